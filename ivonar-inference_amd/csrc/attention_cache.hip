// Attention of a few query rows over the 4-bit cache (layout: cache_layout.hpp).
//
// For a query at position p of its sequence and the keys j <= p, with j > p - window or j < sinks where there is a
// window: x_j = scale * q . k_j, o = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m), in one pass over the keys with a
// running m, sum and o in fp32.  Rows that see no key are zero.
//
// A key/value head is shared by `group` query heads, so its rows are (query token, head of the group), token-major,
// in row tiles of 16 RT.  A wave takes one tile of 32 keys at a time for all rows of the row tile:
//   S^T [key][row]: A = K (converted from 4 bits with its scales in registers, exact in bf16), B = q;
//   P = 2^(x - m), which in the MFMA's result layout is already the B operand of
//   O^T [dim][row] += A = V (converted, then pairs of tokens brought together with v_perm), B = P.
// Nothing of the cache passes through LDS, no register crosses lanes in the loop besides the maxima, and those only
// when some value exceeds the running m by a factor of 2^8 (the exponentials stay below 2^8 until then, which fp32
// and bf16 hold as precisely as values below one).
// q and P are bf16 operands; q in fp16 is split into two bf16 terms and q in fp32 into three (all their bits), and P
// into two or, for fp32 rows, three: a single term of P would leave errors of 2^-8 of sum p |v|, as much as the
// rounding of a bf16 result that does not cancel.
//
// The waves of a block take the tiles of its share of the keys in turn and add their results through LDS; few rows
// and many keys are split over several blocks, whose results (unscaled sums, m, sum) a second kernel adds.
#include "cache_layout.hpp"
#include "ternary_device.hpp"

namespace ivo {
namespace {

constexpr int kWaves = 4;
constexpr float kNoKey = -3.0e38f;  // running maximum before any key
constexpr float kGrowth = 8.0f;

struct Params {
  CacheAttentionArgs a;
  int group;
  int slots;   // row tiles of all sequences (an upper bound), without the slot for rows of no sequence
  int splits;  // blocks that share a row tile's keys
  int chunk;   // key tiles of each of them
  float scale;  // log2(e) * scale
};

// A row tile of a sequence and the key tiles that its rows see: [0, sink_tiles) and [window_tile, end_tile).
struct Span {
  int sequence;
  int row0;        // first row of the sequence in q
  int rows;        // rows of the sequence times group
  int start;       // first row of the row tile
  int first;       // position of the sequence's first query
  int low, high;   // positions of the row tile's first and last rows
  int sink_tiles;
  int window_tile;
  int total;       // key tiles
  __device__ int tile(int i) const { return i < sink_tiles ? i : i - sink_tiles + window_tile; }
};

// Row tile `slot`.  With offsets, sequence b's row tiles are the slots from offsets[b] * group / R + b on, which
// leaves each sequence at least as many as it needs.
template <int R>
__device__ __forceinline__ bool span_of(const Params& p, int slot, Span& s) {
  const CacheAttentionArgs& a = p.a;
  int queries = 1;
  if (a.offsets == nullptr) {
    const int per = (p.group + R - 1) / R;
    s.sequence = slot / per;
    s.start = (slot - s.sequence * per) * R;
    s.row0 = s.sequence;
  } else {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.sequences; base += 64) {
      const int b = base + lane;
      const bool begun = b < a.sequences && (long long)a.offsets[b] * p.group / R + b <= slot;
      before += __popcll(__ballot(begun));
    }
    if (before == 0) return false;
    s.sequence = __builtin_amdgcn_readfirstlane(before - 1);
    s.row0 = a.offsets[s.sequence];
    queries = min(a.offsets[s.sequence + 1], a.rows) - s.row0;
    s.start = (slot - (int)((long long)s.row0 * p.group / R) - s.sequence) * R;
  }
  if (s.sequence >= a.sequences || s.row0 < 0 || queries <= 0) return false;
  s.rows = queries * p.group;
  if (s.start < 0 || s.start >= s.rows) return false;
  // The table's capacity is at most 2^30 tokens, so positions less the window stay within 32 bits.
  const int capacity = (a.table_width << a.page_shift) * kCacheTile;
  const int length = min(max(a.lengths[s.sequence], 0), capacity);
  s.first = length - queries;
  s.low = s.first + s.start / p.group;
  s.high = s.first + (min(s.start + R, s.rows) - 1) / p.group;
  const int end_tile = s.high < 0 ? 0 : s.high / kCacheTile + 1;
  s.window_tile = a.window == 0 || s.low < a.window ? 0 : (s.low - a.window + 1) / kCacheTile;
  s.window_tile = min(s.window_tile, end_tile);
  s.sink_tiles = a.window == 0 ? 0 : min(a.sinks <= 0 ? 0 : (a.sinks - 1) / kCacheTile + 1, s.window_tile);
  s.total = s.sink_tiles + end_tile - s.window_tile;
  return true;
}

// What a lane loads of one tile.
template <int D>
struct Tile {
  static constexpr int W = D / 32, kGroups = W == 8 ? 2 : 1;
  unsigned k[2][W];
  unsigned v[2 * W];
  unsigned k_scale[kGroups];
  uint2 v_scale;
};

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* at, unsigned* to) {
  if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    to[0] = x.x;
    to[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(at + 4 * i);
      to[i] = x.x;
      to[i + 1] = x.y;
      to[i + 2] = x.z;
      to[i + 3] = x.w;
    }
  }
}

template <int D>
__device__ __forceinline__ void load_tile(const uint8_t* base, int lane, Tile<D>& t) {
  constexpr int W = D / 32;
  const int n = lane & 15, b = lane >> 4;
#pragma unroll
  for (int s = 0; s < 2; ++s) load_words<W>(base + (16 * s + n) * (D / 2) + b * (W * 4), t.k[s]);
#pragma unroll
  for (int c = 0; c < W / 2; ++c) load_words<4>(base + 16 * D + c * 1024 + lane * 16, t.v + 4 * c);
  const int k_group = W == 2 ? b >> 1 : W == 4 ? b : 2 * b;
#pragma unroll
  for (int g = 0; g < Tile<D>::kGroups; ++g)
    t.k_scale[g] = *reinterpret_cast<const uint16_t*>(base + 32 * D + (k_group + g) * 32 + n * 2);
  t.v_scale = *reinterpret_cast<const uint2*>(base + 33 * D + (n * W / 16) * 32 + b * 8);
}

// The conversions read the exponent field of the scale operand alone, so a scale byte needs one shift to get there.
__device__ __forceinline__ float scale_operand(unsigned word, int byte) {
  return __uint_as_float(byte == 3 ? word >> 1 : word << (23 - 8 * byte));
}

__device__ __forceinline__ unsigned convert(unsigned word, float scale, int byte) {
  switch (byte) {
    case 0: return bits_as<unsigned>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0));
    case 1: return bits_as<unsigned>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1));
    case 2: return bits_as<unsigned>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2));
    default: return bits_as<unsigned>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3));
  }
}

// x as a sum of NT bf16 terms, x replaced by what is left.
template <int NT>
__device__ __forceinline__ void split_terms(float x, __bf16 (&terms)[NT]) {
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    terms[i] = (__bf16)x;
    if (i + 1 < NT) x -= (float)terms[i];
  }
}

__device__ __forceinline__ float lane_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float lane_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ void store_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_value(Half* p, float x) { p->bits = bits_as<uint16_t>((_Float16)x); }
__device__ __forceinline__ void store_value(Bfloat* p, float x) { p->bits = bits_as<uint16_t>((__bf16)x); }
template <typename Out>
__device__ __forceinline__ void store4(Out* p, const float4& x) {
  store_value(p, x.x);
  store_value(p + 1, x.y);
  store_value(p + 2, x.z);
  store_value(p + 3, x.w);
}

// Zeroes this head's part of the rows that belong to no sequence.
template <int D, typename In>
__device__ __forceinline__ void clear_rows(const Params& p, int head) {
  const CacheAttentionArgs& a = p.a;
  const int begin = a.sequences > 0 ? max(a.offsets[0], 0) : 0;
  const int end = a.sequences > 0 ? a.offsets[a.sequences] : 0;
  In* out = static_cast<In*>(const_cast<void*>(static_cast<const void*>(a.out)));
  const int width = p.group * D;
  for (int row = 0; row < a.rows; ++row) {
    if (row == begin) row = max(end, begin);
    if (row >= a.rows) break;
    In* to = out + ((long long)row * a.heads + (long long)head * p.group) * D;
    for (int i = threadIdx.x; i < width; i += kThreads) store_value(to + i, 0.0f);
  }
}

template <int D, typename In, int RT, int NT>
__global__ __launch_bounds__(kThreads) void cache_attention_kernel(Params p) {
  constexpr int W = D / 32, R = 16 * RT, kTiles = D / 16, kPad = D + 4;
  constexpr int NP = NT < 2 ? 2 : NT;  // terms of a weight
  const CacheAttentionArgs& a = p.a;
  __shared__ float sums[kWaves][16][kPad];
  __shared__ float stats[2][kWaves][R];
  const int lane = threadIdx.x & 63, n = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % a.kv_heads;
  const int unit = blockIdx.x / a.kv_heads;
  const int split = unit % p.splits, slot = unit / p.splits;
  if (slot >= p.slots) {
    if (split == 0) clear_rows<D, In>(p, head);
    return;
  }
  Span s;
  if (!span_of<R>(p, slot, s)) return;
  const int begin = split * p.chunk;
  const int end = split == p.splits - 1 ? s.total : min(s.total, begin + p.chunk);
  if (split > 0 && begin >= end) return;

  // q as the B operand: row n of row tile rt, dims 8 (b W + c) + j.
  bf16x8 q[RT][NT][W];
  int position[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = s.start + rt * 16 + n;
    const bool live = row < s.rows;
    const int token = live ? row / p.group : 0, h = live ? row - token * p.group : 0;
    position[rt] = live ? s.first + token : -1;
    const In* from = static_cast<const In*>(a.q) + (long long)(s.row0 + token) * a.q_strides.token +
                     (long long)(head * p.group + h) * a.q_strides.head + b * (8 * W);
#pragma unroll
    for (int c = 0; c < W; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        __bf16 terms[NT];
        split_terms<NT>(to_float(from[8 * c + j]), terms);
#pragma unroll
        for (int t = 0; t < NT; ++t) q[rt][t][c][j] = terms[t];
      }
  }

  f32x4 o[kTiles][RT];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = kNoKey;
    l[rt] = 0.0f;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i][rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const int* table = a.table + (long long)s.sequence * a.table_width;
  const int page_mask = (1 << a.page_shift) - 1;
  // Tile i of the span: its address, or the first page's where the sequence has no page there.
  auto locate = [&](int i, bool& there) {
    const int tile = s.tile(i);
    const int page = table[tile >> a.page_shift];
    there = (unsigned)page < (unsigned)a.page_count;
    const long long at = ((((long long)(there ? page : 0) * a.kv_heads + head) << a.page_shift) + (tile & page_mask));
    return a.pages + at * cache_tile_bytes(D);
  };

  Tile<D> next;
  bool next_there = false;
  int i = begin + wave;
  if (i < end) load_tile<D>(locate(i, next_there), lane, next);
  for (; i < end; i += kWaves) {
    const Tile<D> t = next;
    const bool there = next_there;
    if (i + kWaves < end) load_tile<D>(locate(i + kWaves, next_there), lane, next);
    if (!there) continue;

    const int key0 = s.tile(i) * kCacheTile;
    f32x4 x[2][RT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) x[h][rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const float scale = scale_operand(t.k_scale[W == 8 ? c / 4 : 0], h);
        u32x4 words;
#pragma unroll
        for (int j = 0; j < 4; ++j) words[j] = convert(t.k[h][c], scale, j);
        const bf16x8 key = bits_as<bf16x8>(words);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int z = 0; z < NT; ++z)
            x[h][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, q[rt][z][c], x[h][rt], 0, 0, 0);
      }
    }

    uint2 v_scale = t.v_scale;
    const bool whole = key0 + kCacheTile - 1 <= s.low &&
                       (a.window == 0 || key0 > s.high - a.window || key0 + kCacheTile <= a.sinks);
    unsigned hidden = 0;  // bit e: the scale of the lane's token e stands for no number
    if (!whole) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = key0 + 16 * h + 4 * b + r;
            const bool seen = key <= position[rt] &&
                              (a.window == 0 || key > position[rt] - a.window || key < a.sinks);
            x[h][rt][r] = seen ? x[h][rt][r] : -INFINITY;
          }
      // A weight of zero times a value that is no number would be no number: such scales become one here, and the
      // rows that do see them get their NaN below.  Scales above kScaleMax are never written, but unwritten bytes
      // may hold them.
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        unsigned& word = e < 4 ? v_scale.x : v_scale.y;
        const int shift = 8 * (e & 3);
        if (((word >> shift) & 255u) > (unsigned)kScaleMax) {
          hidden |= 1u << e;
          word = (word & ~(255u << shift)) | (127u << shift);
        }
      }
    }

    float most[RT];
    bool grows = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const f32x4 u = x[0][rt], w = x[1][rt];
      most[rt] = fmaxf(fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])), fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]))) * p.scale;
      grows |= most[rt] > m[rt] + kGrowth;
    }
    if (__ballot(grows) != 0ull) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        // Only the rows that grow: a row's rounding does not depend on its neighbours.
        const float highest = lane_groups_max(most[rt]);
        const float raised = highest > m[rt] + kGrowth ? highest : m[rt];
        const float factor = __builtin_amdgcn_exp2f(m[rt] - raised);
        m[rt] = raised;
        l[rt] *= factor;
#pragma unroll
        for (int k = 0; k < kTiles; ++k) o[k][rt] *= factor;
      }
    }

    bf16x8 weights[RT][NP];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float sum = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float w = __builtin_amdgcn_exp2f(fmaf(x[h][rt][r], p.scale, -m[rt]));
          sum += w;
          __bf16 terms[NP];
          split_terms<NP>(w, terms);
#pragma unroll
          for (int z = 0; z < NP; ++z) weights[rt][z][4 * h + r] = terms[z];
        }
      l[rt] += sum;
    }

#pragma unroll
    for (int w = 0; w < W; ++w) {
      unsigned pairs[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        constexpr int kPer = 16 / W;
        const int byte = (e % kPer) * W + w;
        pairs[e] = convert(t.v[(e / kPer) * 4 + byte / 4], scale_operand(e < 4 ? v_scale.x : v_scale.y, e & 3),
                           byte & 3);
      }
      u32x4 even, odd;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        even[e] = __builtin_amdgcn_perm(pairs[2 * e + 1], pairs[2 * e], 0x05040100u);
        odd[e] = __builtin_amdgcn_perm(pairs[2 * e + 1], pairs[2 * e], 0x07060302u);
      }
      const bf16x8 value0 = bits_as<bf16x8>(even), value1 = bits_as<bf16x8>(odd);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int z = 0; z < NP; ++z) {
          o[2 * w][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value0, weights[rt][z], o[2 * w][rt], 0, 0, 0);
          o[2 * w + 1][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value1, weights[rt][z], o[2 * w + 1][rt], 0, 0, 0);
        }
    }

    if (!whole && __ballot(hidden != 0u) != 0ull) {
      // How many tokens without a number each row sees, per 2 W dims: the product of the flags and the visibility.
      bf16x8 flags;
#pragma unroll
      for (int e = 0; e < 8; ++e) flags[e] = (__bf16)((hidden >> e) & 1u ? 1.0f : 0.0f);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        bf16x8 seen;
#pragma unroll
        for (int e = 0; e < 8; ++e) seen[e] = (__bf16)(x[e / 4][rt][e & 3] == -INFINITY ? 0.0f : 1.0f);
        f32x4 count = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(flags, seen, count, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (count[r] > 0.0f)
#pragma unroll
            for (int k = 0; k < kTiles; ++k) o[k][rt][r] = NAN;
      }
    }
  }

  // The waves' results, relative to the block's maximum of each row, added in the waves' order.
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] = lane_groups_sum(l[rt]);
    if (b == 0) {
      stats[0][wave][rt * 16 + n] = m[rt];
      stats[1][wave][rt * 16 + n] = l[rt];
    }
  }
  __syncthreads();
  const long long part = ((long long)slot * a.kv_heads + head) * p.splits + split;
  float* sums_out = a.work + part * (R * (D + 2));
  float* stats_out = sums_out + R * D;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float highest = kNoKey;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) highest = fmaxf(highest, stats[0][w][rt * 16 + n]);
    const float factor = __builtin_amdgcn_exp2f(m[rt] - highest);
    if (rt > 0) __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int k = 0; k < kTiles; ++k) sums[wave][n][kTiles * (4 * b + r) + k] = o[k][rt][r] * factor;
    __syncthreads();
    for (int at = threadIdx.x; at < 16 * D / 4; at += kThreads) {
      const int line = at / (D / 4), column = at % (D / 4) * 4;
      const int row = s.start + rt * 16 + line;
      if (row >= s.rows) continue;
      float top = kNoKey, total = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[0][w][rt * 16 + line]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        total += stats[1][w][rt * 16 + line] * __builtin_amdgcn_exp2f(stats[0][w][rt * 16 + line] - top);
      float4 sum = float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(&sums[w][line][column]);
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      if (p.splits == 1) {
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        const int token = row / p.group, h = row - token * p.group;
        In* to = static_cast<In*>(a.out) + ((long long)(s.row0 + token) * a.heads + head * p.group + h) * D + column;
        store4(to, float4{sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse});
      } else {
        *reinterpret_cast<float4*>(sums_out + (rt * 16 + line) * D + column) = sum;
        if (column == 0) {
          stats_out[2 * (rt * 16 + line)] = top;
          stats_out[2 * (rt * 16 + line) + 1] = total;
        }
      }
    }
  }
}

// Adds the parts of a row in their order: a wave per row, D / 64 dims per lane.
template <int D, typename In, int R>
__global__ __launch_bounds__(kThreads) void merge_kernel(Params p) {
  constexpr int kDims = D / 64;
  const CacheAttentionArgs& a = p.a;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long id = (long long)blockIdx.x * kWaves + wave;
  const int line = (int)(id % R);
  const long long unit = id / R;
  const int head = (int)(unit % a.kv_heads), slot = (int)(unit / a.kv_heads);
  Span s;
  if (slot >= p.slots || !span_of<R>(p, slot, s)) return;
  const int row = s.start + line;
  if (row >= s.rows) return;
  const int parts = max(1, min(p.splits, (s.total + p.chunk - 1) / p.chunk));
  const float* from = a.work + unit * p.splits * (R * (D + 2));
  float top = kNoKey;
  for (int i = 0; i < parts; ++i) top = fmaxf(top, from[(long long)i * (R * (D + 2)) + R * D + 2 * line]);
  float total = 0.0f, sum[kDims] = {};
  for (int i = 0; i < parts; ++i) {
    const float* part = from + (long long)i * (R * (D + 2));
    const float factor = __builtin_amdgcn_exp2f(part[R * D + 2 * line] - top);
    total += part[R * D + 2 * line + 1] * factor;
#pragma unroll
    for (int k = 0; k < kDims; ++k) sum[k] += part[line * D + lane * kDims + k] * factor;
  }
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
  const int token = row / p.group, h = row - token * p.group;
  In* to = static_cast<In*>(a.out) + ((long long)(s.row0 + token) * a.heads + head * p.group + h) * D + lane * kDims;
#pragma unroll
  for (int k = 0; k < kDims; ++k) store_value(to + k, sum[k] * inverse);
}

// Row tiles per wave: as many as the sequences' rows fill on average, within the registers.
int row_tiles(const CacheAttentionArgs& a) {
  const long long rows = (long long)a.rows * (a.heads / a.kv_heads) / (a.sequences > 0 ? a.sequences : 1);
  if (rows <= 16 || (a.head_dim == 256 && a.dtype != kBfloat16)) return 1;
  if (rows <= 32 || a.head_dim == 256 || a.dtype == kFloat32) return 2;
  return 4;
}

Params plan(const CacheAttentionArgs& a) {
  Params p{a, a.heads / a.kv_heads, 0, 1, 1, 1.44269504088896340736f * a.scale};
  const int R = 16 * row_tiles(a);
  const long long rows = (long long)a.rows * p.group;
  p.slots = (int)(a.offsets == nullptr ? (long long)a.sequences * ((p.group + R - 1) / R) : rows / R + a.sequences);
  // Key tiles that a row tile sees at most, in shares of at least kLeastTiles such that about kBlocks blocks run.
  constexpr long long kBlocks = 1024, kLeastTiles = 16;
  long long keys = a.max_length;
  if (a.window > 0) keys = min(keys, (long long)a.window + (R + p.group - 1) / p.group + a.sinks + 2 * kCacheTile);
  const long long tiles = max(1LL, (keys + kCacheTile - 1) / kCacheTile);
  const long long live = a.offsets == nullptr ? p.slots : min((long long)p.slots, rows / R + (rows % R > 0) + a.sequences / 2);
  const long long wanted = max(1LL, kBlocks / max(1LL, live * a.kv_heads));
  p.chunk = (int)max(kLeastTiles, (tiles + wanted - 1) / wanted);
  p.splits = (int)((tiles + p.chunk - 1) / p.chunk);
  return p;
}

template <int D, typename In, int RT, int NT>
hipError_t run(hipStream_t stream, const Params& p) {
  const long long blocks = (long long)(p.slots + (p.a.offsets != nullptr ? 1 : 0)) * p.splits * p.a.kv_heads;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((cache_attention_kernel<D, In, RT, NT>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
  if (p.splits > 1) {
    const long long merges = (long long)p.slots * p.a.kv_heads * (16 * RT) / kWaves;
    if (merges > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL((merge_kernel<D, In, 16 * RT>), dim3((unsigned)merges), dim3(kThreads), 0, stream, p);
  }
  return hipGetLastError();
}

template <int D>
hipError_t run_types(hipStream_t stream, const Params& p) {
  const int tiles = row_tiles(p.a);
  if (p.a.dtype == kFloat32) {
    if constexpr (D < 256)
      if (tiles == 2) return run<D, float, 2, 3>(stream, p);
    return run<D, float, 1, 3>(stream, p);
  }
  if (p.a.dtype == kFloat16) {
    if constexpr (D < 256) {
      if (tiles == 4) return run<D, Half, 4, 2>(stream, p);
      if (tiles == 2) return run<D, Half, 2, 2>(stream, p);
    }
    return run<D, Half, 1, 2>(stream, p);
  }
  if constexpr (D < 256)
    if (tiles == 4) return run<D, Bfloat, 4, 1>(stream, p);
  if (tiles == 2) return run<D, Bfloat, 2, 1>(stream, p);
  return run<D, Bfloat, 1, 1>(stream, p);
}

}  // namespace

long long cache_attention_work(const CacheAttentionArgs& a) {
  const Params p = plan(a);
  if (p.splits == 1) return 0;
  return (long long)p.slots * a.kv_heads * p.splits * (16 * row_tiles(a)) * (a.head_dim + 2) * 4;
}

hipError_t launch_cache_attention(hipStream_t stream, const CacheAttentionArgs& a) {
  if (a.rows == 0) return hipSuccess;
  const Params p = plan(a);
  if (a.head_dim == 64) return run_types<64>(stream, p);
  if (a.head_dim == 128) return run_types<128>(stream, p);
  return run_types<256>(stream, p);
}

}  // namespace ivo
