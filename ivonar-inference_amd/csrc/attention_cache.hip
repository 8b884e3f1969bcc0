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
// A wave's tiles come straight from memory into a ring of its own in LDS, three of them (64 dims), two (128) or one
// (256) on their way while one is used, so no barrier stands in the loop.  No register crosses lanes in it besides the
// maxima, and those only when some value exceeds the running m by a factor of 2^8 (the exponentials stay below 2^8
// until then, which fp32 and bf16 hold as precisely as values below one).
// q and P are bf16 operands; q in fp16 is split into two bf16 terms and q in fp32 into three (all their bits), and P
// into two or, for fp32 rows, three: a single term of P would leave errors of 2^-8 of sum p |v|, as much as the
// rounding of a bf16 result that does not cancel.
//
// The waves of a block take the tiles of its share of the keys in turn and add their results through LDS.  Up to 8 rows
// per sequence: the keys of all sequences are dealt out evenly to as many blocks as the device holds; where that cuts a
// row tile's keys, the last of its blocks to end adds the parts (unscaled sums, m, sum).  More rows: row tiles are
// split at equal lengths where there are too few of them, and a second kernel adds their parts.
//
// Measured (MI355X, calls back to back).  One token per sequence, bound by the cache's bytes: 64 sequences of 1000 to
// 8000 tokens (288000 in all), 32/8 heads of 128, bf16: 67 us, 4.7 TB/s (a stream of the same 313 MB reads at 6.5;
// loads alone took 64); one of 131000, fp16: 36.5 us, 3.9 TB/s (142 MB more take 23 us more: the rest is filling the
// device and adding the parts); 128 with a window of 1024, 16/4 heads of 64: 15.2 us, 2.4 TB/s; one of 37, fp32: 6.4 us
// in a graph, a chain of loads.  Chunks, bound by the vector units, which convert the codes and the weights next to the
// matrix units' work: 512 rows over 8702 tokens, 32/8 heads of 128, bf16: 120 us, 590 TFLOP/s (890 counting both terms
// of P); fp16 142 us, fp32 223 us, with more terms of q and P.
#include "buffer_ops.hpp"
#include "cache_layout.hpp"
#include "ternary_device.hpp"

namespace ivo {
namespace {

constexpr int kWaves = 4;
constexpr float kNoKey = -3.0e38f;  // running maximum before any key
constexpr float kGrowth = 8.0f;
constexpr float kFar = 0x1p24f;  // from here on a maximum, x * scale, may be rounded by one and more

struct Params {
  CacheAttentionArgs a;
  int group;
  int slots;     // row tiles of all sequences (an upper bound)
  int splits;    // blocks that share a row tile's keys; 0: the keys of all row tiles are dealt out to `blocks` blocks
  int chunk;     // key tiles of a split, or the least that a block takes of all
  int blocks;    // of each head
  float scale;   // log2(e) * scale
  float inverse;
  bool aligned;  // q's rows start on 16 bytes
  bool stream;   // the cache is loaded past the memory-side cache
  unsigned* counters;  // of dealt out row tiles, by their first block: the parts that have arrived
};

// A row tile of a sequence and the key tiles that its rows see: [0, sink_tiles) and [window_tile, ..), at least one.
struct Span {
  int sequence;
  int row0;       // first row of the sequence in q
  int rows;       // rows of the sequence times group
  int start;      // first row of the row tile
  int first;      // position of the sequence's first query
  int low, high;  // positions of the row tile's first and last rows
  int sink_tiles;
  int window_tile;
  int total;      // key tiles
  __device__ int tile(int i) const { return i < sink_tiles ? i : i - sink_tiles + window_tile; }
};

template <int R>
__device__ __forceinline__ Span make_span(const Params& p, int sequence, int row0, int queries, int length, int start) {
  const CacheAttentionArgs& a = p.a;
  Span s;
  s.sequence = sequence;
  s.row0 = row0;
  s.rows = queries * p.group;
  s.start = start;
  // Rows, the window and the table's tokens are at most 2^30, so positions less any of them stay within 32 bits.
  s.first = max(length, 0) - queries;
  s.low = s.first + start / p.group;
  s.high = s.first + (min(start + R, s.rows) - 1) / p.group;
  // Rows may lie past the table, which has no page for what they see there.
  const int end_tile = s.high < 0 ? 0 : min(s.high / kCacheTile + 1, a.table_width << a.page_shift);
  s.window_tile = a.window == 0 || s.low < a.window ? 0 : (s.low - a.window + 1) / kCacheTile;
  s.window_tile = min(s.window_tile, max(end_tile - 1, 0));
  s.sink_tiles = a.window == 0 ? 0 : min(a.sinks <= 0 ? 0 : (a.sinks - 1) / kCacheTile + 1, s.window_tile);
  s.total = max(1, s.sink_tiles + end_tile - s.window_tile);
  return s;
}

// First row of a sequence and its rows, none where the offsets do not make sense.
__device__ __forceinline__ int rows_of(const CacheAttentionArgs& a, int sequence, int& row0) {
  if (a.offsets == nullptr) {
    row0 = sequence;
    return 1;
  }
  row0 = a.offsets[sequence];
  return row0 < 0 ? 0 : max(0, min(a.offsets[sequence + 1], a.rows) - row0);
}

// Row tile `slot`.  With offsets, sequence b's row tiles are the slots from offsets[b] * group / R + b on, which
// leaves each sequence at least as many as it needs.
template <int R>
__device__ __forceinline__ bool span_of(const Params& p, int slot, Span& s) {
  const CacheAttentionArgs& a = p.a;
  int sequence, start;
  if (a.offsets == nullptr) {
    const int per = (p.group + R - 1) / R;
    sequence = slot / per;
    start = (slot - sequence * per) * R;
  } else {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.sequences; base += 64) {
      const int b = base + lane;
      const bool begun = b < a.sequences && (long long)a.offsets[b] * p.group / R + b <= slot;
      before += __popcll(__ballot(begun));
    }
    if (before == 0) return false;
    sequence = __builtin_amdgcn_readfirstlane(before - 1);
    start = (slot - (int)((long long)a.offsets[sequence] * p.group / R) - sequence) * R;
  }
  if (sequence >= a.sequences) return false;
  int row0;
  const int queries = rows_of(a, sequence, row0);
  if (start < 0 || start >= queries * p.group) return false;
  s = make_span<R>(p, sequence, row0, queries, a.lengths[sequence], start);
  return true;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The key tiles of all sequences in a row: sequence by sequence, its row tiles in order.  A block takes `share`
// neighbouring ones of them for one head, so that blocks end together whatever the lengths are, and the heads' blocks,
// which start together, read the heads' parts of a page at about the same time.
template <int R>
__device__ __forceinline__ long long tiles_of(const Params& p, int sequence) {
  if (sequence >= p.a.sequences) return 0;
  int row0;
  const int queries = rows_of(p.a, sequence, row0), length = p.a.lengths[sequence];
  long long tiles = 0;
  for (int start = 0; start < queries * p.group; start += R)
    tiles += make_span<R>(p, sequence, row0, queries, length, start).total;
  return tiles;
}
__device__ __forceinline__ long long uniform(long long v) {
  const unsigned low = (unsigned)uniform((int)v);
  return (long long)((unsigned long long)(unsigned)uniform((int)(v >> 32)) << 32 | low);
}
// Tiles of the sequences before `upto`.  All lanes of a wave call this together.
template <int R>
__device__ __forceinline__ long long tiles_before(const Params& p, int upto) {
  long long sum = 0;
  for (int b = threadIdx.x & 63; b < upto; b += 64) sum += tiles_of<R>(p, b);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  return uniform(sum);
}
__device__ __forceinline__ long long share_of(const Params& p, long long all) {
  return max((long long)p.chunk, (all + p.blocks - 1) / p.blocks);
}

// What a lane loads of one tile.
template <int D>
struct Tile {
  static constexpr int W = D / 32;
  unsigned k[2 * W];
  unsigned v[2 * W];
  unsigned k_scale[2];
  uint2 v_scale;
};

// A tile on its way from memory to LDS, straight: its 34 D bytes side by side (at D = 64 a dword load of all lanes
// reaches 128 bytes past them, which the buffer's end turns into zeros).
template <int D>
struct Stage {
  static constexpr int kCodeLoads = 32 * D / 1024, kScaleLoads = D == 256 ? 2 : 1;
  static constexpr int kLoads = kCodeLoads + kScaleLoads;
  unsigned char codes[32 * D];
  unsigned char scales[256 * kScaleLoads];
};
template <int D, bool STREAM>
__device__ __forceinline__ void load_tile(const uint8_t* base, unsigned to, int lane) {
  const v4u buffer = wide_buffer(base, cache_tile_bytes(D));
#pragma unroll
  for (int j = 0; j < Stage<D>::kCodeLoads; j += 2)
    dma_pair<STREAM>(buffer, to + j * 1024, 1024, lane * 16, lane * 16, j * 1024, 1024);
#pragma unroll
  for (int j = 0; j < Stage<D>::kScaleLoads; ++j)
    dma4<STREAM>(buffer, to + 32 * D + j * 256, lane * 4, 32 * D + j * 256);
}

template <int N>
__device__ __forceinline__ void read_words(const unsigned char* at, unsigned* to) {
  if constexpr (N == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(at);
    to[0] = x[0];
    to[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(at + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) to[i + j] = x[j];
    }
  }
}

// A lane's keys and values of a tile in LDS.  Of up to 8 rows (NARROW) lane (n, b) takes half a row of key
// 16 (b / 2) + n, else a quarter of the rows of keys n and 16 + n.
template <int D, bool NARROW>
__device__ __forceinline__ void read_tile(const unsigned char* base, int lane, Tile<D>& t) {
  constexpr int W = D / 32;
  const int n = lane & 15, b = lane >> 4;
  if constexpr (NARROW) {
    read_words<2 * W>(base + (16 * (b >> 1) + n) * (D / 2) + (b & 1) * (D / 4), t.k);
#pragma unroll
    for (int g = 0; g < W / 2; ++g) t.k_scale[g] = base[32 * D + ((b & 1) * (W / 2) + g) * 32 + n * 2 + (b >> 1)];
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) read_words<W>(base + (16 * h + n) * (D / 2) + b * (W * 4), t.k + h * W);
    const int group = W == 2 ? b >> 1 : W == 4 ? b : 2 * b;
#pragma unroll
    for (int g = 0; g < (W == 8 ? 2 : 1); ++g)
      t.k_scale[g] = *reinterpret_cast<const uint16_t*>(base + 32 * D + (group + g) * 32 + n * 2);
  }
#pragma unroll
  for (int c = 0; c < W / 2; ++c) read_words<4>(base + 16 * D + c * 1024 + lane * 16, t.v + 4 * c);
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

// The lane 8 further on (or back) of the same 16.
__device__ __forceinline__ unsigned other_half(unsigned v) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, false);  // row_ror:8
}
__device__ __forceinline__ float other_half(float v) { return __uint_as_float(other_half(__float_as_uint(v))); }

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
  In* out = static_cast<In*>(a.out);
  const int width = p.group * D;
  for (int row = 0; row < a.rows; ++row) {
    if (row == begin) row = max(end, begin);
    if (row >= a.rows) break;
    In* to = out + ((long long)row * a.heads + (long long)head * p.group) * D;
    for (int i = threadIdx.x; i < width; i += kThreads) store_value(to + i, 0.0f);
  }
}

// Blocks of 4 waves per CU that the registers leave room for (waves per SIMD).
constexpr int occupancy(int D, int R, int NT) {
  if (R == 8) return D == 128 ? (NT == 1 ? 3 : 2) : NT == 1 ? 4 : 3;
  if (R <= 16) return D == 64 ? (NT == 3 ? 3 : 4) : D == 128 ? (NT == 3 ? 2 : 3) : NT == 3 ? 1 : 2;
  return D == 256 || (D == 128 && NT == 3) ? 1 : D == 64 && NT == 1 ? 3 : 2;
}

// Tiles in a wave's ring: as many as that number of blocks leaves room for in a CU's 160 KB.
constexpr int stages(int D) { return D == 64 ? 4 : D == 128 ? 3 : 2; }

// Tiles of the sequences base .. base + 63, in the lanes, summed up to and including each lane's.
template <int R>
__device__ __forceinline__ long long tiles_up_to(const Params& p, int base) {
  const int lane = threadIdx.x & 63;
  long long sum = tiles_of<R>(p, base + lane);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long lower = __shfl_up(sum, o);
    if (lane >= o) sum += lower;
  }
  return sum;
}

// A run of key tiles of one row tile: tiles begin .. of the row tile at row `start` of the sequence.
struct Run {
  int sequence, start, begin;
  long long at;  // the run's first tile among all of them
};

// Where a share of all key tiles begins, and how many tiles it has.
template <int R>
__device__ __forceinline__ bool share_begin(const Params& p, int block, Run& run, long long& left, long long& share) {
  const CacheAttentionArgs& a = p.a;
  long long sum = tiles_up_to<R>(p, 0);
  const long long all = a.sequences <= 64 ? uniform(__shfl(sum, 63)) : tiles_before<R>(p, a.sequences);
  share = share_of(p, all);
  long long at = block * share;
  if (at >= all) return false;
  run.at = at;
  left = min(share, all - at);
  int base = 0;
  for (;;) {
    const long long here = uniform(__shfl(sum, 63));
    if (at < here) break;
    at -= here;
    base += 64;
    sum = tiles_up_to<R>(p, base);
  }
  const int found = __builtin_ctzll(__ballot(sum > at));
  if (found > 0) at -= uniform(__shfl(sum, found - 1));
  run.sequence = base + found;
  int row0;
  const int queries = rows_of(a, run.sequence, row0), length = a.lengths[run.sequence];
  for (run.start = 0;; run.start += R) {
    const int total = make_span<R>(p, run.sequence, row0, queries, length, run.start).total;
    if (at < total) {
      run.begin = (int)at;
      return true;
    }
    at -= total;
  }
}

// Adds the parts of a row (sums relative to a part's maximum, and the maximum and sum of the weights): a thread takes
// four dims and every `groups`-th part of them, in their order, several on their way at a time.  `first`, then `second`
// and from there on `step` apart: the parts' numbers.
constexpr int kDeviceScope = 16;  // SC1, the scope bit of store_device and load_device, of the wide buffer forms
__device__ __forceinline__ __amdgpu_buffer_rsrc_t parts_buffer(float* work) {
  return __builtin_amdgcn_make_buffer_rsrc(work, 0, 0x7fffffff, 0x00020000);
}
struct RowSum {
  float4 sum;
  float top, total;
};
__device__ __forceinline__ void add_scaled(RowSum& to, const float4& v, float factor) {
  to.sum.x += v.x * factor;
  to.sum.y += v.y * factor;
  to.sum.z += v.z * factor;
  to.sum.w += v.w * factor;
}
template <int D, int R>
__device__ __forceinline__ RowSum add_row(int line, int lane, int groups, int group, __amdgpu_buffer_rsrc_t work,
                                          long long first, long long second, int step, int parts) {
  constexpr int kPart = R * (D + 2), kAtOnce = 8;
  RowSum to{float4{0.0f, 0.0f, 0.0f, 0.0f}, kNoKey, 0.0f};
  for (int base = group; base < parts; base += groups * kAtOnce) {
    float2 stats[kAtOnce];
    float4 values[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = min(base + k * groups, parts - 1);
      const int at = (int)(i == 0 ? first : second + (i - 1) * step) * kPart * 4;
      stats[k] = bits_as<float2>(
          (u32x2)__builtin_amdgcn_raw_buffer_load_b64(work, at + (R * D + 2 * line) * 4, 0, kDeviceScope));
      values[k] = bits_as<float4>(
          (u32x4)__builtin_amdgcn_raw_buffer_load_b128(work, at + (line * D + lane * 4) * 4, 0, kDeviceScope));
    }
    float top = to.top;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) top = fmaxf(top, stats[k].x);
    const float before = __builtin_amdgcn_exp2f(to.top - top);
    to = RowSum{float4{to.sum.x * before, to.sum.y * before, to.sum.z * before, to.sum.w * before}, top,
                to.total * before};
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      // Without a branch, behind which the compiler would load each part by itself.
      const bool live = base + k * groups < parts;
      const float factor = __builtin_amdgcn_exp2f(stats[k].x - top);
      to.total += live ? stats[k].y * factor : 0.0f;
      to.sum.x += live ? values[k].x * factor : 0.0f;
      to.sum.y += live ? values[k].y * factor : 0.0f;
      to.sum.z += live ? values[k].z * factor : 0.0f;
      to.sum.w += live ? values[k].w * factor : 0.0f;
    }
  }
  return to;
}
template <int D, typename In>
__device__ __forceinline__ void store_row(const Params& p, const Span& s, int head, int line, int lane,
                                          const RowSum& from) {
  const float inverse = from.total == 0.0f ? 0.0f : 1.0f / from.total;
  const float4 sum = from.sum;
  const int row = s.start + line, token = row / p.group, h = row - token * p.group;
  In* to = static_cast<In*>(p.a.out) + ((long long)(s.row0 + token) * p.a.heads + head * p.group + h) * D + lane * 4;
  store4(to, float4{sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse});
}

// All rows of a row tile by one block: D / 4 threads per row and group of parts.  room: 6 floats per thread.
template <int D, typename In, int R>
__device__ __forceinline__ void add_parts(const Params& p, const Span& s, int head, __amdgpu_buffer_rsrc_t work,
                                          long long first, long long second, int step, int parts, float* room) {
  constexpr int kLanes = D / 4, kTeams = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, team = (int)threadIdx.x / kLanes;
  const int rows = min(R, s.rows - s.start);
  // Teams per row, a power of two, as many as parts can use.
  int groups = 1;
  while (groups * 2 * rows <= kTeams && groups * 2 <= parts) groups *= 2;
  float4* sums = reinterpret_cast<float4*>(room);
  float2* stats = reinterpret_cast<float2*>(room + 4 * kThreads);
  for (int base = 0; base < rows; base += kTeams / groups) {
    const int line = min(base + team / groups, rows - 1), group = team % groups;
    const RowSum mine = add_row<D, R>(line, lane, groups, group, work, first, second, step, parts);
    __syncthreads();
    sums[threadIdx.x] = mine.sum;
    stats[threadIdx.x] = float2{mine.top, mine.total};
    __syncthreads();
    if (group == 0 && base + team / groups < rows) {
      float top = mine.top;
      for (int k = 1; k < groups; ++k) top = fmaxf(top, stats[threadIdx.x + k * kLanes].x);
      RowSum all{float4{0.0f, 0.0f, 0.0f, 0.0f}, top, 0.0f};
      for (int k = 0; k < groups; ++k) {
        const float2 part = stats[threadIdx.x + k * kLanes];
        const float factor = __builtin_amdgcn_exp2f(part.x - top);
        all.total += part.y * factor;
        add_scaled(all, sums[threadIdx.x + k * kLanes], factor);
      }
      store_row<D, In>(p, s, head, line, lane, all);
    }
  }
}

template <int D, typename In, int R, int NT, bool STREAM>
__global__ __launch_bounds__(kThreads, occupancy(D, R, NT)) void cache_attention_kernel(Params p) {
  static_assert(R != 8 || D < 256, "up to 8 rows, a lane has two scales of K at most");
  constexpr bool kNarrow = R == 8;
  constexpr int RT = kNarrow ? 1 : R / 16, kHalves = kNarrow ? 1 : 2;
  constexpr int W = D / 32, kChunks = kNarrow ? 2 * W : W, kTiles = D / 16, kPad = D + 4;
  constexpr int NP = NT < 2 ? 2 : NT;  // terms of a weight
  const CacheAttentionArgs& a = p.a;
  // A ring of stages per wave, and at the end of a run the waves' sums.
  constexpr int kStages = stages(D);
  union Room {
    Stage<D> ring[kWaves][kStages];
    float sums[kWaves][16][kPad];
  };
  __shared__ __align__(16) unsigned char room_bytes[sizeof(Room)];
  Room& room = *reinterpret_cast<Room*>(room_bytes);
  auto& sums = room.sums;
  __shared__ float stats[2][kWaves][16 * RT];
  __shared__ unsigned arrived;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Keys are dealt out for up to kFewRows rows, which take the smallest row tiles of their head size.
  constexpr bool kDealt = R == 8 || (D == 256 && R == 16);
  const bool shared = kDealt && p.splits == 0;

  // The block's runs of tiles: one, or as many as its share of all tiles has; and where the first one's result goes.
  Run run;
  long long left = 0, share = 0;
  long long part;
  const int head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
  if (shared) {
    if (unit >= p.blocks) {
      clear_rows<D, In>(p, head);
      return;
    }
    if (!share_begin<R>(p, unit, run, left, share)) return;
    part = 2LL * unit * a.kv_heads + head;
  } else {
    const int split = unit % p.splits, slot = unit / p.splits;
    if (slot >= p.slots) {
      if (split == 0) clear_rows<D, In>(p, head);
      return;
    }
    Span s;
    if (!span_of<R>(p, slot, s)) return;
    run.sequence = s.sequence;
    run.start = s.start;
    run.begin = split * p.chunk;
    left = split == p.splits - 1 ? s.total - run.begin : min(s.total - run.begin, p.chunk);
    if (left <= 0) return;
    part = ((long long)slot * p.splits + split) * a.kv_heads + head;
  }

  for (;;) {
    int row0;
    const int sequence = uniform(run.sequence), begin = uniform(run.begin);
    const int queries = uniform(rows_of(a, sequence, row0)), length = a.lengths[sequence];
    const Span s = make_span<R>(p, sequence, uniform(row0), queries, length, uniform(run.start));
    const int end = begin + (int)min((long long)(s.total - begin), uniform(left));
    // Opaque to the compiler, which would otherwise compute every address of the loop's body ahead of it, and hold
    // them in registers throughout.
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, n = lane & 15, b = lane >> 4;
    // In the constant address space, so that pages are looked up by scalar loads: the wait for a vector load would be
    // a wait for every tile under way.
    typedef const __attribute__((address_space(4))) int* Constants;
    const Constants table = (Constants)(uintptr_t)(a.table + (long long)s.sequence * a.table_width);
    const int page_mask = (1 << a.page_shift) - 1;
    // Page of tile i of the span.
    auto page_of = [&](int i) { return table[s.tile(i) >> a.page_shift]; };
    // Begins to load tile i, or the first page's where the sequence has no page there.
    auto load = [&](int i, int page, int stage) {
      const bool there = (unsigned)page < (unsigned)a.page_count;
      const long long at =
          (((long long)(there ? page : 0) * a.kv_heads + head) << a.page_shift) + (s.tile(i) & page_mask);
      load_tile<D, STREAM>(a.pages + at * cache_tile_bytes(D), lds_address(&room.ring[wave][stage]), lane);
      return there;
    };

    // A wave takes every fourth tile, and has up to kStages - 1 of them under way from memory to its ring.
    int i = begin + wave;
    const int last = i < end ? i + (end - 1 - i) / kWaves * kWaves : i;
    unsigned there = 0;  // bit k: the tile k turns ahead has a page
    int page = 0;        // of the next tile to load
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k)
      if (i + k * kWaves <= last && i < end) there |= (unsigned)load(i + k * kWaves, page_of(i + k * kWaves), k) << k;
    if (i < end) page = page_of(min(i + (kStages - 1) * kWaves, last));
    int stage = 0;
    // q as the B operand.  Row n of row tile rt, dims 8 (b W + c) + j; of up to 8 rows, row n % 8 and dims
    // (b % 2) D / 2 + 8 c + j, where the keys b / 2 = n / 8, and zero elsewhere: columns 0 .. 7 of the product are then
    // the rows with the tile's first 16 keys, columns 8 .. 15 with its others, so every lane has logits of its own.
    bf16x8 q[RT][NT][kChunks];
    int position[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = s.start + rt * 16 + (kNarrow ? n & 7 : n);
      const bool live = row < s.rows, mine = !kNarrow || b >> 1 == n >> 3;
      const int token = live ? row / p.group : 0, h = live ? row - token * p.group : 0;
      position[rt] = live ? s.first + token : -1;
      const In* from = static_cast<const In*>(a.q) + (long long)(s.row0 + token) * a.q_strides.token +
                       (long long)(head * p.group + h) * a.q_strides.head + (kNarrow ? b & 1 : b) * (8 * kChunks);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        float x[8];
        load8(from + 8 * c, p.aligned, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          __bf16 terms[NT];
          split_terms<NT>(mine ? x[j] : 0.0f, terms);
#pragma unroll
          for (int z = 0; z < NT; ++z) q[rt][z][c][j] = terms[z];
        }
      }
    }

    f32x4 o[kTiles][RT];
    float m[RT], l[RT];
    bool far = false;  // some row's maximum is
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = kNoKey;
      l[rt] = 0.0f;
#pragma unroll
      for (int k = 0; k < kTiles; ++k) o[k][rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (; i < end; i += kWaves) {
      // This tile has arrived when only the ones after it are under way; towards the end there are fewer of those.
      if (i + (kStages - 2) * kWaves <= last)
        wait_loads<(kStages - 2) * Stage<D>::kLoads>();
      else
        wait_loads<0>();
      // The stage of the tile before this one, which has been used, takes the next tile.
      if (i + (kStages - 1) * kWaves <= last) {
        const int free = stage == 0 ? kStages - 1 : stage - 1;
        there |= (unsigned)load(i + (kStages - 1) * kWaves, page, free) << (kStages - 1);
        page = page_of(min(i + kStages * kWaves, last));
      }
      Tile<D> t;
      read_tile<D, kNarrow>(reinterpret_cast<const unsigned char*>(&room.ring[wave][stage]), lane, t);
      const int key0 = s.tile(i) * kCacheTile;
      const bool whole = (there & 1) != 0 && key0 + kCacheTile - 1 <= s.low &&
                         (a.window == 0 || key0 > s.high - a.window || key0 + kCacheTile <= a.sinks);
      // Zero times a key that is no number would be no number as well.  Where rows see different keys, such scales of
      // up to 8 rows' tiles become one here, and the logits of the keys get their NaN below.  Scales above kScaleMax
      // are never written, but unwritten bytes may hold them.
      unsigned long long strange = 0;
      if (kNarrow && !whole) {
        bool found = false;
#pragma unroll
        for (int g = 0; g < W / 2; ++g) {
          if (t.k_scale[g] > (unsigned)kScaleMax) {
            t.k_scale[g] = 127;
            found = true;
          }
        }
        strange = __ballot(found);
      }
      // x[h][rt][r]: the logit of key 16 h + 4 b + r, or of up to 8 rows 16 (n / 8) + 4 b + r.
      f32x4 x[kHalves][RT];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) x[h][rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        f32x4 upper = f32x4{0.0f, 0.0f, 0.0f, 0.0f};  // of up to 8 rows, a second chain of products
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const float scale =
              kNarrow ? scale_operand(t.k_scale[c / 4], 0) : scale_operand(t.k_scale[W == 8 ? c / 4 : 0], h);
          u32x4 words;
#pragma unroll
          for (int j = 0; j < 4; ++j) words[j] = convert(t.k[h * W + c], scale, j);
          const bf16x8 key = bits_as<bf16x8>(words);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int z = 0; z < NT; ++z) {
              f32x4& sum = kNarrow && c >= kChunks / 2 ? upper : x[h][rt];
              sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, q[rt][z][c], sum, 0, 0, 0);
            }
        }
        if constexpr (kNarrow) x[h][0] += upper;
      }

      uint2 v_scale = t.v_scale;
      unsigned hidden = 0;  // bit e: the scale of the lane's token e stands for no number
      if (!whole) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key = key0 + 16 * (kNarrow ? n >> 3 : h) + 4 * b + r;
              const bool seen = (there & 1) != 0 && key <= position[rt] &&
                                (a.window == 0 || key > position[rt] - a.window || key < a.sinks);
              x[h][rt][r] = seen ? x[h][rt][r] : -INFINITY;
            }
        if (kNarrow && strange != 0) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (((strange >> (32 * (n >> 3) + 4 * b + r)) & 0x10001u) != 0 && x[0][0][r] != -INFINITY) x[0][0][r] = NAN;
        }
        // A weight of zero times a value that is no number likewise: such scales become one, and the rows that do see
        // their tokens get NaN below.
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
        most[rt] = x[0][rt][0];
#pragma unroll
        for (int e = 1; e < 4 * kHalves; ++e) most[rt] = fmaxf(most[rt], x[e / 4][rt][e & 3]);
        most[rt] *= p.scale;
        grows |= most[rt] > m[rt] + kGrowth;
      }
      if (__ballot(grows) != 0ull) {
        bool some = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          // Only the rows that grow: a row's rounding does not depend on its neighbours.
          const float highest = lane_groups_max(kNarrow ? fmaxf(most[rt], other_half(most[rt])) : most[rt]);
          const float raised = highest > m[rt] + kGrowth ? highest : m[rt];
          const float factor = __builtin_amdgcn_exp2f(m[rt] - raised);
          m[rt] = raised;
          some |= fabsf(raised) >= kFar && raised > kNoKey;
          l[rt] *= factor;
#pragma unroll
          for (int k = 0; k < kTiles; ++k) o[k][rt] *= factor;
        }
        far = __ballot(some) != 0ull;
      }
      // x * scale - m in one rounding, unless the rounding of m alone counts; then x becomes what the difference of the
      // two rounded numbers is.  (Costs common logits 1 to 2 %.)
      float shift[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) shift[rt] = m[rt];
      if (__builtin_expect(far, 0)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const bool mine = fabsf(m[rt]) >= kFar && m[rt] > kNoKey;
#pragma unroll
          for (int e = 0; e < 4 * kHalves; ++e)
            x[e / 4][rt][e & 3] = mine ? (x[e / 4][rt][e & 3] * p.scale - m[rt]) * p.inverse : x[e / 4][rt][e & 3];
          shift[rt] = mine ? 0.0f : m[rt];
        }
      }

      // The weights as the B operand: row n, keys 4 b + r and 16 + 4 b + r in elements r and 4 + r.  Of up to 8 rows,
      // columns 0 .. 7 take the first terms of a row's weights and columns 8 .. 15 the second ones, for all of its
      // keys.
      constexpr int kOperands = kNarrow ? NP / 2 + NP % 2 : NP;
      bf16x8 weights[RT][kOperands];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        unsigned words[NP][2 * kHalves];
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4 * kHalves; e += 2) {
          __bf16 terms[2][NP];
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const float w = __builtin_amdgcn_exp2f(fmaf(x[e / 4][rt][(e + f) & 3], p.scale, -shift[rt]));
            sum += w;
            split_terms<NP>(w, terms[f]);
          }
#pragma unroll
          for (int z = 0; z < NP; ++z) words[z][e / 2] = bits_as<unsigned>(bf16x2{terms[0][z], terms[1][z]});
        }
        l[rt] += sum;
        if constexpr (kNarrow) {
          const bool lower = n < 8;
#pragma unroll
          for (int z = 0; z < NP; z += 2) {
            unsigned own[2], others[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const unsigned second = z + 1 < NP ? words[z + 1 < NP ? z + 1 : z][e] : 0u;
              own[e] = lower ? words[z][e] : second;
              others[e] = other_half(lower ? second : words[z][e]);
              if (z + 1 == NP && !lower) others[e] = 0u;
            }
            weights[rt][z / 2] = bits_as<bf16x8>(lower ? u32x4{own[0], own[1], others[0], others[1]}
                                                       : u32x4{others[0], others[1], own[0], own[1]});
          }
        } else {
#pragma unroll
          for (int z = 0; z < NP; ++z)
            weights[rt][z] = bits_as<bf16x8>(u32x4{words[z][0], words[z][1], words[z][2], words[z][3]});
        }
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
          for (int z = 0; z < kOperands; ++z) {
            o[2 * w][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value0, weights[rt][z], o[2 * w][rt], 0, 0, 0);
            o[2 * w + 1][rt] =
                __builtin_amdgcn_mfma_f32_16x16x32_bf16(value1, weights[rt][z], o[2 * w + 1][rt], 0, 0, 0);
          }
      }

      there >>= 1;
      stage = stage == kStages - 1 ? 0 : stage + 1;

      if (!whole && __ballot(hidden != 0u) != 0ull) {
        // How many tokens without a number each row sees, per 2 W dims: the product of the flags and the visibility.
        bf16x8 flags;
#pragma unroll
        for (int e = 0; e < 8; ++e) flags[e] = (__bf16)((hidden >> e) & 1u ? 1.0f : 0.0f);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          bf16x8 seen;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool of_lane = !kNarrow || e / 4 == n >> 3;
            seen[e] = (__bf16)(!of_lane || x[kNarrow ? 0 : e / 4][rt][e & 3] == -INFINITY ? 0.0f : 1.0f);
          }
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

    const bool all = begin == 0 && end == s.total;
    __syncthreads();  // the rings are in use no more
    // The waves' results, relative to the block's maximum of each row, added in the waves' order.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] = lane_groups_sum(kNarrow ? l[rt] + other_half(l[rt]) : l[rt]);
      if (b == 0) {
        stats[0][wave][rt * 16 + n] = m[rt];
        stats[1][wave][rt * 16 + n] = l[rt];
      }
    }
    __syncthreads();
    constexpr int kLines = kNarrow ? 8 : 16;
    const int at_part = (int)part * (R * (D + 2)) * 4;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float highest = kNoKey;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) highest = fmaxf(highest, stats[0][w][rt * 16 + n]);
      const float factor = __builtin_amdgcn_exp2f(m[rt] - highest);
      if (rt > 0) __syncthreads();
      // Of up to 8 rows, columns n and n + 8 hold parts of one row.
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int k = 0; k < kTiles; k += 4)
          *reinterpret_cast<float4*>(&sums[wave][n][kTiles * (4 * b + r) + k]) =
              float4{o[k][rt][r] * factor, o[k + 1][rt][r] * factor, o[k + 2][rt][r] * factor,
                     o[k + 3][rt][r] * factor};
      __syncthreads();
      for (int at = thread; at < kLines * D / 4; at += kThreads) {
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
          if constexpr (kNarrow) {
            const float4 u = *reinterpret_cast<const float4*>(&sums[w][line + 8][column]);
            sum.x += u.x;
            sum.y += u.y;
            sum.z += u.z;
            sum.w += u.w;
          }
        }
        if (all) {
          const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
          const int token = row / p.group, h = row - token * p.group;
          In* to = static_cast<In*>(a.out) + ((long long)(s.row0 + token) * a.heads + head * p.group + h) * D + column;
          store4(to, float4{sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse});
        } else {
          __builtin_amdgcn_raw_buffer_store_b128(bits_as<u32x4>(sum), parts_buffer(a.work),
                                                 at_part + ((rt * 16 + line) * D + column) * 4, 0, kDeviceScope);
          if (column == 0)
            __builtin_amdgcn_raw_buffer_store_b64(bits_as<u32x2>(float2{top, total}), parts_buffer(a.work),
                                                  at_part + (R * D + 2 * (rt * 16 + line)) * 4, 0, kDeviceScope);
        }
      }
    }

    if (shared && !all) {
      // The last part of a row tile to arrive adds them all, by the hand-over of store_device (ternary_device.hpp):
      // nobody waits for anybody.
      const long long first = uniform(run.at) - begin;  // the row tile's first tile among all
      const long long first_block = first / share;
      const int parts = (int)((first + s.total - 1) / share - first_block) + 1;
      unsigned* counter = p.counters + (first_block * a.kv_heads + head) * kAttentionCounterStep;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (arrived == (unsigned)parts - 1) {
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const long long first_part = (2 * first_block + (first == first_block * share ? 0 : 1)) * a.kv_heads + head;
        const long long second_part = 2 * (first_block + 1) * a.kv_heads + head;
        add_parts<D, In, R>(p, s, head, parts_buffer(a.work), first_part, second_part, 2 * a.kv_heads, parts,
                            &sums[0][0][0]);
      }
    }
    run.at += end - begin;
    left -= end - begin;
    if (left <= 0) return;
    // The next run starts with the first tile of the next row tile or sequence.
    part = (2LL * unit + 1) * a.kv_heads + head;
    run.begin = 0;
    run.start = s.start + R;
    if (run.start >= s.rows) {
      run.start = 0;
      do {
        if (++run.sequence >= a.sequences) return;
      } while (rows_of(a, run.sequence, row0) == 0);
    }
    __syncthreads();  // the statistics in LDS have been read
  }
}

// Adds the parts of split row tiles: a wave per row (query token and head).
template <int D, typename In, int R>
__global__ __launch_bounds__(kThreads) void merge_kernel(Params p) {
  const CacheAttentionArgs& a = p.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long id = (long long)blockIdx.x * kWaves + wave;
  const int row = (int)(id / a.heads), h = (int)(id % a.heads);
  int sequence = 0, index = 0;
  if (row >= a.rows || !find_sequence(a.offsets, a.sequences, row, row, sequence, index)) return;
  const int head = h / p.group, line = index * p.group + h % p.group;
  int row0;
  const int queries = rows_of(a, sequence, row0), length = a.lengths[sequence];
  const Span s = make_span<R>(p, sequence, row0, queries, length, line / R * R);
  const int parts = min(p.splits, (s.total + p.chunk - 1) / p.chunk);
  if (parts <= 1) return;  // a single part went to its place at once
  const int first_slot = a.offsets == nullptr ? sequence * ((p.group + R - 1) / R)
                                              : (int)((long long)row0 * p.group / R) + sequence;
  const long long first = (long long)(first_slot + line / R) * p.splits * a.kv_heads + head;
  const int lane = threadIdx.x % (D / 4);
  const RowSum sum =
      add_row<D, R>(line % R, lane, 1, 0, parts_buffer(a.work), first, first + a.kv_heads, a.kv_heads, parts);
  if ((threadIdx.x & 63) < D / 4) store_row<D, In>(p, s, head, line % R, lane, sum);
}

constexpr int kUnitsOnDevice = 256;  // CUs
// Blocks that the row tiles and heads of chunks are split into: as many as the device holds at two per CU.  32/8 heads
// of 128, 9000 tokens: 16 queries 21.3 us and 27.6 with 768 blocks; 64 queries 29, 34 with 768 and 33 with 384.
constexpr int kChunkBlocks = 512;
// Rows per sequence up to which keys are dealt out: the parts of more rows are too much for one block to add.  32/8
// heads of 128: 4 queries over 2000 tokens 12.4 us dealt out, 10.9 split at equal lengths with a second launch; one
// query over 9000 12.4 and 17.3.
constexpr int kFewRows = 8;
// Cached bytes of a call from which on they are loaded past the memory-side cache: half of its 256 MB.  Loads alone
// took 64 us for 313 MB with it and 71 without; 22.6 us for 71 MB with it and 18 without.
constexpr long long kStreamBytes = 128LL << 20;
// A block's share of dealt out tiles: a 32nd of a sequence, since a row's parts are read by one block, 32 of them in
// two turns, but from 8 tiles on (two per wave) and up to 64 (more leave the device half empty).  One sequence, 32/8
// heads of 128: 8000 tokens 11.9 us with 8 tiles and 13.4 with 16; 32000 tokens 17.5 with 31, 22.7 with 11; 131000
// tokens 35.8 with 64, 39.2 with 48 and 37.7 with 43 (as many as fill the device).
constexpr int kLeastTiles = 8, kMostTiles = 64, kParts = 32;
// From so many row tiles and heads on, each with at most so many key tiles is left to one block: handing over the parts
// costs 5 us.
// 64 sequences of 4 heads of 64, 36 tiles: 14.5 us so, 25 dealt out; 60 tiles: 17.3 and 22.7.
constexpr int kWholeUnits = 128, kWholeTiles = 64;

// Rows of a row tile: 8, 16 or 32 as the sequences' rows fill on average, within the registers.  64 rows convert a
// tile's codes for twice the products, but leave room for one wave per SIMD instead of two: 512 queries over 8702
// keys, 32/8 heads of 128, took 139 us with them and take 117 (300 over 3000, 16/4 heads: 58 and 44).
int tile_rows(const CacheAttentionArgs& a) {
  const long long rows = (long long)a.rows * (a.heads / a.kv_heads) / (a.sequences > 0 ? a.sequences : 1);
  if (a.head_dim == 256) return rows <= 16 || a.dtype != kBfloat16 ? 16 : 32;
  return rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
}

Params plan(const CacheAttentionArgs& a) {
  Params p{a, a.heads / a.kv_heads, 0, 1, 0, 0, 1.44269504088896340736f * a.scale, 0.0f, false, false, nullptr};
  p.inverse = 1.0f / p.scale;
  const int size = a.dtype == kFloat32 ? 4 : 2;
  p.aligned =
      (((uintptr_t)a.q | (uintptr_t)(a.q_strides.token * size) | (uintptr_t)(a.q_strides.head * size)) & 15u) == 0;
  const int R = tile_rows(a);
  const long long rows = (long long)a.rows * p.group;
  p.slots = (int)(a.offsets == nullptr ? (long long)a.sequences * ((p.group + R - 1) / R) : rows / R + a.sequences);
  // Key tiles that a row tile sees at most, and the row tiles and heads that there may be.
  long long keys = a.max_length;
  if (a.window > 0) keys = min(keys, (long long)a.window + (R + p.group - 1) / p.group + a.sinks + 2 * kCacheTile);
  const long long tiles = max(1LL, (keys + kCacheTile - 1) / kCacheTile);
  const long long units = (rows / R + (rows % R > 0 || a.offsets == nullptr ? 1 : 0)) * a.kv_heads;
  const int terms = a.dtype == kFloat32 ? 3 : a.dtype == kFloat16 ? 2 : 1;
  static_assert(4 * kUnitsOnDevice <= kAttentionCounters, "a counter per block");
  const int resident = kUnitsOnDevice * occupancy(a.head_dim, R, terms);
  const long long live = max((long long)a.sequences * a.kv_heads, units);
  p.stream = live * tiles * cache_tile_bytes(a.head_dim) > kStreamBytes;
  const bool whole = tiles <= kLeastTiles || (tiles <= kWholeTiles && live >= kWholeUnits);
  const bool dealt = rows <= (long long)a.sequences * kFewRows && a.sequences <= 4096 && !whole;
  if (dealt) {
    p.splits = 0;
    p.chunk = (int)max((long long)kLeastTiles, min((long long)kMostTiles, tiles / kParts));
    p.blocks = (int)max(1LL, min((long long)resident, (live * tiles + p.chunk - 1) / p.chunk) / a.kv_heads);
  } else {
    const long long wanted = whole ? 1 : max(1LL, kChunkBlocks / max(1LL, live));
    p.chunk = (int)max((long long)kLeastTiles, (tiles + wanted - 1) / wanted);
    p.splits = (int)((tiles + p.chunk - 1) / p.chunk);
  }
  return p;
}

template <int D, typename In, int R, int NT>
hipError_t run(hipStream_t stream, const Params& p) {
  const bool clears = p.a.offsets != nullptr;  // rows of no sequence
  const long long units = p.splits == 0 ? (long long)p.blocks : (long long)p.slots * p.splits;
  const long long blocks = (units + (clears ? max(p.splits, 1) : 0)) * p.a.kv_heads;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (R <= 16 && p.stream)
    hipLaunchKernelGGL((cache_attention_kernel<D, In, R, NT, R <= 16>), dim3((unsigned)blocks), dim3(kThreads), 0,
                       stream, p);
  else
    hipLaunchKernelGGL((cache_attention_kernel<D, In, R, NT, false>), dim3((unsigned)blocks), dim3(kThreads), 0, stream,
                       p);
  if (p.splits > 1) {
    const long long merges = ((long long)p.a.rows * p.a.heads + kWaves - 1) / kWaves;
    if (merges > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL((merge_kernel<D, In, R>), dim3((unsigned)merges), dim3(kThreads), 0, stream, p);
  }
  return hipGetLastError();
}

template <int D, typename In, int NT>
hipError_t run_rows(hipStream_t stream, const Params& p) {
  const int rows = tile_rows(p.a);
  if constexpr (D < 256) {
    if (rows == 8) return run<D, In, 8, NT>(stream, p);
    if (rows == 32) return run<D, In, 32, NT>(stream, p);
  } else if constexpr (NT == 1) {
    if (rows == 32) return run<D, In, 32, NT>(stream, p);
  }
  return run<D, In, 16, NT>(stream, p);
}

template <int D>
hipError_t run_types(hipStream_t stream, const Params& p) {
  if (p.a.dtype == kFloat32) return run_rows<D, float, 3>(stream, p);
  if (p.a.dtype == kFloat16) return run_rows<D, Half, 2>(stream, p);
  return run_rows<D, Bfloat, 1>(stream, p);
}

}  // namespace

long long cache_attention_work(const CacheAttentionArgs& a) {
  const Params p = plan(a);
  if (p.splits == 1) return 0;
  const long long parts = (p.splits == 0 ? 2LL * p.blocks : (long long)p.slots * p.splits) * a.kv_heads;
  return parts * tile_rows(a) * (a.head_dim + 2) * 4;
}

hipError_t launch_cache_attention(hipStream_t stream, const CacheAttentionArgs& a) {
  if (a.rows == 0) return hipSuccess;
  Params p = plan(a);
  if (p.splits == 0) {
    Scratch* scratch = nullptr;
    const hipError_t status = scratch_for_stream(stream, &scratch);
    if (status != hipSuccess) return status;
    p.counters = scratch->sync + kAttentionCounterWord;
  }
  if (a.head_dim == 64) return run_types<64>(stream, p);
  if (a.head_dim == 128) return run_types<128>(stream, p);
  return run_types<256>(stream, p);
}

}  // namespace ivo
