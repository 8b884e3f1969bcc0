// Causal attention within packed prompts, over fp16 or bf16 keys and values, with a sliding window and sinks.
//
// The query at position p of its sequence sees the keys j <= p, with j > p - window or j < sinks where there is a
// window: x_j = scale * q . k_j, o = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m), in one pass over the keys with a
// running m, sum and o in fp32; the weights exp(x_j - m) are rounded to the inputs' type, once, for the product with v;
// their sum is not.  That moves a result by up to half a unit of the type in its weights, about as much as its own
// rounding to the type does: the error against 64 bits, relative to the results' norm, is 0.0022 where exact weights
// leave 0.00165 (8192 rows, bf16), and 0.00026 for 0.00020 (6001 rows, fp16).  A second term of the weights, as the
// cache attention has it, would bring the latter figures, but takes 26 % longer here, where products and vector units
// are the bound: 238 us for 189, and 41 for 32.6.
//
// A block takes 128 neighbouring rows of one head, 32 per wave, and the key tiles that any of them sees, which go
// straight from memory to LDS (two buffers: the next tile's loads run while this one is used).  Per tile a wave forms
//   S^T [key][row]: A = K from LDS, B = q, held in registers;
//   P = 2^(x - m), which in the MFMA's result layout is already the B operand of
//   O^T [dim][row] += A = V^T, read from LDS with transposing reads, B = P.
// So a row's maximum and sum need one exchange between the wave's halves, and those of the maximum only when some
// value exceeds the running m by a factor of 2^8 (until then the weights stay below 2^8, which the types hold as
// precisely as values below one).
//
// Bound by issue: the exponentials and conversions of a tile keep the vector units as busy as its products the matrix
// units (41 % and 32 % of the cycles at 128 dims), and two or three waves per SIMD do not overlap them fully.
// Measured (MI355X, in graphs): 8192 rows, 32/8 heads of 128, bf16, window 1024 + 4: 188 us, 686 TFLOP/s of visible
// pairs (a large matrix product reaches 1124); 8 prompts of 6001 rows in all, 16 heads of 64, fp16: 31 us, 331 TFLOP/s
// (short prompts: most of the tiles touch the diagonal or the end); one of 36 rows: 5.7 us, a chain of loads.
#include "buffer_ops.hpp"
#include "cache_layout.hpp"
#include "ternary_device.hpp"

namespace ivo {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;
constexpr float kNoKey = -3.0e38f;  // running maximum before any key
constexpr float kGrowth = 8.0f;
constexpr float kFar = 0x1p24f;  // from here on a maximum, x * scale, may be rounded by one and more

struct Params {
  WindowAttentionArgs a;
  int group;
  int slots;    // row tiles of all sequences (an upper bound)
  float scale;  // log2(e) * scale
  float inverse;
};

struct F16 {
  typedef f16x8 vec;
  static constexpr unsigned kNonFinite = 0x7c00u, kOne = 0x3c00u;
  __device__ static f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static unsigned pack(float x, float y) { return bits_as<unsigned>(f16x2{(_Float16)x, (_Float16)y}); }
};
struct B16 {
  typedef bf16x8 vec;
  static constexpr unsigned kNonFinite = 0x7f80u, kOne = 0x3f80u;
  __device__ static f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static unsigned pack(float x, float y) { return bits_as<unsigned>(bf16x2{(__bf16)x, (__bf16)y}); }
};

// 16-byte piece p of row r of a tile in LDS lies at piece r * D / 8 + (p ^ swizzle).  K: sixteen lanes that read the
// same piece of 16 rows cover all 64 banks once.  V: four rows of 64 bytes that one transposing read takes lie in
// different quarters of the banks.
template <int D>
__device__ __forceinline__ int k_swizzle(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
template <int D>
__device__ __forceinline__ int v_swizzle(int row) { return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }

// Rows [begin, end) of all rows form a sequence; the row tile takes kRows of them from `start` on.
struct Rows {
  int begin, count, start;
};

// Row tile `slot`: sequence b's are the slots from offsets[b] / kRows + b on, which leaves each sequence at least as
// many as it needs.
__device__ __forceinline__ bool rows_of(const Params& p, int slot, Rows& rows) {
  const WindowAttentionArgs& a = p.a;
  if (a.offsets == nullptr) {
    rows.begin = 0;
    rows.count = a.rows;
    rows.start = slot * kRows;
  } else {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.sequences; base += 64) {
      const int b = base + lane;
      before += __popcll(__ballot(b < a.sequences && (long long)(a.offsets[b] / kRows) + b <= slot));
    }
    if (before == 0) return false;
    const int b = __builtin_amdgcn_readfirstlane(before - 1);
    rows.begin = a.offsets[b];
    rows.count = min(a.offsets[b + 1], a.rows) - rows.begin;
    rows.start = (slot - rows.begin / kRows - b) * kRows;
  }
  return rows.begin >= 0 && rows.start >= 0 && rows.start < rows.count;
}

// Zeroes the rows of this head that belong to no sequence.
__device__ __forceinline__ void clear_rows(const Params& p, int head) {
  const WindowAttentionArgs& a = p.a;
  const int begin = a.sequences > 0 ? max(a.offsets[0], 0) : 0;
  const int end = a.sequences > 0 ? max(a.offsets[a.sequences], begin) : 0;
  const int words = a.head_dim / 2;
  for (int row = 0; row < a.rows; ++row) {
    if (row == begin) row = end;
    if (row >= a.rows) break;
    unsigned* to = static_cast<unsigned*>(a.out) + ((long long)row * a.heads + head) * words;
    for (int i = threadIdx.x; i < words; i += kThreads) to[i] = 0u;
  }
}

// Whether a piece of eight values holds one that is no finite number.
template <typename T>
__device__ __forceinline__ bool strange(const u32x4& words) {
  bool found = false;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    found |= (words[j] & T::kNonFinite) == T::kNonFinite || (words[j] >> 16 & T::kNonFinite) == T::kNonFinite;
  return found;
}
// Of two values, a one where one is infinite with this sign or no number, and a zero elsewhere.
template <typename T>
__device__ __forceinline__ unsigned flags_of(unsigned word, unsigned sign) {
  unsigned flags = 0;
#pragma unroll
  for (int shift = 0; shift < 32; shift += 16) {
    const unsigned bits = word >> shift & 0xffffu, size = bits & 0x7fffu;
    if (size > T::kNonFinite || (size == T::kNonFinite && bits >> 15 == sign)) flags |= T::kOne << shift;
  }
  return flags;
}
__device__ __forceinline__ u32x4 piece_of(const unsigned char* rows, int slot) {
  return *reinterpret_cast<const u32x4*>(rows + slot * 16);
}

template <int D, int KEYS>
struct Stage {
  unsigned char k[KEYS * D * 2];
  unsigned char v[KEYS * D * 2];
};

template <typename T, int D, int KEYS>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : D == 128 ? 2 : 3) void window_attention_kernel(Params p) {
  constexpr int kPieces = D / 8, kSubtiles = KEYS / 32, kDims = D / 32, kLoads = KEYS * kPieces / kThreads;
  typedef typename T::vec vec;
  const WindowAttentionArgs& a = p.a;
  __shared__ __align__(16) Stage<D, KEYS> stages[2];
  const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Neighbouring blocks go to different XCDs: those of one XCD take neighbouring heads, which share keys.
  const int turn = blockIdx.x % a.heads;
  const int head = a.heads % 8 == 0 ? turn % 8 * (a.heads / 8) + turn / 8 : turn;
  const int unit = blockIdx.x / a.heads;
  if (unit >= p.slots) {
    clear_rows(p, head);
    return;
  }
  Rows rows;
  if (!rows_of(p, p.slots - 1 - unit, rows)) return;  // the last first: of one prompt, those that see the most keys
  const int kv_head = head / p.group;

  const int low = rows.start + wave * kWaveRows;  // this wave's rows that exist: low .. high
  const int high = min(low + kWaveRows, rows.count) - 1;
  const int position = low + n;
  const int last = min(rows.start + kRows, rows.count) - 1;
  const int end_tile = last / KEYS + 1;
  const int window_tile = a.window == 0 || rows.start < a.window ? 0 : (rows.start - a.window + 1) / KEYS;
  const int sink_tiles = a.window == 0 || a.sinks == 0 ? 0 : min((a.sinks - 1) / KEYS + 1, window_tile);
  const int tiles = sink_tiles + end_tile - window_tile;
  auto tile_of = [&](int i) { return i < sink_tiles ? i : i - sink_tiles + window_tile; };

  // A tile's rows from memory to LDS: a thread takes the same place of kLoads rows kStep apart, whose swizzle is the
  // same (at D = 256, every other's).  Rows past the sequence start past the buffer's end, and are zeros.
  constexpr int kStep = kThreads / kPieces, kPlaces = D == 256 ? 2 : 1;
  const uint16_t* k0 = static_cast<const uint16_t*>(a.k) + rows.begin * a.k_strides.token + kv_head * a.k_strides.head;
  const uint16_t* v0 = static_cast<const uint16_t*>(a.v) + rows.begin * a.v_strides.token + kv_head * a.v_strides.head;
  const int k_step = (int)a.k_strides.token * 2 * kStep, v_step = (int)a.v_strides.token * 2 * kStep;
  int k_at[kPlaces], v_at[kPlaces];
#pragma unroll
  for (int j = 0; j < kPlaces; ++j) {
    const int row = (int)threadIdx.x / kPieces, piece = (int)threadIdx.x % kPieces;
    k_at[j] = row * (int)a.k_strides.token * 2 + (piece ^ k_swizzle<D>(row + j * kStep)) * 16;
    v_at[j] = row * (int)a.v_strides.token * 2 + (piece ^ v_swizzle<D>(row + j * kStep)) * 16;
  }
  // The next tile to load: its first key, and the addresses and sizes of its rows.
  int next_key = tile_of(0) * KEYS;
  const uint16_t *k_next = k0 + next_key * a.k_strides.token, *v_next = v0 + next_key * a.v_strides.token;
  const int k_row = (int)a.k_strides.token * 2, v_row = (int)a.v_strides.token * 2;
  auto load_tile = [&](int i, int stage) {
    const int before = min(KEYS, rows.count - next_key) - 1;
    const v4u k_buffer = wide_buffer(k_next, before * k_row + D * 2);
    const v4u v_buffer = wide_buffer(v_next, before * v_row + D * 2);
    const unsigned to = lds_address(&stages[stage]) + wave * 1024;
#pragma unroll
    for (int j = 0; j < kLoads; j += 2)
      dma_pair<false>(k_buffer, to + j * kThreads * 16, kThreads * 16, k_at[0], k_at[kPlaces - 1], j * k_step, k_step);
#pragma unroll
    for (int j = 0; j < kLoads; j += 2)
      dma_pair<false>(v_buffer, to + KEYS * D * 2 + j * kThreads * 16, kThreads * 16, v_at[0], v_at[kPlaces - 1],
                      j * v_step, v_step);
    const int keys = i + 1 == sink_tiles ? window_tile * KEYS - next_key : KEYS;
    next_key += keys;
    k_next += keys * a.k_strides.token;
    v_next += keys * a.v_strides.token;
  };

  load_tile(0, 0);
  // q as the B operand: row n, dims 16 c + 8 half + j; a row that does not exist takes the last one's.
  vec q[D / 16];
  {
    const uint16_t* from = static_cast<const uint16_t*>(a.q) +
                           (long long)(rows.begin + min(position, rows.count - 1)) * a.q_strides.token +
                           head * a.q_strides.head + half * 8;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) q[c] = *reinterpret_cast<const vec*>(from + c * 16);
    // Waits for q here: a wait inside the loop would be one for the next tile's loads in every turn.
#pragma unroll
    for (int c = 0; c < D / 16; ++c) asm volatile("" : "+v"(q[c]));
  }

  f32x16 o[kDims];
#pragma unroll
  for (int i = 0; i < kDims; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;
  float m = kNoKey, l = 0.0f;
  bool far = false;      // some row's maximum is
  bool cleared = false;  // some value that is no finite number was left out
  bool searched = true;  // every tile was searched for them

  for (int i = 0; i < tiles; ++i) {
    const int key0 = tile_of(i) * KEYS;
    Stage<D, KEYS>& stage = stages[i & 1];
    direct_load_sync();  // this tile has arrived, and nobody reads the other buffer any more
    if (i + 1 < tiles) load_tile(i + 1, (i + 1) & 1);
    // A weight of zero times a value that is no finite number would be no number.  Where rows see different keys, such
    // values become zeros in LDS; the sums of the rows that see them are set at the end.
    const bool edge = key0 + KEYS - 1 > rows.start ||
                      (a.window > 0 && key0 <= last - a.window && key0 + KEYS > a.sinks);
    if (edge) {
      bool found = false;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) found |= strange<T>(piece_of(stage.v, j * kThreads + (int)threadIdx.x));
      if (__syncthreads_or(found)) {
        cleared = true;
#pragma unroll 1
        for (int slot = threadIdx.x; slot < KEYS * kPieces; slot += kThreads) {
          u32x4 words = piece_of(stage.v, slot);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if ((words[j] & T::kNonFinite) == T::kNonFinite) words[j] &= 0xffff0000u;
            if ((words[j] >> 16 & T::kNonFinite) == T::kNonFinite) words[j] &= 0xffffu;
          }
          *reinterpret_cast<u32x4*>(stage.v + slot * 16) = words;
        }
        __syncthreads();
      }
    } else {
      searched = false;
    }
    const bool none = key0 > high || low >= rows.count ||
                      (a.window > 0 && key0 + KEYS - 1 <= low - a.window && key0 >= a.sinks);
    if (none) continue;

    f32x16 x[kSubtiles];
#pragma unroll
    for (int s = 0; s < kSubtiles; ++s) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[s][r] = 0.0f;
      const int row = 32 * s + n;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const vec key = *reinterpret_cast<const vec*>(
            stage.k + (row * kPieces + ((2 * c + half) ^ k_swizzle<D>(row))) * 16);
        x[s] = T::mfma(key, q[c], x[s]);
      }
    }
    // Four reads of K ahead of the products that use them.
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int j = 0; j < kSubtiles * D / 16; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }

    const bool whole = key0 + KEYS - 1 <= low &&
                       (a.window == 0 || key0 > high - a.window || key0 + KEYS <= a.sinks);
    if (!whole) {
#pragma unroll
      for (int s = 0; s < kSubtiles; ++s)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = key0 + 32 * s + 8 * (r / 4) + 4 * half + r % 4;
          const bool seen = key <= position && (a.window == 0 || key > position - a.window || key < a.sinks);
          x[s][r] = seen ? x[s][r] : -INFINITY;
        }
    }
    // Keeps the logits in the registers of the product on either way (they would be copied otherwise).
#pragma unroll
    for (int s = 0; s < kSubtiles; ++s) asm volatile("" : "+v"(x[s]));

    float most = -INFINITY;
#pragma unroll
    for (int s = 0; s < kSubtiles; ++s)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, x[s][r]);
    most *= p.scale;
    if (__ballot(most > m + kGrowth) != 0ull) {
      // Only the rows that grow: a row's rounding does not depend on its neighbours.
      const float highest = fmaxf(most, __shfl_xor(most, 32));
      const float raised = highest > m + kGrowth ? highest : m;
      const float factor = __builtin_amdgcn_exp2f(m - raised);
      m = raised;
      far = __ballot(fabsf(m) >= kFar && m > kNoKey) != 0ull;
      l *= factor;
#pragma unroll
      for (int k = 0; k < kDims; ++k) o[k] *= factor;
    }

    // x * scale - m in one rounding, unless the rounding of m alone counts; then x becomes what the difference of the
    // two rounded numbers is.  (Costs common logits up to 1 %.)
    float shift = m;
    if (far) {
      const bool mine = fabsf(m) >= kFar && m > kNoKey;
#pragma unroll
      for (int s = 0; s < kSubtiles; ++s)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[s][r] = mine ? (x[s][r] * p.scale - m) * p.inverse : x[s][r];
      shift = mine ? 0.0f : m;
    }

    vec weights[2 * kSubtiles];
#pragma unroll
    for (int s = 0; s < kSubtiles; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        u32x4 words;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = __builtin_amdgcn_exp2f(fmaf(x[s][8 * b + 2 * j], p.scale, -shift));
          const float w = __builtin_amdgcn_exp2f(fmaf(x[s][8 * b + 2 * j + 1], p.scale, -shift));
          l += u + w;
          words[j] = T::pack(u, w);
        }
        weights[2 * s + b] = bits_as<vec>(words);
      }

    // V^T as the A operand of 16 keys: dim 32 i + n, keys 4 half + j and 8 + 4 half + j.
    auto value = [&](int block, int k) {
      u32x4 words;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const int row = 16 * block + 8 * part + 4 * half + ((lane & 15) >> 2);
        const int dim = 32 * k + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const unsigned char* at = stage.v + (row * kPieces + ((dim / 8) ^ v_swizzle<D>(row))) * 16 + (dim & 4) * 2;
        const u32x2 got = bits_as<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(at)));
        words[2 * part] = got[0];
        words[2 * part + 1] = got[1];
      }
      return words;
    };
#pragma unroll
    for (int block = 0; block < 2 * kSubtiles; ++block)
#pragma unroll
      for (int k = 0; k < kDims; ++k) o[k] = T::mfma(bits_as<vec>(value(block, k)), weights[block], o[k]);
  }

  l += __shfl_xor(l, 32);
  auto store = [&]() {
    if (position >= rows.count) return;
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* to = static_cast<uint16_t*>(a.out) + ((long long)(rows.begin + position) * a.heads + head) * D + 4 * half;
#pragma unroll
    for (int k = 0; k < kDims; ++k)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<u32x2*>(to + 32 * k + 2 * r) = u32x2{T::pack(o[k][r] * inverse, o[k][r + 1] * inverse),
                                                               T::pack(o[k][r + 2] * inverse, o[k][r + 3] * inverse)};
  };
  store();

  // A row that sees a value that is no finite number gets the infinity, or no number, as its sum.  Such values have
  // been left out, or an infinity met a weight too small for its type in a tile that was not searched: then a row whose
  // logits are numbers has a sum that is none.  In either case the wave goes through its values once more, straight
  // from memory, and stores its rows again (tested before the stores, or by all waves with a barrier, any long prompt
  // takes 2 to 4 % longer).
  bool odd = false;
  if (!searched) {
    float zero[4] = {};
#pragma unroll
    for (int k = 0; k < kDims; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) zero[r & 3] = fmaf(o[k][r], 0.0f, zero[r & 3]);
    odd = !((zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.0f) && l < INFINITY;
  }
  if (low <= high && (cleared || __ballot(odd) != 0ull)) {
#pragma unroll
    for (int k = 0; k < kDims; ++k) {
      // How many infinities of either sign each row sees per dim: the products of their flags and the visibility.
      f32x16 count[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) count[0][r] = count[1][r] = 0.0f;
#pragma unroll 1
      for (int step = 0; step < tiles * (KEYS / 16); ++step) {
        const int key0 = tile_of(step / (KEYS / 16)) * KEYS + step % (KEYS / 16) * 16 + 4 * half;
        u32x4 seen, flags[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          seen[j] = 0;
          unsigned word = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key0 + 8 * (j / 2) + 2 * (j % 2) + e;
            word |= (unsigned)v0[min(key, rows.count - 1) * a.v_strides.token + 32 * k + n] << (16 * e);
            if (key <= position && (a.window == 0 || key > position - a.window || key < a.sinks))
              seen[j] |= T::kOne << (16 * e);
          }
#pragma unroll
          for (unsigned sign = 0; sign < 2; ++sign) flags[sign][j] = flags_of<T>(word, sign);
        }
#pragma unroll
        for (int sign = 0; sign < 2; ++sign)
          count[sign] = T::mfma(bits_as<vec>(flags[sign]), bits_as<vec>(seen), count[sign]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (count[0][r] > 0.0f || count[1][r] > 0.0f)
          o[k][r] = count[1][r] == 0.0f ? INFINITY : count[0][r] == 0.0f ? -INFINITY : NAN;
    }
    store();
  }
}

template <typename T>
void run(hipStream_t stream, const Params& p, unsigned blocks) {
  if (p.a.head_dim == 64)
    hipLaunchKernelGGL((window_attention_kernel<T, 64, 64>), dim3(blocks), dim3(kThreads), 0, stream, p);
  else if (p.a.head_dim == 128)
    hipLaunchKernelGGL((window_attention_kernel<T, 128, 64>), dim3(blocks), dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((window_attention_kernel<T, 256, 32>), dim3(blocks), dim3(kThreads), 0, stream, p);
}

}  // namespace

hipError_t launch_window_attention(hipStream_t stream, const WindowAttentionArgs& a) {
  if (a.rows == 0) return hipSuccess;
  Params p{a, a.heads / a.kv_heads, 0, 1.44269504088896340736f * a.scale, 0.0f};
  p.inverse = 1.0f / p.scale;
  p.slots = a.offsets == nullptr ? (a.rows + kRows - 1) / kRows : a.rows / kRows + a.sequences;
  const long long blocks = (long long)(p.slots + (a.offsets != nullptr ? 1 : 0)) * a.heads;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (a.dtype == kFloat16)
    run<F16>(stream, p, (unsigned)blocks);
  else
    run<B16>(stream, p, (unsigned)blocks);
  return hipGetLastError();
}

}  // namespace ivo
