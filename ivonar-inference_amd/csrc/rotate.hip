// The norm of query and key heads and their rotation by position, in one pass, and with it the write of keys and values
// into the 4-bit cache (layout: cache_layout.hpp).
//
// For a head's row x of D values at position p, with the first 2 H of them rotated (H pairs):
//   y = x * rsqrt(mean(x^2) + eps) * weight, or x where there is no weight;
//   pair i of y, at dims (i, H + i) or (2 i, 2 i + 1), is turned by the angle p f_i:
//   (a, b) -> (a cos - b sin, b cos + a sin).
// Everything is in fp32 but the angle: p f_i / (2 pi) is formed in 64 bits and reduced to half a turn there, since in
// fp32 an angle of 10^5 has lost 2^-8 of a radian; what is left of it is exact to 2^-25 of a turn in fp32.
//
// Bound by the rows' bytes.  A thread takes dims 8 o .. 8 o + 7 of one token and has their sines and cosines for all
// of the heads that it goes through, kBatch heads' loads under way at a time.  A pair's other half lies H dims away: it
// is loaded too (from the vector cache, where a neighbouring lane has just brought it) rather than passed between lanes.
// All lanes of a head are in one wave, which loads all of a head before it stores any of it, so the results may
// replace the inputs.
#include "cache_rows.hpp"

namespace ivo {
namespace {

constexpr int kBatch = 4;

// cos and sin of position * frequency.
__device__ __forceinline__ void turn(long long position, float frequency, float& c, float& s) {
  constexpr double kTurnsPerRadian = 0.15915494309189533577;
  const double turns = (double)position * (double)frequency * kTurnsPerRadian;
  const float part = (float)(turns - rint(turns));
  sincospif(2.0f * part, &s, &c);
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

template <typename In>
__device__ __forceinline__ void store_values(In* p, bool aligned, const float (&x)[8]) {
  if (aligned) {
    store8(p, x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) store_value(p + j, x[j]);
  }
}

// What is left of x after its rounding to the rows' type.
template <typename In>
__device__ __forceinline__ float rounded(float x) {
  In v;
  store_value(&v, x);
  return to_float(v);
}

// Cosines and sines of a thread's eight dims: y[j] = x[j] * cos[j] + partner[j] * sin[j], the sign in sin.
struct Turns {
  float cos[8], sin[8];
  int partner;  // dims between a value and the other half of its pair; 0: neighbours, or not rotated
  bool rotated;
};

template <int D, typename In, bool WRITE>
__global__ __launch_bounds__(kThreads) void rotate_kernel(CacheArgs a, RotateArgs r) {
  constexpr int kLanes = D / 8;
  const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row_id = id / kLanes;
  const int o = (int)(id % kLanes);
  const int row = (int)min(row_id, (long long)a.rows - 1);
  const int first = (int)min((id - (threadIdx.x & 63)) / kLanes, (long long)a.rows - 1);
  int sequence = 0, index = 0;
  const bool live = find_sequence(a.offsets, a.sequences, first, row, sequence, index);
  if (row_id >= a.rows) return;  // all lanes of a head leave together
  In* const q_out = static_cast<In*>(r.q_out) + row * r.q_out_strides.token + o * 8;
  In* const k_out = WRITE ? nullptr : static_cast<In*>(r.k_out) + row * r.k_out_strides.token + o * 8;
  if (!live) {  // a row of no sequence
    const float zero[8] = {};
    for (int head = blockIdx.y; head < r.heads; head += gridDim.y)
      store_values(q_out + head * r.q_out_strides.head, r.out_aligned, zero);
    if constexpr (!WRITE)
      for (int head = blockIdx.y; head < a.kv_heads; head += gridDim.y)
        store_values(k_out + head * r.k_out_strides.head, r.out_aligned, zero);
    return;
  }
  const int start = a.start[sequence];
  const long long position = (long long)start + index;

  Turns t;
  const int half = r.rotary / 2, dim = o * 8;
  t.rotated = dim < r.rotary;
  t.partner = r.interleaved || !t.rotated ? 0 : dim < half ? half : -half;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (r.interleaved && (j & 1)) {
      t.cos[j] = t.cos[j - 1];
      t.sin[j] = -t.sin[j - 1];
      continue;
    }
    const int pair = r.interleaved ? (dim + j) / 2 : dim < half ? dim + j : dim - half + j;
    turn(position, r.frequencies[t.rotated ? pair : 0], t.cos[j], t.sin[j]);
    if (r.interleaved || dim < half) t.sin[j] = -t.sin[j];
  }

  // Heads first, first + step, .. below `heads` of one side, `finish` called with each one's result.
  auto heads_of = [&](const void* rows, RowStrides strides, int heads, const float* norm, auto finish) {
    const In* from = static_cast<const In*>(rows) + row * strides.token + dim;
    float weight[8], partner_weight[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      weight[j] = norm == nullptr ? 1.0f : norm[dim + j];
      partner_weight[j] = norm == nullptr ? 1.0f : norm[dim + t.partner + j];
    }
    for (int head = blockIdx.y; head < heads; head += kBatch * gridDim.y) {
      float x[kBatch][8], other[kBatch][8];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const In* at = from + min(head + i * (int)gridDim.y, heads - 1) * strides.head;
        load8(at, r.aligned, x[i]);
        if (!r.interleaved) load8(at + t.partner, r.aligned, other[i]);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (head + i * (int)gridDim.y >= heads) break;
        float y[8];
        float factor = 1.0f;
        if (norm != nullptr) {
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) sum = fmaf(x[i][j], x[i][j], sum);
          factor = 1.0f / sqrtf(lanes_sum<kLanes>(sum) * (1.0f / D) + r.eps);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[i][j] = x[i][j] * factor * weight[j];
          other[i][j] = other[i][j] * factor * partner_weight[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float partner = r.interleaved ? x[i][j ^ 1] : other[i][j];
          y[j] = t.rotated ? fmaf(partner, t.sin[j], x[i][j] * t.cos[j]) : x[i][j];
        }
        finish(head + i * (int)gridDim.y, y);
      }
    }
  };

  heads_of(r.q, r.q_strides, r.heads, r.q_norm, [&](int head, const float (&y)[8]) {
    store_values(q_out + head * r.q_out_strides.head, r.out_aligned, y);
  });
  if constexpr (!WRITE) {
    heads_of(r.k, r.k_strides, a.kv_heads, r.k_norm, [&](int head, const float (&y)[8]) {
      store_values(k_out + head * r.k_out_strides.head, r.out_aligned, y);
    });
  } else {
    uint8_t* tile = start < 0 ? nullptr : tile_of(a, sequence, position, cache_tile_bytes(D));
    if (tile == nullptr) return;  // all lanes of a token leave together
    const int place = (int)(position & (kCacheTile - 1));
    const long long head_bytes = (long long)cache_tile_bytes(D) << a.page_shift;
    const In* values = static_cast<const In*>(r.v) + row * r.v_strides.token + dim;
    heads_of(r.k, r.k_strides, a.kv_heads, r.k_norm, [&](int head, const float (&y)[8]) {
      uint8_t* at = tile + head * head_bytes;
      float z[8];
      unsigned scale;
      // The rounding that a key between the two calls would have: the cache then holds the same bytes.
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = rounded<In>(y[j]);
      store_key<D>(at, place, o, quantize8(z, scale), scale);
      load8(values + head * r.v_strides.head, r.aligned, z);
      const unsigned codes = quantize8(z, scale);
      store_cached_value<D>(at, place, o, codes, scale);
    });
  }
}

// As the cache's kernels have it: blocks beyond which a thread takes several heads.
constexpr long long kRowBlocks = 2048;

template <int D, typename In>
hipError_t run(hipStream_t stream, const CacheArgs& a, const RotateArgs& r) {
  const long long blocks = ((long long)a.rows * (D / 8) + kThreads - 1) / kThreads;
  const int most = r.heads > a.kv_heads ? r.heads : a.kv_heads;
  long long split = kRowBlocks / blocks;
  split = split < 1 ? 1 : split > most ? most : split;
  const dim3 grid((unsigned)blocks, (unsigned)split);
  if (r.v == nullptr)
    hipLaunchKernelGGL((rotate_kernel<D, In, false>), grid, dim3(kThreads), 0, stream, a, r);
  else
    hipLaunchKernelGGL((rotate_kernel<D, In, true>), grid, dim3(kThreads), 0, stream, a, r);
  return hipGetLastError();
}

template <int D>
hipError_t run_types(hipStream_t stream, const CacheArgs& a, const RotateArgs& r, int dtype) {
  if (dtype == kFloat32) return run<D, float>(stream, a, r);
  if (dtype == kFloat16) return run<D, Half>(stream, a, r);
  return run<D, Bfloat>(stream, a, r);
}

}  // namespace

hipError_t launch_rotate(hipStream_t stream, const CacheArgs& a, RotateArgs r, int head_dim, int dtype) {
  if (a.rows == 0) return hipSuccess;
  const int size = dtype == kFloat32 ? 4 : 2;
  auto at = [&](const void* p, RowStrides s) {
    return (uintptr_t)p | (uintptr_t)(s.token * size) | (uintptr_t)(s.head * size);
  };
  r.aligned = ((at(r.q, r.q_strides) | at(r.k, r.k_strides) | at(r.v, r.v_strides)) & 15u) == 0;
  r.out_aligned = ((at(r.q_out, r.q_out_strides) | at(r.k_out, r.k_out_strides)) & 15u) == 0;
  if (head_dim == 64) return run_types<64>(stream, a, r, dtype);
  if (head_dim == 128) return run_types<128>(stream, a, r, dtype);
  return run_types<256>(stream, a, r, dtype);
}

}  // namespace ivo
