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
// Bound by the rows' bytes.  A thread takes four dims and the four that they are paired with, of one token: no value
// crosses lanes but the sum of squares, and a thread has the four sines and cosines that it needs for all of the heads
// that it goes through, whose loads are under way four at a time while the four before are worked on.  (Eight
// neighbouring dims per thread and their partners' eight loaded as well took 59 us where this takes 29.)  All lanes of
// a head are in one wave, which loads all of a head before it stores any of it, so the results may replace the inputs.
#include "cache_rows.hpp"

namespace ivo {
namespace {

constexpr int kBatch = 4;

// cos and sin of `turns` full turns, |turns| <= 1/2: of the angle left after the nearest quarter by their Taylor
// series, whose first terms left out are below 2^-25 up to an eighth of a turn.
__device__ __forceinline__ void cos_sin(float turns, float& c, float& s) {
  const float quarter = rintf(turns * 4.0f);
  const float x = fmaf(quarter, -0.25f, turns) * 6.28318530717958647693f, y = x * x;
  const float sine = fmaf(fmaf(fmaf(fmaf(1.0f / 362880, y, -1.0f / 5040), y, 1.0f / 120), y, -1.0f / 6) * y, x, x);
  const float cosine =
      fmaf(fmaf(fmaf(fmaf(fmaf(-1.0f / 3628800, y, 1.0f / 40320), y, -1.0f / 720), y, 1.0f / 24), y, -0.5f), y, 1.0f);
  const int q = (int)quarter;
  c = q & 1 ? sine : cosine;
  s = q & 1 ? cosine : sine;
  c = (q + 1) & 2 ? -c : c;
  s = q & 2 ? -s : s;
}
// cos and sin of position * frequency.
__device__ __forceinline__ void turn(double position, float frequency, float& c, float& s) {
  constexpr double kTurnsPerRadian = 0.15915494309189533577;
  const double turns = position * ((double)frequency * kTurnsPerRadian);
  cos_sin((float)(turns - rint(turns)), c, s);
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += xor_lane<1>(v);
  v += xor_lane<2>(v);
  v += xor_lane<4>(v);
  if constexpr (LANES > 8) v += xor_lane<8>(v);
  if constexpr (LANES > 16) v += xor_lane<16>(v);
  return v;
}

// What is left of x after its rounding to the rows' type.
template <typename In>
__device__ __forceinline__ float rounded(float x) {
  In v;
  store_value(&v, x);
  return to_float(v);
}

// Four neighbouring values as they are in memory.
template <typename In>
struct Four {
  In v[4];
};
template <bool ALIGNED, typename In>
__device__ __forceinline__ Four<In> load_four(const In* p) {
  Four<In> f;
  if constexpr (ALIGNED) {
    __builtin_memcpy(&f, __builtin_assume_aligned(p, 4 * sizeof(In)), sizeof(f));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = p[j];
  }
  return f;
}
template <bool ALIGNED, typename In>
__device__ __forceinline__ void store_four(In* p, const float* x) {
  Four<In> f;
#pragma unroll
  for (int j = 0; j < 4; ++j) store_value(&f.v[j], x[j]);
  if constexpr (ALIGNED) {
    __builtin_memcpy(__builtin_assume_aligned(p, 4 * sizeof(In)), &f, sizeof(f));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = f.v[j];
  }
}

__device__ __forceinline__ void load4_values(const float* p, bool aligned, float* x) {
  if (aligned) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = p[j];
  }
}

template <int D, typename In, bool WRITE, bool INTERLEAVED, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void rotate_kernel(CacheArgs a, RotateArgs r) {
  constexpr int kLanes = D / 8;
  __shared__ __align__(16) float rows[WRITE ? kThreads * 8 : 4];  // a key's values on their way to their places
  const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row_id = id / kLanes;
  const int o = (int)(id % kLanes);
  const int row = (int)min(row_id, (long long)a.rows - 1);
  const int half = r.rotary / 2;
  const bool turned = o * 8 < r.rotary, apart = turned && !INTERLEAVED;
  // The thread's dims: dim .. dim + 3 and dim + step .. dim + step + 3.
  const int dim = apart ? o * 4 : o * 8, step = apart ? half : 4;

  // Units: the heads of q, then those of k.  The first ones' loads need no position.
  const int units = r.heads + a.kv_heads, stride = gridDim.y;
  const In* const q = static_cast<const In*>(r.q) + row * r.q_strides.token + dim;
  const In* const k = static_cast<const In*>(r.k) + row * r.k_strides.token + dim;
  Four<In> next[kBatch][2];
  auto load = [&](int unit) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = unit + i * stride;
      if (u >= units) break;
      const In* from = u < r.heads ? q + u * r.q_strides.head : k + (u - r.heads) * r.k_strides.head;
      next[i][0] = load_four<ALIGNED>(from);
      next[i][1] = load_four<ALIGNED>(from + step);
    }
  };
  load(blockIdx.y);

  const int first = (int)min((id - (threadIdx.x & 63)) / kLanes, (long long)a.rows - 1);
  int sequence = 0, index = 0;
  const bool live = find_sequence(a.offsets, a.sequences, first, row, sequence, index);
  if (row_id >= a.rows) return;  // all lanes of a head leave together, here and below
  const int start = live ? a.start[sequence] : 0;
  const long long position = (long long)start + index;
  float cos[4], sin[4];
  float frequencies[4];
  load4_values(r.frequencies + (turned ? o * 4 : 0), r.tables_aligned, frequencies);
#pragma unroll
  for (int j = 0; j < 4; ++j) turn((double)position, frequencies[j], cos[j], sin[j]);
  // The weights of the side whose heads are being worked on.
  float weights[8];
  auto load_weights = [&](const float* norm) {
    if (norm == nullptr) return;
    load4_values(norm + dim, r.tables_aligned, weights);
    load4_values(norm + dim + step, r.tables_aligned, weights + 4);
  };
  const float* norm = (int)blockIdx.y < r.heads ? r.q_norm : r.k_norm;
  load_weights(norm);
  uint8_t* tile = nullptr;
  int place = 0;
  if constexpr (WRITE) {
    if (live && start >= 0) tile = tile_of(a, sequence, position, cache_tile_bytes(D));
    place = (int)(position & (kCacheTile - 1));
  }
  const long long head_bytes = (long long)cache_tile_bytes(D) << a.page_shift;

  for (int unit = blockIdx.y; unit < units; unit += kBatch * stride) {
    Four<In> now[kBatch][2];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      now[i][0] = next[i][0];
      now[i][1] = next[i][1];
    }
    load(unit + kBatch * stride);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = unit + i * stride;
      if (u >= units) break;
      const bool of_q = u < r.heads;
      const int head = of_q ? u : u - r.heads;
      float x[8], y[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = to_float(now[i][0].v[j]);
        x[4 + j] = to_float(now[i][1].v[j]);
      }
      if (!of_q && u - stride < r.heads && u != (int)blockIdx.y) {  // the first of k's
        norm = r.k_norm;
        load_weights(norm);
      }
      if (norm != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
        const float factor = rsqrtf(lanes_sum<kLanes>(sum) * (1.0f / D) + r.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] * factor * weights[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        constexpr int kPair = INTERLEAVED ? 2 : 1, kOther = INTERLEAVED ? 1 : 4;
        const float first = x[kPair * j], second = x[kPair * j + kOther];
        y[kPair * j] = turned ? fmaf(-second, sin[j], first * cos[j]) : first;
        y[kPair * j + kOther] = turned ? fmaf(first, sin[j], second * cos[j]) : second;
      }
      if (!live) {  // a row of no sequence
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = 0.0f;
      }
      if (!WRITE || of_q) {
        In* out = of_q ? static_cast<In*>(r.q_out) + row * r.q_out_strides.token + head * r.q_out_strides.head
                       : static_cast<In*>(r.k_out) + row * r.k_out_strides.token + head * r.k_out_strides.head;
        store_four<ALIGNED>(out + dim, y);
        store_four<ALIGNED>(out + dim + step, y + 4);
      } else if (tile != nullptr) {  // all lanes of a token alike
        // Rounded to the rows' type as between the two calls: the cache then holds the same bytes.
        float* of_token = rows + (threadIdx.x - o) * 8;
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = rounded<In>(y[j]);
        *reinterpret_cast<float4*>(of_token + dim) = float4{z[0], z[1], z[2], z[3]};
        *reinterpret_cast<float4*>(of_token + dim + step) = float4{z[4], z[5], z[6], z[7]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const float4 low = *reinterpret_cast<const float4*>(of_token + o * 8);
        const float4 high = *reinterpret_cast<const float4*>(of_token + o * 8 + 4);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const float key[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
        uint8_t* at = tile + head * head_bytes;
        unsigned scale;
        const unsigned codes = quantize8(key, scale);
        store_key<D>(at, place, o, codes, scale);
        load8(static_cast<const In*>(r.v) + row * r.v_strides.token + head * r.v_strides.head + o * 8, ALIGNED, z);
        const unsigned value_codes = quantize8(z, scale);
        store_cached_value<D>(at, place, o, value_codes, scale);
      }
    }
  }
}

// Blocks of rows that the heads are split between: up to kFullBlocks as long as each thread has a batch of heads, and
// up to kFewBlocks with fewer.  32/8 heads of 128, bf16: 8190 rows 28.8 us, 31.7 with 512 blocks; 1024 rows 6.9 us, 8.6
// with 2048 blocks and single heads; 64 rows 3.8 us, a head to a thread.
constexpr long long kFullBlocks = 2048, kFewBlocks = 1024;

template <int D, typename In, bool WRITE, bool INTERLEAVED>
void launch(hipStream_t stream, dim3 grid, const CacheArgs& a, const RotateArgs& r) {
  if (r.aligned)
    hipLaunchKernelGGL((rotate_kernel<D, In, WRITE, INTERLEAVED, true>), grid, dim3(kThreads), 0, stream, a, r);
  else
    hipLaunchKernelGGL((rotate_kernel<D, In, WRITE, INTERLEAVED, false>), grid, dim3(kThreads), 0, stream, a, r);
}

template <int D, typename In>
hipError_t run(hipStream_t stream, const CacheArgs& a, const RotateArgs& r) {
  const long long blocks = ((long long)a.rows * (D / 8) + kThreads - 1) / kThreads;
  const int units = r.heads + a.kv_heads;
  const long long full = min(kFullBlocks / blocks, (long long)units / kBatch), few = min(kFewBlocks / blocks, (long long)units);
  const long long split = max(1LL, max(full, few));
  const dim3 grid((unsigned)blocks, (unsigned)split);
  if (r.v != nullptr)
    r.interleaved ? launch<D, In, true, true>(stream, grid, a, r) : launch<D, In, true, false>(stream, grid, a, r);
  else
    r.interleaved ? launch<D, In, false, true>(stream, grid, a, r) : launch<D, In, false, false>(stream, grid, a, r);
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
  // Rows are read and written four values at a time where they all start on as many (values for the cache on 16 bytes).
  const uintptr_t four = at(r.q, r.q_strides) | at(r.k, r.k_strides) | at(r.q_out, r.q_out_strides) |
                         at(r.k_out, r.k_out_strides);
  r.tables_aligned = (((uintptr_t)r.q_norm | (uintptr_t)r.k_norm | (uintptr_t)r.frequencies) & 15u) == 0;
  r.aligned = (four & (4 * size - 1)) == 0 && (at(r.v, r.v_strides) & 15u) == 0;
  if (head_dim == 64) return run_types<64>(stream, a, r, dtype);
  if (head_dim == 128) return run_types<128>(stream, a, r, dtype);
  return run_types<256>(stream, a, r, dtype);
}

}  // namespace ivo
