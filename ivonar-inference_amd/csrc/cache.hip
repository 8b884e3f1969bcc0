// Writing rows of keys and values into the 4-bit cache, and reading them back (layout: cache_layout.hpp).
//
// Quantiser, for the 32 values x of a block: a = max |x|; exponent e = floor(log2(a * 8/7)) - 2, at least -100 and at
// most 125, so that a / 2^e < 7 and the largest value is at most half a step from the largest code, 6 (the exponent
// of a alone would leave a / 2^e up to 8 and cut a quarter off); code = the value nearest to x / 2^e, ties to the
// even code, at most 6; scale byte = e + 127.  In bits: the byte is (bits(a) + 0x200000) >> 23, less 2, since adding
// a quarter to the mantissa field carries where the mantissa is 1.75 and more.  A block that holds a NaN or an
// infinity gets the byte 255, which the conversions back turn into NaN.  The division and the rounding are
// v_cvt_scalef32_pk_fp4_f32, which rounds ties to even and saturates.
//
// Both kernels are bound by the rows' bytes: a value costs a handful of instructions.  Measured (MI355X, medians of
// traced calls): 8190 tokens of 8 heads of 128, fp32: written in 16 to 19 us, read back in 17 us, 76 MB each, 4.0 to
// 4.8 and 4.5 TB/s (a copy reaches 5.3); 65000 tokens read as bf16: 70 us, 337 MB, 4.8 TB/s.  A decode step of 64
// tokens takes 3.9 and 3.7 us, a chain of dependent loads (offsets, page, row).
#include "cache_layout.hpp"
#include "ternary_device.hpp"

namespace ivo {
namespace {

__device__ __forceinline__ unsigned quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));  // lane ^ 1
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));  // lane ^ 2
}

// Eight values of a lane, and the scale byte of the block of 32 that four neighbouring lanes hold.
__device__ __forceinline__ unsigned quantize8(const float (&x)[8], unsigned& scale) {
  unsigned most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[j]) & 0x7fffffffu);
  most = quad_max(most);
  const int byte = min(max((int)((most + 0x200000u) >> 23) - 2, kScaleMin), kScaleMax);
  const float s = __uint_as_float((unsigned)byte << 23);
  unsigned codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], s, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], s, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], s, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], s, 3);
  scale = most >= 0x7f800000u ? kScaleNan : (unsigned)byte;
  return codes;
}

// Byte of V codes at which dims 8 o .. 8 o + 7 of token t start (two halves 16 bytes apart at D = 64).
template <int D>
__device__ __forceinline__ int value_offset(int t, int o) {
  constexpr int W = D / 32, kPer = 16 / W;
  const int e = (t >> 4) * 4 + (t & 3), b = (t >> 2) & 3;
  const int n = o * 4 / W;
  return 16 * D + (e / kPer) * 1024 + (b * 16 + n) * 16 + (e % kPer) * W + (W == 8 ? (o & 1) * 4 : 0);
}
template <int D>
__device__ __forceinline__ int key_scale_offset(int t, int group) {
  return 32 * D + group * 32 + (t & 15) * 2 + (t >> 4);
}
template <int D>
__device__ __forceinline__ int value_scale_offset(int t, int group) {
  return 33 * D + group * 32 + ((t >> 2) & 3) * 8 + (t >> 4) * 4 + (t & 3);
}

// Address of the tile of head 0 that holds position p of a sequence, or null where it has no page.
__device__ __forceinline__ uint8_t* tile_of(const CacheArgs& a, int sequence, long long p, int tile_bytes) {
  const long long tile = p / kCacheTile;
  const long long slot = tile >> a.page_shift;
  if (p < 0 || slot >= a.table_width) return nullptr;
  const int page = a.table[(long long)sequence * a.table_width + slot];
  if ((unsigned)page >= (unsigned)a.page_count) return nullptr;
  const int tiles = 1 << a.page_shift;
  return a.pages + ((long long)page * a.kv_heads * tiles + (tile & (tiles - 1))) * tile_bytes;
}

// A thread takes dims 8 o .. 8 o + 7 of a token, for the heads blockIdx.y, blockIdx.y + gridDim.y, ..., of K and V:
// the page is looked up once per token.  D / 8 neighbouring threads hold a row, so a wave reads whole rows, and its
// stores of K are contiguous over its tokens; those of V are words 16 bytes apart, filled by four neighbouring tokens
// (half, a quarter or an eighth of a wave each).
template <int D, typename In>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(CacheArgs a, const In* __restrict__ k,
                                                               const In* __restrict__ v, RowStrides ks, RowStrides vs,
                                                               bool aligned) {
  constexpr int kLanes = D / 8;
  const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row_id = id / kLanes;
  const int o = (int)(id % kLanes);
  const int row = (int)min(row_id, (long long)a.rows - 1);
  const int first = (int)min((id - (threadIdx.x & 63)) / kLanes, (long long)a.rows - 1);
  int sequence = 0, index = 0;
  bool live = find_sequence(a.offsets, a.sequences, first, row, sequence, index) && row_id < a.rows;
  uint8_t* tile = nullptr;
  int t = 0;
  if (live) {
    const long long p = (long long)a.start[sequence] + index;
    tile = a.start[sequence] < 0 ? nullptr : tile_of(a, sequence, p, cache_tile_bytes(D));
    t = (int)(p & (kCacheTile - 1));
  }
  if (tile == nullptr) return;  // four neighbouring lanes share a token, so whole quads leave
  const long long head_bytes = (long long)cache_tile_bytes(D) << a.page_shift;
  for (int head = blockIdx.y; head < a.kv_heads; head += gridDim.y) {
    uint8_t* at = tile + head * head_bytes;
    float x[8];
    unsigned scale;
    load8(k + row * ks.token + head * ks.head + o * 8, aligned, x);
    const unsigned k_codes = quantize8(x, scale);
    *reinterpret_cast<unsigned*>(at + t * (D / 2) + o * 4) = k_codes;
    if ((o & 3) == 0) at[key_scale_offset<D>(t, o >> 2)] = (uint8_t)scale;
    load8(v + row * vs.token + head * vs.head + o * 8, aligned, x);
    const unsigned v_codes = quantize8(x, scale);
    uint8_t* value = at + value_offset<D>(t, o);
    if constexpr (D == 64) {
      *reinterpret_cast<uint16_t*>(value) = (uint16_t)v_codes;
      *reinterpret_cast<uint16_t*>(value + 16) = (uint16_t)(v_codes >> 16);
    } else {
      *reinterpret_cast<unsigned*>(value) = v_codes;
    }
    if ((o & 3) == 0) at[value_scale_offset<D>(t, o >> 2)] = (uint8_t)scale;
  }
}

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = float4{x[0], x[1], x[2], x[3]};
  reinterpret_cast<float4*>(p)[1] = float4{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void store8(Half* p, const float (&x)[8]) {
  f16x8 h;
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = (_Float16)x[j];
  *reinterpret_cast<f16x8*>(p) = h;
}
__device__ __forceinline__ void store8(Bfloat* p, const float (&x)[8]) {
  bf16x8 h;
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = (__bf16)x[j];
  *reinterpret_cast<bf16x8*>(p) = h;
}

// The values that 8 codes and a scale byte stand for: exact in bf16 (two significant bits and its exponent range),
// and then in fp32.
__device__ __forceinline__ void values8(unsigned codes, unsigned scale, float (&x)[8]) {
  const float s = __uint_as_float(scale << 23);
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3);
  x[0] = (float)a[0]; x[1] = (float)a[1]; x[2] = (float)b[0]; x[3] = (float)b[1];
  x[4] = (float)c[0]; x[5] = (float)c[1]; x[6] = (float)d[0]; x[7] = (float)d[1];
}

template <int D, typename Out>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(CacheArgs a, Out* __restrict__ k, Out* __restrict__ v) {
  constexpr int kLanes = D / 8;
  const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row_id = id / kLanes;
  const int o = (int)(id % kLanes);
  const int row = (int)min(row_id, (long long)a.rows - 1);
  const int first = (int)min((id - (threadIdx.x & 63)) / kLanes, (long long)a.rows - 1);
  int sequence = 0, index = 0;
  const bool live = find_sequence(a.offsets, a.sequences, first, row, sequence, index);
  if (row_id >= a.rows) return;
  const uint8_t* tile = nullptr;
  int t = 0;
  if (live) {
    const int start = a.start == nullptr ? 0 : a.start[sequence];
    const long long p = (long long)start + index;
    tile = start < 0 ? nullptr : tile_of(a, sequence, p, cache_tile_bytes(D));
    t = (int)(p & (kCacheTile - 1));
  }
  const long long head_bytes = (long long)cache_tile_bytes(D) << a.page_shift;
  for (int head = blockIdx.y; head < a.kv_heads; head += gridDim.y) {
    float x[8] = {}, y[8] = {};
    if (tile != nullptr) {
      const uint8_t* at = tile + head * head_bytes;
      const unsigned k_codes = *reinterpret_cast<const unsigned*>(at + t * (D / 2) + o * 4);
      const unsigned k_scale = at[key_scale_offset<D>(t, o >> 2)];
      const uint8_t* value = at + value_offset<D>(t, o);
      unsigned v_codes;
      if constexpr (D == 64)
        v_codes = *reinterpret_cast<const uint16_t*>(value) | *reinterpret_cast<const uint16_t*>(value + 16) << 16;
      else
        v_codes = *reinterpret_cast<const unsigned*>(value);
      const unsigned v_scale = at[value_scale_offset<D>(t, o >> 2)];
      values8(k_codes, k_scale, x);
      values8(v_codes, v_scale, y);
    }
    const long long out = ((long long)row * a.kv_heads + head) * D + o * 8;
    store8(k + out, x);
    store8(v + out, y);
  }
}

// Blocks beyond which a thread takes several heads, sharing the page lookup.  65000 tokens read: 73.5 us so, 94.6 with
// a block per head; 64 tokens written and read back: 6.3 us so, 12.3 with all heads in one block.
constexpr long long kRowBlocks = 2048;

dim3 row_grid(const CacheArgs& a, int head_dim) {
  const long long blocks = ((long long)a.rows * (head_dim / 8) + kThreads - 1) / kThreads;
  long long heads = kRowBlocks / blocks;
  heads = heads < 1 ? 1 : heads > a.kv_heads ? a.kv_heads : heads;
  return dim3((unsigned)blocks, (unsigned)heads);
}

template <int D>
hipError_t write_rows(hipStream_t stream, const CacheArgs& a, int dtype, const void* k, const void* v, RowStrides ks,
                      RowStrides vs) {
  // Rows that start on 16 bytes are read in loads of 16 (fp32) or 8 bytes (half types), others value by value.
  const int size = dtype == kFloat32 ? 4 : 2;
  const bool aligned = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(ks.token * size) | (uintptr_t)(ks.head * size) |
                         (uintptr_t)(vs.token * size) | (uintptr_t)(vs.head * size)) & 15u) == 0;
  const dim3 grid = row_grid(a, D);
  if (dtype == kFloat32)
    hipLaunchKernelGGL((cache_write_kernel<D, float>), grid, dim3(kThreads), 0, stream, a,
                       static_cast<const float*>(k), static_cast<const float*>(v), ks, vs, aligned);
  else if (dtype == kFloat16)
    hipLaunchKernelGGL((cache_write_kernel<D, Half>), grid, dim3(kThreads), 0, stream, a, static_cast<const Half*>(k),
                       static_cast<const Half*>(v), ks, vs, aligned);
  else
    hipLaunchKernelGGL((cache_write_kernel<D, Bfloat>), grid, dim3(kThreads), 0, stream, a,
                       static_cast<const Bfloat*>(k), static_cast<const Bfloat*>(v), ks, vs, aligned);
  return hipGetLastError();
}

template <int D>
hipError_t read_rows(hipStream_t stream, const CacheArgs& a, int dtype, void* k, void* v) {
  const dim3 grid = row_grid(a, D);
  if (dtype == kFloat32)
    hipLaunchKernelGGL((cache_read_kernel<D, float>), grid, dim3(kThreads), 0, stream, a, static_cast<float*>(k),
                       static_cast<float*>(v));
  else if (dtype == kFloat16)
    hipLaunchKernelGGL((cache_read_kernel<D, Half>), grid, dim3(kThreads), 0, stream, a, static_cast<Half*>(k),
                       static_cast<Half*>(v));
  else
    hipLaunchKernelGGL((cache_read_kernel<D, Bfloat>), grid, dim3(kThreads), 0, stream, a, static_cast<Bfloat*>(k),
                       static_cast<Bfloat*>(v));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_write(hipStream_t stream, const CacheArgs& a, int head_dim, int dtype, const void* k,
                              const void* v, RowStrides ks, RowStrides vs) {
  if (a.rows == 0) return hipSuccess;
  if (head_dim == 64) return write_rows<64>(stream, a, dtype, k, v, ks, vs);
  if (head_dim == 128) return write_rows<128>(stream, a, dtype, k, v, ks, vs);
  return write_rows<256>(stream, a, dtype, k, v, ks, vs);
}

hipError_t launch_cache_read(hipStream_t stream, const CacheArgs& a, int head_dim, int dtype, void* k, void* v) {
  if (a.rows == 0) return hipSuccess;
  if (head_dim == 64) return read_rows<64>(stream, a, dtype, k, v);
  if (head_dim == 128) return read_rows<128>(stream, a, dtype, k, v);
  return read_rows<256>(stream, a, dtype, k, v);
}

}  // namespace ivo
