// Rows on their way into the 4-bit cache: the quantiser, where a token's codes and scales lie, and stores of eight
// values.
//
// Quantiser, for the 32 values x of a block: a = max |x|; exponent e = floor(log2(a * 8/7)) - 2, at least -100 and at
// most 125, so that a / 2^e < 7 and the largest value is at most half a step from the largest code, 6 (the exponent
// of a alone would leave a / 2^e up to 8 and cut a quarter off); code = the value nearest to x / 2^e, ties to the
// even code, at most 6; scale byte = e + 127.  In bits: the byte is (bits(a) + 0x200000) >> 23, less 2, since adding
// a quarter to the mantissa field carries where the mantissa is 1.75 and more.  A block that holds a NaN or an
// infinity gets the byte 255, which the conversions back turn into NaN.  The division and the rounding are
// v_cvt_scalef32_pk_fp4_f32, which rounds ties to even and saturates.
#pragma once

#include "cache_layout.hpp"

namespace ivo {

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

// A token's eight codes of K, and of V, and (from every fourth lane) the scale byte that four lanes share.
template <int D>
__device__ __forceinline__ void store_key(uint8_t* tile, int t, int o, unsigned codes, unsigned scale) {
  *reinterpret_cast<unsigned*>(tile + t * (D / 2) + o * 4) = codes;
  if ((o & 3) == 0) tile[key_scale_offset<D>(t, o >> 2)] = (uint8_t)scale;
}
template <int D>
__device__ __forceinline__ void store_cached_value(uint8_t* tile, int t, int o, unsigned codes, unsigned scale) {
  uint8_t* value = tile + value_offset<D>(t, o);
  if constexpr (D == 64) {
    *reinterpret_cast<uint16_t*>(value) = (uint16_t)codes;
    *reinterpret_cast<uint16_t*>(value + 16) = (uint16_t)(codes >> 16);
  } else {
    *reinterpret_cast<unsigned*>(value) = codes;
  }
  if ((o & 3) == 0) tile[value_scale_offset<D>(t, o >> 2)] = (uint8_t)scale;
}

__device__ __forceinline__ void store_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_value(Half* p, float x) { p->bits = bits_as<uint16_t>((_Float16)x); }
__device__ __forceinline__ void store_value(Bfloat* p, float x) { p->bits = bits_as<uint16_t>((__bf16)x); }

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

}  // namespace ivo
