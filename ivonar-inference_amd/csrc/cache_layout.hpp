// The 4-bit key/value cache: layout, limits, and device helpers shared by its kernels.
//
// pages: uint8 [pages, kv_heads, tiles, 34 * D], D in {64, 128, 256}.  A page holds `tiles` (a power of two) tiles of
// 32 tokens for every key/value head.  Sequence b's token at position p lies in page table[b, p / (32 * tiles)], tile
// (p / 32) % tiles, place t = p % 32.  A value has 4 bits (E2M1: sign, two exponent bits, one mantissa bit: 0, 0.5, 1,
// 1.5, 2, 3, 4, 6), and 32 neighbouring values of a row share a scale byte (exponent + 127; 255: not a number).
//
// A tile, with W = D / 32 (words of K per lane, bytes of V per lane and token, and scale groups per row alike):
//   K codes   at 0:    token-major rows of D / 2 bytes, byte i = dims 2i (low four bits), 2i + 1;
//   V codes   at 16 D: t = 16 s + 4 b + r, e = 4 s + r, dims 2 W n + 2 w, + 1 in byte w of n = 0..15:
//                      [e / (16 / W)][b][n][e % (16 / W)][w];
//   K scales  at 32 D: [group][t % 16][t / 16];
//   V scales  at 33 D: [group][b][e].
// So 16 bytes that a lane loads are operands of the 16x16x32 MFMA as they are: of K, 8 dims per word of one key (A
// operand: m = key, k = dims); of V, tokens 4b .. 4b + 3 and 16 + 4b .. of dims 2 W n .. (A operand: m = n, k =
// tokens), in the order in which the product of K and q leaves its results in the lanes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "internal.hpp"
#include "ternary_device.hpp"

namespace ivo {

constexpr int kCacheTile = 32;
constexpr int kCacheBlock = 32;  // values that share a scale
// Scale bytes written for finite blocks: 2^-100 keeps products of the pieces that q is split into away from
// subnormals, 2^125 keeps 6 * scale finite in fp32.
constexpr int kScaleMin = 27;
constexpr int kScaleMax = 252;
constexpr unsigned kScaleNan = 255;

__host__ __device__ constexpr bool cache_head_dim(int d) { return d == 64 || d == 128 || d == 256; }
__host__ __device__ constexpr int cache_tile_bytes(int d) { return 34 * d; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename To, typename From>
__device__ __forceinline__ To bits_as(const From& v) {
  static_assert(sizeof(To) == sizeof(From), "same size");
  To out;
  __builtin_memcpy(&out, &v, sizeof(To));
  return out;
}

// Eight neighbouring values as fp32: in loads of 16 or 8 bytes where rows start on 16 bytes, else one by one.
template <typename In>
__device__ __forceinline__ void load8(const In* p, bool aligned, float (&x)[8]) {
  if (aligned) {
    const float4 a = load4(p, 0), b = load4(p, 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = to_float(p[j]);
  }
}

// Which sequence of a ragged batch a row belongs to, and its index there.  offsets is the row prefix [sequences + 1]
// on the device, or null where every sequence has one row.  All lanes of the wave call this together with rows that
// do not decrease from lane to lane; `first` is the wave's smallest row.  A row of no sequence gives false.  One load
// per 64 sequences and a ballot find the first row's sequence (a binary search would wait for log2(sequences)
// dependent loads); the other lanes step on from there.
__device__ __forceinline__ bool find_sequence(const int* offsets, int sequences, int first, int row, int& sequence,
                                              int& index) {
  if (offsets == nullptr) {
    sequence = row;
    index = 0;
    return row < sequences;
  }
  int before = 0;  // sequences whose end lies at or before `first`
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < sequences; base += 64) {
    const bool ended = base + lane < sequences && offsets[1 + base + lane] <= first;
    before += __popcll(__ballot(ended));
  }
  while (before < sequences && offsets[before + 1] <= row) ++before;
  sequence = before;
  if (before >= sequences) return false;
  index = row - offsets[before];
  return index >= 0;
}

}  // namespace ivo
