// Log probabilities of given tokens, the entropy, and the likeliest alternatives, of rows of logits, in one pass.
//
// For a row x of V logits and a temperature T, with m = max x, z_i = (x_i - m) / T, S = sum e^z_i, U = sum z_i e^z_i:
//   log p_i = z_i - log S,   H = -sum p_i log p_i = log S - U / S.
// m, S and U are kept per thread in fp32 and rescaled when a chunk raises m: S' = f S, U' = f (U + d S) for a maximum
// that rises by -d T, f = e^d.  In units of log 2, z = x c - M with c = log2(e) / T and M = m c rounded to fp32: one
// rounding of z itself, and since everything is relative to the same M, that of M does not count as long as it is half a
// unit at most, |M| < 2^24.  From there on it would be the largest weight's exponent (2^128 and more from |M| = 2^31 on,
// as of masked logits or low temperatures), and z = (x - m) c instead.  A logit of -inf has no weight; a row of nothing
// else has log probabilities of -inf and no entropy.  A NaN or +inf makes all of its row's numbers NaN.
//
// The `top` largest logits are found in the same pass.  A logit's key is its value as an ordered number, then its index
// from the end, so no two keys are alike and ties go to the lowest index; a NaN has the lowest value.  A wave keeps the
// 64 largest keys that it has met, or 32 where those are enough, sorted over its lanes, and a bound below which a key cannot be among the row's top:
// the top'th of them, or of the first chunk's per-lane maxima, or what another wave of the row has found.  Most chunks
// hold no logit above the bound, which their maxima tell.  Keys above it go through a buffer in LDS and are sorted and
// merged 64 at a time.
//
// A wave takes 2048 logits at a time, 32 per lane; the next ones are under way while these are used.  Few long rows are
// split between blocks, whose results a second kernel joins.
//
// Bound by the logits' bytes where there are many: 500 rows of 32000 in fp32 14.5 us without alternatives (4.4 TB/s) and
// 18.8 with 5; 2048 rows of 100003 in bf16 95 us with 20 (4.3 TB/s; their rows start anywhere, which costs a tenth),
// where vector instructions take three quarters of the SIMDs' cycles, and as many more where most logits are masked by
// -1e9 (95 us for 87 with masks of -1e4).  One row of 32000 takes 5.8 us, and 11.3 with 20:
// a chain of about fifty compare stages of sorts and merges (with lists of 64 keys, seventy stages, 12.3).
#include "internal.hpp"
#include "ternary_device.hpp"

namespace ivo {
namespace {

constexpr int kWaves = 4;                   // of a block
constexpr int kManyWaves = 16;              // of a block where there are few rows
constexpr int kValues = 32;                 // logits of a lane at a time
constexpr int kWaveChunk = 64 * kValues;    // and of a wave
constexpr int kBuffer = 128;                // keys above the bound that a wave holds before it merges 64
constexpr float kFar = 0x1p24f;             // |m c| from which on the rounding of it counts
constexpr float kOverflow = 0x1p100f;       // |x c| below which z is in range
constexpr int kCrowd = 12;                  // logits of a lane above the first bound that tell of ties
typedef unsigned long long Key;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct Params {
  ScoreArgs a;
  float scale;   // log2(e) / T
  int splits;    // blocks that share a row
  int waves;      // of a block: kWaves or kManyWaves
  int row_waves;  // that share a row
};

constexpr float kLog2 = 0.69314718055994530942f;

// What a part of a row leaves: m, S, U (in units of log 2), and its largest keys.
struct Part {
  float m, sum, weighted;
  Key list;  // of 64, this lane's
};
constexpr int kPartFloats = 4 + 2 * 64;

// 16 bytes of logits as fp32.
template <typename In>
__device__ __forceinline__ void unpack(const u32x4& words, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(In) == 4) {
      x[j] = __uint_as_float(words[j]);
    } else {
      x[2 * j] = to_float(In{(uint16_t)words[j]});
      x[2 * j + 1] = to_float(In{(uint16_t)(words[j] >> 16)});
    }
  }
}

__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned bits = __float_as_uint(x + 0.0f);  // -0 counts as 0
  const unsigned key = bits ^ ((unsigned)((int)bits >> 31) | 0x80000000u);
  return x != x ? 0u : key;
}
__device__ __forceinline__ float value_of(Key key) {
  const unsigned high = (unsigned)(key >> 32);
  if (high == 0u) return NAN;
  return __uint_as_float(high & 0x80000000u ? high ^ 0x80000000u : ~high);
}
__device__ __forceinline__ Key key_of(float x, int index) {
  return (Key)ordered(x) << 32 | (unsigned)~index;
}

template <int X>
__device__ __forceinline__ float keep(float v, bool larger) {
  const float other = xor_lane<X>(v);
  return larger ? fmaxf(v, other) : fminf(v, other);
}

// Compares with lane ^ X and keeps the larger key or the smaller one.
template <int X>
__device__ __forceinline__ Key keep(Key key, bool larger) {
  const Key other = (Key)xor_lane<X>((unsigned)(key >> 32)) << 32 | xor_lane<X>((unsigned)key);
  return (other > key) == larger ? other : key;
}
// Keys (or numbers alone) that rise and then fall, or the reverse, over SIZE lanes, sorted: falling where `falling`.
template <int SIZE, typename V>
__device__ __forceinline__ V merge_lanes(V v, int lane, bool falling) {
  if constexpr (SIZE > 1) {
    v = keep<SIZE / 2>(v, ((lane & (SIZE / 2)) == 0) == falling);
    v = merge_lanes<SIZE / 2>(v, lane, falling);
  }
  return v;
}
template <int SIZE, typename V>
__device__ __forceinline__ V sort_parts(V v, int lane) {
  if constexpr (SIZE > 2) v = sort_parts<SIZE / 2>(v, lane);
  return merge_lanes<SIZE>(v, lane, SIZE < 64 && (lane & SIZE) != 0);
}
// The lane, as a number that the compiler cannot form the stages' masks from ahead of a loop: they would take up most
// of the scalar registers.
__device__ __forceinline__ int opaque_lane() {
  int lane = threadIdx.x;
  asm volatile("" : "+v"(lane));
  return lane;
}
// Sorted over the wave, rising from lane 0 on.
template <typename V>
__device__ __forceinline__ V sort_lanes(V v) { return sort_parts<64>(v, opaque_lane()); }

// The KEEP largest of a falling list and a rising one, over the first KEEP lanes, falling.
template <int KEEP>
__device__ __forceinline__ Key join(Key falling, Key rising) {
  return merge_lanes<KEEP>(falling > rising ? falling : rising, opaque_lane(), true);
}
// The 32 largest of a falling list and of `count` keys, one a lane.
__device__ __forceinline__ Key add_keys32(Key list, Key keys, int count) {
  const int lane = opaque_lane();
  keys = sort_parts<32>(keys, lane);  // the first half rises, the other falls
  list = join<32>(list, keys);
  if (count > 32) list = join<32>(list, __shfl(keys, 63 - lane));
  return list;
}
__device__ __forceinline__ Key lane_key(Key key, int lane) {
  return (Key)(unsigned)__builtin_amdgcn_readlane((int)(key >> 32), lane) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)key, lane);
}

__device__ __forceinline__ float all_max(float v) {
  v = fmaxf(v, xor_lane<1>(v));
  v = fmaxf(v, xor_lane<2>(v));
  v = fmaxf(v, xor_lane<4>(v));
  v = fmaxf(v, xor_lane<8>(v));
  v = fmaxf(v, xor_lane<16>(v));
  return fmaxf(v, xor_lane<32>(v));
}
__device__ __forceinline__ float all_sum(float v) {
  v += xor_lane<1>(v);
  v += xor_lane<2>(v);
  v += xor_lane<4>(v);
  v += xor_lane<8>(v);
  v += xor_lane<16>(v);
  return v + xor_lane<32>(v);
}

// z no further down than where its weight is zero: zero times the result is zero.
__device__ __forceinline__ float bounded(float z) { return fmaxf(z, -1000.0f); }

// M, and none of a maximum of nothing.
__device__ __forceinline__ float scaled(float m, float scale) { return m == -INFINITY ? 0.0f : m * scale; }
// What is relative to m has z = (x - m) c where m is far and else z = x c - M.
__device__ __forceinline__ bool is_far(float m, float scale) { return fabsf(scaled(m, scale)) >= kFar; }
// (x - m) factor, by halves, whose difference is in range.
__device__ __forceinline__ float apart(float x, float m, float factor) {
  return fmaf(0.5f, x, -0.5f * m) * (2.0f * factor);
}

// S and U moved to the maximum `to`.
__device__ __forceinline__ void raise(float& m, float& sum, float& weighted, float to, float scale) {
  const bool from_far = is_far(m, scale), to_far = is_far(to, scale);
  float between = m * scale - to * scale;
  if (from_far || to_far)
    between = !to_far    ? fmaf(m, scale, -(to * scale))
              : from_far ? apart(m, to, scale)
                         : fmaf(-to, scale, m * scale);
  const float d = bounded(between);
  const float factor = __builtin_amdgcn_exp2f(d);
  weighted = fmaf(sum, d, weighted) * factor;
  sum *= factor;
  m = to;
}

// The results of a row, by one wave that holds it whole.
__device__ __forceinline__ void finish(const Params& p, int row, const Part& part) {
  const ScoreArgs& a = p.a;
  const int lane = threadIdx.x & 63;
  const float log_sum = log2f(part.sum);
  const bool none = part.sum == 0.0f, far = is_far(part.m, p.scale);
  auto log_probability = [&](float x) {
    if (none) return -INFINITY;
    // In nats, which may be in range where units of log 2 are not.
    if (far || fabsf(x * p.scale) >= kOverflow) return apart(x, part.m, a.inverse_temperature) - kLog2 * log_sum;
    return kLog2 * (fmaf(x, p.scale, -scaled(part.m, p.scale)) - log_sum);
  };
  if (lane == 0) {
    const int64_t token = a.tokens[row];
    float chosen = -INFINITY;
    if (token >= 0 && token < a.vocab) {
      const long long at = row * a.row_stride + token;
      const float x = a.dtype == kFloat32 ? static_cast<const float*>(a.logits)[at]
                      : a.dtype == kFloat16 ? to_float(static_cast<const Half*>(a.logits)[at])
                                            : to_float(static_cast<const Bfloat*>(a.logits)[at]);
      chosen = log_probability(x);
    }
    a.log_probability[row] = chosen;
    a.entropy[row] = none ? 0.0f : kLog2 * (log_sum - part.weighted / part.sum);
  }
  if (lane < a.top) {
    const long long at = (long long)row * a.top + lane;
    a.top_log_probability[at] = log_probability(value_of(part.list));
    a.top_token[at] = (int64_t)(int)~(unsigned)part.list;
  }
}

// TOP: how many keys a list has, 64, 32 or none.
template <typename In, int TOP, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 4) void score_kernel(Params p) {
  constexpr int kVec = 16 / sizeof(In), kVectors = kValues / kVec;
  const ScoreArgs& a = p.a;
  __shared__ Key buffers[TOP ? WAVES : 1][TOP ? kBuffer : 1];
  __shared__ __align__(16) float places[TOP ? WAVES : 1][TOP ? 64 : 1][kValues];
  __shared__ Key bounds[WAVES];  // of each row of the block, the best bound so far
  __shared__ float sums[WAVES][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sub = wave & (p.row_waves - 1), first_wave = wave - sub;
  const int split = blockIdx.x % p.splits;
  const long long row_id = (long long)(blockIdx.x / p.splits) * (WAVES / p.row_waves) + wave / p.row_waves;
  const bool there = row_id < a.rows;
  const int row = (int)(there ? row_id : a.rows - 1);
  if (TOP) {
    if (threadIdx.x < WAVES) bounds[threadIdx.x] = 0;
    __syncthreads();
  }

  // The row's whole 16-byte vectors in chunks, and up to 2 (kVec - 1) logits before and behind them in a last one.
  const In* begin = static_cast<const In*>(a.logits) + row * a.row_stride;
  const int lead = (int)(((uintptr_t)begin & 15u) / sizeof(In));
  const int head = lead == 0 ? 0 : min(kVec - lead, a.vocab);
  const int vectors = (a.vocab - head) / kVec, whole = (vectors + 64 * kVectors - 1) / (64 * kVectors);
  const int rest = a.vocab - vectors * kVec;  // head + tail
  const int chunks = there ? whole + (rest > 0 ? 1 : 0) : 0;
  const int rest_index = lane < head ? lane : lane < rest ? vectors * kVec + lane : -1;
  const int step = p.splits * p.row_waves;
  const u32x4* const aligned = reinterpret_cast<const u32x4*>(begin + head);
  auto load = [&](int chunk, u32x4 (&to)[kVectors]) {
    if (chunk < whole) {
      // Places past the last vector take that one, and are cleared when they are used.
#pragma unroll
      for (int v = 0; v < kVectors; ++v) to[v] = aligned[min((chunk * kVectors + v) * 64 + lane, vectors - 1)];
    } else {
      In values[kVec];
      values[0] = begin[max(rest_index, 0)];
#pragma unroll
      for (int j = 1; j < kVec; ++j) values[j] = In{};
      __builtin_memcpy(&to[0], values, 16);
    }
  };

  float m = -INFINITY, sum = 0.0f, weighted = 0.0f;
  Key list = 0, bound = 0;
  int held = 0;  // keys in the buffer
  Key* buffer = buffers[TOP ? wave : 0];
  float(*found)[kValues] = places[TOP ? wave : 0];
  // Merges the first `count` keys of the buffer into the list.
  auto merge = [&](int count) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    Key key = buffer[lane];
    key = lane < count ? key : 0;
    if constexpr (TOP == 32)
      list = add_keys32(list, key, count);
    else
      list = join<64>(list, sort_lanes(key));
    const Key last = lane_key(list, a.top - 1);
    bound = last > bound ? last : bound;
    if (lane == 0) atomicMax(&bounds[first_wave], bound);
  };

  u32x4 current[kVectors], next[kVectors];
  int chunk = split * p.row_waves + sub;
  if (chunk < chunks) load(chunk, current);
  for (; chunk < chunks; chunk += step) {
    if (chunk + step < chunks) load(chunk + step, next);
    float x[kValues];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) unpack<In>(current[v], x + v * kVec);
    if (chunk >= whole - 1) {
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        const bool inside = chunk < whole ? (chunk * kVectors + j / kVec) * 64 + lane < vectors
                                          : j == 0 && rest_index >= 0;
        x[j] = inside ? x[j] : -INFINITY;
      }
    }
    float most = x[0];
#pragma unroll
    for (int j = 1; j < kValues; ++j) most = fmaxf(most, x[j]);
    if (most > m) raise(m, sum, weighted, most, p.scale);
    const float shift = scaled(m, p.scale);
    float part_sum[2] = {}, part_weighted[2] = {};
    const bool far = fabsf(shift) >= kFar;
    bool slow = __ballot(far) != 0ull;
    if (!slow) {
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        const float z = fmaf(x[j], p.scale, -shift);
        const float weight = __builtin_amdgcn_exp2f(z);
        part_sum[j & 1] += weight;
        part_weighted[j & 1] = fmaf(z, weight, part_weighted[j & 1]);  // no number for -inf
        if (j % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // or all weights would be held at once
      }
      const float of_sum = part_sum[0] + part_sum[1], of_weighted = part_weighted[0] + part_weighted[1];
      slow = __ballot(of_weighted != of_weighted && of_sum == of_sum) != 0ull;
    }
    if (slow) {
      part_sum[0] = part_sum[1] = part_weighted[0] = part_weighted[1] = 0.0f;
      float again = shift;
      asm volatile("" : "+v"(again));  // or the compiler would hold all z from above for here
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        const float z = far ? apart(x[j], m, p.scale) : fmaf(x[j], p.scale, -again);
        const float weight = __builtin_amdgcn_exp2f(z);
        part_sum[j & 1] += weight;
        part_weighted[j & 1] = fmaf(bounded(z), weight, part_weighted[j & 1]);
        if (j % 8 == 7) __builtin_amdgcn_sched_barrier(0);
      }
    }
    sum += part_sum[0] + part_sum[1];
    weighted += part_weighted[0] + part_weighted[1];

    if constexpr (TOP > 0) {
      const Key shared = *(volatile Key*)&bounds[first_wave];
      bound = shared > bound ? shared : bound;
      // The lane's logit j in the row, outside the vocabulary where it has none.
      const int start = chunk < whole ? head + chunk * kWaveChunk : -1;
      auto index_of = [&](int j) {
        const int vector = (chunk * kVectors + j / kVec) * 64 + lane;
        if (chunk < whole) return vector < vectors ? head + vector * kVec + j % kVec : -1;
        return j == 0 ? rest_index : -1;
      };
      const bool first = bound == 0;
      if (first) {
        // Of the lanes' largest logits the top'th is no larger than that of all.
        const float largest = sort_lanes(fmaxf(most, -INFINITY));
        const float last =
            __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(largest), 64 - a.top));
        // Below the keys of its value: those of the number before it (before +0 comes -0, which compares like it).
        if (last > -INFINITY) bound = ((Key)(ordered(last) - (last == 0.0f ? 1u : 0u)) << 32) - 1;
      }
      unsigned above = 0;  // bit j: logit j may be
      // Behind the bound's index equal logits are below it.  Without a bound, and where it is that of a NaN, all logits
      // may be above it.
      auto compare = [&]() {
        const float least = value_of(bound);
        above = 0;
        if (bound >> 32 != 0 && start > (int)~(unsigned)bound) {
          if (__ballot(most > least) != 0ull)
#pragma unroll
            for (int j = kValues - 1; j >= 0; --j) above = above + above + (x[j] > least ? 1u : 0u);
        } else if (__ballot(!(most < least)) != 0ull) {
#pragma unroll
          for (int j = kValues - 1; j >= 0; --j) above = above + above + (!(x[j] < least) ? 1u : 0u);
        }
      };
      compare();
      if (first && __ballot(__popc(above) >= kCrowd) != 0ull) {
        // Ties: the top'th of the lanes' largest keys.
        int best = -1;
#pragma unroll
        for (int j = kValues - 1; j >= 0; --j) {
          const int index = index_of(j);
          best = x[j] == most && (unsigned)index < (unsigned)a.vocab ? index : best;
        }
        const Key key = sort_lanes(best >= 0 ? key_of(most, best) : 0);
        const Key last = lane_key(key, 64 - a.top);
        bound = last > bound + 1 ? last - 1 : bound;
        compare();
      }
      if (above != 0u) {
        // For the loop below, which takes a lane's logits by number: loads of them, though near, would take longer.
#pragma unroll
        for (int j = 0; j < kValues; j += 4)
          *reinterpret_cast<float4*>(&found[lane][j]) = float4{x[j], x[j + 1], x[j + 2], x[j + 3]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
      while (__ballot(above != 0u) != 0ull) {
        bool add = false;
        Key key = 0;
        if (above != 0u) {
          const int j = __builtin_ctz(above);
          above &= above - 1u;
          const int index = index_of(j);
          if ((unsigned)index < (unsigned)a.vocab) {
            key = key_of(found[lane][j], index);
            add = key > bound;
          }
        }
        const unsigned long long adds = __ballot(add);
        if (add) buffer[held + __popcll(adds & ((1ull << lane) - 1ull))] = key;
        held += __popcll(adds);
        if (held >= 64) {
          merge(64);
          const Key rest = buffer[64 + lane];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          buffer[lane] = rest;
          held -= 64;
        }
      }
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) current[v] = next[v];
  }
  if (TOP && held > 0) merge(held);
  if (TOP == 32 && lane >= 32) list = 0;

  Part part;
  part.m = all_max(m);
  raise(m, sum, weighted, part.m, p.scale);
  part.sum = all_sum(sum);
  part.weighted = all_sum(weighted);
  part.list = list;
  // The parts of a row's waves, four at a time.
  for (int apart = 1; apart < p.row_waves; apart *= 4) {
    if (apart > 1) __syncthreads();  // the parts have been read
    if (lane == 0) {
      sums[wave][0] = part.m;
      sums[wave][1] = part.sum;
      sums[wave][2] = part.weighted;
    }
    if (TOP) buffer[lane] = part.list;
    __syncthreads();
    if (sub % (4 * apart) != 0) continue;
    for (int w = sub + apart; w < min(sub + 4 * apart, p.row_waves); w += apart) {
      float other_m = sums[first_wave + w][0], other_sum = sums[first_wave + w][1];
      float other_weighted = sums[first_wave + w][2];
      const float top = fmaxf(part.m, other_m);
      raise(part.m, part.sum, part.weighted, top, p.scale);
      raise(other_m, other_sum, other_weighted, top, p.scale);
      part.sum += other_sum;
      part.weighted += other_weighted;
      if constexpr (TOP == 64) part.list = join<64>(part.list, buffers[first_wave + w][63 - lane]);
    }
    if constexpr (TOP == 32) {
      // Of 32 keys two lists at a time, in either half of the lanes, the upper one rising, and then those.
      auto key_of_wave = [&](int w, int at) { return w < p.row_waves ? buffers[first_wave + w][at] : 0; };
      const bool low = lane < 32;
      const Key falling = low ? part.list : key_of_wave(sub + 2 * apart, lane & 31);
      const Key rising = key_of_wave(low ? sub + apart : sub + 3 * apart, 31 - (lane & 31));
      const Key two = merge_lanes<32>(falling > rising ? falling : rising, opaque_lane(), low);
      part.list = join<32>(two, (Key)xor_lane<32>((unsigned)(two >> 32)) << 32 | xor_lane<32>((unsigned)two));
      if (!low) part.list = 0;
    }
  }
  if (sub != 0) return;
  if (!there) return;
  if (p.splits == 1) {
    finish(p, row, part);
  } else {
    float* to = a.work + ((long long)row * p.splits + split) * kPartFloats;
    if (lane == 0) *reinterpret_cast<float4*>(to) = float4{part.m, part.sum, part.weighted, 0.0f};
    if (TOP) reinterpret_cast<Key*>(to + 4)[lane] = part.list;
  }
}

// Joins the parts of split rows, a wave per row.
__global__ __launch_bounds__(kThreads) void join_kernel(Params p) {
  const int lane = threadIdx.x & 63;
  const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  if (row >= p.a.rows) return;
  const float* from = p.a.work + (long long)row * p.splits * kPartFloats;
  Part part;
  part.m = -INFINITY;
  part.sum = part.weighted = 0.0f;
  part.list = 0;
  for (int i = lane; i < p.splits; i += 64) {
    float4 other = *reinterpret_cast<const float4*>(from + (long long)i * kPartFloats);
    const float top = fmaxf(part.m, other.x);
    raise(part.m, part.sum, part.weighted, top, p.scale);
    raise(other.x, other.y, other.z, top, p.scale);
    part.sum += other.y;
    part.weighted += other.z;
  }
  const float top = all_max(part.m);
  raise(part.m, part.sum, part.weighted, top, p.scale);
  part.sum = all_sum(part.sum);
  part.weighted = all_sum(part.weighted);
  if (p.a.top > 0) {
    constexpr int kAtOnce = 8;
    for (int base = 0; base < p.splits; base += kAtOnce) {
      Key lists[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const long long i = min(base + k, p.splits - 1);
        lists[k] = reinterpret_cast<const Key*>(from + i * kPartFloats + 4)[63 - lane];
      }
      for (int k = 0; k < kAtOnce && base + k < p.splits; ++k) {
        part.list = join<64>(part.list, lists[0]);
#pragma unroll
        for (int j = 0; j + 1 < kAtOnce; ++j) lists[j] = lists[j + 1];
      }
    }
  }
  finish(p, row, part);
}

// Waves of all rows that keep the device busy, blocks that few long rows are split into, and chunks of a wave that are
// not split.
constexpr int kBusyWaves = 4096, kWantedBlocks = 1024, kLeastChunks = 4;
// Few rows of middling length take a block of sixteen waves each, up to two chunks a wave: top 20 of 1 x 32000 fp32 12.3
// us and of 32 x 50000 bf16 15.8, with four waves 13.7 and 19.3 (lists of 64 keys).  Longer rows are faster in several
// blocks of four waves (1 x 128256 bf16 20.0 us and 22.3), and more rows than compute units fill the device that way.
constexpr int kManyRows = 256, kManyLeast = 8, kManyMost = 32;

Params plan(const ScoreArgs& a) {
  Params p{a, 1.44269504088896340736f * a.inverse_temperature, 1, kWaves, kWaves};
  const int chunks = (int)(((long long)a.vocab + kWaveChunk - 1) / kWaveChunk);
  if (a.rows <= kManyRows && chunks >= kManyLeast && chunks <= kManyMost) p.waves = p.row_waves = kManyWaves;
  while (p.waves == kWaves && p.row_waves > 1 &&
         ((long long)a.rows * p.row_waves >= 2 * kBusyWaves || chunks <= p.row_waves / 2))
    p.row_waves /= 2;
  if (p.row_waves == kWaves)
    p.splits = max(1, min(kWantedBlocks / max(1, a.rows), chunks / (kWaves * kLeastChunks)));
  return p;
}

template <typename In, int WAVES>
void run_waves(hipStream_t stream, const Params& p, unsigned blocks) {
  if (p.a.top > 32)
    hipLaunchKernelGGL((score_kernel<In, 64, WAVES>), dim3(blocks), dim3(WAVES * 64), 0, stream, p);
  else if (p.a.top > 0)
    hipLaunchKernelGGL((score_kernel<In, 32, WAVES>), dim3(blocks), dim3(WAVES * 64), 0, stream, p);
  else
    hipLaunchKernelGGL((score_kernel<In, 0, WAVES>), dim3(blocks), dim3(WAVES * 64), 0, stream, p);
}
template <typename In>
void run(hipStream_t stream, const Params& p, unsigned blocks) {
  if (p.waves == kWaves)
    run_waves<In, kWaves>(stream, p, blocks);
  else
    run_waves<In, kManyWaves>(stream, p, blocks);
}

}  // namespace

long long score_work(const ScoreArgs& a) {
  const Params p = plan(a);
  return p.splits == 1 ? 0 : (long long)a.rows * p.splits * kPartFloats * 4;
}

hipError_t launch_score(hipStream_t stream, const ScoreArgs& a) {
  if (a.rows == 0) return hipSuccess;
  const Params p = plan(a);
  const int block_rows = p.waves / p.row_waves;
  const long long blocks = ((long long)a.rows + block_rows - 1) / block_rows * p.splits;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (a.dtype == kFloat32)
    run<float>(stream, p, (unsigned)blocks);
  else if (a.dtype == kFloat16)
    run<Half>(stream, p, (unsigned)blocks);
  else
    run<Bfloat>(stream, p, (unsigned)blocks);
  if (p.splits > 1)
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)((a.rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace ivo
