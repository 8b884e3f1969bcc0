// Attention of a few query rows over the 4-bit cache (layout: cache_layout.hpp; a run of tiles: attention_cache.hpp).
//
// Up to 8 rows per sequence: the keys of all sequences are dealt out evenly to as many blocks as the device holds;
// where that cuts a row tile's keys, the last of its blocks to end adds the parts (unscaled sums, m, sum).  More rows:
// row tiles are split at equal lengths where there are too few of them, and a second kernel adds their parts.
//
// Measured (MI355X, calls back to back).  One token per sequence, bound by the cache's bytes: 64 sequences of 1000 to
// 8000 tokens (288000 in all), 32/8 heads of 128, bf16: 67 us, 4.7 TB/s (a stream of the same 313 MB reads at 6.5;
// loads alone took 64); one of 131000, fp16: 36.5 us, 3.9 TB/s (142 MB more take 23 us more: the rest is filling the
// device and adding the parts); 128 with a window of 1024, 16/4 heads of 64: 15.2 us, 2.4 TB/s; one of 37, fp32: 6.4 us
// in a graph, a chain of loads.  Chunks, bound by the vector units, which convert the codes and the weights next to the
// matrix units' work: 512 rows over 8702 tokens, 32/8 heads of 128, bf16: 120 us, 590 TFLOP/s (890 counting both terms
// of P); fp16 142 us, fp32 223 us, with more terms of q and P.
#include "attention_cache.hpp"

namespace ivo {
namespace {

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
  constexpr int RT = R == 8 ? 1 : R / 16;
  const CacheAttentionArgs& a = p.a;
  __shared__ __align__(16) unsigned char room_bytes[sizeof(Room<D>)];
  Room<D>& room = *reinterpret_cast<Room<D>*>(room_bytes);
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
    int row0, queries;
    if (!row_tile<R>(p, slot, run.sequence, row0, queries, run.start)) return;
    const Span s = make_span<R>(p, run.sequence, row0, queries, a.lengths[run.sequence], run.start);
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
    const bool all = begin == 0 && end == s.total;
    const int at_part = (int)part * (R * (D + 2)) * 4;
    auto put = [&](int line, int column, int row, float top, float total, const float4& sum) {
      if (all) {
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        const int token = row / p.group, h = row - token * p.group;
        In* to = static_cast<In*>(a.out) + ((long long)(s.row0 + token) * a.heads + head * p.group + h) * D + column;
        store4(to, float4{sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse});
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(bits_as<u32x4>(sum), parts_buffer(a.work),
                                               at_part + (line * D + column) * 4, 0, kDeviceScope);
        if (column == 0)
          __builtin_amdgcn_raw_buffer_store_b64(bits_as<u32x2>(float2{top, total}), parts_buffer(a.work),
                                                at_part + (R * D + 2 * line) * 4, 0, kDeviceScope);
      }
    };
    attend_run<D, In, R, NT, STREAM, false>(p, s, head, begin, end, wave, room, stats, put);

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
                            &room.sums[0][0][0]);
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
  const long long first = (long long)(slot_of<R>(p, sequence, row0) + line / R) * p.splits * a.kv_heads + head;
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
