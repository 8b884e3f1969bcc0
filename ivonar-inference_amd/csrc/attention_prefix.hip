// Attention over the 4-bit cache of sequences that share the pages of a long prefix, group by group (a run of tiles:
// attention_cache.hpp).
//
// The sequences groups[g] .. groups[g + 1] - 1 hold their first prefix[g] tokens in the same pages.  The softmax over all
// of a row's keys is the sum over two stretches of them, each with its own maximum m, sum l and weighted values o:
//   m = max(m1, m2), out = (2^(m1 - m) o1 + 2^(m2 - m) o2) / (2^(m1 - m) l1 + 2^(m2 - m) l2).
// One launch takes the rows of a group together over the prefix, read through a table row of theirs, as
// if they were one sequence's: a tile of keys is loaded and converted once for 32 rows instead of for each sequence's
// few.  The next takes each sequence's own keys behind it and adds the prefix's parts.  A row sees the whole prefix, so
// where a sequence's rows begin before its end, the group's prefix ends there: P_g is the least of prefix[g] and the
// positions of its sequences' first rows, and what lies behind it is read through each sequence's own table row.  Rows
// of a sequence without tokens, as in a padded batch, see nothing, and its group's prefix is as long without it.
//
// The prefix is bound by the instructions that convert keys and values and take the softmax, beside the matrix cores: 256
// sequences of one row over 16000 tokens, 32/8 heads of 128, bf16: 122 us, 550 TFLOP/s (820 with the second terms of the
// weights), vector units busy 60 % of the cycles and matrix units 35 %, which overlap by half at best.  64 rows of a row
// tile instead of 32, so with half the conversions, leave room for one wave per SIMD: 139 us instead of 128.  The tails
// are bound by their bytes: 500 tokens each of the same 256 36 us, 3.9 TB/s.  Short calls are two launches' chains of
// dependent loads (offsets, lengths, page, tile): 8 sequences of 501 tokens 7.6 us and 6.0.  Both in one launch, the tails
// beside the prefix and the join by the last to arrive, took 42 us where two take 25 and 12.
#include "attention_cache.hpp"

namespace ivo {
namespace {

// Blocks per CU that the registers leave room for: as the cache attention's, and three where without its bookkeeping
// they do.
constexpr int resident(int D, int R, int NT) { return D == 64 && R == 32 && NT == 2 ? 3 : occupancy(D, R, NT); }

struct SharedParams {
  Params p;
  const int* groups;
  const int* prefix;
  int group_count;
  int prefix_rows;  // of a row tile over the prefix
  int prefix_slots, prefix_splits, prefix_chunk;
  int tail_splits, tail_chunk;
  int* shared;         // [group_count]: P_g
  float* prefix_work;  // parts, each the row tile's sums, then the maxima and sums of its weights
  float* tail_work;
};

__device__ __forceinline__ int row_before(const CacheAttentionArgs& a, int sequence) {
  return max(0, min(a.offsets == nullptr ? sequence : a.offsets[sequence], a.rows));
}
// A group's sequences and their rows.
struct Group {
  int begin, end;
  int row0, rows;
};
__device__ __forceinline__ Group group_of(const SharedParams& sp, int g) {
  const CacheAttentionArgs& a = sp.p.a;
  Group group;
  group.begin = max(0, min(sp.groups[g], a.sequences));
  group.end = max(group.begin, min(sp.groups[g + 1], a.sequences));
  group.row0 = row_before(a, group.begin);
  group.rows = max(0, row_before(a, group.end) - group.row0);
  return group;
}
// Tokens that all rows of a group see through the shared pages, and the sequence whose table row is read for them, the
// first that has rows.  Sequences without tokens do not count: their rows see nothing.  All lanes of a wave call this
// together.
__device__ __forceinline__ int shared_tokens(const SharedParams& sp, int g, const Group& group, int& source) {
  const CacheAttentionArgs& a = sp.p.a;
  int least = sp.prefix[g], first = group.end;
  for (int b = group.begin + (int)(threadIdx.x & 63); b < group.end; b += 64) {
    int row0;
    const int rows = rows_of(a, b, row0), length = a.lengths[b];
    if (rows > 0 && length > 0) {
      least = min(least, length - rows);
      first = min(first, b);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    least = min(least, __shfl_xor(least, o));
    first = min(first, __shfl_xor(first, o));
  }
  source = uniform(first);
  return source < group.end ? uniform(max(least, 0)) : 0;
}
// First row tile of a group: leaves each group at least as many as it needs.
__device__ __forceinline__ int first_slot(const SharedParams& sp, int g, int row0) {
  return (int)((long long)row0 * sp.p.group / sp.prefix_rows) + g;
}
__device__ __forceinline__ int tiles_in_table(const CacheAttentionArgs& a, int tokens) {
  return min((tokens + kCacheTile - 1) / kCacheTile, a.table_width << a.page_shift);
}

template <int D>
__device__ __forceinline__ constexpr int part_floats(int rows) { return rows * (D + 2); }

template <int D, int R>
__device__ __forceinline__ void store_part(float* part, int line, int column, float top, float total,
                                           const float4& sum) {
  *reinterpret_cast<float4*>(part + line * D + column) = sum;
  if (column == 0) *reinterpret_cast<float2*>(part + R * D + 2 * line) = float2{top, total};
}
// Adds `parts` parts of a row, `step` floats apart, to what there is of it: four dims by this thread.
template <int D>
__device__ __forceinline__ void add_row_parts(RowSum& to, const float* part, long long step, int rows, int line,
                                              int column, int parts) {
  constexpr int kAtOnce = 4;
  for (int base = 0; base < parts; base += kAtOnce) {
    float2 stats[kAtOnce];
    float4 values[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float* from = part + min(base + k, parts - 1) * step;
      stats[k] = *reinterpret_cast<const float2*>(from + rows * D + 2 * line);
      values[k] = *reinterpret_cast<const float4*>(from + line * D + column);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const bool live = base + k < parts;
      const float top = live ? fmaxf(to.top, stats[k].x) : to.top;
      const float before = __builtin_amdgcn_exp2f(to.top - top);
      const float factor = __builtin_amdgcn_exp2f(stats[k].x - top);
      to.top = top;
      to.total = to.total * before + (live ? stats[k].y * factor : 0.0f);
      to.sum.x = to.sum.x * before + (live ? values[k].x * factor : 0.0f);
      to.sum.y = to.sum.y * before + (live ? values[k].y * factor : 0.0f);
      to.sum.z = to.sum.z * before + (live ? values[k].z * factor : 0.0f);
      to.sum.w = to.sum.w * before + (live ? values[k].w * factor : 0.0f);
    }
  }
}
// Where the prefix's parts of a sequence's rows lie.
struct PrefixParts {
  int tokens;     // P_g, 0: none
  int row0;       // the group's first row
  int first_slot;
  int parts;
};
__device__ __forceinline__ PrefixParts prefix_parts(const SharedParams& sp, int sequence) {
  // The last group that begins at or before the sequence, if that has it.
  int before = 0;
  for (int base = 0; base < sp.group_count; base += 64) {
    const int g = base + (int)(threadIdx.x & 63);
    before += __popcll(__ballot(g < sp.group_count && sp.groups[g] <= sequence));
  }
  PrefixParts of{0, 0, 0, 0};
  const int g = uniform(before) - 1;
  if (g < 0 || sequence >= sp.groups[g + 1] || sp.p.a.lengths[sequence] <= 0) return of;
  of.tokens = max(sp.shared[g], 0);
  if (of.tokens == 0) return of;
  of.row0 = row_before(sp.p.a, max(0, min(sp.groups[g], sp.p.a.sequences)));
  of.first_slot = first_slot(sp, g, of.row0);
  const int tiles = tiles_in_table(sp.p.a, of.tokens);
  of.parts = min(sp.prefix_splits, (tiles + sp.prefix_chunk - 1) / sp.prefix_chunk);
  return of;
}
// Adds the prefix's parts of a row, `index` being the row's query token among all of q's.
template <int D>
__device__ __forceinline__ void add_prefix(const SharedParams& sp, const PrefixParts& of, RowSum& to, int head, int index,
                                           int h, int column) {
  if (of.parts == 0) return;
  const int line = (index - of.row0) * sp.p.group + h, slot = of.first_slot + line / sp.prefix_rows;
  if (line < 0 || slot >= sp.prefix_slots) return;  // offsets that decrease: within the parts all the same
  const long long floats = part_floats<D>(sp.prefix_rows);
  const float* part = sp.prefix_work + ((long long)slot * sp.prefix_splits * sp.p.a.kv_heads + head) * floats;
  add_row_parts<D>(to, part, floats * sp.p.a.kv_heads, sp.prefix_rows, line % sp.prefix_rows, column, of.parts);
}
template <int D, typename In>
__device__ __forceinline__ void store_result(const CacheAttentionArgs& a, const RowSum& from, int row, int head,
                                             int column) {
  const float inverse = from.total == 0.0f ? 0.0f : 1.0f / from.total;
  store4(static_cast<In*>(a.out) + ((long long)row * a.heads + head) * D + column,
         float4{from.sum.x * inverse, from.sum.y * inverse, from.sum.z * inverse, from.sum.w * inverse});
}

// The rows of a group over its prefix: a part per row tile, share of the keys, and head.
template <int D, typename In, int R, int NT>
__global__ __launch_bounds__(kThreads, resident(D, R, NT)) void prefix_kernel(SharedParams sp) {
  const Params& p = sp.p;
  const CacheAttentionArgs& a = p.a;
  __shared__ __align__(16) unsigned char room_bytes[sizeof(Room<D>)];
  Room<D>& room = *reinterpret_cast<Room<D>*>(room_bytes);
  __shared__ float stats[2][kWaves][R == 8 ? 16 : R];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
  const int split = unit % sp.prefix_splits, slot = unit / sp.prefix_splits;

  int before = 0;
  for (int base = 0; base < sp.group_count; base += 64) {
    const int g = base + (int)(threadIdx.x & 63);
    bool begun = false;
    if (g < sp.group_count) begun = first_slot(sp, g, row_before(a, max(0, min(sp.groups[g], a.sequences)))) <= slot;
    before += __popcll(__ballot(begun));
  }
  const int g = uniform(before) - 1;
  if (g < 0) return;
  const Group group = group_of(sp, g);
  Span s;
  s.start = (slot - first_slot(sp, g, group.row0)) * R;
  s.rows = group.rows * p.group;
  if (s.start < 0 || s.start >= s.rows) return;
  int source;
  const int tokens = shared_tokens(sp, g, group, source);
  if (slot == first_slot(sp, g, group.row0) && split == 0 && head == 0 && threadIdx.x == 0) sp.shared[g] = tokens;
  s.sequence = s.table_row = source;
  s.row0 = group.row0;
  s.first = s.low = s.high = tokens - 1;
  s.sink_tiles = s.window_tile = s.from = s.step = 0;
  s.total = tiles_in_table(a, tokens);
  const int begin = split * sp.prefix_chunk;
  const int end = split == sp.prefix_splits - 1 ? s.total : min(s.total, begin + sp.prefix_chunk);
  if (begin >= end) return;
  float* part = sp.prefix_work + (((long long)slot * sp.prefix_splits + split) * a.kv_heads + head) * part_floats<D>(R);
  attend_run<D, In, R, NT, false, true>(p, s, head, begin, end, wave, room, stats,
                                        [&](int line, int column, int, float top, float total, const float4& sum) {
                                          store_part<D, R>(part, line, column, top, total, sum);
                                        });
}

// The span of a sequence's rows over its keys from `tokens` on.
template <int R>
__device__ __forceinline__ Span tail_span(const SharedParams& sp, int sequence, int row0, int queries, int start,
                                          int tokens) {
  Span s = make_span<R>(sp.p, sequence, row0, queries, sp.p.a.lengths[sequence], start);
  s.table_row = sequence;
  s.from = tokens;
  s.step = 1;
  s.window_tile = min(tokens / kCacheTile, s.total);
  s.total -= s.window_tile;
  return s;
}

// The rows of each sequence over its own keys: the results where they are not split, else a part per row tile, share
// and head.
template <int D, typename In, int R, int NT>
__global__ __launch_bounds__(kThreads, resident(D, R, NT)) void tail_kernel(SharedParams sp) {
  const Params& p = sp.p;
  const CacheAttentionArgs& a = p.a;
  __shared__ __align__(16) unsigned char room_bytes[sizeof(Room<D>)];
  Room<D>& room = *reinterpret_cast<Room<D>*>(room_bytes);
  __shared__ float stats[2][kWaves][R == 8 ? 16 : R];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
  const int split = unit % sp.tail_splits, slot = unit / sp.tail_splits;
  if (slot >= p.slots) {
    if (split == 0) clear_rows<D, In>(p, head);
    return;
  }
  int sequence, row0, queries, start;
  if (!row_tile<R>(p, slot, sequence, row0, queries, start)) return;
  const PrefixParts of = prefix_parts(sp, sequence);
  const Span s = tail_span<R>(sp, sequence, row0, queries, start, of.tokens);
  const int begin = split * sp.tail_chunk;
  const int end = split == sp.tail_splits - 1 ? s.total : min(s.total, begin + sp.tail_chunk);
  if (sp.tail_splits == 1) {
    attend_run<D, In, R, NT, false, true>(
        p, s, head, 0, s.total, wave, room, stats,
        [&](int, int column, int row, float top, float total, const float4& sum) {
          RowSum all{sum, top, total};
          const int token = row / p.group, h = row - token * p.group;
          add_prefix<D>(sp, of, all, head, s.row0 + token, h, column);
          store_result<D, In>(a, all, s.row0 + token, head * p.group + h, column);
        });
  } else if (begin < end) {
    float* part = sp.tail_work + (((long long)slot * sp.tail_splits + split) * a.kv_heads + head) * part_floats<D>(R);
    attend_run<D, In, R, NT, false, true>(p, s, head, begin, end, wave, room, stats,
                                          [&](int line, int column, int, float top, float total, const float4& sum) {
                                            store_part<D, R>(part, line, column, top, total, sum);
                                          });
  }
}

// Adds the parts of split tails and of the prefix: a wave per row (query token and head).
template <int D, typename In, int R>
__global__ __launch_bounds__(kThreads) void join_kernel(SharedParams sp) {
  const Params& p = sp.p;
  const CacheAttentionArgs& a = p.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long id = (long long)blockIdx.x * kWaves + wave;
  const int row = (int)(id / a.heads), h = (int)(id % a.heads);
  int sequence = 0, index = 0;
  if (row >= a.rows || !find_sequence(a.offsets, a.sequences, row, row, sequence, index)) return;
  const int head = h / p.group, line = index * p.group + h % p.group;
  int row0;
  const int queries = rows_of(a, sequence, row0);
  const PrefixParts of = prefix_parts(sp, sequence);
  const Span s = tail_span<R>(sp, sequence, row0, queries, line / R * R, of.tokens);
  const int column = (threadIdx.x & 63) * 4;
  if (column >= D) return;
  RowSum all{float4{0.0f, 0.0f, 0.0f, 0.0f}, kNoKey, 0.0f};
  const int slot = slot_of<R>(p, sequence, row0) + line / R;
  const long long floats = part_floats<D>(R);
  const int parts = min(sp.tail_splits, (s.total + sp.tail_chunk - 1) / sp.tail_chunk);
  add_row_parts<D>(all, sp.tail_work + ((long long)slot * sp.tail_splits * a.kv_heads + head) * floats,
                   floats * a.kv_heads, R, line % R, column, parts);
  add_prefix<D>(sp, of, all, head, row, h % p.group, column);
  store_result<D, In>(a, all, row, h, column);
}

// Keys are split where row tiles and heads make fewer blocks than the device holds at a time, but not below so many
// tiles.  Four groups of 16 sequences with 4 rows each over 3957 tokens, 16/4 heads of 64, fp16: 22.1 us with as many
// blocks as it holds, 768, and 24.9 with 512 or 1024.
constexpr int kDeviceUnits = 256, kLeastTiles = 8;  // CUs
constexpr int kWholeUnits = 128, kWholeTiles = 64;

// Rows of a row tile: 8, 16 or 32, as `rows` of them fill.
int tile_rows(const CacheAttentionArgs& a, long long rows) {
  if (a.head_dim == 256) return rows <= 16 || a.dtype != kBfloat16 ? 16 : 32;
  return rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
}

struct Plan {
  SharedParams sp;
  int tail_rows;
  long long prefix_bytes, tail_bytes, shared_bytes;
};

Plan plan(const PrefixAttentionArgs& args) {
  const CacheAttentionArgs& a = args.a;
  Plan plan{};
  SharedParams& sp = plan.sp;
  sp.p = Params{a, a.heads / a.kv_heads, 0, 1, 0, 0, 1.44269504088896340736f * a.scale, 0.0f, false, false, nullptr};
  Params& p = sp.p;
  p.inverse = 1.0f / p.scale;
  const int size = a.dtype == kFloat32 ? 4 : 2;
  p.aligned =
      (((uintptr_t)a.q | (uintptr_t)(a.q_strides.token * size) | (uintptr_t)(a.q_strides.head * size)) & 15u) == 0;
  sp.groups = args.groups;
  sp.prefix = args.prefix;
  sp.group_count = args.group_count;
  const long long rows = (long long)a.rows * p.group;
  const int terms = a.dtype == kFloat32 ? 3 : a.dtype == kFloat16 ? 2 : 1;
  auto split = [&](int R, long long tiles, long long units, int& splits, int& chunk) {
    const long long wanted = max(1LL, kDeviceUnits * resident(a.head_dim, R, terms) / max(1LL, units));
    const long long each = max((long long)kLeastTiles, (tiles + wanted - 1) / wanted);
    chunk = (int)each;
    splits = (int)max(1LL, (tiles + each - 1) / each);
  };

  const int R = sp.prefix_rows = tile_rows(a, rows / max(1, args.group_count));
  sp.prefix_slots = (int)(rows / R + args.group_count);
  // Where nothing is known of the prefixes, they may be all of the longest sequence, and so may what lies behind them.
  // 32/8 heads of 128, bf16: eight rows over 480 shared and 19520 own keys 51 us so, 135 with tails taken for short, one
  // over 130000 own 54 and 783; eight over 480 and 21 pay 4 us for the third launch, 21 and 17.
  const bool known = args.max_prefix >= 0;
  const int longest_prefix = known ? args.max_prefix : a.max_length;
  split(R, ((long long)longest_prefix + kCacheTile - 1) / kCacheTile, ((rows + R - 1) / R) * a.kv_heads, sp.prefix_splits,
        sp.prefix_chunk);
  const int T = plan.tail_rows = tile_rows(a, rows / max(1, a.sequences));
  p.slots = (int)(a.offsets == nullptr ? (long long)a.sequences * ((p.group + T - 1) / T) : rows / T + a.sequences);
  const long long tiles = max(0, a.max_length - (known ? args.max_prefix : 0)) / kCacheTile + 2;
  const long long units = max((long long)a.sequences, rows / T) * a.kv_heads;
  if (tiles <= kLeastTiles || (tiles <= kWholeTiles && units >= kWholeUnits)) {
    sp.tail_splits = 1;
    sp.tail_chunk = 1;
  } else {
    split(T, tiles, units, sp.tail_splits, sp.tail_chunk);
  }
  const long long floats = a.head_dim + 2;
  plan.shared_bytes = ((long long)args.group_count * 4 + 15) & ~15LL;
  plan.prefix_bytes = (long long)sp.prefix_slots * sp.prefix_splits * a.kv_heads * R * floats * 4;
  plan.tail_bytes = sp.tail_splits == 1 ? 0 : (long long)p.slots * sp.tail_splits * a.kv_heads * T * floats * 4;
  return plan;
}

template <int D, typename In, int R, int NT>
hipError_t run_prefix(hipStream_t stream, const Plan& plan) {
  const SharedParams& sp = plan.sp;
  const long long blocks = (long long)sp.prefix_slots * sp.prefix_splits * sp.p.a.kv_heads;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (blocks > 0)
    hipLaunchKernelGGL((prefix_kernel<D, In, R, NT>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, sp);
  return hipGetLastError();
}

template <int D, typename In, int R, int NT>
hipError_t run_tails(hipStream_t stream, const Plan& plan) {
  const SharedParams& sp = plan.sp;
  const long long clears = sp.p.a.offsets != nullptr ? sp.tail_splits : 0;  // rows of no sequence
  const long long blocks = ((long long)sp.p.slots * sp.tail_splits + clears) * sp.p.a.kv_heads;
  const long long joins = ((long long)sp.p.a.rows * sp.p.a.heads + kWaves - 1) / kWaves;
  if (blocks > 0x7fffffffLL || joins > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((tail_kernel<D, In, R, NT>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, sp);
  if (sp.tail_splits > 1)
    hipLaunchKernelGGL((join_kernel<D, In, R>), dim3((unsigned)joins), dim3(kThreads), 0, stream, sp);
  return hipGetLastError();
}

template <int D, typename In, int NT, bool TAILS, int R>
hipError_t run(hipStream_t stream, const Plan& plan) {
  if constexpr (TAILS)
    return run_tails<D, In, R, NT>(stream, plan);
  else
    return run_prefix<D, In, R, NT>(stream, plan);
}
template <int D, typename In, int NT, bool TAILS>
hipError_t run_rows(hipStream_t stream, const Plan& plan) {
  const int rows = TAILS ? plan.tail_rows : plan.sp.prefix_rows;
  if constexpr (D < 256) {
    if (rows == 8) return run<D, In, NT, TAILS, 8>(stream, plan);
    if (rows == 32) return run<D, In, NT, TAILS, 32>(stream, plan);
  } else if constexpr (NT == 1) {
    if (rows == 32) return run<D, In, NT, TAILS, 32>(stream, plan);
  }
  return run<D, In, NT, TAILS, 16>(stream, plan);
}
template <int D, bool TAILS>
hipError_t run_types(hipStream_t stream, const Plan& plan) {
  if (plan.sp.p.a.dtype == kFloat32) return run_rows<D, float, 3, TAILS>(stream, plan);
  if (plan.sp.p.a.dtype == kFloat16) return run_rows<D, Half, 2, TAILS>(stream, plan);
  return run_rows<D, Bfloat, 1, TAILS>(stream, plan);
}
template <int D>
hipError_t run_both(hipStream_t stream, const Plan& plan) {
  const hipError_t status = run_types<D, false>(stream, plan);
  return status != hipSuccess ? status : run_types<D, true>(stream, plan);
}

}  // namespace

long long prefix_attention_work(const PrefixAttentionArgs& args) {
  const Plan p = plan(args);
  return p.shared_bytes + p.prefix_bytes + p.tail_bytes;
}

hipError_t launch_prefix_attention(hipStream_t stream, const PrefixAttentionArgs& args) {
  if (args.a.rows == 0) return hipSuccess;
  Plan p = plan(args);
  char* work = reinterpret_cast<char*>(args.a.work);
  p.sp.shared = reinterpret_cast<int*>(work);
  p.sp.prefix_work = reinterpret_cast<float*>(work + p.shared_bytes);
  p.sp.tail_work = reinterpret_cast<float*>(work + p.shared_bytes + p.prefix_bytes);
  if (args.a.head_dim == 64) return run_both<64>(stream, p);
  if (args.a.head_dim == 128) return run_both<128>(stream, p);
  return run_both<256>(stream, p);
}

}  // namespace ivo
