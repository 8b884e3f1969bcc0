// The pages of a cache, kept on the device: given to sequences that grow, shared by forks, taken back, moved together.
//
// refs [pages]: how many table entries hold a page.  free [pages / 32]: bit p % 32 of word p / 32 is set where none
// does.  A page is given lowest number first, in the order of the sequences and of their slots, so a pool and its
// tables are a function of the calls made on them: ranks come from prefix sums, and what goes through atomics (counts
// up and down, bits set) does not depend on their order.
//
// The bookkeeping is a chain of a few dependent loads in one block, since every rank depends on all before it: the
// free words' population counts, summed over the block, give every thread the ranks of the free pages in its words, and
// a request of rank r finds its page by a binary search in those sums and then in the words of one thread.  Measured:
// a step of 64 sequences in a pool of 4096 pages reserved in 3.8 us and their windows released in 3.4; 4 sequences forked
// into 64 in 6.4 and 1.3; a pool of 6000 pages compacted in 7.2 and 1.6 to 4.  Pages' bytes are moved by a kernel of
// their own that reads what to move from the device, for each layer's cache.
#include "internal.hpp"
#include "ternary_device.hpp"

namespace ivo {
namespace {

constexpr int kBlock = 1024;  // threads of the bookkeeping
constexpr int kBlockWaves = kBlock / 64;

__device__ __forceinline__ bool is_page(const PoolArgs& p, int page) { return (unsigned)page < (unsigned)p.pages; }

// Sum of v over the threads before this one, and over all.
__device__ __forceinline__ int block_scan(int v, int* totals, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int lower = __shfl_up(sum, o);
    if (lane >= o) sum += lower;
  }
  __syncthreads();  // the totals of a scan before this one have been read
  if (lane == 63) totals[wave] = sum;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kBlockWaves; ++w) {
    before += w < wave ? totals[w] : 0;
    all += totals[w];
  }
  return before + sum - v;
}

// Sum of v over the block, in thread 0.
__device__ __forceinline__ long long block_sum(long long v, long long* totals) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) totals[threadIdx.x >> 6] = v;
  __syncthreads();
  long long all = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < kBlockWaves; ++w) all += totals[w];
  return all;
}

// Word w of the free pages; bits past the last page do not count.
__device__ __forceinline__ unsigned free_word(const PoolArgs& p, int w) {
  const int left = p.pages - w * 32;
  return (unsigned)p.free[w] & (left < 32 ? (1u << left) - 1u : ~0u);
}

// The free pages in order, over a block: thread t has the words [t * per, (t + 1) * per).
struct FreePages {
  int per;
  int own;        // free pages of this thread's words
  int before;     // and of those before
  int available;
  const int* sums;  // [kBlock] in LDS: `before` of every thread
};
__device__ __forceinline__ FreePages scan_free(const PoolArgs& p, int* sums, int* totals) {
  FreePages f;
  const int words = (p.pages + 31) / 32;
  f.per = (words + kBlock - 1) / kBlock;
  f.own = 0;
  const int begin = threadIdx.x * f.per, end = min(begin + f.per, words);
  for (int w = begin; w < end; ++w) f.own += __popc(free_word(p, w));
  f.before = block_scan(f.own, totals, f.available);
  sums[threadIdx.x] = f.before;
  f.sums = sums;
  __syncthreads();
  return f;
}
// The free page of a rank below `available`.  (The walk ends with the words all the same where another call on the pool,
// against the order that they need, has taken pages since the scan.)
__device__ __forceinline__ int free_page(const PoolArgs& p, const FreePages& f, int rank) {
  int thread = 0;
#pragma unroll
  for (int step = kBlock / 2; step > 0; step >>= 1)
    if (f.sums[thread + step] <= rank) thread += step;
  rank -= f.sums[thread];
  const int words = (p.pages + 31) / 32;
  int w = min(thread * f.per, words - 1);
  unsigned word = free_word(p, w);
  for (int count = __popc(word); rank >= count && w + 1 < words; count = __popc(word)) {
    rank -= count;
    word = free_word(p, ++w);
  }
  for (; rank > 0; --rank) word &= word - 1u;
  return word == 0u ? 0 : w * 32 + __builtin_ctz(word);
}
// Clears the bits of the first `given` free pages.  No thread may look for a page any more.
__device__ __forceinline__ void take_free(const PoolArgs& p, const FreePages& f, int given) {
  int mine = min(given - f.before, f.own);
  for (int w = threadIdx.x * f.per; mine > 0 && w < min((int)(threadIdx.x + 1) * f.per, (p.pages + 31) / 32); ++w) {
    unsigned word = free_word(p, w);
    for (; word != 0u && mine > 0; --mine) word &= word - 1u;
    p.free[w] = (int)word;
  }
}

// Slots that a sequence's next tokens need: [first, last).
__device__ __forceinline__ void slots_of(int length, int count, int page_shift, long long& first, long long& last) {
  const long long page = 1LL << page_shift, from = max(length, 0);
  first = (from + page - 1) >> page_shift;
  last = (from + max(count, 0) + page - 1) >> page_shift;
}

constexpr int kShort = 4;  // slots up to which a lane goes through a sequence's by itself

// Calls visit(sequence of the lane, slot, needs a page, ..) so that a wave goes through 64 sequences' slots in their
// order: `one` for a lane's slot, `many` for 64 slots of one sequence.
template <typename One, typename Many>
__device__ __forceinline__ void visit_slots(const PoolArgs& p, const int* table, int width, int sequence, long long first,
                                            long long last, One one, Many many) {
  const int lane = threadIdx.x & 63;
  const bool is_short = last - first <= kShort;
  if (is_short)
    for (long long slot = first; slot < last; ++slot)
      if (!is_page(p, table[(long long)sequence * width + slot])) one((int)slot);
  unsigned long long others = __ballot(!is_short);
  while (others != 0ull) {
    const int from = __builtin_ctzll(others);
    others &= others - 1ull;
    const int b = __shfl(sequence, from), begin = __shfl((int)first, from), end = __shfl((int)last, from);
    for (int base = begin; base < end; base += 64) {
      const int slot = base + lane;
      const bool need = slot < end && !is_page(p, table[(long long)b * width + slot]);
      many(from, b, slot, need, __ballot(need));
    }
  }
}

__global__ __launch_bounds__(kBlock) void reserve_kernel(PoolArgs p, int* table, int width, const int* lengths,
                                                         const int* counts, int sequences, int* missing) {
  __shared__ int sums[kBlock];
  __shared__ int totals[kBlockWaves];
  __shared__ long long totals_outside[kBlockWaves];
  const FreePages f = scan_free(p, sums, totals);
  const int lane = threadIdx.x & 63;
  int given = 0;             // ranks of the sequences before these
  long long outside = 0;     // slots past the table, of this thread's sequences
  for (int base = 0; base < sequences; base += kBlock) {
    const int b = base + (int)threadIdx.x;
    long long first = 0, last = 0;
    if (b < sequences) slots_of(lengths[b], counts[b], p.page_shift, first, last);
    outside += max(last, (long long)width) - max(first, (long long)width);
    first = min(first, (long long)width);
    last = min(last, (long long)width);
    int needed = 0;
    visit_slots(p, table, width, b, first, last, [&](int) { ++needed; },
                [&](int from, int, int, bool, unsigned long long mask) { needed += lane == from ? __popcll(mask) : 0; });
    int all = 0;
    int rank = given + block_scan(needed, totals, all);
    auto give = [&](int sequence, int slot, int r) {
      if (r >= f.available) return;
      const int page = free_page(p, f, r);
      table[(long long)sequence * width + slot] = page;
      p.refs[page] = 1;
    };
    if (all > 0)
      visit_slots(p, table, width, b, first, last, [&](int slot) { give(b, slot, rank++); },
                  [&](int from, int sequence, int slot, bool need, unsigned long long mask) {
                    const int r = __shfl(rank, from) + __popcll(mask & ((1ull << lane) - 1ull));
                    if (need) give(sequence, slot, r);
                    if (lane == from) rank += __popcll(mask);
                  });
    given += all;
  }
  outside = block_sum(outside, totals_outside);  // and everybody has found its pages
  take_free(p, f, min(given, f.available));
  if (threadIdx.x == 0) *missing = (int)min(max(given - f.available, 0) + outside, 0x7fffffffLL);
}

// One holder of a page less.
__device__ __forceinline__ void drop(const PoolArgs& p, int page) {
  const int before = atomicSub(p.refs + page, 1);
  if (before == 1) atomicOr(reinterpret_cast<unsigned*>(p.free) + page / 32, 1u << (page & 31));
  if (before <= 0) atomicAdd(p.refs + page, 1);  // the counts were wrong: no page has fewer than none
}

__global__ __launch_bounds__(kThreads) void release_kernel(PoolArgs p, int* table, int width, const int* first,
                                                           const int* last, int sequences) {
  const int b = blockIdx.y + blockIdx.z * 65535;
  if (b >= sequences) return;
  const int slot = blockIdx.x * kThreads + (int)threadIdx.x;
  if (slot >= width || (first != nullptr && slot < first[b]) || (last != nullptr && slot >= last[b])) return;
  int* entry = table + (long long)b * width + slot;
  const int page = *entry;
  if (!is_page(p, page)) return;
  *entry = -1;
  drop(p, page);
}

__device__ __forceinline__ int whole_pages(const PoolArgs& p, int length) { return max(length, 0) >> p.page_shift; }

// Block 0 writes the rows' slots with unfinished pages, and all lengths and copies: it gives out pages to the rows that
// share their parent with an earlier row, and to the others (a parent's heirs) whose unfinished page is in more entries
// of the table than theirs.  The other blocks write the rows' other slots, each kBlock slots of one row.  They may
// count up a page while block 0 looks at its count, but only one that is in two entries before.
__global__ __launch_bounds__(kBlock) void fork_kernel(PoolArgs p, ForkArgs a) {
  __shared__ int sums[kBlock];
  __shared__ int totals[kBlockWaves];
  if (blockIdx.x > 0) {
    const int blocks = (a.width + kBlock - 1) / kBlock;
    const int r = (blockIdx.x - 1) / blocks, slot = (blockIdx.x - 1) % blocks * kBlock + (int)threadIdx.x;
    const int parent = a.parents[r];
    const bool there = (unsigned)parent < (unsigned)a.sequences;
    bool taken = false;
    if (there)
      for (int i = threadIdx.x; i < r; i += kBlock) taken |= a.parents[i] == parent;
    const bool heir = !__syncthreads_or(taken);
    if (slot >= a.width) return;
    int page = -1;
    if (there) {
      const int length = a.lengths[parent], whole = whole_pages(p, length);
      if (slot == whole && max(length, 0) & ((1 << p.page_shift) - 1)) return;  // block 0's
      if (heir || slot < whole) page = a.table[(long long)parent * a.width + slot];
    }
    a.out_table[(long long)r * a.width + slot] = page;
    if (is_page(p, page)) atomicAdd(p.refs + page, 1);
    return;
  }
  extern __shared__ int first[];  // [sequences]: the first row of a parent
  for (int b = threadIdx.x; b < a.sequences; b += kBlock) first[b] = a.rows;
  const FreePages f = scan_free(p, sums, totals);
  for (int r = threadIdx.x; r < a.rows; r += kBlock) {
    const int parent = a.parents[r];
    if ((unsigned)parent < (unsigned)a.sequences) atomicMin(first + parent, r);
  }
  __syncthreads();
  int given = 0;
  for (int base = 0; base < a.rows; base += kBlock) {
    const int r = base + (int)threadIdx.x;
    int length = 0, whole = 0, source = -1;
    bool slot = false, heir = false;  // this block writes the row's slot `whole`
    if (r < a.rows) {
      const int parent = a.parents[r];
      if ((unsigned)parent < (unsigned)a.sequences) {
        length = max(a.lengths[parent], 0);
        whole = whole_pages(p, length);
        heir = first[parent] == r;
        slot = whole < a.width && (length & ((1 << p.page_shift) - 1)) != 0;
        if (slot) source = a.table[(long long)parent * a.width + whole];
      }
    }
    const bool wants = is_page(p, source) && (!heir || p.refs[source] > 1);
    int all = 0;
    const int rank = given + block_scan(wants ? 1 : 0, totals, all);
    int page = heir && !wants ? source : -1;
    if (is_page(p, page)) atomicAdd(p.refs + page, 1);
    if (wants && rank < f.available) {
      page = free_page(p, f, rank);
      p.refs[page] = 1;
      a.copies[2 * rank] = source;
      a.copies[2 * rank + 1] = page;
    }
    if (wants && page < 0) length = whole << p.page_shift;  // the tokens of the unfinished page are lost
    if (slot) a.out_table[(long long)r * a.width + whole] = page;
    if (r < a.rows) a.out_lengths[r] = length;
    given += all;
  }
  __syncthreads();  // everybody has found its pages
  const int got = min(given, f.available);
  take_free(p, f, got);
  for (int i = 2 * got + (int)threadIdx.x; i < 2 * a.rows; i += kBlock) a.copies[i] = -1;
  if (threadIdx.x == 0) *a.missing = given - got;
}

// The old rows hold their pages no more.
__global__ __launch_bounds__(kThreads) void drop_kernel(PoolArgs p, const int* table, long long entries) {
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i < entries && is_page(p, table[i])) drop(p, table[i]);
}

// The held pages from `live` on go to the free ones below it, in order.
__global__ __launch_bounds__(kBlock) void compact_kernel(PoolArgs p, int* copies, int* moved, int* live_out) {
  __shared__ int sums[kBlock];
  __shared__ int totals[kBlockWaves];
  __shared__ int holes;
  const FreePages f = scan_free(p, sums, totals);
  const int live = p.pages - f.available, most = p.pages / 2;
  if (threadIdx.x == 0) holes = live == p.pages ? f.available : -1;
  for (int page = live + (int)threadIdx.x; page < p.pages; page += kBlock) moved[page] = page;
  __syncthreads();
  const int begin = threadIdx.x * f.per, end = min(begin + f.per, (p.pages + 31) / 32);
  // Free pages before `live`, by the thread that has its word.
  if (live / 32 >= begin && live / 32 < end) {
    int count = f.before;
    for (int w = begin; w < live / 32; ++w) count += __popc(free_word(p, w));
    holes = count + __popc(free_word(p, live / 32) & ((1u << (live & 31)) - 1u));
  }
  __syncthreads();
  const int count = holes;
  int rank = f.before;
  for (int w = begin; w < end; ++w) {
    const unsigned word = free_word(p, w);
    const int base = w * 32, limit = min(32, p.pages - base);
    for (unsigned bits = word; bits != 0u && base + __builtin_ctz(bits) < live; bits &= bits - 1u)
      copies[2 * (rank + __popc(word & ((bits & -bits) - 1u))) + 1] = base + __builtin_ctz(bits);
    unsigned held = ~word & (limit == 32 ? ~0u : (1u << limit) - 1u);
    if (base + 31 < live) held = 0u;
    if (base < live && live - base < 32) held &= ~((1u << (live - base)) - 1u);
    // A held page's rank among all held ones is its number less the free pages before it.
    for (; held != 0u; held &= held - 1u) {
      const int bit = __builtin_ctz(held);
      const int before = rank + __popc(word & ((1u << bit) - 1u));
      copies[2 * (base + bit - before - (live - count))] = base + bit;
    }
    rank += __popc(word);
  }
  for (int i = count + (int)threadIdx.x; i < most; i += kBlock) copies[2 * i] = copies[2 * i + 1] = -1;
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kBlock) {
    const int source = copies[2 * i], target = copies[2 * i + 1];
    moved[source] = target;
    p.refs[target] = p.refs[source];
    p.refs[source] = 0;
  }
  for (int w = begin; w < end; ++w) {
    const int base = w * 32;
    unsigned word = base + 32 <= live ? 0u : base >= live ? ~0u : ~((1u << (live - base)) - 1u);
    if (p.pages - base < 32) word &= (1u << (p.pages - base)) - 1u;
    p.free[w] = (int)word;
  }
  if (threadIdx.x == 0) *live_out = live;
}

__global__ __launch_bounds__(kThreads) void renumber_kernel(PoolArgs p, int* table, long long entries, const int* moved,
                                                            const int* live) {
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= entries) return;
  const int page = table[i];
  if (is_page(p, page) && page >= *live) table[i] = moved[page];
}

// A block takes 4 KB, 16 bytes a thread, of every gridDim.y'th page of the list.  It looks at 64 rows of the list at a
// time, most of which hold no copy when a cache is compacted.  Pages of 68 KB: 60 copied in 3.2 us and 900 in 20 (6.4
// TB/s); with two to four loads before their stores in a thread 16.5 and 28.
constexpr int kCopyBytes = kThreads * 16;
__global__ __launch_bounds__(kThreads) void copy_kernel(uint8_t* pages, int page_count, long long page_bytes,
                                                        const int* copies, int count) {
  const int lane = threadIdx.x & 63;
  const long long at = (long long)blockIdx.x * kThreads + threadIdx.x;
  const bool inside = at < page_bytes / 16;
  for (long long base = blockIdx.y; base < count; base += 64LL * gridDim.y) {
    const long long i = base + (long long)lane * gridDim.y;
    const int2 copy = i < count ? reinterpret_cast<const int2*>(copies)[i] : int2{-1, -1};
    unsigned long long live = __ballot((unsigned)copy.x < (unsigned)page_count && (unsigned)copy.y < (unsigned)page_count &&
                                       copy.x != copy.y);
    for (; live != 0ull; live &= live - 1ull) {
      const int row = __builtin_ctzll(live);
      const float4* from = reinterpret_cast<const float4*>(pages + __shfl(copy.x, row) * page_bytes);
      float4* to = reinterpret_cast<float4*>(pages + __shfl(copy.y, row) * page_bytes);
      if (inside) to[at] = from[at];
    }
  }
}
constexpr int kCopyBlocks = 8192;

}  // namespace

hipError_t launch_page_reserve(hipStream_t stream, const PoolArgs& p, int* table, int width, const int* lengths,
                               const int* counts, int sequences, int* missing) {
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kBlock), 0, stream, p, table, width, lengths, counts, sequences,
                     missing);
  return hipGetLastError();
}

hipError_t launch_page_release(hipStream_t stream, const PoolArgs& p, int* table, int width, const int* first,
                               const int* last, int sequences) {
  if (sequences == 0) return hipSuccess;
  const unsigned y = (unsigned)(sequences < 65535 ? sequences : 65535), z = (unsigned)((sequences + 65534) / 65535);
  hipLaunchKernelGGL(release_kernel, dim3((unsigned)((width + kThreads - 1) / kThreads), y, z), dim3(kThreads), 0, stream,
                     p, table, width, first, last, sequences);
  return hipGetLastError();
}

hipError_t launch_page_fork(hipStream_t stream, const PoolArgs& p, const ForkArgs& a) {
  const long long blocks = 1 + (long long)a.rows * ((a.width + kBlock - 1) / kBlock);
  const long long entries = (long long)a.sequences * a.width;
  const long long drops = (entries + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL || drops > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(fork_kernel, dim3((unsigned)blocks), dim3(kBlock), a.sequences * sizeof(int), stream, p, a);
  if (drops > 0)
    hipLaunchKernelGGL(drop_kernel, dim3((unsigned)drops), dim3(kThreads), 0, stream, p, a.table, entries);
  return hipGetLastError();
}

hipError_t launch_page_compact(hipStream_t stream, const PoolArgs& p, int* table, long long entries, int* copies,
                               int* moved, int* live) {
  const long long blocks = (entries + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kBlock), 0, stream, p, copies, moved, live);
  if (blocks > 0)
    hipLaunchKernelGGL(renumber_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p, table, entries, moved,
                       live);
  return hipGetLastError();
}

hipError_t launch_page_copy(hipStream_t stream, uint8_t* pages, int page_count, long long page_bytes, const int* copies,
                            int count) {
  if (count == 0) return hipSuccess;
  const long long chunks = (page_bytes + kCopyBytes - 1) / kCopyBytes;
  const long long rows = kCopyBlocks / chunks;
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)chunks, (unsigned)(rows < 1 ? 1 : rows < count ? rows : count)),
                     dim3(kThreads), 0, stream, pages, page_count, page_bytes, copies, count);
  return hipGetLastError();
}

}  // namespace ivo
