// CacheCopy, CacheFork, CacheGrow, CacheFree and CacheCompact for gfx950: the pages of a cache copied, shared, given, taken back
// and moved together, on tables that stay on the device.
//
// State: refs[p] rows hold page p (0: free). Nothing else says what is free, so there is no list that could disagree with it:
// the free pages are found anew by each call, lowest first, from a bitmap that one launch makes of refs (4 bytes a page: 5.7 us
// for four million pages, 3.3 of them HBM time, and little beside the launch for the usual tens of thousands). That launch's
// counts for each 1,024 pages let any thread of the next find the r-th free page by a search of two levels, so requests are
// served side by side and get the pages that serving them in order would give them.
//
// Copies are the rest: pages are `column`s of 16 bytes over every layer of every pool, a thread takes one column of up to
// eight pages, all loads before the stores.

#include "cache_f4.h"

namespace {

using namespace roost_dev;

constexpr uint32_t kThreads = 256;
constexpr uint32_t kChunk = 1024;                // pages that one count stands for
constexpr uint32_t kWords = kChunk / 64;         // words of the bitmap in it
constexpr uint32_t kMaxPages = 4u << 20;
constexpr uint32_t kMaxChunks = kMaxPages / kChunk;
constexpr uint32_t kMaxRequests = 1024;
constexpr uint32_t kMaxPairs = 65536;
constexpr int kBatch = 8;                        // pages a thread copies at once
constexpr uint32_t kTile = 1024;                 // pairs that are held against each other; more go by bitmaps

typedef uint32_t U4 __attribute__((ext_vector_type(4)));

// ---- Columns of a page over all pools -----------------------------------------------------------------------------------

struct Pools {
  struct One {
    unsigned char* address;
    uint64_t page_bytes, layer_bytes;
    uint32_t columns, per_page;  // 16-byte columns of the pool's pages over all layers, and of one layer
  } pool[ROOST_AMD_MAX_PAGE_POOLS];
  uint32_t count;
  uint32_t columns;  // of all pools
};

// Page 0's address of column c, and the bytes between pages.
__device__ __forceinline__ unsigned char* ColumnAt(const Pools& p, uint32_t c, uint64_t& page_bytes) {
  uint32_t i = 0;
  while (i + 1 < p.count && c >= p.pool[i].columns) c -= p.pool[i].columns, ++i;
  const Pools::One& o = p.pool[i];
  const uint32_t layer = c / o.per_page;
  page_bytes = o.page_bytes;
  return o.address + layer * o.layer_bytes + uint64_t{16} * (c - layer * o.per_page);
}

// Copied and moved pages are passed through once: their lines give way first in the L2 (1,200 pages of 408 KiB copied: 209 us,
// 215 by ordinary accesses). A fork's parent page is not: its other children read it too (128 forks of 16: 44 us, 54 so).
__device__ __forceinline__ U4 Load(const unsigned char* at) { return __builtin_nontemporal_load(reinterpret_cast<const U4*>(at)); }
__device__ __forceinline__ void Store(unsigned char* at, U4 v) { __builtin_nontemporal_store(v, reinterpret_cast<U4*>(at)); }

// ---- CacheCopy ------------------------------------------------------------------------------------------------------------

// Whether pair (src, dst) has to keep its place among the others: it reads or writes a page that another writes, or writes
// one that another reads.
__device__ __forceinline__ bool Meets(int2 a, int2 b) { return a.x == b.y || a.y == b.x || a.y == b.y; }
__device__ __forceinline__ bool InPools(int2 p, uint32_t pages) {
  return static_cast<uint32_t>(p.x) < pages && static_cast<uint32_t>(p.y) < pages;
}

// What a long list's pairs do with each page, as bitmaps over the pages.
struct PageMarks {
  uint32_t *from, *to, *to_twice;  // [words] each
  uint32_t words;
};

__global__ void __launch_bounds__(kThreads) ClearMarksKernel(PageMarks m) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i < 3 * m.words) m.from[i] = 0;  // the three lie one behind the other
}

__global__ void __launch_bounds__(kThreads) MarkKernel(PageMarks m, const int2* __restrict__ pairs, uint32_t count,
                                                       uint32_t pages) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= count) return;
  const int2 p = pairs[i];
  if (!InPools(p, pages)) return;
  const uint32_t to = 1u << (p.y % 32);
  atomicOr(&m.from[p.x / 32], 1u << (p.x % 32));
  if (atomicOr(&m.to[p.y / 32], to) & to) atomicOr(&m.to_twice[p.y / 32], to);
}

__device__ __forceinline__ bool Meets(const PageMarks& m, int2 p) {
  const auto at = [](const uint32_t* bits, int32_t page) { return (bits[page / 32] >> (page % 32) & 1) != 0; };
  return at(m.to, p.x) || at(m.from, p.y) || at(m.to_twice, p.y);
}

// blockIdx.x: 256 columns. blockIdx.y > 0: a group of `per` pairs, those of them that meet no other pair. blockIdx.y = 0: the
// pairs that meet another, one after the other; each thread sees its column alone, so their order is its own.
// kMarked: the pairs that meet others are told by the bitmaps, else every pair is held against all kTile of them or fewer.
template <bool kMarked>
__global__ void __launch_bounds__(kThreads) CacheCopyKernel(Pools pools, const int2* __restrict__ pairs, uint32_t count,
                                                            uint32_t pages, uint32_t per, PageMarks marks) {
  __shared__ int2 all[kMarked ? 1 : kTile];
  __shared__ uint32_t meets[kThreads / 32];
  const uint32_t c = blockIdx.x * kThreads + threadIdx.x;
  uint64_t page_bytes = 0;
  unsigned char* const at = ColumnAt(pools, min(c, pools.columns - 1), page_bytes);
  const bool mine = c < pools.columns;
  if constexpr (!kMarked) {
    for (uint32_t j = threadIdx.x; j < count; j += kThreads) all[j] = pairs[j];
  }

  if (blockIdx.y > 0) {
    const uint32_t first = (blockIdx.y - 1) * per, n = min(per, count - first);
    if (threadIdx.x == 0) meets[0] = 0;
    __syncthreads();
    for (uint32_t i = 0; i < n; ++i) {
      const int2 p = pairs[first + i];
      if (!InPools(p, pages)) {
        if (threadIdx.x == 0) atomicOr(&meets[0], 1u << i);
        continue;
      }
      bool met = false;
      if constexpr (kMarked) {
        met = threadIdx.x == 0 && Meets(marks, p);
      } else {
        for (uint32_t j = threadIdx.x; j < count; j += kThreads) {
          met |= j != first + i && InPools(all[j], pages) && Meets(p, all[j]);
        }
      }
      if (met) atomicOr(&meets[0], 1u << i);
    }
    __syncthreads();
    const uint32_t skip = meets[0];
    U4 v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (mine && i < static_cast<int>(n) && !(skip >> i & 1)) {
        v[i] = Load(at + pairs[first + i].x * page_bytes);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (mine && i < static_cast<int>(n) && !(skip >> i & 1)) {
        Store(at + pairs[first + i].y * page_bytes, v[i]);
      }
    }
    return;
  }

  for (uint32_t first = 0; first < count; first += kThreads) {
    __syncthreads();
    if (threadIdx.x < kThreads / 32) meets[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t i = first + threadIdx.x;
    bool met = false;
    if (i < count) {
      const int2 p = pairs[i];
      if (InPools(p, pages)) {
        if constexpr (kMarked) {
          met = Meets(marks, p);
        } else {
          for (uint32_t j = 0; j < count; ++j) met |= j != i && InPools(all[j], pages) && Meets(p, all[j]);
        }
      }
    }
    if (met) atomicOr(&meets[threadIdx.x / 32], 1u << (threadIdx.x % 32));
    __syncthreads();
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
      for (uint32_t bits = meets[w]; bits != 0; bits &= bits - 1) {
        const int2 p = pairs[first + 32 * w + __builtin_ctz(bits)];
        if (mine) *reinterpret_cast<U4*>(at + p.y * page_bytes) = *reinterpret_cast<const U4*>(at + p.x * page_bytes);
      }
    }
  }
}

// ---- The tables -------------------------------------------------------------------------------------------------------------

struct Tables {
  int32_t *blocks, *lengths, *refs;
  uint32_t sequences, max_blocks, pages, page_shift;
};

// The workspace: a bitmap of the pages asked for (free or used), their number in each chunk, and either what the requests
// were found to need or, for compact, the pages that move, those they move to and each moving page's place among them.
struct Scratch {
  uint64_t* bits;      // [chunks * kWords]
  uint32_t* counts;    // [chunks]
  int32_t *first, *need;  // [kMaxRequests]
  int32_t *movers, *holes, *place;  // [pages]
  uint32_t chunks;
};

__host__ __device__ constexpr uint64_t ScratchBytes(uint32_t pages) {
  const uint64_t chunks = (pages + kChunk - 1) / kChunk;
  return chunks * kWords * 8 + chunks * 4 + 8 * kMaxRequests + 12 * uint64_t{pages} + 256;
}

struct Requests {
  const int32_t* list;
  const int32_t* cu;
  int64_t* slots;
  uint64_t slot_count;
  int32_t* status;
  uint32_t count;
};

__device__ __forceinline__ int32_t PagesOf(int64_t tokens, uint32_t shift) {
  return static_cast<int32_t>((tokens + (int64_t{1} << shift) - 1) >> shift);
}
// A sequence's length as its row can hold it.
__device__ __forceinline__ int64_t LengthOf(const Tables& t, uint32_t s) {
  return min(static_cast<int64_t>(max(t.lengths[s], 0)), static_cast<int64_t>(t.max_blocks) << t.page_shift);
}

// The sum over the threads before this one; `total`: over all. lds: kThreads / 64 words.
__device__ __forceinline__ uint32_t Before(uint32_t v, uint32_t* lds, uint32_t& total) {
  uint32_t sum = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = static_cast<uint32_t>(__shfl_up(static_cast<int>(sum), d));
    if (static_cast<int>(threadIdx.x % 64) >= d) sum += o;
  }
  __syncthreads();
  if (threadIdx.x % 64 == 63) lds[threadIdx.x / 64] = sum;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
  for (uint32_t w = 0; w < kThreads / 64; ++w) {
    if (w < threadIdx.x / 64) before += lds[w];
    total += lds[w];
  }
  return before + sum - v;
}

// Block c < chunks: chunk c's bits (used == 0: of its free pages, else of its used ones) and count. The last block, if there
// is one more: what each request needs and how many pages the earlier ones do. kFork: one page where the parent's last is
// partly filled. Otherwise (grow): the pages of the new tokens.
template <bool kFork>
__global__ void __launch_bounds__(kThreads) ScanKernel(Tables t, Scratch s, Requests r, int used) {
  __shared__ uint32_t lds[kThreads / 64];
  if (blockIdx.x < s.chunks) {
    const uint32_t base = blockIdx.x * kChunk;
    uint32_t n = 0;
#pragma unroll
    for (uint32_t k = 0; k < kChunk / kThreads; ++k) {
      const uint32_t p = base + k * kThreads + threadIdx.x;
      const uint64_t word = __ballot(p < t.pages && (t.refs[p] > 0) == (used != 0));
      if (threadIdx.x % 64 == 0) s.bits[(base + k * kThreads + threadIdx.x) / 64] = word;
      n += static_cast<uint32_t>(__popcll(word));
    }
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t sum = 0;
      for (uint32_t w = 0; w < kThreads / 64; ++w) sum += lds[w];
      s.counts[blockIdx.x] = sum;
    }
    return;
  }

  __shared__ __attribute__((aligned(16))) int32_t named[kMaxRequests];  // the sequence that a request writes
  for (uint32_t i = threadIdx.x; i < r.count; i += kThreads) named[i] = kFork ? r.list[2 * i + 1] : r.list[i];
  __syncthreads();
  const auto needed = [&](uint32_t i) -> int32_t {  // pages, or -1 for a request that is refused
    const int32_t to = named[i];
    if (static_cast<uint32_t>(to) >= t.sequences) return -1;
    // Four names a read and no way out of the loop: the reads overlap (128 requests: 13 us one by one).
    bool again = false;
#pragma unroll 4
    for (uint32_t j = 0; j < i; j += 4) {
      const int4 four = *reinterpret_cast<const int4*>(&named[j]);
      again |= (four.x == to) | (j + 1 < i && four.y == to) | (j + 2 < i && four.z == to) | (j + 3 < i && four.w == to);
    }
    if (again) return -1;
    const int64_t have = LengthOf(t, to);
    if constexpr (kFork) {
      const int32_t from = r.list[2 * i];
      if (static_cast<uint32_t>(from) >= t.sequences || have > 0) return -1;
      const int64_t len = LengthOf(t, from);
      return len > 0 ? (len & ((int64_t{1} << t.page_shift) - 1)) != 0 : -1;
    } else {
      const int64_t more = static_cast<int64_t>(r.cu[i + 1]) - r.cu[i];
      if (more < 0 || r.cu[i] < 0 || have + more > static_cast<int64_t>(t.max_blocks) << t.page_shift ||
          have + more > 0x7FFFFFFF) {
        return -1;
      }
      return PagesOf(have + more, t.page_shift) - PagesOf(have, t.page_shift);
    }
  };
  uint32_t carry = 0;
  for (uint32_t first = 0; first < r.count; first += kThreads) {
    const uint32_t i = first + threadIdx.x;
    const int32_t need = i < r.count ? needed(i) : 0;
    uint32_t total;
    // A need above all pages there can be counts as that: the sums stay in 32 bits.
    const uint32_t at = carry + Before(min(static_cast<uint32_t>(max(need, 0)), kMaxPages + 1), lds, total);
    if (i < r.count) {
      s.first[i] = static_cast<int32_t>(min(at, 0x7FFFFFFFu));
      s.need[i] = need;
    }
    carry = min(carry + total, 0x7FFFFFFFu);
  }
}

// ends[c]: bits set in chunks 0 .. c, in LDS, for every chunk of the workgroup's `chunks`; returns the last.
__device__ __forceinline__ uint32_t SumCounts(const Scratch& s, uint32_t* ends, uint32_t* lds) {
  constexpr uint32_t kEach = kMaxChunks / kThreads;
  const uint32_t each = (s.chunks + kThreads - 1) / kThreads;
  uint32_t sum = 0;
  for (uint32_t k = 0; k < kEach && k < each; ++k) {
    const uint32_t c = threadIdx.x * each + k;
    sum += c < s.chunks ? s.counts[c] : 0;
  }
  uint32_t total;
  uint32_t at = Before(sum, lds, total);
  for (uint32_t k = 0; k < kEach && k < each; ++k) {
    const uint32_t c = threadIdx.x * each + k;
    if (c >= s.chunks) break;
    at += s.counts[c];
    ends[c] = at;
  }
  __syncthreads();
  return total;
}

// The page of the rank-th set bit (from 0; there is one).
__device__ __forceinline__ uint32_t Select(const Scratch& s, const uint32_t* ends, uint32_t rank) {
  uint32_t lo = 0, hi = s.chunks - 1;  // the first chunk whose end is above the rank
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (ends[mid] > rank) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  rank -= lo > 0 ? ends[lo - 1] : 0;
  const uint64_t* words = s.bits + uint64_t{lo} * kWords;
  uint32_t w = 0;
  uint64_t word = words[0];
  for (uint32_t n = static_cast<uint32_t>(__popcll(word)); w + 1 < kWords && rank >= n; n = static_cast<uint32_t>(__popcll(word))) {
    rank -= n;
    word = words[++w];
  }
  for (; rank > 0; --rank) word &= word - 1;
  return lo * kChunk + 64 * w + static_cast<uint32_t>(__builtin_ctzll(word));
}

// Block (i, 0): request i's tables. Block (i, y > 0): 256 columns' share of its page's copy.
__global__ void __launch_bounds__(kThreads) ForkKernel(Tables t, Scratch s, Requests r, Pools pools) {
  __shared__ uint32_t ends[kMaxChunks];
  __shared__ uint32_t lds[kThreads / 64];
  const uint32_t i = blockIdx.x;
  const int32_t need = s.need[i];
  if (need < 0 || (need == 0 && blockIdx.y > 0)) {
    if (need < 0 && blockIdx.y == 0 && threadIdx.x == 0 && r.status != nullptr) r.status[i] = 0;
    return;
  }
  uint32_t page = 0;
  bool given = true;
  if (need > 0) {
    const uint32_t rank = static_cast<uint32_t>(s.first[i]);
    given = rank < SumCounts(s, ends, lds);
    if (given) page = Select(s, ends, rank);
  }
  if (blockIdx.y == 0 && threadIdx.x == 0 && r.status != nullptr) r.status[i] = given;
  if (!given) return;
  const uint32_t parent = static_cast<uint32_t>(r.list[2 * i]), child = static_cast<uint32_t>(r.list[2 * i + 1]);
  const int64_t len = LengthOf(t, parent);
  const uint32_t whole = static_cast<uint32_t>(len >> t.page_shift);
  const int32_t* from = t.blocks + uint64_t{parent} * t.max_blocks;
  if (blockIdx.y == 0) {
    int32_t* to = t.blocks + uint64_t{child} * t.max_blocks;
    for (uint32_t b = threadIdx.x; b < whole; b += kThreads) {
      const int32_t p = from[b];
      to[b] = p;
      if (static_cast<uint32_t>(p) < t.pages) atomicAdd(&t.refs[p], 1);
    }
    if (threadIdx.x == 0) {
      if (need > 0) {
        to[whole] = static_cast<int32_t>(page);
        t.refs[page] = 1;
      }
      t.lengths[child] = static_cast<int32_t>(len);
    }
    return;
  }
  const int32_t old = from[whole];
  if (static_cast<uint32_t>(old) >= t.pages) return;
  for (uint32_t c = (blockIdx.y - 1) * kThreads + threadIdx.x; c < pools.columns; c += (gridDim.y - 1) * kThreads) {
    uint64_t bytes;
    unsigned char* const at = ColumnAt(pools, c, bytes);
    *reinterpret_cast<U4*>(at + page * bytes) = *reinterpret_cast<const U4*>(at + old * bytes);
  }
}

// Block i: request i.
__global__ void __launch_bounds__(kThreads) GrowKernel(Tables t, Scratch s, Requests r) {
  __shared__ uint32_t ends[kMaxChunks];
  __shared__ uint32_t lds[kThreads / 64];
  const uint32_t i = blockIdx.x;
  const int32_t need = s.need[i];
  const uint32_t rank = static_cast<uint32_t>(s.first[i]);
  bool given = need >= 0;
  if (need > 0) given = uint64_t{rank} + static_cast<uint32_t>(need) <= SumCounts(s, ends, lds);
  if (threadIdx.x == 0 && r.status != nullptr) r.status[i] = given;
  const int64_t begin = r.cu[i], more = static_cast<int64_t>(r.cu[i + 1]) - begin;
  const auto slot_at = [&](int64_t k) { return static_cast<uint64_t>(begin + k) < r.slot_count; };
  if (!given) {
    for (int64_t k = threadIdx.x; begin >= 0 && k < more; k += kThreads) {
      if (!slot_at(k)) break;
      r.slots[begin + k] = -1;
    }
    return;
  }
  const uint32_t seq = static_cast<uint32_t>(r.list[i]);
  const int64_t have = LengthOf(t, seq);
  int32_t* row = t.blocks + uint64_t{seq} * t.max_blocks;
  const int32_t had = PagesOf(have, t.page_shift);
  for (int32_t k = static_cast<int32_t>(threadIdx.x); k < need; k += kThreads) {
    const uint32_t page = Select(s, ends, rank + static_cast<uint32_t>(k));
    row[had + k] = static_cast<int32_t>(page);
    t.refs[page] = 1;
  }
  __syncthreads();  // the row, written by this workgroup, is read below; nobody else writes it
  for (int64_t k = threadIdx.x; k < more; k += kThreads) {
    if (!slot_at(k)) break;
    const int64_t pos = have + k;
    const int32_t page = row[pos >> t.page_shift];
    const int64_t offset = pos & ((int64_t{1} << t.page_shift) - 1);
    r.slots[begin + k] = static_cast<uint32_t>(page) < t.pages ? (static_cast<int64_t>(page) << t.page_shift) + offset : -1;
  }
  if (threadIdx.x == 0) t.lengths[seq] = static_cast<int32_t>(have + more);
}

// Block i: request i's sequence. Whoever takes its length frees it, so one named twice is freed once.
__global__ void __launch_bounds__(kThreads) FreeKernel(Tables t, Requests r) {
  __shared__ int32_t length;
  const int32_t seq = r.list[blockIdx.x];
  if (static_cast<uint32_t>(seq) >= t.sequences) return;
  if (threadIdx.x == 0) length = atomicExch(&t.lengths[seq], 0);
  __syncthreads();
  const int64_t len = min(static_cast<int64_t>(max(length, 0)), static_cast<int64_t>(t.max_blocks) << t.page_shift);
  int32_t* row = t.blocks + static_cast<uint64_t>(seq) * t.max_blocks;
  for (int32_t b = static_cast<int32_t>(threadIdx.x); b < PagesOf(len, t.page_shift); b += kThreads) {
    const int32_t p = row[b];
    if (static_cast<uint32_t>(p) < t.pages) {
      atomicSub(&t.refs[p], 1);
      row[b] = -1;
    }
  }
}

// Chunk blockIdx.x: the places of its used pages from page `live` on among the movers, and of its free pages below among the
// holes. Both have the same number: live - (used pages below live) = (free pages below live).
__global__ void __launch_bounds__(kThreads) PlacesKernel(Tables t, Scratch s, int32_t* status) {
  __shared__ uint32_t ends[kMaxChunks];
  __shared__ uint32_t lds[kThreads / 64];
  __shared__ uint32_t below_live, words[kWords];
  const uint32_t live = SumCounts(s, ends, lds);
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0 && status != nullptr) status[0] = static_cast<int32_t>(live);
    // Used pages below page `live`: the movers' places start behind them.
    const uint32_t c = live / kChunk;
    uint32_t n = c > 0 ? ends[c - 1] : 0;
    if (c < s.chunks) {
      const uint64_t* w = s.bits + uint64_t{c} * kWords;
      const uint32_t in = live % kChunk;
      for (uint32_t k = 0; k < in / 64; ++k) n += static_cast<uint32_t>(__popcll(w[k]));
      if (in % 64 != 0) n += static_cast<uint32_t>(__popcll(w[in / 64] & ((uint64_t{1} << (in % 64)) - 1)));
    }
    below_live = n;
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + kWords) {  // used pages before each of the chunk's words
    const uint32_t k = threadIdx.x - 64;
    const uint64_t* w = s.bits + uint64_t{blockIdx.x} * kWords;
    uint32_t before = blockIdx.x > 0 ? ends[blockIdx.x - 1] : 0;
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) before += i < k ? static_cast<uint32_t>(__popcll(w[i])) : 0;
    words[k] = before;
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) s.counts[s.chunks] = live - below_live;  // movers
  for (uint32_t k = threadIdx.x; k < kChunk; k += kThreads) {
    const uint32_t p = blockIdx.x * kChunk + k;
    if (p >= t.pages) break;
    const uint64_t word = s.bits[p / 64];
    const bool used = word >> (p % 64) & 1;
    const uint32_t before = words[k / 64] + static_cast<uint32_t>(__popcll(word & ((uint64_t{1} << (p % 64)) - 1)));
    if (used && p >= live) {
      s.movers[before - below_live] = static_cast<int32_t>(p);
      s.place[p] = static_cast<int32_t>(before - below_live);
    } else {
      s.place[p] = -1;
      if (!used && p < live) s.holes[p - before] = static_cast<int32_t>(p);
    }
  }
}

// Every sequence's row, dealt over the grid; and blockIdx.x: 256 columns of the moving pages, kBatch at a time, whose groups
// blockIdx.y deals. A thread keeps its column, so an address is one product a page.
__global__ void __launch_bounds__(kThreads) MoveKernel(Tables t, Scratch s, Pools pools) {
  const uint32_t movers = s.counts[s.chunks];
  if (movers == 0) return;
  for (uint64_t q = uint64_t{blockIdx.y} * gridDim.x + blockIdx.x; q < t.sequences; q += uint64_t{gridDim.y} * gridDim.x) {
    int32_t* row = t.blocks + q * t.max_blocks;
    const int32_t n = PagesOf(LengthOf(t, static_cast<uint32_t>(q)), t.page_shift);
    for (int32_t b = static_cast<int32_t>(threadIdx.x); b < n; b += kThreads) {
      const int32_t p = row[b];
      if (static_cast<uint32_t>(p) >= t.pages) continue;
      const int32_t place = s.place[p];
      if (place >= 0) row[b] = s.holes[place];
    }
  }
  const uint32_t c = blockIdx.x * kThreads + threadIdx.x;
  const bool mine = c < pools.columns;
  uint64_t bytes;
  unsigned char* const at = ColumnAt(pools, min(c, pools.columns - 1), bytes);
  for (uint32_t first = blockIdx.y * kBatch; first < movers; first += gridDim.y * kBatch) {
    const uint32_t n = min(movers - first, uint32_t{kBatch});
    if (blockIdx.x == 0 && threadIdx.x < n) {
      const int32_t from = s.movers[first + threadIdx.x], to = s.holes[first + threadIdx.x];
      t.refs[to] = t.refs[from];
      t.refs[from] = 0;
    }
    U4 v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (mine && i < static_cast<int>(n)) v[i] = Load(at + s.movers[first + i] * bytes);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (mine && i < static_cast<int>(n)) Store(at + s.holes[first + i] * bytes, v[i]);
    }
  }
}

// ---- Admission ----------------------------------------------------------------------------------------------------------------

roost::Extent PoolExtent(const RoostAmdPagePool& p, uint32_t pages) {
  return roost::ExtentOf(p.address, p.layers, p.layers > 1 ? p.layer_bytes : 0, p.page_bytes * pages);
}

void AdmitPools(roost::Gate& gate, const RoostAmdPagePool* pools, uint32_t count, uint32_t pages, Pools& out) {
  gate.Expect(pools != nullptr && count > 0 && count <= ROOST_AMD_MAX_PAGE_POOLS, ROOST_STATUS_INVALID_ARGUMENT,
              "%u pools at %p: 1 to %u are taken", count, static_cast<const void*>(pools), ROOST_AMD_MAX_PAGE_POOLS);
  if (!gate.ok()) return;
  out = Pools{};
  out.count = count;
  uint64_t columns = 0;
  for (uint32_t i = 0; i < count; ++i) {
    const RoostAmdPagePool& p = pools[i];
    gate.Expect(p.reserved0 == 0, ROOST_STATUS_INVALID_ARGUMENT, "pool %u: reserved0 = %u, must be 0", i, p.reserved0)
        .Expect(p.address != nullptr && roost::IsAligned(p.address, 16), ROOST_STATUS_INVALID_ARGUMENT,
                "pool %u: address %p is NULL or not 16-byte aligned", i, p.address)
        .Expect(p.layers > 0 && p.page_bytes > 0 && p.page_bytes % 16 == 0, ROOST_STATUS_INVALID_ARGUMENT,
                "pool %u: %u layers of pages of %llu bytes; pages are multiples of 16 bytes", i, p.layers,
                static_cast<unsigned long long>(p.page_bytes))
        .Expect(p.page_bytes <= (uint64_t{1} << 34), ROOST_STATUS_UNSUPPORTED, "pool %u: pages of %llu bytes, above 2^34", i,
                static_cast<unsigned long long>(p.page_bytes))
        .Expect(p.layers == 1 || (p.layer_bytes % 16 == 0 && p.layer_bytes >= p.page_bytes * pages &&
                                  p.layer_bytes <= (uint64_t{1} << 40)),
                ROOST_STATUS_INVALID_ARGUMENT,
                "pool %u: layers %llu bytes apart: no multiple of 16, below %u pages of %llu, or above 2^40", i,
                static_cast<unsigned long long>(p.layer_bytes), pages, static_cast<unsigned long long>(p.page_bytes));
    if (!gate.ok()) return;
    const uint64_t mine = p.page_bytes / 16 * p.layers;
    columns += mine;
    gate.Expect(columns <= 0x7FFFFFFF, ROOST_STATUS_UNSUPPORTED, "a page of all pools is above 2^35 bytes");
    for (uint32_t j = 0; j < i && gate.ok(); ++j) {
      gate.Expect(!roost::Overlap(PoolExtent(p, pages), PoolExtent(pools[j], pages)), ROOST_STATUS_INVALID_ARGUMENT,
                  "pools %u and %u overlap", j, i);
    }
    if (!gate.ok()) return;
    out.pool[i] = {static_cast<unsigned char*>(p.address), p.page_bytes, p.layer_bytes, static_cast<uint32_t>(mine),
                   static_cast<uint32_t>(p.page_bytes / 16)};
  }
  out.columns = static_cast<uint32_t>(columns);
}

constexpr char kCopy[] = "cache_copy";

RoostStatus AdmitCopy(const RoostAmdCacheCopyParams& p, Pools& pools) {
  roost::Gate gate(kCopy);
  gate.Expect(p.reserved0 == 0, ROOST_STATUS_INVALID_ARGUMENT, "reserved0 = %u, must be 0", p.reserved0)
      .Expect(p.pages > 0 && p.pages <= kMaxPages, ROOST_STATUS_UNSUPPORTED, "pages = %u, not 1 to %u", p.pages, kMaxPages)
      .Expect(p.count <= kMaxPairs, ROOST_STATUS_UNSUPPORTED, "count = %u, above %u", p.count, kMaxPairs)
      .Tensor("pairs", p.pairs, ROOST_DTYPE_I32, 2 * uint64_t{p.count})
      .Aligned("pairs", p.pairs.address, 8);
  ROOST_GATE_RETURN(gate);
  AdmitPools(gate, p.pools, p.pool_count, p.pages, pools);
  for (uint32_t i = 0; gate.ok() && i < p.pool_count; ++i) {
    gate.Expect(!roost::Overlap(PoolExtent(p.pools[i], p.pages), roost::ExtentOf(p.pairs.address, 8 * uint64_t{p.count})),
                ROOST_STATUS_INVALID_ARGUMENT, "pool %u overlaps pairs", i);
  }
  return gate.status();
}

uint64_t CopyScratchBytes(const RoostAmdCacheCopyParams& p) { return p.count <= kTile ? 0 : 12 * ((uint64_t{p.pages} + 31) / 32); }

enum class Call { kFork, kGrow, kFree, kCompact };

struct Admitted {
  Tables tables{};
  Requests requests{};
  Pools pools{};
};

RoostStatus Admit(const RoostAmdCachePagesParams& p, const char* op, Call call, Admitted& a) {
  roost::Gate gate(op);
  const uint64_t entries = uint64_t{p.sequences} * p.max_blocks;
  gate.Expect(p.sequences > 0 && p.max_blocks > 0 && entries <= 0x7FFFFFFF && p.sequences <= (1u << 24), ROOST_STATUS_UNSUPPORTED,
              "block_tables of %u x %u: 1 to 2^31 - 1 entries of up to 2^24 sequences are taken", p.sequences, p.max_blocks)
      .Expect(p.pages > 0 && p.pages <= kMaxPages, ROOST_STATUS_UNSUPPORTED, "pages = %u, not 1 to %u", p.pages, kMaxPages)
      .Expect(roost::IsPow2(p.page_size) && p.page_size <= (1u << 20), ROOST_STATUS_UNSUPPORTED,
              "page_size = %u is no power of two up to 2^20", p.page_size)
      .Expect(p.count <= kMaxRequests, ROOST_STATUS_UNSUPPORTED, "count = %u, above %u", p.count, kMaxRequests)
      .Tensor("block_tables", p.block_tables, ROOST_DTYPE_I32, entries)
      .Tensor("lengths", p.lengths, ROOST_DTYPE_I32, p.sequences)
      .Tensor("refs", p.refs, ROOST_DTYPE_I32, p.pages)
      .Aligned("block_tables", p.block_tables.address, 4)
      .Aligned("lengths", p.lengths.address, 4)
      .Aligned("refs", p.refs.address, 4);
  ROOST_GATE_RETURN(gate);
  if (call != Call::kCompact) {
    gate.Tensor("requests", p.requests, ROOST_DTYPE_I32, uint64_t{p.count} * (call == Call::kFork ? 2 : 1))
        .Aligned("requests", p.requests.address, 4);
  }
  if (call == Call::kGrow) {
    gate.Tensor("cu_seqlens", p.cu_seqlens, ROOST_DTYPE_I32, p.count ? p.count + 1 : 0)
        .Aligned("cu_seqlens", p.cu_seqlens.address, 4)
        .Tensor("slot_mapping", p.slot_mapping, ROOST_DTYPE_I64, 0)
        .Expect(p.slot_mapping.address != nullptr || p.slot_mapping.length == 0, ROOST_STATUS_INVALID_ARGUMENT,
                "slot_mapping: address is NULL")
        .Aligned("slot_mapping", p.slot_mapping.address, 8);
  }
  const uint64_t statuses = call == Call::kCompact ? 1 : p.count;
  if (call != Call::kFree) {
    gate.OptionalTensor("status", p.status, ROOST_DTYPE_I32, statuses).Aligned("status", p.status.address, 4);
  }
  ROOST_GATE_RETURN(gate);
  const bool pools = call == Call::kFork || call == Call::kCompact;
  if (pools) AdmitPools(gate, p.pools, p.pool_count, p.pages, a.pools);
  ROOST_GATE_RETURN(gate);
  const auto of = [](const RoostDeviceSpan& s, uint64_t elements, uint64_t bytes) {
    return roost::ExtentOf(s.address, elements * bytes);
  };
  // Everything that the call writes, then what it only reads.
  const uint64_t requests = call == Call::kCompact ? 0 : uint64_t{p.count} * (call == Call::kFork ? 2 : 1);
  const roost::Extent spans[] = {of(p.block_tables, entries, 4),
                                 of(p.lengths, p.sequences, 4),
                                 of(p.refs, p.pages, 4),
                                 call == Call::kFree ? roost::Extent{} : of(p.status, statuses, 4),
                                 call == Call::kGrow ? of(p.slot_mapping, p.slot_mapping.length, 8) : roost::Extent{},
                                 of(p.requests, requests, 4),
                                 call == Call::kGrow ? of(p.cu_seqlens, p.count + 1, 4) : roost::Extent{}};
  for (int i = 0; i < 7; ++i) {
    for (int j = 0; j < i && j < 5; ++j) {
      gate.Expect(!roost::Overlap(spans[i], spans[j]), ROOST_STATUS_INVALID_ARGUMENT, "spans of the call overlap");
    }
    for (uint32_t k = 0; pools && k < p.pool_count; ++k) {
      gate.Expect(!roost::Overlap(spans[i], PoolExtent(p.pools[k], p.pages)), ROOST_STATUS_INVALID_ARGUMENT,
                  "pool %u overlaps a table of the call", k);
    }
  }
  ROOST_GATE_RETURN(gate);
  a.tables = {static_cast<int32_t*>(p.block_tables.address), static_cast<int32_t*>(p.lengths.address),
              static_cast<int32_t*>(p.refs.address), p.sequences, p.max_blocks, p.pages,
              static_cast<uint32_t>(__builtin_ctz(p.page_size))};
  a.requests = {static_cast<const int32_t*>(p.requests.address), static_cast<const int32_t*>(p.cu_seqlens.address),
                static_cast<int64_t*>(p.slot_mapping.address), p.slot_mapping.length,
                static_cast<int32_t*>(p.status.address), p.count};
  return ROOST_STATUS_OK;
}

Scratch ScratchOf(const RoostWorkspace* ws, uint32_t pages) {
  Scratch s{};
  s.chunks = (pages + kChunk - 1) / kChunk;
  s.bits = static_cast<uint64_t*>(ws->device);
  s.first = reinterpret_cast<int32_t*>(s.bits + uint64_t{s.chunks} * kWords);
  s.need = s.first + kMaxRequests;
  s.movers = s.need + kMaxRequests;
  s.holes = s.movers + pages;
  s.place = s.holes + pages;
  s.counts = reinterpret_cast<uint32_t*>(s.place + pages);  // chunks + 1
  return s;
}

RoostStatus Run(RoostContext* ctx, const void* params, const RoostWorkspace* ws, void* stream, const char* op, Call call) {
  roost::Gate gate(op);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed")
      .Header(params, sizeof(RoostAmdCachePagesParams));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdCachePagesParams*>(params);
  return roost::CatchAll(op, [&]() -> RoostStatus {
    Admitted a;
    ROOST_RETURN_IF_FAILED(Admit(p, op, call, a));
    const uint64_t bytes = call == Call::kFree ? 0 : ScratchBytes(p.pages);
    gate.Expect(roost::HasDeviceRegion(ws, bytes), ROOST_STATUS_WORKSPACE_TOO_SMALL,
                "the call needs %llu bytes of 256-byte aligned device workspace", static_cast<unsigned long long>(bytes));
    ROOST_GATE_RETURN(gate);
    if (call != Call::kCompact && p.count == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    const hipStream_t st = roost::Stream(stream);
    if (call == Call::kFree) {
      FreeKernel<<<p.count, kThreads, 0, st>>>(a.tables, a.requests);
      return roost::HipStatus(hipGetLastError(), op, "kernel launch");
    }
    const Scratch s = ScratchOf(ws, p.pages);
    if (call == Call::kFork) {
      ScanKernel<true><<<s.chunks + 1, kThreads, 0, st>>>(a.tables, s, a.requests, 0);
      // A page's columns over at most 64 workgroups of each request: enough for one fork of a large page to fill the chip's
      // memory pipes, and few enough that many forks do not pay for idle ones.
      const auto pieces = static_cast<uint32_t>(std::min<uint64_t>(roost::CeilDiv(a.pools.columns, kThreads), 64));
      ForkKernel<<<dim3(p.count, 1 + pieces), kThreads, 0, st>>>(a.tables, s, a.requests, a.pools);
    } else if (call == Call::kGrow) {
      ScanKernel<false><<<s.chunks + 1, kThreads, 0, st>>>(a.tables, s, a.requests, 0);
      GrowKernel<<<p.count, kThreads, 0, st>>>(a.tables, s, a.requests);
    } else {
      ScanKernel<false><<<s.chunks, kThreads, 0, st>>>(a.tables, s, a.requests, 1);
      PlacesKernel<<<s.chunks, kThreads, 0, st>>>(a.tables, s, a.requests.status);
      // The number of moving pages is the device's, at most half the pool's. 64 workgroups a CU end evenly over the chip (910 MB
      // moved: 369 us, 460 with 8), and 16,384 that find nothing to move cost 5 us.
      const auto pieces = static_cast<uint32_t>(roost::CeilDiv(a.pools.columns, kThreads));
      const uint64_t groups =
          std::min<uint64_t>(roost::CeilDiv(p.pages, 2 * kBatch), roost::CeilDiv(uint64_t{64} * ctx->compute_units, pieces));
      MoveKernel<<<dim3(pieces, static_cast<uint32_t>(groups)), kThreads, 0, st>>>(a.tables, s, a.pools);
    }
    return roost::HipStatus(hipGetLastError(), op, "kernel launch");
  });
}

}  // namespace

extern "C" ROOST_API RoostStatus roost_amd_cache_copy_workspace(RoostContext* ctx, const void* params,
                                                                RoostWorkspaceSizes* sizes) {
  roost::Gate gate(kCopy);
  gate.Expect(ctx != nullptr && sizes != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "a context and a sizes record are required")
      .Header(params, sizeof(RoostAmdCacheCopyParams));
  ROOST_GATE_RETURN(gate);
  gate.Header(sizes, sizeof(RoostWorkspaceSizes));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdCacheCopyParams*>(params);
  return roost::CatchAll(kCopy, [&]() -> RoostStatus {
    Pools pools;
    ROOST_RETURN_IF_FAILED(AdmitCopy(p, pools));
    sizes->device_bytes = CopyScratchBytes(p);
    sizes->pinned_host_bytes = sizes->plan_bytes = 0;
    sizes->device_alignment = 256;
    return ROOST_STATUS_OK;
  });
}

extern "C" ROOST_API RoostStatus roost_amd_cache_copy_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                          void* stream) {
  roost::Gate gate(kCopy);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed")
      .Header(params, sizeof(RoostAmdCacheCopyParams));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdCacheCopyParams*>(params);
  return roost::CatchAll(kCopy, [&]() -> RoostStatus {
    Pools pools;
    ROOST_RETURN_IF_FAILED(AdmitCopy(p, pools));
    gate.Expect(roost::HasDeviceRegion(ws, CopyScratchBytes(p)), ROOST_STATUS_WORKSPACE_TOO_SMALL,
                "the call needs %llu bytes of 256-byte aligned device workspace",
                static_cast<unsigned long long>(CopyScratchBytes(p)));
    ROOST_GATE_RETURN(gate);
    if (p.count == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    const hipStream_t s = roost::Stream(stream);
    const auto* pairs = static_cast<const int2*>(p.pairs.address);
    const auto pieces = static_cast<uint32_t>(roost::CeilDiv(pools.columns, kThreads));
    // Few pairs go one to a workgroup, so that their copies lie side by side; many by eight, one column's address for all.
    const uint32_t per = uint64_t{pieces} * p.count <= 4 * ctx->compute_units ? 1 : kBatch;
    const dim3 grid(pieces, 1 + static_cast<uint32_t>(roost::CeilDiv(p.count, per)));
    if (p.count <= kTile) {
      CacheCopyKernel<false><<<grid, kThreads, 0, s>>>(pools, pairs, p.count, p.pages, per, PageMarks{});
    } else {
      const uint32_t words = (p.pages + 31) / 32;
      auto* bits = static_cast<uint32_t*>(ws->device);
      const PageMarks marks{bits, bits + words, bits + 2 * words, words};
      ClearMarksKernel<<<static_cast<uint32_t>(roost::CeilDiv(3 * words, kThreads)), kThreads, 0, s>>>(marks);
      MarkKernel<<<static_cast<uint32_t>(roost::CeilDiv(p.count, kThreads)), kThreads, 0, s>>>(marks, pairs, p.count, p.pages);
      CacheCopyKernel<true><<<grid, kThreads, 0, s>>>(pools, pairs, p.count, p.pages, per, marks);
    }
    return roost::HipStatus(hipGetLastError(), kCopy, "kernel launch");
  });
}

extern "C" ROOST_API RoostStatus roost_amd_cache_pages_workspace(RoostContext* ctx, const void* params,
                                                                 RoostWorkspaceSizes* sizes) {
  roost::Gate gate("cache_pages");
  gate.Expect(ctx != nullptr && sizes != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "a context and a sizes record are required")
      .Header(params, sizeof(RoostAmdCachePagesParams));
  ROOST_GATE_RETURN(gate);
  gate.Header(sizes, sizeof(RoostWorkspaceSizes));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdCachePagesParams*>(params);
  gate.Expect(p.pages > 0 && p.pages <= kMaxPages, ROOST_STATUS_UNSUPPORTED, "pages = %u, not 1 to %u", p.pages, kMaxPages);
  ROOST_GATE_RETURN(gate);
  sizes->device_bytes = ScratchBytes(p.pages);
  sizes->pinned_host_bytes = sizes->plan_bytes = 0;
  sizes->device_alignment = 256;
  return ROOST_STATUS_OK;
}

extern "C" ROOST_API RoostStatus roost_amd_cache_fork_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                          void* stream) {
  return Run(ctx, params, ws, stream, "cache_fork", Call::kFork);
}

extern "C" ROOST_API RoostStatus roost_amd_cache_grow_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                          void* stream) {
  return Run(ctx, params, ws, stream, "cache_grow", Call::kGrow);
}

extern "C" ROOST_API RoostStatus roost_amd_cache_free_run(RoostContext* ctx, const void* params, void* stream) {
  return Run(ctx, params, nullptr, stream, "cache_free", Call::kFree);
}

extern "C" ROOST_API RoostStatus roost_amd_cache_compact_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                             void* stream) {
  return Run(ctx, params, ws, stream, "cache_compact", Call::kCompact);
}
