// The bookkeeping of a paged key-value cache, on the device: pages are given, shared, moved and taken back by kernels, so that a decode
// step needs no word from the host and can be captured.
//
// A page is free where no table holds it (refs = 0), and the lowest free ones are taken first, in the order of the call's sequences: what a call does
// follows from the state alone, never from the schedule, and a pool stays dense at its front without a list that has to be kept in order.
//
// A call that gives pages is one block that plans (checks everything, counts what is needed and what there is, and only then
// writes: all or nothing) and, where data has to move, one grid that copies by the plan's list of moves.  The plan is bound by the latency of its passes
// over refs (4 bytes for each page of the pool, 4096 pages a pass); copies of whole pages by memory (74 % of its rate): a page of all layers is one piece of it; of one that is
// filled in part, the filled rows of each (layer, key or value, head) are, and the addresses of their 16 bytes take 57 % of the issue slots beside 24 % of the memory.
#include "rollout.cuh"

namespace metis {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kScan = 4;                   // pages a thread looks at in one pass
constexpr int kPass = kPlanThreads * kScan;
constexpr int kNear = 1024;
constexpr int64_t kMaxSequences = 1 << 17; // a bit for each in shared memory

// A workspace: the header, for each sequence of the call what it needs in front of it, its source and its length, then the moves or the
// pages' new numbers.
struct Header {
  int32_t moves;                           // -1: the call is refused
  int32_t live;
};
struct Move { int32_t from, to, filled, unused; };     // filled: rows of the page
struct Work {
  Header* header;
  int64_t* needs;                          // [n + 1]
  int32_t *from, *to, *length;             // [n]: sequences (-1: none) and what the source holds
  Move* moves;                             // [pages]
  int32_t* renumbered;                     // [pages]
};
__host__ __device__ inline int64_t round16(int64_t v) { return (v + 15) / 16 * 16; }
__host__ __device__ inline int64_t work_bytes(int64_t n, int64_t pages) { return 16 + round16((n + 1) * 8) + 3 * round16(n * 4) + pages * 16 + round16(pages * 4); }
__host__ __device__ inline Work work_view(void* p, int64_t n, int64_t pages) {
  char* at = static_cast<char*>(p);
  Work w;
  w.header = reinterpret_cast<Header*>(at); at += 16;
  w.needs = reinterpret_cast<int64_t*>(at); at += round16((n + 1) * 8);
  w.from = reinterpret_cast<int32_t*>(at); at += round16(n * 4);
  w.to = reinterpret_cast<int32_t*>(at); at += round16(n * 4);
  w.length = reinterpret_cast<int32_t*>(at); at += round16(n * 4);
  w.moves = reinterpret_cast<Move*>(at); at += pages * 16;
  w.renumbered = reinterpret_cast<int32_t*>(at);
  return w;
}

__device__ __forceinline__ void refuse(int32_t* status, int32_t code) { atomicCAS(status, 0, code); }

struct PlanShared {
  int64_t sums[kPlanThreads / 32];
  int32_t code;                            // why the call is refused, the largest of the reasons
  int32_t found[kPass];                    // free pages of a pass, in order
  int32_t needs[kNear];                    // those of the call's sequences where it has no more: a search of the others goes to memory at every step
};

__device__ __forceinline__ void reason(PlanShared& sh, int32_t code) { atomicMax(&sh.code, code); }

// Which of the thread's pages of a pass, from `at`, have what `test` asks of refs: a bit for each.
template <typename Test>
__device__ __forceinline__ uint32_t pages_with(const CacheView& c, int64_t at, const Test& test) {
  static_assert(kScan == 4, "one 16-byte load");
  if (at + kScan <= c.pages && (reinterpret_cast<uintptr_t>(c.refs) & 15) == 0) {
    const int4 v = *reinterpret_cast<const int4*>(c.refs + at);
    return (test(v.x, at) ? 1u : 0u) | (test(v.y, at + 1) ? 2u : 0u) | (test(v.z, at + 2) ? 4u : 0u) | (test(v.w, at + 3) ? 8u : 0u);
  }
  uint32_t with = 0;
  for (int i = 0; i < kScan; ++i) with |= (at + i < c.pages && test(c.refs[at + i], at + i) ? 1u : 0u) << i;
  return with;
}

// Free pages in the order of their numbers: take(rank, page) for each of the first `want`; false, and nothing taken, where there are not so many.  The first kPass are
// kept in shared memory while they are counted; a call for more goes through refs once more.
template <typename Take>
__device__ bool take_lowest(const CacheView& c, int64_t want, PlanShared& sh, const Take& take) {
  auto pass = [&](int64_t base, int64_t found, int64_t from) -> int64_t {        // found: before this pass; from: the rank that sh.found begins with
    const int64_t at = base + (int64_t)threadIdx.x * kScan;
    uint32_t free_ = pages_with(c, at, [](int32_t refs, int64_t) { return refs == 0; });
    int64_t all, rank = found - from + block_exclusive<kPlanThreads>((int64_t)__popc(free_), sh.sums, all);
    for (; free_; free_ &= free_ - 1, ++rank)
      if (rank < kPass) sh.found[rank] = (int32_t)(at + __ffs(free_) - 1);
    return all;
  };
  int64_t found = 0;
  for (int64_t base = 0; base < c.pages && found < want; base += kPass) found += pass(base, found, 0);
  if (found < want) return false;
  __syncthreads();
  if (want <= kPass) {
    for (int64_t r = threadIdx.x; r < want; r += kPlanThreads) take(r, (int64_t)sh.found[r]);
    return true;
  }
  found = 0;
  for (int64_t base = 0; base < c.pages && found < want; base += kPass) {
    const int64_t all = pass(base, found, found);
    __syncthreads();
    for (int64_t r = threadIdx.x; r < all && found + r < want; r += kPlanThreads) take(found + r, (int64_t)sh.found[r]);
    found += all;
    // (the next pass writes behind block_exclusive's barriers)
  }
  return true;
}

// The call's sequence that the rank-th page is for: the last whose needs begin at or before it.
__device__ __forceinline__ int64_t owner_of(const PlanShared& sh, const int64_t* needs, int64_t n, int64_t rank) {
  int64_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if ((n <= kNear ? (int64_t)sh.needs[mid] : needs[mid]) <= rank) lo = mid; else hi = mid;
  }
  return lo;
}

// need(i) -> pages that the call's sequence i takes (checks what it has to); exclusive sums of it in w.needs.
template <typename Need>
__device__ int64_t count_needs(const Work& w, int64_t n, PlanShared& sh, const Need& need) {
  int64_t total = 0;
  for (int64_t base = 0; base < n; base += kPlanThreads) {
    const int64_t i = base + threadIdx.x;
    int64_t all;
    const int64_t before = total + block_exclusive<kPlanThreads>(i < n ? need(i) : (int64_t)0, sh.sums, all);
    if (i < n) w.needs[i] = before;
    if (i < n && n <= kNear) sh.needs[i] = (int32_t)min(before, (int64_t)1 << 30);       // (a call that asks for so many is refused)
    total += all;
  }
  if (threadIdx.x == 0) w.needs[n] = total;
  __syncthreads();
  return total;
}

// Marks a sequence; whether it was marked before.
__device__ __forceinline__ bool marked(uint32_t* marks, int64_t sequence) {
  const uint32_t bit = 1u << (sequence & 31);
  return (atomicOr(&marks[sequence >> 5], bit) & bit) != 0;
}
__device__ __forceinline__ void clear_marks(uint32_t* marks, int64_t sequences) {
  for (int64_t i = threadIdx.x; i < (sequences + 31) / 32; i += kPlanThreads) marks[i] = 0;
}

// The call's sequences have no room for what comes to their ends: append goes by it.
__device__ __forceinline__ void hold_back(const CacheView& c, const void* slots, bool wide, int64_t n) {
  if (!c.refused) return;
  for (int64_t i = threadIdx.x; i < n; i += kPlanThreads) {
    const int64_t slot = slots ? load_index(slots, wide, i) : i;
    if (slot >= 0 && slot < c.sequences) c.refused[slot] = 1;
  }
}

// Whether the call goes ahead; all threads.
__device__ __forceinline__ bool agreed(const CacheView& c, PlanShared& sh, Header* header) {
  __syncthreads();
  if (sh.code == 0) return true;
  if (threadIdx.x == 0) {
    refuse(c.status, sh.code);
    header->moves = -1;
  }
  return false;
}

// ---- reserve --------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(const CacheView c, const void* slots, const void* counts, int64_t count, bool wide, int64_t n, const Work w) {
  extern __shared__ uint32_t marks[];
  __shared__ PlanShared sh;
  grid_dependency_wait();
  if (threadIdx.x == 0) sh.code = 0;
  clear_marks(marks, c.sequences);
  __syncthreads();
  const int64_t page = c.page_size;
  const int64_t want = count_needs(w, n, sh, [&](int64_t i) -> int64_t {
    const int64_t slot = slots ? load_index(slots, wide, i) : i, more = counts ? load_index(counts, wide, i) : count;
    w.to[i] = -1;
    if (slot < 0) return 0;
    if (slot >= c.sequences) { reason(sh, METIS_CACHE_BAD_SLOT); return 0; }
    if (marked(marks, slot)) { reason(sh, METIS_CACHE_TWICE); return 0; }
    const int64_t length = c.lengths[slot];
    // (a count near 2^63 is too long, not negative again; nor is a length taken that no call has left)
    if (length < 0 || more < 0 || more > c.width * page || length + more > c.width * page) { reason(sh, METIS_CACHE_TOO_LONG); return 0; }
    w.to[i] = (int32_t)slot;
    w.length[i] = (int32_t)(length + more);
    return (length + more + page - 1) / page - (length + page - 1) / page;
  });
  if (!agreed(c, sh, w.header)) {
    hold_back(c, slots, wide, n);
    return;
  }
  const bool done = take_lowest(c, want, sh, [&](int64_t rank, int64_t p) {
    const int64_t i = owner_of(sh, w.needs, n, rank), slot = w.to[i];
    const int64_t first = (c.lengths[slot] + page - 1) / page;
    c.tables[slot * c.width + first + rank - w.needs[i]] = (int32_t)p;
    c.refs[p] = 1;
  });
  if (!done) {
    if (threadIdx.x == 0) refuse(c.status, METIS_CACHE_NO_PAGES);
    hold_back(c, slots, wide, n);
    return;
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < n; i += kPlanThreads)
    if (w.to[i] >= 0) {
      c.lengths[w.to[i]] = w.length[i];
      if (c.refused) c.refused[w.to[i]] = 0;
    }
}

// ---- fork -----------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const CacheView c, const void* src, const void* dst, bool wide, int64_t n, bool share, const Work w) {
  extern __shared__ uint32_t marks[];
  __shared__ PlanShared sh;
  grid_dependency_wait();
  if (threadIdx.x == 0) sh.code = 0;
  clear_marks(marks, c.sequences);
  __syncthreads();
  const int64_t page = c.page_size;
  // A page that is absent in the source is absent in its fork: one of its own would hold keys of whoever had it before.
  auto present = [&](int64_t from, int64_t e) {
    const int32_t p = c.tables[from * c.width + e];
    return p >= 0 && p < c.pages;
  };
  const int64_t want = count_needs(w, n, sh, [&](int64_t i) -> int64_t {
    const int64_t from = load_index(src, wide, i), to = load_index(dst, wide, i);
    w.to[i] = -1;
    if (from < 0 || to < 0) return 0;
    if (from >= c.sequences || to >= c.sequences) { reason(sh, METIS_CACHE_BAD_SLOT); return 0; }
    if (marked(marks, to)) { reason(sh, METIS_CACHE_TWICE); return 0; }
    if (c.lengths[to] != 0) { reason(sh, METIS_CACHE_NOT_EMPTY); return 0; }
    const int64_t length = c.lengths[from];
    if (length < 0 || length > c.width * page) { reason(sh, METIS_CACHE_TOO_LONG); return 0; }
    w.from[i] = (int32_t)from;
    w.to[i] = (int32_t)to;
    w.length[i] = (int32_t)length;
    int64_t there = 0;
#pragma unroll 16
    for (int64_t e = share ? length / page : 0; e * page < length; ++e) there += present(from, e);
    return there;
  });
  if (!agreed(c, sh, w.header)) return;
  // (a destination is empty, so that no source's table is written here)
  const bool done = take_lowest(c, want, sh, [&](int64_t rank, int64_t p) {
    const int64_t i = owner_of(sh, w.needs, n, rank), from = w.from[i], to = w.to[i], length = w.length[i];
    const int64_t first = share ? length / page : 0, last = (length - 1) / page, mine = rank - w.needs[i];
    int64_t entry = first + mine;
    if (w.needs[i + 1] - w.needs[i] != last + 1 - first) {      // (some are absent)
      entry = first;
      for (int64_t ahead = mine; entry < last && (!present(from, entry) || ahead-- > 0); ) ++entry;
    }
    c.tables[to * c.width + entry] = (int32_t)p;
    c.refs[p] = 1;
    const int32_t old = c.tables[from * c.width + entry];
    w.moves[rank] = Move{old, (int32_t)p, (int32_t)min(page, length - entry * page), 0};
  });
  if (!done) {
    if (threadIdx.x == 0) {
      refuse(c.status, METIS_CACHE_NO_PAGES);
      w.header->moves = -1;
    }
    return;
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < n; i += kPlanThreads)
    if (w.to[i] >= 0) {
      c.lengths[w.to[i]] = w.length[i];
      if (c.refused) c.refused[w.to[i]] = 0;
    }
  if (threadIdx.x == 0) w.header->moves = (int32_t)want;
}

// ---- compact --------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CacheView c, int32_t* live_out, const Work w) {
  __shared__ PlanShared sh;
  grid_dependency_wait();
  // how many pages are held
  int64_t mine = 0, live;
  for (int64_t p = threadIdx.x; p < c.pages; p += kPlanThreads) mine += c.refs[p] > 0;
  block_exclusive<kPlanThreads>(mine, sh.sums, live);
  // holes below that number and pages at or above it, both in order: as many of the one as of the other
  int64_t holes = 0, movers = 0;
  for (int64_t base = 0; base < c.pages; base += kPass) {
    const int64_t at = base + (int64_t)threadIdx.x * kScan;
    uint32_t hole = pages_with(c, at, [&](int32_t refs, int64_t p) { return refs <= 0 && p < live; });
    uint32_t mover = pages_with(c, at, [&](int32_t refs, int64_t p) { return refs > 0 && p >= live; });
    for (int i = 0; i < kScan; ++i)
      if (at + i < c.pages && !(mover >> i & 1u)) w.renumbered[at + i] = (int32_t)(at + i);
    int64_t all, rank = holes + block_exclusive<kPlanThreads>((int64_t)__popc(hole), sh.sums, all);
    holes += all;
    for (; hole; hole &= hole - 1) w.moves[rank++].to = (int32_t)(at + __ffs(hole) - 1);
    rank = movers + block_exclusive<kPlanThreads>((int64_t)__popc(mover), sh.sums, all);
    movers += all;
    for (; mover; mover &= mover - 1) w.moves[rank++].from = (int32_t)(at + __ffs(mover) - 1);
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < holes; i += kPlanThreads) {
    w.moves[i].filled = c.page_size;
    w.renumbered[w.moves[i].from] = w.moves[i].to;
  }
  if (threadIdx.x == 0) {
    w.header->moves = (int32_t)holes;
    w.header->live = (int32_t)live;
    *live_out = (int32_t)live;
  }
}

// ---- free -----------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(256) free_kernel(const CacheView c, const void* slots, bool wide, int64_t n) {
  __shared__ int32_t length;
  grid_dependency_wait();
  // A block goes through all of the list before it empties anything: a call that names a sequence that the cache does not have does nothing.
  if (slots) {
    bool bad = false;
    for (int64_t i = threadIdx.x; i < n; i += 256) bad |= load_index(slots, wide, i) >= c.sequences;
    if (__syncthreads_or(bad)) {
      if (blockIdx.x == 0 && threadIdx.x == 0) refuse(c.status, METIS_CACHE_BAD_SLOT);
      return;
    }
  }
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int64_t slot = slots ? load_index(slots, wide, i) : i;
    if (slot < 0 || slot >= c.sequences) continue;
    __syncthreads();
    if (threadIdx.x == 0) length = atomicExch(&c.lengths[slot], 0);          // (whoever comes second finds it empty)
    __syncthreads();
    const int64_t held = min(((int64_t)length + c.page_size - 1) / c.page_size, c.width);
    for (int64_t e = threadIdx.x; e < held; e += 256) {
      int32_t* entry = &c.tables[slot * c.width + e];
      const int32_t p = *entry;
      *entry = -1;
      if (p >= 0 && p < c.pages) atomicSub(&c.refs[p], 1);
    }
  }
}

// ---- moves ----------------------------------------------------------------------------------------------------------

enum MoveKind { kFork, kCompact };

// Rows of kRun moves in a row of the plan's list, as pieces of V (16 bytes, or 8 where the rows of 8-bit elements end on half a piece): the filled rows
// of a page lie in `places`, one for each layer, key or value and head, and are taken as one list, so that all threads have work whatever a page is filled with.
// A block takes kBatch pieces a thread, all of its loads before its first store; what a prompt's group of answers copies is read once for kRun of them.  Forks, which
// write more than they read, take four (88 registers a thread are 59): 32 prompts for 16 answers each, 500 tokens, 28 layers of 2 heads of 128, 32.4 -> 28.8 us with
// free (511 tokens, last pages all but full: 56.5 -> 58.4); compactions eight (64 sequences of 30 pages of 28 layers: 293 us, 302 with four).  Runs of 8 or 16: 30.3 and 33.5.
constexpr int kRun = 4;
template <int kBatch, typename V>
__device__ __forceinline__ void move_rows(const CacheView& c, const Move* moves, int count, int place_bytes, int places, int part) {
  const int row = c.head_dim * c.item;
  V v[kBatch];
  int32_t at_from = -1, at_filled = -1;
#pragma unroll 1
  for (int m = 0; m < count; ++m) {
    const Move mv = moves[m];
    if (mv.from < 0 || mv.from >= c.pages) continue;
    const int in_place = mv.filled * row / (int)sizeof(V), all = in_place * places;
    int at = part * kBatch * kMoveThreads + (int)threadIdx.x;
    if (at >= all) continue;
    int place = at / in_place, inside = at - place * in_place;
    const int step_places = kMoveThreads / in_place, step_inside = kMoveThreads - step_places * in_place;
    const bool fresh = mv.from != at_from || mv.filled != at_filled;
    const char* from = c.pool + mv.from * c.page_bytes;
    char* to = c.pool + mv.to * c.page_bytes;
    int off[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      off[i] = at < all ? place * place_bytes + inside * (int)sizeof(V) : -1;
      if (fresh && at < all) v[i] = *reinterpret_cast<const V*>(from + off[i]);
      at += kMoveThreads;
      place += step_places;
      inside += step_inside;
      if (inside >= in_place) { inside -= in_place; ++place; }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (off[i] >= 0) *reinterpret_cast<V*>(to + off[i]) = v[i];
    at_from = mv.from;
    at_filled = mv.filled;
  }
}

// The plan's moves, and what goes with them: of a fork with shared pages the tables' rows and one more holder for each page; of a compaction the
// pages' new numbers in all tables, and their holders.
template <MoveKind kKind>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const CacheView c, const Work w, int64_t n, bool share) {
  constexpr int kBatch = kKind == kFork ? 4 : 8;
  grid_dependency_wait();
  const int32_t moves = w.header->moves;
  if (moves < 0) return;
  const int64_t threads = (int64_t)gridDim.x * kMoveThreads, thread = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x;
  if constexpr (kKind == kFork) {
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
      if (w.to[i] < 0) continue;
      // the entries that the plan has not written are the source's: those that are shared, and absent ones
      const int64_t from = w.from[i], to = w.to[i], length = w.length[i];
      const int64_t shared = share ? length / c.page_size : 0, entries = (length + c.page_size - 1) / c.page_size;
      const bool absent = w.needs[i + 1] - w.needs[i] != entries - shared;
      for (int64_t e = threadIdx.x; e < (absent ? entries : shared); e += kMoveThreads) {
        const int32_t p = c.tables[from * c.width + e];
        const bool there = p >= 0 && p < c.pages;
        if (e < shared || !there) c.tables[to * c.width + e] = there ? p : -1;
        if (e < shared && there) atomicAdd(&c.refs[p], 1);
      }
    }
  } else {
    for (int64_t i = thread; i < moves; i += threads) {
      const Move m = w.moves[i];
      c.refs[m.to] = c.refs[m.from];
      c.refs[m.from] = 0;
    }
    if (moves > 0)
      for (int64_t i = thread; i < c.sequences * c.width; i += threads) {
        const int64_t slot = i / c.width, e = i - slot * c.width;
        if (e * c.page_size >= c.lengths[slot]) continue;
        const int32_t p = c.tables[i];
        if (p >= 0 && p < c.pages) c.tables[i] = w.renumbered[p];
      }
  }
  const int row = c.head_dim * c.item, piece = row * c.page_size, pieces = (int)(c.page_bytes / piece);
  const int unit = row % 16 == 0 ? 16 : 8;
  const int parts = (int)((c.page_bytes / unit + kBatch * kMoveThreads - 1) / (kBatch * kMoveThreads));      // of a full page
  const int run = kKind == kFork ? kRun : 1;
  const int64_t runs = (moves + run - 1) / run;
  for (int64_t j = blockIdx.x; j < runs * parts; j += gridDim.x) {
    const int64_t r = j / parts;
    const int part = (int)(j - r * parts), count = (int)min((int64_t)run, moves - r * run);
    if (unit == 16) move_rows<kBatch, uint4>(c, w.moves + r * run, count, piece, pieces, part);
    else            move_rows<kBatch, uint2>(c, w.moves + r * run, count, piece, pieces, part);
  }
}

int32_t check_call(const metis_cache* cache, CacheView* c, int64_t n, const void* workspace, int64_t bytes) {
  if (const int32_t rc = check_cache(cache, c)) return rc;
  if (n <= 0 || n >= ((int64_t)1 << 31)) return fail(METIS_ERR_BAD_SHAPE, "the number of sequences must be positive");
  if (!workspace || !aligned16(workspace)) return fail(METIS_ERR_BAD_ARGUMENT, "the workspace must be 16-byte aligned");
  if (bytes < work_bytes(n, c->pages)) return fail(METIS_ERR_WORKSPACE, "the workspace has %lld bytes, %lld are needed", (long long)bytes, (long long)work_bytes(n, c->pages));
  return METIS_OK;
}

size_t mark_bytes(const CacheView& c) { return (size_t)((c.sequences + 31) / 32) * 4; }

cudaError_t launch_moves(const CacheView& c, const Work& w, MoveKind kind, int64_t n, bool share, cudaStream_t st) {
  return launch_overlapped(kLaunchShort, kind == kFork ? move_kernel<kFork> : move_kernel<kCompact>, dim3((unsigned)device_sm_count() * 8), dim3(kMoveThreads), 0, st, c, w, n, share);
}

std::atomic<int64_t> launches{0};

}  // namespace

void count_rollout_launches(int n) { launches.fetch_add(n, std::memory_order_relaxed); }

int32_t check_cache(const metis_cache* c, CacheView* v) {
  if (!c || !c->pool || !c->tables || !c->lengths || !c->refs || !c->status) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  if (c->dtype != METIS_DTYPE_BF16 && c->dtype != METIS_DTYPE_E4M3) return fail(METIS_ERR_BAD_ARGUMENT, "the cache's dtype must be bf16 or e4m3");
  if ((c->dtype == METIS_DTYPE_E4M3) != (c->scales != nullptr)) return fail(METIS_ERR_BAD_ARGUMENT, "scales go with e4m3, and with nothing else");
  if (c->flags == METIS_CACHE_HAS_REFUSED && !c->refused) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  const int item = c->dtype == METIS_DTYPE_BF16 ? 2 : 1;
  if (c->pages <= 0 || c->pages >= ((int64_t)1 << 31) || c->layers <= 0 || c->kv_heads <= 0 || c->sequences <= 0 || c->sequences > kMaxSequences || c->width <= 0)
    return fail(METIS_ERR_BAD_SHAPE, "pages, layers, heads, sequences and width must be positive, sequences at most 2^17");
  if (c->page_size <= 0 || c->page_size % 16 != 0) return fail(METIS_ERR_BAD_SHAPE, "page_size must be a multiple of 16");
  if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim % 8 != 0) return fail(METIS_ERR_BAD_SHAPE, "head_dim must be a multiple of 8 up to 256");
  if (c->width > (((int64_t)1 << 31) - 1) / c->page_size) return fail(METIS_ERR_TOO_LARGE, "lengths are 32-bit numbers");
  if ((int64_t)c->layers * 2 * c->kv_heads * c->page_size * c->head_dim >= (int64_t)1 << 30) return fail(METIS_ERR_TOO_LARGE, "a page of all layers has less than 2^30 elements");
  if (!aligned16(c->pool)) return fail(METIS_ERR_BAD_ALIGNMENT, "the pool must be 16-byte aligned");
  *v = {static_cast<char*>(c->pool), (int64_t)c->layers * 2 * c->kv_heads * c->page_size * c->head_dim * item, c->pages, c->tables, c->sequences, c->width, c->lengths,
        c->refs, c->status, c->flags == METIS_CACHE_HAS_REFUSED ? c->refused : nullptr, c->layers, c->kv_heads, c->page_size, c->head_dim, item};
  return METIS_OK;
}

}  // namespace metis

using namespace metis;

extern "C" int64_t metis_rollout_launches(void) { return launches.load(std::memory_order_relaxed); }

extern "C" int32_t metis_cache_check(const metis_cache* cache) {
  CacheView c;
  return check_cache(cache, &c);
}

extern "C" int64_t metis_cache_workspace_bytes(const metis_cache* cache, int64_t n) { return cache && cache->pages > 0 && n >= 0 ? work_bytes(n, cache->pages) : 0; }

extern "C" int32_t metis_cache_reserve(const metis_cache* cache, const void* slots, const void* counts, int64_t count, int32_t index_64, int64_t n, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  CacheView c;
  if (const int32_t rc = check_call(cache, &c, n, workspace, workspace_bytes)) return rc;
  METIS_CUDA_OK(launch_overlapped(kLaunchShort, reserve_kernel, dim3(1), dim3(kPlanThreads), mark_bytes(c), static_cast<cudaStream_t>(stream), c, slots, counts, count,
                                  index_64 != 0, n, work_view(workspace, n, c.pages)));
  count_rollout_launches(1);
  return METIS_OK;
}

extern "C" int32_t metis_cache_fork(const metis_cache* cache, const void* src, const void* dst, int32_t index_64, int64_t n, int32_t share, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  CacheView c;
  if (const int32_t rc = check_call(cache, &c, n, workspace, workspace_bytes)) return rc;
  if (!src || !dst) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Work w = work_view(workspace, n, c.pages);
  METIS_CUDA_OK(launch_overlapped(kLaunchShort, fork_plan_kernel, dim3(1), dim3(kPlanThreads), mark_bytes(c), st, c, src, dst, index_64 != 0, n, share != 0, w));
  METIS_CUDA_OK(launch_moves(c, w, kFork, n, share != 0, st));
  count_rollout_launches(2);
  return METIS_OK;
}

extern "C" int32_t metis_cache_free(const metis_cache* cache, const void* slots, int32_t index_64, int64_t n, void* stream) {
  CacheView c;
  if (const int32_t rc = check_cache(cache, &c)) return rc;
  if (n <= 0 || n >= ((int64_t)1 << 31)) return fail(METIS_ERR_BAD_SHAPE, "the number of sequences must be positive");
  const int64_t most = (int64_t)device_sm_count() * 8;
  METIS_CUDA_OK(launch_overlapped(kLaunchShort, free_kernel, dim3((unsigned)(n < most ? n : most)), dim3(256), 0, static_cast<cudaStream_t>(stream), c, slots, index_64 != 0, n));
  count_rollout_launches(1);
  return METIS_OK;
}

extern "C" int32_t metis_cache_compact(const metis_cache* cache, int32_t* live, void* workspace, int64_t workspace_bytes, void* stream) {
  CacheView c;
  if (const int32_t rc = check_call(cache, &c, 1, workspace, workspace_bytes)) return rc;
  if (!live) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Work w = work_view(workspace, 1, c.pages);
  METIS_CUDA_OK(launch_overlapped(kLaunchShort, compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, c, live, w));
  METIS_CUDA_OK(launch_moves(c, w, kCompact, 1, false, st));
  count_rollout_launches(2);
  return METIS_OK;
}
