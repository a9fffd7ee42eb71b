// paged.cu — a K/V cache in pages: allocation, writes, roll-back of rejected
// drafts, forks, frees and compaction, all on the device without host reads.
//
// Pools: (L, P, H_kv, page, D), one page of one layer contiguous, one head of it
// contiguous in turn.  Bookkeeping, shared by all layers: table (S, M) page ids
// of each slot (-1 beyond the slot's pages), lengths (S,), refs (P,) = number of
// slots that hold the page.  A page with refs = 0 is free; allocation takes the
// lowest free pages in the order of the call's entries, so results do not depend
// on any hidden list.  A part-filled page is never shared.
//
// Every operation is a plan of one CTA (checks everything, scans refs, and leaves
// its decisions in the workspace) and an apply that writes the new table and
// lengths and moves rows: over all SMs in a second launch, or, for small calls, by
// the plan's own CTA.  If the plan rejects the call, it sets the status word and the
// apply copies the bookkeeping through.
//
// Bound: the moves are HBM copies; the plan is latency (a few dependent loads and
// block scans), which is why it is one CTA and the apply starts while it drains.
// A call of 64 slots is 6 to 9 us; fork + free + compact of 64 sequences (236 MB of
// rows moved) 101 us, of which the moves are 73: DRAM reads 237 MB and writes 186, the
// rest of what is written being in L2 still, 5.8 TB/s.  The plans walk all of refs: of
// 5,000 / 20,000 / 100,000 pages a reserve takes 8.6 / 11 / 39 us, an accept 9.7 / 10 / 23,
// a free 5.4 / 6.7 / 13, a compaction that moves little 7.9 / 12 / 50.
#include <algorithm>
#include "common.cuh"

namespace scree {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kThreads = 256;
constexpr int kMaxSlots = 65536;
constexpr int kHereEntries = 2048, kHereWarps = 32;  // see apply_by_plan
constexpr int kSitePagedArgs = 60;    // a slot, count, length or path out of range
constexpr int kSitePagedFull = 61;    // not enough free pages
constexpr int kSitePagedShared = 62;  // a draft, or rows to write, on pages that other slots hold
constexpr int kSitePagedTable = 63;   // a page id out of range

// Decisions of a plan (int32 words at the start of the workspace), then
// slot_of (S), and per entry first / last / start, then page lists.
struct Plan {
  int32_t ok;
  int32_t moves;
};
constexpr int64_t kPlanWords = 16;

struct Book {  // bookkeeping of a call, input and output (never the same memory)
  const int32_t *table, *lengths, *refs;
  int32_t *table_out, *lengths_out, *refs_out;
  int S, M, P, page;
  int32_t* ws;
  int* status;
  __device__ __forceinline__ Plan* plan() const { return reinterpret_cast<Plan*>(ws); }
  __device__ __forceinline__ int32_t* slot_of() const { return ws + kPlanWords; }
  __device__ __forceinline__ int32_t* first() const { return slot_of() + S; }
  __device__ __forceinline__ int32_t* last(int n) const { return first() + n; }
  __device__ __forceinline__ int32_t* start(int n) const { return first() + 2 * (int64_t)n; }
  __device__ __forceinline__ int32_t* list(int n) const { return first() + 3 * (int64_t)n; }
};

struct Pools {
  char *k, *v;
  int L, H;
  int64_t row_bytes;   // D elements
  int64_t page_bytes;  // H * page * row_bytes
  int64_t layer_bytes; // P * page_bytes
};

template <int W> struct Vec;
template <> struct Vec<16> { using T = uint4; };
template <> struct Vec<8> { using T = uint2; };
template <> struct Vec<4> { using T = uint32_t; };
template <> struct Vec<2> { using T = uint16_t; };
template <> struct Vec<1> { using T = uint8_t; };

// ------------------------------------------------------------------ plan pieces

// A plan waits for what came before it on the stream (it may be the apply of an
// earlier call on the same cache) and lets its own apply be launched meanwhile.
__device__ __forceinline__ void begin_plan() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
}

// Exclusive sum over the block (1024 threads) and its total.
__device__ int block_scan(int v, int* total) {
  __shared__ int warp_sum[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // an earlier call's readers are done
  if (lane == 31) warp_sum[w] = x;
  __syncthreads();
  int s = warp_sum[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  const int before = __shfl_sync(0xffffffffu, s, w > 0 ? w - 1 : 0);
  return x - v + (w > 0 ? before : 0);
}

struct SlotSet {  // slots named by the call, for the check that they differ
  uint32_t bits[kMaxSlots / 32];
};

// Warp w of the plan owns the pages [lo, hi).  Pass 1 copies refs and counts the
// pages that match; pass 2 lists matching pages by rank.
__device__ __forceinline__ void warp_pages(int P, int& lo, int& hi, int warp, int warps) {
  const int per = (int)((((int64_t)P + warps - 1) / warps + 31) / 32 * 32);
  lo = min((int64_t)P, (int64_t)warp * per);
  hi = min((int64_t)P, (int64_t)lo + per);
}
__device__ __forceinline__ void warp_pages(int P, int& lo, int& hi) { warp_pages(P, lo, hi, threadIdx.x >> 5, 32); }
// (By warp `warp` of `warps`.)
__device__ int copy_and_count(const Book& b, bool used, int warp, int warps) {
  int lo, hi;
  warp_pages(b.P, lo, hi, warp, warps);
  const int lane = threadIdx.x & 31;
  int n = 0;
  constexpr int U = 8;  // loads in flight per lane
  for (int p0 = lo; p0 < hi; p0 += 32 * U) {
    int r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * 32 + lane;
      r[u] = p < hi ? b.refs[p] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * 32 + lane;
      if (p < hi) {
        if (b.refs_out != nullptr) b.refs_out[p] = r[u];
        n += used ? r[u] > 0 : r[u] == 0;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}
__device__ __forceinline__ int copy_and_count(const Book& b, bool used) {
  return copy_and_count(b, used, threadIdx.x >> 5, 32);
}
// The lowest `want` free pages into list; false if there are fewer.
__device__ bool list_free(const Book& b, int want, int32_t* list) {
  const int n = copy_and_count(b, false);
  int total;
  int rank = block_scan((threadIdx.x & 31) == 0 ? n : 0, &total);
  rank = __shfl_sync(0xffffffffu, rank, 0);
  if (total < want) return false;
  int lo, hi;
  warp_pages(b.P, lo, hi);
  const int lane = threadIdx.x & 31;
  for (int p0 = lo; p0 < hi && rank < want; p0 += 32) {
    const int p = p0 + lane;
    const bool f = p < hi && b.refs[p] == 0;
    const unsigned m = __ballot_sync(0xffffffffu, f);
    const int r = rank + __popc(m & ((1u << lane) - 1));
    if (f && r < want) list[r] = p;
    rank += __popc(m);
  }
  return true;
}

// Marks the n slots in slot_of; false in `good` if one is out of range or named twice.
__device__ bool mark_slots(const Book& b, const int32_t* slots, int n, SlotSet* set) {
  for (int i = threadIdx.x; i < (b.S + 31) / 32; i += blockDim.x) set->bits[i] = 0;
  for (int i = threadIdx.x; i < b.S; i += blockDim.x) b.slot_of()[i] = -1;
  __syncthreads();
  bool good = true;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = slots[i];
    if ((unsigned)s >= (unsigned)b.S) {
      good = false;
      continue;
    }
    const uint32_t bit = 1u << (s & 31);
    if (atomicOr(&set->bits[s >> 5], bit) & bit) good = false;
    b.slot_of()[s] = i;
  }
  return good;
}

// A length that its table row can hold.
__device__ __forceinline__ bool length_ok(const Book& b, int64_t len) {
  return len >= 0 && len <= (int64_t)b.M * b.page;
}
__device__ __forceinline__ int pages_of(int64_t len, int page) { return (int)((len + page - 1) / page); }

// Ends a plan: records the first error, publishes ok.
__device__ void end_plan(const Book& b, int bad_site, int moves) {
  const int any = __syncthreads_or(bad_site != 0);
  if (bad_site != 0) record_device_error(b.status, SCREE_DEVERR_BAD_INPUT, bad_site);
  if (threadIdx.x == 0) {
    b.plan()->ok = !any;
    b.plan()->moves = any ? 0 : moves;
  }
}
// An earlier error stands: nothing is planned (refs still copied through).
__device__ bool plan_stopped(const Book& b) {
  const bool stop = b.status != nullptr && *reinterpret_cast<volatile int*>(b.status) != 0;
  if (!__syncthreads_or(stop)) return false;
  copy_and_count(b, false);
  if (threadIdx.x == 0) b.plan()->ok = b.plan()->moves = 0;
  return true;
}

// ------------------------------------------------------------------ apply

// Rows of `bytes` bytes as W-byte vectors by one warp.
template <int W>
__device__ __forceinline__ void warp_copy(char* dst, const char* src, int64_t bytes, int lane) {
  using V = typename Vec<W>::T;
  const int64_t n = bytes / W;
  constexpr int U = 4;
  int64_t i = lane;
  for (; i + 32 * (U - 1) < n; i += 32 * U) {
    V r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = reinterpret_cast<const V*>(src)[i + 32 * u];
#pragma unroll
    for (int u = 0; u < U; ++u) reinterpret_cast<V*>(dst)[i + 32 * u] = r[u];
  }
  for (; i < n; i += 32) reinterpret_cast<V*>(dst)[i] = reinterpret_cast<const V*>(src)[i];
}

enum BookOp { kReserve, kFork, kFree, kAccept, kCompact };

// One entry of the new table (and what it does to refs); the thread of column 0
// writes the slot's length.
template <int OP>
__device__ __forceinline__ void book_entry(const Book& b, bool ok, const int32_t* aux, int n, int64_t at) {
  const int s = (int)((unsigned)at / (unsigned)b.M), c = (int)(at - (int64_t)s * b.M);  // S * M < 2^31
  int32_t e = b.table[at];
  int32_t len = b.lengths[s];
  if (ok) {
    if constexpr (OP == kCompact) {
      if (e >= 0 && e < b.P) e = b.list(0)[e];
    } else {
      const int i = b.slot_of()[s];
      if (i >= 0) {
        if constexpr (OP == kReserve) {  // aux = counts
          if (c >= b.first()[i] && c < b.last(n)[i]) {
            e = b.list(n)[b.start(n)[i] + c - b.first()[i]];
            b.refs_out[e] = 1;
          }
          len += aux[i];
        } else if constexpr (OP == kFork) {  // aux = parents
          const int p = aux[i];
          e = -1;
          len = b.lengths[p];
          if (c < b.first()[i]) {
            e = b.table[(int64_t)p * b.M + c];
            if ((unsigned)e < (unsigned)b.P) atomicAdd(&b.refs_out[e], 1);
            else record_device_error(b.status, SCREE_DEVERR_BAD_INPUT, kSitePagedTable);
          } else if (c < b.last(n)[i]) {
            e = b.list(n)[b.start(n)[i]];
            b.refs_out[e] = 1;
          }
        } else if constexpr (OP == kFree) {
          if (c < pages_of(len, b.page)) {
            if ((unsigned)e < (unsigned)b.P) atomicSub(&b.refs_out[e], 1);
            else record_device_error(b.status, SCREE_DEVERR_BAD_INPUT, kSitePagedTable);
          }
          e = -1;
          len = 0;
        } else {  // aux = drafted
          if (c >= b.first()[i] && c < b.last(n)[i]) {
            b.refs_out[e] = 0;  // held by this slot alone, as the plan has checked
            e = -1;
          }
          len += b.start(n)[i] - aux[i];
        }
      }
    }
  }
  b.table_out[at] = e;
  if (c == 0) b.lengths_out[s] = len;
}

// The whole new table by threads [thread, ...) of `threads`.
template <int OP>
__device__ __forceinline__ void apply_table(const Book& b, bool ok, const int32_t* aux, int n, int64_t thread,
                                            int64_t threads) {
  const int64_t all = (int64_t)b.S * b.M;
  for (int64_t at = thread; at < all; at += threads) book_entry<OP>(b, ok, aux, n, at);
}

// The rows that an accepted call moves, by warp `warp` of `warps`.
template <int OP, int W>
__device__ __forceinline__ void apply_moves(const Book& b, const Pools& pl, const int32_t* slots, const int32_t* aux,
                                            const int32_t* path, int depth, int n, int64_t warp, int64_t warps) {
  const int lane = threadIdx.x & 31;
  if constexpr (OP == kFork) {
    // Filled rows of the parent's last page, one head at a time.
    const int64_t tasks = (int64_t)n * pl.L * 2 * pl.H;
    for (int64_t t = warp; t < tasks; t += warps) {
      const int h = (int)(t % pl.H);
      const int64_t r = t / pl.H;
      const int pool = (int)(r & 1), layer = (int)((r >> 1) % pl.L), i = (int)((r >> 1) / pl.L);
      const int full = b.first()[i];
      if (b.last(n)[i] == full) continue;
      const int parent = slots[i];
      const int old = b.table[(int64_t)parent * b.M + full], fresh = b.list(n)[b.start(n)[i]];
      if ((unsigned)old >= (unsigned)b.P) {
        record_device_error(b.status, SCREE_DEVERR_BAD_INPUT, kSitePagedTable);
        continue;
      }
      char* base = (pool ? pl.v : pl.k) + layer * pl.layer_bytes + (int64_t)h * b.page * pl.row_bytes;
      warp_copy<W>(base + fresh * pl.page_bytes, base + old * pl.page_bytes,
                   (b.lengths[parent] % b.page) * pl.row_bytes, lane);
    }
  } else if constexpr (OP == kCompact) {
    // Whole pages, an eighth of one to each warp.
    constexpr int kParts = 8;
    const int moves = b.plan()->moves;
    const int32_t *hole = b.list(0) + b.P, *mover = hole + b.P;
    const int64_t vecs = pl.page_bytes / W, per = (vecs + kParts - 1) / kParts;
    const int64_t tasks = (int64_t)moves * pl.L * 2 * kParts;
    for (int64_t t = warp; t < tasks; t += warps) {
      const int part = (int)(t % kParts);
      const int64_t r = t / kParts;
      const int pool = (int)(r & 1), layer = (int)((r >> 1) % pl.L), i = (int)((r >> 1) / pl.L);
      char* base = (pool ? pl.v : pl.k) + layer * pl.layer_bytes;
      const int64_t lo = min(vecs, part * per), hi = min(vecs, lo + per);
      warp_copy<W>(base + hole[i] * pl.page_bytes + lo * W, base + mover[i] * pl.page_bytes + lo * W,
                   (hi - lo) * W, lane);
    }
  } else if constexpr (OP == kAccept) {
    // Row d of the path moves to row d of the draft.  A task is an entry's rows in
    // one pool of one layer, a run of 32 W-byte columns of them; a lane owns a
    // column and moves it through the whole path: rows only move down (path[d] >=
    // d, ascending), so reading a batch of rows before writing it reads nothing
    // that an earlier batch wrote.
    using V = typename Vec<W>::T;
    const unsigned vpr = (unsigned)(pl.row_bytes / W), cols = pl.H * vpr, runs = (cols + 31) / 32;
    const unsigned pools = (unsigned)pl.L * 2 * runs;
    constexpr int U = 8;
    for (int64_t t = warp; t < (int64_t)n * pools; t += warps) {
      const int i = (int)(t / pools);
      const unsigned r = (unsigned)(t - (int64_t)i * pools), pool = r / runs, col = (r - pool * runs) * 32 + lane;
      const int kept = b.start(n)[i];
      const int s = slots[i];
      const int begin = b.lengths[s] - aux[i];
      const int32_t* row = b.table + (int64_t)s * b.M;
      char* base = (pool & 1 ? pl.v : pl.k) + (pool >> 1) * pl.layer_bytes +
                   (int64_t)(col / vpr) * b.page * pl.row_bytes + (int64_t)(col % vpr) * W;
      // Byte offset of a row of the draft in its layer.
      auto place = [&](int d) {
        const unsigned pos = (unsigned)(begin + d), pg = pos / (unsigned)b.page;
        return row[pg] * pl.page_bytes + (int64_t)(pos - pg * b.page) * pl.row_bytes;
      };
      for (int d0 = 0; d0 < kept; d0 += 32) {
        // 32 steps of the path at a time in the lanes.
        int64_t src = 0, dst = 0;
        if (d0 + lane < kept) {
          src = place(path[(int64_t)i * depth + d0 + lane]);
          dst = place(d0 + lane);
        }
        const int here = min(32, kept - d0);
        for (int e0 = 0; e0 < here; e0 += U) {
          V x[U];
          int64_t from[U], to[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            from[u] = __shfl_sync(0xffffffffu, src, (e0 + u) & 31);
            to[u] = __shfl_sync(0xffffffffu, dst, (e0 + u) & 31);
            if (e0 + u < here && from[u] != to[u] && col < cols) x[u] = *reinterpret_cast<const V*>(base + from[u]);
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (e0 + u < here && from[u] != to[u] && col < cols) *reinterpret_cast<V*>(base + to[u]) = x[u];
        }
      }
    }
  }
}

// Blocks [0, table_blocks) write the table, the others move rows.
template <int OP, int W>
__global__ void __launch_bounds__(kThreads)
    apply_kernel(const Book b, const Pools pl, const int32_t* slots, const int32_t* aux,
                 const int32_t* path, int depth, int n, int table_blocks) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const bool ok = b.plan()->ok != 0;
  if ((int)blockIdx.x < table_blocks) {
    apply_table<OP>(b, ok, aux, n, (int64_t)blockIdx.x * kThreads + threadIdx.x, (int64_t)table_blocks * kThreads);
  } else if (ok) {
    apply_moves<OP, W>(b, pl, slots, aux, path, depth, n,
                       (int64_t)(blockIdx.x - table_blocks) * (kThreads / 32) + (threadIdx.x >> 5),
                       (int64_t)(gridDim.x - table_blocks) * (kThreads / 32));
  }
}

// A small call's apply, by its plan's own CTA (rows in 16-byte vectors).
template <int OP, bool MOVES>
__device__ __forceinline__ void apply_here(const Book& b, const Pools& pl, const int32_t* slots, const int32_t* aux,
                                           const int32_t* path, int depth, int n) {
  __syncthreads();
  const bool ok = b.plan()->ok != 0;
  apply_table<OP>(b, ok, aux, n, threadIdx.x, blockDim.x);
  if (MOVES && ok) apply_moves<OP, 16>(b, pl, slots, aux, path, depth, n, threadIdx.x >> 5, blockDim.x >> 5);
}

// ------------------------------------------------------------------ plans

template <bool HERE>
__global__ void __launch_bounds__(kPlanThreads) plan_reserve_kernel(const Book b, const int32_t* slots,
                                                                    const int32_t* counts, int n) {
  __shared__ SlotSet set;
  begin_plan();
  if (plan_stopped(b)) {
    if (HERE) apply_here<kReserve, false>(b, Pools{}, slots, counts, nullptr, 0, n);
    return;
  }
  int bad = mark_slots(b, slots, n, &set) ? 0 : kSitePagedArgs;
  int64_t want = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0, f = 0;
    if (i < n) {
      const int s = slots[i];
      const int64_t cnt = counts[i];
      if ((unsigned)s < (unsigned)b.S) {
        const int64_t len = b.lengths[s];
        if (cnt < 0 || !length_ok(b, len) || !length_ok(b, len + cnt)) {
          bad = kSitePagedArgs;
        } else {
          f = pages_of(len, b.page);
          need = pages_of(len + cnt, b.page) - f;
        }
      }
    }
    int total;
    const int before = block_scan(need, &total);
    if (i < n) {
      b.first()[i] = f;
      b.last(n)[i] = f + need;
      b.start(n)[i] = (int)min(want + before, (int64_t)b.P);
    }
    want += total;
  }
  const bool fits = list_free(b, (int)min(want, (int64_t)b.P), b.list(n)) && want <= b.P;
  if (!fits && bad == 0) bad = kSitePagedFull;
  end_plan(b, bad, 0);
  if (HERE) apply_here<kReserve, false>(b, Pools{}, slots, counts, nullptr, 0, n);
}

template <bool HERE>
__global__ void __launch_bounds__(kPlanThreads) plan_fork_kernel(const Book b, const Pools pl, const int32_t* parents,
                                                                 const int32_t* children, int n) {
  __shared__ SlotSet set;
  begin_plan();
  if (plan_stopped(b)) {
    if (HERE) apply_here<kFork, true>(b, pl, parents, parents, nullptr, 0, n);
    return;
  }
  int bad = mark_slots(b, children, n, &set) ? 0 : kSitePagedArgs;
  __syncthreads();
  int64_t want = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0, full = 0;
    if (i < n) {
      const int p = parents[i], c = children[i];
      if ((unsigned)p >= (unsigned)b.S || (unsigned)c >= (unsigned)b.S || b.lengths[c] != 0 ||
          (set.bits[p >> 5] >> (p & 31) & 1) || !length_ok(b, b.lengths[p])) {
        bad = kSitePagedArgs;
      } else {
        full = b.lengths[p] / b.page;
        need = b.lengths[p] % b.page != 0;
      }
    }
    int total;
    const int before = block_scan(need, &total);
    if (i < n) {
      b.first()[i] = full;
      b.last(n)[i] = full + need;
      b.start(n)[i] = (int)min(want + before, (int64_t)b.P);
    }
    want += total;
  }
  const bool fits = list_free(b, (int)min(want, (int64_t)b.P), b.list(n)) && want <= b.P;
  if (!fits && bad == 0) bad = kSitePagedFull;
  end_plan(b, bad, 0);
  if (HERE) apply_here<kFork, true>(b, pl, parents, parents, nullptr, 0, n);
}

template <bool HERE>
__global__ void __launch_bounds__(kPlanThreads) plan_free_kernel(const Book b, const int32_t* slots, int n) {
  __shared__ SlotSet set;
  begin_plan();
  if (plan_stopped(b)) {
    if (HERE) apply_here<kFree, false>(b, Pools{}, slots, nullptr, nullptr, 0, n);
    return;
  }
  int bad = mark_slots(b, slots, n, &set) ? 0 : kSitePagedArgs;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = slots[i];
    if ((unsigned)s < (unsigned)b.S && !length_ok(b, b.lengths[s])) bad = kSitePagedArgs;
  }
  copy_and_count(b, false);
  end_plan(b, bad, 0);
  if (HERE) apply_here<kFree, false>(b, Pools{}, slots, nullptr, nullptr, 0, n);
}

// last[i] = pages before, first[i] = pages after, start[i] = rows kept of the draft.
template <bool HERE>
__global__ void __launch_bounds__(kPlanThreads) plan_accept_kernel(const Book b, const Pools pl, const int32_t* slots,
                                                                   const int32_t* drafted,
                                                                   const int32_t* path, int depth, int n) {
  __shared__ SlotSet set;
  begin_plan();
  if (plan_stopped(b)) {
    if (HERE) apply_here<kAccept, true>(b, pl, slots, drafted, path, depth, n);
    return;
  }
  int bad = mark_slots(b, slots, n, &set) ? 0 : kSitePagedArgs;
  // One warp per entry: lanes read the path and the draft's pages side by side.
  // The last eight warps copy refs meanwhile.
  const int lane = threadIdx.x & 31;
  constexpr int kCopyWarps = 8, kCheckWarps = kPlanThreads / 32 - kCopyWarps;
  if (threadIdx.x >> 5 >= kCheckWarps) copy_and_count(b, false, (threadIdx.x >> 5) - kCheckWarps, kCopyWarps);
  for (int i = threadIdx.x >> 5; i < n && threadIdx.x >> 5 < kCheckWarps; i += kCheckWarps) {
    const int s = slots[i];
    if ((unsigned)s >= (unsigned)b.S) continue;  // reported above
    const int64_t len = b.lengths[s], m = drafted[i];
    if (m < 0 || m > len || !length_ok(b, len)) {
      bad = kSitePagedArgs;
      continue;
    }
    int kept = 0, prev = -1;
    for (int d0 = 0; d0 < depth; d0 += 32) {
      const int node = d0 + lane < depth ? path[(int64_t)i * depth + d0 + lane] : -1;
      const unsigned ends = __ballot_sync(0xffffffffu, node < 0);
      const int here = ends ? __ffs(ends) - 1 : 32;  // nodes before the first -1
      int before = __shfl_up_sync(0xffffffffu, node, 1);
      if (lane == 0) before = prev;
      if (lane < here && (node <= before || node >= m)) bad = kSitePagedArgs;
      prev = __shfl_sync(0xffffffffu, node, 31);
      kept += here;
      if (here < 32) break;
    }
    const int64_t begin = len - m;
    const int pages = pages_of(len, b.page);
    for (int c = (int)(begin / b.page) + lane; c < pages; c += 32) {
      const int p = b.table[(int64_t)s * b.M + c];
      if ((unsigned)p >= (unsigned)b.P) bad = kSitePagedTable;
      else if (m > 0 && b.refs[p] != 1) bad = kSitePagedShared;
    }
    if (lane == 0) {
      b.last(n)[i] = pages;
      b.first()[i] = pages_of(begin + kept, b.page);
      b.start(n)[i] = kept;
    }
  }
  end_plan(b, bad, 0);
  if (HERE) apply_here<kAccept, true>(b, pl, slots, drafted, path, depth, n);
}

// list = new id of each page, then the holes and the pages that fill them.
__global__ void __launch_bounds__(kPlanThreads) plan_compact_kernel(const Book b) {
  begin_plan();
  if (plan_stopped(b)) return;
  int32_t *to = b.list(0), *hole = to + b.P, *mover = hole + b.P;
  const int lane = threadIdx.x & 31;
  const int mine = copy_and_count(b, true);
  int used;
  block_scan(lane == 0 ? mine : 0, &used);
  int lo, hi;
  warp_pages(b.P, lo, hi);
  int nh = 0, nm = 0;
  for (int p0 = lo; p0 < hi; p0 += 32) {
    const int p = p0 + lane, r = p < hi ? b.refs[p] : 0;
    nh += __popc(__ballot_sync(0xffffffffu, p < hi && r <= 0 && p < used));
    nm += __popc(__ballot_sync(0xffffffffu, p < hi && r > 0 && p >= used));
  }
  int holes, movers;
  int rh = block_scan(lane == 0 ? nh : 0, &holes);
  int rm = block_scan(lane == 0 ? nm : 0, &movers);
  rh = __shfl_sync(0xffffffffu, rh, 0);
  rm = __shfl_sync(0xffffffffu, rm, 0);
  for (int p0 = lo; p0 < hi; p0 += 32) {
    const int p = p0 + lane, r = p < hi ? b.refs[p] : 0;
    const bool h = p < hi && r <= 0 && p < used, m = p < hi && r > 0 && p >= used;
    const unsigned bh = __ballot_sync(0xffffffffu, h), bm = __ballot_sync(0xffffffffu, m);
    const unsigned lt = (1u << lane) - 1;
    if (p < hi) to[p] = p;
    if (h) hole[rh + __popc(bh & lt)] = p;
    if (m) mover[rm + __popc(bm & lt)] = p;
    rh += __popc(bh);
    rm += __popc(bm);
  }
  __syncthreads();  // also orders the lists for this block's readers
  // As many used pages stand above `used` as free ones below it.
  for (int i = threadIdx.x; i < movers; i += blockDim.x) {
    const int src = mover[i], dst = hole[i];
    to[src] = dst;
    b.refs_out[dst] = b.refs[src];
    b.refs_out[src] = 0;
  }
  end_plan(b, 0, movers);
}

// ------------------------------------------------------------------ write

// Sequence that holds packed row t: the last b with offs[b] <= t, by a 32-way
// search of the whole warp.
__device__ __forceinline__ int64_t warp_find_seq(const void* offs, int is64, int64_t B, int64_t t, int lane) {
  int64_t lo = 0, n = B;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int64_t step = (n + 31) / 32;
    const int64_t at = lo + lane * step;
    const bool le = lane * step < n && load_offset(offs, is64, at) <= t;
    const int k = __popc(__ballot_sync(0xffffffffu, le));  // a prefix: offsets do not decrease
    const int64_t skip = (k > 0 ? k - 1 : 0) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// Up to so many entries each block of a write looks for a slot that is named twice;
// of more, one block does in a launch of its own.  One token an entry, by the blocks /
// by a launch (us; neither: 3.5, 3.9, 6.7, 29): 256 entries 3.8 / 4.9, 1,024 5.0 / 5.6,
// 4,096 13.3 / 9.3, 16,384 107 / 35.
constexpr int64_t kCompareEntries = 1024;

// Records that two entries with tokens name one slot, or that k's and v's offsets (or
// nullptr: the same) differ; by one block, ahead of the write.
__global__ void __launch_bounds__(kPlanThreads)
    check_entries_kernel(const int32_t* slots, const void* offs, const void* v_offs, int is64, int64_t B, int S,
                         int* status) {
  __shared__ SlotSet set;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  for (int i = threadIdx.x; i < kMaxSlots / 32; i += blockDim.x) set.bits[i] = 0;
  __syncthreads();
  bool bad = false;
  if (v_offs != nullptr)
    for (int64_t i = threadIdx.x; i <= B; i += blockDim.x)
      bad |= load_offset(offs, is64, i) != load_offset(v_offs, is64, i);
  constexpr int C = 4;  // loads under way
  for (int64_t i0 = threadIdx.x; i0 < B; i0 += C * kPlanThreads) {
    int s[C];
    bool some[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int64_t i = i0 + c * kPlanThreads;
      s[c] = i < B ? slots[i] : -1;
      some[c] = i < B && load_offset(offs, is64, i + 1) > load_offset(offs, is64, i);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      // (Neighbouring slots in words of their own.)
      const uint32_t bit = 1u << ((unsigned)s[c] / (kMaxSlots / 32) & 31);
      if ((unsigned)s[c] < (unsigned)S && some[c])
        bad |= (atomicOr(&set.bits[s[c] % (kMaxSlots / 32)], bit) & bit) != 0;
    }
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) record_device_error(status, SCREE_DEVERR_BAD_INPUT, kSitePagedArgs);
}

// One warp per token: its K and V rows.  The rows of entry b are the last
// offs[b+1] - offs[b] of its slot.  The first loads of the rows are under way
// while the chain offsets -> slot -> length -> page id finds where they go.
// Entries with tokens that name one slot would write the same rows: none of them
// does.  The block's threads look for such entries side by side, behind the loads of
// the chain.
// 64 entries of 256 tokens of 8 x 128 16-bit elements: 24.6 us, 5.5 TB/s; of 64: 6.8;
// one of six: 2.9, which is the chain.  (Without the look at refs 23.3, 6.7 and 2.9.)
template <int W>
__global__ void __launch_bounds__(kThreads, 4)
    paged_write_kernel(const Pools pl, int layer, const char* k, int64_t k_rb, int64_t k_hb, const char* v,
                       int64_t v_rb, int64_t v_hb, const void* offs, int is64, int64_t B, int64_t T,
                       const int32_t* slots, const int32_t* table, const int32_t* lengths, const int32_t* refs, int S,
                       int M, int P, int page, int* status) {
  using V = typename Vec<W>::T;
  constexpr int kWarps = kThreads / 32;
  __shared__ int sm_slot[kWarps], sm_entry[kWarps];
  __shared__ uint32_t sm_twice;  // of the warps: their slot is another entry's too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const bool stopped = status != nullptr && *reinterpret_cast<volatile int*>(status) != 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  const unsigned vpr = (unsigned)(pl.row_bytes / W), all = t < T ? vpr * (unsigned)pl.H : 0;
  const int first = threadIdx.x < B ? slots[threadIdx.x] : -1;
  constexpr int U = 4;
  V x[2][U];
  auto load = [&](unsigned i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = i0 + 32 * u;
      if (i < all) {
        x[0][u] = *reinterpret_cast<const V*>(k + t * k_rb + (i / vpr) * k_hb + (int64_t)(i % vpr) * W);
        x[1][u] = *reinterpret_cast<const V*>(v + t * v_rb + (i / vpr) * v_hb + (int64_t)(i % vpr) * W);
      }
    }
  };
  load(lane);
  // Where the row goes, or the site of what is wrong.
  int site = 0, s = -1, p = 0;
  int64_t b = 0;
  unsigned at = 0, row = 0;
  if (t < T) {
    b = warp_find_seq(offs, is64, B, t, lane);
    const int64_t lo = load_offset(offs, is64, b), hi = load_offset(offs, is64, b + 1);
    s = slots[b];
    if ((unsigned)s >= (unsigned)S || lo < 0 || t < lo || t >= hi || hi > T) {
      site = kSitePagedArgs;
    } else {
      const int64_t pos = (int64_t)lengths[s] - (hi - t);
      if (pos < 0 || pos >= (int64_t)M * page) {
        site = kSitePagedArgs;
      } else {
        at = (unsigned)pos / (unsigned)page;
        row = (unsigned)pos - at * page;
        p = table[(int64_t)s * M + at];
        if ((unsigned)p >= (unsigned)P) site = kSitePagedTable;
        else if (refs != nullptr && refs[p] > 1) site = kSitePagedShared;
      }
    }
  }
  if (B > 1 && B <= kCompareEntries) {
    if (lane == 0) {
      sm_slot[warp] = s;
      sm_entry[warp] = (int)b;
      if (warp == 0) sm_twice = 0;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < (int)B; i += kThreads) {
      const int named = i < kThreads ? first : __ldg(slots + i);
      uint32_t same = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) same |= named == sm_slot[w] && i != sm_entry[w] ? 1u << w : 0u;
      if (same != 0 && load_offset(offs, is64, i + 1) > load_offset(offs, is64, i)) atomicOr(&sm_twice, same);
    }
    __syncthreads();
    if (site == 0 && (sm_twice >> warp & 1)) site = kSitePagedArgs;
  }
  if (stopped || t >= T) return;
  if (site != 0) {
    if (lane == 0) record_device_error(status, SCREE_DEVERR_BAD_INPUT, site);
    return;
  }
  const int64_t to = layer * pl.layer_bytes + p * pl.page_bytes + (int64_t)row * pl.row_bytes;
  const int64_t dst_hb = (int64_t)page * pl.row_bytes;
  for (unsigned i0 = lane; i0 < all; i0 += 32 * U) {
    if (i0 != (unsigned)lane) load(i0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = i0 + 32 * u;
      if (i < all) {
        const int64_t d = to + (i / vpr) * dst_hb + (int64_t)(i % vpr) * W;
        *reinterpret_cast<V*>(pl.k + d) = x[0][u];
        *reinterpret_cast<V*>(pl.v + d) = x[1][u];
      }
    }
  }
}

// ------------------------------------------------------------------ tree mask

// Bit j of row i: node j is i or an ancestor of i.  One thread per node walks to
// its root; a parent must come before its child, so the walk ends.
__global__ void __launch_bounds__(kThreads)
    tree_mask_kernel(const int32_t* parents, const void* offs, int is64, int64_t B, int64_t T, int words,
                     unsigned long long* mask, int* status) {
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int lane = threadIdx.x & 31;
  // The search is of the whole warp: its lanes look for the warp's first row, then walk on.
  const int64_t t0 = min(t - lane, T - 1);
  int64_t b = warp_find_seq(offs, is64, B, t0, lane);
  if (t >= T) return;
  while (b + 1 < B && load_offset(offs, is64, b + 1) <= t) ++b;
  const int64_t lo = load_offset(offs, is64, b), hi = load_offset(offs, is64, b + 1);
  unsigned long long* row = mask + t * words;
  for (int w = 0; w < words; ++w) row[w] = 0;
  if (lo < 0 || t < lo || t >= hi || hi > T || hi - lo > (int64_t)words * 64) {
    record_device_error(status, SCREE_DEVERR_BAD_INPUT, kSitePagedArgs);
    return;
  }
  int node = (int)(t - lo);
  while (true) {
    row[node >> 6] |= 1ull << (node & 63);
    const int up = parents[lo + node];
    if (up < 0) break;
    if (up >= node) {
      record_device_error(status, SCREE_DEVERR_BAD_INPUT, kSitePagedArgs);
      break;
    }
    node = up;
  }
}

// ------------------------------------------------------------------ host side

int pick_width(int64_t bytes, std::initializer_list<uintptr_t> addrs) {
  int w = 16;
  while (w > 1 && bytes % w != 0) w >>= 1;
  for (uintptr_t a : addrs)
    while (w > 1 && a % w != 0) w >>= 1;
  return w;
}

int check_book(const char* what, const scree_paged_book* k, int64_t n, const void* ws, size_t ws_bytes) {
  SCREE_CHECK_ARG(k != nullptr, "%s: null bookkeeping", what);
  SCREE_CHECK_ARG(k->S >= 1 && k->S <= kMaxSlots && k->M >= 1 && k->P >= 1 && k->page >= 1 &&
                      k->S * k->M < (1ll << 31) && k->P < (1ll << 30) && k->page <= (1 << 20) &&
                      k->M * k->page < (1ll << 31),
                  "%s: bad sizes S=%lld M=%lld P=%lld page=%lld", what, (long long)k->S,
                  (long long)k->M, (long long)k->P, (long long)k->page);
  SCREE_CHECK_ARG(n >= 0 && n <= k->S, "%s: %lld entries for %lld slots", what, (long long)n, (long long)k->S);
  SCREE_CHECK_ARG(k->table && k->lengths && k->refs && k->table_out && k->lengths_out && k->refs_out,
                  "%s: null pointer", what);
  SCREE_CHECK_ARG(k->table != k->table_out && k->lengths != k->lengths_out && k->refs != k->refs_out,
                  "%s: outputs must not be the inputs", what);
  SCREE_CHECK_ARG(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= scree_paged_workspace_size(k->S, k->P),
                  "%s: workspace too small", what);
  return SCREE_OK;
}
Book make_book(const scree_paged_book* k, void* ws) {
  Book b;
  b.table = k->table;
  b.lengths = k->lengths;
  b.refs = k->refs;
  b.table_out = k->table_out;
  b.lengths_out = k->lengths_out;
  b.refs_out = k->refs_out;
  b.S = (int)k->S;
  b.M = (int)k->M;
  b.P = (int)k->P;
  b.page = (int)k->page;
  b.ws = reinterpret_cast<int32_t*>(ws);
  b.status = device_status_ptr();
  return b;
}
int make_pools(const char* what, const scree_paged_pools* p, int64_t P, int64_t page, Pools* out) {
  SCREE_CHECK_ARG(p != nullptr && p->k && p->v, "%s: null pools", what);
  SCREE_CHECK_ARG(p->L >= 1 && p->L < (1 << 20) && p->H >= 1 && p->H < (1 << 16) && p->row_bytes >= 1 &&
                      p->row_bytes <= (1 << 20),
                  "%s: bad pool sizes L=%lld H=%lld row_bytes=%lld", what, (long long)p->L,
                  (long long)p->H, (long long)p->row_bytes);
  out->k = reinterpret_cast<char*>(p->k);
  out->v = reinterpret_cast<char*>(p->v);
  out->L = (int)p->L;
  out->H = (int)p->H;
  out->row_bytes = p->row_bytes;
  out->page_bytes = p->H * page * p->row_bytes;
  out->layer_bytes = P * out->page_bytes;
  return SCREE_OK;
}

template <int OP, int W>
int launch_apply_w(const Book& b, const Pools& pl, const int32_t* slots, const int32_t* aux,
                   const int32_t* path, int depth, int n, int table_blocks, int move_blocks, cudaStream_t s) {
  SCREE_CUDA_TRY(launch_dependent(apply_kernel<OP, W>, dim3((unsigned)(table_blocks + move_blocks)),
                                  dim3(kThreads), 0, s, 1, b, pl, slots, aux, path, depth, n, table_blocks));
  count_launch();
  return SCREE_OK;
}
// A call is applied by its plan's CTA if that takes it about as long as a second
// launch, which costs the host 3 us more.  Reserve, by the plan's CTA / by a
// launch of its own: 4.4 / 4.4 us at 256 table entries, 5.9 / 5.8 at 2,048, 7.0 /
// 6.6 at 4,096, 15.1 / 9.4 at 16,384.  Fork and accept with one moving task per
// warp (32): 8.4 / 7.2 and 7.5 / 5.8 us; with four: 16.2 / 7.5 and 17.9 / 6.0.
bool apply_by_plan(const Book& b, int64_t units, int w) {
  return (int64_t)b.S * b.M <= kHereEntries && units <= kHereWarps && w == 16;
}

// `units`: warps of row-moving work (an upper bound where only the device knows).
template <int OP>
int launch_apply(const Book& b, const Pools& pl, const int32_t* slots, const int32_t* aux,
                 const int32_t* path, int depth, int n, int64_t units, cudaStream_t s) {
  const int table_blocks = (int)std::min<int64_t>(((int64_t)b.S * b.M + kThreads - 1) / kThreads, 2 * num_sms());
  const int move_blocks = (int)std::min<int64_t>((units + kThreads / 32 - 1) / (kThreads / 32), 8 * num_sms());
  const int w = units == 0 ? 16
                           : pick_width(pl.row_bytes, {(uintptr_t)pl.k, (uintptr_t)pl.v});
  switch (w) {
    case 16: return launch_apply_w<OP, 16>(b, pl, slots, aux, path, depth, n, table_blocks, move_blocks, s);
    case 8: return launch_apply_w<OP, 8>(b, pl, slots, aux, path, depth, n, table_blocks, move_blocks, s);
    case 4: return launch_apply_w<OP, 4>(b, pl, slots, aux, path, depth, n, table_blocks, move_blocks, s);
    case 2: return launch_apply_w<OP, 2>(b, pl, slots, aux, path, depth, n, table_blocks, move_blocks, s);
    default: return launch_apply_w<OP, 1>(b, pl, slots, aux, path, depth, n, table_blocks, move_blocks, s);
  }
}

}  // namespace
}  // namespace scree

using namespace scree;

extern "C" size_t scree_paged_workspace_size(int64_t S, int64_t P) {
  if (S < 1 || P < 1) return 0;
  return 4 * (size_t)(kPlanWords + 4 * S + 3 * P);
}

extern "C" int scree_paged_reserve(const scree_paged_book* book, const int32_t* slots, const int32_t* counts,
                                   int64_t n, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_book("paged_reserve", book, n, workspace, workspace_bytes);
  if (rc != SCREE_OK) return rc;
  SCREE_CHECK_ARG(n == 0 || (slots && counts), "paged_reserve: null pointer");
  SCREE_BIND_DEVICE(stream, book->table);
  const Book b = make_book(book, workspace);
  cudaStream_t s = (cudaStream_t)stream;
  const bool here = apply_by_plan(b, 0, 16);
  SCREE_CUDA_TRY(launch_dependent(here ? plan_reserve_kernel<true> : plan_reserve_kernel<false>, dim3(1),
                                  dim3(kPlanThreads), 0, s, 1, b, slots, counts, (int)n));
  count_launch();
  if (here) return SCREE_OK;
  return launch_apply<kReserve>(b, Pools{}, slots, counts, nullptr, 0, (int)n, 0, s);
}

extern "C" int scree_paged_accept(const scree_paged_book* book, const scree_paged_pools* pools,
                                  const int32_t* slots, const int32_t* drafted, const int32_t* path,
                                  int64_t depth, int64_t n, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  int rc = check_book("paged_accept", book, n, workspace, workspace_bytes);
  if (rc != SCREE_OK) return rc;
  SCREE_CHECK_ARG(depth >= 0 && depth < (1ll << 31), "paged_accept: bad depth %lld", (long long)depth);
  SCREE_CHECK_ARG(n == 0 || (slots && drafted && (path || depth == 0)), "paged_accept: null pointer");
  Pools pl;
  if ((rc = make_pools("paged_accept", pools, book->P, book->page, &pl)) != SCREE_OK) return rc;
  SCREE_BIND_DEVICE(stream, book->table);
  const Book b = make_book(book, workspace);
  cudaStream_t s = (cudaStream_t)stream;
  const int w = pick_width(pl.row_bytes, {(uintptr_t)pl.k, (uintptr_t)pl.v});
  const int64_t units = depth == 0 ? 0 : n * pl.L * 2 * ((pl.H * (pl.row_bytes / w) + 31) / 32);
  const bool here = apply_by_plan(b, units, w);
  SCREE_CUDA_TRY(launch_dependent(here ? plan_accept_kernel<true> : plan_accept_kernel<false>, dim3(1),
                                  dim3(kPlanThreads), 0, s, 1, b, pl, slots, drafted, path, (int)depth, (int)n));
  count_launch();
  if (here) return SCREE_OK;
  return launch_apply<kAccept>(b, pl, slots, drafted, path, (int)depth, (int)n, units, s);
}

extern "C" int scree_paged_fork(const scree_paged_book* book, const scree_paged_pools* pools,
                                const int32_t* parents, const int32_t* children, int64_t n, void* workspace,
                                size_t workspace_bytes, void* stream) {
  int rc = check_book("paged_fork", book, n, workspace, workspace_bytes);
  if (rc != SCREE_OK) return rc;
  SCREE_CHECK_ARG(n == 0 || (parents && children), "paged_fork: null pointer");
  Pools pl;
  if ((rc = make_pools("paged_fork", pools, book->P, book->page, &pl)) != SCREE_OK) return rc;
  SCREE_BIND_DEVICE(stream, book->table);
  const Book b = make_book(book, workspace);
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t units = n * pl.L * 2 * pl.H;
  const bool here = apply_by_plan(b, units, pick_width(pl.row_bytes, {(uintptr_t)pl.k, (uintptr_t)pl.v}));
  SCREE_CUDA_TRY(launch_dependent(here ? plan_fork_kernel<true> : plan_fork_kernel<false>, dim3(1),
                                  dim3(kPlanThreads), 0, s, 1, b, pl, parents, children, (int)n));
  count_launch();
  if (here) return SCREE_OK;
  return launch_apply<kFork>(b, pl, parents, parents, nullptr, 0, (int)n, units, s);
}

extern "C" int scree_paged_free(const scree_paged_book* book, const int32_t* slots, int64_t n, void* workspace,
                                size_t workspace_bytes, void* stream) {
  int rc = check_book("paged_free", book, n, workspace, workspace_bytes);
  if (rc != SCREE_OK) return rc;
  SCREE_CHECK_ARG(n == 0 || slots, "paged_free: null pointer");
  SCREE_BIND_DEVICE(stream, book->table);
  const Book b = make_book(book, workspace);
  cudaStream_t s = (cudaStream_t)stream;
  const bool here = apply_by_plan(b, 0, 16);
  SCREE_CUDA_TRY(launch_dependent(here ? plan_free_kernel<true> : plan_free_kernel<false>, dim3(1),
                                  dim3(kPlanThreads), 0, s, 1, b, slots, (int)n));
  count_launch();
  if (here) return SCREE_OK;
  return launch_apply<kFree>(b, Pools{}, slots, nullptr, nullptr, 0, (int)n, 0, s);
}

extern "C" int scree_paged_compact(const scree_paged_book* book, const scree_paged_pools* pools,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_book("paged_compact", book, 0, workspace, workspace_bytes);
  if (rc != SCREE_OK) return rc;
  Pools pl;
  if ((rc = make_pools("paged_compact", pools, book->P, book->page, &pl)) != SCREE_OK) return rc;
  SCREE_BIND_DEVICE(stream, book->table);
  const Book b = make_book(book, workspace);
  cudaStream_t s = (cudaStream_t)stream;
  SCREE_CUDA_TRY(launch_dependent(plan_compact_kernel, dim3(1), dim3(kPlanThreads), 0, s, 1, b));
  count_launch();
  // At most half of the pages can move.
  return launch_apply<kCompact>(b, pl, nullptr, nullptr, nullptr, 0, 0, (book->P / 2 + 1) * pl.L * 2 * 8, s);
}

extern "C" int scree_paged_write_ex(const scree_paged_pools* pools, const int32_t* table, const int32_t* lengths,
                                    const int32_t* refs, int64_t S, int64_t M, int64_t P, int64_t page,
                                    int64_t layer, const int32_t* slots, const void* k, int64_t k_row_bytes,
                                    int64_t k_head_bytes, const void* v, int64_t v_row_bytes,
                                    int64_t v_head_bytes, const void* offsets, const void* v_offsets,
                                    int offs_is_i64, int64_t B, int64_t T, void* stream) {
  SCREE_CHECK_ARG(S >= 1 && S <= kMaxSlots && M >= 1 && P >= 1 && P < (1ll << 30) && page >= 1 &&
                      M * page < (1ll << 31),
                  "paged_write: bad sizes S=%lld M=%lld P=%lld page=%lld", (long long)S, (long long)M,
                  (long long)P, (long long)page);
  SCREE_CHECK_ARG(B >= (T > 0) && T >= 0 && T < (1ll << 31), "paged_write: bad sizes B=%lld T=%lld", (long long)B,
                  (long long)T);
  Pools pl;
  int rc = make_pools("paged_write", pools, P, page, &pl);
  if (rc != SCREE_OK) return rc;
  SCREE_CHECK_ARG(layer >= 0 && layer < pl.L, "paged_write: layer %lld of %d", (long long)layer, pl.L);
  if (T == 0) return SCREE_OK;
  SCREE_CHECK_ARG(table && lengths && slots && k && v && offsets, "paged_write: null pointer");
  SCREE_BIND_DEVICE(stream, k);
  const int w = pick_width(pl.row_bytes, {(uintptr_t)pl.k, (uintptr_t)pl.v, (uintptr_t)k, (uintptr_t)v,
                                          (uintptr_t)k_row_bytes, (uintptr_t)k_head_bytes,
                                          (uintptr_t)v_row_bytes, (uintptr_t)v_head_bytes});
  const unsigned grid = (unsigned)((T + kThreads / 32 - 1) / (kThreads / 32));
  cudaStream_t s = (cudaStream_t)stream;
  if (B > kCompareEntries || v_offsets != nullptr) {
    SCREE_CUDA_TRY(launch_dependent(check_entries_kernel, dim3(1), dim3(kPlanThreads), 0, s, 1, slots, offsets,
                                    v_offsets, offs_is_i64, B, (int)S, device_status_ptr()));
    count_launch();
  }
#define SCREE_WRITE(WW)                                                                                   \
  SCREE_CUDA_TRY(launch_dependent(                                                                        \
      paged_write_kernel<WW>, dim3(grid), dim3(kThreads), 0, s, 1, pl, (int)layer, (const char*)k,        \
      k_row_bytes, k_head_bytes, (const char*)v, v_row_bytes, v_head_bytes, offsets, offs_is_i64, B, T,   \
      slots, table, lengths, refs, (int)S, (int)M, (int)P, (int)page, device_status_ptr()))
  switch (w) {
    case 16: SCREE_WRITE(16); break;
    case 8: SCREE_WRITE(8); break;
    case 4: SCREE_WRITE(4); break;
    case 2: SCREE_WRITE(2); break;
    default: SCREE_WRITE(1); break;
  }
#undef SCREE_WRITE
  count_launch();
  return SCREE_OK;
}

extern "C" int scree_paged_write(const scree_paged_pools* pools, const int32_t* table, const int32_t* lengths,
                                 int64_t S, int64_t M, int64_t P, int64_t page, int64_t layer,
                                 const int32_t* slots, const void* k, int64_t k_row_bytes,
                                 int64_t k_head_bytes, const void* v, int64_t v_row_bytes,
                                 int64_t v_head_bytes, const void* offsets, int offs_is_i64, int64_t B,
                                 int64_t T, void* stream) {
  return scree_paged_write_ex(pools, table, lengths, nullptr, S, M, P, page, layer, slots, k, k_row_bytes,
                              k_head_bytes, v, v_row_bytes, v_head_bytes, offsets, nullptr, offs_is_i64, B, T, stream);
}

extern "C" int scree_tree_mask(const int32_t* parents, const void* offsets, int offs_is_i64, int64_t B,
                               int64_t T, int64_t words, uint64_t* mask, void* stream) {
  SCREE_CHECK_ARG(B >= (T > 0) && T >= 0 && T < (1ll << 31) && words >= 1 && words < (1 << 20),
                  "tree_mask: bad sizes B=%lld T=%lld words=%lld", (long long)B, (long long)T, (long long)words);
  if (T == 0) return SCREE_OK;
  SCREE_CHECK_ARG(parents && offsets && mask, "tree_mask: null pointer");
  SCREE_BIND_DEVICE(stream, parents);
  tree_mask_kernel<<<(unsigned)((T + kThreads - 1) / kThreads), kThreads, 0, (cudaStream_t)stream>>>(
      parents, offsets, offs_is_i64, B, T, (int)words, reinterpret_cast<unsigned long long*>(mask),
      device_status_ptr());
  SCREE_LAUNCH_CHECK();
  return SCREE_OK;
}
