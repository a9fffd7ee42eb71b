// attn_paged.cuh — what the two kernels of attention over a paged cache share:
// the call's parameters, the cut of the work into equal runs, and their entry.
#pragma once
#include "attn_common.cuh"

namespace scree {

constexpr int kPagedKeys = 16;      // pages hold a multiple of this many keys
constexpr int kPagedMaxSeqs = 4096; // sequences of a call (their prefix sits in shared memory)
constexpr int kSitePagedAttn = 70, kSitePagedAttnPage = 71, kSitePagedAttnWait = 72;

// What the join needs of worker c: the segment that its first piece continues
// (on = 0: none; written for every worker of the grid).
struct PagedDesc {
  int32_t on;
  int32_t w0, np;    // the segment's first worker, its pieces
  int32_t row0;      // packed row (token) of the tile's first query
  int32_t h, i0, n;  // K/V head; index of the tile's first row (or token), new tokens of the sequence
};

struct PagedParams {
  const char* q;
  int64_t q_rs, q_hs;  // bytes
  const void* offs;
  int is64;
  const int32_t *slots, *table, *lengths;
  const unsigned long long* mask;
  int words;
  int B, S, M, P, page;
  int H, Hkv, G;
  int64_t T;
  int64_t layer_row;  // first row of the layer in the pools' row view
  const void* v;      // the V pool
  float sl2;          // scale log2 e
  char* o;
  int64_t o_rs, o_hs;
  float* lse;
  int* status;
  PagedDesc* desc;
  float2* part_ml;
  float* part_o;
};

// Division of non-negative numbers, in 32 bits where they fit (a 64-bit division
// takes several hundred cycles, and a worker's start needs half a dozen).
__device__ __forceinline__ int64_t udiv(int64_t a, int64_t b) {
  if (((uint64_t)(a | b) >> 32) == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
  return a / b;
}
// Units [start(w), start(w + 1)) are worker w's: U / N each, one more for the first
// U % N; the worker that holds unit u.
struct PagedCut {
  int64_t q, r;
  __device__ __forceinline__ PagedCut(int64_t U, int64_t N) {
    q = udiv(U, N);
    r = U - q * N;
  }
  __device__ __forceinline__ int64_t start(int64_t w) const { return w * q + min(w, r); }
  __device__ __forceinline__ int64_t of(int64_t u) const {
    return u < r * (q + 1) ? udiv(u, q + 1) : r + udiv(u - r * (q + 1), q);
  }
};

// Fills pre[b] = units of the sequences before b (units(n, len) of each), by the
// whole block of 32 * WARPS threads; false for every thread if the call is to be
// left alone (an error stands, or the input is invalid, which is recorded).
template <int WARPS, typename Units>
__device__ __forceinline__ bool paged_prefix(const PagedParams& p, int64_t* pre, Units units_of) {
  __shared__ int64_t warp_sum[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool bad = p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != 0;
  const bool stopped = bad;
  int64_t carry = 0;
  for (int base = 0; base < p.B; base += WARPS * 32) {
    const int b = base + threadIdx.x;
    int64_t units = 0;
    if (b < p.B) {
      const int s = p.slots[b];
      const int64_t lo = load_offset(p.offs, p.is64, b), hi = load_offset(p.offs, p.is64, b + 1);
      const int64_t n = hi - lo;
      if ((unsigned)s >= (unsigned)p.S || lo < 0 || n < 0 || hi > p.T || (b == 0 && lo != 0) ||
          (b == p.B - 1 && hi != p.T)) {
        bad = true;
      } else {
        const int64_t len = p.lengths[s];
        if (len < n || len > (int64_t)p.M * p.page || (p.mask != nullptr && n > (int64_t)p.words * 64)) bad = true;
        else units = units_of(n, len);
      }
    }
    int64_t x = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int64_t before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    if (b < p.B) pre[b + 1] = before + x;
    carry = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) pre[0] = 0;
  if (__syncthreads_or(bad)) {
    if (bad && !stopped) record_device_error(p.status, SCREE_DEVERR_BAD_INPUT, kSitePagedAttn);
    return false;
  }
  return true;
}
// Sequence of unit u: the last b with pre[b] <= u (those without units hold none).
__device__ __forceinline__ int paged_find(const int64_t* pre, int B, int64_t u) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Wait that gives up after its own limit only: an error that other work has
// recorded (a page id out of range is read as page 0 and recorded) stops nothing
// half way, so no CTA leaves copies in flight behind.
__device__ __forceinline__ bool paged_wait(const PagedParams& p, uint64_t* bar, uint32_t parity, volatile int* abort) {
  const bool ok = mbar_wait_impl(bar, parity & 1, abort, nullptr, kSitePagedAttnWait);
  if (!ok) record_device_error(p.status, SCREE_DEVERR_WAIT_TIMEOUT, kSitePagedAttnWait);
  return ok;
}

// Exit path: waits, as long at most, for a copy that may still be under way, so no
// CTA ends with a copy to its shared memory in flight.
__device__ __forceinline__ void paged_drain(uint64_t* bar, uint32_t parity) {
  volatile int quiet = 0;
  mbar_wait_impl(bar, parity & 1, &quiet, nullptr, kSitePagedAttnWait);
}

// Page that holds key group g (16 keys) of a slot; a bad id is recorded and read as page 0.
__device__ __forceinline__ int paged_page(const PagedParams& p, int slot, int g) {
  const int page = p.table[(int64_t)slot * p.M + (unsigned)g * kPagedKeys / (unsigned)p.page];
  if ((unsigned)page < (unsigned)p.P) return page;
  record_device_error(p.status, SCREE_DEVERR_BAD_INPUT, kSitePagedAttnPage);
  return 0;
}

// Visibility of keys [k0, k0 + N), N <= 64, for query i of a sequence (row of the
// packed queries): all keys before c0 = len - n, of the n new ones those of the
// mask row (or j <= i), none from len on.
template <int N>
__device__ __forceinline__ unsigned long long paged_visible(const PagedParams& p, int64_t row, int i, int k0,
                                                            int c0, int len) {
  constexpr unsigned long long kAll = N == 64 ? ~0ull : (1ull << (N & 63)) - 1;
  unsigned long long v = kAll;
  const int t0 = k0 - c0;  // index of key k0 among the new ones
  if (t0 > -N) {
    if (p.mask == nullptr) {
      const int last = i - t0;  // last visible key of the group
      v = last >= N - 1 ? kAll : last < 0 ? 0ull : (2ull << last) - 1;
    } else {
      const unsigned long long* m = p.mask + row * p.words;
      if (t0 < 0) {
        v = (m[0] << -t0) | ((1ull << -t0) - 1);
      } else {
        const int w = t0 >> 6, o = t0 & 63;
        v = w < p.words ? m[w] >> o : 0ull;
        if (o > 64 - N && w + 1 < p.words) v |= m[w + 1] << (64 - o);
      }
      v &= kAll;
    }
  }
  const int left = len - k0;
  return left >= N ? v : left <= 0 ? 0ull : v & ((1ull << left) - 1);
}

// 2^x, x <= 0, as the weight of what has been summed so far.  It is never 0: an
// infinity that a row has taken in stays one (0 * inf = NaN), whatever comes behind it
// and wherever the run is cut.  2^-149 of a finite sum is below its rounding.
__device__ __forceinline__ float ex2_weight(float x) { return fmaxf(ex2_approx(x), __uint_as_float(1u)); }

// All ones in the exponent: infinity or NaN, of either half of a word.
template <typename T> __device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
  return ((w & E) == E ? 0xFFFFu : 0u) | (((w >> 16) & E) == E ? 0xFFFF0000u : 0u);
}

// Tensor map over the pools' rows {D, rows} (16-bit), boxes of box_rows rows.
int make_pool_map(CUtensorMap* map, const void* base, int64_t rows, int D, int box_rows, bool bf16);

// attn_paged_tc.cu: row tiles of 2 x 128 on the tensor cores' own instructions.
size_t attn_paged_tc_workspace(int D);
int attn_paged_tc(const PagedParams& p, const void* k, const void* v, int64_t pool_rows, int D, bool bf16,
                  void* workspace, cudaStream_t s);

}  // namespace scree
