// logprobs.cu — log probabilities of given tokens, entropies and top
// alternatives of (N, V) logits, and the gradient of the logits.
//
//   s1 = sum e^(x - m),  s2 = sum e^(x - m) (x - m),  m = max x
//   log p = (x - m) - log s1,  H = -sum p log p = log s1 - s2 / s1
//   dx_v = g_logp [v = target] + sum_j g_top_j [v = id_j]
//          - p_v (g_logp + sum_j g_top_j) - g_H p_v (log p_v + H)
//
// Forward: each logit is read from HBM once, and that bounds it.  Persistent CTAs
// stream rows in chunks of 16 KB: one warp copies them into a ring with bulk
// copies, running on into the CTA's next row while eight read one, so 3 CTAs keep
// up to 144 KB per SM in flight.  The eight never meet at a barrier: each thread
// keeps its own maximum, s1 and s2 (rescaled only when a chunk raises the maximum),
// and a tenth warp joins them, two rows behind at most.  Of few rows each is cut
// into segments for the CTAs of a cluster, which hand their results to its first
// CTA through shared memory.  6,144 x 128,000 in 16 bits: 270 us (5.8 TB/s), with
// four alternatives 274; 4,099 x 65,539 with eight: 107; 16,384 x 16,384: 111, with
// four 182 (the tenth warp's pace: 5 us a row); 1 x 131,072 with twenty: 8.4.  (With
// the eight warps joining and merging at barriers between rows: 276, 332, 152, 178,
// 318 and 11.6.)
//
// Alternatives: a thread notes the maximum of its elements of each chunk (a pair:
// thread, chunk), so the streaming loop pays one store a chunk.  After kWin chunks or
// at the row's end the tenth warp takes the top-th largest of 64 thread maxima as a
// bound; the few pairs that reach it can hold one of the best elements, and those
// are read again, from L2, and ranked with the list so far, while the eight go on.
// That is once per row of up to 131,000 16-bit logits.  (Pushing elements above a
// running bound as they stream past cost 4,000 cycles each time a warp met one,
// twice the time of a chunk.)  Equal values are taken in the order of their
// indices: keys hold both, and a pair whose lowest index is behind the list's last
// is passed over, so floods of equal values end early.
//
// Numerics: sums in fp32, exponents in units of log2 (one FMA and one ex2 per
// element; the product x log2e is not rounded before m is subtracted; see shift).
#include <algorithm>
#include "common.cuh"
#include "sm100.cuh"

namespace scree {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;     // one alternative per lane when lists are merged
constexpr int kU = 4;           // vectors of a thread per chunk
constexpr int kCtasPerSm = 3;
constexpr int kStages = 3;      // ring of chunks
constexpr int kChunkBytes = kThreads * kU * 16;
constexpr int kWinRow = 32 + 4;  // a thread's maxima over a window (a word more: its rows start in different banks)
constexpr int kWinBytes = kWinRow * kThreads;
constexpr int kRingSmem = kStages * kChunkBytes + 2 * kWinBytes + 128;
constexpr int kWarps = kThreads / 32;      // that work; one more copies, one finishes rows
constexpr int kMaxSegs = 8;     // a portable cluster
constexpr int kSiteRing = 51;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kSiteTarget = 50, kSiteAlternative = 52;

template <typename T> struct Lv {  // elements of one 16-byte vector
  static constexpr int N = 16 / sizeof(T);
};
template <typename T> __device__ __forceinline__ uint32_t neg_inf_word();
template <> __device__ __forceinline__ uint32_t neg_inf_word<__nv_bfloat16>() { return 0xFF80FF80u; }
template <> __device__ __forceinline__ uint32_t neg_inf_word<__half>() { return 0xFC00FC00u; }
template <> __device__ __forceinline__ uint32_t neg_inf_word<float>() { return 0xFF800000u; }

template <typename T> __device__ __forceinline__ void unpack_vec(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Largest element of a vector, NaN if it holds one (16-bit types two at a time).
template <typename T> __device__ __forceinline__ float vec_max(const uint4& v) {
  if constexpr (std::is_same<T, float>::value) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                   max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    auto b = [](uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); };
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(b(v.x), b(v.y)), __hmax2_nan(b(v.z), b(v.w)));
    return max_nan(__low2float(m), __high2float(m));
  } else {
    auto h = [](uint32_t u) { return *reinterpret_cast<__half2*>(&u); };
    const __half2 m = __hmax2_nan(__hmax2_nan(h(v.x), h(v.y)), __hmax2_nan(h(v.z), h(v.w)));
    return max_nan(__low2float(m), __high2float(m));
  }
}

// x log2e - m log2e in one FMA rounds m log2e first.  All terms are off by the same
// 2^shift(m), so sums are kept as they are and the shift is taken out where maxima meet
// and at the row's end: log p depends on differences alone.  From 1024 on (a row, or all
// that a thread has seen of it, masked with a large number) x - m is taken first.
constexpr float kFar = 1024.f;
__device__ __forceinline__ float shift(float m) {
  return fabsf(m) >= kFar ? 0.f : fmaf(m, kLog2e, -__fmul_rn(m, kLog2e));
}
// -inf must not meet its own weight, 0 * -inf = NaN: elements near the
// type's lowest value are raised to `low`, two at a time for the 16-bit types.  With |m| < kFar their weight
// is 0 either way and (x - m) log2e is finite.  NaN stays.
template <typename T> struct Far;
template <> struct Far<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t two(uint32_t w) {
    const uint32_t low = 0xFE96FE96u;  // -9.97e37
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&low));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint4 raise(const uint4& v) { return make_uint4(two(v.x), two(v.y), two(v.z), two(v.w)); }
};
template <> struct Far<__half> {
  static __device__ __forceinline__ uint32_t two(uint32_t w) {
    const uint32_t low = 0xFBFFFBFFu;  // -65504
    const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&w), *reinterpret_cast<const __half2*>(&low));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint4 raise(const uint4& v) { return make_uint4(two(v.x), two(v.y), two(v.z), two(v.w)); }
};
template <> struct Far<float> {
  static __device__ __forceinline__ uint32_t one(uint32_t w) { return __float_as_uint(max_nan(__uint_as_float(w), -1e38f)); }
  static __device__ __forceinline__ uint4 raise(const uint4& v) { return make_uint4(one(v.x), one(v.y), one(v.z), one(v.w)); }
};

// Order of the alternatives: larger value first (NaN above all, -0 = +0), then
// lower index.  Keys of valid elements are never 0.
__device__ __forceinline__ uint32_t order_bits(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
  if (o == 0xFFFFFFFFu) return __uint_as_float(0x7FFFFFFFu);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ unsigned long long order_key(float x, uint32_t idx) {
  return ((unsigned long long)order_bits(x) << 32) | (0xFFFFFFFFu - idx);
}

// Running statistics: m, s1, and s2 in units of log2, both sums' terms 2^shift(m) too
// large; s1 = 0 when empty.
struct Stat {
  float m, s1, s2;
};
// s1 and s2 moved from maximum m to the maximum `to` >= m.
__device__ __forceinline__ void stat_move(Stat& s, float to) {
  float d = __fmul_rn(s.m, kLog2e) - __fmul_rn(to, kLog2e);  // both near: what the terms were taken at
  if (!(fmaxf(fabsf(s.m), fabsf(to)) < kFar))
    d = (s.m - (to == -INFINITY ? 0.f : to)) * kLog2e + (shift(to) - shift(s.m));
  const float w = ex2_approx(d);
  // An empty side has d = -inf: its weight is 0 and its (bounded) shift is not used.
  s.s2 = w * (s.s2 + fmaxf(d, -1000.f) * s.s1);
  s.s1 *= w;
  s.m = to;
}
__device__ __forceinline__ float max_nan_warp(float v) {
  float d;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}
// Joined over the first W lanes (in lane 0; the others empty, or W = 32: in all).
template <int W = 32> __device__ __forceinline__ Stat stat_warp(Stat s) {
  const float m = max_nan_warp(s.m);
  stat_move(s, m);
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    s.s1 += __shfl_xor_sync(0xffffffffu, s.s1, o);
    s.s2 += __shfl_xor_sync(0xffffffffu, s.s2, o);
  }
  return s;
}

// Bitonic networks over the lanes of a warp, descending.
template <typename K> __device__ __forceinline__ K lane_merge(K v, int lane) {
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const K o = __shfl_xor_sync(0xffffffffu, v, j);
    v = ((lane & j) == 0) == (v > o) ? v : o;
  }
  return v;
}
// The 32 largest of two descending lists of 32.
template <typename K> __device__ __forceinline__ K lane_join(K a, K b, int lane) {
  const K r = __shfl_sync(0xffffffffu, b, 31 - lane);
  return lane_merge(a > r ? a : r, lane);
}

// 32 keys in descending order.
template <typename K> __device__ __forceinline__ K lane_sort(K v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const K o = __shfl_xor_sync(0xffffffffu, v, j);
      v = (((lane & j) == 0) == ((lane & k) == 0)) == (v > o) ? v : o;
    }
  return v;
}

struct FwdArgs {
  const void* x;
  int64_t row_stride, N;
  int V;
  int chunks, segs;  // chunks of a row, segments that they are dealt to (= CTAs of a cluster)
  int seg_bits;      // segs = 1 << seg_bits
  const void* targets;
  int t64;
  int top;
  float *logp, *entropy;
  float2* norm;  // maximum and log of the sum: log p = (x - norm.x) - norm.y
  float* top_logp;
  int64_t* top_ids;
  int* status;
};

// The row's outputs from its joined statistics (s2: lane 0's); `key` is the lane's alternative, t
// the target and xt its logit (lane 0).
template <typename T>
__device__ __forceinline__ void finish_row(const FwdArgs& a, int64_t n, const Stat& s, unsigned long long key,
                                           int64_t t, float xt, int lane) {
  // A row with nothing left (every logit -inf): logp = -inf, H = 0.
  const bool empty = s.m == -INFINITY;
  const float l2 = log2f(s.s1), ls = (l2 - shift(s.m)) * kLn2;
  if (lane == 0) {
    if (a.norm != nullptr) a.norm[n] = make_float2(s.m, empty ? -INFINITY : ls);
    a.entropy[n] = empty ? 0.f : (l2 - __fdividef(s.s2, s.s1)) * kLn2;  // (both hold the shift)
    float lp = 0.f;  // negative target: no token given
    if (t >= (int64_t)a.V) {
      record_device_error(a.status, SCREE_DEVERR_BAD_INPUT, kSiteTarget);
      lp = __uint_as_float(0x7FFFFFFFu);
    } else if (t >= 0) {
      lp = empty ? -INFINITY : (xt - s.m) - ls;
    }
    a.logp[n] = lp;
  }
  if (lane < a.top) {
    a.top_ids[n * a.top + lane] = (int64_t)(0xFFFFFFFFu - (uint32_t)key);
    const float x = order_value((uint32_t)(key >> 32));
    a.top_logp[n * a.top + lane] = empty ? -INFINITY : (x - s.m) - ls;
  }
}

// Wait on the ring.  It records its own time-out but does not stop for an error
// that another row has recorded (a target out of range spoils no other row).
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  const bool ok = mbar_wait_impl(bar, parity, abort, nullptr, kSiteRing);
  if (!ok) record_device_error(status, SCREE_DEVERR_WAIT_TIMEOUT, kSiteRing);
  return ok;
}

// Vector at element e0 of a row (e0 a multiple of the vector size from a 16-byte
// boundary); elements outside [0, V) read as -inf.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* row, int e0, int V) {
  constexpr int VE = Lv<T>::N;
  if (e0 >= 0 && e0 + VE <= V) return *reinterpret_cast<const uint4*>(row + e0);
  uint32_t w[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) w[u] = neg_inf_word<T>();
  if (e0 + VE > 0 && e0 < V) {
    T* el = reinterpret_cast<T*>(w);
#pragma unroll
    for (int u = 0; u < VE; ++u)
      if (e0 + u >= 0 && e0 + u < V) el[u] = row[e0 + u];
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A vector at element e0 of a row, its elements outside [0, V) replaced by -inf.
template <typename T> __device__ __forceinline__ uint4 keep_row(const uint4& v, int e0, int V) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t m;
    if constexpr (sizeof(T) == 4) m = (unsigned)(e0 + j) < (unsigned)V ? 0xFFFFFFFFu : 0u;
    else m = ((unsigned)(e0 + 2 * j) < (unsigned)V ? 0xFFFFu : 0u) | ((unsigned)(e0 + 2 * j + 1) < (unsigned)V ? 0xFFFF0000u : 0u);
    r[j] = (w[j] & m) | (neg_inf_word<T>() & ~m);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename T> constexpr int kWin = 32 / (int)sizeof(T);  // chunks of a window

// A bound as a value of type T, and which of a word's elements reach it, which are
// beyond it (NaN always, and everything if it is NaN): bit 0, and bit 16 of 16-bit
// types.
template <typename T> struct Bound;
template <> struct Bound<float> {
  float v;
  __device__ __forceinline__ explicit Bound(float f) : v(f) {}
  __device__ __forceinline__ uint32_t reach(uint32_t w) const { return __uint_as_float(w) < v ? 0u : 1u; }
  __device__ __forceinline__ uint32_t beyond(uint32_t w) const { return __uint_as_float(w) <= v ? 0u : 1u; }
};
template <> struct Bound<__nv_bfloat16> {
  __nv_bfloat162 v;
  __device__ __forceinline__ explicit Bound(float f) : v(__bfloat162bfloat162(__float2bfloat16_rd(f))) {}
  __device__ __forceinline__ uint32_t reach(uint32_t w) const {
    return ~__hlt2_mask(*reinterpret_cast<__nv_bfloat162*>(&w), v) & 0x00010001u;
  }
  __device__ __forceinline__ uint32_t beyond(uint32_t w) const {
    return ~__hle2_mask(*reinterpret_cast<__nv_bfloat162*>(&w), v) & 0x00010001u;
  }
};
template <> struct Bound<__half> {
  __half2 v;
  __device__ __forceinline__ explicit Bound(float f) : v(__half2half2(__float2half_rd(f))) {}
  __device__ __forceinline__ uint32_t reach(uint32_t w) const {
    return ~__hlt2_mask(*reinterpret_cast<__half2*>(&w), v) & 0x00010001u;
  }
  __device__ __forceinline__ uint32_t beyond(uint32_t w) const {
    return ~__hle2_mask(*reinterpret_cast<__half2*>(&w), v) & 0x00010001u;
  }
};
// Bit b of the words' reach(), word w shifted by w: which element of them it is.
template <typename T> __device__ __forceinline__ int reach_element(int b) {
  return sizeof(T) == 4 ? b : (b & 15) * 2 + (b >> 4);
}

// Scratch of the merging warp.
constexpr int kManyKeys = 12;  // elements of a pair that are sorted into the list at once
constexpr int kCand = 96;      // elements that wait for their ranks
struct MergeScratch {
  unsigned long long cand[kCand + 32];  // (and the list, when they are ranked)
  unsigned long long sorted[32];
  int queue[64];                        // pairs to look at: their first elements
  uint32_t queue_max[64];               // and order_bits of their maxima
  uint16_t threads[kThreads];           // those whose maximum reaches the bound
};

// Merges the window of `nch` chunks from chunk c0 on into the list (32 keys in the
// lanes, descending; the first `top` count).  wm: the window's maxima, kWinRow
// bytes a thread; tm: the threads' maxima over the window.  By one warp, once a row:
// what it costs is the fetching of its instructions and its chains of dependent
// ones, so it is loops of few instructions, and lanes that each take a pair.
template <typename T>
__device__ __forceinline__ unsigned long long merge_window(unsigned long long best, int top, const T* row, int mis,
                                                           int V, const uint8_t* wm, const float* tm, int c0, int nch,
                                                           MergeScratch& sc, int lane) {
  constexpr int VE = Lv<T>::N, CV = kThreads * kU, E = kU * VE, G = kThreads / 32;
  const uint32_t lt = (1u << lane) - 1;
  const int base0 = c0 * CV * VE - mis;  // first element of the window's first thread
  // A bound from below: the top-th largest of 64 maxima over four threads each.
  float m[G];  // (-inf of threads without elements)
#pragma unroll
  for (int g = 0; g < G; ++g) m[g] = tm[g * 32 + lane];
  uint32_t tau;
  {
    const uint32_t a = order_bits(max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3])));
    const uint32_t b = order_bits(max_nan(max_nan(m[4], m[5]), max_nan(m[6], m[7])));
    tau = __shfl_sync(0xffffffffu, lane_join(lane_sort(a, lane), lane_sort(b, lane), lane), top - 1);
  }
  unsigned long long kth = __shfl_sync(0xffffffffu, best, top - 1);
  tau = max(tau, (uint32_t)(kth >> 32));
  const float tau_f = order_value(tau);
  const Bound<T> bound(tau_f);
  int flagged = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const bool in = !(m[g] < tau_f);
    const uint32_t b = __ballot_sync(0xffffffffu, in);
    if (in) sc.threads[flagged + __popc(b & lt)] = (uint16_t)(g * 32 + lane);
    flagged += __popc(b);
  }
  __syncwarp();
  int queued = 0, waiting = 0;
  // The waiting elements enter the list.  Keys differ, so a key's place is the number
  // of larger ones.
  auto rank = [&]() {
    const int had = __popc(__ballot_sync(0xffffffffu, best != 0));
    if (lane < had) sc.cand[waiting + lane] = best;
    sc.sorted[lane] = 0;
    __syncwarp();
    const int n = waiting + had;
#pragma unroll 1
    for (int i = lane; i - lane < n; i += 32) {
      const unsigned long long key = i < n ? sc.cand[i] : 0;
      int above = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) above += sc.cand[j] > key;
      if (i < n && above < 32) sc.sorted[above] = key;
    }
    __syncwarp();
    best = sc.sorted[lane];
    kth = __shfl_sync(0xffffffffu, best, top - 1);
    waiting = 0;
  };
  // The queued pairs' elements that reach the bound and are above the list's last; a
  // lane reads a pair.
  auto drain = [&]() {
    __syncwarp();
#pragma unroll 1
    for (int at = 0; at < queued; at += 32) {
      const bool in = at + lane < queued;
      const int e0 = in ? sc.queue[at + lane] : 0;
      const unsigned long long most = in ? (unsigned long long)sc.queue_max[at + lane] << 32 | (0xFFFFFFFFu - max(e0, 0)) : 0;
      uint32_t pass = 0;
      if (most > kth) {
        uint4 v[kU];
#pragma unroll
        for (int i = 0; i < kU; ++i) v[i] = load_vec<T>(row, e0 + i * kThreads * VE, V);
#pragma unroll
        for (int i = 0; i < kU; ++i)
          pass |= bound.reach(v[i].x) << (4 * i) | bound.reach(v[i].y) << (4 * i + 1) | bound.reach(v[i].z) << (4 * i + 2) |
                  bound.reach(v[i].w) << (4 * i + 3);
      }
      // Pairs with many such elements by the whole warp.
      uint32_t left = 0xFFFFFFFFu;  // lanes not looked at yet
      while (true) {
        const uint32_t many = __ballot_sync(0xffffffffu, __popc(pass) >= kManyKeys && most > kth) & left;
        if (many == 0) break;
        const int src = __ffs(many) - 1;
        left = ~((2u << src) - 1);
        const int e = __shfl_sync(0xffffffffu, e0, src) + lane / VE * kThreads * VE + lane % VE;
        unsigned long long key = lane < E && e >= 0 && e < V ? order_key(Cvt<T>::to_f(row[e]), (uint32_t)e) : 0;
        if (key <= kth) key = 0;
        best = lane_join(best, lane_sort(key, lane), lane);
        kth = __shfl_sync(0xffffffffu, best, top - 1);
      }
      if (__popc(pass) >= kManyKeys) pass = 0;
#pragma unroll 1
      while (__any_sync(0xffffffffu, pass != 0)) {
        const int x = reach_element<T>(__ffs(pass) - 1), e = e0 + x / VE * kThreads * VE + x % VE;
        unsigned long long key = 0;
        if (pass != 0 && e >= 0 && e < V) key = order_key(Cvt<T>::to_f(row[e]), (uint32_t)e);
        pass &= pass - 1;
        const uint32_t b = __ballot_sync(0xffffffffu, key > kth);
        if (key > kth) sc.cand[waiting + __popc(b & lt)] = key;
        waiting += __popc(b);
        if (waiting > kCand - 32) rank();
      }
    }
    __syncwarp();
    queued = 0;
  };
  // A pair can matter if its maximum, at its lowest index, is above the list's last.
  // Of 32 threads at a time: of equal values the first ones come early.
#pragma unroll 1
  for (int f0 = 0; f0 < flagged; f0 += 32) {
    const int th = sc.threads[min(f0 + lane, flagged - 1)], e0 = base0 + th * VE;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(wm + th * kWinRow);
    // Behind the list's last an equal value does not count.
    const Bound<T> last(order_value((uint32_t)(kth >> 32)));
    const bool behind = kth != 0 && e0 > (int)(0xFFFFFFFFu - (uint32_t)kth);
    uint32_t pass = 0;
#pragma unroll
    for (int i = 0; i < kWinRow / 4 - 1; ++i) pass |= (behind ? last.beyond(w[i]) : bound.reach(w[i])) << i;
    // Chunks in which the thread has elements.
    const int have = f0 + lane < flagged && e0 < V ? min(nch, (V - e0 + CV * VE - 1) / (CV * VE)) : 0;
    pass &= sizeof(T) == 4 ? (1u << have) - 1 : ((1u << ((have + 1) >> 1)) - 1) | ((1u << (have >> 1)) - 1) << 16;
#pragma unroll 1
    while (__any_sync(0xffffffffu, pass != 0)) {
      bool in = pass != 0;
      const int q = in ? reach_element<T>(__ffs(pass) - 1) : 0, e = e0 + q * CV * VE;
      const uint32_t o = order_bits(Cvt<T>::to_f(reinterpret_cast<const T*>(w)[q]));
      in = in && ((unsigned long long)o << 32 | (0xFFFFFFFFu - max(e, 0))) > kth;
      pass &= pass - 1;
      const uint32_t b = __ballot_sync(0xffffffffu, in);
      if (in) {
        sc.queue[queued + __popc(b & lt)] = e;
        sc.queue_max[queued + __popc(b & lt)] = o;
      }
      queued += __popc(b);
      if (queued >= 32) drain();
    }
  }
  if (queued > 0) drain();
  if (waiting > 0) rank();
  return best;
}

// What a row's other segments hand to its first CTA.
struct SegOut {
  Stat stat[kMaxSegs];
  unsigned long long keys[kMaxSegs][kMaxTop];
};
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kThreads + 64, kCtasPerSm) logprobs_kernel(const FwdArgs a) {
  constexpr int VE = Lv<T>::N, CV = kThreads * kU;  // elements of a vector, vectors of a chunk
  extern __shared__ __align__(16) uint8_t ring[];
  uint8_t* wm = ring + kStages * kChunkBytes;  // two windows' maxima
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * kChunkBytes + 2 * kWinBytes);
  uint64_t* empty = full + kStages;
  uint64_t* win_full = empty + kStages;  // [2] a window has been read: its maxima, and the row's sums behind its last
  uint64_t* win_empty = win_full + 2;    // [2] they have been taken
  volatile int* abort_flag = reinterpret_cast<volatile int*>(win_empty + 2);
  __shared__ Stat sm_stat[2][kWarps];
  __shared__ float tm[2][kThreads];  // the threads' maxima over a window
  __shared__ MergeScratch scratch;
  __shared__ SegOut so;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&win_full[i], kWarps);
      mbar_init(&win_empty[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (a.segs > 1) cluster_sync();  // the first CTA is there to be written to
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  // Item = segment of a row; with several segments a CTA has one item, and the
  // segment is its rank in the cluster.
  const int64_t items = a.N * a.segs;
  // Vectors start at 16-byte boundaries: a row begins `mis` elements into its first
  // one.  A row's vectors go through the ring with what its neighbours have in the
  // first and the last; only where that would leave the tensor the copying warp
  // fetches their elements one by one.
  auto row_of = [&](int64_t n) { return reinterpret_cast<const T*>(a.x) + n * a.row_stride; };
  auto mis_of = [](const T* row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); };
  auto seg_begin = [&](int seg) { return (int)(((int64_t)a.chunks * seg) >> a.seg_bits); };
  // (A row's alignment may leave it one chunk less; a segment has one at least.)
  auto seg_end = [&](int seg, int mis) {
    const int own = (a.V + mis + VE * CV - 1) / (VE * CV);
    return max(seg_begin(seg) + 1, min(seg_begin(seg + 1), own));
  };

  if (warp == kWarps) {
    // ---------------------------------------------------------------- copies
    int k = 0;  // chunks issued
    bool ok = true;
    for (int64_t item = blockIdx.x; lane == 0 && ok && item < items; item += gridDim.x) {
      const T* row = row_of(item >> a.seg_bits);
      const int seg = (int)item & (a.segs - 1), mis = mis_of(row), v_end = (a.V + mis + VE - 1) / VE;
      const int v_lo = row - mis < row_of(0) ? 1 : 0;
      const int v_hi = row - mis + (int64_t)v_end * VE > row_of(a.N - 1) + a.V ? (a.V + mis) / VE : v_end;
      const int c1 = seg_end(seg, mis);
      for (int c = seg_begin(seg); c < c1; ++c, ++k) {
        const int st = k % kStages;
        if (k >= kStages &&
            !(ok = ring_wait(&empty[st], ((k / kStages) - 1) & 1, abort_flag, a.status)))
          break;
        const int lo = max(c * CV, v_lo), hi = min((c + 1) * CV, v_hi);
        auto fetch = [&](int v) {
          T* to = reinterpret_cast<T*>(ring + st * kChunkBytes) + (v - c * CV) * VE;
          for (int e = max(v * VE - mis, 0); e < min((v + 1) * VE - mis, a.V); ++e) to[e - (v * VE - mis)] = row[e];
          fence_proxy_async_smem();  // the place's next copy
        };
        if (c == 0 && v_lo > 0) fetch(0);
        if (v_hi < v_end && v_hi >= max(c * CV, v_lo) && v_hi < (c + 1) * CV) fetch(v_hi);
        if (lo < hi) {
          mbar_expect_tx(&full[st], (uint32_t)(hi - lo) * 16);
          bulk_load_1d(ring + st * kChunkBytes + (lo - c * CV) * 16, row + (int64_t)lo * VE - mis,
                       (uint32_t)(hi - lo) * 16, &full[st]);
        } else {
          mbar_arrive(&full[st]);
        }
      }
    }
    if (lane == 0 && !ok) {  // give copies in flight time to land before the CTA ends
      volatile int quiet = 0;
      for (int i = max(0, k - kStages); i < k; ++i)
        mbar_wait_impl(&full[i % kStages], (i / kStages) & 1, &quiet, nullptr, kSiteRing);
    }
    __syncwarp();
    if (a.segs > 1) cluster_sync();
    return;
  }

  if (warp == kWarps + 1) {
    // ---------------------------------------------------------------- alternatives, results
    // A wait that gives up has set the status word; the work runs on (its results
    // do not count) so that all warps come to their ends.
    auto target_of = [&](int64_t item) {
      const int64_t n = item >> a.seg_bits;
      return item >= items ? -1
             : a.t64       ? reinterpret_cast<const int64_t*>(a.targets)[n]
                           : (int64_t)reinterpret_cast<const int32_t*>(a.targets)[n];
    };
    auto logit_of = [&](int64_t item, int64_t t) {
      return t >= 0 && t < a.V ? row_of(item >> a.seg_bits)[t] : T();
    };
    int w = 0;  // windows taken
    int64_t t0 = target_of(blockIdx.x), t1 = target_of(blockIdx.x + (int64_t)gridDim.x);
    T x0 = logit_of(blockIdx.x, t0);
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
      const int64_t n = item >> a.seg_bits;
      const int seg = (int)item & (a.segs - 1);
      const T* row = row_of(n);
      const int mis = mis_of(row), c1 = seg_end(seg, mis);
      // The targets and their logits are loaded rows ahead.
      const int64_t t = t0;
      const T xt = x0;
      t0 = t1;
      x0 = logit_of(item + gridDim.x, t0);
      t1 = target_of(item + 2 * (int64_t)gridDim.x);
      unsigned long long best = 0;
      for (int c = seg_begin(seg);; ++w) {
        const int buf = w & 1, nch = a.top > 0 ? min(kWin<T>, c1 - c) : c1 - c;
        ring_wait(&win_full[buf], (w >> 1) & 1, abort_flag, a.status);
        if (a.top > 0)
          best = merge_window<T>(best, a.top, row, mis, a.V, wm + buf * kWinBytes, tm[buf], c, nch, scratch, lane);
        c += nch;
        Stat s = lane < kWarps ? sm_stat[buf][lane] : Stat{-INFINITY, 0.f, 0.f};  // (read in vain but behind the last)
        __syncwarp();
        if (lane == 0) mbar_arrive(&win_empty[buf]);
        if (c < c1) continue;
        ++w;
        s = stat_warp<kWarps>(s);
        if (a.segs > 1) {
          if (seg > 0) {
            const uint32_t at = smem_peer(smem_u32(&so.stat[seg]), 0);
            if (lane == 0) {
              st_cluster(at, s.m);
              st_cluster(at + 4, s.s1);
              st_cluster(at + 8, s.s2);
            }
            if (a.top > 0) st_cluster(smem_peer(smem_u32(&so.keys[seg][lane]), 0), best);
          }
          __syncwarp();
          cluster_sync();
          if (seg > 0) break;
          const Stat o = lane > 0 && lane < a.segs ? so.stat[lane] : Stat{-INFINITY, 0.f, 0.f};
          s = stat_warp<kMaxSegs>(lane == 0 ? s : o);
          if (a.top > 0)
            for (int j = 1; j < a.segs; ++j) best = lane_join(best, so.keys[j][lane], lane);
        }
        s.s1 = __shfl_sync(0xffffffffu, s.s1, 0);
        finish_row<T>(a, n, s, best, t, Cvt<T>::to_f(xt), lane);
        break;
      }
    }
    return;
  }

  const int tid = threadIdx.x;
  int k = 0, w = 0;  // chunks, windows taken
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t n = item >> a.seg_bits;
    const int seg = (int)item & (a.segs - 1);
    const T* row = row_of(n);
    const int mis = mis_of(row);
    const int c0 = seg_begin(seg), c1 = seg_end(seg, mis);
    const int v_end = (a.V + mis + VE - 1) / VE;
    Stat st{-INFINITY, 0.f, 0.f};
    for (int c = c0; c < c1; ++w) {
      const int buf = w & 1, end = a.top > 0 ? min(c1, c + kWin<T>) : c1;
      if (w >= 2) ring_wait(&win_empty[buf], ((w >> 1) - 1) & 1, abort_flag, a.status);
      T* out = reinterpret_cast<T*>(wm + buf * kWinBytes + tid * kWinRow);
      float top_max = -INFINITY;  // this thread's maximum over the window
#pragma unroll 1
      for (; c < end; ++c, ++k) {
        const int slot = k % kStages;
        ring_wait(&full[slot], (k / kStages) & 1, abort_flag, a.status);
        const uint4* src = reinterpret_cast<const uint4*>(ring + slot * kChunkBytes) + tid;
        float cm = -INFINITY;
        if (c * CV + (tid & ~31) < v_end) {
          auto vec = [&](int i) {
            const int e = (c * CV + i * kThreads + tid) * VE - mis, e0 = e - lane * VE;  // of the thread, of the warp
            if (e0 >= 0 && e0 + 32 * VE <= a.V) return src[i * kThreads];
            if (e0 >= a.V)
              return make_uint4(neg_inf_word<T>(), neg_inf_word<T>(), neg_inf_word<T>(), neg_inf_word<T>());
            return keep_row<T>(src[i * kThreads], e, a.V);
          };
          uint4 d[kU];
          if (c * CV * VE >= mis && (c + 1) * CV * VE <= a.V + mis) {
#pragma unroll
            for (int i = 0; i < kU; ++i) d[i] = src[i * kThreads];
          } else {
#pragma unroll
            for (int i = 0; i < kU; ++i) d[i] = vec(i);
          }
          cm = vec_max<T>(d[0]);
#pragma unroll
          for (int i = 1; i < kU; ++i) cm = max_nan(cm, vec_max<T>(d[i]));
          if (!(cm <= st.m)) stat_move(st, cm);
          if (!(fabsf(st.m) >= kFar)) {
            const uint64_t l2 = f2_pack(kLog2e, kLog2e), nm = f2_pack(-__fmul_rn(st.m, kLog2e), -__fmul_rn(st.m, kLog2e));
            uint64_t s1[2] = {0, 0}, s2[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < kU; ++i) {
              float f[VE];
              unpack_vec<T>(Far<T>::raise(d[i]), f);
#pragma unroll
              for (int u = 0; u < VE; u += 2) {
                const uint64_t t = f2_fma(f2_pack(f[u], f[u + 1]), l2, nm);
                float t0, t1;
                f2_unpack(t, t0, t1);
                const uint64_t e = f2_pack(ex2_approx(t0), ex2_approx(t1));
                s1[(u >> 1) & 1] = f2_add(s1[(u >> 1) & 1], e);
                s2[(u >> 1) & 1] = f2_fma(e, t, s2[(u >> 1) & 1]);
              }
            }
            float x, y;
            f2_unpack(f2_add(s1[0], s1[1]), x, y);
            st.s1 += x + y;
            f2_unpack(f2_add(s2[0], s2[1]), x, y);
            st.s2 += x + y;
          } else if (st.m != -INFINITY) {  // (nothing but -inf so far, or no element in the chunk)
            // A far maximum (-inf differs from the lowest value here), or an infinity.
#pragma unroll 1
            for (int i = 0; i < kU; ++i) {
              float f[VE];
              unpack_vec<T>(vec(i), f);
#pragma unroll
              for (int u = 0; u < VE; ++u) {
                const float t = (f[u] - st.m) * kLog2e, e = ex2_approx(t);
                st.s1 += e;
                st.s2 = fmaf(e, fmaxf(t, -1000.f), st.s2);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[slot]);
        if (a.top == 0) continue;
        *out++ = Cvt<T>::from_f(cm);  // exact: an element's value
        top_max = max_nan(top_max, cm);
      }
      if (a.top > 0) tm[buf][tid] = top_max;
      if (c == c1) {
        st = stat_warp(st);
        if (lane == 0) sm_stat[buf][warp] = st;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&win_full[buf]);
    }
  }
  if (a.segs > 1) cluster_sync();
}

struct BwdArgs {
  const void* x;
  int64_t row_stride, N;
  int V;
  int slices;
  const void* targets;
  int t64;
  int top;
  const float2* norm;
  const float* entropy;
  const int64_t* top_ids;
  const float *g_logp, *g_entropy, *g_top;  // each may be null
  void* dx;                                 // (N, V) contiguous
  int* status;
};

// The 16 bytes of a and b (the 16 behind a) from byte `bytes` < 16 on.
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int bytes) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (bytes & 8) {
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
  }
  if (bytes & 4) {
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
  }
  const int bits = (bytes & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// dx = -p (gs + gH (H + log p)), then the given token and the alternatives.
// HBM-bound: one read and one write of each logit; 6,144 x 128,000 in 16 bits: 527 us,
// 6.0 TB/s (16 vectors a thread: 700, 4: 549; plain loads: 542).  Where a row begins
// at another place of a 16-byte block than dx's does (rows of a padded vocabulary),
// 16-bit types are stored in dx's vectors, each put together from two of the row's:
// 8,192 x 50,257 of 50,304 453 us (element by element 978; without padding 324); fp32
// element by element: 4,096 rows 289 (in vectors 329; without padding 258).
template <typename T, int NV>
__global__ void __launch_bounds__(kThreads) logprobs_bwd_kernel(const BwdArgs a) {
  constexpr int VE = Lv<T>::N;
  __shared__ float sm_gs;
  const int64_t n = blockIdx.x / (unsigned)a.slices;
  const int slice = blockIdx.x % (unsigned)a.slices;
  const T* row = reinterpret_cast<const T*>(a.x) + n * a.row_stride;
  T* out = reinterpret_cast<T*>(a.dx) + n * (int64_t)a.V;
  constexpr bool kByRow = sizeof(T) == 4;  // vectors of the row, not of dx
  const int at = (int)(((uintptr_t)row & 15) / sizeof(T));
  const int mis = kByRow ? at : (int)(((uintptr_t)out & 15) / sizeof(T));
  const int k = (at - mis) & (VE - 1);  // where dx's vectors begin in the row's
  const bool same = !kByRow || (((uintptr_t)row ^ (uintptr_t)out) & 15) == 0;
  const int v0 = slice * kThreads * NV;  // first vector of the slice
  uint4 d[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (v0 + i * kThreads + (int)threadIdx.x) * VE - mis - k;
    d[i] = e >= 0 && e + VE <= a.V ? __ldcs(reinterpret_cast<const uint4*>(row + e)) : load_vec<T>(row, e, a.V);
  }
  if (!kByRow && k != 0) {  // the rest of a vector is in the next lane's
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint4 b;
      b.x = __shfl_down_sync(0xffffffffu, d[i].x, 1);
      b.y = __shfl_down_sync(0xffffffffu, d[i].y, 1);
      b.z = __shfl_down_sync(0xffffffffu, d[i].z, 1);
      b.w = __shfl_down_sync(0xffffffffu, d[i].w, 1);
      if (lane == 31) b = load_vec<T>(row, (v0 + i * kThreads + (int)threadIdx.x + 1) * VE - mis - k, a.V);
      d[i] = shifted(d[i], b, k * (int)sizeof(T));
    }
  }
  // The given token and the alternatives as one list of (index, weight): entry 0
  // is the target, entry 1 + j alternative j; index -1 has no weight.
  auto entry = [&](int j, int64_t& idx) -> float {
    if (j == 0) {
      idx = a.t64 ? reinterpret_cast<const int64_t*>(a.targets)[n]
                  : (int64_t)reinterpret_cast<const int32_t*>(a.targets)[n];
      if (idx < 0 || idx >= a.V || a.g_logp == nullptr) idx = -1;
      return idx < 0 ? 0.f : a.g_logp[n];
    }
    idx = a.top_ids[n * a.top + j - 1];
    return a.g_top[n * a.top + j - 1];
  };
  const int entries = 1 + (a.g_top != nullptr ? a.top : 0);
  if (threadIdx.x < 32) {
    float g = 0.f;
    int64_t idx;
    for (int j = threadIdx.x; j < entries; j += 32) g += entry(j, idx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) g += __shfl_xor_sync(0xffffffffu, g, o);
    if (threadIdx.x == 0) sm_gs = g;
  }
  __syncthreads();
  const float2 nm = a.norm[n];
  const float gh = a.g_entropy != nullptr ? a.g_entropy[n] : 0.f;
  const bool empty = nm.x == -INFINITY;  // nothing left in the row: no gradient
  // log2 p = x log2e - l2, l2 = (m + log s1) log2e rounded once: what that leaves out, rest,
  // is the row's, and so goes into the row's factors.  Far maxima: (x - m) log2e - s2.
  const bool far = fabsf(nm.x) >= kFar;
  const float m2 = __fmul_rn(nm.x, kLog2e), s2 = __fmul_rn(nm.y, kLog2e), l2 = __fadd_rn(m2, s2);
  float rest = fmaf(nm.y, kLog2e, -s2);
  if (!far) {
    const float part = __fsub_rn(l2, m2);
    rest += fmaf(nm.x, kLog2e, -m2) + (__fsub_rn(m2, __fsub_rn(l2, part)) + __fsub_rn(s2, part));
  }
  const float y = -rest * kLn2, c = fmaf(y, fmaf(0.5f, y, 1.f), 1.f);  // c = 2^-rest, |rest| < 2^-12
  const float base = c * fmaf(gh, a.entropy[n] + y, sm_gs), ghc = c * gh;
  auto grad = [&](float x) {
    const float d2 = far ? fmaf(x - nm.x, kLog2e, -s2) : fmaf(x, kLog2e, -l2);  // log2 p + rest
    // The bound only matters at p = 0, where it keeps 0 * inf out.
    return -ex2_approx(d2) * fmaf(ghc, fmaxf(d2, -1000.f) * kLn2, base);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e0 = (v0 + i * kThreads + (int)threadIdx.x) * VE - mis;
    if (e0 + VE <= 0 || e0 >= a.V) continue;
    float f[VE];
    unpack_vec<T>(d[i], f);
#pragma unroll
    for (int u = 0; u < VE; ++u) f[u] = empty ? 0.f : grad(f[u]);
    __align__(16) T o[VE];
    cvt_from_f<T, VE>(f, o);
    if (same && e0 >= 0 && e0 + VE <= a.V) {
      __stcs(reinterpret_cast<uint4*>(out + e0), *reinterpret_cast<const uint4*>(o));
    } else {
#pragma unroll
      for (int u = 0; u < VE; ++u)
        if (e0 + u >= 0 && e0 + u < a.V) out[e0 + u] = o[u];
    }
  }
  // The listed elements of this slice, written again with their weights (after
  // the barrier, so over the plain value).  Entries with one index write one value.
  __syncthreads();
  if (threadIdx.x < entries && !empty) {
    int64_t idx;
    entry(threadIdx.x, idx);
    const int lo = v0 * VE - mis;
    if (threadIdx.x > 0 && (idx < 0 || idx >= a.V)) {  // an id that is none: nothing to write
      record_device_error(a.status, SCREE_DEVERR_BAD_INPUT, kSiteAlternative);
    } else if (idx >= 0 && idx >= lo && idx < lo + kThreads * NV * VE) {
      float g = 0.f;
      for (int j = 0; j < entries; ++j) {
        int64_t other;
        const float w = entry(j, other);
        if (other == idx) g += w;
      }
      out[idx] = Cvt<T>::from_f(g + grad(Cvt<T>::to_f(row[idx])));
    }
  }
}

// Vectors of a row (which may begin inside its first one).
int64_t row_vecs(int64_t V, int dtype) {
  const int64_t ve = 16 / (int64_t)dtype_size(dtype);
  return (V + ve - 1 + ve - 1) / ve;
}
int64_t row_chunks(int64_t V, int dtype) { return (row_vecs(V, dtype) + kThreads * kU - 1) / (kThreads * kU); }
// Rows are cut while the segments' CTAs still have an SM each.  Measured (us; bf16,
// eight alternatives; 1 / 2 / 4 / 8 segments): 131,072 logits, 1 row 14.2 / 10.6 / 8.6
// / 8.0, 64 rows 14.3 / 11.5 / 11.4 / 16.2, 128 rows 14.7 / 15.5 / 19.2 / 23.9, 444
// rows 27 / 33 / 49 / 78; 32,000 logits, 1 row 7.9 / 7.4 / 7.2, 128 rows 8.3 / 9.2 /
// 14.0, 1,300 rows 24 / 49 / 88.
int row_segs(int64_t N, int64_t V, int dtype) {
  int segs = 1;
  while (segs < kMaxSegs && 2 * N * segs <= num_sms() && 2 * segs <= row_chunks(V, dtype)) segs *= 2;
  return segs;
}
constexpr int kNV = 8;  // vectors of a thread, backward
int64_t bwd_slices(int64_t V, int dtype) { return (row_vecs(V, dtype) + kThreads * kNV - 1) / (kThreads * kNV); }

int check_sizes(const char* what, int64_t N, int64_t V, int64_t row_stride, int top, int dtype) {
  SCREE_CHECK_ARG(dtype == SCREE_F16 || dtype == SCREE_BF16 || dtype == SCREE_F32,
                  "%s: fp16, bf16 or fp32 only", what);
  SCREE_CHECK_ARG(N >= 0 && V >= 1 && V < (1ll << 30), "%s: bad sizes N=%lld V=%lld", what,
                  (long long)N, (long long)V);
  SCREE_CHECK_ARG(row_stride >= V || N <= 1, "%s: rows overlap (row stride %lld, V=%lld)", what,
                  (long long)row_stride, (long long)V);
  SCREE_CHECK_ARG(top >= 0 && top <= kMaxTop && top <= V,
                  "%s: top must be between 0 and %d and at most V (got %d)", what, kMaxTop, top);
  SCREE_CHECK_ARG(N * row_chunks(V, dtype) < (1ll << 31), "%s: N=%lld too large", what,
                  (long long)N);
  return SCREE_OK;
}

template <typename T> int launch_fwd(const FwdArgs& a, cudaStream_t s) {
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63]) {
    SCREE_CUDA_TRY(cudaFuncSetAttribute(logprobs_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
    attr_set[dev & 63] = true;
  }
  const int64_t grid = a.segs > 1 ? a.N * a.segs : std::min<int64_t>(a.N, (int64_t)kCtasPerSm * num_sms());
  SCREE_CUDA_TRY(launch_dependent(logprobs_kernel<T>, dim3((unsigned)grid), dim3(kThreads + 64), kRingSmem, s, a.segs, a));
  count_launch();
  return SCREE_OK;
}
template <typename T> int launch_bwd(const BwdArgs& a, cudaStream_t s) {
  logprobs_bwd_kernel<T, kNV><<<(unsigned)(a.N * a.slices), kThreads, 0, s>>>(a);
  SCREE_LAUNCH_CHECK();
  return SCREE_OK;
}

}  // namespace
}  // namespace scree

using namespace scree;

extern "C" int scree_token_logprobs_fwd(const void* logits, int64_t row_stride, const void* targets,
                                        int targets_is_i64, int64_t N, int64_t V, int top,
                                        int dtype, float* logp, float* entropy, float* norm,
                                        float* top_logp, int64_t* top_ids, void* stream) {
  int rc = check_sizes("token_logprobs", N, V, row_stride, top, dtype);
  if (rc != SCREE_OK) return rc;
  if (N == 0) return SCREE_OK;
  SCREE_CHECK_ARG(logits && targets && logp && entropy && (top == 0 || (top_logp && top_ids)),
                  "token_logprobs: null pointer");
  SCREE_CHECK_ARG((uintptr_t)logits % dtype_size(dtype) == 0 && (uintptr_t)norm % 8 == 0,
                  "token_logprobs: misaligned logits or norm");
  SCREE_BIND_DEVICE(stream, logits);
  FwdArgs a;
  a.x = logits;
  a.row_stride = row_stride;
  a.N = N;
  a.V = (int)V;
  a.chunks = (int)row_chunks(V, dtype);
  a.segs = row_segs(N, V, dtype);
  a.seg_bits = 0;
  while (1 << a.seg_bits < a.segs) ++a.seg_bits;
  a.targets = targets;
  a.t64 = targets_is_i64;
  a.top = top;
  a.logp = logp;
  a.entropy = entropy;
  a.norm = (float2*)norm;
  a.top_logp = top_logp;
  a.top_ids = top_ids;
  a.status = device_status_ptr();
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SCREE_F32) return launch_fwd<float>(a, s);
  return dtype == SCREE_BF16 ? launch_fwd<__nv_bfloat16>(a, s) : launch_fwd<__half>(a, s);
}

extern "C" int scree_token_logprobs_bwd(const void* logits, int64_t row_stride, const void* targets,
                                        int targets_is_i64, const float* norm, const float* entropy,
                                        const int64_t* top_ids, const float* g_logp,
                                        const float* g_entropy, const float* g_top, int64_t N,
                                        int64_t V, int top, int dtype, void* d_logits,
                                        void* stream) {
  int rc = check_sizes("token_logprobs backward", N, V, row_stride, top, dtype);
  if (rc != SCREE_OK) return rc;
  if (N == 0) return SCREE_OK;
  SCREE_CHECK_ARG(logits && targets && norm && entropy && d_logits && (top == 0 || g_top == nullptr || top_ids),
                  "token_logprobs backward: null pointer");
  SCREE_CHECK_ARG((uintptr_t)logits % dtype_size(dtype) == 0 && (uintptr_t)d_logits % dtype_size(dtype) == 0 &&
                      (uintptr_t)norm % 8 == 0,
                  "token_logprobs backward: misaligned logits or norm");
  SCREE_BIND_DEVICE(stream, logits);
  BwdArgs a;
  a.x = logits;
  a.row_stride = row_stride;
  a.N = N;
  a.V = (int)V;
  a.slices = (int)bwd_slices(V, dtype);
  a.targets = targets;
  a.t64 = targets_is_i64;
  a.top = top;
  a.norm = (const float2*)norm;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.g_logp = g_logp;
  a.g_entropy = g_entropy;
  a.g_top = top > 0 ? g_top : nullptr;
  a.dx = d_logits;
  a.status = device_status_ptr();
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SCREE_F32) return launch_bwd<float>(a, s);
  return dtype == SCREE_BF16 ? launch_bwd<__nv_bfloat16>(a, s) : launch_bwd<__half>(a, s);
}
