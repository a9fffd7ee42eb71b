// logprobs.cu — log probabilities of given tokens, entropies and top
// alternatives of (N, V) logits, and the gradient of the logits.
//
//   lse = m + log s1,  s1 = sum e^(x - m),  s2 = sum e^(x - m) (x - m),  m = max x
//   logp = x[target] - lse,  H = -sum p log p = log s1 - s2 / s1
//   dx_v = g_logp [v = target] + sum_j g_top_j [v = id_j]
//          - p_v (g_logp + sum_j g_top_j) - g_H p_v (log p_v + H)
//
// Forward: each logit is read from HBM once.  A CTA takes a slice of a row
// (kThreads x NV 16-byte vectors), keeps it in registers as it was loaded, and
// forms per thread the maximum, then s1 and s2 against that maximum, so there
// is no rescaling in the element loop.  The k-th largest of the threads' maxima
// bounds the slice's k-th largest element from below; only elements that reach
// it (about k of them) are ranked.  Slices are joined by a second kernel, one
// warp per row, or in place when a row is one slice.
//
// Numerics: sums in fp32, in units of log2 (one FMA and one ex2 per element;
// the product x log2e is not rounded before m is subtracted).
#include <algorithm>
#include "common.cuh"
#include "sm100.cuh"

namespace scree {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;     // one alternative per lane when lists are merged
constexpr int kCand = 512;      // ranked candidates of a slice; more take the slow exact path
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kSiteTarget = 50;

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

// Running statistics: m2 = m log2e, s1, s2 (log2 units); s1 = 0 when empty.
struct Stat {
  float m2, s1, s2;
};
__device__ __forceinline__ Stat stat_join(const Stat& a, const Stat& b) {
  Stat r;
  r.m2 = max_nan(a.m2, b.m2);
  const float ref = r.m2 == -INFINITY ? 0.f : r.m2;
  // An empty side has m2 = -inf: its weight is 0 and its (finite) shift is not used.
  const float da = fmaxf(a.m2 - ref, -1000.f), db = fmaxf(b.m2 - ref, -1000.f);
  const float wa = ex2_approx(a.m2 - ref), wb = ex2_approx(b.m2 - ref);
  r.s1 = a.s1 * wa + b.s1 * wb;
  r.s2 = wa * (a.s2 + da * a.s1) + wb * (b.s2 + db * b.s1);
  return r;
}
__device__ __forceinline__ Stat stat_warp(Stat s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat t;
    t.m2 = __shfl_xor_sync(0xffffffffu, s.m2, o);
    t.s1 = __shfl_xor_sync(0xffffffffu, s.s1, o);
    t.s2 = __shfl_xor_sync(0xffffffffu, s.s2, o);
    s = stat_join(s, t);
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
template <typename K> __device__ __forceinline__ K lane_sort(K v, int lane) {
#pragma unroll
  for (int k = 2; k <= 16; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const K o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool up = ((lane & k) == 0) == ((lane & j) == 0);
      v = up == (v > o) ? v : o;
    }
  return lane_merge(v, lane);
}
// The 32 largest of two descending lists of 32.
template <typename K> __device__ __forceinline__ K lane_join(K a, K b, int lane) {
  const K r = __shfl_sync(0xffffffffu, b, 31 - lane);
  return lane_merge(a > r ? a : r, lane);
}

struct FwdArgs {
  const void* x;
  int64_t row_stride, N;
  uint32_t V;
  int slices;
  const void* targets;
  int t64;
  int top;
  float *logp, *entropy, *lse, *top_logp;
  int64_t* top_ids;
  Stat* part;                  // (N, slices)
  unsigned long long* part_keys;  // (N, slices, top)
  int* status;
};

// The row's outputs from its joined statistics; `key` is the lane's alternative.
template <typename T>
__device__ __forceinline__ void finish_row(const FwdArgs& a, int64_t n, const Stat& s,
                                           unsigned long long key, int lane) {
  // A row with nothing left (every logit -inf): lse = logp = -inf, H = 0.
  const bool empty = s.m2 == -INFINITY;
  const float lse = empty ? -INFINITY : (s.m2 + log2f(s.s1)) * kLn2;
  if (lane == 0) {
    a.lse[n] = lse;
    a.entropy[n] = empty ? 0.f : (log2f(s.s1) - s.s2 / s.s1) * kLn2;
    const int64_t t = a.t64 ? reinterpret_cast<const int64_t*>(a.targets)[n]
                            : (int64_t)reinterpret_cast<const int32_t*>(a.targets)[n];
    float lp = 0.f;  // negative target: no token given
    if (t >= (int64_t)a.V) {
      record_device_error(a.status, SCREE_DEVERR_BAD_INPUT, kSiteTarget);
      lp = __uint_as_float(0x7FFFFFFFu);
    } else if (t >= 0) {
      const float x = Cvt<T>::to_f(reinterpret_cast<const T*>(a.x)[n * a.row_stride + t]);
      lp = empty ? -INFINITY : x - lse;
    }
    a.logp[n] = lp;
  }
  if (lane < a.top) {
    a.top_ids[n * a.top + lane] = (int64_t)(0xFFFFFFFFu - (uint32_t)key);
    const float x = order_value((uint32_t)(key >> 32));
    a.top_logp[n * a.top + lane] = empty ? -INFINITY : x - lse;
  }
}

template <typename T, int NV>
__global__ void __launch_bounds__(kThreads) logprobs_slice_kernel(const FwdArgs a) {
  constexpr int VE = Lv<T>::N;
  __shared__ Stat sm_stat[kThreads / 32];
  __shared__ uint32_t sm_max[kThreads / 32][32];
  __shared__ unsigned long long sm_cand[kCand];
  __shared__ unsigned long long sm_top[kMaxTop];
  __shared__ unsigned long long sm_red[kThreads / 32];
  __shared__ int sm_count;
  __shared__ uint32_t sm_tau;
  asm volatile("griddepcontrol.launch_dependents;");
  const int64_t n = blockIdx.x / (unsigned)a.slices;
  const int slice = blockIdx.x % (unsigned)a.slices;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* row = reinterpret_cast<const T*>(a.x) + n * a.row_stride;
  // Vectors start at 16-byte boundaries: the row begins `mis` elements into its
  // first vector.  A vector that crosses an end of the row is read element by element.
  const int mis = (int)(((uintptr_t)row & 15) / sizeof(T));
  const int64_t v0 = (int64_t)slice * kThreads * NV;  // first vector of the slice
  uint4 d[NV];
  // Index of element 0 of vector i of this thread (may be negative or past V).
  auto first = [&](int i) { return (v0 + i * kThreads + threadIdx.x) * VE - mis; };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t e0 = first(i);
    if (e0 >= 0 && e0 + VE <= (int64_t)a.V) {
      d[i] = __ldcs(reinterpret_cast<const uint4*>(row + e0));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = neg_inf_word<T>();
      if (e0 + VE > 0 && e0 < (int64_t)a.V) {
        T* el = reinterpret_cast<T*>(w);
#pragma unroll
        for (int u = 0; u < VE; ++u)
          if (e0 + u >= 0 && e0 + u < (int64_t)a.V) el[u] = row[e0 + u];
      }
      d[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  float vm[NV], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vm[i] = vec_max<T>(d[i]);
    m = max_nan(m, vm[i]);
  }
  Stat st{-INFINITY, 0.f, 0.f};
  if (m != -INFINITY) {
    st.m2 = m * kLog2e;
    const uint64_t l2 = f2_pack(kLog2e, kLog2e), nm = f2_pack(-st.m2, -st.m2);
    uint64_t s1a = 0, s1b = 0, s2a = 0, s2b = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VE];
      unpack_vec<T>(d[i], f);
#pragma unroll
      for (int u = 0; u < VE; u += 4) {
        auto two = [&](int j, uint64_t& s1, uint64_t& s2) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(f[j], f[j + 1]), l2, nm), x0, x1);
          const uint64_t e = f2_pack(ex2_approx(x0), ex2_approx(x1));
          s1 = f2_add(s1, e);
          // -inf has e = 0; the bound keeps its term 0 instead of 0 * inf.
          s2 = f2_fma(e, f2_pack(fmaxf(x0, -1000.f), fmaxf(x1, -1000.f)), s2);
        };
        two(u, s1a, s2a);
        two(u + 2, s1b, s2b);
      }
    }
    float p, q;
    f2_unpack(f2_add(s1a, s1b), p, q);
    st.s1 = p + q;
    f2_unpack(f2_add(s2a, s2b), p, q);
    st.s2 = p + q;
  }
  st = stat_warp(st);
  if (lane == 0) sm_stat[warp] = st;

  if (a.top > 0) {
    // Bound: the top-th largest thread maximum (threads without a valid element count as 0).
    const bool any = first(0) + VE > 0 && first(0) < (int64_t)a.V;
    sm_max[warp][lane] = lane_sort<uint32_t>(any ? order_bits(m) : 0u, lane);
    if (threadIdx.x == 0) sm_count = 0;
    __syncthreads();
    if (warp == 0) {
      uint32_t best = sm_max[0][lane];
#pragma unroll
      for (int w = 1; w < kThreads / 32; ++w) best = lane_join(best, sm_max[w][lane], lane);
      if (lane == a.top - 1) sm_tau = best;
    }
    __syncthreads();
    const uint32_t tau = sm_tau;
    if (any && order_bits(m) >= tau) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (order_bits(vm[i]) < tau) continue;
        float f[VE];
        unpack_vec<T>(d[i], f);
        const int64_t e0 = first(i);
#pragma unroll
        for (int u = 0; u < VE; ++u) {
          if (order_bits(f[u]) >= tau && e0 + u >= 0 && e0 + u < (int64_t)a.V) {
            const int at = atomicAdd(&sm_count, 1);
            if (at < kCand) sm_cand[at] = order_key(f[u], (uint32_t)(e0 + u));
          }
        }
      }
    }
    __syncthreads();
    const int cnt = sm_count;
    if (threadIdx.x < kMaxTop) sm_top[threadIdx.x] = 0;
    __syncthreads();
    if (cnt <= kCand) {
      // Keys differ, so a candidate's rank is the number of larger ones, whatever
      // order the candidates arrived in.
      for (int i = threadIdx.x; i < cnt; i += kThreads) {
        const unsigned long long key = sm_cand[i];
        int rank = 0;
        for (int j = 0; j < cnt; ++j) rank += sm_cand[j] > key;
        if (rank < a.top) sm_top[rank] = key;
      }
      __syncthreads();
    } else {
      // Many equal elements: take the largest remaining key, `top` times.
      unsigned long long last = ~0ull;
      for (int r = 0; r < a.top; ++r) {
        unsigned long long best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float f[VE];
          unpack_vec<T>(d[i], f);
          const int64_t e0 = first(i);
#pragma unroll
          for (int u = 0; u < VE; ++u) {
            if (e0 + u < 0 || e0 + u >= (int64_t)a.V) continue;
            const unsigned long long key = order_key(f[u], (uint32_t)(e0 + u));
            if (key < last && key > best) best = key;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long t = __shfl_xor_sync(0xffffffffu, best, o);
          best = t > best ? t : best;
        }
        if (lane == 0) sm_red[warp] = best;
        __syncthreads();
        best = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) best = sm_red[w] > best ? sm_red[w] : best;
        if (threadIdx.x == 0) sm_top[r] = best;
        last = best;
        __syncthreads();
      }
    }
  } else {
    __syncthreads();
  }
  if (warp == 0) {
    Stat s = lane < kThreads / 32 ? sm_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
    s = stat_warp(s);
    if (a.slices == 1) {
      finish_row<T>(a, n, s, lane < a.top ? sm_top[lane] : 0, lane);
    } else {
      if (lane == 0) a.part[n * a.slices + slice] = s;
      if (lane < a.top) a.part_keys[(n * a.slices + slice) * a.top + lane] = sm_top[lane];
    }
  }
}

// One warp per row joins the slices.
template <typename T>
__global__ void __launch_bounds__(128) logprobs_join_kernel(const FwdArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  Stat s{-INFINITY, 0.f, 0.f};
  for (int j = lane; j < a.slices; j += 32) s = stat_join(s, a.part[n * a.slices + j]);
  s = stat_warp(s);
  unsigned long long best = 0;
  if (a.top > 0) {
    const unsigned long long* keys = a.part_keys + n * a.slices * a.top;
    for (int j = 0; j < a.slices; ++j) {
      const unsigned long long k = lane < a.top ? keys[(int64_t)j * a.top + lane] : 0;
      best = j == 0 ? k : lane_join(best, k, lane);
    }
  }
  finish_row<T>(a, n, s, best, lane);
}

struct BwdArgs {
  const void* x;
  int64_t row_stride, N;
  uint32_t V;
  int slices;
  const void* targets;
  int t64;
  int top;
  const float *lse, *entropy;
  const int64_t* top_ids;
  const float *g_logp, *g_entropy, *g_top;  // each may be null
  void* dx;                                 // (N, V) contiguous
};

// dx = -p (gs + gH (H + log p)), then the given token and the alternatives.
// HBM-bound: one read and one write of each logit.
template <typename T, int NV>
__global__ void __launch_bounds__(kThreads) logprobs_bwd_kernel(const BwdArgs a) {
  constexpr int VE = Lv<T>::N;
  __shared__ float sm_gs;
  const int64_t n = blockIdx.x / (unsigned)a.slices;
  const int slice = blockIdx.x % (unsigned)a.slices;
  const T* row = reinterpret_cast<const T*>(a.x) + n * a.row_stride;
  T* out = reinterpret_cast<T*>(a.dx) + n * (int64_t)a.V;
  const int mis = (int)(((uintptr_t)row & 15) / sizeof(T));
  const bool same = (((uintptr_t)row ^ (uintptr_t)out) & 15) == 0;
  const int64_t v0 = (int64_t)slice * kThreads * NV;
  uint4 d[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t e0 = (v0 + i * kThreads + threadIdx.x) * VE - mis;
    if (e0 >= 0 && e0 + VE <= (int64_t)a.V) {
      d[i] = __ldcs(reinterpret_cast<const uint4*>(row + e0));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = neg_inf_word<T>();
      if (e0 + VE > 0 && e0 < (int64_t)a.V) {
        T* el = reinterpret_cast<T*>(w);
#pragma unroll
        for (int u = 0; u < VE; ++u)
          if (e0 + u >= 0 && e0 + u < (int64_t)a.V) el[u] = row[e0 + u];
      }
      d[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  // The given token and the alternatives as one list of (index, weight): entry 0
  // is the target, entry 1 + j alternative j; index -1 has no weight.
  auto entry = [&](int j, int64_t& idx) -> float {
    if (j == 0) {
      idx = a.t64 ? reinterpret_cast<const int64_t*>(a.targets)[n]
                  : (int64_t)reinterpret_cast<const int32_t*>(a.targets)[n];
      if (idx < 0 || idx >= (int64_t)a.V || a.g_logp == nullptr) idx = -1;
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
  const float lse = a.lse[n];
  const float gh = a.g_entropy != nullptr ? a.g_entropy[n] : 0.f;
  const bool empty = lse == -INFINITY;  // nothing left in the row: no gradient
  const float base = sm_gs + gh * a.entropy[n];
  const float l2 = lse * kLog2e;
  auto grad = [&](float x) {
    const float d2 = fmaf(x, kLog2e, -l2);  // log2 p
    // The bound only matters at p = 0, where it keeps 0 * inf out.
    return -ex2_approx(d2) * fmaf(gh, fmaxf(d2, -1000.f) * kLn2, base);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t e0 = (v0 + i * kThreads + threadIdx.x) * VE - mis;
    if (e0 + VE <= 0 || e0 >= (int64_t)a.V) continue;
    float f[VE];
    unpack_vec<T>(d[i], f);
#pragma unroll
    for (int u = 0; u < VE; ++u) f[u] = empty ? 0.f : grad(f[u]);
    __align__(16) T o[VE];
    cvt_from_f<T, VE>(f, o);
    if (same && e0 >= 0 && e0 + VE <= (int64_t)a.V) {
      __stcs(reinterpret_cast<uint4*>(out + e0), *reinterpret_cast<const uint4*>(o));
    } else {
#pragma unroll
      for (int u = 0; u < VE; ++u)
        if (e0 + u >= 0 && e0 + u < (int64_t)a.V) out[e0 + u] = o[u];
    }
  }
  // The listed elements of this slice, written again with their weights (after
  // the barrier, so over the plain value).  Entries with one index write one value.
  __syncthreads();
  if (threadIdx.x < entries && !empty) {
    int64_t idx;
    entry(threadIdx.x, idx);
    const int64_t lo = v0 * VE - mis;
    if (idx >= 0 && idx >= lo && idx < lo + (int64_t)kThreads * NV * VE) {
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

constexpr int kNV = 8;
template <typename T> int64_t slice_elems() { return (int64_t)kThreads * kNV * Lv<T>::N; }
int64_t row_slices(int64_t V, int dtype) {
  const int64_t per = dtype == SCREE_F32 ? slice_elems<float>() : slice_elems<__half>();
  const int64_t lead = dtype == SCREE_F32 ? 3 : 7;  // a row may begin inside its first vector
  return (V + lead + per - 1) / per;
}

int check_sizes(const char* what, int64_t N, int64_t V, int64_t row_stride, int top, int dtype) {
  SCREE_CHECK_ARG(dtype == SCREE_F16 || dtype == SCREE_BF16 || dtype == SCREE_F32,
                  "%s: fp16, bf16 or fp32 only", what);
  SCREE_CHECK_ARG(N >= 0 && V >= 1 && V < (1ll << 31), "%s: bad sizes N=%lld V=%lld", what,
                  (long long)N, (long long)V);
  SCREE_CHECK_ARG(row_stride >= V || N <= 1, "%s: rows overlap (row stride %lld, V=%lld)", what,
                  (long long)row_stride, (long long)V);
  SCREE_CHECK_ARG(top >= 0 && top <= kMaxTop && top <= V,
                  "%s: top must be between 0 and %d and at most V (got %d)", what, kMaxTop, top);
  SCREE_CHECK_ARG(N * row_slices(V, dtype) < (1ll << 31), "%s: N=%lld too large", what,
                  (long long)N);
  return SCREE_OK;
}

template <typename T> int launch_fwd(const FwdArgs& a, cudaStream_t s) {
  logprobs_slice_kernel<T, kNV><<<(unsigned)(a.N * a.slices), kThreads, 0, s>>>(a);
  SCREE_LAUNCH_CHECK();
  if (a.slices > 1) {
    SCREE_CUDA_TRY(launch_dependent(logprobs_join_kernel<T>, dim3((unsigned)((a.N + 3) / 4)),
                                    dim3(128), 0, s, a));
    count_launch();
  }
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

extern "C" size_t scree_token_logprobs_workspace_size(int64_t N, int64_t V, int top, int dtype) {
  const int64_t sl = row_slices(V, dtype);
  if (N <= 0 || V <= 0 || sl == 1) return 0;
  return (size_t)(N * sl) * (16 + 8 * (size_t)(top > 0 ? top : 0));
}

extern "C" int scree_token_logprobs_fwd(const void* logits, int64_t row_stride, const void* targets,
                                        int targets_is_i64, int64_t N, int64_t V, int top,
                                        int dtype, float* logp, float* entropy, float* lse,
                                        float* top_logp, int64_t* top_ids, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  int rc = check_sizes("token_logprobs", N, V, row_stride, top, dtype);
  if (rc != SCREE_OK) return rc;
  if (N == 0) return SCREE_OK;
  SCREE_CHECK_ARG(logits && targets && logp && entropy && lse && (top == 0 || (top_logp && top_ids)),
                  "token_logprobs: null pointer");
  SCREE_CHECK_ARG((uintptr_t)logits % dtype_size(dtype) == 0, "token_logprobs: misaligned logits");
  const size_t need = scree_token_logprobs_workspace_size(N, V, top, dtype);
  SCREE_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
                  "token_logprobs: workspace too small");
  SCREE_BIND_DEVICE(stream, logits);
  FwdArgs a;
  a.x = logits;
  a.row_stride = row_stride;
  a.N = N;
  a.V = (uint32_t)V;
  a.slices = (int)row_slices(V, dtype);
  a.targets = targets;
  a.t64 = targets_is_i64;
  a.top = top;
  a.logp = logp;
  a.entropy = entropy;
  a.lse = lse;
  a.top_logp = top_logp;
  a.top_ids = top_ids;
  a.part_keys = reinterpret_cast<unsigned long long*>(workspace);
  a.part = reinterpret_cast<Stat*>(reinterpret_cast<char*>(workspace) + 8 * (size_t)(N * a.slices) * top);
  a.status = device_status_ptr();
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SCREE_F32) return launch_fwd<float>(a, s);
  return dtype == SCREE_BF16 ? launch_fwd<__nv_bfloat16>(a, s) : launch_fwd<__half>(a, s);
}

extern "C" int scree_token_logprobs_bwd(const void* logits, int64_t row_stride, const void* targets,
                                        int targets_is_i64, const float* lse, const float* entropy,
                                        const int64_t* top_ids, const float* g_logp,
                                        const float* g_entropy, const float* g_top, int64_t N,
                                        int64_t V, int top, int dtype, void* d_logits,
                                        void* stream) {
  int rc = check_sizes("token_logprobs backward", N, V, row_stride, top, dtype);
  if (rc != SCREE_OK) return rc;
  if (N == 0) return SCREE_OK;
  SCREE_CHECK_ARG(logits && targets && lse && entropy && d_logits && (top == 0 || g_top == nullptr || top_ids),
                  "token_logprobs backward: null pointer");
  SCREE_CHECK_ARG((uintptr_t)logits % dtype_size(dtype) == 0 && (uintptr_t)d_logits % dtype_size(dtype) == 0,
                  "token_logprobs backward: misaligned logits");
  SCREE_BIND_DEVICE(stream, logits);
  BwdArgs a;
  a.x = logits;
  a.row_stride = row_stride;
  a.N = N;
  a.V = (uint32_t)V;
  a.slices = (int)row_slices(V, dtype);
  a.targets = targets;
  a.t64 = targets_is_i64;
  a.top = top;
  a.lse = lse;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.g_logp = g_logp;
  a.g_entropy = g_entropy;
  a.g_top = top > 0 ? g_top : nullptr;
  a.dx = d_logits;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == SCREE_F32) return launch_bwd<float>(a, s);
  return dtype == SCREE_BF16 ? launch_bwd<__nv_bfloat16>(a, s) : launch_bwd<__half>(a, s);
}
