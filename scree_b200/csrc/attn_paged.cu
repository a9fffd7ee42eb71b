// attn_paged.cu — attention of new tokens (single ones, chunks, trees of drafted
// tokens) over a paged K/V cache.
//
//   S = Q K^T scale over the visible keys, P = softmax(S), O = P V, LSE = m + ln l
//
// The rows that share a K/V head (token i, query head h * G + g -> row i G + g)
// form row tiles of R rows; a (sequence, K/V head, row tile) is a segment, its
// units groups of KEYS keys (and kLead more).  All segments laid end to end are cut into
// equal runs of groups, one run per worker, so the cache is read evenly by the
// whole GPU whatever the lengths are: a long sequence is spread over many
// workers, short ones share a worker.  A worker is one warp with a ring of
// shared memory of its own, filled by TMA one group ahead of the next; the
// warps of a CTA never wait for one another.  A segment that one worker holds
// whole is written out by it; pieces of a split segment go to the workspace as
// (m, l, O) and a second kernel joins them.
//
// Bound: HBM, 4 D bytes per key and K/V head (R = 16 rows of mma.sync work per
// key hide under that).  64 sequences of 2048 keys on average, lengths spread 0.6
// log-normal, 8 K/V heads of 128: 113 us for 621 MB, 5.5 TB/s; the SMs end between 90
// and 104 us, the join takes the rest.  (The last sixth of the groups handed out from
// a counter instead: 117.6 us against 115.9 on the same build, its join slower.)  A group is as many keys as make 8 KB of K and V: the
// chain scores -> maximum -> exponentials -> product takes a warp about 1,000
// cycles whatever the number of keys, and with 16 keys at D = 64 that, not HBM,
// set the pace (2 x 131071 keys: main kernel 25 us against 21).  It is loaded in
// boxes of 16 keys, which never span pages.
//
// P goes to the product with V in the queries' 16-bit type, as mma.sync takes it and as
// in attn_fwd.cu: each weight is off by half a unit of that type, the row sums l and the
// pieces are fp32.
#include <algorithm>
#include "attn_paged.cuh"

namespace scree {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kBox = kPagedKeys;     // keys of a box
constexpr int R = 16;                // rows of a tile: one mma
// A segment's units are kLead idle ones, which stand for what starting a piece
// costs a worker, and its groups.
constexpr int kLead = 1;

template <int D> struct Cfg {
  static constexpr int GP = 128 / D;               // boxes of a group
  static constexpr int KEYS = GP * kBox;
  static constexpr int ROWB = D >= 64 ? 128 : 64;  // bytes of a box row (= swizzle span)
  static constexpr int NB = D * 2 / ROWB;          // boxes across D
  static constexpr int BOX = kBox * ROWB;
  static constexpr int PART = GP * NB * BOX;       // K (or V) of a group
  static constexpr int STAGE = 2 * PART;           // 8 KB
  static constexpr int STAGES = 3;                 // 24 KB in flight per warp, 192 KB per SM
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr int smem(int64_t B) {
    return 1024 + RING + kWarps * STAGES * 8 + 64 + (int)(B + 1) * 8;
  }
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  T o[2];
  const float f[2] = {a, b};
  cvt_from_f<T, 2>(f, o);
  return (uint32_t)*reinterpret_cast<uint16_t*>(&o[0]) | ((uint32_t)*reinterpret_cast<uint16_t*>(&o[1]) << 16);
}
template <int D, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    attn_paged_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const PagedParams p) {
  using C = Cfg<D>;
  constexpr int KK = D / 16;  // k-steps of Q K^T = pairs of 8-column tiles of O
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::RING);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kWarps * C::STAGES);
  int64_t* pre = reinterpret_cast<int64_t*>(reinterpret_cast<uint8_t*>(bars + kWarps * C::STAGES) + 64);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  if (threadIdx.x < kWarps * C::STAGES) mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_mbar_init();
  // Units before each sequence, by every CTA for itself (a launch of its own
  // would cost more than these few loads).
  if (!paged_prefix<kWarps>(p, pre, [&](int64_t n, int64_t len) {
        return (int64_t)((unsigned)(n * p.G + R - 1) / R) * (kLead + (unsigned)(len + C::KEYS - 1) / C::KEYS) * p.Hkv;
      }))
    return;
  const int64_t U = pre[p.B];  // > 0: T = 0 does not launch, and a new token is a key
  const int64_t N = min((int64_t)gridDim.x * kWarps, U);
  // Neighbouring runs go to different SMs, so few workers are spread out too.
  const int64_t w = (int64_t)warp * gridDim.x + blockIdx.x;
  if (w >= N) {
    if (lane == 0) p.desc[w].on = 0;
    return;
  }
  const PagedCut cut(U, N);
  const int64_t u0 = cut.start(w), u1 = cut.start(w + 1);

  struct Seg {
    int b, h, rt, slot, len;
    int64_t s0, s1;
  };
  auto find = [&](int64_t u) {
    const int lo = paged_find(pre, p.B, u);
    Seg g;
    g.b = lo;
    g.slot = p.slots[lo];
    g.len = p.lengths[g.slot];
    const unsigned groups = (unsigned)(g.len + C::KEYS - 1) / C::KEYS, seg = kLead + groups;
    const int64_t at = udiv(u - pre[lo], seg);  // segment within the sequence
    const unsigned rts = (unsigned)udiv(pre[lo + 1] - pre[lo], seg) / (unsigned)p.Hkv;  // row tiles
    g.h = (int)((unsigned)at / rts);
    g.rt = (int)((unsigned)at - g.h * rts);
    g.s0 = pre[lo] + at * seg + kLead;  // the unit of group 0
    g.s1 = g.s0 + groups;
    return g;
  };

  uint8_t* ring = smem + warp * C::STAGES * C::STAGE;
  const uint32_t ring_s = smem_u32(ring);
  uint64_t* full = bars + warp * C::STAGES;

  // Loads run ahead of the work, across segments.  The page ids of 32 boxes at a
  // time sit in the lanes (past the end those of the last box: its keys are masked
  // and its V is taken out).
  int64_t ui = u0;
  Seg gi = find(u0);
  int64_t win = -1;  // first unit of the window of page ids
  int my_page = 0;
  int ist = 0;
  auto issue = [&]() {
    if (ui >= gi.s1 && ui < u1) {
      gi = find(ui);
      win = -1;
    }
    ui = max(ui, gi.s0);  // past the segment's lead
    if (ui >= u1) return;
    const int last = (gi.len - 1) / kBox;
    if (win < 0 || ui >= win + 32 / C::GP) {
      win = ui;
      my_page = paged_page(p, gi.slot, min((int)(ui - gi.s0) * C::GP + lane, last));
    }
    int page[C::GP];
#pragma unroll
    for (int q = 0; q < C::GP; ++q)
      page[q] = __shfl_sync(0xffffffffu, my_page, (int)(ui - win) * C::GP + q);
    if (lane == 0) {
      uint8_t* st = ring + ist * C::STAGE;
      mbar_expect_tx(&full[ist], C::STAGE);
#pragma unroll
      for (int q = 0; q < C::GP; ++q) {
        const unsigned box = (unsigned)min((int)(ui - gi.s0) * C::GP + q, last);
        const int row = (int)(p.layer_row + ((int64_t)page[q] * p.Hkv + gi.h) * p.page + box * kBox % (unsigned)p.page);
#pragma unroll
        for (int c = 0; c < C::NB; ++c) {
          uint8_t* at = st + (q * C::NB + c) * C::BOX;
          tma_load_2d(at, &tm_k, &full[ist], c * (C::ROWB / 2), row);
          tma_load_2d(at + C::PART, &tm_v, &full[ist], c * (C::ROWB / 2), row);
        }
      }
    }
    ist = ist + 1 == C::STAGES ? 0 : ist + 1;
    ++ui;
  };
#pragma unroll 1
  for (int i = 0; i < C::STAGES; ++i) issue();

  // Byte offset of 16-byte chunk c of key k of a box (TMA's swizzle).
  auto chunk = [](int k, int c) -> uint32_t {
    constexpr int CPR = C::ROWB / 16;
    const int sw = C::ROWB == 128 ? (k & 7) : ((k >> 1) & 3);
    return (uint32_t)((c / CPR) * C::BOX + k * C::ROWB + (((c % CPR) ^ sw) << 4));
  };
  const int mi = lane >> 3;
  const int k_key = (mi >> 1) * 8 + (lane & 7), k_c = mi & 1;  // ldmatrix rows of K
  const int v_key = (mi & 1) * 8 + (lane & 7), v_c = mi >> 1;  // and of V
  const int qr = lane >> 2, qc = (lane & 3) * 2;               // row and column in mma tiles

  int cst = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t u = u0; ok && u < u1;) {
    const Seg g = find(u);
    const bool run_start = u == u0;
    u = max(u, g.s0);
    const int64_t begin = u, end = min(u1, g.s1);
    const int64_t q0 = load_offset(p.offs, p.is64, g.b);
    const int n = (int)(load_offset(p.offs, p.is64, g.b + 1) - q0);
    if (run_start && lane == 0) {
      const int w0 = (int)cut.of(g.s0);
      p.desc[w] = PagedDesc{u0 > g.s0 ? 1 : 0, w0, (int)cut.of(g.s1 - 1) - w0 + 1, (int)q0, g.h, g.rt * R, n};
    }
    if (u >= u1) break;  // the run ends in a segment's lead
    const int c0 = g.len - n;
    const int rows = min(R, n * p.G - g.rt * R);
    // Rows of this lane: half r -> row r * 8 + qr of the tile.
    auto row_of = [&](int r) { return r * 8 + qr; };
    uint32_t qf[KK][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = row_of(r);
      const int a = g.rt * R + row;
      const bool in = row < rows;
      const char* src = p.q + (q0 + (in ? a / p.G : 0)) * p.q_rs + (int64_t)(g.h * p.G + (in ? a % p.G : 0)) * p.q_hs;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        qf[kk][r] = in ? *reinterpret_cast<const uint32_t*>(src + (kk * 16 + qc) * 2) : 0u;
        qf[kk][2 + r] = in ? *reinterpret_cast<const uint32_t*>(src + (kk * 16 + 8 + qc) * 2) : 0u;
      }
    }
    float o[2 * KK][4];
    float m[2], l[2];
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * KK; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
#pragma unroll 1
    for (; u < end; ++u) {
      ok = paged_wait(p, &full[cst], phase, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const uint32_t ks = ring_s + cst * C::STAGE, vs = ks + C::PART;
      constexpr int NT = 2 * C::GP;  // 8-key tiles of the scores
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int q = 0; q < C::GP; ++q) {
          uint32_t kf[4];
          ldsm_x4(ks + q * C::NB * C::BOX + chunk(k_key, kk * 2 + k_c), kf);
          mma16816<T>(s[2 * q], qf[kk], kf[0], kf[1]);
          mma16816<T>(s[2 * q + 1], qf[kk], kf[2], kf[3]);
        }
      const int k0 = (int)(u - g.s0) * C::KEYS;
      const bool edge = k0 + C::KEYS > c0;  // holds new tokens, or runs past the end
      unsigned long long vis[2];
      if (edge) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = row_of(r), i = row < rows ? (g.rt * R + row) / p.G : 0;
          vis[r] = paged_visible<C::KEYS>(p, q0 + i, i, k0, c0, g.len);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!(vis[r] >> (t * 8 + qc + e) & 1)) s[t][r * 2 + e] = -INFINITY;
        }
      }
      // Running maximum; rescaled only when it grew by more than 2^8 (P stays <= 256).
      float alpha[2];
      bool need = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(s[0][r * 2], s[0][r * 2 + 1]);
#pragma unroll
        for (int t = 1; t < NT; ++t) mx = fmax3(mx, s[t][r * 2], s[t][r * 2 + 1]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mc = mx * p.sl2;
        alpha[r] = 1.f;
        if (mc > m[r] + 8.f) {
          alpha[r] = ex2_weight(m[r] - mc);
          m[r] = mc;
          need = true;
        }
      }
      if (__any_sync(0xffffffffu, need)) {
        l[0] *= alpha[0];
        l[1] *= alpha[1];
#pragma unroll
        for (int j = 0; j < 2 * KK; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][e] *= alpha[e >> 1];
      }
      uint32_t pf[C::GP][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float mm = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float e0 = ex2_approx(fmaf(s[t][r * 2], p.sl2, -mm));
          const float e1 = ex2_approx(fmaf(s[t][r * 2 + 1], p.sl2, -mm));
          l[r] += e0 + e1;
          pf[t >> 1][(t & 1) * 2 + r] = pack2<T>(e0, e1);
        }
      }
      if (!edge) {
#pragma unroll
        for (int q = 0; q < C::GP; ++q)
#pragma unroll
          for (int j = 0; j < KK; ++j) {
            uint32_t vf[4];
            ldsm_x4_t(vs + q * C::NB * C::BOX + chunk(v_key, j * 2 + v_c), vf);
            mma16816<T>(o[2 * j], pf[q], vf[0], vf[1]);
            mma16816<T>(o[2 * j + 1], pf[q], vf[2], vf[3]);
          }
      } else {
        // A key that a row does not see must not reach it even if its V is an
        // infinity or NaN (0 * NaN): such elements, and the rows past the end of
        // the sequence, are taken out of the product; the infinities and NaN are
        // then added for the rows that do see them.
        const int left = g.len - k0;
        auto live = [&](int k) { return (k < left ? 0xFFFFu : 0u) | (k + 1 < left ? 0xFFFF0000u : 0u); };
        bool special = false;
#pragma unroll
        for (int q = 0; q < C::GP; ++q) {
          const uint32_t live_lo = live(q * kBox + qc), live_hi = live(q * kBox + qc + 8);
#pragma unroll
          for (int j = 0; j < KK; ++j) {
            uint32_t vf[4];
            ldsm_x4_t(vs + q * C::NB * C::BOX + chunk(v_key, j * 2 + v_c), vf);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              vf[e] &= (e & 1) ? live_hi : live_lo;
              const uint32_t nf = nonfinite_halves<T>(vf[e]);
              special |= nf != 0;
              vf[e] &= ~nf;
            }
            mma16816<T>(o[2 * j], pf[q], vf[0], vf[1]);
            mma16816<T>(o[2 * j + 1], pf[q], vf[2], vf[3]);
          }
        }
        if (__any_sync(0xffffffffu, special)) {
#pragma unroll 1
          for (int k = 0; k < min(left, C::KEYS); ++k) {
#pragma unroll
            for (int j = 0; j < 2 * KK; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint8_t* at =
                    ring + cst * C::STAGE + C::PART + k / kBox * C::NB * C::BOX + chunk(k % kBox, j) + (qc + e) * 2;
                const uint16_t h = *reinterpret_cast<const uint16_t*>(at);
                if (nonfinite_halves<T>(h) & 0xFFFFu) {
                  const float x = Cvt<T>::to_f(*reinterpret_cast<const T*>(&h));
#pragma unroll
                  for (int r = 0; r < 2; ++r)
                    if (vis[r] >> k & 1) o[j][r * 2 + e] += x;  // P > 0
                }
              }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      issue();
      cst = cst + 1 == C::STAGES ? 0 : cst + 1;
      if (cst == 0) phase ^= 1;
    }
    if (!ok) {  // stages cst up to ist are in flight
      do {
        paged_drain(&full[cst], phase);
        cst = cst + 1 == C::STAGES ? 0 : cst + 1;
        if (cst == 0) phase ^= 1;
      } while (cst != ist);
      break;
    }
    // ---------------------------------------------------------------- piece done
    const bool whole = begin == g.s0 && end == g.s1;
    // A run has at most one piece that continues a segment and one that leaves one.
    const int64_t slot = 2 * w + (begin > g.s0 ? 0 : 1);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float sum = l[r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int row = row_of(r);
      if (row >= rows) continue;
      if (whole) {
        const int a = g.rt * R + row, hq = g.h * p.G + a % p.G;
        const int64_t tok = q0 + a / p.G;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        char* dst = p.o + tok * p.o_rs + hq * p.o_hs;
#pragma unroll
        for (int j = 0; j < 2 * KK; ++j)
          *reinterpret_cast<uint32_t*>(dst + (j * 8 + qc) * 2) =
              pack2<T>(o[j][r * 2] * inv, o[j][r * 2 + 1] * inv);
        if (p.lse != nullptr && (lane & 3) == 0)
          p.lse[tok * p.H + hq] = sum == 0.f ? -INFINITY : (m[r] + log2f(sum)) * 0.69314718055994531f;
      } else {
        float* dst = p.part_o + (slot * R + row) * D;
#pragma unroll
        for (int j = 0; j < 2 * KK; ++j)
          *reinterpret_cast<float2*>(dst + j * 8 + qc) = make_float2(o[j][r * 2], o[j][r * 2 + 1]);
        if ((lane & 3) == 0) p.part_ml[slot * R + row] = make_float2(m[r], sum);
      }
    }
  }
}

// Joins the pieces of a split segment: O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i.
// The workers that continue a segment (all of its pieces but the first) lend a
// block each; they deal its rows among them.  Where a segment has many pieces
// (one long sequence over the whole GPU) the warps of a block share a row's
// pieces, else each warp takes rows of its own.
constexpr int kJoinWarps = 8;
constexpr int64_t kManyPieces = 16;
template <int D, typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_paged_join_kernel(const PagedParams p) {
  constexpr int E = D / 32;         // columns of a lane
  constexpr int kLoads = E == 4 ? 8 : 16;  // O rows under way at a time
  __shared__ float sm_o[kJoinWarps][D];
  __shared__ float2 sm_ml[kJoinWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != 0) return;
  const PagedDesc d = p.desc[blockIdx.x + 1];
  if (!d.on) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int np = d.np, rows = min(R, d.n * p.G - d.i0), nth = (int)blockIdx.x - d.w0;
  auto slot_of = [&](int i) { return (int64_t)(i == 0 ? 2 * d.w0 + 1 : 2 * (d.w0 + i)); };
  const int share = np >= kManyPieces ? kJoinWarps : 1;  // warps of one row
  const int sub = warp % share;
  const int step = (np - 1) * (kJoinWarps / share);
  for (int row = nth * (kJoinWarps / share) + warp / share; row < rows; row += step) {
    // This warp's pieces sub, sub + share, ...: 32 at a time their (m, l) in the
    // lanes, their O rows kLoads at a time.
    float mx = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int i0 = sub; i0 < np; i0 += 32 * share) {
      const int mine = i0 + lane * share;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (mine < np) ml = p.part_ml[slot_of(mine) * R + row];
      const int here = min(32, (np - i0 + share - 1) / share);
      float x[kLoads][E];
      auto load = [&](int t0) {
#pragma unroll
        for (int t = 0; t < kLoads; ++t) {
          const int i = min(i0 + (t0 + t) * share, np - 1);
          const float* src = p.part_o + (slot_of(i) * R + row) * D + lane * E;
          if constexpr (E == 4) *reinterpret_cast<float4*>(x[t]) = *reinterpret_cast<const float4*>(src);
          else if constexpr (E == 2) *reinterpret_cast<float2*>(x[t]) = *reinterpret_cast<const float2*>(src);
          else x[t][0] = *src;
        }
      };
      load(0);
      float m2 = ml.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m2 = fmaxf(m2, __shfl_xor_sync(0xffffffffu, m2, o));
      m2 = fmaxf(m2, mx);
      const float ref = m2 == -INFINITY ? 0.f : m2, scale = ex2_weight(mx - ref), wt = ex2_weight(ml.x - ref);
      mx = m2;
      sum = sum * scale + wt * ml.y;  // (a lane's own pieces)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= scale;
      for (int t0 = 0; t0 < here; t0 += kLoads) {
        if (t0 > 0) load(t0);
#pragma unroll
        for (int t = 0; t < kLoads; ++t) {
          const float f = __shfl_sync(0xffffffffu, wt, (t0 + t) & 31);
          if (t0 + t < here) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(f, x[t][e], acc[e]);
          }
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (share > 1) {
      __syncthreads();  // the row before has been read
#pragma unroll
      for (int e = 0; e < E; ++e) sm_o[warp][lane * E + e] = acc[e];
      if (lane == 0) sm_ml[warp] = make_float2(mx, sum);
      __syncthreads();
      if (warp > 0) continue;
      mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) mx = fmaxf(mx, sm_ml[w].x);
      const float ref = mx == -INFINITY ? 0.f : mx;
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        const float f = ex2_weight(sm_ml[w].x - ref);
        sum = fmaf(f, sm_ml[w].y, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(f, sm_o[w][lane * E + e], acc[e]);
      }
    }
    const int a = d.i0 + row, hq = d.h * p.G + a % p.G;
    const int64_t tok = d.row0 + a / p.G;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = Cvt<T>::from_f(acc[e] * inv);
    char* dst = p.o + tok * p.o_rs + hq * p.o_hs + lane * E * 2;
    if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(y);
    else if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<uint32_t*>(y);
    else *reinterpret_cast<T*>(dst) = y[0];
    if (p.lse != nullptr && lane == 0)
      p.lse[tok * p.H + hq] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
  }
}

// Which kernel: this one pads a tile's rows to 16 and reads the cache once per tile;
// the tensor-core one pads them to 128 and runs at its softmax's pace.  Measured (us,
// this / that) at 16, 32 and 64 rows a K/V head:
//   D 128, 8 K/V heads    512 x 64 keys   61 / 206,   94 / 205,  172 / 206
//   (4 query heads each)  128 x 256       48 / 100,   70 / 100,  109 / 103
//                         64 x 2,048     106 / 138,  190 / 143,  358 / 144
//                         16 x 4,096      62 / 69,   102 / 72,   154 / 72
//                         1,024 x 1,024  718 / 1218, 1412 / 1208, 2791 / 1250
//   D 64, 2 K/V heads     512 x 64        25 / 52,    35 / 52,    47 / 52
//   (8 query heads each)  64 x 2,048      25 / 38,    33 / 39,    49 / 39
//                         16 x 4,096      21 / 26,    27 / 26,    31 / 26
//                         1,024 x 1,024  112 / 256,  191 / 257,  354 / 264
// (D 32 as D 64; one query head a K/V head as four.)  One tile of rows is better here
// throughout, and the rule's limit.  Two are better here too at D 64 and over short
// contexts, which the rule leaves aside: it goes by the rows alone.  The rows of a
// sequence are known on the device only; their mean decides.  A tensor-core tile holds
// whole tokens, so at most 128 heads a group.
bool few_rows(int64_t B, int64_t T, int64_t H, int64_t H_kv) {
  return T * (H / H_kv) <= R * B || H / H_kv > 128;
}
int64_t max_workers() { return (int64_t)num_sms() * kWarps; }
size_t ws_bytes(bool few, int D) {
  if (!few) return attn_paged_tc_workspace(D);
  const int64_t N = max_workers();
  return (size_t)N * sizeof(PagedDesc) / 16 * 16 + 16 + (size_t)(2 * N) * R * (8 + 4 * (size_t)D);
}

template <int D, typename T>
int launch_paged(const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p, cudaStream_t s) {
  auto kern = attn_paged_kernel<D, T>;
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63]) {
    SCREE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::smem(kPagedMaxSeqs)));
    attr_set[dev & 63] = true;
  }
  ProfScope prof(PROF_ATTN_FWD, s);
  SCREE_CUDA_TRY(launch_dependent(kern, dim3((unsigned)num_sms()), dim3(kThreads), Cfg<D>::smem(p.B), s, 1, tk, tv, p));
  count_launch();
  SCREE_CUDA_TRY(launch_dependent(attn_paged_join_kernel<D, T>, dim3((unsigned)max_workers() - 1),
                                  dim3(kJoinWarps * 32), 0, s, 1, p));
  count_launch();
  return SCREE_OK;
}

}  // namespace

int make_pool_map(CUtensorMap* map, const void* base, int64_t rows, int D, int box_rows, bool bf16) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) {
    set_last_error("cuTensorMapEncodeTiled is unavailable from the driver");
    return SCREE_ERR_CUDA;
  }
  cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  cuuint32_t box[2] = {(cuuint32_t)std::min(D, 64), (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1u, 1u};
  CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                   const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   D >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled failed (CUresult %d): pool of %lld rows, D=%d", (int)r,
                   (long long)rows, D);
    return SCREE_ERR_CUDA;
  }
  return SCREE_OK;
}

}  // namespace scree

using namespace scree;

extern "C" size_t scree_attn_fwd_paged_workspace_size(int64_t B, int64_t T, int64_t H, int64_t H_kv, int D) {
  if (B < 1 || T < 0 || H < 1 || H_kv < 1 || H % H_kv != 0) return 0;
  return ws_bytes(few_rows(B, T, H, H_kv), D);
}

extern "C" int scree_attn_fwd_paged(const void* q, int64_t q_rs, int64_t q_hs, const scree_paged_pools* pools,
                                    int64_t layer, const int32_t* table, const int32_t* lengths, int64_t S,
                                    int64_t M, int64_t P, int64_t page, const int32_t* slots,
                                    const void* offsets, int offs_is_i64, int64_t B, int64_t T, int64_t H,
                                    int D, int dtype, float scale, const uint64_t* mask, int64_t words,
                                    void* o, int64_t o_rs, int64_t o_hs, float* lse, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  SCREE_CHECK_ARG(pools != nullptr, "attn_fwd_paged: null pools");
  const int64_t H_kv = pools->H;
  SCREE_CHECK_ARG(H_kv >= 1 && H >= 1 && H % H_kv == 0 && H < 65536,
                  "attn_fwd_paged: query heads (%lld) must be a multiple of K/V heads (%lld)", (long long)H,
                  (long long)H_kv);
  SCREE_CHECK_ARG(B >= (T > 0) && B <= kPagedMaxSeqs && T >= 0 && T < (1ll << 31) && T * (H / H_kv) < (1ll << 31),
                  "attn_fwd_paged: bad sizes B=%lld (at most %d) T=%lld", (long long)B, kPagedMaxSeqs, (long long)T);
  if (D != 32 && D != 64 && D != 128) {
    set_last_error("attn_fwd_paged: head_dim %d unsupported (32, 64, 128)", D);
    return SCREE_ERR_UNSUPPORTED;
  }
  if (dtype != SCREE_F16 && dtype != SCREE_BF16) {
    set_last_error("attn_fwd_paged: fp16 / bf16 only");
    return SCREE_ERR_UNSUPPORTED;
  }
  SCREE_CHECK_ARG(pools->row_bytes == 2 * D, "attn_fwd_paged: pool rows of %lld bytes for head_dim %d",
                  (long long)pools->row_bytes, D);
  SCREE_CHECK_ARG(S >= 1 && M >= 1 && P >= 1 && P < (1ll << 30) && page >= kBox && page % kBox == 0 &&
                      M * page < (1ll << 31),
                  "attn_fwd_paged: bad cache sizes S=%lld M=%lld P=%lld page=%lld (a multiple of %d)",
                  (long long)S, (long long)M, (long long)P, (long long)page, kBox);
  SCREE_CHECK_ARG(layer >= 0 && layer < pools->L, "attn_fwd_paged: layer %lld of %lld", (long long)layer,
                  (long long)pools->L);
  const int64_t pool_rows = pools->L * P * H_kv * page;
  SCREE_CHECK_ARG(pool_rows < (1ll << 31), "attn_fwd_paged: pools of %lld rows are too large", (long long)pool_rows);
  SCREE_CHECK_ARG(mask == nullptr || (words >= 1 && words < (1 << 20)), "attn_fwd_paged: bad mask width");
  SCREE_CHECK_ARG(scale > 0.f, "attn_fwd_paged: scale %g must be positive", (double)scale);
  if (T == 0) return SCREE_OK;
  SCREE_CHECK_ARG(q && pools->k && pools->v && table && lengths && slots && offsets && o, "attn_fwd_paged: null pointer");
  SCREE_CHECK_ARG((uintptr_t)pools->k % 16 == 0 && (uintptr_t)pools->v % 16 == 0,
                  "attn_fwd_paged: pools must be 16-byte aligned");
  SCREE_CHECK_ARG((uintptr_t)q % 16 == 0 && q_rs % 8 == 0 && q_hs % 8 == 0,
                  "attn_fwd_paged: q must be 16-byte aligned with strides multiple of 8");
  SCREE_CHECK_ARG((uintptr_t)o % 16 == 0 && o_rs % 8 == 0 && o_hs % 8 == 0,
                  "attn_fwd_paged: output must be 16-byte aligned with strides multiple of 8");
  SCREE_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0, "attn_fwd_paged: workspace must be 16-byte aligned");
  SCREE_BIND_DEVICE(stream, q);
  const bool few = few_rows(B, T, H, H_kv);
  SCREE_CHECK_ARG(workspace_bytes >= ws_bytes(few, D), "attn_fwd_paged: workspace too small");
  const bool bf16 = dtype == SCREE_BF16;
  PagedParams p;
  p.q = (const char*)q;
  p.q_rs = q_rs * 2;
  p.q_hs = q_hs * 2;
  p.offs = offsets;
  p.is64 = offs_is_i64;
  p.slots = slots;
  p.table = table;
  p.lengths = lengths;
  p.mask = reinterpret_cast<const unsigned long long*>(mask);
  p.words = (int)words;
  p.B = (int)B;
  p.S = (int)S;
  p.M = (int)M;
  p.P = (int)P;
  p.page = (int)page;
  p.H = (int)H;
  p.Hkv = (int)H_kv;
  p.G = (int)(H / H_kv);
  p.T = T;
  p.layer_row = layer * P * H_kv * page;
  p.v = pools->v;
  p.sl2 = scale * 1.4426950408889634f;
  p.o = (char*)o;
  p.o_rs = o_rs * 2;
  p.o_hs = o_hs * 2;
  p.lse = lse;
  p.status = device_status_ptr();
  cudaStream_t s = (cudaStream_t)stream;
  if (!few) return attn_paged_tc(p, pools->k, pools->v, pool_rows, D, bf16, workspace, s);
  CUtensorMap tk, tv;
  int rc;
  if ((rc = make_pool_map(&tk, pools->k, pool_rows, D, kBox, bf16))) return rc;
  if ((rc = make_pool_map(&tv, pools->v, pool_rows, D, kBox, bf16))) return rc;
  char* w = (char*)workspace;
  const int64_t N = max_workers();
  p.desc = (PagedDesc*)w;
  w += N * sizeof(PagedDesc) / 16 * 16 + 16;
  p.part_ml = (float2*)w;
  p.part_o = (float*)(w + 2 * N * R * 8);
#define SCREE_PAGED_CASE(DD)                                                                         \
  if (D == DD)                                                                                       \
    return bf16 ? launch_paged<DD, __nv_bfloat16>(tk, tv, p, s) : launch_paged<DD, __half>(tk, tv, p, s);
  SCREE_PAGED_CASE(128)
  SCREE_PAGED_CASE(64)
  SCREE_PAGED_CASE(32)
#undef SCREE_PAGED_CASE
  return SCREE_ERR_UNSUPPORTED;
}
