// attn_paged_tc.cu — attention over a paged K/V cache for many rows per K/V head
// (trees of drafted tokens, chunks of a prompt), on tcgen05 tensor cores.
//
// The rows that share a K/V head (new token t, query head g of the group: row
// t G + g) are cut into tiles of 128 rows of whole tokens; a segment is a
// (sequence, K/V head, pair of tiles A and B), its units are tiles of 128 keys
// (and kLead more).
// As in attn_paged.cu all units laid end to end are cut into equal runs, one per
// CTA (one CTA per SM), and pieces of split segments are joined by a second
// kernel.  A and B share every K/V tile in shared memory, and the tensor core
// works on one while the softmax of the other runs.  Where a segment has but one
// tile of rows, A takes its even key tiles and B the odd ones, and A's warps join
// the two when they store the piece (one alone left half of the softmax warps idle:
// 64 x 2048 keys, 64 rows, 176 us against 148).
//
//   warp 8   finds the CTA's pieces, publishes their records through a ring,
//            loads Q and the K ring (TMA; a tile is 128 / box rows boxes, since
//            its pages lie anywhere; the lanes issue them side by side)
//   warp 10  the V ring, likewise
//   warp 9   one thread issues tcgen05.mma: S_X = Q_X K^T, O_X += P_X V
//   warps 0-3 / 4-7  softmax of tile A / B: a thread owns a row (a TMEM lane),
//            writes P (16-bit) over S in TMEM, rescales O when the maximum grew
//            by more than 2^8, and stores the piece
//
// TMEM columns: S_A [0,128), S_B [128,256), O_A [256,256+D), O_B [256+D,256+2D);
// P_X lies over the first 64 columns of S_X.  One thread issues all MMAs, which
// run in order, so S_X of the next tile may follow O_X += P_X V at once.
//
// Only tiles that reach the new tokens are masked.  There the softmax warps also
// clear, in shared memory, the V rows past the sequence's end and the infinities
// and NaN of drafted tokens' V (0 * NaN would reach rows that do not see them);
// rows that do see them get them back when the piece is stored.
//
// Bound: the chain scores -> softmax -> product of a pair of tiles, 2.3 us per 128
// keys (the tensor pipe is active 42% of the time, HBM at 38% of its peak), then the
// start and end of a run: finding its pieces, 7.5 us with the first tile; storing a
// piece, 4 us; the join, 14.  16 sequences of 4096 keys, 61 drafted tokens, 32 heads over
// 8 of 128: 113 us, 0.61 PFLOP/s of visible pairs; its bytes alone would take 54.  P is
// held in the queries' 16-bit type, as the tensor cores take it; l and O are fp32.
#include <algorithm>
#include "attn_paged.cuh"

namespace scree {
namespace {

constexpr int BM = 128, BN = 128;
// 8 softmax warps and a warpgroup of TMA (K), MMA, TMA (V) and one idle warp;
// registers as in attn_fwd.cu: 256 x 208 + 128 x 88 = 64,512 = 384 x 168.
constexpr int kThreads = 384, kWarps = kThreads / 32;
constexpr int kRegsSoftmax = 208, kRegsOther = 88;
constexpr int kRing = 4;                     // piece records in flight
constexpr int kReaders = 1 + 1 + 256;        // V warp, MMA thread, softmax threads
constexpr int kLanesPerTile = BN / kPagedKeys;

template <int D> struct Cfg {
  static constexpr int SWB = D >= 64 ? 128 : 64;  // swizzle span = bytes of a box row
  static constexpr int CHUNK = SWB / 2;
  static constexpr int NCHUNK = D / CHUNK;
  static constexpr uint32_t SWZ = SWB == 128 ? SW_128B : SW_64B;
  static constexpr int KSTAGES = D == 128 ? 2 : 3;
  static constexpr int VSTAGES = 3;
  static constexpr int Q_BYTES = BM * D * 2;
  static constexpr int KV_BYTES = BN * D * 2;
  static constexpr int OFF_K = 2 * Q_BYTES;
  static constexpr int OFF_V = OFF_K + KSTAGES * KV_BYTES;
  static constexpr int OFF_BAR = OFF_V + VSTAGES * KV_BYTES;
  static constexpr int OFF_END = OFF_BAR + 512;
  static constexpr int COL_S = 0, COL_O = 256;
};

struct Rec {  // a piece: key tiles [t0, t1) of a segment; t0 < 0: no more
  int32_t row0;      // packed row (token) of the first query
  int32_t ntok;      // tokens of the sequence from there on
  int32_t i0;        // its index among the sequence's new tokens
  int32_t c0, len;   // first new key, keys
  int32_t h, slot;
  int32_t t0, t1;
  int32_t part;      // partial slot, -1: the whole segment
  int32_t special;   // some drafted V is not finite
};

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// Key tiles of the rt-th row tile pair: up to its last row's last visible key.
__device__ __forceinline__ int64_t seg_tiles(const PagedParams& p, int64_t n, int64_t len, int64_t rt, int tok2) {
  const int64_t keys = p.mask != nullptr ? len : len - n + min(n, (rt + 1) * tok2);
  return (unsigned)(keys + BN - 1) / BN;
}
// A segment's units are kLead idle ones, which stand for what starting and storing
// a piece costs (5 us, where a tile takes 2.3), and its tiles.
constexpr int kLead = 4;
// Units of one K/V head of a sequence.
__device__ __forceinline__ int64_t head_units(const PagedParams& p, int64_t n, int64_t len, int tok2) {
  const int64_t rts = (unsigned)(n + tok2 - 1) / (unsigned)tok2;
  if (p.mask != nullptr) return rts * (kLead + (unsigned)(len + BN - 1) / BN);
  int64_t u = 0;
  for (int64_t r = 0; r < rts; ++r) u += kLead + seg_tiles(p, n, len, r, tok2);
  return u;
}

template <int D, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    attn_paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const PagedParams p, const int box) {
  using C = Cfg<D>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = make_idesc_f16(BM, BN, kBF16, false, false);
  constexpr uint32_t IDESC_O = make_idesc_f16(BM, D, kBF16, false, true);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tpt = BM / p.G, tok2 = 2 * tpt;  // tokens of a tile, of a pair
  // The sequences' prefix lies in the Q buffer for as long as it takes to find the
  // run's first sequence; from there on warp 8 walks the sequences in turn.
  int64_t* pre = reinterpret_cast<int64_t*>(smem);
  if (!paged_prefix<kWarps>(p, pre, [&](int64_t n, int64_t len) { return head_units(p, n, len, tok2) * p.Hkv; }))
    return;
  const int64_t U = pre[p.B], N = min((int64_t)gridDim.x, U), w = blockIdx.x;
  if (w >= N) {
    if (threadIdx.x == 0) p.desc[w].on = 0;
    return;
  }
  const PagedCut cut(U, N);
  const int64_t u0 = cut.start(w), u1 = cut.start(w + 1);
  const int b_first = paged_find(pre, p.B, u0);
  const int64_t pre_first = pre[b_first];
  __syncthreads();  // the prefix has been read: its memory becomes the Q buffer

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + C::KSTAGES;
  uint64_t* v_full = k_empty + C::KSTAGES;
  uint64_t* v_empty = v_full + C::VSTAGES;
  uint64_t* s_full = v_empty + C::VSTAGES;   // [2]
  uint64_t* p_half = s_full + 2;             // [2] first 64 keys of P_X
  uint64_t* p_full = p_half + 2;             // [2]
  uint64_t* pv_done = p_full + 2;            // [2]
  uint64_t* q_empty = pv_done + 2;
  uint64_t* o_empty = q_empty + 1;           // [2]
  uint64_t* ml_full = o_empty + 2;           // B's (m, l) of a split piece are there
  uint64_t* ml_free = ml_full + 1;           // and have been read
  uint64_t* mma_end = ml_free + 1;           // all MMAs are done
  uint64_t* rec_full = mma_end + 1;          // [kRing]
  uint64_t* rec_empty = rec_full + kRing;    // [kRing]
  Rec* ring = reinterpret_cast<Rec*>(rec_empty + kRing);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ring + kRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((1 + 2 * C::KSTAGES + 2 * C::VSTAGES + 8 + 6 + 2 * kRing) * 8 + kRing * sizeof(Rec) + 8 <= 512,
                "barrier area");
  const uint32_t sQ = smem_u32(smem), sK = smem_u32(smem + C::OFF_K), sV = smem_u32(smem + C::OFF_V);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(ml_full, 128);
    mbar_init(ml_free, 128);
    mbar_init(mma_end, 1);
    for (int i = 0; i < C::KSTAGES; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < C::VSTAGES; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_half[x], 128);
      mbar_init(&p_full[x], 128);
      mbar_init(&pv_done[x], 1);
      mbar_init(&o_empty[x], 128);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&rec_full[i], 1);
      mbar_init(&rec_empty[i], kReaders);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc<512>(tmem_slot);
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  fence_proxy_async_smem();  // the prefix was written through the generic proxy
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return paged_wait(p, bar, parity, abort_flag);
  };
  // Record of the CTA's k-th piece (t0 < 0: none left); false if the wait gave up.
  auto take = [&](int k, Rec& e) {
    if (!wait(&rec_full[k % kRing], k / kRing)) return false;
    e = ring[k % kRing];
    return true;
  };
  // A piece of one tile of rows and at least two of keys is split by keys between A and B.
  auto is_split = [&](const Rec& e) { return e.ntok <= tpt && e.t1 - e.t0 >= 2; };
  // Tile t's keys by one warp: lane l < 8 knows the page of key group 8 t + l (the
  // last valid group beyond the end: its keys are masked, its V cleared).
  auto tile_pages = [&](const Rec& e, int t) {
    if (lane >= kLanesPerTile) return 0;
    const int last = (e.len - 1) / kPagedKeys, per = box / kPagedKeys;
    const int g = min(t * kLanesPerTile + lane, last / per * per);
    return paged_page(p, e.slot, g);
  };
  auto load_tile = [&](const Rec& e, int t, int my_page, const CUtensorMap* map, uint8_t* dst, uint64_t* bar) {
    const int nbox = BN / box, per = box / kPagedKeys;
    const int b = lane % nbox, c = lane / nbox;
    const int page = __shfl_sync(0xffffffffu, my_page, b * per);
    if (lane == 0) mbar_expect_tx(bar, C::KV_BYTES);
    __syncwarp();
    if (c < C::NCHUNK) {
      const int last = (e.len - 1) / kPagedKeys;
      const int g = min(t * kLanesPerTile + b * per, last / per * per);
      const int row = (int)(p.layer_row + ((int64_t)page * p.Hkv + e.h) * p.page + (unsigned)g * kPagedKeys % (unsigned)p.page);
      tma_load_2d(dst + c * BN * C::SWB + b * box * C::SWB, map, bar, c * C::CHUNK, row);
    }
  };

  if (warp == 8) {
    // ------------------------------------------------------------ pieces, Q, K
    regs_dec<kRegsOther>();
    int kc = 0, k = 0, qc = 0, splits = 0;
    bool ok = true, was_split = false;
    int b = b_first, of = -1;
    int64_t pre_b = pre_first, hu = 0;  // units before sequence b; of one K/V head of sequence `of`
    for (int64_t u = u0; ok; ++k) {
      const int slot = k % kRing;
      if (k >= kRing && !(ok = __all_sync(0xffffffffu, wait(&rec_empty[slot], k / kRing - 1)))) break;
      Rec e;
      e.t0 = -1;
      while (u < u1) {
        int64_t q0 = 0, n = 0, len = 0;
        while (true) {  // the sequence of unit u (those after the run's first, in turn)
          q0 = load_offset(p.offs, p.is64, b);
          n = load_offset(p.offs, p.is64, b + 1) - q0;
          e.slot = p.slots[b];
          len = p.lengths[e.slot];
          if (of != b) hu = head_units(p, n, len, tok2);
          of = b;
          if (u < pre_b + hu * p.Hkv || b + 1 >= p.B) break;
          pre_b += hu * p.Hkv;
          ++b;
        }
        e.h = (int)udiv(u - pre_b, hu);
        int64_t s0 = pre_b + e.h * hu, rt = 0, tiles;
        if (p.mask != nullptr) {
          tiles = seg_tiles(p, n, len, 0, tok2);
          rt = udiv(u - s0, kLead + tiles);
          s0 += rt * (kLead + tiles);
        } else {
          while (u >= s0 + kLead + (tiles = seg_tiles(p, n, len, rt, tok2))) {
            s0 += kLead + tiles;
            ++rt;
          }
        }
        s0 += kLead;  // the unit of tile 0
        const int64_t s1 = s0 + tiles, from = max(u, s0), end = min(u1, s1);
        const bool start = u == u0;
        u = max(end, from);
        if (start && lane == 0) {
          const int w0 = (int)cut.of(s0);
          p.desc[w] = PagedDesc{u0 > s0 ? 1 : 0, w0, (int)cut.of(s1 - 1) - w0 + 1, (int)q0, e.h, (int)rt * tok2, (int)n};
        }
        if (end <= s0) continue;  // the run ends in the segment's lead
        e.i0 = (int)rt * tok2;
        e.row0 = (int)q0 + e.i0;
        e.ntok = (int)n - e.i0;
        e.c0 = (int)(len - n);
        e.len = (int)len;
        e.t0 = (int)(from - s0);
        e.t1 = (int)(end - s0);
        // A run has at most one piece that continues a segment and one that leaves one.
        e.part = from == s0 && end == s1 ? -1 : (int)(2 * w + (from > s0 ? 0 : 1));
        e.special = 0;
        break;
      }
      if (lane == 0) {
        ring[slot] = e;
        mbar_arrive(&rec_full[slot]);
      }
      __syncwarp();
      if (e.t0 < 0) break;
      if (k > 0 && !(ok = __all_sync(0xffffffffu, wait(q_empty, k - 1)))) break;
      // Q_B's place holds (m, l) at the end of a split piece.
      if (was_split && !(ok = __all_sync(0xffffffffu, wait(ml_free, splits - 1)))) break;
      was_split = is_split(e);
      splits += was_split;
      const bool two = e.ntok > tpt;
      if (lane == 0) {
        mbar_expect_tx(q_full, (two ? 2 : 1) * tpt * p.G * D * 2);
        for (int x = 0; x < (two ? 2 : 1); ++x)
#pragma unroll
          for (int c = 0; c < C::NCHUNK; ++c)
            tma_load_3d(smem + x * C::Q_BYTES + c * BM * C::SWB, &tm_q, q_full, c * C::CHUNK, e.h * p.G,
                        e.row0 + x * tpt);
      }
      __syncwarp();
      ++qc;
      int page = tile_pages(e, e.t0);
      for (int t = e.t0; t < e.t1; ++t, ++kc) {
        const int st = kc % C::KSTAGES;
        const int next = t + 1 < e.t1 ? tile_pages(e, t + 1) : 0;
        if (kc >= C::KSTAGES && !(ok = __all_sync(0xffffffffu, wait(&k_empty[st], kc / C::KSTAGES - 1)))) break;
        load_tile(e, t, page, &tm_k, smem + C::OFF_K + st * C::KV_BYTES, &k_full[st]);
        page = next;
      }
    }
    if (qc > 0) paged_drain(q_full, qc - 1);
    for (int i = max(0, kc - C::KSTAGES); i < kc; ++i) paged_drain(&k_full[i % C::KSTAGES], i / C::KSTAGES);
  } else if (warp == 10) {
    // ------------------------------------------------------------ V
    regs_dec<kRegsOther>();
    int vc = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      Rec e;
      ok = __all_sync(0xffffffffu, take(k, e));
      if (!ok) break;
      if (lane == 0) mbar_arrive(&rec_empty[k % kRing]);
      if (e.t0 < 0) break;
      int page = tile_pages(e, e.t0);
      for (int t = e.t0; t < e.t1; ++t, ++vc) {
        const int st = vc % C::VSTAGES;
        const int next = t + 1 < e.t1 ? tile_pages(e, t + 1) : 0;
        if (vc >= C::VSTAGES && !(ok = __all_sync(0xffffffffu, wait(&v_empty[st], vc / C::VSTAGES - 1)))) break;
        load_tile(e, t, page, &tm_v, smem + C::OFF_V + st * C::KV_BYTES, &v_full[st]);
        page = next;
      }
    }
    for (int i = max(0, vc - C::VSTAGES); i < vc; ++i) paged_drain(&v_full[i % C::VSTAGES], i / C::VSTAGES);
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    regs_dec<kRegsOther>();
    if (elect_one()) {
      auto kstep = [](int kk, int rows) -> uint32_t {
        const int e = kk * 16;
        return (uint32_t)(((e / C::CHUNK) * rows * C::SWB + (e % C::CHUNK) * 2) >> 4);
      };
      auto issue_s = [&](int x, int qx, int kpos) {
        const uint64_t dq = make_sdesc(sQ + qx * C::Q_BYTES, 16, 8 * C::SWB, C::SWZ);
        const uint64_t dk = make_sdesc(sK + (kpos % C::KSTAGES) * C::KV_BYTES, 16, 8 * C::SWB, C::SWZ);
        const uint32_t dt = tmem + C::COL_S + x * BN;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_ss(dt, dq + kstep(kk, BM), dk + kstep(kk, BN), IDESC_S, kk > 0 ? 1u : 0u);
        umma_commit(&s_full[x]);
      };
      // O_X += P_X V over keys [16 kk0, 16 kk1); V is the MN-major operand.
      auto issue_pv = [&](int x, bool first, int vpos, int kk0, int kk1) {
        const uint64_t dv = make_sdesc(sV + (vpos % C::VSTAGES) * C::KV_BYTES, BN * C::SWB, 8 * C::SWB, C::SWZ);
        const uint32_t pt = tmem + C::COL_S + x * BN, dt = tmem + C::COL_O + x * D;
#pragma unroll
        for (int kk = kk0; kk < kk1; ++kk)
          umma_f16_ts(dt, pt + kk * 8, dv + (uint32_t)((kk * 16 * C::SWB) >> 4), IDESC_O, (!first || kk > 0) ? 1u : 0u);
      };
      int kc = 0, vc = 0;
      int sc[2] = {0, 0};  // rounds of tile X so far
      int xc[2] = {0, 0};  // pieces of tile X so far
      bool ok = true;
      for (int k = 0; ok; ++k) {
        Rec e;
        if (!(ok = take(k, e))) break;
        mbar_arrive(&rec_empty[k % kRing]);
        if (e.t0 < 0) break;
        const int nt = e.t1 - e.t0, nx = e.ntok > tpt ? 2 : 1;
        if (!(ok = wait(q_full, k))) break;
        // O_X += P_X V of ring position vpos, round r of the piece.
        auto pv = [&](int x, int r, int vpos) {
          // O_X is overwritten once the piece before has been read out of it.
          if (r == 0 && xc[x] > 0 && !wait(&o_empty[x], xc[x] - 1)) return false;
          if (!wait(&p_half[x], sc[x] + r)) return false;
          tc_fence_after();
          issue_pv(x, r == 0, vpos, 0, BN / 32);
          if (!wait(&p_full[x], sc[x] + r)) return false;
          tc_fence_after();
          issue_pv(x, r == 0, vpos, BN / 32, BN / 16);
          umma_commit(&pv_done[x]);
          return true;
        };
        if (is_split(e)) {
          // S_A of tile 0 and S_B of tile 1, then each tile's product and S of the tile after next.
          auto s_of = [&](int j) {
            const int kn = kc + j;
            if (!wait(&k_full[kn % C::KSTAGES], kn / C::KSTAGES)) return false;
            tc_fence_after();
            issue_s(j & 1, 0, kn);
            umma_commit(&k_empty[kn % C::KSTAGES]);
            if (j + 1 == nt) umma_commit(q_empty);  // the last S product
            return true;
          };
          ok = s_of(0) && s_of(1);
          for (int j = 0; ok && j < nt; ++j) {
            const int vpos = vc + j;
            if (!(ok = wait(&v_full[vpos % C::VSTAGES], vpos / C::VSTAGES))) break;
            if (!(ok = pv(j & 1, j >> 1, vpos))) break;
            umma_commit(&v_empty[vpos % C::VSTAGES]);
            if (j + 2 < nt) ok = s_of(j + 2);
          }
          kc += nt;
          vc += nt;
          for (int x = 0; x < 2; ++x) {
            sc[x] += (nt + 1 - x) / 2;
            ++xc[x];
          }
          continue;
        }
        if (!(ok = wait(&k_full[kc % C::KSTAGES], kc / C::KSTAGES))) break;
        tc_fence_after();
        for (int x = 0; x < nx; ++x) issue_s(x, x, kc);
        umma_commit(&k_empty[kc % C::KSTAGES]);
        if (nt == 1) umma_commit(q_empty);
        for (int j = 0; ok && j < nt; ++j) {
          const int vpos = vc + j, kn = kc + j + 1;
          const bool more = j + 1 < nt;
          if (!(ok = wait(&v_full[vpos % C::VSTAGES], vpos / C::VSTAGES))) break;
          if (more && !(ok = wait(&k_full[kn % C::KSTAGES], kn / C::KSTAGES))) break;
          for (int x = 0; ok && x < nx; ++x) {
            if (!(ok = pv(x, j, vpos))) break;
            if (more) issue_s(x, x, kn);
          }
          if (!ok) break;
          if (j + 2 == nt) umma_commit(q_empty);  // the last S products have been issued
          umma_commit(&v_empty[vpos % C::VSTAGES]);
          if (more) umma_commit(&k_empty[kn % C::KSTAGES]);
        }
        kc += nt;
        vc += nt;
        for (int x = 0; x < nx; ++x) {
          sc[x] += nt;
          ++xc[x];
        }
      }
      umma_commit(mma_end);  // TMEM is freed behind the last product
      paged_drain(mma_end, 0);
    }
  } else if (warp == 11) {
    regs_dec<kRegsOther>();  // idle: only completes its warpgroup's register release
  } else {
    // ------------------------------------------------------------ softmax
    regs_inc<kRegsSoftmax>();
    const int x = warp >> 2;                // tile
    const int r = (warp & 3) * 32 + lane;   // row of the tile = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t col_s = lane_base + C::COL_S + x * BN, col_o = lane_base + C::COL_O + x * D;
    const float sl2 = p.sl2;
    const int tok = r / p.G, hq = r - tok * p.G;  // token of the tile, head of the group
    float2* ml_b = reinterpret_cast<float2*>(smem + C::Q_BYTES);  // (m, l) of B's rows of a split piece
    int sc = 0, sc_b = 0, vc = 0, splits = 0;  // rounds of this tile so far, of B's; key tiles; split pieces
    bool ok = true;
    for (int k = 0; ok; ++k) {
      Rec e;
      ok = __all_sync(0xffffffffu, take(k, e));
      if (!ok || e.t0 < 0) break;
      const bool split = is_split(e);
      const int tiles = e.t1 - e.t0;
      const int nt_b = split ? tiles / 2 : e.ntok > tpt ? tiles : 0;  // rounds of B
      const int nt = x == 1 ? nt_b : tiles - (split ? nt_b : 0);
      const int first_tok = split ? 0 : x * tpt;  // of this tile of rows
      const bool row_ok = r < tpt * p.G && first_tok + tok < e.ntok;
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < nt; ++j) {
        const int tile = split ? 2 * j + x : j;
        const int k0 = (e.t0 + tile) * BN;
        const bool edge = k0 + BN > e.c0;
        ok = wait(&s_full[x], sc + j);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (edge) {
          // V row r of the tile: cleared past the end; of a drafted token, without
          // its infinities and NaN.  Both tiles' warps do this, each before it lets
          // its product start; whoever clears an element has set the mark first.
          // The scores come first: their MMA is issued behind the products of two
          // tiles earlier (or of the pieces before), which have taken every V tile up
          // to there, so the place's last fill, three tiles back, has landed and the
          // parity names this tile's phase alone.
          const int vpos = vc + tile, st = vpos % C::VSTAGES;
          ok = wait(&v_full[st], vpos / C::VSTAGES);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          uint8_t* vrow = smem + C::OFF_V + st * C::KV_BYTES + r * C::SWB;
          if (k0 + r >= e.len) {
#pragma unroll
            for (int c = 0; c < C::NCHUNK; ++c)
              for (int i = 0; i < C::SWB / 16; ++i)
                *reinterpret_cast<uint4*>(vrow + c * BN * C::SWB + ((i + r) % (C::SWB / 16)) * 16) = make_uint4(0, 0, 0, 0);
          } else if (k0 + r >= e.c0) {
            for (int c = 0; c < C::NCHUNK; ++c)
              for (int i = 0; i < C::SWB / 16; ++i) {
                uint4* at = reinterpret_cast<uint4*>(vrow + c * BN * C::SWB + ((i + r) % (C::SWB / 16)) * 16);
                const uint4 v = *at;
                const uint4 f = make_uint4(nonfinite_halves<T>(v.x), nonfinite_halves<T>(v.y),
                                           nonfinite_halves<T>(v.z), nonfinite_halves<T>(v.w));
                if ((f.x | f.y | f.z | f.w) != 0) {
                  *reinterpret_cast<volatile int32_t*>(&ring[k % kRing].special) = 1;
                  __threadfence_block();
                  *at = make_uint4(v.x & ~f.x, v.y & ~f.y, v.z & ~f.z, v.w & ~f.w);
                }
              }
          }
          fence_proxy_async_smem();
        }
        float s[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld32(col_s + c * 32, *reinterpret_cast<float(*)[32]>(&s[c * 32]));
        tmem_wait_ld();
        tmem_regs_ready<BN>(s);
        if (edge) {
          const int i = e.i0 + first_tok + (row_ok ? tok : 0);
          const int64_t qrow = (int64_t)e.row0 + first_tok + (row_ok ? tok : 0);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const unsigned long long v = row_ok ? paged_visible<64>(p, qrow, i, k0 + hf * 64, e.c0, e.len) : 0ull;
#pragma unroll
            for (int c = 0; c < 64; ++c)
              if (!((c < 32 ? (uint32_t)v >> c : (uint32_t)(v >> 32) >> (c - 32)) & 1)) s[hf * 64 + c] = -INFINITY;
          }
        }
        float mx8[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) mx8[a] = fmaxf(s[a], s[8 + a]);
#pragma unroll
        for (int c = 16; c < BN; c += 16)
#pragma unroll
          for (int a = 0; a < 8; ++a) mx8[a] = fmax3(mx8[a], s[c + a], s[c + 8 + a]);
        const float mx = fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
        const float m_cand = mx * sl2;
        float alpha = 1.f;
        bool need = false;
        if (m_cand > m_used + 8.0f) {
          need = true;
          alpha = ex2_weight(m_used - m_cand);
          m_used = m_cand;
        }
        const float m_eff = m_used == -INFINITY ? 0.f : m_used;
        const uint64_t sl2x2 = f2_pack(sl2, sl2), negm2 = f2_pack(-m_eff, -m_eff);
        uint64_t rs4[4] = {0ull, 0ull, 0ull, 0ull};
        uint32_t pk[BN / 2];
        auto exp_pack = [&](int c0, int c1) {
#pragma unroll
          for (int c = c0; c < c1; c += 2) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(s[c], s[c + 1]), sl2x2, negm2), x0, x1);
            const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
            rs4[(c / 2) & 3] = f2_add(rs4[(c / 2) & 3], f2_pack(e0, e1));
            pk[c / 2] = pack2<T>(e0, e1);
          }
        };
        exp_pack(0, BN / 2);
        if (j >= 1) {
          // O_X += P_X V of the tile before must be complete before O_X is rescaled
          // and before P_X is overwritten; it is, as s_full covers it.
          ok = wait(&pv_done[x], sc + j - 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (__any_sync(0xffffffffu, need)) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tmem_ld32_sync(col_o + c * 32, o);
#pragma unroll
              for (int q = 0; q < 32; ++q) o[q] *= alpha;
              tmem_st32(col_o + c * 32, o);
            }
          }
        }
        tmem_st32u(col_s, *reinterpret_cast<uint32_t(*)[32]>(&pk[0]));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_half[x]);
        exp_pack(BN / 2, BN);
        tmem_st32u(col_s + 32, *reinterpret_cast<uint32_t(*)[32]>(&pk[32]));
        float ra, rb;
        f2_unpack(f2_add(f2_add(rs4[0], rs4[1]), f2_add(rs4[2], rs4[3])), ra, rb);
        l = l * alpha + (ra + rb);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[x]);
      }
      // ------------------------------------------------------------ the piece is done
      if (ok && nt > 0) {
        ok = wait(&pv_done[x], sc + nt - 1);
        ok = __all_sync(0xffffffffu, ok);
      }
      float fa = 1.f, fb = 0.f;  // weights of O_A and O_B in a split piece
      if (ok && split) {
        // B's warps leave (m, l) and go on; A's join the two and store the piece.
        // (B cannot come here again before A has read: its next O waits for that.)
        if (x == 1) {
          ml_b[r] = make_float2(m_used, l);
          mbar_arrive(ml_full);
        } else {
          ok = __all_sync(0xffffffffu, wait(ml_full, splits) && wait(&pv_done[1], sc_b + nt_b - 1));
          const float2 o = ml_b[r];
          fence_proxy_async_smem();
          mbar_arrive(ml_free);
          const float m = fmaxf(m_used, o.x), ref = m == -INFINITY ? 0.f : m;
          fa = ex2_weight(m_used - ref);
          fb = ex2_weight(o.x - ref);
          l = fa * l + fb * o.y;
          m_used = m;
        }
      }
      if (ok && nt > 0 && !(split && x == 1)) {
        tc_fence_after();
        const bool special = *reinterpret_cast<volatile int32_t*>(&ring[k % kRing].special) != 0;
        const int64_t qrow = (int64_t)e.row0 + first_tok + tok;
        const int head = e.h * p.G + hq;
        const bool whole = e.part < 0;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* orow = reinterpret_cast<T*>(p.o + qrow * p.o_rs + (int64_t)head * p.o_hs);
        float4* part = reinterpret_cast<float4*>(p.part_o) + ((int64_t)(whole ? 0 : e.part) * 2 + x) * (D / 4) * BM + r;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          tmem_ld32_sync(col_o + c * 32, o);
          if (split) {
            float ob[32];
            tmem_ld32_sync(col_o + D + c * 32, ob);
#pragma unroll
            for (int q = 0; q < 32; ++q) o[q] = fa * o[q] + fb * ob[q];
          }
          if (special && row_ok) {
            // The infinities and NaN that were taken out of V, for the keys that this row sees.
            for (int kk = max(e.c0, e.t0 * BN); kk < min(e.len, e.t1 * BN); ++kk) {
              if (!(paged_visible<16>(p, qrow, e.i0 + first_tok + tok, kk, e.c0, e.len) & 1)) continue;
              const int page = paged_page(p, e.slot, kk / kPagedKeys);
              const uint32_t* v = reinterpret_cast<const uint32_t*>(
                  reinterpret_cast<const T*>(p.v) +
                  (p.layer_row + ((int64_t)page * p.Hkv + e.h) * p.page + kk % p.page) * D + c * 32);
#pragma unroll
              for (int q = 0; q < 16; ++q) {
                const uint32_t wv = v[q], f = nonfinite_halves<T>(wv);
                const uint16_t lo = (uint16_t)wv, hi = (uint16_t)(wv >> 16);
                if (f & 0xFFFFu) o[2 * q] += Cvt<T>::to_f(*reinterpret_cast<const T*>(&lo));
                if (f >> 16) o[2 * q + 1] += Cvt<T>::to_f(*reinterpret_cast<const T*>(&hi));
              }
            }
          }
          if (row_ok && whole) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 y;
              y.x = pack2<T>(o[q * 8 + 0] * inv, o[q * 8 + 1] * inv);
              y.y = pack2<T>(o[q * 8 + 2] * inv, o[q * 8 + 3] * inv);
              y.z = pack2<T>(o[q * 8 + 4] * inv, o[q * 8 + 5] * inv);
              y.w = pack2<T>(o[q * 8 + 6] * inv, o[q * 8 + 7] * inv);
              *reinterpret_cast<uint4*>(orow + c * 32 + q * 8) = y;
            }
          } else if (row_ok) {
            // [column / 4][row]: a warp's stores are contiguous.
#pragma unroll
            for (int q = 0; q < 8; ++q)
              part[(int64_t)(c * 8 + q) * BM] = make_float4(o[q * 4], o[q * 4 + 1], o[q * 4 + 2], o[q * 4 + 3]);
          }
        }
        tc_fence_before();
        mbar_arrive(&o_empty[x]);  // O_X has been read
        if (split) mbar_arrive(&o_empty[1]);
        if (row_ok && !whole) p.part_ml[((int64_t)e.part * 2 + x) * BM + r] = make_float2(m_used, l);
        if (row_ok && whole && p.lse != nullptr)
          p.lse[qrow * p.H + head] = l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.69314718055994531f;
      }
      mbar_arrive(&rec_empty[k % kRing]);
      sc += nt;
      sc_b += nt_b;
      vc += tiles;
      splits += split;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

// Joins the pieces of a split segment (see attn_paged.cu).  Block (c - 1, y): the
// segment whose second worker is c, rows [32 y, 32 y + 32) of its two tiles; a lane
// is a row, a warp takes every eighth float4 of its columns.
constexpr int kJoinWarps = 8;
template <int D, typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_paged_tc_join_kernel(const PagedParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != 0) return;
  const PagedDesc d = p.desc[blockIdx.x + 1];
  if (!d.on || d.w0 != (int)blockIdx.x) return;
  const int np = d.np, tpt = BM / p.G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int x = blockIdx.y >> 2, r = (blockIdx.y & 3) * 32 + lane;
  const int tok = r / p.G, hq = r - tok * p.G;
  const int i = d.i0 + x * tpt + tok;  // new token of the sequence
  if (r >= tpt * p.G || i >= d.n) return;
  auto part_of = [&](int j) { return (int64_t)(j == 0 ? 2 * d.w0 + 1 : 2 * (d.w0 + j)) * 2 + x; };
  constexpr int E = D / 4 / kJoinWarps;  // float4 of a warp
  constexpr int J = 2;                   // pieces loaded side by side
  float mx = -INFINITY, sum = 0.f;
  float4 acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* po = reinterpret_cast<const float4*>(p.part_o);
#pragma unroll 1
  for (int j0 = 0; j0 < np; j0 += J) {
    float2 ml[J];
    float4 v[J][E];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t part = part_of(min(j0 + j, np - 1));
      ml[j] = j0 + j < np ? p.part_ml[part * BM + r] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) v[j][e] = po[(part * (D / 4) + warp * E + e) * BM + r];
    }
    const float m2 = fmaxf(mx, fmaxf(ml[0].x, ml[1].x));
    const float ref = m2 == -INFINITY ? 0.f : m2, scale = ex2_weight(mx - ref);
    mx = m2;
    sum *= scale;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[e].x *= scale;
      acc[e].y *= scale;
      acc[e].z *= scale;
      acc[e].w *= scale;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (j0 + j >= np) continue;
      const float f = ex2_weight(ml[j].x - ref);
      sum = fmaf(f, ml[j].y, sum);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        acc[e].x = fmaf(f, v[j][e].x, acc[e].x);
        acc[e].y = fmaf(f, v[j][e].y, acc[e].y);
        acc[e].z = fmaf(f, v[j][e].z, acc[e].z);
        acc[e].w = fmaf(f, v[j][e].w, acc[e].w);
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int head = d.h * p.G + hq;
  T* orow = reinterpret_cast<T*>(p.o + ((int64_t)d.row0 + i) * p.o_rs + (int64_t)head * p.o_hs) + warp * E * 4;
#pragma unroll
  for (int e = 0; e < E; ++e)
    *reinterpret_cast<uint2*>(orow + e * 4) = make_uint2(pack2<T>(acc[e].x * inv, acc[e].y * inv),
                                                         pack2<T>(acc[e].z * inv, acc[e].w * inv));
  if (warp == 0 && p.lse != nullptr)
    p.lse[((int64_t)d.row0 + i) * p.H + head] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
}

// Tensor map over q viewed as {D, H, T}: a box is the G heads of a K/V head of
// `tokens` tokens, which lie in shared memory as rows token * G + head.
int make_q_map(CUtensorMap* map, const PagedParams& p, int D, int tokens, bool bf16) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) {
    set_last_error("cuTensorMapEncodeTiled is unavailable from the driver");
    return SCREE_ERR_CUDA;
  }
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.H, (cuuint64_t)p.T};
  cuuint64_t strides[2] = {(cuuint64_t)p.q_hs, (cuuint64_t)p.q_rs};
  cuuint32_t box[3] = {(cuuint32_t)std::min(D, 64), (cuuint32_t)p.G, (cuuint32_t)tokens};
  cuuint32_t es[3] = {1u, 1u, 1u};
  CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                   const_cast<char*>(p.q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   D >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled failed (CUresult %d): q of %lld tokens, strides %lld, %lld bytes", (int)r,
                   (long long)p.T, (long long)p.q_rs, (long long)p.q_hs);
    return SCREE_ERR_CUDA;
  }
  return SCREE_OK;
}

template <int D, typename T>
int launch_tc(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p, int box,
              cudaStream_t s) {
  auto kern = attn_paged_tc_kernel<D, T>;
  // At least 120 KB, so that two CTAs (each holds all of TMEM) never share an SM.
  constexpr int smem = std::max(Cfg<D>::OFF_END + 1024, 120 * 1024);
  static_assert(smem <= 232448 && (kPagedMaxSeqs + 1) * 8 <= Cfg<D>::OFF_BAR, "shared memory");
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63]) {
    SCREE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set[dev & 63] = true;
  }
  ProfScope prof(PROF_ATTN_FWD, s);
  SCREE_CUDA_TRY(launch_dependent(kern, dim3((unsigned)num_sms()), dim3(kThreads), smem, s, 1, tq, tk, tv, p, box));
  count_launch();
  SCREE_CUDA_TRY(launch_dependent(attn_paged_tc_join_kernel<D, T>, dim3((unsigned)std::max(1, num_sms() - 1), 8),
                                  dim3(kJoinWarps * 32), 0, s, 1, p));
  count_launch();
  return SCREE_OK;
}

}  // namespace

size_t attn_paged_tc_workspace(int D) {
  const size_t N = (size_t)num_sms();
  return N * sizeof(PagedDesc) / 16 * 16 + 16 + 2 * N * 2 * BM * (8 + 4 * (size_t)D);
}

int attn_paged_tc(const PagedParams& in, const void* k, const void* v, int64_t pool_rows, int D, bool bf16,
                  void* workspace, cudaStream_t s) {
  PagedParams p = in;
  const size_t N = (size_t)num_sms();
  char* w = (char*)workspace;
  p.desc = (PagedDesc*)w;
  w += N * sizeof(PagedDesc) / 16 * 16 + 16;
  p.part_ml = (float2*)w;
  p.part_o = (float*)(w + 2 * N * 2 * BM * 8);
  // Boxes as tall as pages allow: rows of a box are consecutive in a page.
  int box = kPagedKeys;
  while (box < BN && p.page % (2 * box) == 0) box *= 2;
  CUtensorMap tq, tk, tv;
  int rc;
  if ((rc = make_q_map(&tq, p, D, BM / p.G, bf16))) return rc;
  if ((rc = make_pool_map(&tk, k, pool_rows, D, box, bf16))) return rc;
  if ((rc = make_pool_map(&tv, v, pool_rows, D, box, bf16))) return rc;
#define SCREE_TC_CASE(DD)                                                              \
  if (D == DD)                                                                         \
    return bf16 ? launch_tc<DD, __nv_bfloat16>(tq, tk, tv, p, box, s) : launch_tc<DD, __half>(tq, tk, tv, p, box, s);
  SCREE_TC_CASE(128)
  SCREE_TC_CASE(64)
  SCREE_TC_CASE(32)
#undef SCREE_TC_CASE
  return SCREE_ERR_UNSUPPORTED;
}

}  // namespace scree
