// head_bwd_tc.cu — gradients of masked attention with heads on the tensor
// memory (tcgen05), bf16. The operator is defined in head_attn.cu, its row
// statistics come from head_delta_kernel.
//
// Two kernels of one shape, each forming S and dP again tile by tile:
// * dq: a block owns 128 query rows (Q, dout staged once) and streams 128-key
//   tiles of K and V: S = Q K^T, dP = dout V^T, dS = P (dP - D) in registers
//   (rows are queries), dQ += dS K.
// * dk, dv: a block owns 128 keys of a key head and streams 128-row tiles of Q
//   and dout of all query heads that share it: S^T = K Q^T, dP^T = V dout^T,
//   dV += P^T dout, dK += dS^T Q. Shared heads add up in TMEM.
// P and dS return to TMEM as bf16, over the columns S and dP had, and are the
// A operands of the aggregates, so they never pass through shared memory.
// Roles of the 20 warps (two idle): 16 form the weights of one tile together (a thread
// has one row and 32 of the 128 columns), one thread feeds the TMA rings, one
// issues products. The two halves of a tile's work overlap the products of the
// other half: while P of tile t + 1 is formed the tensor core runs dK (or dQ)
// of tile t and dP of t + 1; while dS of tile t is formed it runs dV of t and
// S of t + 1 (dq: S is held twice and runs two tiles ahead).
// P and dS of columns 32 c .. 32 c + 31 sit at column 32 c of their region, so
// that no group of warps writes over what another has still to read.
// TMEM columns: dk, dv: dV, dK in [0, 256), S at 256, dP at 384; dq: dQ in
// [0, 128), S at 128 and 256, dP at 384.
// Bound: 7 products for the 5 that the gradient needs (P is formed twice
// rather than added up across blocks with atomics, so two calls give the same
// bits) and two exponentials per pair, 1024 clocks of the special-function
// unit per 128 x 128 tile against 256 d / 64 for a product. Measured on B200:
// 8192 causal rows of 16 heads on 4, d = 128: dk, dv 424 us, dq 308 us (365
// and 264 us for the products and hand-overs alone, in an earlier form), 939
// TFLOP/s of the five products' flops; 32 x 1024 rows of 8 heads, d = 64: 187
// and 155 us.
// Every wait is bounded; one that runs out ends all roles once their copies
// and products have landed, and every row is written, NaN or right.
#include <type_traits>

#include "head_tc.cuh"

namespace tarmac {

int head_sm_count();

namespace {

constexpr int HB_THREADS = 640;
// the issuing warps come first: older warps win the issue slots, and a late
// product stalls all others
constexpr int HB_MMA_WARP = 0, HB_TMA_WARP = 1, HB_W0 = 4;
constexpr int HB_T = 128;  // streamed rows per tile
constexpr float HB_LOG2E = 1.4426950408889634f;

// Rings: X is what S contracts with and the last aggregate reads again (Q, or
// K for dq), Y the other tensor (dout, or V for dq).
template <int DP, bool DQ>
struct HbPlan {
  static constexpr int TILE = 128 * DP * 2;  // bytes of 128 rows
  static constexpr int NX = DP == 64 || DQ ? 3 : 2;
  static constexpr int NY = 2;
  static constexpr int STATS = DQ ? 0 : 2 * HB_T * 4;  // lse2 and D of an X tile
  static constexpr int SMEM = (2 + NX + NY) * TILE + NX * STATS + 1024;
};

template <int NX, int NY>
struct HbShared {
  uint64_t own_full, own_empty, xfull[NX], xempty[NX], yfull[NY], yempty[NY];
  uint64_t sfull[2], dpfull, pfull, dsfull, acc_full, acc_empty, drain;
  uint32_t tmem;
  int abort_flag;
};

struct HbItem {
  int b, h, hk;  // h: query head (dq)
  int x0;        // first owned row
  int start, len;
  int t0, nper;  // dk, dv: first streamed tile, tiles per query head
  int n;         // streamed tiles
};

}  // namespace

struct HbGrid {
  int tiles, items, tile_major;
};

template <bool DQ>
__device__ __forceinline__ HbItem hb_item(const HeadAttnParams& p, const HbGrid& gr, int item) {
  HbItem w;
  const int heads = DQ ? p.H : p.Hk;
  const int bh = p.B * heads;
  const int t = gr.tile_major ? item / bh : item % gr.tiles;
  const int x = gr.tile_major ? item % bh : item / gr.tiles;
  w.h = x % heads;
  w.hk = DQ ? w.h / p.G : w.h;
  w.b = x / heads;
  w.start = ht::first_pos(p, w.b);
  w.len = ht::key_count(p, w.b);
  w.t0 = 0;
  if constexpr (DQ) {  // last tiles first: the most keys under the past rule
    w.x0 = (gr.tiles - 1 - t) * 128;
    w.nper = w.n = cdiv(ht::key_limit(p, w.start + min(p.Nq, w.x0 + 128) - 1, w.len), HB_T);
  } else {  // first tiles first: the most queries
    w.x0 = t * 128;
    w.nper = 0;
    if (w.x0 < w.len) {
      // first query that sees a key of the tile
      const int i0 = p.peers == PEERS_PAST ? max(0, w.x0 - w.start) : 0;
      if (i0 < p.Nq) {
        w.t0 = i0 / HB_T;
        w.nper = cdiv(p.Nq, HB_T) - w.t0;
      }
    }
    w.n = w.nper * p.G;
  }
  return w;
}

__device__ __forceinline__ int hb_next(int k) {
  const int g = (int)gridDim.x, x = (int)blockIdx.x;
  return k * g + ((k & 1) ? g - 1 - x : x);
}

// 32 x 32 bits across a warp: lane L's result holds in bit e what lane e's
// word had in bit L
__device__ __forceinline__ uint32_t warp_transpose(uint32_t x, int lane) {
  constexpr uint32_t M[5] = {0x0000ffffu, 0x00ff00ffu, 0x0f0f0f0fu, 0x33333333u, 0x55555555u};
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const int s = 16 >> i;
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, s);
    x = (lane & s) ? (((y >> s) & M[i]) | (x & ~M[i])) : ((x & M[i]) | ((y & M[i]) << s));
  }
  return x;
}

// DQ: own tiles Q and dout, streamed K and V; else own K and V, streamed Q
// and dout. m[0..3]: tensor maps of q, k, v, dout.
template <int NKS, bool DQ>
__global__ void __launch_bounds__(HB_THREADS, 1)
    head_bwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                       const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mg,
                       HeadAttnParams p, HbGrid gr, int64_t nqp) {
  constexpr int DP = ht::width(NKS);
  using Plan = HbPlan<DP, DQ>;
  constexpr int NX = Plan::NX, NY = Plan::NY, TILE = Plan::TILE;
  constexpr int NSB = DQ ? 2 : 1;                      // copies of S
  constexpr uint32_t COL_S = DQ ? 128 : 256, COL_DP = 384;
  extern __shared__ unsigned char hb_raw[];
  __shared__ HbShared<NX, NY> sh;
  const uint32_t base = (tc::smem_addr(hb_raw) + 1023u) & ~1023u;
  const uint32_t own = base, xr = base + 2 * TILE, yr = xr + NX * TILE, stats = yr + NY * TILE;
  const float* stats_ptr =
      reinterpret_cast<const float*>(hb_raw + (stats - tc::smem_addr(hb_raw)));
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tc::mbar_init(&sh.own_full, 1);
    tc::mbar_init(&sh.own_empty, 1);
    for (int s = 0; s < NX; ++s) {
      tc::mbar_init(&sh.xfull[s], 1);
      tc::mbar_init(&sh.xempty[s], 1);
    }
    for (int s = 0; s < NY; ++s) {
      tc::mbar_init(&sh.yfull[s], 1);
      tc::mbar_init(&sh.yempty[s], 1);
    }
    for (int s = 0; s < 2; ++s) tc::mbar_init(&sh.sfull[s], 1);
    tc::mbar_init(&sh.dpfull, 1);
    tc::mbar_init(&sh.pfull, 16);
    tc::mbar_init(&sh.dsfull, 16);
    tc::mbar_init(&sh.acc_full, 1);
    tc::mbar_init(&sh.acc_empty, 16);
    tc::mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    tc::mbar_init_fence();
  }
  if (warp == HB_MMA_WARP) tc::tmem_alloc(&sh.tmem, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sh.tmem;
  const int64_t stat_plane = (int64_t)p.B * p.H * nqp;

  if (warp == HB_TMA_WARP) {
    if (lane == 0) {
      uint32_t xc = 0, yc = 0, oc = 0;  // copies issued: X, Y and own tiles
      for (int k = 0;; ++k) {
        const int item = hb_next(k);
        if (item >= gr.items) break;
        if (ht::gives_up(ht::ROLE_LOADER, k)) {
          *abort_flag = 1;
          break;
        }
        const HbItem w = hb_item<DQ>(p, gr, item);
        if (w.n == 0) continue;
        if (!ws::wait(&sh.own_empty, (oc & 1) ^ 1, abort_flag)) goto tma_done;
        ++oc;
        ht::expect_tx(&sh.own_full, 2 * TILE);
        ht::tma_tile<DP, 128>(own, DQ ? &mq : &mk, &sh.own_full, w.h, w.x0, w.b);
        ht::tma_tile<DP, 128>(own + TILE, DQ ? &mg : &mv, &sh.own_full, w.h, w.x0, w.b);
        int g = 0, t = w.t0;
        for (int x = 0; x < w.n; ++x) {
          const int sx = xc % NX, sy = yc % NY;
          const int head = DQ ? w.hk : w.hk * p.G + g;
          if (!ws::wait(&sh.xempty[sx], ((xc / NX) & 1) ^ 1, abort_flag)) goto tma_done;
          ht::expect_tx(&sh.xfull[sx], TILE + Plan::STATS);
          ht::tma_tile<DP, HB_T>(xr + sx * TILE, DQ ? &mk : &mq, &sh.xfull[sx], head, t * HB_T,
                                 w.b);
          if constexpr (!DQ) {
            const float* st = p.delta + ((int64_t)w.b * p.H + head) * nqp + t * HB_T;
            ht::bulk_copy(stats + sx * Plan::STATS, st, HB_T * 4, &sh.xfull[sx]);
            ht::bulk_copy(stats + sx * Plan::STATS + HB_T * 4, st + stat_plane, HB_T * 4,
                          &sh.xfull[sx]);
          }
          ++xc;
          if (!ws::wait(&sh.yempty[sy], ((yc / NY) & 1) ^ 1, abort_flag)) goto tma_done;
          ht::expect_tx(&sh.yfull[sy], TILE);
          ht::tma_tile<DP, HB_T>(yr + sy * TILE, DQ ? &mv : &mg, &sh.yfull[sy], head, t * HB_T,
                                 w.b);
          ++yc;
          if (++t == w.t0 + w.nper) {
            t = w.t0;
            ++g;
          }
        }
      }
    tma_done:
      // the copies in flight land before the block ends, whoever gave up
      ht::drain_copies(&sh.own_full, 1, oc);
      ht::drain_copies(sh.xfull, NX, xc);
      ht::drain_copies(sh.yfull, NY, yc);
    }
    __syncwarp();
  } else if (warp == HB_MMA_WARP) {
    constexpr uint32_t id_s = tc::idesc_bf16(128, HB_T, false, false);
    constexpr uint32_t id_o = tc::idesc_bf16(128, NKS * 16, false, true);
    const uint64_t da0 = ht::desc128(own, 16), dx0 = ht::desc128(xr, 16),
                   dy0 = ht::desc128(yr, 16);
    const uint64_t nx0 = ht::desc128(xr, HB_T * 128), ny0 = ht::desc128(yr, HB_T * 128);
    const uint32_t b_own_full = tc::smem_addr(&sh.own_full), b_own_empty = tc::smem_addr(&sh.own_empty);
    const uint32_t b_xfull = tc::smem_addr(&sh.xfull[0]), b_xempty = tc::smem_addr(&sh.xempty[0]);
    const uint32_t b_yfull = tc::smem_addr(&sh.yfull[0]), b_yempty = tc::smem_addr(&sh.yempty[0]);
    const uint32_t b_sfull = tc::smem_addr(&sh.sfull[0]), b_dpfull = tc::smem_addr(&sh.dpfull);
    const uint32_t b_pfull = tc::smem_addr(&sh.pfull), b_dsfull = tc::smem_addr(&sh.dsfull);
    const uint32_t b_acc_full = tc::smem_addr(&sh.acc_full), b_acc_empty = tc::smem_addr(&sh.acc_empty);
    const bool leader = ht::elect_one();
    // next X tile to score, next X tile to aggregate, next Y tile of each
    ht::RingPos<NX> xs, xa;
    ht::RingPos<NY> ys, ya;
    uint32_t c = 0, oc = 0, sbuf = 0;
    bool ok = true;
    auto issue_s = [&] {
      ok = ok && ht::wait_at(b_xfull + 8 * xs.s, xs.ph, abort_flag);
      tc::fence_after_sync();
      if (ok && leader) {
        ht::issue_scores<NKS, HB_T>(tmem + COL_S + sbuf * 128, da0,
                                    dx0 + (uint64_t)(xs.s * (TILE >> 4)), id_s);
        ht::commit_at(b_sfull + 8 * sbuf);
      }
      __syncwarp();
      xs.next();
      if (NSB == 2) sbuf ^= 1;
    };
    auto issue_dp = [&] {
      ok = ok && ht::wait_at(b_yfull + 8 * ys.s, ys.ph, abort_flag);
      tc::fence_after_sync();
      if (ok && leader) {
        ht::issue_scores<NKS, HB_T>(tmem + COL_DP, da0 + (uint64_t)(TILE >> 4),
                                    dy0 + (uint64_t)(ys.s * (TILE >> 4)), id_s);
        ht::commit_at(b_dpfull);
        if (DQ) ht::commit_at(b_yempty + 8 * ys.s);  // V is read once
      }
      __syncwarp();
      ys.next();
    };
    for (int k = 0; ok; ++k) {
      const int item = hb_next(k);
      if (item >= gr.items) break;
      const int n = hb_item<DQ>(p, gr, item).n;
      if (n == 0) continue;
      ok = ht::wait_at(b_own_full, oc & 1, abort_flag);
      issue_s();
      issue_dp();
      if (DQ && n > 1) issue_s();
      if (n == 1 && ok && leader) ht::commit_at(b_own_empty);
      __syncwarp();
      // the accumulators of the item before have been read
      ok = ht::agree(ok && ht::wait_at(b_acc_empty, (oc & 1) ^ 1, abort_flag));
      ++oc;
      for (int t = 0; t < n && ok; ++t, ++c) {
        if constexpr (!DQ) {
          ok = ht::wait_at(b_pfull, c & 1, abort_flag);
          tc::fence_after_sync();
          if (ok && leader) {  // dV += P^T dout
            ht::issue_aggregate<HB_T, 32>(tmem, tmem + COL_S,
                                          ny0 + (uint64_t)(ya.s * (TILE >> 4)), id_o, t > 0);
            ht::commit_at(b_yempty + 8 * ya.s);
          }
          __syncwarp();
          ya.next();
          if (t + 1 < n) issue_s();
        }
        ok = ok && ht::wait_at(b_dsfull, c & 1, abort_flag);
        tc::fence_after_sync();
        if (ok && leader) {  // dK += dS^T Q, or dQ += dS K
          ht::issue_aggregate<HB_T, 32>(tmem + (DQ ? 0 : DP), tmem + COL_DP,
                                        nx0 + (uint64_t)(xa.s * (TILE >> 4)), id_o, t > 0);
          ht::commit_at(b_xempty + 8 * xa.s);
        }
        __syncwarp();
        xa.next();
        if (t + 1 < n) issue_dp();
        // the last S and dP are issued: the next item's own tiles may load
        if (t + 2 == n && ok && leader) ht::commit_at(b_own_empty);
        __syncwarp();
        if (DQ && t + 2 < n) issue_s();
        ok = ht::agree(ok);
      }
      if (ok && leader) ht::commit_at(b_acc_full);
      __syncwarp();
    }
    // the last commits land before the block ends
    for (uint32_t x = c > (uint32_t)NX ? c - NX : 0; x < c && ok; ++x)
      ok = ht::wait_at(b_xempty + 8 * (x % NX), (x / NX) & 1, abort_flag);
    if (oc && ok) ok = ht::wait_at(b_own_empty, (oc - 1) & 1, abort_flag);
    if (!ht::agree(ok)) ht::drain_products(&sh.drain, leader);
    __syncwarp();
  } else if (warp >= HB_W0) {
    // ---------------- weights ----------------
    // columns [32 part, 32 part + 32) of each tile
    const int part = (warp - HB_W0) >> 2, row = threadIdx.x & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + COL_S + part * 32 + lane_off;
    const uint32_t t_dp = tmem + COL_DP + part * 32 + lane_off;
    const float c2 = p.scale * HB_LOG2E;
    const uint64_t cc2 = pack2(c2, c2);
    uint32_t c = 0, ac = 0;
    bool ok = true;
    // warps that gave up walk on over the block's items and write NaN
    for (int k = 0;; ++k) {
      const int item = hb_next(k);
      if (item >= gr.items) break;
      if (ht::gives_up(ht::ROLE_WEIGHTS, k) && part == 1) {
        ok = false;
        *abort_flag = 1;
      }
      const HbItem it = hb_item<DQ>(p, gr, item);
      const int own_row = it.x0 + row;
      float nlse = -INFINITY, ndelta = 0.f;  // -lse2 and -D of a query row
      int jlim = 0, self = -1;
      const uint32_t* words = nullptr;
      if constexpr (DQ) {
        if (own_row < p.Nq) {
          const int64_t srow = ((int64_t)it.b * p.H + it.h) * nqp + own_row;
          nlse = p.delta[srow];
          ndelta = p.delta[stat_plane + srow];
        }
        jlim = ht::key_limit(p, it.start + own_row, it.len);
        self = p.peers == PEERS_OTHERS ? it.start + own_row : -1;
        if (p.bits)
          words = p.bits + it.b * p.bits_b + (int64_t)min(own_row, p.Nq - 1) * p.bits_w;
      }
      // keys: the query (as an index) that stands at this key's position
      const int twin = own_row - it.start;
      int tt = it.t0;  // streamed tile inside its head
      for (int t = 0; t < it.n && ok; ++t) {
        const uint32_t x = c + t;
        const int x0 = tt * HB_T + part * 32;  // first column of this thread
        if (++tt == it.t0 + it.nper) tt = it.t0;
        const int sx = x % NX;
        uint32_t seen = 0xffffffffu;
        bool edge;
        if constexpr (DQ) {
          edge = words || x0 + 32 > jlim || (self >= x0 && self < x0 + 32);
          if (edge) {
            uint32_t bits = 0xffffffffu;
            if (words) bits = (x0 >> 5) < p.bits_w ? __ldg(words + (x0 >> 5)) : 0u;
            seen = ht::key_word(x0, jlim, self, bits);
          }
        } else {
          const int e = twin - x0;  // column of the twin
          edge = p.bits || (p.peers == PEERS_PAST ? e > 0
                                                  : p.peers == PEERS_OTHERS && e >= 0 && e < 32);
          if (p.bits) {
            const int kw = (it.x0 >> 5) + (warp & 3), i = x0 + lane;
            uint32_t bits = 0u;
            if (i < p.Nq && kw < p.bits_w)
              bits = __ldg(p.bits + it.b * p.bits_b + (int64_t)i * p.bits_w + kw);
            seen = warp_transpose(bits, lane);
          }
          if (p.peers == PEERS_PAST)
            seen &= e <= 0 ? 0xffffffffu : (e >= 32 ? 0u : 0xffffffffu << e);
          else if (p.peers == PEERS_OTHERS && e >= 0 && e < 32)
            seen &= ~(1u << e);
        }
        // dk, dv: the statistics came with the Q tile; dq: its K tile may
        // have rows to clear
        const bool tail = DQ && it.len < p.Nk && x0 - part * 32 + HB_T > it.len;
        if (!DQ || tail) ok = ht::warp_wait(&sh.xfull[sx], (x / NX) & 1, abort_flag);
        if (ok)
          ok = ht::warp_wait(&sh.sfull[NSB == 2 ? (x & 1) : 0], (NSB == 2 ? x >> 1 : x) & 1,
                             abort_flag);
        if (!ok) break;
        tc::fence_after_sync();
        const float* st = stats_ptr + sx * (Plan::STATS / 4) + part * 32;
        uint32_t sv[32];
        ht::tmem_ld(t_s + (NSB == 2 ? (x & 1) * 128 : 0), sv);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          uint64_t l0 = pack2(nlse, nlse), l1 = l0;
          if constexpr (!DQ) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(st + e);
            l0 = q.x;
            l1 = q.y;
          }
          const float2 y0 = unpack2(ffma2(ht::pair(sv[e], sv[e + 1]), cc2, l0));
          const float2 y1 = unpack2(ffma2(ht::pair(sv[e + 2], sv[e + 3]), cc2, l1));
          sv[e] = __float_as_uint(tc::ex2_approx(y0.x));
          sv[e + 1] = __float_as_uint(tc::ex2_approx(y0.y));
          sv[e + 2] = __float_as_uint(tc::ex2_approx(y1.x));
          sv[e + 3] = __float_as_uint(tc::ex2_approx(y1.y));
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((seen >> e) & 1u)) sv[e] = 0u;
        }
        uint32_t pk[16];
        if constexpr (!DQ) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            pk[e] = tc::pack_bf16x2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1]));
          ht::tmem_st(t_s, pk);
          ht::st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) ws::arrive(&sh.pfull);
        }
        ok = ht::warp_wait(&sh.dpfull, x & 1, abort_flag);
        if (!ok) break;
        tc::fence_after_sync();
        uint32_t dv[32];
        ht::tmem_ld(t_dp, dv);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          uint64_t d0 = pack2(ndelta, ndelta), d1 = d0;
          if constexpr (!DQ) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(st + HB_T + e);
            d0 = q.x;
            d1 = q.y;
          }
          const float2 y0 = unpack2(
              ht::fmul2(ht::pair(sv[e], sv[e + 1]), ht::fadd2(ht::pair(dv[e], dv[e + 1]), d0)));
          const float2 y1 = unpack2(ht::fmul2(ht::pair(sv[e + 2], sv[e + 3]),
                                              ht::fadd2(ht::pair(dv[e + 2], dv[e + 3]), d1)));
          pk[e / 2] = tc::pack_bf16x2(y0.x, y0.y);
          pk[e / 2 + 1] = tc::pack_bf16x2(y1.x, y1.y);
        }
        if (edge) {  // a masked pair's dP may be anything
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (!((seen >> (2 * e)) & 1u)) pk[e] &= 0xffff0000u;
            if (!((seen >> (2 * e)) & 2u)) pk[e] &= 0x0000ffffu;
          }
        }
        ht::tmem_st(t_dp, pk);
        if (tail) {
          // K rows beyond the length may hold anything: dS is zero there, the
          // rows become zero too (S has been formed)
          const int r0 = it.len - (x0 - part * 32);
          const uint32_t kt = xr + sx * TILE;
          for (int e = threadIdx.x - HB_W0 * 32; e < (HB_T - r0) * (DP / 8); e += 512) {
            const int r = r0 + e / (DP / 8), cc = e % (DP / 8);
            st_shared_zero16(kt + (uint32_t)((cc >> 3) * HB_T * 128 + r * 128 + (cc & 7) * 16));
          }
          tc::fence_async_smem();
        }
        ht::st_wait();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) ws::arrive(&sh.dsfull);
      }
      c += (uint32_t)it.n;
      if (ok && it.n > 0) {
        ok = ht::warp_wait(&sh.acc_full, ac & 1, abort_flag);
        ++ac;
        tc::fence_after_sync();
      }
      // dq: each group stores a quarter of the columns; dk, dv: groups 0 and
      // 1 the halves of dv, 2 and 3 those of dk
      const int own_n = DQ ? p.Nq : p.Nk, heads = DQ ? p.H : p.Hk;
      const bool second = !DQ && part >= 2;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(DQ ? p.dq : (second ? p.dk : p.dv)) +
                           (((int64_t)it.b * own_n + own_row) * heads + it.h) * p.d;
      float f = DQ || second ? p.scale : 1.f;
      if (!ok) f = __int_as_float(0x7fffffff);
      const bool zero = it.n == 0 || (!DQ && own_row >= it.len);
      const int c0 = DQ ? part * (DP / 4) : (part & 1) * (DP / 2);
      const int c1 = c0 + (DQ ? DP / 4 : DP / 2);
      const uint32_t t_acc = tmem + lane_off + (second ? DP : 0);
      for (int cc = c0; cc < c1 && cc < p.d; cc += 16) {
        uint32_t o[16];
        if (it.n > 0 && ok) {
          ht::tmem_ld(t_acc + cc, o);
        } else {
#pragma unroll
          for (int u = 0; u < 16; ++u) o[u] = 0u;
        }
        if (own_row < own_n) {
#pragma unroll
          for (int u = 0; u < 16; u += 8) {
            if (cc + u >= p.d) break;
            uint4 q = make_uint4(0, 0, 0, 0);
            if (!zero) {
              q.x = tc::pack_bf16x2(__uint_as_float(o[u]) * f, __uint_as_float(o[u + 1]) * f);
              q.y = tc::pack_bf16x2(__uint_as_float(o[u + 2]) * f, __uint_as_float(o[u + 3]) * f);
              q.z = tc::pack_bf16x2(__uint_as_float(o[u + 4]) * f, __uint_as_float(o[u + 5]) * f);
              q.w = tc::pack_bf16x2(__uint_as_float(o[u + 6]) * f, __uint_as_float(o[u + 7]) * f);
            }
            *reinterpret_cast<uint4*>(out + cc + u) = q;
          }
        }
      }
      if (it.n > 0 && ok) {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) ws::arrive(&sh.acc_empty);
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == HB_MMA_WARP) tc::tmem_dealloc(tmem, 512);
}

template <int NKS, bool DQ>
static cudaError_t bwd_tc_go(const CUtensorMap* m, const HeadAttnParams& p, int64_t nqp,
                             cudaStream_t s) {
  const int sms = head_sm_count();
  HbGrid gr;
  gr.tiles = cdiv(DQ ? p.Nq : p.Nk, 128);
  const int64_t bh = (int64_t)p.B * (DQ ? p.H : p.Hk);
  gr.items = (int)(bh * gr.tiles);
  gr.tile_major = p.peers == PEERS_PAST && bh <= sms;
  const int grid = gr.items < sms ? gr.items : sms;
  constexpr int SMEM = HbPlan<ht::width(NKS), DQ>::SMEM;
  const void* fn = reinterpret_cast<const void*>(&head_bwd_tc_kernel<NKS, DQ>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  head_bwd_tc_kernel<NKS, DQ><<<grid, HB_THREADS, SMEM, s>>>(m[0], m[1], m[2], m[3], p, gr, nqp);
  return cudaGetLastError();
}

// Whether these kernels take a bf16 call: rows on the 16-byte grid, by the
// rules below.
bool head_bwd_tc_takes(const HeadAttnParams& p) {
  // Short sets leave the 128 x 128 tiles mostly empty; the kernels of
  // head_attn.cu were faster there. Measured, those against these, dq and dk,
  // dv together (us): 512 x 8 heads, d = 64: N = 64 138 / 220, N = 96 305 /
  // 234, N = 256 1175 / 591; 128 x 8 heads, d = 64, rows x keys: 32 x 512 171 /
  // 178, 40 x 512 213 / 181, 1024 x 40 406 / 334. d = 32, 512 x 4 heads:
  // N = 192 238 / 259, N = 224 347 / 261; d = 16, 256 x 4 heads: N = 192 88 /
  // 121, N = 256 142 / 121.
  const int longer = p.Nq > p.Nk ? p.Nq : p.Nk;
  if (!p.vec || p.Nk < 1 || p.Nq <= 32 || longer <= (p.d > 32 ? 64 : 192)) return false;
  if ((int64_t)p.B * p.H * cdiv(p.Nq, 128) > (1 << 30) ||
      (int64_t)p.B * p.Hk * cdiv(p.Nk, 128) > (1 << 30))
    return false;
  return head_map_ok(p.sq, p.B, p.Nq, p.H) && head_map_ok(p.sk, p.B, p.Nk, p.Hk) &&
         head_map_ok(p.sv, p.B, p.Nk, p.Hk) && head_map_ok(p.sg, p.B, p.Nq, p.H);
}

// The row statistics are in p.delta already. *done says whether the call was
// taken.
cudaError_t launch_head_bwd_tc(const HeadAttnParams& p, int64_t nqp, cudaStream_t s, bool* done) {
  *done = false;
  if (!head_bwd_tc_takes(p)) return cudaSuccess;
  CUtensorMap m[4];
  if (!head_tensor_map(&m[0], p.q, p.sq, p.B, p.Nq, p.H, p.d) ||
      !head_tensor_map(&m[1], p.k, p.sk, p.B, p.Nk, p.Hk, p.d) ||
      !head_tensor_map(&m[2], p.v, p.sv, p.B, p.Nk, p.Hk, p.d) ||
      !head_tensor_map(&m[3], p.g, p.sg, p.B, p.Nq, p.H, p.d))
    return cudaSuccess;
  *done = true;
  auto both = [&](auto nks) {
    constexpr int NKS = decltype(nks)::value;
    const cudaError_t e = bwd_tc_go<NKS, false>(m, p, nqp, s);
    return e != cudaSuccess ? e : bwd_tc_go<NKS, true>(m, p, nqp, s);
  };
  if (p.d <= 32) return both(std::integral_constant<int, 2>());
  if (p.d <= 64) return both(std::integral_constant<int, 4>());
  if (p.d <= 96) return both(std::integral_constant<int, 6>());
  return both(std::integral_constant<int, 8>());
}

}  // namespace tarmac
