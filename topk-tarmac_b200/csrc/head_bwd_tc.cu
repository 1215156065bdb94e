// head_bwd_tc.cu — gradients of masked attention with heads on the tensor
// memory (tcgen05), bf16. The operator is defined in head_attn.cu, its row
// statistics come from head_delta_kernel.
//
// Two kernels of one shape, each forming S and dP again tile by tile:
// * dq: a block owns 128 query rows (Q, dout staged once) and streams 64-key
//   tiles of K and V: S = Q K^T, dP = dout V^T, dS = P (dP - D) in registers
//   (a thread per query row), dQ += dS K.
// * dk, dv: a block owns 128 keys of a key head and streams 64-row tiles of Q
//   and dout of all query heads that share it: S^T = K Q^T, dP^T = V dout^T,
//   then dV += P^T dout and dK += dS^T Q. Shared heads add up in TMEM.
// P and dS return to TMEM as bf16, over the columns S and dP had, and are the
// A operands of the aggregates, so they never pass through shared memory.
// Roles of the 18 warps: two pairs of warpgroups that take tiles in turn (while
// one pair computes weights, the tensor core serves the other; each group of
// a pair has 32 of the 64 columns), one thread for the TMA ring, one thread
// that issues products. TMEM: accumulators in columns [0, 256), stage w (S,
// dP: 64 columns each) at 256 + 128 w. P and dS of columns 32 c .. 32 c + 31
// sit at column 32 c of their region, so that no group writes over what the
// other has still to read.
// Bound: 7 products for the 5 that the gradient needs (P is formed twice
// rather than added up across blocks with atomics, so two calls give the same
// bits) and two exponentials per pair.
// Every wait is bounded; one that runs out ends all roles and the rows
// concerned are written as NaN.
#include <type_traits>

#include "head_tc.cuh"

namespace tarmac {

int head_sm_count();

namespace {

constexpr int HB_THREADS = 576;
constexpr int HB_TMA_WARP = 16, HB_MMA_WARP = 17;
constexpr int HB_T = 64;  // streamed rows per tile
constexpr float HB_LOG2E = 1.4426950408889634f;

template <int DP>
struct HbPlan {
  static constexpr int OWN = 128 * DP * 2;   // an owned tile
  static constexpr int RUN = HB_T * DP * 2;  // a streamed tile
  static constexpr int NS = DP == 64 ? 6 : 4;
  static constexpr int STATS = 2 * HB_T * 4;  // lse2 and D of 64 rows
  static constexpr int SMEM = 2 * OWN + NS * (2 * RUN + STATS) + 1024;
};

template <int NS>
struct HbShared {
  uint64_t own_full, own_empty, full[NS], empty[NS], sfull[2], pfull[2], acc_full, acc_empty;
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
  w.start = p.q_start ? __ldg(p.q_start + w.b) : p.Nk - p.Nq;
  int len = p.key_len ? __ldg(p.key_len + w.b) : p.Nk;
  w.len = max(0, min(len, p.Nk));
  w.t0 = 0;
  if constexpr (DQ) {  // last tiles first: the most keys under the past rule
    w.x0 = (gr.tiles - 1 - t) * 128;
    int kend = w.len;
    if (p.peers == PEERS_PAST) {
      const int64_t last = (int64_t)w.start + min(p.Nq, w.x0 + 128) - 1;
      kend = (int)max((int64_t)0, min((int64_t)w.len, last + 1));
    }
    w.nper = w.n = cdiv(kend, HB_T);
  } else {  // first tiles first: the most queries
    w.x0 = t * 128;
    w.nper = 0;
    if (w.x0 < w.len) {
      int64_t i0 = 0;  // first query that sees a key of the tile
      if (p.peers == PEERS_PAST) i0 = max((int64_t)0, (int64_t)w.x0 - w.start);
      if (i0 < p.Nq) {
        w.t0 = (int)i0 / HB_T;
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
  using Plan = HbPlan<DP>;
  constexpr int NS = Plan::NS, OWN = Plan::OWN, RUN = Plan::RUN, SLOT = 2 * RUN;
  extern __shared__ unsigned char hb_raw[];
  __shared__ HbShared<NS> sh;
  const uint32_t base = (tc::smem_addr(hb_raw) + 1023u) & ~1023u;
  const uint32_t own = base, ring = base + 2 * OWN, stats = ring + NS * SLOT;
  const float* stats_ptr =
      reinterpret_cast<const float*>(hb_raw + (stats - tc::smem_addr(hb_raw)));
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tc::mbar_init(&sh.own_full, 1);
    tc::mbar_init(&sh.own_empty, 1);
    for (int s = 0; s < NS; ++s) {
      tc::mbar_init(&sh.full[s], 1);
      tc::mbar_init(&sh.empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      tc::mbar_init(&sh.sfull[w], 1);
      tc::mbar_init(&sh.pfull[w], 8);
    }
    tc::mbar_init(&sh.acc_full, 1);
    tc::mbar_init(&sh.acc_empty, 16);
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
      uint32_t c = 0, oc = 0;
      for (int k = 0;; ++k) {
        const int item = hb_next(k);
        if (item >= gr.items) break;
        const HbItem w = hb_item<DQ>(p, gr, item);
        if (w.n == 0) continue;
        if (!ws::wait(&sh.own_empty, (oc & 1) ^ 1, abort_flag)) goto tma_done;
        ++oc;
        ht::expect_tx(&sh.own_full, 2 * OWN);
        ht::tma_tile<DP, 128>(own, DQ ? &mq : &mk, &sh.own_full, w.h, w.x0, w.b);
        ht::tma_tile<DP, 128>(own + OWN, DQ ? &mg : &mv, &sh.own_full, w.h, w.x0, w.b);
        int g = 0, t = w.t0;
        for (int x = 0; x < w.n; ++x, ++c) {
          const int s = c % NS;
          if (!ws::wait(&sh.empty[s], ((c / NS) & 1) ^ 1, abort_flag)) goto tma_done;
          const uint32_t slot = ring + s * SLOT;
          ht::expect_tx(&sh.full[s], SLOT + (DQ ? 0 : Plan::STATS));
          const int head = DQ ? w.hk : w.hk * p.G + g;
          ht::tma_tile<DP, HB_T>(slot, DQ ? &mk : &mq, &sh.full[s], head, t * HB_T, w.b);
          ht::tma_tile<DP, HB_T>(slot + RUN, DQ ? &mv : &mg, &sh.full[s], head, t * HB_T, w.b);
          if constexpr (!DQ) {
            const float* st = p.delta + ((int64_t)w.b * p.H + head) * nqp + t * HB_T;
            ht::bulk_copy(stats + s * Plan::STATS, st, HB_T * 4, &sh.full[s]);
            ht::bulk_copy(stats + s * Plan::STATS + HB_T * 4, st + stat_plane, HB_T * 4,
                          &sh.full[s]);
          }
          if (++t == w.t0 + w.nper) {
            t = w.t0;
            ++g;
          }
        }
      }
    tma_done:
      if (*abort_flag) {  // the copies in flight land before the block ends
        if (oc) tc::mbar_wait(&sh.own_full, (oc - 1) & 1, 1u << 16);
        for (uint32_t x = c > (uint32_t)NS ? c - NS : 0; x < c; ++x)
          tc::mbar_wait(&sh.full[x % NS], (x / NS) & 1, 1u << 16);
      }
    }
    __syncwarp();
  } else if (warp == HB_MMA_WARP) {
    if (lane == 0) {
      const uint32_t id_s = tc::idesc_bf16(128, HB_T, false, false);
      const uint32_t id_o = tc::idesc_bf16(128, NKS * 16, false, true);
      const uint64_t da0 = ht::desc128(own, 16), db0 = ht::desc128(ring, 16);
      const uint64_t dn0 = ht::desc128(ring, HB_T * 128);  // streamed tile, MN-major
      uint32_t c = 0, oc = 0, pc[2] = {0, 0};
      // S and dP of streamed tile number x (counted over all items)
      auto issue = [&](uint32_t x) {
        const int s = x % NS, w = x & 1;
        if (!ws::wait(&sh.full[s], (x / NS) & 1, abort_flag)) return false;
        tc::fence_after_sync();
        const uint64_t db = db0 + (uint64_t)((s * SLOT) >> 4);
        const uint32_t d0 = tmem + 256 + w * 128;
        ht::issue_scores<NKS, HB_T>(d0, da0, db, id_s);
        ht::issue_scores<NKS, HB_T>(d0 + 64, da0 + (uint64_t)(OWN >> 4), db + (uint64_t)(RUN >> 4),
                                    id_s);
        tc::mma_commit(&sh.sfull[w]);
        return true;
      };
      for (int k = 0;; ++k) {
        const int item = hb_next(k);
        if (item >= gr.items) break;
        const HbItem it = hb_item<DQ>(p, gr, item);
        if (it.n == 0) continue;
        if (!ws::wait(&sh.own_full, oc & 1, abort_flag)) goto mma_done;
        if (!issue(c)) goto mma_done;
        if (it.n > 1 && !issue(c + 1)) goto mma_done;
        if (it.n <= 2) tc::mma_commit(&sh.own_empty);
        // the accumulators of the item before have been read
        if (!ws::wait(&sh.acc_empty, (oc & 1) ^ 1, abort_flag)) goto mma_done;
        ++oc;
        for (int t = 0; t < it.n; ++t) {
          const uint32_t x = c + t;
          const int s = x % NS, w = x & 1;
          if (!ws::wait(&sh.pfull[w], pc[w] & 1, abort_flag)) goto mma_done;
          ++pc[w];
          tc::fence_after_sync();
          const uint64_t dn = dn0 + (uint64_t)((s * SLOT) >> 4);
          const uint32_t a0 = tmem + 256 + w * 128;
          if constexpr (!DQ)  // dV += P^T dout
            ht::issue_aggregate<HB_T, 32>(tmem, a0, dn + (uint64_t)(RUN >> 4), id_o, t > 0);
          // dK += dS^T Q, or dQ += dS K
          ht::issue_aggregate<HB_T, 32>(tmem + (DQ ? 0 : DP), a0 + 64, dn, id_o, t > 0);
          tc::mma_commit(&sh.empty[s]);
          if (t + 2 < it.n) {
            if (!issue(x + 2)) goto mma_done;
            if (t + 3 == it.n) tc::mma_commit(&sh.own_empty);
          }
        }
        tc::mma_commit(&sh.acc_full);
        c += (uint32_t)it.n;
      }
      // the last commits land before the block ends
      for (uint32_t x = c > (uint32_t)NS ? c - NS : 0; x < c; ++x)
        if (!ws::wait(&sh.empty[x % NS], (x / NS) & 1, abort_flag)) break;
    mma_done:;
    }
    __syncwarp();
  } else {
    // ---------------- weights ----------------
    // group: stage w, columns [32 half, 32 half + 32) of its tiles
    const int w = warp >> 3, half = (warp >> 2) & 1, row = threadIdx.x & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + 256 + w * 128 + half * 32 + lane_off, t_dp = t_s + 64;
    const float c2 = p.scale * HB_LOG2E;
    const uint64_t cc2 = pack2(c2, c2);
    uint32_t c = 0, sc = 0, ac = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int item = hb_next(k);
      if (item >= gr.items) break;
      const HbItem it = hb_item<DQ>(p, gr, item);
      const int own_row = it.x0 + row;
      float lse2 = INFINITY, delta = 0.f;
      int jlim = 0, self = -1;
      const uint32_t* words = nullptr;
      if constexpr (DQ) {
        if (own_row < p.Nq) {
          const int64_t srow = ((int64_t)it.b * p.H + it.h) * nqp + own_row;
          lse2 = p.delta[srow];
          delta = p.delta[stat_plane + srow];
        }
        const int64_t pos = (int64_t)it.start + own_row;
        jlim = p.peers == PEERS_PAST ? (int)max((int64_t)0, min((int64_t)it.len, pos + 1)) : it.len;
        self = p.peers == PEERS_OTHERS && pos >= 0 && pos < p.Nk ? (int)pos : -1;
        if (p.bits)
          words = p.bits + it.b * p.bits_b + (int64_t)min(own_row, p.Nq - 1) * p.bits_w;
      }
      // keys: the query (as an index) that stands at this key's position
      const int64_t twin = (int64_t)own_row - it.start;
      int tt = it.t0;  // streamed tile inside its head
      for (int t = 0; t < it.n; ++t) {
        const uint32_t x = c + t;
        const int x0 = tt * HB_T + half * 32;  // first column of this group
        if (++tt == it.t0 + it.nper) tt = it.t0;
        if ((int)(x & 1) != w) continue;
        const int s = x % NS;
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
          const int64_t e = twin - x0;  // column of the twin
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
          // the statistics came with the tile
          if (!ht::warp_wait(&sh.full[s], (x / NS) & 1, abort_flag)) {
            ok = false;
            break;
          }
        }
        if (!ht::warp_wait(&sh.sfull[w], sc & 1, abort_flag)) {
          ok = false;
          break;
        }
        ++sc;
        tc::fence_after_sync();
        const float* st = stats_ptr + s * (Plan::STATS / 4) + half * 32;
        uint32_t sv[32];
        ht::tmem_ld(t_s, sv);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          uint64_t l0 = pack2(-lse2, -lse2), l1 = l0;
          if constexpr (!DQ) {
            const float4 q = *reinterpret_cast<const float4*>(st + e);
            l0 = pack2(-q.x, -q.y);
            l1 = pack2(-q.z, -q.w);
          }
          const float2 y0 = unpack2(
              ffma2(pack2(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), cc2, l0));
          const float2 y1 = unpack2(
              ffma2(pack2(__uint_as_float(sv[e + 2]), __uint_as_float(sv[e + 3])), cc2, l1));
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
        }
        uint32_t dv[32];
        ht::tmem_ld(t_dp, dv);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float de[4] = {delta, delta, delta, delta};
          if constexpr (!DQ) {
            const float4 q = *reinterpret_cast<const float4*>(st + HB_T + e);
            de[0] = q.x;
            de[1] = q.y;
            de[2] = q.z;
            de[3] = q.w;
          }
          float y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            y[u] = __uint_as_float(sv[e + u]) * (__uint_as_float(dv[e + u]) - de[u]);
          if (edge) {  // a masked pair's dP may be anything
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (!((seen >> (e + u)) & 1u)) y[u] = 0.f;
          }
          pk[e / 2] = tc::pack_bf16x2(y[0], y[1]);
          pk[e / 2 + 1] = tc::pack_bf16x2(y[2], y[3]);
        }
        ht::tmem_st(t_dp, pk);
        if constexpr (DQ) {
          const int k0 = x0 - half * 32;
          if (it.len < p.Nk && k0 + HB_T > it.len) {
            // K rows beyond the length may hold anything: dS is zero there,
            // the rows become zero too (S has been formed)
            if (!ht::warp_wait(&sh.full[s], (x / NS) & 1, abort_flag)) {
              ok = false;
              break;
            }
            const int r0 = it.len - k0;
            const uint32_t kt = ring + s * SLOT;
            for (int e = half * 128 + row; e < (HB_T - r0) * (DP / 8); e += 256) {
              const int r = r0 + e / (DP / 8), cc = e % (DP / 8);
              st_shared_zero16(kt + (uint32_t)((cc >> 3) * HB_T * 128 + r * 128 + (cc & 7) * 16));
            }
            tc::fence_async_smem();
          }
        }
        ht::st_wait();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) ws::arrive(&sh.pfull[w]);
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
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(DQ ? p.dq : (w ? p.dk : p.dv)) +
                           (((int64_t)it.b * own_n + own_row) * heads + it.h) * p.d;
      float f = DQ || w ? p.scale : 1.f;
      if (!ok) f = __int_as_float(0x7fffffff);
      const bool zero = it.n == 0 || (!DQ && own_row >= it.len);
      const int c0 = DQ ? (2 * w + half) * (DP / 4) : half * (DP / 2);
      const int c1 = c0 + (DQ ? DP / 4 : DP / 2);
      const uint32_t t_acc = tmem + lane_off + (DQ ? 0 : (w ? DP : 0));
      for (int cc = c0; cc < c1 && cc < p.d; cc += 16) {
        uint32_t o[16];
        if (it.n > 0) ht::tmem_ld(t_acc + cc, o);
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
      if (it.n > 0) {
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
  constexpr int SMEM = HbPlan<ht::width(NKS)>::SMEM;
  const void* fn = reinterpret_cast<const void*>(&head_bwd_tc_kernel<NKS, DQ>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  head_bwd_tc_kernel<NKS, DQ><<<grid, HB_THREADS, SMEM, s>>>(m[0], m[1], m[2], m[3], p, gr, nqp);
  return cudaGetLastError();
}

// bf16 rows on the 16-byte grid, at least 64 queries and 64 keys; the row
// statistics are in p.delta already. *done says whether the call was taken.
cudaError_t launch_head_bwd_tc(const HeadAttnParams& p, int64_t nqp, cudaStream_t s, bool* done) {
  *done = false;
  if (!p.vec || p.Nq < 64 || p.Nk < 64) return cudaSuccess;
  if ((int64_t)p.B * p.H * cdiv(p.Nq, 128) > (1 << 30) ||
      (int64_t)p.B * p.Hk * cdiv(p.Nk, 128) > (1 << 30))
    return cudaSuccess;
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
