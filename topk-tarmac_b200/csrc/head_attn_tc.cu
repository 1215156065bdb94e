// head_attn_tc.cu — forward masked attention with heads on the tensor memory
// (tcgen05), bf16. The operator is defined in head_attn.cu.
//
// A block owns two 128-row query tiles of one key head — two heads of the
// same rows, or neighbouring tiles — that share every staged K and V tile of
// 128 keys. Roles of its 20 warps (two idle):
// * warps 4..11 and 12..19: two warpgroups per tile, two threads per row with 64
//   of the 128 columns each. They read S from TMEM, mask, run the softmax in
//   base 2 and write P as bf16 to TMEM. The reference maximum moves, and O is
//   rescaled, only when a score of some row exceeds it by 2^8, which few tiles
//   do: one barrier with a vote settles the others, and only those that move
//   exchange row maxima through shared memory.
// * warp 1: one thread issues the TMA loads (Q once, K and V in a ring).
// * warp 0: one thread issues the products, alternating the tiles:
//   S_g = Q_g K^T, then O_g += P_g V with P from TMEM. While one tile is in
//   its softmax the tensor core serves the other.
// TMEM columns: S_g at 128 g (P_g over the columns of S_g that a group owns),
// O_g at 256 + DP g. A P_g with columns of its own, which lets S of the next
// key tile run under the exponentials, was no faster at d = 64 (32 x 8 heads of
// 1024 rows: 128 against 129 us) and slower with masks (204 against 184 us).
// Bound: of a tile's 1900 to 2000 clocks the special-function unit's 16
// exponentials per clock take 1024 (128 x 128 scores), the two products 256 d /
// 64 each; the rest is the chain from S to P and back, which two tiles in turn
// hide in part. Forming an eighth, a quarter or half of the exponentials as a
// polynomial on the FMA pipe gave 127, 131 and 142 us where this takes 127;
// P V in two halves, the first under the exponentials of the second, 132.
// Measured on B200: 2 x 8192 causal rows of 16 heads on 4, d = 128:
// 491 us, 1.12 PFLOP/s (557 us in a long run under the power limit); 32 x 1024
// rows of 8 heads, d = 64: 129 us, 533 TFLOP/s (its 268 M exponentials alone
// take 63 us at 1.8 GHz); 256 x 512 rows of 4 heads on 2, d = 64, with
// visibility words 180 us, without 143 us.
// Blocks are persistent, one per SM, and walk their items in
// alternating direction, so that under the past rule each gets long and short
// tiles.
// Every wait is bounded; one that runs out raises a flag that ends all roles
// once their copies and products have landed, and every row is written, NaN or
// right.
#include "head_tc.cuh"

namespace tarmac {

namespace {

constexpr int HT_THREADS = 640;
// the issuing warps come first: older warps win the issue slots, and a late
// product stalls all others
constexpr int HT_MMA_WARP = 0, HT_TMA_WARP = 1, HT_W0 = 4;
constexpr int HT_KEYS = 128;
constexpr float HT_LOG2E = 1.4426950408889634f;
constexpr float HT_LN2 = 0.6931471805599453f;
constexpr float HT_MOVE = 8.0f;  // exponent units

template <int DP>
struct HtPlan {
  static constexpr int TILE = 128 * DP * 2;                 // bytes of 128 rows
  static constexpr int NS = DP == 64 ? 4 : 2;               // ring stages (K and V)
  static constexpr int SMEM = 2 * TILE + NS * 2 * TILE + 1024;
};

template <int NS>
struct HtShared {
  uint64_t qfull, qempty, kfull[NS], vfull[NS], empty[NS], sfull[2], pfull[2], odone[2], drain;
  uint32_t tmem;
  int abort_flag;
  float top[2][2][2][128];  // row maxima: tile, step parity, group, row
  float sum[2][2][128];     // row sums: tile, group, row
};

struct HtItem {
  int b, hk, n;       // n: key tiles that either tile needs
  int tile[2], g[2];  // query tile and head inside the group (tile -1: none)
  int nt[2];          // key tiles of each
};

}  // namespace

struct HtGrid {
  int nqt, pairs, items, pair_major;
};

// item -> its two tiles. Tiles run from the last to the first, as the last
// have the most keys under the past rule.
__device__ __forceinline__ HtItem ht_item(const HeadAttnParams& p, const HtGrid& gr, int item) {
  HtItem w;
  const int bh = p.B * p.Hk;
  const int pair = gr.pair_major ? item / bh : item % gr.pairs;
  const int x = gr.pair_major ? item % bh : item / gr.pairs;
  w.hk = x % p.Hk;
  w.b = x / p.Hk;
  const int start = ht::first_pos(p, w.b), len = ht::key_count(p, w.b);
  w.n = 0;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int unit = 2 * pair + u;
    w.tile[u] = -1;
    w.g[u] = 0;
    w.nt[u] = 0;
    if (unit >= gr.nqt * p.G) continue;
    w.tile[u] = gr.nqt - 1 - unit / p.G;
    w.g[u] = unit % p.G;
    w.nt[u] = cdiv(ht::key_limit(p, start + min(p.Nq, (w.tile[u] + 1) * 128) - 1, len), HT_KEYS);
    w.n = max(w.n, w.nt[u]);
  }
  return w;
}

// items of this block, in alternating direction
__device__ __forceinline__ int ht_next(int k) {
  const int g = (int)gridDim.x, x = (int)blockIdx.x;
  return k * g + ((k & 1) ? g - 1 - x : x);
}

template <int NKS>
__global__ void __launch_bounds__(HT_THREADS, 1)
    head_fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                       const __grid_constant__ CUtensorMap mv, HeadAttnParams p, HtGrid gr) {
  constexpr int DP = ht::width(NKS);
  using Plan = HtPlan<DP>;
  constexpr int NS = Plan::NS, TILE = Plan::TILE;
  extern __shared__ unsigned char ht_raw[];
  __shared__ HtShared<NS> sh;
  // 1024-byte grid of the swizzle
  const uint32_t base = (tc::smem_addr(ht_raw) + 1023u) & ~1023u;
  const uint32_t qa = base, kva = base + 2 * TILE;
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tc::mbar_init(&sh.qfull, 1);
    tc::mbar_init(&sh.qempty, 1);
    for (int s = 0; s < NS; ++s) {
      tc::mbar_init(&sh.kfull[s], 1);
      tc::mbar_init(&sh.vfull[s], 1);
      tc::mbar_init(&sh.empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      tc::mbar_init(&sh.sfull[w], 1);
      tc::mbar_init(&sh.pfull[w], 8);
      tc::mbar_init(&sh.odone[w], 1);
    }
    tc::mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    tc::mbar_init_fence();
  }
  if (warp == HT_MMA_WARP) tc::tmem_alloc(&sh.tmem, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sh.tmem;

  if (warp == HT_TMA_WARP) {
    if (lane == 0) {
      uint32_t kc = 0, qc = 0;  // copies issued: K and V tiles, Q tiles
      for (int k = 0;; ++k) {
        const int item = ht_next(k);
        if (item >= gr.items) break;
        if (ht::gives_up(ht::ROLE_LOADER, k)) {
          *abort_flag = 1;
          break;
        }
        const HtItem w = ht_item(p, gr, item);
        if (!ws::wait(&sh.qempty, (k & 1) ^ 1, abort_flag)) goto tma_done;
        const int both = w.tile[1] >= 0;
        ht::expect_tx(&sh.qfull, (uint32_t)(TILE * (1 + both)));
        for (int u = 0; u <= both; ++u)
          ht::tma_tile<DP, 128>(qa + u * TILE, &mq, &sh.qfull, w.hk * p.G + w.g[u],
                                w.tile[u] * 128, w.b);
        ++qc;
        for (int t = 0; t < w.n; ++t, ++kc) {
          const int s = kc % NS;
          if (!ws::wait(&sh.empty[s], ((kc / NS) & 1) ^ 1, abort_flag)) goto tma_done;
          const uint32_t slot = kva + s * 2 * TILE;
          ht::expect_tx(&sh.kfull[s], TILE);
          ht::tma_tile<DP, 128>(slot, &mk, &sh.kfull[s], w.hk, t * HT_KEYS, w.b);
          ht::expect_tx(&sh.vfull[s], TILE);
          ht::tma_tile<DP, 128>(slot + TILE, &mv, &sh.vfull[s], w.hk, t * HT_KEYS, w.b);
        }
      }
    tma_done:
      // the copies in flight land before the block ends, whoever gave up
      ht::drain_copies(&sh.qfull, 1, qc);
      ht::drain_copies(sh.kfull, NS, kc);
      ht::drain_copies(sh.vfull, NS, kc);
    }
    __syncwarp();
  } else if (warp == HT_MMA_WARP) {
    constexpr uint32_t id_s = tc::idesc_bf16(128, HT_KEYS, false, false);
    constexpr uint32_t id_o = tc::idesc_bf16(128, NKS * 16, false, true);
    const uint64_t dq0 = ht::desc128(qa, 16), dk0 = ht::desc128(kva, 16);
    const uint64_t dv0 = ht::desc128(kva + TILE, 128 * 128);
    const uint32_t b_qfull = tc::smem_addr(&sh.qfull), b_qempty = tc::smem_addr(&sh.qempty);
    const uint32_t b_kfull = tc::smem_addr(&sh.kfull[0]), b_vfull = tc::smem_addr(&sh.vfull[0]);
    const uint32_t b_empty = tc::smem_addr(&sh.empty[0]), b_sfull = tc::smem_addr(&sh.sfull[0]);
    const uint32_t b_pfull = tc::smem_addr(&sh.pfull[0]), b_odone = tc::smem_addr(&sh.odone[0]);
    const bool leader = ht::elect_one();
    ht::RingPos<NS> kr, vr;  // next K tile to score, next V tile to aggregate
    uint32_t pc0 = 0, pc1 = 0, kc = 0;
    bool ok = true;
    auto scores = [&](int w) {  // S_w from the K tile at kr
      if (ok && leader) {
        ht::issue_scores<NKS, 128>(tmem + w * 128, dq0 + (uint64_t)(w * (TILE >> 4)),
                                   dk0 + (uint64_t)(kr.s * (2 * TILE >> 4)), id_s);
        ht::commit_at(b_sfull + 8 * w);
      }
      __syncwarp();
    };
    auto wait_k = [&] {
      ok = ok && ht::wait_at(b_kfull + 8 * kr.s, kr.ph, abort_flag);
      tc::fence_after_sync();
    };
    for (int k = 0; ok; ++k) {
      const int item = ht_next(k);
      if (item >= gr.items) break;
      const HtItem it = ht_item(p, gr, item);
      const int n = it.n, n0 = it.nt[0], n1 = it.nt[1];
      ok = ht::wait_at(b_qfull, k & 1, abort_flag);
      if (n > 0) {
        wait_k();
        if (n0 > 0) scores(0);
        if (n1 > 0) scores(1);
        kr.next();
      }
      if (n <= 1 && ok && leader) ht::commit_at(b_qempty);
      ok = ht::agree(ok);
      for (int t = 0; t < n && ok; ++t, ++kc) {
        ok = ht::wait_at(b_vfull + 8 * vr.s, vr.ph, abort_flag);
        if (t + 1 < n) wait_k();
        const uint64_t dv = dv0 + (uint64_t)(vr.s * (2 * TILE >> 4));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int nw = w ? n1 : n0;
          if (t >= nw) continue;
          ok = ok && ht::wait_at(b_pfull + 8 * w, (w ? pc1 : pc0) & 1, abort_flag);
          if (w) ++pc1; else ++pc0;
          tc::fence_after_sync();
          if (ok && leader) {
            ht::issue_aggregate<HT_KEYS, 64>(tmem + 256 + w * DP, tmem + w * 128, dv, id_o, t > 0);
            if (t + 1 == nw) ht::commit_at(b_odone + 8 * w);
          }
          __syncwarp();
          if (t + 1 < nw) scores(w);
        }
        if (ok && leader) {
          ht::commit_at(b_empty + 8 * vr.s);
          if (t + 2 == n) ht::commit_at(b_qempty);
        }
        ok = ht::agree(ok);
        vr.next();
        if (t + 1 < n) kr.next();
      }
    }
    // the last commits land before the block ends
    for (uint32_t c = kc > (uint32_t)NS ? kc - NS : 0; c < kc && ok; ++c)
      ok = ht::wait_at(b_empty + 8 * (c % NS), (c / NS) & 1, abort_flag);
    if (!ht::agree(ok)) ht::drain_products(&sh.drain, leader);
    __syncwarp();
  } else if (warp >= HT_W0) {
    // ---------------- softmax groups ----------------
    // tile w of the item, columns [64 half, 64 half + 64) of its key tiles
    const int w = (warp - HT_W0) >> 3, half = ((warp - HT_W0) >> 2) & 1, row = threadIdx.x & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + w * 128 + half * 64 + lane_off;
    const uint32_t t_o = tmem + 256 + w * DP + half * (DP / 2) + lane_off;
    const int c_lo = half * (DP / 2), c_n = max(0, min(DP / 2, p.d - c_lo));  // columns of O
    const float c2 = p.scale * HT_LOG2E;
    auto pair_sync = [&] { asm volatile("bar.sync %0, 256;" ::"r"(1 + w) : "memory"); };
    // does any of the pair's threads say so? (a barrier)
    auto pair_any = [&](bool x) {
      uint32_t r;
      asm volatile(
          "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, %2, 256, p;\n"
          "selp.u32 %0, 1, 0, q;\n}\n"
          : "=r"(r)
          : "r"((uint32_t)x), "r"(1 + w)
          : "memory");
      return r != 0;
    };
    uint32_t kc = 0, sc = 0, oc = 0;
    bool ok = true;
    // a group that gave up keeps meeting its partner: it skips the bounded
    // waits, never the barrier
    for (int k = 0;; ++k) {
      const int item = ht_next(k);
      if (item >= gr.items) break;
      const HtItem it = ht_item(p, gr, item);
      if (ht::gives_up(ht::ROLE_WEIGHTS, k) && half) {
        ok = false;
        *abort_flag = 1;
      }
      const uint32_t kc0 = kc;
      kc += (uint32_t)it.n;
      const int tile = w ? it.tile[1] : it.tile[0], nt = w ? it.nt[1] : it.nt[0];
      if (tile < 0) continue;
      const int h = it.hk * p.G + (w ? it.g[1] : it.g[0]);
      const int i = tile * 128 + row;
      const int pos = ht::first_pos(p, it.b) + i, len = ht::key_count(p, it.b);
      const int jlim = ht::key_limit(p, pos, len);
      const int self = p.peers == PEERS_OTHERS ? pos : -1;
      const uint32_t* words =
          p.bits ? p.bits + it.b * p.bits_b + (int64_t)min(i, p.Nq - 1) * p.bits_w : nullptr;
      float mref = -INFINITY;  // reference maximum in exponent units
      float l = 0.f;           // this group's part of the sum
      // the visibility words of the next key tile are on their way while this
      // one is worked on
      auto fetch_words = [&](int t, uint32_t (&bits)[2]) {
        const int j = t * (HT_KEYS / 32) + half * 2;
#pragma unroll
        for (int x = 0; x < 2; ++x)
          bits[x] = words ? (j + x < p.bits_w ? __ldg(words + j + x) : 0u) : 0xffffffffu;
      };
      uint32_t bits[2];
      fetch_words(0, bits);
      for (int t = 0; t < nt; ++t) {
        const int k0 = t * HT_KEYS + half * 64;
        const bool edge = words || k0 + 64 > jlim || (self >= k0 && self < k0 + 64);
        uint32_t seen[2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
          seen[x] = edge ? ht::key_word(k0 + 32 * x, jlim, self, bits[x]) : 0xffffffffu;
        if (words) fetch_words(t + 1, bits);
        if (ok) ok = ht::warp_wait(&sh.sfull[w], sc & 1, abort_flag);
        ++sc;
        tc::fence_after_sync();
        uint32_t s[64];
        ht::tmem_ld(t_s, s);
        if (edge) {
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (!((seen[e >> 5] >> (e & 31)) & 1u)) s[e] = 0xff800000u;  // -inf
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 64; x += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            mx[u] = max3f(mx[u], __uint_as_float(s[x + 2 * u]), __uint_as_float(s[x + 2 * u + 1]));
        const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (t == 0 ||
            pair_any(mine * c2 > mref + HT_MOVE || (mref == -INFINITY && mine != -INFINITY))) {
          sh.top[w][t & 1][half][row] = mine;
          pair_sync();
          const float m2 = fmaxf(mine, sh.top[w][t & 1][half ^ 1][row]) * c2;
          float alpha = 1.f;
          const bool move = m2 > mref + HT_MOVE || (mref == -INFINITY && m2 != -INFINITY);
          if (move) {
            alpha = tc::ex2_approx(mref - m2);
            l *= alpha;
            mref = m2;
          }
          // rescale O where any lane of the warp moved (P V of the last tile is
          // complete: it was issued before the S that just arrived)
          if (t > 0 && __any_sync(0xffffffffu, move)) {
            for (int c = 0; c < c_n; c += 16) {
              uint32_t o[16];
              ht::tmem_ld(t_o + c, o);
#pragma unroll
              for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * alpha);
              ht::tmem_st(t_o + c, o);
            }
          }
        }
        const float mb = mref == -INFINITY ? 0.f : -mref;
        const uint64_t cc = pack2(c2, c2), mm = pack2(mb, mb);
        uint64_t l2[2] = {0, 0};
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 y = unpack2(ffma2(ht::pair(s[2 * e], s[2 * e + 1]), cc, mm));
          const float a = tc::ex2_approx(y.x), b = tc::ex2_approx(y.y);
          l2[e & 1] = ht::fadd2(l2[e & 1], pack2(a, b));
          pk[e] = tc::pack_bf16x2(a, b);
        }
        ht::tmem_st(t_s, pk);
        l += hsum2(ht::fadd2(l2[0], l2[1]));
        const int kt = t * HT_KEYS;
        if (len < p.Nk && kt + HT_KEYS > len) {
          // keys beyond the length may hold anything: their weights are zero,
          // their V rows become zero too
          const uint32_t s_ = (kc0 + t) % NS;
          if (ok) ok = ht::warp_wait(&sh.vfull[s_], ((kc0 + t) / NS) & 1, abort_flag);
          const int r0 = len - kt;  // > 0: the tile has a visible key
          const uint32_t v = kva + s_ * 2 * TILE + TILE;
          for (int e = half * 128 + row; e < (128 - r0) * (DP / 8); e += 256) {
            const int r = r0 + e / (DP / 8), c = e % (DP / 8);
            st_shared_zero16(v + (uint32_t)((c >> 3) * 128 * 128 + r * 128 + (c & 7) * 16));
          }
          tc::fence_async_smem();
        }
        ht::st_wait();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) ws::arrive(&sh.pfull[w]);
      }
      if (nt > 0) {
        if (ok) ok = ht::warp_wait(&sh.odone[w], oc & 1, abort_flag);
        ++oc;
        tc::fence_after_sync();
        // a row whose other half gave up is NaN as a whole: its reference
        // maximum and its sum have both halves' parts
        if (!ok) l = __int_as_float(0x7fffffff);
        sh.sum[w][half][row] = l;
        pair_sync();
        l += sh.sum[w][half ^ 1][row];
      }
      const float inv = !ok ? __int_as_float(0x7fffffff) : (l == 0.f ? 0.f : 1.f / l);
      __nv_bfloat16* O = static_cast<__nv_bfloat16*>(p.o) +
                         (((int64_t)it.b * p.Nq + i) * p.H + h) * p.d + c_lo;
      for (int c = 0; c < c_n; c += 16) {
        uint32_t o[16];
        if (nt > 0) {
          ht::tmem_ld(t_o + c, o);
        } else {
#pragma unroll
          for (int u = 0; u < 16; ++u) o[u] = 0u;
        }
        if (i < p.Nq) {
#pragma unroll
          for (int u = 0; u < 16; u += 8) {
            if (c + u >= c_n) break;
            uint4 x;
            x.x = tc::pack_bf16x2(__uint_as_float(o[u]) * inv, __uint_as_float(o[u + 1]) * inv);
            x.y = tc::pack_bf16x2(__uint_as_float(o[u + 2]) * inv, __uint_as_float(o[u + 3]) * inv);
            x.z = tc::pack_bf16x2(__uint_as_float(o[u + 4]) * inv, __uint_as_float(o[u + 5]) * inv);
            x.w = tc::pack_bf16x2(__uint_as_float(o[u + 6]) * inv, __uint_as_float(o[u + 7]) * inv);
            *reinterpret_cast<uint4*>(O + c + u) = x;
          }
        }
      }
      tc::fence_before_sync();
      if (half == 0 && p.lse && i < p.Nq)
        p.lse[((int64_t)it.b * p.H + h) * p.Nq + i] =
            !ok ? inv : (l == 0.f ? -INFINITY : (mref + log2f(l)) * HT_LN2);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == HT_MMA_WARP) tc::tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// tensor maps and launch
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return static_cast<EncodeTiledFn>(nullptr);
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// strides of the heads, rows and episodes in bytes; false where TMA cannot
// take them
static bool map_strides(const HeadStrides& s, int B, int N, int h, int es, cuuint64_t (&bytes)[3]) {
  const int64_t st[3] = {s.h, s.n, s.b};
  const int size[3] = {h, N, B};
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of one is never used
    const int64_t e = size[i] == 1 ? 16 / es : st[i];
    if (e <= 0 || e * es % 16 || e * es >= ((int64_t)1 << 40)) return false;
    bytes[i] = (cuuint64_t)(e * es);
  }
  return true;
}
bool head_map_ok(const HeadStrides& s, int B, int N, int h) {
  cuuint64_t bytes[3];
  return map_strides(s, B, N, h, 2, bytes);
}

bool head_box_map(CUtensorMap* map, const void* ptr, const HeadStrides& s, int B, int N, int h,
                  int d, bool f32, int box_rows) {
  const EncodeTiledFn fn = encode_fn();
  cuuint64_t bytes[3];
  if (!fn || (uintptr_t)ptr % 16 || !map_strides(s, B, N, h, f32 ? 4 : 2, bytes)) return false;
  const cuuint64_t size[4] = {(cuuint64_t)d, (cuuint64_t)h, (cuuint64_t)N, (cuuint64_t)B};
  const cuuint32_t box[4] = {f32 ? 32u : 64u, 1, (cuuint32_t)box_rows, 1}, one[4] = {1, 1, 1, 1};
  return fn(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
            const_cast<void*>(ptr), size, bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool head_tensor_map(CUtensorMap* map, const void* ptr, const HeadStrides& s, int B, int N, int h,
                     int d) {
  return head_box_map(map, ptr, s, B, N, h, d, false, ht::BOX_ROWS);
}

template <int NKS>
static cudaError_t fwd_tc_go(const CUtensorMap* m, const HeadAttnParams& p, const HtGrid& gr,
                             int grid, cudaStream_t s) {
  constexpr int SMEM = HtPlan<ht::width(NKS)>::SMEM;
  const void* fn = reinterpret_cast<const void*>(&head_fwd_tc_kernel<NKS>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  head_fwd_tc_kernel<NKS><<<grid, HT_THREADS, SMEM, s>>>(m[0], m[1], m[2], p, gr);
  return cudaGetLastError();
}

int head_sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

// Items of a bf16 call that these kernels take, 0 for one that they leave:
// rows on the 16-byte grid, by the rules below.
int64_t head_fwd_tc_items(const HeadAttnParams& p) {
  // Short sets of rows leave these 128-row tiles half empty, and for narrow
  // rows the products weigh little; the kernels of head_attn.cu were faster
  // there. Measured, those against these (us): 512 x 8 heads, d = 64: N = 64
  // 58 / 103, N = 96 140 / 113, N = 256 379 / 208; 512 x 4 heads, d = 32:
  // N = 128 44 / 51, N = 192 82 / 91, N = 224 132 / 93; d = 16, 256 x 4 heads:
  // N = 192 32 / 45, N = 512 152 / 130.
  if (!p.vec || p.Nk < 1 || p.Nq <= (p.d > 32 ? 64 : 192)) return 0;
  const int64_t pairs = ((int64_t)cdiv(p.Nq, 128) * p.G + 1) / 2;
  const int64_t items = pairs * p.B * p.Hk;
  if (items > (1 << 30)) return 0;
  // With few items those kernels fill the GPU by splitting the key axis. 128
  // rows of 8 heads, d = 64, against 2048 and 8192 keys: 40 items 28 / 27 and
  // 67 / 92 us, 56 items 36 / 27 and 85 / 93, 128 items 63 / 28 and 161 / 96.
  if (p.splits > 1 && items < 56) return 0;
  const bool maps = head_map_ok(p.sq, p.B, p.Nq, p.H) && head_map_ok(p.sk, p.B, p.Nk, p.Hk) &&
                    head_map_ok(p.sv, p.B, p.Nk, p.Hk);
  return maps ? items : 0;
}

// *done says whether the call was taken.
cudaError_t launch_head_fwd_tc(const HeadAttnParams& p, cudaStream_t s, bool* done) {
  *done = false;
  const int64_t items = head_fwd_tc_items(p);
  if (!items) return cudaSuccess;
  HtGrid gr;
  gr.nqt = cdiv(p.Nq, 128);
  CUtensorMap m[3];
  if (!head_tensor_map(&m[0], p.q, p.sq, p.B, p.Nq, p.H, p.d) ||
      !head_tensor_map(&m[1], p.k, p.sk, p.B, p.Nk, p.Hk, p.d) ||
      !head_tensor_map(&m[2], p.v, p.sv, p.B, p.Nk, p.Hk, p.d))
    return cudaSuccess;
  const int sms = head_sm_count();
  gr.pairs = cdiv(gr.nqt * p.G, 2);
  gr.items = (int)items;
  gr.pair_major = p.peers == PEERS_PAST && p.B * p.Hk <= sms;
  const int grid = items < sms ? (int)items : sms;
  *done = true;
  if (p.d <= 32) return fwd_tc_go<2>(m, p, gr, grid, s);
  if (p.d <= 64) return fwd_tc_go<4>(m, p, gr, grid, s);
  if (p.d <= 96) return fwd_tc_go<6>(m, p, gr, grid, s);
  return fwd_tc_go<8>(m, p, gr, grid, s);
}

}  // namespace tarmac
