// decay_tc.cu — attention with a decay for each head on the tensor memory
// (tcgen05), bf16 rows of 40 to 128 columns. The form is that of decay.cuh, in
// chunks of 128 rows:
//   P = a b^T, out = (l^(i-j) P, j <= i) c + l^(i+1) a S,
//   S = l^n S + (l^(n-1-j) b)^T c.
//
// decay_rows_tc_kernel gives the rows. A block walks over one unit: a head of
// an episode, or two heads of up to 64 columns (the two 64-column halves of a
// tile), in one segment of the row axis. Roles of its 20 warps (two idle):
// * warp 1: one thread loads a, b, c tiles by TMA, two chunks deep.
// * warp 0: one thread issues the products P, a S, the state's and P c.
// * warps 4..11 weight P (TMEM, back to TMEM as bf16, the A operand of P c) and
//   store the rows.
// * warps 12..19 keep the state (fp32 in TMEM: scaled by l^n before the product
//   adds to it; a bf16 copy in shared memory multiplies a), weight b for the
//   state's product, in two bf16 parts over b and a once those are used, and
//   scale a S by l^(i+1) before P c adds to it.
// TMEM columns: P of a unit's head u at 128 u, out at 256, S at 384. S has the
// columns of c as lanes, those of b as columns; with two heads the product
// forms all four blocks of 64 x 64 and only the two of one head each are used.
// Roundings to bf16, one on the way of each term and the size of the output's
// own: the weighted P and the copy of S. One part for the weighted b would be
// a second for what passes through S (2.6e-3 of the rows' norm, where two give
// 2.3e-3 and the output's rounding alone is 1.7e-3).
//
// decay_state_tc_kernel gives what each segment adds to the state, in fp32
// registers: the weighted b in two bf16 parts for states that only feed the
// rows, in three (24 bits) for those that the caller gets.
//
// Bound by memory: four tiles a chunk (a, b, c, out), 128 KB for 2048 clocks of
// products at d = 128 (about 5600 clocks of one SM's share of HBM).
// Every wait is bounded; one that runs out ends all roles once their copies
// and products have landed, and every row is written, NaN or right.
#include "decay.cuh"
#include "head_tc.cuh"

namespace tarmac {

int head_sm_count();

namespace {

constexpr int DT_THREADS = 640;
constexpr int DT_MMA_WARP = 0, DT_TMA_WARP = 1, DT_W0 = 4;
constexpr int DT_T = DECAY_TC_CHUNK;
constexpr int DT_TILE = DT_T * 128 * 2;   // bytes: two halves of 64 columns
constexpr int DT_HALF = DT_TILE / 2;
constexpr float DT_LOG2E = 1.4426950408889634f;

struct DtGrid {
  int units, head_units, chunks;
};

// One unit: episode, first head, rows, and the chunks k in [k0, k1) in the
// order they are walked; those in [a0, a1) have rows.
struct DtUnit {
  int b, h, seg, len, k0, k1, a0, a1;
};
template <bool PAIR>
__device__ __forceinline__ DtUnit dt_unit(const DecayParams& p, const DtGrid& g, int unit) {
  DtUnit w;
  const int x = unit % g.head_units, y = unit / g.head_units;
  w.h = PAIR ? 2 * x : x;
  w.b = y % p.B;
  w.seg = y / p.B;
  w.len = decay_len(p, w.b);
  const int full = cdiv(w.len, DT_T);
  w.k0 = w.seg * p.seg_chunks;
  w.k1 = min(w.k0 + p.seg_chunks, g.chunks);
  w.a0 = p.reverse ? max(w.k0, g.chunks - full) : w.k0;
  w.a1 = p.reverse ? w.k1 : min(w.k1, full);
  w.a1 = max(w.a1, w.a0);
  return w;
}
__device__ __forceinline__ int dt_chunk(const DecayParams& p, const DtGrid& g, int k) {
  return p.reverse ? g.chunks - 1 - k : k;
}
__device__ __forceinline__ int dt_rows(const DtUnit& w, int chunk) {
  return min(DT_T, w.len - chunk * DT_T);
}
__device__ __forceinline__ float power(float l2, int e) { return tc::ex2_approx(l2 * (float)e); }

// a tile of 128 rows: both halves of one head, or one half of each of two
template <bool PAIR>
__device__ __forceinline__ void dt_load(uint32_t dst, const CUtensorMap* map, uint64_t* mbar,
                                        const DecayParams& p, const DtUnit& w, int share, int row) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int head = (PAIR ? min(w.h + u, p.H - 1) : w.h) / share;
#pragma unroll
    for (int r = 0; r < DT_T / 64; ++r)
      ht::tma_box(dst + u * DT_HALF + r * ht::BOX_BYTES, map, mbar, PAIR ? 0 : u * 64, head,
                  row + r * 64, w.b);
  }
}

// Rows of a staged tile by 16-byte pieces: piece e of a half holds row e / 8,
// wherever the swizzle put its columns.
__device__ __forceinline__ uint4 ld_piece(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void st_piece(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}
__device__ __forceinline__ float lo_half(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_half(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// the pair of fp32 bits (a, b) w, as bf16
__device__ __forceinline__ uint32_t scaled_f32(uint32_t a, uint32_t b, float w) {
  return tc::pack_bf16x2(__uint_as_float(a) * w, __uint_as_float(b) * w);
}
// the pair (a, b) as bf16; what the rounding left stays
__device__ __forceinline__ uint32_t split_off(float& a, float& b) {
  const uint32_t h = tc::pack_bf16x2(a, b);
  a -= lo_half(h);
  b -= hi_half(h);
  return h;
}

__device__ __forceinline__ void tmem_ld_n(uint32_t t, uint32_t (&r)[16]) { ht::tmem_ld(t, r); }
__device__ __forceinline__ void tmem_ld_n(uint32_t t, uint32_t (&r)[32]) { ht::tmem_ld(t, r); }

// D[tmem] (+)= C^T B over 128 rows; both tiles by rows (MN-major operands)
__device__ __forceinline__ void issue_state(uint32_t tmem_d, uint64_t dc, uint64_t db,
                                            uint32_t idesc, bool add) {
#pragma unroll
  for (int ks = 0; ks < DT_T / 16; ++ks)
    tc::mma_bf16(tmem_d, dc + (uint64_t)((ks * 2048) >> 4), db + (uint64_t)((ks * 2048) >> 4),
                 idesc, add || ks > 0);
}

struct DtShared {
  uint64_t full_ab[2], full_c[2], empty[2];
  uint64_t pdone, s16, o1done, oscaled, conv, udone, pready[2], pvdone, ofree, drain;
  uint32_t tmem;
  int abort_flag;
  alignas(16) float steps[2][16];  // powers inside a group of 16 columns, by head of the unit
};

constexpr int dt_smem(bool pair) { return 6 * DT_TILE + (pair ? DT_HALF : DT_TILE) + 1024; }

template <int NKS, bool PAIR>
__global__ void __launch_bounds__(DT_THREADS, 1)
    decay_rows_tc_kernel(const __grid_constant__ CUtensorMap ma,
                         const __grid_constant__ CUtensorMap mb,
                         const __grid_constant__ CUtensorMap mc, DecayParams p, DtGrid g) {
  constexpr int HEADS = PAIR ? 2 : 1;
  extern __shared__ unsigned char dt_raw[];
  __shared__ DtShared sh;
  const uint32_t base = (tc::smem_addr(dt_raw) + 1023u) & ~1023u;
  const uint32_t s16 = base + 6 * DT_TILE;
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&sh.full_ab[s], 1);
      tc::mbar_init(&sh.full_c[s], 1);
      tc::mbar_init(&sh.empty[s], 1);
      tc::mbar_init(&sh.pready[s], 8 / HEADS);
    }
    tc::mbar_init(&sh.pdone, 1);
    tc::mbar_init(&sh.o1done, 1);
    tc::mbar_init(&sh.udone, 1);
    tc::mbar_init(&sh.pvdone, 1);
    tc::mbar_init(&sh.drain, 1);
    tc::mbar_init(&sh.s16, 8);
    tc::mbar_init(&sh.oscaled, 8);
    tc::mbar_init(&sh.conv, 8);
    tc::mbar_init(&sh.ofree, 8);
    sh.abort_flag = 0;
    tc::mbar_init_fence();
  }
  if (warp == DT_MMA_WARP) tc::tmem_alloc(&sh.tmem, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sh.tmem, t_out = tmem + 256, t_state = tmem + 384;
  // does a unit's first chunk start from a state?
  auto starts = [&](const DtUnit& w) { return p.part ? w.seg > 0 || p.start : p.start != nullptr; };

  if (warp == DT_TMA_WARP) {
    if (lane == 0) {
      uint32_t c = 0;
      for (int k = 0, unit = blockIdx.x; unit < g.units; unit += gridDim.x, ++k) {
        if (ht::gives_up(ht::ROLE_LOADER, k)) {
          *abort_flag = 1;
          break;
        }
        const DtUnit w = dt_unit<PAIR>(p, g, unit);
        for (int x = w.a0; x < w.a1; ++x, ++c) {
          const int s = c & 1, row = dt_chunk(p, g, x) * DT_T;
          if (!ws::wait(&sh.empty[s], ((c >> 1) & 1) ^ 1, abort_flag)) goto tma_done;
          const uint32_t at = base + s * 3 * DT_TILE;
          ht::expect_tx(&sh.full_ab[s], 2 * DT_TILE);
          dt_load<PAIR>(at, &ma, &sh.full_ab[s], p, w, p.ga, row);
          dt_load<PAIR>(at + DT_TILE, &mb, &sh.full_ab[s], p, w, p.gb, row);
          ht::expect_tx(&sh.full_c[s], DT_TILE);
          dt_load<PAIR>(at + 2 * DT_TILE, &mc, &sh.full_c[s], p, w, p.gc, row);
        }
      }
    tma_done:
      ht::drain_copies(sh.full_ab, 2, c);
      ht::drain_copies(sh.full_c, 2, c);
    }
    __syncwarp();
  } else if (warp == DT_MMA_WARP) {
    constexpr uint32_t id_p = tc::idesc_bf16(128, 128, false, false);
    constexpr uint32_t id_1 = tc::idesc_bf16(128, NKS * 16, false, false);
    constexpr uint32_t id_s = tc::idesc_bf16(128, 128, true, true);
    constexpr uint32_t id_2 = tc::idesc_bf16(128, NKS * 16, false, true);
    const bool leader = ht::elect_one();
    bool ok = true;
    uint32_t c = 0, states = 0;  // chunks, and those with a state
    auto wait = [&](uint64_t& bar, uint32_t parity) {
      ok = ok && ht::wait_at(tc::smem_addr(&bar), parity, abort_flag);
    };
    for (int unit = blockIdx.x; unit < g.units && ok; unit += gridDim.x) {
      const DtUnit w = dt_unit<PAIR>(p, g, unit);
      for (int x = w.a0; x < w.a1 && ok; ++x, ++c) {
        const bool state = x > w.a0 || starts(w);
        const uint32_t s = c & 1, ph = (c >> 1) & 1, odd = c & 1;
        const uint32_t at = base + s * 3 * DT_TILE;
        const uint64_t da = ht::desc128(at, 16), db = ht::desc128(at + DT_TILE, 16);
        const uint64_t dc = ht::desc128(at + 2 * DT_TILE, DT_HALF);
        wait(sh.full_ab[s], ph);
        tc::fence_after_sync();
        if (ok && leader) {
#pragma unroll
          for (int u = 0; u < HEADS; ++u)
            ht::issue_scores<NKS, 128>(tmem + u * 128, da + u * (DT_HALF >> 4),
                                       db + u * (DT_HALF >> 4), id_p);
          ht::commit_at(tc::smem_addr(&sh.pdone));
        }
        __syncwarp();
        wait(sh.ofree, odd ^ 1);  // the rows of the chunk before are out
        if (state) {
          wait(sh.s16, states & 1);
          tc::fence_after_sync();
          if (ok && leader) {
#pragma unroll
            for (int u = 0; u < HEADS; ++u)
              ht::issue_scores<NKS, 128>(t_out + u * 64, da + u * (DT_HALF >> 4),
                                         ht::desc128(s16 + u * 64 * 128, 16), id_1);
            ht::commit_at(tc::smem_addr(&sh.o1done));
          }
          __syncwarp();
        }
        wait(sh.full_c[s], ph);
        wait(sh.conv, odd);
        tc::fence_after_sync();
        if (x + 1 < w.a1) {
          if (ok && leader) {
            issue_state(t_state, dc, ht::desc128(at + DT_TILE, DT_HALF), id_s, state);
            issue_state(t_state, dc, ht::desc128(at, DT_HALF), id_s, true);
            ht::commit_at(tc::smem_addr(&sh.udone));
          }
          __syncwarp();
        }
        if (state) {
          wait(sh.oscaled, states & 1);
          ++states;
        }
#pragma unroll
        for (int u = 0; u < HEADS; ++u) {
          wait(sh.pready[u], odd);
          tc::fence_after_sync();
          if (ok && leader)
            ht::issue_aggregate<DT_T, 64>(t_out + u * 64, tmem + u * 128,
                                          dc + u * (DT_HALF >> 4), id_2, state);
          __syncwarp();
        }
        if (ok && leader) {
          ht::commit_at(tc::smem_addr(&sh.pvdone));
          ht::commit_at(tc::smem_addr(&sh.empty[s]));
        }
        ok = ht::agree(ok);
      }
    }
    // the last commits land before the block ends
    for (uint32_t i = c > 2 ? c - 2 : 0; i < c && ok; ++i)
      ok = ht::wait_at(tc::smem_addr(&sh.empty[i & 1]), (i >> 1) & 1, abort_flag);
    if (!ht::agree(ok)) ht::drain_products(&sh.drain, leader);
    __syncwarp();
  } else if (warp >= DT_W0 && warp < DT_W0 + 8) {
    // ---------------- weights of P, and the rows ----------------
    // one head: columns [64 half, 64 half + 64) of P and of the rows; two:
    // all of head `half`
    const int half = (warp - DT_W0) >> 2, i = threadIdx.x & 127, w0 = (warp & 3) * 32;
    const uint32_t lane_off = (uint32_t)w0 << 16;
    const int c_lo = PAIR ? 0 : half * 64, c_n = max(0, min(64, p.d - c_lo));
    float* steps = sh.steps[half];
    bool ok = true;
    uint32_t c = 0;
    for (int k = 0, unit = blockIdx.x; unit < g.units; unit += gridDim.x, ++k) {
      const DtUnit w = dt_unit<PAIR>(p, g, unit);
      if (ht::gives_up(ht::ROLE_WEIGHTS, k)) {
        ok = false;
        *abort_flag = 1;
      }
      const int h = PAIR ? min(w.h + half, p.H - 1) : w.h;
      const bool mine = !PAIR || w.h + half < p.H;
      const float l2 = decay_rate(p.log_decay, h) * DT_LOG2E;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
      if (i < 16) steps[i] = power(l2, p.reverse ? i : 15 - i);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
      for (int x = w.k0; x < w.k1; ++x) {
        const int chunk = dt_chunk(p, g, x), row = chunk * DT_T + i;
        const bool live = x >= w.a0 && x < w.a1;
        const int n = live ? dt_rows(w, chunk) : 0;
        if (live) {
          if (ok) ok = ht::warp_wait(&sh.pdone, c & 1, abort_flag);
          tc::fence_after_sync();
#pragma unroll 1
          for (int piece = 0; piece < HEADS; ++piece) {
            const int j0 = PAIR ? piece * 64 : half * 64;
            const uint32_t t_p = tmem + (PAIR ? half * 128 : 0) + j0 + lane_off;
            uint32_t pk[32];
            if (p.reverse ? w0 > j0 + 63 || j0 >= n : w0 + 31 < j0) {
#pragma unroll
              for (int e = 0; e < 32; ++e) pk[e] = 0u;
            } else {
              uint32_t s[64];
              ht::tmem_ld(t_p, s);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int jb = j0 + 16 * q;
                if (p.reverse ? jb >= w0 + 31 && jb + 15 < n : w0 >= jb + 15) {
                  const float f = p.in_scale * power(l2, p.reverse ? jb - i : i - jb - 15);
                  const uint64_t ff = pack2(f, f);
#pragma unroll
                  for (int e = 0; e < 16; e += 4) {
                    const float4 t = *reinterpret_cast<const float4*>(steps + e);
                    const float2 y = unpack2(ht::fmul2(ht::fmul2(pack2(t.x, t.y), ff),
                                                       ht::pair(s[16 * q + e], s[16 * q + e + 1])));
                    const float2 z = unpack2(ht::fmul2(ht::fmul2(pack2(t.z, t.w), ff),
                                                       ht::pair(s[16 * q + e + 2], s[16 * q + e + 3])));
                    pk[8 * q + e / 2] = tc::pack_bf16x2(y.x, y.y);
                    pk[8 * q + e / 2 + 1] = tc::pack_bf16x2(z.x, z.y);
                  }
                } else if (p.reverse ? jb + 15 < w0 || jb >= n : w0 + 31 < jb) {
#pragma unroll
                  for (int e = 0; e < 8; ++e) pk[8 * q + e] = 0u;
                } else {
#pragma unroll
                  for (int e = 0; e < 16; e += 2) {
                    float y[2];
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                      const int j = jb + e + v, gap = p.reverse ? j - i : i - j;
                      const bool see = gap >= 0 && (!p.reverse || j < n);
                      y[v] = see ? __uint_as_float(s[16 * q + e + v]) * p.in_scale *
                                       power(l2, max(gap, 0))
                                 : 0.f;
                    }
                    pk[8 * q + e / 2] = tc::pack_bf16x2(y[0], y[1]);
                  }
                }
              }
            }
            ht::tmem_st(t_p, pk);
          }
          ht::st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (ok && lane == 0) ws::arrive(&sh.pready[PAIR ? half : 0]);
          if (ok) ok = ht::warp_wait(&sh.pvdone, c & 1, abort_flag);
          tc::fence_after_sync();
          ++c;
        }
        const bool store = mine && row < p.N;
        const int64_t at = (((int64_t)w.b * p.N + row) * p.H + h) * p.d + c_lo;
        const float f = !ok ? __int_as_float(0x7fffffff) : p.out_scale;
        const bool zero = ok && i >= n;
#pragma unroll 1
        for (int cc = 0; cc < c_n; cc += 32) {
          uint32_t o[32];
          if (live) ht::tmem_ld(t_out + half * 64 + cc + lane_off, o);
          if (!live || zero) {
#pragma unroll
            for (int u = 0; u < 32; ++u) o[u] = 0u;
          }
          if (store) {
            if (p.out_f32) {
              float* dst = static_cast<float*>(p.out) + at + cc;
#pragma unroll
              for (int u = 0; u < 32; u += 4)
                if (cc + u < c_n)
                  *reinterpret_cast<float4*>(dst + u) =
                      make_float4(__uint_as_float(o[u]) * f, __uint_as_float(o[u + 1]) * f,
                                  __uint_as_float(o[u + 2]) * f, __uint_as_float(o[u + 3]) * f);
            } else {
              __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + at + cc;
#pragma unroll
              for (int u = 0; u < 32; u += 8)
                if (cc + u < c_n)
                  *reinterpret_cast<uint4*>(dst + u) = make_uint4(
                      scaled_f32(o[u], o[u + 1], f), scaled_f32(o[u + 2], o[u + 3], f),
                      scaled_f32(o[u + 4], o[u + 5], f), scaled_f32(o[u + 6], o[u + 7], f));
            }
          }
          __syncwarp();
        }
        if (live) {
          tc::fence_before_sync();
          __syncwarp();
          if (ok && lane == 0) ws::arrive(&sh.ofree);
        }
      }
    }
  } else if (warp >= DT_W0 + 8) {
    // ---------------- the state ----------------
    const int half = (warp - DT_W0 - 8) >> 2, r = threadIdx.x & 127;
    const int tid = threadIdx.x - (DT_W0 + 8) * 32;  // 0 .. 255
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    // this thread's part of S: row r (a column of c), SN columns (of b)
    constexpr int SP = PAIR ? 1 : 2;  // pieces of 32 columns
    const int s_head = PAIR ? r >> 6 : 0;
    const int s_col = half * (PAIR ? 32 : 64);  // first column inside the head
    const uint32_t t_s = t_state + (PAIR ? s_head * 64 : 0) + s_col + lane_off;
    const uint32_t t_o = t_out + half * 64 + lane_off;
    bool ok = true;
    uint32_t c = 0, states = 0, us = 0;
    for (int unit = blockIdx.x; unit < g.units; unit += gridDim.x) {
      const DtUnit w = dt_unit<PAIR>(p, g, unit);
      const int h0 = w.h, h1 = PAIR ? min(w.h + 1, p.H - 1) : w.h;
      const float l2_0 = decay_rate(p.log_decay, h0) * DT_LOG2E;
      const float l2_1 = decay_rate(p.log_decay, h1) * DT_LOG2E;
      const float l2_s = s_head ? l2_1 : l2_0, l2_o = PAIR && half ? l2_1 : l2_0;
      const int hs = s_head ? h1 : h0, rc = PAIR ? r & 63 : r;
      const float* start = nullptr;
      if (starts(w))
        start = (p.part ? p.part + (int64_t)w.seg * p.B * p.H * p.d * p.d : p.start) +
                ((int64_t)w.b * p.H + hs) * p.d * p.d;
      for (int x = w.a0; x < w.a1; ++x, ++c) {
        const int chunk = dt_chunk(p, g, x), n = dt_rows(w, chunk);
        const bool state = x > w.a0 || start;
        const uint32_t at = base + (c & 1) * 3 * DT_TILE;
        if (state) {
          // the state before this chunk: its copy, and what the product adds to
          const float all = power(l2_s, n);
          if (x > w.a0) {
            if (ok) ok = ht::warp_wait(&sh.udone, us & 1, abort_flag);
            ++us;
            tc::fence_after_sync();
          }
#pragma unroll 1
          for (int q = 0; q < SP; ++q) {
            uint32_t s[32];
            const int b0 = s_col + 32 * q;
            if (x > w.a0) {
              ht::tmem_ld(t_s + 32 * q, s);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const int bc = b0 + e;
                const bool in = rc < p.d && bc < p.d;
                s[e] = in ? __float_as_uint(__ldg(start + (p.transposed ? rc * p.d + bc
                                                                        : bc * p.d + rc)))
                          : 0u;
              }
            }
            const uint32_t row = s16 + (PAIR ? 0 : (b0 >> 6) * DT_HALF) + r * 128;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              st_piece(row + (((((b0 & 63) + e) >> 3) ^ (r & 7)) << 4),
                       make_uint4(scaled_f32(s[e], s[e + 1], 1.f), scaled_f32(s[e + 2], s[e + 3], 1.f),
                                  scaled_f32(s[e + 4], s[e + 5], 1.f),
                                  scaled_f32(s[e + 6], s[e + 7], 1.f)));
            }
            if (x + 1 < w.a1) {
#pragma unroll
              for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * all);
              ht::tmem_st(t_s + 32 * q, s);
            }
          }
          ht::st_wait();
          tc::fence_before_sync();
          tc::fence_async_smem();
          __syncwarp();
          if (ok && lane == 0) ws::arrive(&sh.s16);
        }
        // b, weighted, in two parts: over b and over a, once P and a S are formed
        if (ok) ok = ht::warp_wait(&sh.full_ab[c & 1], (c >> 1) & 1, abort_flag);
        if (ok) ok = ht::warp_wait(&sh.pdone, c & 1, abort_flag);
        if (state) {
          if (ok) ok = ht::warp_wait(&sh.o1done, states & 1, abort_flag);
          ++states;
        }
        if (x + 1 < w.a1) {
#pragma unroll 4
          for (int e = 0; e < 8; ++e) {
            const int piece = tid + 256 * e, row = (piece & 1023) >> 3;
            const float l2 = PAIR && e >= 4 ? l2_1 : l2_0;
            const float f = row < n ? p.in_scale * power(l2, p.reverse ? row + 1 : n - 1 - row) : 0.f;
            const uint4 v = ld_piece(at + DT_TILE + piece * 16);
            const uint32_t in[4] = {v.x, v.y, v.z, v.w};
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float y = lo_half(in[i]) * f, z = hi_half(in[i]) * f;
              if (row >= n) y = z = 0.f;
              hi[i] = split_off(y, z);
              lo[i] = tc::pack_bf16x2(y, z);
            }
            st_piece(at + DT_TILE + piece * 16, make_uint4(hi[0], hi[1], hi[2], hi[3]));
            st_piece(at + piece * 16, make_uint4(lo[0], lo[1], lo[2], lo[3]));
          }
        }
        if (n < DT_T && w.len < p.N) {
          // rows from the length on may hold anything: those of c become zero
          if (ok) ok = ht::warp_wait(&sh.full_c[c & 1], (c >> 1) & 1, abort_flag);
#pragma unroll 1
          for (int piece = tid; piece < 2048; piece += 256)
            if (((piece & 1023) >> 3) >= n) st_shared_zero16(at + 2 * DT_TILE + piece * 16);
        }
        tc::fence_async_smem();
        __syncwarp();
        if (ok && lane == 0) ws::arrive(&sh.conv);
        if (state) {
          tc::fence_after_sync();
          const float f = power(l2_o, max(0, p.reverse ? n - 1 - r : r + 1));
#pragma unroll 1
          for (int q = 0; q < 2; ++q) {
            uint32_t o[32];
            ht::tmem_ld(t_o + 32 * q, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            ht::tmem_st(t_o + 32 * q, o);
          }
          ht::st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (ok && lane == 0) ws::arrive(&sh.oscaled);
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == DT_MMA_WARP) tc::tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// what each segment adds to the state
// ---------------------------------------------------------------------------
template <int PLANES>
struct DsTcPlan {
  static constexpr int NS = 2;
  // places of the lower parts; with two, a chunk is split while the product of
  // the one before runs
  static constexpr int LOW = PLANES == 2 ? 2 : 1;
  static constexpr int SMEM = (2 * NS + LOW * (PLANES - 1)) * DT_TILE + 1024;
};
template <int NS>
struct DsTcShared {
  uint64_t full[NS], empty[NS], conv, udone[2], drain;
  uint32_t tmem;
  int abort_flag;
};

template <bool PAIR, int PLANES>
__global__ void __launch_bounds__(DT_THREADS, 1)
    decay_state_tc_kernel(const __grid_constant__ CUtensorMap mb,
                          const __grid_constant__ CUtensorMap mc, DecayParams p, DtGrid g) {
  constexpr int NS = DsTcPlan<PLANES>::NS, LOW = DsTcPlan<PLANES>::LOW;
  extern __shared__ unsigned char dt_raw[];
  __shared__ DsTcShared<NS> sh;
  const uint32_t base = (tc::smem_addr(dt_raw) + 1023u) & ~1023u;
  const uint32_t extra = base + 2 * NS * DT_TILE;  // the lower parts
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      tc::mbar_init(&sh.full[s], 1);
      tc::mbar_init(&sh.empty[s], 1);
    }
    tc::mbar_init(&sh.conv, 16);
    tc::mbar_init(&sh.udone[0], 1);
    tc::mbar_init(&sh.udone[1], 1);
    tc::mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    tc::mbar_init_fence();
  }
  if (warp == DT_MMA_WARP) tc::tmem_alloc(&sh.tmem, 256);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sh.tmem;

  if (warp == DT_TMA_WARP) {
    if (lane == 0) {
      uint32_t c = 0;
      for (int k = 0, unit = blockIdx.x; unit < g.units; unit += gridDim.x, ++k) {
        if (ht::gives_up(ht::ROLE_LOADER, k)) {
          *abort_flag = 1;
          break;
        }
        const DtUnit w = dt_unit<PAIR>(p, g, unit);
        for (int x = w.a0; x < w.a1; ++x, ++c) {
          const int s = c % NS, row = dt_chunk(p, g, x) * DT_T;
          if (!ws::wait(&sh.empty[s], ((c / NS) & 1) ^ 1, abort_flag)) goto tma_done;
          const uint32_t at = base + s * 2 * DT_TILE;
          ht::expect_tx(&sh.full[s], 2 * DT_TILE);
          dt_load<PAIR>(at, &mb, &sh.full[s], p, w, p.gb, row);
          dt_load<PAIR>(at + DT_TILE, &mc, &sh.full[s], p, w, p.gc, row);
        }
      }
    tma_done:
      ht::drain_copies(sh.full, NS, c);
    }
    __syncwarp();
  } else if (warp == DT_MMA_WARP) {
    constexpr uint32_t id_s = tc::idesc_bf16(128, 128, true, true);
    const bool leader = ht::elect_one();
    bool ok = true;
    uint32_t c = 0;
    for (int unit = blockIdx.x; unit < g.units && ok; unit += gridDim.x) {
      const DtUnit w = dt_unit<PAIR>(p, g, unit);
      for (int x = w.a0; x < w.a1 && ok; ++x, ++c) {
        const uint32_t s = c % NS, at = base + s * 2 * DT_TILE;
        const uint64_t dc = ht::desc128(at + DT_TILE, DT_HALF);
        ok = ht::wait_at(tc::smem_addr(&sh.conv), c & 1, abort_flag);
        tc::fence_after_sync();
        if (ok && leader) {
          const uint32_t d = tmem + (c & 1) * 128;
          issue_state(d, dc, ht::desc128(at, DT_HALF), id_s, false);
#pragma unroll
          for (int q = 1; q < PLANES; ++q)
            issue_state(d, dc, ht::desc128(extra + ((c % LOW) + q - 1) * DT_TILE, DT_HALF), id_s,
                        true);
          ht::commit_at(tc::smem_addr(&sh.udone[c & 1]));
          ht::commit_at(tc::smem_addr(&sh.empty[s]));
        }
        __syncwarp();
        ok = ht::agree(ok);
      }
    }
    for (uint32_t i = c > (uint32_t)NS ? c - NS : 0; i < c && ok; ++i)
      ok = ht::wait_at(tc::smem_addr(&sh.empty[i % NS]), (i / NS) & 1, abort_flag);
    if (!ht::agree(ok)) ht::drain_products(&sh.drain, leader);
    __syncwarp();
  } else if (warp >= DT_W0) {
    constexpr int SC = PAIR ? 16 : 32;  // columns of S that a thread holds
    const int grp = (warp - DT_W0) >> 2, r = threadIdx.x & 127, tid = threadIdx.x - DT_W0 * 32;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const int s_head = PAIR ? r >> 6 : 0, rc = PAIR ? r & 63 : r;
    const uint32_t t_s = tmem + (PAIR ? s_head * 64 : 0) + grp * SC + lane_off;
    bool ok = true;
    uint32_t c = 0;
    for (int unit = blockIdx.x; unit < g.units; unit += gridDim.x) {
      const DtUnit w = dt_unit<PAIR>(p, g, unit);
      const int h0 = w.h, h1 = PAIR ? min(w.h + 1, p.H - 1) : w.h;
      const float l2_0 = decay_rate(p.log_decay, h0) * DT_LOG2E;
      const float l2_1 = decay_rate(p.log_decay, h1) * DT_LOG2E;
      const float l2_s = s_head ? l2_1 : l2_0;
      float S[SC];
#pragma unroll
      for (int e = 0; e < SC; ++e) S[e] = 0.f;
      // S = l^n S + the product of chunk c_
      auto take = [&](uint32_t c_, int n) {
        if (ok) ok = ht::warp_wait(&sh.udone[c_ & 1], (c_ >> 1) & 1, abort_flag);
        tc::fence_after_sync();
        uint32_t u[SC];
        tmem_ld_n(t_s + (c_ & 1) * 128, u);
        const float all = power(l2_s, n);
#pragma unroll
        for (int e = 0; e < SC; ++e) S[e] = fmaf(all, S[e], __uint_as_float(u[e]));
        tc::fence_before_sync();
      };
      int n_before = 0;
      for (int x = w.a0; x < w.a1; ++x, ++c) {
        const int n = dt_rows(w, dt_chunk(p, g, x)), s = c % NS;
        if (LOW == 1 && x > w.a0) take(c - 1, n_before);
        if (ok) ok = ht::warp_wait(&sh.full[s], (c / NS) & 1, abort_flag);
        const uint32_t at = base + s * 2 * DT_TILE;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int piece = tid + 512 * e, row = (piece & 1023) >> 3;
          const float l2 = PAIR && e >= 2 ? l2_1 : l2_0;
          const float f = row < n ? p.in_scale * power(l2, p.reverse ? row + 1 : n - 1 - row) : 0.f;
          const uint4 v = ld_piece(at + piece * 16);
          const uint32_t in[4] = {v.x, v.y, v.z, v.w};
          uint32_t part[PLANES][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a = lo_half(in[i]) * f, b = hi_half(in[i]) * f;
            if (row >= n) a = b = 0.f;
#pragma unroll
            for (int q = 0; q < PLANES; ++q) part[q][i] = split_off(a, b);
          }
          st_piece(at + piece * 16, make_uint4(part[0][0], part[0][1], part[0][2], part[0][3]));
#pragma unroll
          for (int q = 1; q < PLANES; ++q)
            st_piece(extra + ((c % LOW) + q - 1) * DT_TILE + piece * 16,
                     make_uint4(part[q][0], part[q][1], part[q][2], part[q][3]));
          if (row >= n && w.len < p.N) st_shared_zero16(at + DT_TILE + piece * 16);
        }
        tc::fence_async_smem();
        __syncwarp();
        if (ok && lane == 0) ws::arrive(&sh.conv);
        if (LOW == 2 && x > w.a0) take(c - 1, n_before);
        n_before = n;
      }
      if (w.a1 > w.a0) take(c - 1, n_before);
      const bool mine = !PAIR || w.h + s_head < p.H;
      if (mine && rc < p.d) {
        float* dst = p.part + (((int64_t)w.seg * p.B + w.b) * p.H + (s_head ? h1 : h0)) * p.d * p.d;
#pragma unroll
        for (int e = 0; e < SC; ++e) {
          const int bc = grp * SC + e;
          if (bc < p.d) dst[bc * p.d + rc] = ok ? S[e] : __int_as_float(0x7fffffff);
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == DT_MMA_WARP) tc::tmem_dealloc(tmem, 256);
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------
DtGrid dt_grid(const DecayParams& p, int segs) {
  DtGrid g;
  g.head_units = p.d <= 64 ? cdiv(p.H, 2) : p.H;
  g.chunks = cdiv(p.N, DT_T);
  g.units = g.head_units * p.B * segs;
  return g;
}
int dt_blocks(const DtGrid& g) {
  const int sms = head_sm_count();
  return g.units < sms ? g.units : sms;
}

template <int NKS, bool PAIR>
cudaError_t rows_go(const CUtensorMap* m, const DecayParams& p, const DtGrid& g, cudaStream_t s) {
  constexpr int SMEM = dt_smem(PAIR);
  const void* fn = reinterpret_cast<const void*>(&decay_rows_tc_kernel<NKS, PAIR>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  decay_rows_tc_kernel<NKS, PAIR><<<dt_blocks(g), DT_THREADS, SMEM, s>>>(m[0], m[1], m[2], p, g);
  return cudaGetLastError();
}
template <bool PAIR, int PLANES>
cudaError_t state_go(const CUtensorMap* m, const DecayParams& p, const DtGrid& g, cudaStream_t s) {
  constexpr int SMEM = DsTcPlan<PLANES>::SMEM;
  const void* fn = reinterpret_cast<const void*>(&decay_state_tc_kernel<PAIR, PLANES>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  decay_state_tc_kernel<PAIR, PLANES><<<dt_blocks(g), DT_THREADS, SMEM, s>>>(m[0], m[1], p, g);
  return cudaGetLastError();
}

bool map_of(CUtensorMap* m, const DecayParams& p, const void* ptr, const HeadStrides& s,
            int share) {
  return head_tensor_map(m, ptr, s, p.B, p.N, p.H / share, p.d);
}

}  // namespace

// Segments of a call: the walk over the longest block, with the states' pass
// where there are segments (about half the rows' time) and what a unit costs
// beside its chunks (about one chunk). Host arithmetic for 148 SMs, so that a
// caller can ask for the scratch without a GPU.
DecayPlan decay_plan_tc(int B, int N, int H, int d) {
  const int64_t heads = (int64_t)B * (d <= 64 ? cdiv(H, 2) : H);
  const int chunks = cdiv(N, DT_T);
  DecayPlan best = {1, chunks};
  double least = 0;
  for (int want = 1; want <= chunks && want <= 256; ++want) {
    const int per = cdiv(chunks, want), segs = cdiv(chunks, per);
    const double turns = (double)((heads * segs + 147) / 148);
    const double cost = turns * (per + 1) * (segs > 1 ? 1.5 : 1.0) + (segs > 1 ? 2.0 : 0.0);
    if (want == 1 || cost < least) {
      least = cost;
      best = DecayPlan{segs, per};
    }
  }
  return best;
}

cudaError_t launch_decay_states_tc(const DecayParams& p, cudaStream_t s) {
  // the last segment's share counts only where the state after it is wanted
  const DtGrid g = dt_grid(p, p.last ? p.segs : p.segs - 1);
  if (g.units == 0) return cudaSuccess;
  CUtensorMap m[2];
  if (!map_of(&m[0], p, p.b, p.sb, p.gb) || !map_of(&m[1], p, p.c, p.sc, p.gc))
    return cudaErrorInvalidValue;
  if (p.d <= 64) return p.planes > 2 ? state_go<true, 3>(m, p, g, s) : state_go<true, 2>(m, p, g, s);
  return p.planes > 2 ? state_go<false, 3>(m, p, g, s) : state_go<false, 2>(m, p, g, s);
}

cudaError_t launch_decay_rows_tc(const DecayParams& p, cudaStream_t s) {
  CUtensorMap m[3];
  if (!map_of(&m[0], p, p.a, p.sa, p.ga) || !map_of(&m[1], p, p.b, p.sb, p.gb) ||
      !map_of(&m[2], p, p.c, p.sc, p.gc))
    return cudaErrorInvalidValue;
  const DtGrid g = dt_grid(p, p.segs);
  if (p.d <= 64) return rows_go<4, true>(m, p, g, s);
  if (p.d <= 96) return rows_go<6, false>(m, p, g, s);
  return rows_go<8, false>(m, p, g, s);
}

}  // namespace tarmac
