// decay_tc.cu — attention with a decay for each head on the tensor memory
// (tcgen05), bf16 rows of 16 to 128 columns. The form is that of decay.cuh, in
// chunks of 128 rows:
//   P = a b^T, out = (l^(i-j) P, j <= i) c + l^(i+1) a S,
//   S = l^n S + (l^(n-1-j) b)^T c.
//
// decay_rows_tc_kernel gives the rows, of one sum or of the gradients' three. A
// block walks over one unit: a head of an episode, or two heads of up to 64
// columns (the two 64-column halves of a tile), in one segment of the row axis.
// Roles of its 20 warps (two idle):
// * warp 1: one thread loads a, b, c tiles by TMA ahead of the products.
// * warp 0: one thread issues the products P, a S, the state's and P c.
// * warps 4..11 weight P (TMEM, back to TMEM as bf16, the A operand of P c) and
//   store the rows, through the tile of a.
// * warps 12..19 keep the state (fp32 in TMEM: scaled by l^n before the product
//   adds to it; a copy in shared memory multiplies a), weight b in place for
//   the state's product once P is formed, and scale a S by l^(i+1) before P c
//   adds to it.
// TMEM columns: P of a unit's head u at 128 u (one head: of two chunks in
// turn), out at 256, S at 384. S has the columns of c as lanes, those of b as
// columns; with two heads the product forms all four blocks of 64 x 64 and only
// the two of one head each are used.
// Roundings to bf16, one on the way of each term and the size of the output's
// own: the weighted P and the weighted b. The copy of S is in two bf16 parts; in
// one it would be a second rounding for what passes through S (2.6e-3 of the
// rows' norm, where this gives 2.3e-3 and the output's rounding alone 1.7e-3).
//
// decay_state_tc_kernel gives what each segment adds to the state, in fp32
// registers: the weighted b as in the rows' kernel for states that only feed
// the rows, in three bf16 parts (24 bits) for those that the caller gets.
//
// Measured: 2 x 8192 rows of 16 heads, d = 128, the gradients 190-196 us (64 chunks
// of 5800 clocks in each of 96 blocks), the forward pass 28 us of states, 5 of
// joining and 56 of rows; 32 x 1024 rows of 8 heads, d = 64, 37 and 93 us. A
// chunk at d = 128 has 1280 clocks of products and four tiles to move, 128 KB or
// 5700 clocks of an SM's share of HBM where no other block reads them too. The
// chain bounds the rest: state, a S, out, rows follow one another, and what runs
// beside them is the next P and the weights (tensor pipe 25-37 %, issue 35-43 %).
// Bound of the states' pass: issue of the split (58 %; two halves a chunk in turn
// 34 us, a whole chunk at once 43: 2 x 8192 rows of 16 heads on 4, d = 128).
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
  int units, head_units, chunks;  // units of a job
};
// One sum, the forward pass, or the gradients' three over the same heads and rows
// in one launch. A block stays with one job; those of the three lie side by side,
// as they read the same tensors.
template <int JOBS>
struct DtJobs {
  CUtensorMap map[JOBS][4];  // a, b, c, out
  DecayParams p[JOBS];
};

// One unit: episode, first head, rows, and the chunks k in [k0, k1) in the
// order they are walked; those in [a0, a1) have rows.
struct DtUnit {
  int b, h, seg, len, k0, k1, a0, a1;
};
template <bool PAIR>
__device__ __forceinline__ DtUnit dt_unit(const DecayParams& p, const DtGrid& g, int unit) {
  DtUnit w;
  const unsigned y = (unsigned)unit / (unsigned)g.head_units, x = unit - y * g.head_units;
  w.h = PAIR ? 2 * x : x;
  w.seg = y / (unsigned)p.B;
  w.b = y - w.seg * p.B;
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

// eight bf16 times f
__device__ __forceinline__ uint4 weighted(uint4 v, float f) {
  const uint64_t ff = pack2(f, f);
  uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = unpack2(ht::fmul2(pack2(lo_half(x[i]), hi_half(x[i])), ff));
    x[i] = tc::pack_bf16x2(a.x, a.y);
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
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

// A warp's 32 rows of 128 bytes in shared memory, each lane's own, 16-byte
// pieces swizzled by row as TMA reads them.
__device__ __forceinline__ void stage_row(uint32_t stage, int lane, int piece,
                                          const uint32_t (&o)[32]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      x[u] = tc::pack_bf16x2(__uint_as_float(o[8 * e + 2 * u]), __uint_as_float(o[8 * e + 2 * u + 1]));
    st_piece(stage + lane * 128 + (((piece + e) ^ (lane & 7)) << 4),
             make_uint4(x[0], x[1], x[2], x[3]));
  }
}
__device__ __forceinline__ void stage_row32(uint32_t stage, int lane, const uint32_t (&o)[32]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    st_piece(stage + lane * 128 + ((e ^ (lane & 7)) << 4),
             make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
}
// Those rows to a tensor with boxes of 32 rows, rows and columns beyond it left
// out. One lane; the same lane waits for their having been read.
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t stage, int col, int head,
                                          int row, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];\n"
      "cp.async.bulk.commit_group;" ::"l"(map),
      "r"(stage), "r"(col), "r"(head), "r"(row), "r"(b)
      : "memory");
}
__device__ __forceinline__ void stores_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
// 32 rows from memory address dst on, `step` elements apart, all of one word: the
// first n columns, where they exist; `each`: elements of 16 bytes
template <typename T>
__device__ __forceinline__ void fill_rows(T* dst, uint32_t word, int lane, int left, int64_t step,
                                          int n, int each) {
  for (int r = lane >> 3; r < min(left, 32); r += 4)
    for (int c = (lane & 7) * each; c < n; c += 8 * each)
      *reinterpret_cast<uint4*>(dst + r * step + c) = make_uint4(word, word, word, word);
}

// Decays below 2^-7 a row: l^-15 nears the end of fp32's range.
constexpr float DT_STRONG = -7.f;

// 32 columns j0 .. of row i of P, weighted, back to TMEM as bf16. Columns
// 64 c .. 64 c + 63 take the 32 TMEM columns from 64 c on. w0: the warp's first
// row. In each group of 16 columns from jb on, l^(i-j) = l^(i-jb-15) l^(15-x)
// with the second factor from `steps` (backwards l^(jb-i) l^x); on the diagonal
// the first is above 1, where a strong decay takes an exponential for each
// element instead. Elements that a row does not see become zero whatever
// they are.
template <bool REV>
__device__ __forceinline__ void weigh(uint32_t t_p, int j0, int i, int w0, int n, float l2,
                                      float in_scale, const uint64_t (&steps)[8]) {
  uint32_t pk[16];
  const uint32_t to = t_p + (j0 & ~63) + (j0 & 32) / 2;
  if (REV ? w0 > j0 + 31 || j0 >= n : w0 + 31 < j0) {  // no row sees any
#pragma unroll
    for (int e = 0; e < 16; ++e) pk[e] = 0u;
  } else {
    uint32_t s[32];
    ht::tmem_ld(t_p + j0, s);
    const bool whole = REV ? j0 >= w0 + 31 && j0 + 32 <= n : w0 >= j0 + 31;
    if (whole || l2 >= DT_STRONG) {
      float f = in_scale * power(l2, REV ? j0 - i : i - j0 - 15);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint64_t ff = pack2(f, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 y = unpack2(ht::fmul2(ht::fmul2(steps[e], ff),
                                             ht::pair(s[16 * g + 2 * e], s[16 * g + 2 * e + 1])));
          s[16 * g + 2 * e] = __float_as_uint(y.x);
          s[16 * g + 2 * e + 1] = __float_as_uint(y.y);
        }
        if (g == 0) f = in_scale * power(l2, REV ? j0 + 16 - i : i - j0 - 31);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const int gap = max(0, REV ? j0 + e - i : i - j0 - e);
        s[e] = __float_as_uint(__uint_as_float(s[e]) * in_scale * power(l2, gap));
      }
    }
    if (!whole) {
      const int lo = REV ? i - j0 : 0, hi = REV ? n - 1 - j0 : i - j0;  // columns that count
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if ((REV && e < lo) || e > hi) s[e] = 0u;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      pk[e] = tc::pack_bf16x2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
  }
  ht::tmem_st(to, pk);
}

// 32 values times f
__device__ __forceinline__ void times(uint32_t (&v)[32], float f) {
  const uint64_t ff = pack2(f, f);
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const float2 y = unpack2(ht::fmul2(ht::pair(v[e], v[e + 1]), ff));
    v[e] = __float_as_uint(y.x);
    v[e + 1] = __float_as_uint(y.y);
  }
}

// D[tmem] (+)= C^T B over ROWS rows; both tiles by rows (MN-major operands)
template <int ROWS = DT_T>
__device__ __forceinline__ void issue_state(uint32_t tmem_d, uint64_t dc, uint64_t db,
                                            uint32_t idesc, bool add) {
#pragma unroll
  for (int ks = 0; ks < ROWS / 16; ++ks)
    tc::mma_bf16(tmem_d, dc + (uint64_t)((ks * 2048) >> 4), db + (uint64_t)((ks * 2048) >> 4),
                 idesc, add || ks > 0);
}

// C[tmem_d] += A . B^T, as ht::issue_scores
template <int NKS, int RB>
__device__ __forceinline__ void issue_scores_add(uint32_t tmem_d, uint64_t da, uint64_t db,
                                                 uint32_t idesc) {
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks)
    tc::mma_bf16(tmem_d, da + ht::kstep(ks, 128), db + ht::kstep(ks, RB), idesc, true);
}

// Shared memory: a and b of two chunks, c of one (two with two heads a unit,
// whose state is half as large), the state's copy in two parts.
template <bool PAIR>
struct DtPlan {
  static constexpr int CS = PAIR ? 2 : 1;
  static constexpr int COPY = PAIR ? DT_HALF : DT_TILE;
  static constexpr int AT_C = 4 * DT_TILE, AT_COPY = AT_C + CS * DT_TILE;
  static constexpr int SMEM = AT_COPY + 2 * COPY + 1024;
};

struct DtShared {
  // by chunk, in turn of two: pdone[c & 1] is P of chunk c, and so on
  uint64_t full_ab[2], empty_ab[2], full_c[2], empty_c[2], pdone[2], conv[2];
  uint64_t pready[2];  // by chunk, with two heads by head
  uint64_t s16, o1done, oscaled, udone, pvdone, ofree, drain;
  uint32_t tmem;
  int abort_flag;
};

template <int NKS, bool PAIR, int JOBS>
__global__ void __launch_bounds__(DT_THREADS, 1)
    decay_rows_tc_kernel(const __grid_constant__ DtJobs<JOBS> jobs, DtGrid g) {
  using Plan = DtPlan<PAIR>;
  constexpr int HEADS = PAIR ? 2 : 1, CS = Plan::CS;
  extern __shared__ unsigned char dt_raw[];
  __shared__ DtShared sh;
  const uint32_t base = (tc::smem_addr(dt_raw) + 1023u) & ~1023u;
  const uint32_t copy = base + Plan::AT_COPY;
  auto tile_a = [&](uint32_t c) { return base + (c & 1) * 2 * DT_TILE; };
  auto tile_b = [&](uint32_t c) { return base + (c & 1) * 2 * DT_TILE + DT_TILE; };
  auto tile_c = [&](uint32_t c) { return base + Plan::AT_C + (c % CS) * DT_TILE; };
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int job = JOBS == 1 ? 0 : blockIdx.x % JOBS;
  const int first_unit = blockIdx.x / JOBS, unit_step = gridDim.x / JOBS;
  const DecayParams& p = jobs.p[job];
  const CUtensorMap* map = jobs.map[job];
  const bool rev = JOBS > 1 && p.reverse, f32 = JOBS > 1 && p.out_f32;
  const bool transposed = JOBS > 1 && p.transposed;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&sh.full_ab[s], 1);
      tc::mbar_init(&sh.full_c[s], 1);
      tc::mbar_init(&sh.empty_ab[s], 8);
      tc::mbar_init(&sh.empty_c[s], 1);
      tc::mbar_init(&sh.pdone[s], 1);
      tc::mbar_init(&sh.conv[s], 8);
      tc::mbar_init(&sh.pready[s], 8 / HEADS);
    }
    tc::mbar_init(&sh.o1done, 1);
    tc::mbar_init(&sh.udone, 1);
    tc::mbar_init(&sh.pvdone, 1);
    tc::mbar_init(&sh.drain, 1);
    tc::mbar_init(&sh.s16, 8);
    tc::mbar_init(&sh.oscaled, 8);
    tc::mbar_init(&sh.ofree, 8);
    sh.abort_flag = 0;
    tc::mbar_init_fence();
  }
  if (warp == DT_MMA_WARP) tc::tmem_alloc(&sh.tmem, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sh.tmem, t_out = tmem + 256, t_state = tmem + 384;
  // P of a chunk: the unit's heads side by side, or two chunks in turn
  auto tmem_p = [&](uint32_t c, int u) { return tmem + (PAIR ? u : (int)(c & 1)) * 128; };
  // does a unit's first chunk start from a state?
  auto starts = [&](const DtUnit& w) {
    return p.part ? w.seg > 0 || p.start : p.start != nullptr;
  };

  if (warp == DT_TMA_WARP) {
    if (lane == 0) {
      uint32_t c = 0, cc = 0;  // copies of a and b, of c
      for (int k = 0, unit = first_unit; unit < g.units; unit += unit_step, ++k) {
        if (ht::gives_up(ht::ROLE_LOADER, k)) {
          *abort_flag = 1;
          break;
        }
        const DtUnit w = dt_unit<PAIR>(p, g, unit);
        for (int x = w.a0; x < w.a1; ++x) {
          const int s = c & 1, row = dt_chunk(p, g, x) * DT_T;
          if (!ws::wait(&sh.empty_ab[s], ((c >> 1) & 1) ^ 1, abort_flag)) goto tma_done;
          ht::expect_tx(&sh.full_ab[s], 2 * DT_TILE);
          dt_load<PAIR>(tile_a(c), map, &sh.full_ab[s], p, w, p.ga, row);
          dt_load<PAIR>(tile_b(c), map + 1, &sh.full_ab[s], p, w, p.gb, row);
          ++c;
          const int t = cc % CS;
          if (!ws::wait(&sh.empty_c[t], ((cc / CS) & 1) ^ 1, abort_flag)) goto tma_done;
          ht::expect_tx(&sh.full_c[t], DT_TILE);
          dt_load<PAIR>(tile_c(cc), map + 2, &sh.full_c[t], p, w, p.gc, row);
          ++cc;
        }
      }
    tma_done:
      ht::drain_copies(sh.full_ab, 2, c);
      ht::drain_copies(sh.full_c, CS, cc);
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
    bool formed = false;         // is P of chunk c?
    auto wait = [&](uint64_t& bar, uint32_t parity) {
      ok = ok && ht::wait_at(tc::smem_addr(&bar), parity, abort_flag);
    };
    // have a and b of chunk c_ landed?
    auto landed = [&](uint32_t c_) {
      return __all_sync(0xffffffffu, ws::test(&sh.full_ab[c_ & 1], (c_ >> 1) & 1));
    };
    auto form_p = [&](uint32_t c_) {  // P of chunk c_
      wait(sh.full_ab[c_ & 1], (c_ >> 1) & 1);
      tc::fence_after_sync();
      if (ok && leader) {
#pragma unroll
        for (int u = 0; u < HEADS; ++u)
          ht::issue_scores<NKS, 128>(tmem_p(c_, u), ht::desc128(tile_a(c_) + u * DT_HALF, 16),
                                     ht::desc128(tile_b(c_) + u * DT_HALF, 16), id_p);
        ht::commit_at(tc::smem_addr(&sh.pdone[c_ & 1]));
      }
      __syncwarp();
    };
    for (int unit = first_unit; unit < g.units && ok; unit += unit_step) {
      const DtUnit w = dt_unit<PAIR>(p, g, unit);
      for (int x = w.a0; x < w.a1 && ok; ++x, ++c) {
        const bool state = x > w.a0 || starts(w);
        const uint32_t odd = c & 1, ph = (c >> 1) & 1;
        if (!formed) form_p(c);
        formed = false;
        wait(sh.ofree, odd ^ 1);  // the rows of the chunk before are out
        if (state) {
          wait(sh.s16, states & 1);
          tc::fence_after_sync();
          if (ok && leader) {
#pragma unroll
            for (int u = 0; u < HEADS; ++u) {
              const uint64_t da = ht::desc128(tile_a(c) + u * DT_HALF, 16);
              const uint32_t at = copy + u * 64 * 128;
              ht::issue_scores<NKS, 128>(t_out + u * 64, da, ht::desc128(at, 16), id_1);
              issue_scores_add<NKS, 128>(t_out + u * 64, da, ht::desc128(at + Plan::COPY, 16), id_1);
            }
            ht::commit_at(tc::smem_addr(&sh.o1done));
          }
          __syncwarp();
        }
        wait(sh.full_c[c % CS], (c / CS) & 1);
        wait(sh.conv[odd], ph);
        tc::fence_after_sync();
        const uint64_t dc = ht::desc128(tile_c(c), DT_HALF);
        if (x + 1 < w.a1) {
          if (ok && leader) {
            issue_state(t_state, dc, ht::desc128(tile_b(c), DT_HALF), id_s, state);
            ht::commit_at(tc::smem_addr(&sh.udone));
          }
          __syncwarp();
        }
        // one head: the next chunk's P, this unit's or the next one's, goes ahead of
        // this one's P c
        if (!PAIR && landed(c + 1)) {
          form_p(c + 1);
          formed = true;
        }
        if (state) {
          wait(sh.oscaled, states & 1);
          ++states;
        }
#pragma unroll
        for (int u = 0; u < HEADS; ++u) {
          wait(sh.pready[PAIR ? u : odd], PAIR ? odd : ph);
          tc::fence_after_sync();
          if (ok && leader)
            ht::issue_aggregate<DT_T, 64>(t_out + u * 64, tmem_p(c, u), dc + u * (DT_HALF >> 4),
                                          id_2, state);
          __syncwarp();
        }
        if (ok && leader) {
          ht::commit_at(tc::smem_addr(&sh.pvdone));
          ht::commit_at(tc::smem_addr(&sh.empty_c[c % CS]));
        }
        ok = ht::agree(ok);
      }
    }
    // the last products are done before the block ends
    if (c > 0 && ok)
      ok = ht::wait_at(tc::smem_addr(&sh.empty_c[(c - 1) % CS]), ((c - 1) / CS) & 1, abort_flag);
    if (!ht::agree(ok)) ht::drain_products(&sh.drain, leader);
    __syncwarp();
  } else if (warp >= DT_W0 && warp < DT_W0 + 8) {
    // ---------------- weights of P, and the rows ----------------
    // one head: columns [64 half, 64 half + 64) of P and of the rows; two:
    // all of head `half`
    const int half = (warp - DT_W0) >> 2, i = threadIdx.x & 127, w0 = (warp & 3) * 32;
    const uint32_t lane_off = (uint32_t)w0 << 16;
    const int c_lo = PAIR ? 0 : half * 64, c_n = max(0, min(64, p.d - c_lo));
    // The tile that holds the rows of chunk c - 1 may be loaded again once they
    // have been read: asked for only when the next chunk is under way.
    bool held = false;
    uint32_t c = 0;
    auto release = [&] {
      if (held && lane == 0) {
        stores_read();
        ws::arrive(&sh.empty_ab[(c - 1) & 1]);
      }
      held = false;
      __syncwarp();
    };
    // the rows have been read from TMEM
    auto rows_free = [&] {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) ws::arrive(&sh.ofree);
    };
    bool ok = true;
    for (int k = 0, unit = first_unit; unit < g.units; unit += unit_step, ++k) {
      const DtUnit w = dt_unit<PAIR>(p, g, unit);
      if (ht::gives_up(ht::ROLE_WEIGHTS, k)) {
        ok = false;
        *abort_flag = 1;
      }
      const int h = PAIR ? min(w.h + half, p.H - 1) : w.h;
      const bool mine = !PAIR || w.h + half < p.H;
      const float l2 = decay_rate(p.log_decay, h) * DT_LOG2E;
      uint64_t steps[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        steps[e] = rev ? pack2(power(l2, 2 * e), power(l2, 2 * e + 1))
                       : pack2(power(l2, 15 - 2 * e), power(l2, 14 - 2 * e));
      for (int x = w.k0; x < w.k1; ++x) {
        const int chunk = dt_chunk(p, g, x);
        const bool live = x >= w.a0 && x < w.a1;
        const int n = live ? dt_rows(w, chunk) : 0;
        if (live) {
          if (ok) ok = ht::warp_wait(&sh.pdone[c & 1], (c >> 1) & 1, abort_flag);
          if (ok) {
            tc::fence_after_sync();
#pragma unroll 1
            for (int j0 = PAIR ? 0 : half * 64, q = 0; q < 2 * HEADS; ++q, j0 += 32) {
              if (q == HEADS) release();
              const uint32_t t_p = tmem_p(c, half) + lane_off;
              if (rev)
                weigh<true>(t_p, j0, i, w0, n, l2, p.in_scale, steps);
              else
                weigh<false>(t_p, j0, i, w0, n, l2, p.in_scale, steps);
            }
            ht::st_wait();
            tc::fence_before_sync();
          }
          __syncwarp();
          if (ok && lane == 0) ws::arrive(&sh.pready[PAIR ? half : c & 1]);
          if (ok) ok = ht::warp_wait(&sh.pvdone, c & 1, abort_flag);
          tc::fence_after_sync();
          ++c;
        }
        const int64_t first = (((int64_t)w.b * p.N + chunk * DT_T + w0) * p.H + h) * p.d + c_lo;
        const int left = mine ? p.N - chunk * DT_T - w0 : 0;  // rows of this warp to write
        if (live && ok) {
          // through shared memory (the chunk's a has been used), so that a
          // store takes whole lines
          const uint32_t stage = tile_a(c - 1) + (warp - DT_W0) * 4096;
          uint32_t o[32];
          auto part = [&](int col) {
            ht::tmem_ld(t_out + half * 64 + col + lane_off, o);
            times(o, p.out_scale);
            if (n < DT_T && i >= n) {  // padding
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
          };
          auto store = [&](int col) {
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0 && left > 0) store_box(map + 3, stage, c_lo + col, h, chunk * DT_T + w0, w.b);
            __syncwarp();
          };
          part(0);
          if (!f32) {
            stage_row(stage, lane, 0, o);
            part(32);
            stage_row(stage, lane, 4, o);
            rows_free();
            if (c_n > 0) store(0);
          } else {
            stage_row32(stage, lane, o);
            if (c_n > 0) store(0);
            part(32);
            rows_free();
            if (lane == 0) stores_read();
            __syncwarp();
            stage_row32(stage, lane, o);
            if (c_n > 32) store(32);
          }
          held = true;
        } else {
          // padding, or rows given up
          if (f32)
            fill_rows(static_cast<float*>(p.out) + first, ok ? 0u : 0x7fffffffu, lane, left,
                      (int64_t)p.H * p.d, c_n, 4);
          else
            fill_rows(static_cast<__nv_bfloat16*>(p.out) + first, ok ? 0u : 0x7fff7fffu, lane, left,
                      (int64_t)p.H * p.d, c_n, 8);
        }
      }
    }
    release();
  } else if (warp >= DT_W0 + 8) {
    // ---------------- the state ----------------
    const int half = (warp - DT_W0 - 8) >> 2, r = threadIdx.x & 127;
    const int tid = threadIdx.x - (DT_W0 + 8) * 32;  // 0 .. 255
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    // this thread's part of S: row r (a column of c), from column s_col on
    constexpr int SP = PAIR ? 1 : 2;  // pieces of 32 columns (of b)
    const int s_head = PAIR ? r >> 6 : 0;
    const int s_col = half * (PAIR ? 32 : 64);  // inside the head
    const uint32_t t_s = t_state + (PAIR ? s_head * 64 : 0) + s_col + lane_off;
    const uint32_t t_o = t_out + half * 64 + lane_off;
    // a warp that gave up leaves: it must not touch what the others still use
    bool ok = true;
    uint32_t c = 0, states = 0, us = 0;
    for (int unit = first_unit; unit < g.units && ok; unit += unit_step) {
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
      // weights of a whole chunk; a chunk of fewer rows makes its own. `whole` is off
      // by up to 2^-22 in every chunk, 5e-5 of the norm after 512 of slow decays: below
      // the rows' bf16, where what the states' kernel does about it took 3 to 20 %.
      float f0[4], f1[4];
      auto weights = [&](int n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = (tid >> 3) + 32 * e, to = max(0, rev ? row + 1 : n - 1 - row);
          f0[e] = p.in_scale * power(l2_0, to);
          f1[e] = PAIR ? p.in_scale * power(l2_1, to) : 0.f;
        }
      };
      weights(DT_T);
      const float whole = power(l2_s, DT_T), row_whole = power(l2_o, rev ? DT_T - 1 - r : r + 1);
      // b of chunk c_, the unit's x_, weighted in place once P is formed
      auto convert = [&](uint32_t c_, int x_) {
        const int n = dt_rows(w, dt_chunk(p, g, x_));
        ok = ht::warp_wait(&sh.full_ab[c_ & 1], (c_ >> 1) & 1, abort_flag) &&
             ht::warp_wait(&sh.pdone[c_ & 1], (c_ >> 1) & 1, abort_flag);
        if (!ok) return;
        if (x_ + 1 < w.a1) {
          if (n < DT_T) weights(n);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const uint32_t at = tile_b(c_) + hf * DT_HALF + tid * 16;
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = ld_piece(at + e * 4096);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              st_piece(at + e * 4096, weighted(v[e], PAIR && hf ? f1[e] : f0[e]));
          }
          if (n < DT_T) {
            weights(DT_T);
#pragma unroll 1
            for (int piece = tid; piece < 2048; piece += 256)
              if (((piece & 1023) >> 3) >= n) st_shared_zero16(tile_b(c_) + piece * 16);
          }
        }
        if (n < DT_T && w.len < p.N) {
          // rows from the length on may hold anything: those of c become zero
          ok = ht::warp_wait(&sh.full_c[c_ % CS], (c_ / CS) & 1, abort_flag);
          if (!ok) return;
#pragma unroll 1
          for (int piece = tid; piece < 2048; piece += 256)
            if (((piece & 1023) >> 3) >= n) st_shared_zero16(tile_c(c_) + piece * 16);
        }
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) ws::arrive(&sh.conv[c_ & 1]);
      };
      for (int x = w.a0; x < w.a1; ++x, ++c) {
        const int chunk = dt_chunk(p, g, x), n = dt_rows(w, chunk);
        const bool state = x > w.a0 || start;
        if (state) {
          // the state before this chunk: its copy, and what the product adds to
          const float all = n < DT_T ? power(l2_s, n) : whole;
          if (x > w.a0) {
            ok = ht::warp_wait(&sh.udone, us & 1, abort_flag);
            if (!ok) break;
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
                s[e] = in ? __float_as_uint(__ldg(start + (transposed ? rc * p.d + bc
                                                                        : bc * p.d + rc)))
                          : 0u;
              }
            }
            const uint32_t row = copy + (PAIR ? 0 : (b0 >> 6) * DT_HALF) + r * 128;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                float y = __uint_as_float(s[e + 2 * v]), z = __uint_as_float(s[e + 2 * v + 1]);
                hi[v] = split_off(y, z);
                lo[v] = tc::pack_bf16x2(y, z);
              }
              const uint32_t to = row + (((((b0 & 63) + e) >> 3) ^ (r & 7)) << 4);
              st_piece(to, make_uint4(hi[0], hi[1], hi[2], hi[3]));
              st_piece(to + Plan::COPY, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            if (x + 1 < w.a1) {
              times(s, all);
              ht::tmem_st(t_s + 32 * q, s);
            }
          }
          ht::st_wait();
          tc::fence_before_sync();
          tc::fence_async_smem();
          __syncwarp();
          if (lane == 0) ws::arrive(&sh.s16);
        }
        convert(c, x);
        if (!ok) break;
        if (state) {
          ok = ht::warp_wait(&sh.o1done, states & 1, abort_flag);
          if (!ok) break;
          ++states;
          tc::fence_after_sync();
          const float f = rev && n < DT_T ? power(l2_o, max(0, n - 1 - r)) : row_whole;
#pragma unroll 1
          for (int q = 0; q < 2; ++q) {
            uint32_t o[32];
            ht::tmem_ld(t_o + 32 * q, o);
            times(o, f);
            ht::tmem_st(t_o + 32 * q, o);
          }
          ht::st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) ws::arrive(&sh.oscaled);
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
// A chunk is split and multiplied by halves of 64 rows: one half's product runs
// while the other is split, and the lower parts need one place only.
template <int PLANES>
struct DsTcPlan {
  static constexpr int NS = PLANES == 1 ? 3 : 2;
  static constexpr int SMEM = (2 * NS + PLANES - 1) * DT_TILE + 1024;
};
template <int NS>
struct DsTcShared {
  uint64_t full[NS], empty[NS];
  uint64_t conv[2], done[2];  // by half: split, multiplied
  uint64_t drain;
  uint32_t tmem;
  int abort_flag;
};

// The decay l^128 = hi + lo of whole chunks; out of line, as most of the kernel never
// needs its registers (2 x 8192 rows of 16 heads on 4: 33.9 us, 34.6 in line).
__device__ __noinline__ DecayFactor whole_chunk(const float* log_decay, int h) {
  return DecayFactor::make(decay_rate(log_decay, h), (float)DT_T);
}
// That of the k-th whole chunk of a walk: fp32 numbers around l^128, in [1/2, 1] where
// lo is not zero, whose sum is that of as many l^128 to 2^-24. One number for all
// would be off by the same rounding, the exponential's 2^-22, in every chunk (512
// chunks of slow decays: 1.8e-5 of the state's norm off 64 bits, 7e-7).
__device__ __forceinline__ float chunk_decay(const DecayFactor& l, int k) {
  auto steps = [](float x) { return (x + 0.75f) - 0.75f; };  // to a multiple of 2^-24
  return l.hi + (steps((float)(k + 1) * l.lo) - steps((float)k * l.lo));
}

template <bool PAIR, int PLANES>
__global__ void __launch_bounds__(DT_THREADS, 1)
    decay_state_tc_kernel(const __grid_constant__ CUtensorMap mb,
                          const __grid_constant__ CUtensorMap mc, DecayParams p, DtGrid g) {
  constexpr int NS = DsTcPlan<PLANES>::NS;
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
    for (int q = 0; q < 2; ++q) {
      tc::mbar_init(&sh.conv[q], 16);
      tc::mbar_init(&sh.done[q], 1);
    }
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
        const uint32_t d = tmem + (c & 1) * 128;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          ok = ok && ht::wait_at(tc::smem_addr(&sh.conv[hf]), c & 1, abort_flag);
          tc::fence_after_sync();
          if (ok && leader) {
            const uint32_t rows = hf * DT_HALF / 2;  // bytes of half a tile's rows
            const uint64_t dc = ht::desc128(at + DT_TILE + rows, DT_HALF);
#pragma unroll
            for (int q = 0; q < PLANES; ++q)
              issue_state<DT_T / 2>(
                  d, dc, ht::desc128((q ? extra + (q - 1) * DT_TILE : at) + rows, DT_HALF), id_s,
                  hf || q);
            ht::commit_at(tc::smem_addr(&sh.done[hf]));
            if (hf) ht::commit_at(tc::smem_addr(&sh.empty[s]));
          }
          __syncwarp();
        }
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
      DecayFactor whole = {};  // once the first chunk is under way
      float S[SC];
#pragma unroll
      for (int e = 0; e < SC; ++e) S[e] = 0.f;
      // S = l^n S + the product of chunk c_, the unit's k-th
      auto take = [&](uint32_t c_, int n, int k) {
        if (ok) ok = ht::warp_wait(&sh.done[1], c_ & 1, abort_flag);
        if (!ok) return;
        tc::fence_after_sync();
        uint32_t u[SC];
        tmem_ld_n(t_s + (c_ & 1) * 128, u);
        const float all = n < DT_T || k == 0 ? power(l2_s, n) : chunk_decay(whole, k);
#pragma unroll
        for (int e = 0; e < SC; ++e) S[e] = fmaf(all, S[e], __uint_as_float(u[e]));
        tc::fence_before_sync();
      };
      int n_before = 0;
      // weights of a whole chunk; a chunk of fewer rows makes its own
      float f[4];
      auto weights = [&](int n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = ((tid + 512 * e) & 1023) >> 3;
          f[e] = p.in_scale * power(PAIR && e >= 2 ? l2_1 : l2_0,
                                    max(0, p.reverse ? row + 1 : n - 1 - row));
        }
      };
      weights(DT_T);
      for (int x = w.a0; x < w.a1; ++x, ++c) {
        const int n = dt_rows(w, dt_chunk(p, g, x)), s = c % NS;
        if (n < DT_T) weights(n);
        if (ok) ok = ht::warp_wait(&sh.full[s], (c / NS) & 1, abort_flag);
        // a warp that gave up does not touch what the others still use
        if (!ok) continue;
        const uint32_t at = base + s * 2 * DT_TILE;
        // pieces tid + 512 e: those with e = hf and hf + 2 are rows of half hf
        uint4 v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ld_piece(at + (tid + 512 * e) * 16);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          // This half of the chunk before is multiplied: its lower parts may go, and
          // the issuing warp has seen its conv. (A unit ends with a take.)
          if (x > w.a0) {
            if (hf)
              take(c - 1, n_before, x - 1 - w.a0);
            else
              ok = ht::warp_wait(&sh.done[0], (c - 1) & 1, abort_flag);
          }
          if (!ok) break;
#pragma unroll
          for (int e = hf; e < 4; e += 2) {
            const int piece = tid + 512 * e;
            if constexpr (PLANES == 1) {
              st_piece(at + piece * 16, weighted(v[e], f[e]));
            } else {
              const uint32_t in[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
              uint32_t part[PLANES][4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float a = lo_half(in[i]) * f[e], b = hi_half(in[i]) * f[e];
#pragma unroll
                for (int q = 0; q < PLANES; ++q) part[q][i] = split_off(a, b);
              }
              st_piece(at + piece * 16, make_uint4(part[0][0], part[0][1], part[0][2], part[0][3]));
#pragma unroll
              for (int q = 1; q < PLANES; ++q)
                st_piece(extra + (q - 1) * DT_TILE + piece * 16,
                         make_uint4(part[q][0], part[q][1], part[q][2], part[q][3]));
            }
          }
          if (n < (hf + 1) * DT_T / 2) {  // rows that are not there, whatever the tiles hold
#pragma unroll 1
            for (int e = hf; e < 4; e += 2) {
              const int piece = tid + 512 * e;
              if (((piece & 1023) >> 3) < n) continue;
              st_shared_zero16(at + piece * 16);
              for (int q = 1; q < PLANES; ++q)
                st_shared_zero16(extra + (q - 1) * DT_TILE + piece * 16);
              if (w.len < p.N) st_shared_zero16(at + DT_TILE + piece * 16);
            }
          }
          tc::fence_async_smem();
          __syncwarp();
          if (lane == 0) ws::arrive(&sh.conv[hf]);
        }
        if (n < DT_T) weights(DT_T);
        if (x == w.a0 && x + 1 < w.a1)
          whole = whole_chunk(p.log_decay, s_head ? h1 : h0);
        n_before = n;
      }
      if (w.a1 > w.a0) take(c - 1, n_before, w.a1 - 1 - w.a0);
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
int dt_blocks(const DtGrid& g, int jobs) {
  const int most = head_sm_count() / jobs;
  return jobs * (g.units < most ? g.units : most);
}

template <int NKS, bool PAIR, int JOBS>
cudaError_t rows_go(const DtJobs<JOBS>& jobs, const DtGrid& g, cudaStream_t s) {
  constexpr int SMEM = DtPlan<PAIR>::SMEM;
  const void* fn = reinterpret_cast<const void*>(&decay_rows_tc_kernel<NKS, PAIR, JOBS>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  decay_rows_tc_kernel<NKS, PAIR, JOBS><<<dt_blocks(g, JOBS), DT_THREADS, SMEM, s>>>(jobs, g);
  return cudaGetLastError();
}
template <bool PAIR, int PLANES>
cudaError_t state_go(const CUtensorMap* m, const DecayParams& p, const DtGrid& g, cudaStream_t s) {
  constexpr int SMEM = DsTcPlan<PLANES>::SMEM;
  const void* fn = reinterpret_cast<const void*>(&decay_state_tc_kernel<PAIR, PLANES>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  decay_state_tc_kernel<PAIR, PLANES><<<dt_blocks(g, 1), DT_THREADS, SMEM, s>>>(m[0], m[1], p, g);
  return cudaGetLastError();
}

bool map_of(CUtensorMap* m, const DecayParams& p, const void* ptr, const HeadStrides& s,
            int share) {
  return head_tensor_map(m, ptr, s, p.B, p.N, p.H / share, p.d);
}

}  // namespace

// Segments of a call of `jobs` sums, by the longest walk of a block in chunks: a
// unit costs one and a half beside its own, a chunk of the states' pass two
// thirds of one, its launch and the joining four. The gradients' three sums need
// two such passes. Host arithmetic for 148 SMs, so that a caller can ask for the
// scratch without a GPU. 2 x 8192 rows of 16 heads, d = 128, gradients: 96 units
// of 64 chunks 184 us, three segments with their states 219 (an earlier form of
// the rows' kernel).
DecayPlan decay_plan_tc(int B, int N, int H, int d, int jobs) {
  const int64_t heads = (int64_t)B * (d <= 64 ? cdiv(H, 2) : H);
  const int chunks = cdiv(N, DT_T);
  DecayPlan best = {1, chunks};
  double least = 0;
  for (int want = 1; want <= chunks && want <= 256; ++want) {
    const int per = cdiv(chunks, want), segs = cdiv(chunks, per);
    const int blocks = 148 / jobs;
    double cost = (double)((heads * segs + blocks - 1) / blocks) * (per + 1.5);
    if (segs > 1)
      cost += (jobs > 1 ? 2 : 1) *
              ((double)((heads * (segs - 1) + 147) / 148) * (per + 1.5) * 0.65 + 4.0);
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
  if (p.d <= 64) return p.planes > 2 ? state_go<true, 3>(m, p, g, s) : state_go<true, 1>(m, p, g, s);
  return p.planes > 2 ? state_go<false, 3>(m, p, g, s) : state_go<false, 1>(m, p, g, s);
}

template <int JOBS>
cudaError_t launch_jobs(const DecayParams* p, cudaStream_t s) {
  DtJobs<JOBS> all;
  for (int j = 0; j < JOBS; ++j) {
    const DecayParams& q = p[j];
    const HeadStrides so = {(int64_t)q.N * q.H * q.d, (int64_t)q.H * q.d, q.d};
    CUtensorMap* m = all.map[j];
    if (!map_of(&m[0], q, q.a, q.sa, q.ga) || !map_of(&m[1], q, q.b, q.sb, q.gb) ||
        !map_of(&m[2], q, q.c, q.sc, q.gc) ||
        !head_box_map(&m[3], q.out, so, q.B, q.N, q.H, q.d, q.out_f32, 32))
      return cudaErrorInvalidValue;
    all.p[j] = q;
  }
  const DtGrid g = dt_grid(p[0], p[0].segs);
  if (p[0].d <= 64) return rows_go<4, true, JOBS>(all, g, s);
  if (p[0].d <= 96) return rows_go<6, false, JOBS>(all, g, s);
  return rows_go<8, false, JOBS>(all, g, s);
}
cudaError_t launch_decay_rows_tc(const DecayParams* p, int jobs, cudaStream_t s) {
  if (jobs == 3) return launch_jobs<3>(p, s);
  // a single one is the forward pass's
  if (jobs != 1 || p->reverse || p->transposed || p->out_f32) return cudaErrorInvalidValue;
  return launch_jobs<1>(p, s);
}

}  // namespace tarmac
