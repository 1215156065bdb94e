// decay_scan.cu — attention with a decay for each head over a set of rows, the
// recurrent form (fp32 rows, and bf16 rows that decay_tc.cu leaves), and what
// joins the states of segments.
//
//   S = l S + b c^T,  out = S^T a,  row_out = S e   for one row after the other.
// In fp32 this form takes 5 d^2 operations a row, fewer than any chunk form
// (three tf32 products for one on the tensor cores: 64 x 512 rows of 4 heads,
// d = 16, with gradients 166 us), and no operand is rounded. Up to 32 columns
// the gradients need no transposed state: dq = S dout is a row_out, and one
// walk backwards over R = l R + q dout^T gives dv = R^T k and dk = R v.
//
// A warp takes 32 columns of c of one head (two heads of up to 16 columns) and
// walks over the rows of a segment with its part of S in registers: lanes are
// NG groups of rows by 32 / NG groups of columns, a lane holds R rows (of b) by
// C columns. a and b are read from shared memory by the lanes of a row group, c
// and e by those of a column group; the sum over the row groups halves the
// columns with each exchange. For that a lane holds column j ^ (its row group)
// in place j: what it passes on is always the upper half. Rows come in tiles by
// asynchronous copies, one tile ahead.
// Bound by issue: at d = 32 a row takes 96 clocks of a scheduler's FMA pipe and
// about as many slots for reads, copies into pairs and sums. Measured, gradients
// with the forward pass: 64 x 512 rows of 4 heads, d = 16, 84 us; 300 x 723 rows
// of 8 heads, d = 32, 1211 us (FMA pipe 56-62 %, issue 51-60 % of the peak); 32 x
// 512 rows of 4 heads, d = 64, 351 us.
//
// Where episodes and heads are too few to fill the GPU the row axis is cut in
// segments: a first launch forms what each segment adds to the state; up to 32
// columns the rows' kernel puts those before its segment together itself, else a
// second launch joins them.
#include <type_traits>

#include "decay.cuh"

namespace tarmac {

namespace {

constexpr int SC_WARPS = 2;  // of a block; they do not meet

template <typename T, int DP>
struct ScPlan {
  static constexpr int NG = DP == 16 ? 4 : 8;       // groups of rows (of S)
  static constexpr int C = DP == 16 ? 4 : 8;        // columns of a lane
  static constexpr int R = DP / NG;                 // rows of a lane
  static constexpr int HEADS = DP == 16 ? 2 : 1;    // heads of a warp
  static constexpr int COLS = DP == 16 ? 16 : 32;   // columns of a warp and head
  static constexpr int PARTS = DP / COLS;           // warps of a head
  static constexpr bool WHOLE = PARTS == 1;         // the warp has all of S
  static constexpr int TT = DP >= 128 ? 4 : (DP >= 64 ? 8 : 16);  // rows of a tile
  static constexpr int BLOCKS = DP == 16 ? 10 : (DP == 32 ? 8 : (DP == 64 ? 6 : 4));  // of an SM
};

enum ScMode { SC_STATES = 0, SC_COLS = 1, SC_ROWS = 2 };  // SC_COLS | SC_ROWS: both

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The rows of a lane as pairs: four neighbours of each 4 NG, so that the lanes
// of a load are neighbours too. p: its first.
template <int R, int NG>
__device__ __forceinline__ void read_pairs(uint64_t (&x)[R / 2], const float* p) {
#pragma unroll
  for (int i = 0; i < R / 2; i += 2) {
    const float4 v = *reinterpret_cast<const float4*>(p + 2 * i * NG);
    x[i] = pack2(v.x, v.y);
    x[i + 1] = pack2(v.z, v.w);
  }
}
template <int R, int NG>
__device__ __forceinline__ void read_pairs(uint64_t (&x)[R / 2], const __nv_bfloat16* p) {
#pragma unroll
  for (int i = 0; i < R / 2; i += 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p + 2 * i * NG);
    x[i] = pack2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u));
    x[i + 1] = pack2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
  }
}

template <typename T, int DP, bool REV, int MODE>
__global__ void __launch_bounds__(SC_WARPS * 32, ScPlan<T, DP>::BLOCKS)
    decay_scan_kernel(DecayParams p, unsigned warps) {
  using Plan = ScPlan<T, DP>;
  constexpr int NG = Plan::NG, C = Plan::C, R = Plan::R, HEADS = Plan::HEADS, TT = Plan::TT;
  constexpr int COLS = Plan::COLS, PARTS = Plan::PARTS, E = 16 / (int)sizeof(T);
  constexpr bool OUT_C = MODE & SC_COLS, OUT_R = MODE & SC_ROWS, STATES = MODE == SC_STATES;
  // The states' walk runs against the rows': S = sum_j l^(n-1-j) b_j c_j^T needs
  // no decay of S then, only the weight of each b.
  constexpr int DIR = REV != STATES ? -1 : 1;
  static_assert(!OUT_R || Plan::WHOLE, "row_out needs all columns");
  // a staged row: b, c, and a or e or both; a head's tile, off the banks of the
  // other's
  constexpr int AT_C = DP, AT_A = AT_C + COLS, AT_E = AT_A + (OUT_C ? DP : 0);
  constexpr int ROW = AT_E + (OUT_R ? COLS : 0);
  constexpr int HEAD = TT * ROW + (HEADS == 2 ? 64 / (int)sizeof(T) : 0), TILE = HEADS * HEAD;
  extern __shared__ __align__(16) unsigned char sc_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, seg = blockIdx.y;
  const unsigned unit = blockIdx.x * SC_WARPS + warp;
  if (unit >= warps) return;
  T* tiles = reinterpret_cast<T*>(sc_smem) + warp * 2 * TILE;
  const int part = unit % PARTS;
  const unsigned heads = (unsigned)p.B * (unsigned)p.H, bh0 = unit / PARTS * HEADS;
  const int own = HEADS == 2 ? lane >> 4 : 0;  // this lane's head of the warp
  const int sub = HEADS == 2 ? lane & 15 : lane;
  const int rg = sub % NG, cg = sub / NG;
  const int s0 = seg * p.seg_chunks * DECAY_CHUNK;
  // rows in the order they enter S, x in [s0, s1): backwards from the end of the
  // last chunk, so that segments are the same rows in either direction
  const int end = REV ? cdiv(p.N, DECAY_CHUNK) * DECAY_CHUNK : p.N;
  const int s1 = min(end, s0 + p.seg_chunks * DECAY_CHUNK);
  // the warp's heads: operands from row 0 on, and rows
  const T *src_a[HEADS], *src_b[HEADS], *src_c[HEADS], *src_e[HEADS];
  int src_len[HEADS], b = 0, h = 0, len = 0, most = 0;
  {
    int ub = bh0 / (unsigned)p.H, uh = bh0 - (unsigned)ub * p.H;
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      const bool there = bh0 + u < heads;
      const int xb = there ? ub : 0, xh = there ? uh : 0;
      src_len[u] = there ? decay_len(p, xb) : 0;
      most = max(most, src_len[u]);
      src_b[u] = static_cast<const T*>(p.b) + xb * p.sb.b + (xh / p.gb) * p.sb.h;
      src_c[u] = static_cast<const T*>(p.c) + xb * p.sc.b + (xh / p.gc) * p.sc.h + part * COLS;
      if (OUT_C) src_a[u] = static_cast<const T*>(p.a) + xb * p.sa.b + (xh / p.ga) * p.sa.h;
      if (OUT_R) src_e[u] = static_cast<const T*>(p.e) + xb * p.se.b + (xh / p.ge) * p.se.h;
      if (u == own) {
        b = xb;
        h = xh;
        len = src_len[u];
      }
      if (++uh == p.H) {
        uh = 0;
        ++ub;
      }
    }
  }
  const bool there = bh0 + own < heads;
  // A rounded decay would be off by the same 2^-25 in every row: one row in 16 takes
  // one that makes up for the 16 and for what its own rounding left before (16384
  // rows of slow decays: 1.9e-6 of the norm off 64 bits, with one that repeats its
  // rounding 1.3e-5).
  const float rate = decay_rate(p.log_decay, h);
  // FAR: what that takes stays in shared memory between uses, where registers are
  // short (300 x 512 rows of 8 heads, d = 32: 259 us, 289 without; the other kernels
  // are up to 6 % slower with it).
  constexpr bool FAR = DP == 32 && MODE == SC_COLS;
  DecayFactor l16 = DecayFactor::make(rate, 1.f, 16.f);
  const float l = l16.hi;
  __shared__ float2 far[FAR ? SC_WARPS * 32 : 1];
  if (FAR) far[threadIdx.x] = make_float2(l16.lo, l16.left);
  // those that some head of the warp has, and how they are walked: y in [0, n)
  const int x0 = REV ? max(s0, end - most) : s0, x1 = REV ? s1 : min(s1, most);
  const int rows = x1 - x0, row0 = REV ? (STATES ? end - x1 : end - 1 - x0) : (STATES ? x1 - 1 : x0);
  auto row_at = [&](int y) { return row0 + DIR * y; };

  // first row of pair i and column of place j, inside the head
  auto row_of = [&](int i) { return (i >> 1) * 4 * NG + rg * 4 + (i & 1) * 2; };
  auto place = [&](int j) { return OUT_C ? j ^ rg : j; };  // column of place j in its group
  auto col_of = [&](int j) { return part * COLS + cg * C + place(j); };
  const int dd = p.d * p.d;
  const int64_t state_at = ((int64_t)b * p.H + h) * dd;
  auto state_index = [&](int r, int c) { return p.transposed ? c * p.d + r : r * p.d + c; };
  // rows of this lane's head in segment s
  auto rows_in = [&](int s) {
    const int t0 = s * p.seg_chunks * DECAY_CHUNK, t1 = min(end, t0 + p.seg_chunks * DECAY_CHUNK);
    return REV ? max(0, t1 - max(t0, end - len)) : max(0, min(t1, len) - t0);
  };
  // S over in_scale: in_scale comes back with the rows and the state
  uint64_t S[R / 2][C];
#pragma unroll
  for (int i = 0; i < R / 2; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) S[i][j] = 0;
  const bool parts = Plan::WHOLE && p.segs > 1;  // p.part as the lanes hold it
  constexpr int LANE_PARTS = 32 * (R / 2) * C;   // pairs of a warp
  uint64_t* own_part =
      reinterpret_cast<uint64_t*>(p.part) + (int64_t)unit * LANE_PARTS + lane;
  const int64_t part_step = (int64_t)warps * LANE_PARTS;  // from segment to segment
  const float* src = nullptr;
  if (!STATES && there)
    src = p.segs > 1 && !parts ? p.part + (int64_t)seg * heads * dd + state_at
                               : (p.start ? p.start + state_at : nullptr);
  if (src) {
    const float inv = 1.f / p.in_scale;
#pragma unroll
    for (int i = 0; i < R / 2; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int r = row_of(i), c = col_of(j);
        const float x = r < p.d && c < p.d ? src[state_index(r, c)] * inv : 0.f;
        const float y = r + 1 < p.d && c < p.d ? src[state_index(r + 1, c)] * inv : 0.f;
        S[i][j] = pack2(x, y);
      }
  }
  if (!STATES && parts) {
    // joined: the segments before as one; else one after the other (the loads of
    // several in flight together spill)
    const int step = p.seg_chunks * DECAY_CHUNK;
    DecayFactor whole = DecayFactor::make(rate, (float)step);
    for (int s = p.joined ? seg : 0; s < (p.joined ? seg + 1 : seg); ++s) {
      const int n = !p.joined ? rows_in(s)
                    : REV     ? max(0, s0 - max(0, end - len))
                              : min(s0, len);
      const float all = !p.joined && n == step ? whole.next() : expf(rate * (float)n);
      const uint64_t a2 = pack2(all, all);
#pragma unroll
      for (int i = 0; i < R / 2; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j)
          S[i][j] = ffma2(a2, S[i][j], own_part[s * part_step + (i * C + place(j)) * 32]);
    }
  }
  // W columns of the rows [y, y + TT) of the walk, from `from` (row 0) on, to
  // `to`; rows that the head does not have and columns from `cols` on are zero
  auto fetch_part = [&](auto width, T* to, const T* from, int64_t stride, int y, int n, int cols) {
    constexpr int W = decltype(width)::value;
    if (p.vec) {
      constexpr int PR = W / E, RP = 32 / PR;  // pieces of a row, rows at a time
      const int c = lane % PR * E;
      int t = lane / PR;
      const int64_t step = DIR * RP * stride;
      const T* at = from + row_at(y + t) * stride + c;
      uint32_t dst = tc_smem_base(to + t * ROW + c);
#pragma unroll
      for (; t < TT; t += RP, at += step, dst += RP * ROW * (int)sizeof(T)) {
        const bool in = y + t < rows && row_at(y + t) < n && c < cols;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
                     "l"(in ? at : from), "r"(in ? 16 : 0)
                     : "memory");
      }
    } else {
      for (int e = lane; e < TT * W; e += 32) {
        const int t = e / W, c = e % W;
        const bool in = y + t < rows && row_at(y + t) < n && c < cols;
        to[t * ROW + c] = in ? from[row_at(y + t) * stride + c] : from_f32<T>(0.f);
      }
    }
  };
  auto fetch = [&](int slot, int y) {
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      T* to = tiles + slot * TILE + u * HEAD;
      const std::integral_constant<int, DP> wide;
      const std::integral_constant<int, COLS> part_wide;
      fetch_part(wide, to, src_b[u], p.sb.n, y, src_len[u], p.d);
      fetch_part(part_wide, to + AT_C, src_c[u], p.sc.n, y, src_len[u], p.d - part * COLS);
      if constexpr (OUT_C) fetch_part(wide, to + AT_A, src_a[u], p.sa.n, y, src_len[u], p.d);
      if constexpr (OUT_R) fetch_part(part_wide, to + AT_E, src_e[u], p.se.n, y, src_len[u], p.d);
    }
    cp_async_commit();
  };
  const uint64_t ll = pack2(l, l);
  uint64_t ll_mend = ll;
  // Rows: the decay of S before each; backwards it follows the sum, so the first
  // has none. States: the weight of b.
  uint64_t w = REV != STATES ? pack2(1.f, 1.f) : ll;
  const float f = p.in_scale * p.out_scale;
  // what this lane writes: a column of out, a row of row_out
  const int my_col = col_of(0);
  const int my_row = rg * 4 + (cg & 2) + (cg & 1);
  const bool mine = there && my_col < p.d, mine_r = there && my_row < p.d;
  const int es = p.out_f32 ? 4 : (int)sizeof(T);
  const int64_t out_step = (int64_t)(REV ? -1 : 1) * p.H * p.d * es;
  const int64_t first = (((int64_t)b * p.N + row0) * p.H + h) * p.d;
  char* out = static_cast<char*>(p.out) + (first + my_col) * es;
  char* out_r = static_cast<char*>(p.row_out) + (first + my_row) * es;
  auto write = [&](char* at, float x) {
    if (p.out_f32)
      *reinterpret_cast<float*>(at) = x;
    else
      *reinterpret_cast<T*>(at) = from_f32<T>(x);
  };
  const int a_at = rg * 4, c_at = cg * C;
  // the C columns of a lane at `at`
  auto read_cols = [&](float (&x)[C], const T* at) {
    if constexpr (OUT_C) {
#pragma unroll
      for (int j = 0; j < C; ++j) x[j] = to_f32<T>(at[c_at + (j ^ rg)]);
    } else {
#pragma unroll
      for (int j = 0; j < C; j += 4) {
        uint64_t y[2];
        read_pairs<4, 1>(y, at + c_at + j);
        const float2 u = unpack2(y[0]), v = unpack2(y[1]);
        x[j] = u.x;
        x[j + 1] = u.y;
        x[j + 2] = v.x;
        x[j + 3] = v.y;
      }
    }
  };
  if (rows > 0) fetch(0, 0);
  for (int y = 0, slot = 0; y < rows; y += TT, slot ^= 1) {
    if (y + TT < rows) {
      fetch(slot ^ 1, y + TT);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncwarp();
    const T* tile = tiles + slot * TILE + own * HEAD;
    const int n = min(TT, rows - y);
    if (TT == 16 || (y & 15) == 8) {  // the tile has a row 8 of 16
      if (FAR) l16 = DecayFactor{l, far[threadIdx.x].x, far[threadIdx.x].y};
      const float mend = l16.next();
      if (FAR) far[threadIdx.x].y = l16.left;
      ll_mend = pack2(mend, mend);
    }
#pragma unroll 2
    for (int t = 0; t < n; ++t) {
      const T* row = tile + t * ROW;
      uint64_t av[R / 2], bv[R / 2], acc_r[R / 2];
      read_pairs<R, NG>(bv, row + a_at);
      if constexpr (OUT_C) read_pairs<R, NG>(av, row + AT_A + a_at);
      // a row that this lane's head does not have leaves S alone
      const bool live = HEADS == 1 || row_at(y + t) < len;
      const uint64_t lt = ((y + t) & 15) == 8 ? ll_mend : ll;
      if (!STATES && !REV) w = lt;
      const uint64_t wt = STATES || live ? w : pack2(1.f, 1.f);
      if constexpr (STATES) {
#pragma unroll
        for (int i = 0; i < R / 2; ++i) bv[i] = mul2(bv[i], wt);
        if (live) w = mul2(w, lt);
      } else if (REV && live) {
        w = lt;
      }
      float o[C], cv[C], ev[OUT_R ? C : 1];
      read_cols(cv, row + AT_C);
      if constexpr (OUT_R) read_cols(ev, row + AT_E);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const uint64_t cc = pack2(cv[j], cv[j]);
        uint64_t acc = 0, ee = 0;
        if constexpr (OUT_R) ee = pack2(ev[j], ev[j]);
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
          if constexpr (STATES)
            S[i][j] = ffma2(bv[i], cc, S[i][j]);
          else
            S[i][j] = ffma2(wt, S[i][j], mul2(bv[i], cc));
          if constexpr (OUT_C) acc = i == 0 ? mul2(av[i], S[i][j]) : ffma2(av[i], S[i][j], acc);
          if constexpr (OUT_R) acc_r[i] = j == 0 ? mul2(ee, S[i][j]) : ffma2(ee, S[i][j], acc_r[i]);
        }
        if constexpr (OUT_C) o[j] = hsum2(acc);
      }
      if constexpr (OUT_C) {
#pragma unroll
        for (int m = C / 2; m > 0; m >>= 1)
#pragma unroll
          for (int j = 0; j < m; ++j) o[j] += __shfl_xor_sync(0xffffffffu, o[j + m], m);
        if (mine && live) write(out, o[0] * f);
        out += out_step;
      }
      if constexpr (OUT_R) {
        // four rows over the four column groups: a lane keeps one
        const uint64_t keep = cg & 2 ? acc_r[1] : acc_r[0], pass = cg & 2 ? acc_r[0] : acc_r[1];
        const float2 k2 = unpack2(keep), p2 = unpack2(pass);
        const float y0 = k2.x + __shfl_xor_sync(0xffffffffu, p2.x, 2 * NG);
        const float y1 = k2.y + __shfl_xor_sync(0xffffffffu, p2.y, 2 * NG);
        const float z = (cg & 1 ? y1 : y0) + __shfl_xor_sync(0xffffffffu, cg & 1 ? y0 : y1, NG);
        if (mine_r && live) write(out_r, z * f);
        out_r += out_step;
      }
    }
    __syncwarp();  // the tile is free again
  }
  if (!STATES && there) {
    // padding: rows [len, N) of the segment
    const int t0 = max(len, REV ? end - s1 : s0), t1 = min(p.N, REV ? end - s0 : s1);
    for (int t = t0; t < t1; ++t) {
      const int64_t at = (((int64_t)b * p.N + t) * p.H + h) * p.d;
      if (OUT_C && mine) write(static_cast<char*>(p.out) + (at + my_col) * es, 0.f);
      if (OUT_R && mine_r) write(static_cast<char*>(p.row_out) + (at + my_row) * es, 0.f);
    }
  }
  // what the segment adds, or the state after the last
  const bool any = rows_in(seg) > 0;
  const uint64_t g = REV && any && !STATES ? ll : pack2(1.f, 1.f);
  if (STATES && parts) {
#pragma unroll
    for (int i = 0; i < R / 2; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j)
        own_part[seg * part_step + (i * C + place(j)) * 32] = S[i][j];
    return;
  }
  float* dst = nullptr;
  if (STATES)
    dst = p.part + (int64_t)seg * heads * dd + state_at;
  else if (p.last && seg == p.segs - 1)
    dst = p.last + state_at;
  if (!dst || !there) return;
  // no rows: as it was, to the bit
  const bool as_was = !any && src && !(parts && len > 0);
#pragma unroll
  for (int i = 0; i < R / 2; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int r = row_of(i), c = col_of(j);
      const float2 x = unpack2(mul2(mul2(S[i][j], g), pack2(p.in_scale, p.in_scale)));
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (r + u < p.d && c < p.d) {
          const int e = state_index(r + u, c);
          dst[e] = as_was ? src[e] : (u ? x.y : x.x);
        }
    }
}

// part[s] (what segment s adds) becomes the state before segment s:
//   X_0 = start, X_(s+1) = l^(rows of s) X_s + part[s];
// p.last, where given, the state after the last one. Whole segments have one decay,
// whose rounding must not add up (683 segments of 96 rows: 9e-6 of the norm off 64
// bits with one fp32 number, 8e-7 with DecayFactor). V elements a thread.
template <int V>
__global__ void __launch_bounds__(128) decay_join_kernel(DecayParams p, int64_t stride, int rows) {
  const int64_t e = ((int64_t)blockIdx.x * 128 + threadIdx.x) * V;
  if (e >= stride) return;
  struct alignas(4 * V) Vec {
    float x[V];
  };
  const unsigned dd = p.d * p.d;
  const int bh = V == 1 || stride >> 32 ? (int)(e / dd) : (int)((unsigned)e / dd), b = bh / p.H;
  const int len = decay_len(p, b), chunk_rows = p.seg_chunks * rows;
  const int chunks = cdiv(p.N, rows), parts = p.last ? p.segs : p.segs - 1;
  const float rate = decay_rate(p.log_decay, bh % p.H);
  DecayFactor whole = DecayFactor::make(rate, (float)chunk_rows);
  Vec x = {};
  if (p.start) x = *reinterpret_cast<const Vec*>(p.start + e);
  float* at = p.part + e;
  for (int s0 = 0; s0 < p.segs; s0 += 8) {
    Vec add[8] = {};  // eight loads in flight
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (s0 + u < parts) add[u] = *reinterpret_cast<const Vec*>(at + (s0 + u) * stride);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u;
      if (s >= p.segs) break;
      *reinterpret_cast<Vec*>(at + s * stride) = x;
      // rows [t0, t1) of segment s
      const int t0 = p.reverse ? max(0, chunks - (s + 1) * p.seg_chunks) * rows : s * chunk_rows;
      const int t1 = p.reverse ? (chunks - s * p.seg_chunks) * rows : t0 + chunk_rows;
      const int n = max(0, min(len, t1) - t0);
      const float all = n == chunk_rows ? whole.next() : expf(rate * (float)n);
#pragma unroll
      for (int v = 0; v < V; ++v) x.x[v] = fmaf(all, x.x[v], add[u].x[v]);
    }
  }
  if (p.last) *reinterpret_cast<Vec*>(p.last + e) = x;
}

// The same for parts as the lanes hold them (pairs; a warp has 512 of each of
// `per` heads' in turn of 16 lanes), without the state before the first.
__global__ void __launch_bounds__(256)
    decay_join_lanes_kernel(DecayParams p, int64_t pairs, int per) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= pairs) return;
  const int64_t warp_pairs = per == 2 ? 256 : 512;
  const int64_t bh = e / warp_pairs * per + (per == 2 ? (int)(e >> 4) & 1 : 0);
  if (bh >= (int64_t)p.B * p.H) return;
  const int len = decay_len(p, (int)(bh / p.H)), step = p.seg_chunks * DECAY_CHUNK;
  const int end = cdiv(p.N, DECAY_CHUNK) * DECAY_CHUNK;
  const float rate = decay_rate(p.log_decay, (int)(bh % p.H));
  DecayFactor whole = DecayFactor::make(rate, (float)step);
  uint64_t x = 0, *at = reinterpret_cast<uint64_t*>(p.part) + e;
  for (int s0 = 0; s0 < p.segs; s0 += 8) {
    uint64_t add[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) add[u] = s0 + u < p.segs - 1 ? at[(s0 + u) * pairs] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u;
      if (s >= p.segs) break;
      at[s * pairs] = x;
      const int t0 = s * step, t1 = t0 + step;
      const int n = p.reverse ? max(0, min(t1, end) - max(t0, end - len))
                              : max(0, min(t1, len) - t0);
      const float all = n == step ? whole.next() : expf(rate * (float)n);
      x = ffma2(pack2(all, all), x, add[u]);
    }
  }
}

// out[., hk, .] = sum over the G heads of a key head; blockIdx.y: of the two
// tensors. V elements a thread, all G loads in flight; bound by memory.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    decay_share_kernel(const float* x, int64_t x_step, T* out0, T* out1, int64_t n, int G, int d) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (e >= n) return;
  struct alignas(4 * V) In {
    float x[V];
  };
  struct alignas(sizeof(T) * V) Out {
    T x[V];
  };
  const int64_t row = n >> 32 ? e / d : (int64_t)((unsigned)e / (unsigned)d);  // [B, N, Hk]
  const float* src = x + blockIdx.y * x_step + row * G * d + (e - row * d);
  In s = {};
#pragma unroll 4
  for (int g = 0; g < G; ++g) {
    const In y = *reinterpret_cast<const In*>(src + (int64_t)g * d);
#pragma unroll
    for (int v = 0; v < V; ++v) s.x[v] += y.x[v];
  }
  Out o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.x[v] = from_f32<T>(s.x[v]);
  *reinterpret_cast<Out*>((blockIdx.y ? out1 : out0) + e) = o;
}

template <typename T>
cudaError_t share_go(const float* x, int64_t x_step, void* out0, void* out1, int64_t n, int G,
                     int d, cudaStream_t s) {
  const int V = d % 4 == 0 ? 4 : 1;
  const dim3 grid((unsigned)((n / V + 255) / 256), 2);
  T *o0 = static_cast<T*>(out0), *o1 = static_cast<T*>(out1);
  if (V == 4)
    decay_share_kernel<T, 4><<<grid, 256, 0, s>>>(x, x_step, o0, o1, n, G, d);
  else
    decay_share_kernel<T, 1><<<grid, 256, 0, s>>>(x, x_step, o0, o1, n, G, d);
  return cudaGetLastError();
}

template <typename T, int DP, bool REV, int MODE>
cudaError_t scan_go(const DecayParams& p, cudaStream_t s) {
  using Plan = ScPlan<T, DP>;
  const int row = DP + Plan::COLS + (MODE & SC_COLS ? DP : 0) + (MODE & SC_ROWS ? Plan::COLS : 0);
  const int smem = SC_WARPS * 2 * Plan::HEADS *
                   (Plan::TT * row * (int)sizeof(T) + (Plan::HEADS == 2 ? 64 : 0));
  const void* fn = reinterpret_cast<const void*>(&decay_scan_kernel<T, DP, REV, MODE>);
  const cudaError_t e = raise_smem_limit(fn, smem);
  if (e != cudaSuccess) return e;
  const int64_t heads = (int64_t)p.B * p.H;
  const unsigned warps = (unsigned)((heads + Plan::HEADS - 1) / Plan::HEADS * Plan::PARTS);
  // the last segment's share of the state is nobody's start
  const dim3 grid((warps + SC_WARPS - 1) / SC_WARPS, MODE == SC_STATES ? p.segs - 1 : p.segs);
  decay_scan_kernel<T, DP, REV, MODE><<<grid, SC_WARPS * 32, smem, s>>>(p, warps);
  return cudaGetLastError();
}
template <typename T, bool REV>
cudaError_t scan_mode(const DecayParams& p, int mode, cudaStream_t s) {
  if (p.d > 32) {
    if (mode == SC_STATES)
      return p.d <= 64 ? scan_go<T, 64, REV, SC_STATES>(p, s) : scan_go<T, 128, REV, SC_STATES>(p, s);
    return p.d <= 64 ? scan_go<T, 64, REV, SC_COLS>(p, s) : scan_go<T, 128, REV, SC_COLS>(p, s);
  }
  if (mode == SC_STATES)
    return p.d <= 16 ? scan_go<T, 16, REV, SC_STATES>(p, s) : scan_go<T, 32, REV, SC_STATES>(p, s);
  if constexpr (REV) {  // both gradients of a walk backwards
    return p.d <= 16 ? scan_go<T, 16, true, SC_COLS | SC_ROWS>(p, s)
                     : scan_go<T, 32, true, SC_COLS | SC_ROWS>(p, s);
  } else {
    if (mode == SC_ROWS)
      return p.d <= 16 ? scan_go<T, 16, false, SC_ROWS>(p, s) : scan_go<T, 32, false, SC_ROWS>(p, s);
    return p.d <= 16 ? scan_go<T, 16, false, SC_COLS>(p, s) : scan_go<T, 32, false, SC_COLS>(p, s);
  }
}
cudaError_t launch_scan(const DecayParams& p, int mode, bool bf16, cudaStream_t s) {
  if (bf16)
    return p.reverse ? scan_mode<__nv_bfloat16, true>(p, mode, s)
                     : scan_mode<__nv_bfloat16, false>(p, mode, s);
  return p.reverse ? scan_mode<float, true>(p, mode, s) : scan_mode<float, false>(p, mode, s);
}

}  // namespace

DecayPlan decay_plan(int B, int N, int H, int d, bool tc, int jobs) {
  if (B < 1 || N < 1) return DecayPlan{1, 1};
  if (tc) return decay_plan_tc(B, N, H, d, jobs);
  const int64_t heads = (int64_t)B * H;
  const int64_t warps = d <= 16 ? (heads + 1) / 2 : heads * (d <= 32 ? 1 : (d <= 64 ? 2 : 4));
  const int chunks = cdiv(N, DECAY_CHUNK);
  // one wave of what the SMs hold
  const int64_t wave = 148 * 2 * (d <= 16 ? 10 : (d <= 32 ? 8 : (d <= 64 ? 6 : 4)));
  int64_t segs = 2 * warps >= wave ? 1 : wave / warps;
  if (segs > chunks / 2) segs = chunks / 2;
  if (segs < 1) segs = 1;
  DecayPlan g;
  g.seg_chunks = cdiv(chunks, (int)segs);
  g.segs = cdiv(chunks, g.seg_chunks);
  return g;
}

bool decay_tc_sizes(int B, int N, int H, int d, bool bf16) {
  // Measured, the tensor memory against the recurrent form (us, the forward pass
  // with the gradients): d = 64: 2048 heads, 12 rows 103 / 88, 16 rows 104 / 108,
  // 32 rows 104 / 184; 4 heads, 12 to 32 rows 18 / 29 to 49; d = 128, 2048 heads:
  // 16 rows 161 / 342; d = 32: 2048 heads, 16 rows 104 / 43, 4 heads 18 / 27, 32 x
  // 4096 rows of 8 heads 446 / 992; d = 16, 64 x 4096 rows 808 / 823.
  return bf16 && d >= 16 && d % 8 == 0 && N >= (d > 64 ? 12 : (d > 32 ? 16 : 24));
}
bool decay_one_walk(int d, bool tc) { return !tc && d <= 32; }

int64_t decay_part_bytes(const DecayPlan& g, int B, int H, int d, bool tc) {
  const int64_t heads = (int64_t)B * H;
  if (!decay_one_walk(d, tc)) return g.segs * heads * d * d * 4;
  // as the lanes hold it: whole warps of 16 x 16 or 32 x 32
  return g.segs * (d <= 16 ? (heads + 1) / 2 * 2 * 1024 : heads * 4096);
}

cudaError_t launch_decay_states(const DecayParams& p, bool bf16, cudaStream_t s) {
  if (!decay_uses_part(DecayPlan{p.segs, p.seg_chunks}, p.tc, p.last)) return cudaSuccess;
  DecayParams q = p;
  if (!p.tc) q.last = nullptr;
  const cudaError_t e = p.tc ? launch_decay_states_tc(p, s) : launch_scan(p, SC_STATES, bf16, s);
  if (e != cudaSuccess) return e;
  if (!p.joined) return e;
  if (decay_one_walk(p.d, p.tc)) {
    const int64_t heads = (int64_t)p.B * p.H;
    const int64_t pairs = p.d <= 16 ? (heads + 1) / 2 * 256 : heads * 512;
    decay_join_lanes_kernel<<<(unsigned)((pairs + 255) / 256), 256, 0, s>>>(p, pairs,
                                                                            p.d <= 16 ? 2 : 1);
    return cudaGetLastError();
  }
  const int64_t stride = (int64_t)p.B * p.H * p.d * p.d;
  const int chunk = p.tc ? DECAY_TC_CHUNK : DECAY_CHUNK;
  if (p.d % 4 == 0 && (uintptr_t)p.start % 16 == 0 && (uintptr_t)q.last % 16 == 0)
    decay_join_kernel<4><<<(unsigned)((stride / 4 + 127) / 128), 128, 0, s>>>(q, stride, chunk);
  else
    decay_join_kernel<1><<<(unsigned)((stride + 127) / 128), 128, 0, s>>>(q, stride, chunk);
  return cudaGetLastError();
}

cudaError_t launch_decay_rows(const DecayParams& p, bool bf16, cudaStream_t s) {
  if (p.tc) return launch_decay_rows_tc(&p, 1, s);
  return launch_scan(p, p.row_out && !p.out ? SC_ROWS : SC_COLS, bf16, s);
}

cudaError_t launch_decay_share(const float* x, int64_t x_step, void* out0, void* out1,
                               int64_t rows, int Hk, int G, int d, bool bf16, cudaStream_t s) {
  const int64_t n = rows * Hk * d;
  return bf16 ? share_go<__nv_bfloat16>(x, x_step, out0, out1, n, G, d, s)
              : share_go<float>(x, x_step, out0, out1, n, G, d, s);
}

}  // namespace tarmac
