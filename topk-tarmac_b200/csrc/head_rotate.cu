// head_rotate.cu — norms of queries and keys for each head with the position
// rotation in the same pass, forward and backward.
//
// For a row x of d columns, weights w and the row's tables cos, sin [r / 2]:
//   s = (mean_c x_c^2 + eps)^(-1/2),  z = x s w,
//   (y_a, y_b) = (z_a cos - z_b sin, z_a sin + z_b cos) for each of the r / 2
//   column pairs (a, b); columns from r on pass through.
// Pairs are (i, i + r / 2), or (2i, 2i + 1) when interleaved. Backward, with
// dz the inverse rotation of dy and g = w dz:
//   dw = sum over rows of dz x s,   dx = s (g - x s^2 mean_c(g_c x_c)).
//
// Both directions are bound by memory: each element is read once and written
// once (backward: two reads). A row belongs to LPR lanes, and each lane holds
// E column pairs as two vectors of E elements, so the rotation never leaves
// the lane and the only exchange is the row's sum. Columns without a rotation
// take cos = 1, sin = 0, which makes every lane run the same code. A lane
// group keeps its row's tables and weights in registers and runs over up to
// four heads of the same (episode, row), with their loads in flight together.
#include "heads.cuh"

namespace tarmac {

constexpr int ROT_THREADS = 256;
constexpr int ROT_HC = 4;           // heads per unit
constexpr int ROT_BWD_BLOCKS = 148 * 4;

// E consecutive elements as one load or store
template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
  T x[E];
};

template <typename T, int E>
__device__ __forceinline__ void ld_pack(float (&f)[E], const T* p, bool ok) {
  if (ok) {
    const Pack<T, E> v = *reinterpret_cast<const Pack<T, E>*>(p);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = to_f32<T>(v.x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = 0.f;
  }
}
template <typename T, int E>
__device__ __forceinline__ void st_pack(T* p, const float (&f)[E], bool ok) {
  if (!ok) return;
  Pack<T, E> v;
#pragma unroll
  for (int e = 0; e < E; ++e) v.x[e] = from_f32<T>(f[e]);
  *reinterpret_cast<Pack<T, E>*>(p) = v;
}

// The columns of one lane: vectors A and B of E elements starting at ca and
// cb (ok_*: inside the row). Its E pairs are (A[e], B[e]), or, when the pairs
// are adjacent and E >= 2 (ADJ), neighbours inside A and then inside B.
template <int E, bool ADJ>
struct LaneCols {
  int ca, cb;
  bool ok_a, ok_b, adjacent;
  __device__ __forceinline__ LaneCols(int slot, int d, int r, bool interleaved)
      : adjacent(interleaved) {
    const int nrot = r / 2 / E;
    if (ADJ || interleaved) {
      ca = 2 * E * slot;
      cb = ca + E;
    } else if (slot < nrot) {
      ca = E * slot;
      cb = r / 2 + ca;
    } else {
      ca = r + 2 * E * (slot - nrot);
      cb = ca + E;
    }
    ok_a = ca < d;
    ok_b = cb < d;
  }
  // table entry of pair e, or -1 for columns that are not rotated
  __device__ __forceinline__ int entry(int e, int r) const {
    if (ADJ || adjacent) {
      const int c = ADJ ? (e < E / 2 ? ca + 2 * e : cb + 2 * e - E) : ca;
      return c < r ? c / 2 : -1;
    }
    return ca < r / 2 ? ca + e : -1;
  }
};

template <int E, bool ADJ>
__device__ __forceinline__ void turn(float (&a)[E], float (&b)[E], const float (&c)[E],
                                     const float (&s)[E]) {
  if constexpr (ADJ) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float x = a[2 * e], y = a[2 * e + 1];
      a[2 * e] = x * c[e] - y * s[e];
      a[2 * e + 1] = x * s[e] + y * c[e];
      const float u = b[2 * e], v = b[2 * e + 1];
      b[2 * e] = u * c[E / 2 + e] - v * s[E / 2 + e];
      b[2 * e + 1] = u * s[E / 2 + e] + v * c[E / 2 + e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = a[e], y = b[e];
      a[e] = x * c[e] - y * s[e];
      b[e] = x * s[e] + y * c[e];
    }
  }
}

// sum over the LPR lanes of a row (LPR a power of two)
__device__ __forceinline__ float row_sum(float v, int lpr) {
  for (int o = lpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One slot of a lane: its columns, weights and table values.
template <int E, bool ADJ>
struct Slot {
  LaneCols<E, ADJ> col;
  float wa[E], wb[E], c[E], s[E];
  __device__ __forceinline__ Slot(int slot, int d, int r, bool interleaved)
      : col(slot, d, r, interleaved) {}
  __device__ __forceinline__ void weights(const float* w) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      wa[e] = col.ok_a ? (w ? __ldg(w + col.ca + e) : 1.f) : 0.f;
      wb[e] = col.ok_b ? (w ? __ldg(w + col.cb + e) : 1.f) : 0.f;
    }
  }
  __device__ __forceinline__ void tables(const float* cs, const float* sn, int r) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int t = col.entry(e, r);
      c[e] = t >= 0 ? __ldg(cs + t) : 1.f;
      s[e] = t >= 0 ? __ldg(sn + t) : 0.f;
    }
  }
};

// NP slots of E pairs per lane; LPR lanes per row.
template <typename T, int E, bool ADJ, int NP>
__global__ void __launch_bounds__(ROT_THREADS) rotate_kernel(RotateParams p, int lpr) {
  const int per_warp = 32 / lpr;
  const int lane = threadIdx.x & 31;
  const int sub = lane % lpr;
  const int64_t group = (int64_t)(blockIdx.x * (ROT_THREADS / 32) + (threadIdx.x >> 5)) *
                            per_warp + lane / lpr;
  const int cq = cdiv(p.H, ROT_HC), chunks = cq + cdiv(p.Hk, ROT_HC);
  const int64_t tokens = (int64_t)p.B * p.N;
  const int64_t unit = group;
  // lanes of a warp leave together only (the row sums are warp shuffles)
  const bool live = unit < tokens * chunks;
  const int64_t token = live ? unit / chunks : 0;
  const int chunk = live ? (int)(unit - token * chunks) : 0;
  const bool is_q = chunk < cq;
  const int h0 = (is_q ? chunk : chunk - cq) * ROT_HC;
  const int heads = is_q ? p.H : p.Hk;
  const int b = (int)(token / p.N), n = (int)(token - (int64_t)b * p.N);
  const HeadStrides st = is_q ? p.sq : p.sk;
  const T* src = static_cast<const T*>(is_q ? p.q : p.k) + b * st.b + n * st.n + h0 * st.h;
  T* dst = static_cast<T*>(is_q ? p.oq : p.ok) + (token * heads + h0) * p.d;

  float a[ROT_HC][NP][E], bb[ROT_HC][NP][E];
#pragma unroll
  for (int h = 0; h < ROT_HC; ++h)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const LaneCols<E, ADJ> col(sub + i * lpr, p.d, p.r, p.interleaved);
      const bool ok = live && h0 + h < heads;
      ld_pack<T, E>(a[h][i], src + h * st.h + col.ca, ok && col.ok_a);
      ld_pack<T, E>(bb[h][i], src + h * st.h + col.cb, ok && col.ok_b);
    }
  float rs[ROT_HC];
#pragma unroll
  for (int h = 0; h < ROT_HC; ++h) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e)
        ss = fmaf(a[h][i][e], a[h][i][e], fmaf(bb[h][i][e], bb[h][i][e], ss));
    rs[h] = rsqrtf(row_sum(ss, lpr) / (float)p.d + p.eps);
  }
  if (!live) return;
  const int64_t tab = b * p.table_b + (int64_t)n * (p.r / 2);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    Slot<E, ADJ> sl(sub + i * lpr, p.d, p.r, p.interleaved);
    sl.weights(is_q ? p.wq : p.wk);
    sl.tables(p.cos + tab, p.sin + tab, p.r);
#pragma unroll
    for (int h = 0; h < ROT_HC; ++h) {
      if (h0 + h >= heads) break;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        a[h][i][e] *= rs[h] * sl.wa[e];
        bb[h][i][e] *= rs[h] * sl.wb[e];
      }
      turn<E, ADJ>(a[h][i], bb[h][i], sl.c, sl.s);
      st_pack<T, E>(dst + (int64_t)h * p.d + sl.col.ca, a[h][i], sl.col.ok_a);
      st_pack<T, E>(dst + (int64_t)h * p.d + sl.col.cb, bb[h][i], sl.col.ok_b);
    }
  }
}

// Blocks [0, nq) take the query heads, the others the key heads, so that a
// lane's sums for dw belong to one weight; each block leaves one row of d
// sums in `work` and rotate_dw_kernel adds the rows in order: the result does
// not depend on which block ran when.
template <typename T, int E, bool ADJ, int NP>
__global__ void __launch_bounds__(ROT_THREADS) rotate_bwd_kernel(RotateParams p, int lpr,
                                                                 int nq_blocks) {
  constexpr int HC = 2;
  __shared__ float red[ROT_THREADS / 32][128];
  const bool is_q = (int)blockIdx.x < nq_blocks;
  const int blk = is_q ? blockIdx.x : blockIdx.x - nq_blocks;
  const int nblk = is_q ? nq_blocks : gridDim.x - nq_blocks;
  const int per_warp = 32 / lpr;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % lpr;
  const int heads = is_q ? p.H : p.Hk;
  const int chunks = cdiv(heads, HC);
  const int64_t units = (int64_t)p.B * p.N * chunks;
  const HeadStrides st = is_q ? p.sq : p.sk, sg = is_q ? p.sgq : p.sgk;
  const T* X = static_cast<const T*>(is_q ? p.q : p.k);
  const T* Gr = static_cast<const T*>(is_q ? p.gq : p.gk);
  T* D = static_cast<T*>(is_q ? p.oq : p.ok);
  const float inv_d = 1.f / (float)p.d;

  Slot<E, ADJ> sl0(sub, p.d, p.r, p.interleaved);
  Slot<E, ADJ> sl1(sub + (NP > 1 ? lpr : 0), p.d, p.r, p.interleaved);
  sl0.weights(is_q ? p.wq : p.wk);
  if constexpr (NP > 1) sl1.weights(is_q ? p.wq : p.wk);
  float dwa[NP][E], dwb[NP][E];
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) dwa[i][e] = dwb[i][e] = 0.f;

  const int64_t step = (int64_t)nblk * (ROT_THREADS / 32) * per_warp;
  const int64_t first = ((int64_t)blk * (ROT_THREADS / 32) + warp) * per_warp;
  for (int64_t u0 = first; u0 < units; u0 += step) {  // warp-uniform bound
    const int64_t unit = u0 + lane / lpr;
    const bool live = unit < units;
    const int64_t token = live ? unit / chunks : 0;
    const int h0 = live ? (int)(unit - token * chunks) * HC : 0;
    const int b = (int)(token / p.N), n = (int)(token - (int64_t)b * p.N);
    const T* src = X + b * st.b + n * st.n + h0 * st.h;
    const T* gsrc = Gr + b * sg.b + n * sg.n + h0 * sg.h;
    T* dst = D + (token * heads + h0) * p.d;
    float a[HC][NP][E], bb[HC][NP][E], ga[HC][NP][E], gb[HC][NP][E];
#pragma unroll
    for (int h = 0; h < HC; ++h)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const Slot<E, ADJ>& sl = i ? sl1 : sl0;
        const bool ok = live && h0 + h < heads;
        ld_pack<T, E>(a[h][i], src + h * st.h + sl.col.ca, ok && sl.col.ok_a);
        ld_pack<T, E>(bb[h][i], src + h * st.h + sl.col.cb, ok && sl.col.ok_b);
        ld_pack<T, E>(ga[h][i], gsrc + h * sg.h + sl.col.ca, ok && sl.col.ok_a);
        ld_pack<T, E>(gb[h][i], gsrc + h * sg.h + sl.col.cb, ok && sl.col.ok_b);
      }
    const int64_t tab = b * p.table_b + (int64_t)n * (p.r / 2);
    sl0.tables(p.cos + tab, p.sin + tab, p.r);
    if constexpr (NP > 1) sl1.tables(p.cos + tab, p.sin + tab, p.r);
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const Slot<E, ADJ>& sl = i ? sl1 : sl0;
        float ns[E];
#pragma unroll
        for (int e = 0; e < E; ++e) ns[e] = -sl.s[e];
        turn<E, ADJ>(ga[h][i], gb[h][i], sl.c, ns);  // dz
#pragma unroll
        for (int e = 0; e < E; ++e) {
          ss = fmaf(a[h][i][e], a[h][i][e], fmaf(bb[h][i][e], bb[h][i][e], ss));
          dot = fmaf(ga[h][i][e] * sl.wa[e], a[h][i][e],
                     fmaf(gb[h][i][e] * sl.wb[e], bb[h][i][e], dot));
        }
      }
      const float rs = rsqrtf(row_sum(ss, lpr) * inv_d + p.eps);
      const float m = row_sum(dot, lpr) * inv_d * rs * rs;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const Slot<E, ADJ>& sl = i ? sl1 : sl0;
        float xa[E], xb[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          dwa[i][e] = fmaf(ga[h][i][e], a[h][i][e] * rs, dwa[i][e]);
          dwb[i][e] = fmaf(gb[h][i][e], bb[h][i][e] * rs, dwb[i][e]);
          xa[e] = rs * fmaf(-a[h][i][e], m, ga[h][i][e] * sl.wa[e]);
          xb[e] = rs * fmaf(-bb[h][i][e], m, gb[h][i][e] * sl.wb[e]);
        }
        const bool ok = live && h0 + h < heads;
        st_pack<T, E>(dst + (int64_t)h * p.d + sl.col.ca, xa, ok && sl.col.ok_a);
        st_pack<T, E>(dst + (int64_t)h * p.d + sl.col.cb, xb, ok && sl.col.ok_b);
      }
    }
  }
  // the warp's groups, then the block's warps, in a fixed order
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const Slot<E, ADJ>& sl = i ? sl1 : sl0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float x = dwa[i][e], y = dwb[i][e];
      for (int o = lpr; o < 32; o <<= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
      }
      if (lane < lpr) {
        if (sl.col.ok_a) red[warp][sl.col.ca + e] = x;
        if (sl.col.ok_b) red[warp][sl.col.cb + e] = y;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < p.d) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < ROT_THREADS / 32; ++w) t += red[w][threadIdx.x];
    p.work[(int64_t)blockIdx.x * p.d + threadIdx.x] = t;
  }
}

// block 0: dwq from the rows [0, nq) of the per-block sums; block 1: dwk from
// the rows [nq, n). 8 slices of rows per column, joined in order.
__global__ void __launch_bounds__(1024) rotate_dw_kernel(const float* work, int nq, int n,
                                                         int d, float* dwq, float* dwk) {
  __shared__ float red[8][128];
  const int c = threadIdx.x & 127, slice = threadIdx.x >> 7;
  const int lo = blockIdx.x ? nq : 0, hi = blockIdx.x ? n : nq;
  float t = 0.f;
  if (c < d)
    for (int i = lo + slice; i < hi; i += 8) t += work[(int64_t)i * d + c];
  red[slice][c] = t;
  __syncthreads();
  float* out = blockIdx.x ? dwk : dwq;
  if (slice == 0 && c < d && out) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += red[i][c];
    out[c] = t;
  }
}

int64_t rotate_bwd_work(int d) { return (int64_t)ROT_BWD_BLOCKS * d; }

static int pow2_at_least(int x) {
  int r = 1;
  while (r < x) r <<= 1;
  return r;
}

// Widest vector (in elements) that every row start, head start and column
// group of these tensors allows.
static int rotate_width(const RotateParams& p, int es, bool bwd) {
  int e = 16 / es;
  auto fits = [&](int w) {
    const uintptr_t a = (uintptr_t)(w * es - 1);
    auto ok = [&](const void* ptr, const HeadStrides& s) {
      return ((uintptr_t)ptr & a) == 0 && s.b % w == 0 && s.n % w == 0 && s.h % w == 0;
    };
    if (p.d % w || (p.interleaved ? false : (p.r / 2) % w)) return false;
    if (!ok(p.q, p.sq) || !ok(p.k, p.sk)) return false;
    if (bwd && (!ok(p.gq, p.sgq) || !ok(p.gk, p.sgk))) return false;
    const HeadStrides z{0, 0, 0};
    return ok(p.oq, z) && ok(p.ok, z);
  };
  while (e > 1 && !fits(e)) e >>= 1;
  return e;
}

// lanes per row for vectors of e elements (a power of two, at most 32)
static int rotate_lanes(const RotateParams& p, int e) {
  const int rot = p.interleaved ? 0 : p.r / 2 / e;
  const int rest = cdiv(p.interleaved ? p.d : p.d - p.r, 2 * e);
  const int l = pow2_at_least(rot + rest);
  return l > 32 ? 32 : l;
}

template <typename T, int E, bool ADJ>
static cudaError_t rotate_go(const RotateParams& p, bool bwd, cudaStream_t s) {
  constexpr int NP = E == 1 ? 2 : 1;  // scalar columns: up to 64 pairs a row
  const int lpr = E == 1 ? 32 : rotate_lanes(p, E);
  const int groups = ROT_THREADS / lpr;
  const int64_t tokens = (int64_t)p.B * p.N;
  if (!bwd) {
    const int64_t units = tokens * (cdiv(p.H, ROT_HC) + cdiv(p.Hk, ROT_HC));
    const int64_t blocks = (units + groups - 1) / groups;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    rotate_kernel<T, E, ADJ, NP><<<(unsigned)blocks, ROT_THREADS, 0, s>>>(p, lpr);
    return cudaGetLastError();
  }
  // enough blocks for the work, at most ROT_BWD_BLOCKS, shared out by heads
  const int64_t uq = tokens * cdiv(p.H, 2), uk = tokens * cdiv(p.Hk, 2);
  int64_t want = (uq + uk + groups - 1) / groups;
  if (want > ROT_BWD_BLOCKS) want = ROT_BWD_BLOCKS;
  if (want < 2) want = 2;
  int nq = (int)((want * uq + (uq + uk) / 2) / (uq + uk));
  if (nq < 1) nq = 1;
  if (nq > want - 1) nq = (int)want - 1;
  rotate_bwd_kernel<T, E, ADJ, NP><<<(unsigned)want, ROT_THREADS, 0, s>>>(p, lpr, nq);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (p.dwq || p.dwk)
    rotate_dw_kernel<<<2, 1024, 0, s>>>(p.work, nq, (int)want, p.d, p.dwq, p.dwk);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t rotate_any(const RotateParams& p, bool bwd, cudaStream_t s) {
  const int e = rotate_width(p, (int)sizeof(T), bwd);
  const bool adj = p.interleaved != 0;
  if constexpr (sizeof(T) == 2) {
    if (e == 8) return adj ? rotate_go<T, 8, true>(p, bwd, s) : rotate_go<T, 8, false>(p, bwd, s);
  }
  if (e == 4) return adj ? rotate_go<T, 4, true>(p, bwd, s) : rotate_go<T, 4, false>(p, bwd, s);
  if (e == 2) return adj ? rotate_go<T, 2, true>(p, bwd, s) : rotate_go<T, 2, false>(p, bwd, s);
  return rotate_go<T, 1, false>(p, bwd, s);
}

cudaError_t launch_rotate(const RotateParams& p, bool bf16, cudaStream_t s) {
  return bf16 ? rotate_any<__nv_bfloat16>(p, false, s) : rotate_any<float>(p, false, s);
}
cudaError_t launch_rotate_bwd(const RotateParams& p, bool bf16, cudaStream_t s) {
  return bf16 ? rotate_any<__nv_bfloat16>(p, true, s) : rotate_any<float>(p, true, s);
}

}  // namespace tarmac
