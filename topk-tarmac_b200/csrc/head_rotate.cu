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
// once (backward: two reads). Measured on B200, bf16: 4 x 8192 rows of 20
// heads, d = 128: 61 us, 5.6 TB/s; 1024 x 512 rows of 6 heads, d = 64, a table
// per episode: 162 us, 5.4 TB/s, backward 291 us, 4.4 TB/s: issue is active
// half the time there and loads are waited for, as the staging leaves three
// blocks per SM. A row belongs to LPR lanes, and each lane holds
// E column pairs as two vectors of E elements, so the rotation never leaves
// the lane and the only exchange is the row's sum. Columns without a rotation
// take cos = 1, sin = 0, which makes every lane run the same code. A lane
// group keeps the weights of its columns in registers, walks over rows
// (episode, position) with a fixed stride, loads a row's table once and runs
// over its heads, the loads of two to four heads in flight together.
#include <type_traits>

#include "heads.cuh"

namespace tarmac {

constexpr int ROT_THREADS = 256;
constexpr int ROT_TILES = 4;    // backward: row tiles per block
constexpr int ROT_SLICES = 64;  // first stage of the sums for dw

// E consecutive elements as one load or store
template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
  T x[E];
};

template <typename T, int E>
__device__ __forceinline__ void st_pack(T* p, const float (&f)[E], bool ok) {
  if (!ok) return;
  if constexpr (sizeof(T) == 2 && E % 2 == 0) {
    Pack<__nv_bfloat162, E / 2> v;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v.x[e] = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    *reinterpret_cast<Pack<__nv_bfloat162, E / 2>*>(p) = v;
  } else {
    Pack<T, E> v;
#pragma unroll
    for (int e = 0; e < E; ++e) v.x[e] = from_f32<T>(f[e]);
    *reinterpret_cast<Pack<T, E>*>(p) = v;
  }
}

// The columns of one lane: vectors A and B of E elements starting at ca and
// cb (ok_*: inside the row). Its E pairs are (A[e], B[e]), or, when the pairs
// are adjacent and E >= 2 (ADJ), neighbours inside A and then inside B.
template <int E, bool ADJ>
struct LaneCols {
  int ca, cb;
  bool ok_a, ok_b, adjacent;
  __device__ __forceinline__ void init(int slot, int d, int r, bool interleaved) {
    adjacent = interleaved;
    const int nrot = r / 2 / E;
    if (ADJ || interleaved) {
      ca = 2 * E * slot;
      cb = ca + E;
    } else if (slot < nrot) {
      ca = E * slot;
      cb = r / 2 + ca;
    } else {  // neighbouring lanes take neighbouring columns here too
      const int pairs = cdiv(d - r, 2 * E);
      ca = r + E * (slot - nrot);
      cb = ca + E * pairs;
      if (slot - nrot >= pairs) ca = cb = d;  // no columns
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

// Elementwise arithmetic on E values, two per instruction (fma.rn.f32x2 and
// its kin: the same IEEE results); these kernels are otherwise bound by issue.
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// d = a b + c
template <int E>
__device__ __forceinline__ void vfma(float (&d)[E], const float (&a)[E], const float (&b)[E],
                                     const float (&c)[E]) {
  if constexpr (E % 2 == 0) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 r = unpack2(ffma2(pack2(a[e], a[e + 1]), pack2(b[e], b[e + 1]),
                                     pack2(c[e], c[e + 1])));
      d[e] = r.x;
      d[e + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = fmaf(a[e], b[e], c[e]);
  }
}
template <int E>
__device__ __forceinline__ void vmul(float (&d)[E], const float (&a)[E], const float (&b)[E]) {
  if constexpr (E % 2 == 0) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 r = unpack2(mul2(pack2(a[e], a[e + 1]), pack2(b[e], b[e + 1])));
      d[e] = r.x;
      d[e + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = a[e] * b[e];
  }
}
// d = a f + c, d = a f with one factor for all
template <int E>
__device__ __forceinline__ void vfma1(float (&d)[E], const float (&a)[E], float f,
                                      const float (&c)[E]) {
  float ff[E];
#pragma unroll
  for (int e = 0; e < E; ++e) ff[e] = f;
  vfma<E>(d, a, ff, c);
}
template <int E>
__device__ __forceinline__ void vmul1(float (&d)[E], const float (&a)[E], float f) {
  float ff[E];
#pragma unroll
  for (int e = 0; e < E; ++e) ff[e] = f;
  vmul<E>(d, a, ff);
}
template <int E>
__device__ __forceinline__ float vsum(const float (&a)[E]) {
  float t = a[0];
#pragma unroll
  for (int e = 1; e < E; ++e) t += a[e];
  return t;
}

// Rotate the pairs of (a, b) by (c, s); ns = -s. The inverse takes (ns, s).
template <int E, bool ADJ>
__device__ __forceinline__ void turn(float (&a)[E], float (&b)[E], const float (&c)[E],
                                     const float (&s)[E], const float (&ns)[E]) {
  if constexpr (ADJ) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float x = a[2 * e], y = a[2 * e + 1];
      a[2 * e] = fmaf(x, c[e], y * ns[e]);
      a[2 * e + 1] = fmaf(x, s[e], y * c[e]);
      const float u = b[2 * e], v = b[2 * e + 1];
      b[2 * e] = fmaf(u, c[E / 2 + e], v * ns[E / 2 + e]);
      b[2 * e + 1] = fmaf(u, s[E / 2 + e], v * c[E / 2 + e]);
    }
  } else {
    float t[E], u[E];
    vmul<E>(t, b, ns);
    vmul<E>(u, b, c);
    vfma<E>(b, a, s, u);
    vfma<E>(a, a, c, t);
  }
}

// sum over the lanes of a row (a power of two): LPR of them, or lpr when LPR is 0
template <int LPR>
__device__ __forceinline__ float row_sum(float v, int lpr) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < (LPR ? LPR : lpr)) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// How a launch is laid out; divisions by N are a multiplication with
// ceil(2^(31 + ceil(log2 N)) / N), exact for dividends below 2^31.
struct RotGrid {
  int lpr, lpr_log2;  // lanes per row
  int parts, parts_q; // units per row, and those of query heads
  int four_q, four_k; // units of four heads (else two)
  int table_vec, weight_vec;
  float inv_d;
  uint32_t mul, shift;
  __device__ __forceinline__ uint32_t episode(uint32_t token) const {
    return mul ? __umulhi(token, mul) >> shift : token;
  }
};

// One slot of a lane: its columns and the row's table values.
template <int E, bool ADJ>
struct Slot {
  LaneCols<E, ADJ> col;
  float c[E], s[E];
  __device__ __forceinline__ void weights(const float* w, float (&wa)[E], float (&wb)[E],
                                          bool vec) const {
    if (E >= 4 && vec && w && col.ok_b) {
#pragma unroll
      for (int e = 0; e + 3 < E; e += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(w + col.ca + e));
        const float4 y = __ldg(reinterpret_cast<const float4*>(w + col.cb + e));
        wa[e] = x.x; wa[e + 1] = x.y; wa[e + 2] = x.z; wa[e + 3] = x.w;
        wb[e] = y.x; wb[e + 1] = y.y; wb[e + 2] = y.z; wb[e + 3] = y.w;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      wa[e] = col.ok_a ? (w ? __ldg(w + col.ca + e) : 1.f) : 0.f;
      wb[e] = col.ok_b ? (w ? __ldg(w + col.cb + e) : 1.f) : 0.f;
    }
  }
  // a lane's E entries are neighbours; `vec`: on the 16-byte grid
  __device__ __forceinline__ void tables(const float* cs, const float* sn, int r, bool vec) {
    const int first = ADJ ? col.ca / 2 : col.ca;
    if (E >= 4 && vec && first + E <= r / 2) {
#pragma unroll
      for (int e = 0; e + 3 < E; e += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(cs + first + e));
        const float4 y = __ldg(reinterpret_cast<const float4*>(sn + first + e));
        c[e] = x.x; c[e + 1] = x.y; c[e + 2] = x.z; c[e + 3] = x.w;
        s[e] = y.x; s[e + 1] = y.y; s[e + 2] = y.z; s[e + 3] = y.w;
      }
    } else if ((ADJ || !col.adjacent) && first >= r / 2) {  // not rotated
#pragma unroll
      for (int e = 0; e < E; ++e) {
        c[e] = 1.f;
        s[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int t = col.entry(e, r);
        c[e] = t >= 0 ? __ldg(cs + t) : 1.f;
        s[e] = t >= 0 ? __ldg(sn + t) : 0.f;
      }
    }
  }
};

// global to shared, asynchronously; zeros when not ok
template <typename T, int E>
__device__ __forceinline__ void fetch_pack(Pack<T, E>* dst, const T* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(tc_smem_base(dst)), "l"(src),
               "n"(sizeof(T) * E), "r"(ok ? (int)sizeof(T) * E : 0)
               : "memory");
}

// A vector of E elements as loaded, widened when it is used.
template <typename T, int E>
struct Raw {
  Pack<T, E> v;
  __device__ __forceinline__ void load(const T* p, bool ok) {
    if (ok) {
      v = *reinterpret_cast<const Pack<T, E>*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v.x[e] = from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void widen(float (&f)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = to_f32<T>(v.x[e]);
  }
};

// Where a block's rows and heads are: it takes one unit — HC heads, all query
// or all key heads — of consecutive rows; the units of a row are neighbouring
// blocks, so its table is in L2 after the first. HC is 4 where the head count
// is a multiple of four (more independent work to hide the row sums), else 2.
struct RotUnit {
  uint32_t tblock;
  int chunk;
  bool is_q;
  __device__ __forceinline__ RotUnit(const RotGrid& g) {
    tblock = blockIdx.x / (uint32_t)g.parts;
    chunk = (int)(blockIdx.x - tblock * (uint32_t)g.parts);
    is_q = chunk < g.parts_q;
    if (!is_q) chunk -= g.parts_q;
  }
};

// NP slots of E pairs per lane.
template <typename T, int E, bool ADJ, int NP, int LPR, int HC>
__device__ __forceinline__ void rotate_unit(const RotateParams& p, const RotGrid& g,
                                            const RotUnit& w) {
  constexpr bool FULL = LPR > 0;
  const int lane = threadIdx.x & 31;
  const int sub = lane & (g.lpr - 1);
  const bool is_q = w.is_q;
  const int h0 = w.chunk * HC;
  const int heads = is_q ? p.H : p.Hk;
  // lanes of a warp leave together only (the row sums are warp shuffles)
  uint32_t token = w.tblock * (ROT_THREADS >> g.lpr_log2) + (threadIdx.x >> g.lpr_log2);
  const bool live = token < (uint32_t)p.B * (uint32_t)p.N;
  if (!live) token = 0;
  const uint32_t b = g.episode(token), n = token - b * (uint32_t)p.N;
  const int64_t sh = is_q ? p.sq.h : p.sk.h;
  const T* src = is_q ? static_cast<const T*>(p.q) + b * p.sq.b + n * p.sq.n
                      : static_cast<const T*>(p.k) + b * p.sk.b + n * p.sk.n;
  src += h0 * sh;
  T* dst = static_cast<T*>(is_q ? p.oq : p.ok) + ((int64_t)token * heads + h0) * p.d;
  Slot<E, ADJ> sl[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) sl[i].col.init(sub + i * g.lpr, p.d, p.r, p.interleaved);
  Raw<T, E> a[HC][NP], bb[HC][NP];
#pragma unroll
  for (int h = 0; h < HC; ++h)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const bool ok = FULL || (live && h0 + h < heads);
      a[h][i].load(src + h * sh + sl[i].col.ca, ok && (FULL || sl[i].col.ok_a));
      bb[h][i].load(src + h * sh + sl[i].col.cb, ok && (FULL || sl[i].col.ok_b));
    }
  const int64_t tab = (int64_t)b * p.table_b + (int64_t)n * (p.r / 2);
  float wa[NP][E], wb[NP][E];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    sl[i].tables(p.cos + tab, p.sin + tab, p.r, g.table_vec != 0);
    sl[i].weights(is_q ? p.wq : p.wk, wa[i], wb[i], g.weight_vec != 0);
  }
  float ns[NP][E];
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) ns[i][e] = -sl[i].s[e];
#pragma unroll
  for (int h = 0; h < HC; ++h) {
    float x[NP][E], y[NP][E], acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      a[h][i].widen(x[i]);
      bb[h][i].widen(y[i]);
      vfma<E>(acc, x[i], x[i], acc);
      vfma<E>(acc, y[i], y[i], acc);
    }
    const float rs = rsqrtf(fmaf(row_sum<LPR>(vsum<E>(acc), g.lpr), g.inv_d, p.eps));
    const bool ok = live && (FULL || h0 + h < heads);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      vmul1<E>(x[i], x[i], rs);
      vmul1<E>(y[i], y[i], rs);
      vmul<E>(x[i], x[i], wa[i]);
      vmul<E>(y[i], y[i], wb[i]);
      turn<E, ADJ>(x[i], y[i], sl[i].c, sl[i].s, ns[i]);
      st_pack<T, E>(dst + h * p.d + sl[i].col.ca, x[i], ok && (FULL || sl[i].col.ok_a));
      st_pack<T, E>(dst + h * p.d + sl[i].col.cb, y[i], ok && (FULL || sl[i].col.ok_b));
    }
  }
}

template <typename T, int E, bool ADJ, int NP, int LPR>
__global__ void __launch_bounds__(ROT_THREADS, 4) rotate_kernel(RotateParams p, RotGrid g) {
  const RotUnit w(g);
  if (w.is_q ? g.four_q : g.four_k)
    rotate_unit<T, E, ADJ, NP, LPR, 4>(p, g, w);
  else
    rotate_unit<T, E, ADJ, NP, LPR, 2>(p, g, w);
}

// Laid out as the forward pass, ROT_TILES tiles of rows per block. A lane sums
// its columns' dw over its rows and heads, the block its lanes', and each block
// leaves one row of d sums in `work`; rotate_dw_kernel adds those rows in a
// fixed order, so the result does not depend on which block ran when.
template <typename T, int E, bool ADJ, int NP, int LPR, int HC>
__device__ __forceinline__ void rotate_bwd_unit(const RotateParams& p, const RotGrid& g,
                                                const RotUnit& w, float (&red)[ROT_THREADS / 32][128],
                                                Pack<T, E>* stage) {
  constexpr bool STAGED = E == 4;  // NP is 1
  constexpr bool FULL = LPR > 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane & (g.lpr - 1);
  const uint32_t tblock = w.tblock;
  const bool is_q = w.is_q;
  const int h0 = w.chunk * HC;
  const int heads = is_q ? p.H : p.Hk;
  const uint32_t tokens = (uint32_t)p.B * (uint32_t)p.N;
  const HeadStrides st = is_q ? p.sq : p.sk, sg = is_q ? p.sgq : p.sgk;
  const T* X = static_cast<const T*>(is_q ? p.q : p.k) + h0 * st.h;
  const T* Gr = static_cast<const T*>(is_q ? p.gq : p.gk) + h0 * sg.h;
  T* D = static_cast<T*>(is_q ? p.oq : p.ok) + h0 * p.d;

  Slot<E, ADJ> sl[NP];
  float wa[NP][E], wb[NP][E], dwa[NP][E], dwb[NP][E];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    sl[i].col.init(sub + i * g.lpr, p.d, p.r, p.interleaved);
    sl[i].weights(is_q ? p.wq : p.wk, wa[i], wb[i], g.weight_vec != 0);
#pragma unroll
    for (int e = 0; e < E; ++e) dwa[i][e] = dwb[i][e] = 0.f;
  }
  // STAGED: the vectors of tile it + 1 are on their way to shared memory, each
  // lane's to its own place, while tile it is in work (1024 x 512 rows of 6
  // bf16 heads, d = 64: 321 us, loads to registers 360)
  Raw<T, E> raw[STAGED ? 1 : HC][4][NP];
  auto place = [&](int it, int h, int v) {
    return stage + (((it & 1) * HC + h) * 4 + v) * ROT_THREADS + threadIdx.x;
  };
  uint32_t token;
  bool live;
  float tc[NP][E], ts[NP][E];  // its table values
  auto fetch = [&](int it) {
    token = (tblock * ROT_TILES + it) * (ROT_THREADS >> g.lpr_log2) + (threadIdx.x >> g.lpr_log2);
    live = token < tokens;
    if (!live) token = 0;
    const uint32_t b = g.episode(token), n = token - b * (uint32_t)p.N;
    const T* src = X + b * st.b + n * st.n;
    const T* gsrc = Gr + b * sg.b + n * sg.n;
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      const bool ok = FULL || (live && h0 + h < heads);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const bool ok_a = ok && (FULL || sl[i].col.ok_a), ok_b = ok && (FULL || sl[i].col.ok_b);
        if constexpr (STAGED) {
          fetch_pack(place(it, h, 0), ok_a ? src + h * st.h + sl[i].col.ca : X, ok_a);
          fetch_pack(place(it, h, 1), ok_b ? src + h * st.h + sl[i].col.cb : X, ok_b);
          fetch_pack(place(it, h, 2), ok_a ? gsrc + h * sg.h + sl[i].col.ca : Gr, ok_a);
          fetch_pack(place(it, h, 3), ok_b ? gsrc + h * sg.h + sl[i].col.cb : Gr, ok_b);
        } else {
          raw[h][0][i].load(src + h * st.h + sl[i].col.ca, ok_a);
          raw[h][1][i].load(src + h * st.h + sl[i].col.cb, ok_b);
          raw[h][2][i].load(gsrc + h * sg.h + sl[i].col.ca, ok_a);
          raw[h][3][i].load(gsrc + h * sg.h + sl[i].col.cb, ok_b);
        }
      }
    }
    if constexpr (STAGED) cp_async_commit();
    const int64_t tab = (int64_t)b * p.table_b + (int64_t)n * (p.r / 2);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      sl[i].tables(p.cos + tab, p.sin + tab, p.r, g.table_vec != 0);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        tc[i][e] = sl[i].c[e];
        ts[i][e] = sl[i].s[e];
      }
    }
  };
  if constexpr (STAGED) fetch(0);
  for (int it = 0; it < ROT_TILES; ++it) {
    if constexpr (!STAGED) fetch(it);
    if (__all_sync(0xffffffffu, !live)) break;
    const bool here = live;
    T* dst = D + (int64_t)token * heads * p.d;
    float cs[NP][E], sn[NP][E];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        cs[i][e] = tc[i][e];
        sn[i][e] = ts[i][e];
      }
    if constexpr (STAGED) {
      if (it + 1 < ROT_TILES) {
        fetch(it + 1);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
    }
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      float x[NP][E], y[NP][E], ga[NP][E], gb[NP][E];  // ga, gb: dz
      float acc[E], dot[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = dot[e] = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if constexpr (STAGED)
#pragma unroll
          for (int v = 0; v < 4; ++v) raw[0][v][i].v = *place(it, h, v);
        auto& r = raw[STAGED ? 0 : h];
        r[0][i].widen(x[i]);
        r[1][i].widen(y[i]);
        r[2][i].widen(ga[i]);
        r[3][i].widen(gb[i]);
        float ns[E];
#pragma unroll
        for (int e = 0; e < E; ++e) ns[e] = -sn[i][e];
        turn<E, ADJ>(ga[i], gb[i], cs[i], ns, sn[i]);
        vfma<E>(acc, x[i], x[i], acc);
        vfma<E>(acc, y[i], y[i], acc);
        float t[E];
        vmul<E>(t, ga[i], wa[i]);
        vfma<E>(dot, t, x[i], dot);
        vmul<E>(t, gb[i], wb[i]);
        vfma<E>(dot, t, y[i], dot);
      }
      const bool ok = here && (FULL || h0 + h < heads);
      float rs = rsqrtf(fmaf(row_sum<LPR>(vsum<E>(acc), g.lpr), g.inv_d, p.eps));
      if (!ok) rs = 0.f;  // no row: with eps 0 it would add 0 inf to dw
      const float m = row_sum<LPR>(vsum<E>(dot), g.lpr) * g.inv_d * rs * rs;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        float t[E], u[E];
        vmul1<E>(t, x[i], rs);
        vfma<E>(dwa[i], ga[i], t, dwa[i]);
        vmul1<E>(t, y[i], rs);
        vfma<E>(dwb[i], gb[i], t, dwb[i]);
        vmul<E>(t, ga[i], wa[i]);
        vfma1<E>(u, x[i], -m, t);
        vmul1<E>(u, u, rs);
        st_pack<T, E>(dst + h * p.d + sl[i].col.ca, u, ok && (FULL || sl[i].col.ok_a));
        vmul<E>(t, gb[i], wb[i]);
        vfma1<E>(u, y[i], -m, t);
        vmul1<E>(u, u, rs);
        st_pack<T, E>(dst + h * p.d + sl[i].col.cb, u, ok && (FULL || sl[i].col.ok_b));
      }
    }
  }
  if constexpr (STAGED) cp_async_wait<0>();
  // the warp's groups, then the block's warps, in a fixed order
#pragma unroll
  for (int i = 0; i < NP; ++i) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float x = dwa[i][e], y = dwb[i][e];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1)
        if (o >= g.lpr) {
          x += __shfl_xor_sync(0xffffffffu, x, o);
          y += __shfl_xor_sync(0xffffffffu, y, o);
        }
      if (lane < g.lpr) {
        if (sl[i].col.ok_a) red[warp][sl[i].col.ca + e] = x;
        if (sl[i].col.ok_b) red[warp][sl[i].col.cb + e] = y;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < p.d) {
    float t = 0.f;
#pragma unroll
    for (int x = 0; x < ROT_THREADS / 32; ++x) t += red[x][threadIdx.x];
    p.work[(int64_t)blockIdx.x * p.d + threadIdx.x] = t;
  }
}

template <typename T, int E, bool ADJ, int NP, int LPR>
__global__ void __launch_bounds__(ROT_THREADS, E == 4 ? 3 : 2) rotate_bwd_kernel(RotateParams p, RotGrid g) {
  extern __shared__ __align__(16) unsigned char rot_stage[];
  __shared__ float red[ROT_THREADS / 32][128];
  const RotUnit w(g);
  auto* stage = reinterpret_cast<Pack<T, E>*>(rot_stage);
  if (w.is_q ? g.four_q : g.four_k)
    rotate_bwd_unit<T, E, ADJ, NP, LPR, 4>(p, g, w, red, stage);
  else
    rotate_bwd_unit<T, E, ADJ, NP, LPR, 2>(p, g, w, red, stage);
}

// Sum rows of `src`, [tb, parts] rows of d: block (x, 0) adds the query
// chunks, (x, 1) the key chunks of its share of tb, into row x of dst_q or
// dst_k (rows `dst_stride` apart). Eight lines of rows per column, joined in
// order.
__global__ void __launch_bounds__(1024) rotate_dw_kernel(const float* src, int tb, int parts,
                                                         int cq, int d, float* dst_q,
                                                         float* dst_k, int dst_stride) {
  __shared__ float red[8][128];
  const int c = threadIdx.x & 127, line = threadIdx.x >> 7;
  const int per = cdiv(tb, (int)gridDim.x), lo = (int)blockIdx.x * per, hi = min(tb, lo + per);
  const int c0 = blockIdx.y ? cq : 0, c1 = blockIdx.y ? parts : cq;
  float* dst = blockIdx.y ? dst_k : dst_q;
  if (!dst) return;
  float t = 0.f;
  if (c < d)
    for (int i = lo + line; i < hi; i += 8)
      for (int x = c0; x < c1; ++x) t += src[((int64_t)i * parts + x) * d + c];
  red[line][c] = t;
  __syncthreads();
  if (line == 0 && c < d) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += red[i][c];
    dst[(int64_t)blockIdx.x * dst_stride + c] = t;
  }
}


static int64_t rotate_row_blocks(int64_t tokens, int lpr) {
  const int64_t rows = (int64_t)ROT_TILES * (ROT_THREADS / lpr);
  return (tokens + rows - 1) / rows;
}

int64_t rotate_bwd_work(int64_t tokens, int H, int Hk, int d) {
  // the narrowest rows of blocks: 32 lanes a row
  return (rotate_row_blocks(tokens, 32) * (cdiv(H, 2) + cdiv(Hk, 2)) +
          2 * ROT_SLICES) * d;
}

static int pow2_at_least(int x) {
  int r = 1;
  while (r < x) r <<= 1;
  return r;
}

// Widest vector (in elements, at most 4) that every row start, head start and
// column group of these tensors allows. bf16 vectors of 8 were slower: their
// weights, tables and sums take 176 registers a thread, which leaves too few
// loads in flight (forward, 4 x 8192 rows of 20 heads, d = 128: 157 us, with
// vectors of 4 then 70 and now 61).
static int rotate_width(const RotateParams& p, int es, bool bwd) {
  int e = 4;
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
  auto grid16 = [](const void* x) { return (uintptr_t)x % 16 == 0; };
  RotGrid g = {};
  g.lpr = E == 1 ? 32 : rotate_lanes(p, E);
  while ((1 << g.lpr_log2) < g.lpr) ++g.lpr_log2;
  g.inv_d = 1.f / (float)p.d;
  g.table_vec = p.r / 2 % 4 == 0 && p.table_b % 4 == 0 && grid16(p.cos) && grid16(p.sin);
  g.weight_vec = p.d % 4 == 0 && grid16(p.wq) && grid16(p.wk);
  if (p.N > 1) {
    int l = 0;
    while (((uint64_t)1 << l) < (uint64_t)p.N) ++l;
    g.shift = (uint32_t)l - 1;
    g.mul = (uint32_t)((((uint64_t)1 << (31 + l)) + (uint64_t)p.N - 1) / (uint64_t)p.N);
  }
  const int groups = ROT_THREADS / g.lpr;
  const int64_t tokens = (int64_t)p.B * p.N;
  const bool four = !bwd || sizeof(T) == 2;  // fp32 backward: the stages' size
  g.four_q = four && p.H % 4 == 0;
  g.four_k = four && p.Hk % 4 == 0;
  const int cq = cdiv(p.H, g.four_q ? 4 : 2);
  g.parts_q = cq;
  g.parts = cq + cdiv(p.Hk, g.four_k ? 4 : 2);
  // Rows that fill their lanes, in even numbers of heads, need no tests of
  // columns and heads, and their sums no more steps than they have lanes
  // (1024 x 512 rows of 6 bf16 heads, d = 64: 172 to 163 us, backward 321 to
  // 295).
  auto with_lpr = [&](auto go) {
    if constexpr (E == 4) {
      if (p.d == 2 * E * g.lpr && p.H % 2 == 0 && p.Hk % 2 == 0) {
        if (g.lpr == 2) return go(std::integral_constant<int, 2>());
        if (g.lpr == 4) return go(std::integral_constant<int, 4>());
        if (g.lpr == 8) return go(std::integral_constant<int, 8>());
        if (g.lpr == 16) return go(std::integral_constant<int, 16>());
      }
    }
    return go(std::integral_constant<int, 0>());
  };
  if (!bwd) {
    const int64_t blocks = (tokens + groups - 1) / groups * g.parts;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    with_lpr([&](auto lpr) {
      rotate_kernel<T, E, ADJ, NP, decltype(lpr)::value>
          <<<(unsigned)blocks, ROT_THREADS, 0, s>>>(p, g);
    });
    return cudaGetLastError();
  }
  const int64_t tb = rotate_row_blocks(tokens, g.lpr);
  if (tb * g.parts > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const int smem =
      E == 4 ? 2 * (g.four_q || g.four_k ? 4 : 2) * 4 * ROT_THREADS * E * (int)sizeof(T) : 0;
  cudaError_t e = with_lpr([&](auto lpr) {
    auto* fn = &rotate_bwd_kernel<T, E, ADJ, NP, decltype(lpr)::value>;
    const cudaError_t x = raise_smem_limit(reinterpret_cast<const void*>(fn), smem);
    if (x != cudaSuccess) return x;
    fn<<<(unsigned)(tb * g.parts), ROT_THREADS, smem, s>>>(p, g);
    return cudaGetLastError();
  });
  if (e != cudaSuccess || (!p.dwq && !p.dwk)) return e;
  if (tb <= ROT_SLICES) {
    rotate_dw_kernel<<<dim3(1, 2), 1024, 0, s>>>(p.work, (int)tb, g.parts, cq, p.d, p.dwq, p.dwk,
                                                 0);
  } else {
    float* part = p.work + tb * g.parts * p.d;  // [ROT_SLICES][2][d]
    rotate_dw_kernel<<<dim3(ROT_SLICES, 2), 1024, 0, s>>>(p.work, (int)tb, g.parts, cq, p.d, part,
                                                          part + p.d, 2 * p.d);
    rotate_dw_kernel<<<dim3(1, 2), 1024, 0, s>>>(part, ROT_SLICES, 2, 1, p.d, p.dwq, p.dwk, 0);
  }
  return cudaGetLastError();
}

template <typename T>
static cudaError_t rotate_any(const RotateParams& p, bool bwd, cudaStream_t s) {
  const int e = rotate_width(p, (int)sizeof(T), bwd);
  const bool adj = p.interleaved != 0;
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
