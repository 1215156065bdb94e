// block_norm.cu — the norm after a block, its gate and residual scale, the sum
// with the stream and the norm before the next block, in one pass; and the
// gradients.
//
// For a row of D columns, s = sigmoid(gate):
//   yn = y / sqrt(mean y^2 + eps),  u = yn w_post,  h = x + scale s u,
//   hn = h / sqrt(mean h^2 + eps),  z = hn w_pre.
// Backward, with rh, ry the two reciprocal roots and a = w_pre dz:
//   e = dh + rh (a - hn mean(a hn)),  dx = e,
//   dgate = e scale u s (1 - s),  dscale = sum e s u,  dw_pre = sum dz hn,
//   b = e scale s,  dw_post = sum b yn,
//   dy = ry (w_post b - yn mean(w_post b yn)).
// z and e follow from the unrounded h, which the backward pass forms again from
// x: it reads x in place of h. With q = sum e s yn, a row of sums, dscale is
// w_post q and dw_post scale q.
//
// Bound by memory: three tensors in and two out, five in and three out. A row
// belongs to a group of threads with eight columns each, as vectors of V: part
// of a warp or a warp up to 256 columns, a block beyond. The group walks over
// rows with its weights in registers, so that nothing but the rows moves, and
// computes on pairs (two fp32 operations an issue slot), as issue is the next
// bound. The sums for the weights are added up in registers over a thread's
// rows, then over the block's groups, and leave two rows a block; a second
// kernel adds those in a fixed order. Measured: 4 x 8192 rows of 2048 bf16 columns
// 114 us (5.9 TB/s, 90 % of the copy rate); 1024 x 512 rows of 256 with a gate 219
// us (6.1 TB/s), gradients 347 + 4 us (6.2 TB/s), 8192 columns' gradients 41 % of
// it: a block of 1024 threads has no registers to fetch ahead.
#include "block_norm.cuh"

namespace tarmac {

namespace {

constexpr int BN_THREADS = 256;  // where a row is at most a warp
constexpr int BN_E = 8;          // columns of a thread
constexpr int BN_P = BN_E / 2;   // as pairs

struct NormGrid {
  int lanes;        // threads of a row: 1 .. 32, or whole warps
  int groups;       // rows of a block at a time
  int64_t rows;
};

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t both(float x) { return pack2(x, x); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T x[V];
};

// the pair of bf16 values in a word
__device__ __forceinline__ uint64_t widen2(uint32_t w) {
  return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Columns of a thread: vectors v at (slot + v lanes) V.
template <typename T, int V>
struct Cols {
  static constexpr int NV = BN_E / V;
  int slot, lanes, D;
  __device__ __forceinline__ int at(int v) const { return (slot + v * lanes) * V; }
  struct Raw {
    Vec<T, V> v[NV];
  };
  __device__ __forceinline__ void load(Raw& r, const T* p) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (at(v) < D) {
        r.v[v] = *reinterpret_cast<const Vec<T, V>*>(p + at(v));
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) r.v[v].x[e] = from_f32<T>(0.f);
      }
    }
  }
  static __device__ __forceinline__ void widen(uint64_t (&f)[BN_P], const Raw& r) {
    if constexpr (sizeof(T) == 2 && V >= 2) {
#pragma unroll
      for (int i = 0; i < BN_P; ++i)
        f[i] = widen2(reinterpret_cast<const uint32_t*>(&r.v[2 * i / V])[2 * i % V / 2]);
    } else {
#pragma unroll
      for (int i = 0; i < BN_P; ++i)
        f[i] = pack2(to_f32<T>(r.v[2 * i / V].x[2 * i % V]),
                     to_f32<T>(r.v[(2 * i + 1) / V].x[(2 * i + 1) % V]));
    }
  }
  __device__ __forceinline__ void store(T* p, const uint64_t (&f)[BN_P]) const {
    float x[BN_E];
    split(x, f);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Vec<T, V> r;
#pragma unroll
      for (int e = 0; e < V; ++e) r.x[e] = from_f32<T>(x[v * V + e]);
      if (at(v) < D) *reinterpret_cast<Vec<T, V>*>(p + at(v)) = r;
    }
  }
  static __device__ __forceinline__ void split(float (&x)[BN_E], const uint64_t (&f)[BN_P]) {
#pragma unroll
    for (int i = 0; i < BN_P; ++i) {
      const float2 y = unpack2(f[i]);
      x[2 * i] = y.x;
      x[2 * i + 1] = y.y;
    }
  }
  // fp32 weights of these columns, ones where there are none, zero beyond D
  __device__ __forceinline__ void weights(uint64_t (&f)[BN_P], const float* w) const {
#pragma unroll
    for (int i = 0; i < BN_P; ++i) {
      float y[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = 2 * i + u, c = at(e / V) + e % V;
        y[u] = at(e / V) < D ? (w ? __ldg(w + c) : 1.f) : 0.f;
      }
      f[i] = pack2(y[0], y[1]);
    }
  }
};

// sum of K values over a row's threads; WIDE: through part [2][K][32]
template <bool WIDE>
struct RowSum {
  float* part;
  int lanes, flip = 0;
  template <int K>
  __device__ __forceinline__ void operator()(float (&x)[K]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (WIDE || o < lanes)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] += __shfl_xor_sync(0xffffffffu, x[k], o);
    if constexpr (WIDE) {
      // The buffers alternate: a warp that writes the next sum may be ahead of
      // one that still reads this one, never by two. Places of warps that the
      // block does not have hold zeros.
      float* buf = part + flip * 64;
      flip ^= 1;
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) buf[32 * k + (threadIdx.x >> 5)] = x[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < lanes >> 5; w += 4) {
          const float4 y = *reinterpret_cast<const float4*>(buf + 32 * k + w);
          s.x += y.x;
          s.y += y.y;
          s.z += y.z;
          s.w += y.w;
        }
        x[k] = (s.x + s.y) + (s.z + s.w);
      }
    }
  }
};

// 1 / (1 + 2^(-x log2 e)), by the special-function unit (an exponent's error
// of |x| 2^-24 and a few 2^-23)
__device__ __forceinline__ void sigmoid(uint64_t (&g)[BN_P]) {
#pragma unroll
  for (int i = 0; i < BN_P; ++i) {
    const float2 x = unpack2(mul2(g[i], both(-1.4426950408889634f)));
    float y[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float e;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(u ? x.y : x.x));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y[u]) : "f"(1.f + e));
    }
    g[i] = pack2(y[0], y[1]);
  }
}

// What a thread of the gradients keeps from row to row, K arrays of its columns:
// in registers, or, where a block of 1024 threads leaves 64 a thread, in its own
// places of shared memory.
template <int K, bool SHARED>
struct Kept {
  uint64_t r[SHARED ? 1 : K][BN_P];
  uint64_t* s;
  __device__ __forceinline__ void init(void* smem) {
    s = SHARED ? static_cast<uint64_t*>(smem) + threadIdx.x : nullptr;
  }
  __device__ __forceinline__ uint64_t get(int k, int i) const {
    return SHARED ? s[(k * BN_P + i) * 1024] : r[SHARED ? 0 : k][i];
  }
  __device__ __forceinline__ void set(int k, int i, uint64_t x) {
    if (SHARED)
      s[(k * BN_P + i) * 1024] = x;
    else
      r[SHARED ? 0 : k][i] = x;
  }
};
constexpr int BN_KEPT_BYTES = 4 * BN_P * 1024 * 8;

template <typename T>
__device__ __forceinline__ const T* row_of(const void* p, const RowStrides& s, uint32_t b,
                                           uint32_t n) {
  return static_cast<const T*>(p) + (int64_t)b * s.b + (int64_t)n * s.n;
}

// THREADS: the most of a block; WIDE where a row is a block
template <typename T, int V, int THREADS, bool WIDE, bool GATE>
__global__ void __launch_bounds__(THREADS, WIDE ? 1024 / THREADS : 5)
    norm_kernel(NormParams p, NormGrid g) {
  using C = Cols<T, V>;
  __shared__ alignas(16) float part[WIDE ? 128 : 1];
  if constexpr (WIDE) {
    for (int i = threadIdx.x; i < 128; i += blockDim.x) part[i] = 0.f;
    __syncthreads();
  }
  const int group = WIDE ? 0 : threadIdx.x / g.lanes;
  const C c = {WIDE ? (int)threadIdx.x : (int)(threadIdx.x & (g.lanes - 1)), g.lanes, p.D};
  RowSum<WIDE> total = {part, g.lanes};
  uint64_t ws[BN_P], wi[BN_P];  // scale w_post, w_pre
  {
    uint64_t sc[BN_P];
    c.weights(ws, p.w_post);
    c.weights(sc, p.scale);
    c.weights(wi, p.w_pre);
#pragma unroll
    for (int i = 0; i < BN_P; ++i) ws[i] = mul2(ws[i], sc[i]);
  }
  const float inv = 1.f / (float)p.D;
  const int64_t step = (int64_t)gridDim.x * g.groups;
  typename C::Raw rx, ry, rg;
  auto fetch = [&](int64_t r0) {  // a turn's rows
    const uint32_t row = (uint32_t)(r0 + group < g.rows ? r0 + group : r0);
    const uint32_t b = row / (uint32_t)p.N, n = row - b * (uint32_t)p.N;
    c.load(ry, row_of<T>(p.y, p.sy, b, n));
    c.load(rx, row_of<T>(p.x, p.sx, b, n));
    if constexpr (GATE) c.load(rg, row_of<T>(p.gate, p.sg, b, n));
  };
  const int64_t first = (int64_t)blockIdx.x * g.groups;
  if (WIDE && first < g.rows) fetch(first);
  // all threads of a block take the same number of turns
  for (int64_t r0 = first; r0 < g.rows; r0 += step) {
    const bool live = r0 + group < g.rows;
    const uint32_t row = (uint32_t)(live ? r0 + group : r0);
    if (!WIDE) fetch(r0);
    uint64_t x[BN_P], y[BN_P], gt[BN_P], acc = 0;
    C::widen(y, ry);
    C::widen(x, rx);
    if constexpr (GATE) C::widen(gt, rg);
    // a block's rows come one after the other: the next is on its way
    if (WIDE && r0 + step < g.rows) fetch(r0 + step);
#pragma unroll
    for (int i = 0; i < BN_P; ++i) acc = ffma2(y[i], y[i], acc);
    float s[1] = {hsum2(acc)};
    total(s);
    const uint64_t rn = both(rsqrtf(fmaf(s[0], inv, p.eps)));
    if constexpr (GATE) {
      sigmoid(gt);
#pragma unroll
      for (int i = 0; i < BN_P; ++i) y[i] = mul2(y[i], gt[i]);
    }
    acc = 0;
#pragma unroll
    for (int i = 0; i < BN_P; ++i) {
      x[i] = ffma2(mul2(y[i], rn), ws[i], x[i]);
      acc = ffma2(x[i], x[i], acc);
    }
    s[0] = hsum2(acc);
    total(s);
    const uint64_t rh = both(rsqrtf(fmaf(s[0], inv, p.eps)));
    const int64_t at = (int64_t)row * p.D;
    if (live) c.store(static_cast<T*>(p.h) + at, x);
#pragma unroll
    for (int i = 0; i < BN_P; ++i) x[i] = mul2(mul2(x[i], rh), wi[i]);
    if (live) c.store(static_cast<T*>(p.z) + at, x);
  }
}

template <typename T, int V, int THREADS, bool WIDE, bool GATE>
__global__ void __launch_bounds__(THREADS, WIDE ? 1 : 2)
    norm_bwd_kernel(NormParams p, NormGrid g) {
  using C = Cols<T, V>;
  // The next row's vectors are on their way while this row is worked on, at
  // the price of a third block per SM (1024 x 512 rows of 256 bf16 columns:
  // 349 us, three blocks without 455); 1024 threads have no room for them.
  constexpr bool AHEAD = THREADS <= 512;
  __shared__ alignas(16) float part[WIDE ? 128 : 1];
  __shared__ float acc[WIDE ? 1 : BN_THREADS / 32][WIDE ? 1 : 32 * BN_E];
  if constexpr (WIDE) {
    for (int i = threadIdx.x; i < 128; i += blockDim.x) part[i] = 0.f;
    __syncthreads();
  }
  const int group = WIDE ? 0 : threadIdx.x / g.lanes;
  const C c = {WIDE ? (int)threadIdx.x : (int)(threadIdx.x & (g.lanes - 1)), g.lanes, p.D};
  RowSum<WIDE> total = {part, g.lanes};
  extern __shared__ __align__(16) unsigned char bn_smem[];
  enum { WS, WI, Q, PRE };  // scale w_post, w_pre, the sums q and for w_pre
  Kept<4, THREADS == 1024> kept;
  kept.init(bn_smem);
  {
    uint64_t ws[BN_P], sc[BN_P], wi[BN_P];
    c.weights(ws, p.w_post);
    c.weights(sc, p.scale);
    c.weights(wi, p.w_pre);
#pragma unroll
    for (int i = 0; i < BN_P; ++i) {
      kept.set(WS, i, mul2(ws[i], sc[i]));
      kept.set(WI, i, wi[i]);
      kept.set(Q, i, 0);
      kept.set(PRE, i, 0);
    }
  }
  const float inv = 1.f / (float)p.D;
  const int64_t step = (int64_t)gridDim.x * g.groups;
  typename C::Raw rx, ry, rg, rdh = {}, rdz = {};
  auto fetch = [&](int64_t r0) {
    const uint32_t row = (uint32_t)(r0 + group < g.rows ? r0 + group : r0);
    const uint32_t b = row / (uint32_t)p.N, n = row - b * (uint32_t)p.N;
    c.load(ry, row_of<T>(p.y, p.sy, b, n));
    c.load(rx, row_of<T>(p.x, p.sx, b, n));
    if constexpr (GATE) c.load(rg, row_of<T>(p.gate, p.sg, b, n));
    if (p.dz) c.load(rdz, row_of<T>(p.dz, p.sdz, b, n));
    if (p.dh) c.load(rdh, row_of<T>(p.dh, p.sdh, b, n));
  };
  const int64_t first = (int64_t)blockIdx.x * g.groups;
  if (AHEAD && first < g.rows) fetch(first);
  for (int64_t r0 = first; r0 < g.rows; r0 += step) {
    const bool live = r0 + group < g.rows;
    const uint32_t row = (uint32_t)(live ? r0 + group : r0);
    if (!AHEAD) fetch(r0);
    uint64_t h[BN_P], y[BN_P], gt[BN_P], dz[BN_P], e[BN_P], t0 = 0, t1 = 0;
    C::widen(y, ry);
    C::widen(h, rx);
    C::widen(dz, rdz);
    C::widen(e, rdh);
    if constexpr (GATE) C::widen(gt, rg);
    if (AHEAD && r0 + step < g.rows) fetch(r0 + step);
#pragma unroll
    for (int i = 0; i < BN_P; ++i) t0 = ffma2(y[i], y[i], t0);
    float s1[1] = {hsum2(t0)};
    total(s1);
    const float rn = rsqrtf(fmaf(s1[0], inv, p.eps));
    if constexpr (GATE) sigmoid(gt);
    t0 = 0;
#pragma unroll
    for (int i = 0; i < BN_P; ++i) {
      y[i] = mul2(y[i], both(rn));  // yn
      h[i] = ffma2(GATE ? mul2(gt[i], y[i]) : y[i], kept.get(WS, i), h[i]);
      t0 = ffma2(h[i], h[i], t0);
      t1 = ffma2(mul2(dz[i], kept.get(WI, i)), h[i], t1);
    }
    float s2[2] = {hsum2(t0), hsum2(t1)};
    total(s2);
    const float rh = rsqrtf(fmaf(s2[0], inv, p.eps));
    const uint64_t m = both(-s2[1] * inv * rh * rh);  // -mean(a hn) / rms(h)
    const uint64_t rh2 = both(rh);
    const int64_t at = (int64_t)row * p.D;
    t0 = 0;
#pragma unroll
    for (int i = 0; i < BN_P; ++i) {
      const uint64_t hn = mul2(h[i], rh2);
      e[i] = ffma2(rh2, mul2(dz[i], kept.get(WI, i)), ffma2(m, hn, e[i]));
      const uint64_t es = GATE ? mul2(e[i], gt[i]) : e[i];
      if (live) {
        kept.set(PRE, i, ffma2(dz[i], hn, kept.get(PRE, i)));
        kept.set(Q, i, ffma2(es, y[i], kept.get(Q, i)));
      }
      h[i] = mul2(es, kept.get(WS, i));  // w_post b
      const uint64_t hy = mul2(h[i], y[i]);
      t0 = ffma2(h[i], y[i], t0);
      if constexpr (GATE) gt[i] = ffma2(mul2(hy, both(-1.f)), gt[i], hy);  // dgate
    }
    if (live) c.store(static_cast<T*>(p.dx) + at, e);
    if constexpr (GATE)
      if (live) c.store(static_cast<T*>(p.dgate) + at, gt);
    s1[0] = hsum2(t0);
    total(s1);
    const uint64_t my = both(-s1[0] * inv);
#pragma unroll
    for (int i = 0; i < BN_P; ++i) h[i] = mul2(both(rn), ffma2(my, y[i], h[i]));
    if (live) c.store(static_cast<T*>(p.dy) + at, h);
  }
  // this block's sums for the weights
  float* work = p.work + (int64_t)blockIdx.x * 2 * p.D;
  auto leave = [&](int which, float* out) {
    uint64_t f[BN_P];
#pragma unroll
    for (int i = 0; i < BN_P; ++i) f[i] = kept.get(which, i);
    float x[BN_E];
    C::split(x, f);
    if constexpr (WIDE) {
#pragma unroll
      for (int v = 0; v < C::NV; ++v)
        if (c.at(v) < p.D)
#pragma unroll
          for (int e = 0; e < V; ++e) out[c.at(v) + e] = x[v * V + e];
    } else {
      // the groups of a warp by shuffles, the warps through shared memory
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o >= g.lanes)
#pragma unroll
          for (int e = 0; e < BN_E; ++e) x[e] += __shfl_xor_sync(0xffffffffu, x[e], o);
      __syncthreads();
      if (lane < g.lanes)
#pragma unroll
        for (int v = 0; v < C::NV; ++v)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[warp][c.at(v) + e] = x[v * V + e];
      __syncthreads();
      for (int i = threadIdx.x; i < p.D; i += BN_THREADS) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < BN_THREADS / 32; ++w) s += acc[w][i];
        out[i] = s;
      }
    }
  };
  leave(Q, work);
  leave(PRE, work + p.D);
}

// column sums of work [blocks][2 D], in a fixed order, to the weights' gradients
__global__ void __launch_bounds__(1024) norm_sums_kernel(NormParams p, int blocks) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x, n = 2 * p.D;
  float s = 0.f;
  if (col < n)
    for (int i = threadIdx.y; i < blocks; i += 32) s += p.work[(int64_t)i * n + col];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < n) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[i][threadIdx.x];
    if (col < p.D) {
      if (p.dw_post) p.dw_post[col] = s * (p.scale ? __ldg(p.scale + col) : 1.f);
      if (p.dscale) p.dscale[col] = s * (p.w_post ? __ldg(p.w_post + col) : 1.f);
    } else if (p.dw_pre) {
      p.dw_pre[col - p.D] = s;
    }
  }
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

constexpr int BN_MAX_BLOCKS = 1024;  // of a backward launch

struct NormLaunch {
  NormGrid g;
  int threads, blocks;
};
// per_sm: resident threads of an SM
NormLaunch norm_layout(int64_t rows, int D, int per_sm, int cap) {
  NormLaunch l;
  l.g.rows = rows;
  const int need = cdiv(D, BN_E);
  if (need > 32) {
    l.g.lanes = cdiv(need, 32) * 32;
    l.g.groups = 1;
    l.threads = l.g.lanes;
  } else {
    l.g.lanes = 1;
    while (l.g.lanes < need) l.g.lanes *= 2;
    l.g.groups = BN_THREADS / l.g.lanes;
    l.threads = BN_THREADS;
  }
  int64_t most = (int64_t)sm_count() * (per_sm > l.threads ? per_sm / l.threads : 1);
  if (most > cap) most = cap;
  const int64_t want = (rows + l.g.groups - 1) / l.g.groups;
  l.blocks = (int)(want < most ? want : most);
  return l;
}

// widest vectors, in elements, that every row allows
template <typename T>
int vector_width(const NormParams& p, bool backward) {
  const void* ptr[8] = {p.x, p.y, p.gate, p.dh, p.dz, backward ? p.dx : p.h,
                        backward ? p.dy : p.z, p.dgate};
  const RowStrides st[5] = {p.sx, p.sy, p.sg, p.sdh, p.sdz};
  uintptr_t bits = (uintptr_t)p.D * sizeof(T);
  for (int i = 0; i < 8; ++i) {
    if (!ptr[i]) continue;
    bits |= (uintptr_t)ptr[i];
    if (i < 5) bits |= (uintptr_t)(st[i].b * (int64_t)sizeof(T)) | (uintptr_t)(st[i].n * (int64_t)sizeof(T));
  }
  int v = 16 / (int)sizeof(T);
  while (v > 1 && bits % (v * sizeof(T))) v /= 2;
  return v;
}

template <typename T, int V, int THREADS, bool WIDE, bool GATE>
cudaError_t norm_go(const NormParams& p, bool backward, cudaStream_t s) {
  // as the launch bounds leave it
  const int per_sm = backward ? (THREADS == 1024 ? 1024 : 512) : (WIDE ? 1024 : 5 * BN_THREADS);
  const NormLaunch l =
      norm_layout((int64_t)p.B * p.N, p.D, per_sm, backward ? BN_MAX_BLOCKS : 1 << 30);
  if (!backward) {
    norm_kernel<T, V, THREADS, WIDE, GATE><<<l.blocks, l.threads, 0, s>>>(p, l.g);
    return cudaGetLastError();
  }
  const int smem = THREADS == 1024 ? BN_KEPT_BYTES : 0;
  cudaError_t e = cudaSuccess;
  if (smem)
    e = raise_smem_limit(reinterpret_cast<const void*>(&norm_bwd_kernel<T, V, THREADS, WIDE, GATE>),
                         smem);
  if (e != cudaSuccess) return e;
  norm_bwd_kernel<T, V, THREADS, WIDE, GATE><<<l.blocks, l.threads, smem, s>>>(p, l.g);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  norm_sums_kernel<<<cdiv(2 * p.D, 32), dim3(32, 32), 0, s>>>(p, l.blocks);
  return cudaGetLastError();
}
template <typename T, int V, bool GATE>
cudaError_t norm_rows(const NormParams& p, bool backward, cudaStream_t s) {
  if (p.D <= 32 * BN_E) return norm_go<T, V, BN_THREADS, false, GATE>(p, backward, s);
  if (p.D <= 512 * BN_E) return norm_go<T, V, 512, true, GATE>(p, backward, s);
  return norm_go<T, V, 1024, true, GATE>(p, backward, s);
}
template <typename T, int V>
cudaError_t norm_pick(const NormParams& p, bool backward, cudaStream_t s) {
  return p.gate ? norm_rows<T, V, true>(p, backward, s) : norm_rows<T, V, false>(p, backward, s);
}
template <typename T>
cudaError_t norm_launch(const NormParams& p, bool backward, cudaStream_t s) {
  const int v = vector_width<T>(p, backward);
  if constexpr (sizeof(T) == 2)
    if (v == 8) return norm_pick<T, 8>(p, backward, s);
  if (v == 4) return norm_pick<T, 4>(p, backward, s);
  if (v == 2) return norm_pick<T, 2>(p, backward, s);
  return norm_pick<T, 1>(p, backward, s);
}

}  // namespace

cudaError_t launch_residual_norm(const NormParams& p, bool bf16, cudaStream_t s) {
  return bf16 ? norm_launch<__nv_bfloat16>(p, false, s) : norm_launch<float>(p, false, s);
}
cudaError_t launch_residual_norm_bwd(const NormParams& p, bool bf16, cudaStream_t s) {
  return bf16 ? norm_launch<__nv_bfloat16>(p, true, s) : norm_launch<float>(p, true, s);
}
int64_t residual_norm_bwd_work(int64_t rows, int D) {
  const int need = cdiv(D, BN_E);
  int lanes = 1;
  while (lanes < need && lanes < 32) lanes *= 2;
  const int64_t groups = need > 32 ? 1 : BN_THREADS / lanes;
  int64_t blocks = (rows + groups - 1) / groups;
  if (blocks > BN_MAX_BLOCKS) blocks = BN_MAX_BLOCKS;
  return blocks * 2 * D;
}

}  // namespace tarmac
