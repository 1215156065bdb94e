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
// x: it reads x in place of h.
//
// Bound by memory: three tensors in and two out, five in and three out. A row
// belongs to a group of threads with eight columns each, as vectors of V: part
// of a warp or a warp up to 256 columns, a block beyond. The group walks over
// rows with its weights in registers, so that nothing but the rows moves. The
// weights' gradients are added up in registers over a thread's rows, then over
// the block's groups, and leave one row of sums a block; a second kernel adds
// those in a fixed order.
#include "block_norm.cuh"

namespace tarmac {

namespace {

constexpr int BN_THREADS = 256;  // where a row is at most a warp
constexpr int BN_E = 8;          // columns of a thread

struct NormGrid {
  int lanes;        // threads of a row: 1 .. 32, or whole warps
  int groups;       // rows of a block at a time
  int64_t rows;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T x[V];
};

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
  static __device__ __forceinline__ void widen(float (&f)[BN_E], const Raw& r) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) f[v * V + e] = to_f32<T>(r.v[v].x[e]);
  }
  __device__ __forceinline__ void store(T* p, const float (&f)[BN_E]) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Vec<T, V> r;
#pragma unroll
      for (int e = 0; e < V; ++e) r.x[e] = from_f32<T>(f[v * V + e]);
      if (at(v) < D) *reinterpret_cast<Vec<T, V>*>(p + at(v)) = r;
    }
  }
  // fp32 weights of these columns, ones where there are none, zero beyond D
  __device__ __forceinline__ void weights(float (&f)[BN_E], const float* w) const {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e)
        f[v * V + e] = at(v) < D ? (w ? __ldg(w + at(v) + e) : 1.f) : 0.f;
  }
};

// sums over a row's threads of K values each
template <int K, bool WIDE>
struct RowSum {
  float (*part)[K][32];  // two buffers [2][K][warps]
  int lanes, flip = 0;
  __device__ __forceinline__ void operator()(float (&x)[K]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (WIDE || o < lanes)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] += __shfl_xor_sync(0xffffffffu, x[k], o);
    if constexpr (WIDE) {
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = lanes >> 5;
      // the buffers alternate: a warp that writes the next sum may be ahead of
      // one that still reads this one, never by two
      float (*buf)[32] = part[flip];
      flip ^= 1;
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) buf[k][warp] = x[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float s = lane < warps ? buf[k][lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        x[k] = s;
      }
    }
  }
};

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

template <typename T>
__device__ __forceinline__ const T* row_of(const void* p, const RowStrides& s, uint32_t b,
                                           uint32_t n) {
  return static_cast<const T*>(p) + (int64_t)b * s.b + (int64_t)n * s.n;
}

template <typename T, int V, bool WIDE, bool GATE>
__global__ void __launch_bounds__(WIDE ? 1024 : BN_THREADS)
    norm_kernel(NormParams p, NormGrid g) {
  using C = Cols<T, V>;
  __shared__ float part[2][1][32];
  const int group = WIDE ? 0 : threadIdx.x / g.lanes;
  const C c = {WIDE ? (int)threadIdx.x : (int)(threadIdx.x & (g.lanes - 1)), g.lanes, p.D};
  RowSum<1, WIDE> total = {part, g.lanes};
  float wo[BN_E], wi[BN_E];  // scale w_post, w_pre
  {
    float sc[BN_E];
    c.weights(wo, p.w_post);
    c.weights(sc, p.scale);
    c.weights(wi, p.w_pre);
#pragma unroll
    for (int e = 0; e < BN_E; ++e) wo[e] *= sc[e];
  }
  const float inv = 1.f / (float)p.D;
  const int64_t step = (int64_t)gridDim.x * g.groups;
  // all threads of a block take the same number of turns
  for (int64_t r0 = (int64_t)blockIdx.x * g.groups; r0 < g.rows; r0 += step) {
    const bool live = r0 + group < g.rows;
    const uint32_t row = (uint32_t)(live ? r0 + group : r0);
    const uint32_t b = row / (uint32_t)p.N, n = row - b * (uint32_t)p.N;
    typename C::Raw rx, ry, rg;
    c.load(ry, row_of<T>(p.y, p.sy, b, n));
    c.load(rx, row_of<T>(p.x, p.sx, b, n));
    if constexpr (GATE) c.load(rg, row_of<T>(p.gate, p.sg, b, n));
    float x[BN_E], y[BN_E], s[1] = {0.f};
    C::widen(y, ry);
    C::widen(x, rx);
#pragma unroll
    for (int e = 0; e < BN_E; ++e) s[0] = fmaf(y[e], y[e], s[0]);
    total(s);
    const float rn = rsqrtf(fmaf(s[0], inv, p.eps));
    if constexpr (GATE) {
      float gt[BN_E];
      C::widen(gt, rg);
#pragma unroll
      for (int e = 0; e < BN_E; ++e) y[e] *= sigmoid(gt[e]);
    }
    s[0] = 0.f;
#pragma unroll
    for (int e = 0; e < BN_E; ++e) {
      x[e] = fmaf(y[e] * rn, wo[e], x[e]);
      s[0] = fmaf(x[e], x[e], s[0]);
    }
    total(s);
    const float rh = rsqrtf(fmaf(s[0], inv, p.eps));
    const int64_t at = (int64_t)row * p.D;
    if (live) c.store(static_cast<T*>(p.h) + at, x);
#pragma unroll
    for (int e = 0; e < BN_E; ++e) x[e] = x[e] * rh * wi[e];
    if (live) c.store(static_cast<T*>(p.z) + at, x);
  }
}

template <typename T, int V, bool WIDE, bool GATE>
__global__ void __launch_bounds__(WIDE ? 1024 : BN_THREADS)
    norm_bwd_kernel(NormParams p, NormGrid g) {
  using C = Cols<T, V>;
  __shared__ float part[2][2][32];
  __shared__ float acc[WIDE ? 1 : BN_THREADS / 32][WIDE ? 1 : 32 * BN_E];
  const int group = WIDE ? 0 : threadIdx.x / g.lanes;
  const C c = {WIDE ? (int)threadIdx.x : (int)(threadIdx.x & (g.lanes - 1)), g.lanes, p.D};
  RowSum<2, WIDE> total = {part, g.lanes};
  float wo[BN_E], wi[BN_E], sc[BN_E], d_post[BN_E], d_pre[BN_E], d_sc[BN_E];
  c.weights(wo, p.w_post);
  c.weights(wi, p.w_pre);
  c.weights(sc, p.scale);
#pragma unroll
  for (int e = 0; e < BN_E; ++e) d_post[e] = d_pre[e] = d_sc[e] = 0.f;
  const float inv = 1.f / (float)p.D;
  const int64_t step = (int64_t)gridDim.x * g.groups;
  for (int64_t r0 = (int64_t)blockIdx.x * g.groups; r0 < g.rows; r0 += step) {
    const bool live = r0 + group < g.rows;
    const uint32_t row = (uint32_t)(live ? r0 + group : r0);
    const uint32_t b = row / (uint32_t)p.N, n = row - b * (uint32_t)p.N;
    typename C::Raw rx, ry, rg, rdh, rdz;
    c.load(ry, row_of<T>(p.y, p.sy, b, n));
    c.load(rx, row_of<T>(p.x, p.sx, b, n));
    if constexpr (GATE) c.load(rg, row_of<T>(p.gate, p.sg, b, n));
    float h[BN_E], y[BN_E], gt[BN_E], dz[BN_E], t[2] = {0.f, 0.f};
    if (p.dz) {
      c.load(rdz, row_of<T>(p.dz, p.sdz, b, n));
      C::widen(dz, rdz);
    } else {
#pragma unroll
      for (int e = 0; e < BN_E; ++e) dz[e] = 0.f;
    }
    float ed[BN_E];
    if (p.dh) {
      c.load(rdh, row_of<T>(p.dh, p.sdh, b, n));
      C::widen(ed, rdh);
    } else {
#pragma unroll
      for (int e = 0; e < BN_E; ++e) ed[e] = 0.f;
    }
    C::widen(y, ry);
    C::widen(h, rx);
#pragma unroll
    for (int e = 0; e < BN_E; ++e) t[0] = fmaf(y[e], y[e], t[0]);
    total(t);
    const float rn = rsqrtf(fmaf(t[0], inv, p.eps));
    if constexpr (GATE) {
      C::widen(gt, rg);
#pragma unroll
      for (int e = 0; e < BN_E; ++e) gt[e] = sigmoid(gt[e]);
    } else {
#pragma unroll
      for (int e = 0; e < BN_E; ++e) gt[e] = 1.f;
    }
    t[0] = t[1] = 0.f;
#pragma unroll
    for (int e = 0; e < BN_E; ++e) {
      y[e] *= rn;  // yn
      h[e] = fmaf(gt[e] * y[e], wo[e] * sc[e], h[e]);
      t[0] = fmaf(h[e], h[e], t[0]);
      t[1] = fmaf(dz[e] * wi[e], h[e], t[1]);
    }
    total(t);
    const float rh = rsqrtf(fmaf(t[0], inv, p.eps));
    const float m = t[1] * inv * rh * rh;  // mean(a hn) rh
    const int64_t at = (int64_t)row * p.D;
    t[0] = t[1] = 0.f;
    float dg[BN_E];
#pragma unroll
    for (int e = 0; e < BN_E; ++e) {
      const float hn = h[e] * rh;
      ed[e] = fmaf(rh, dz[e] * wi[e], fmaf(-m, hn, ed[e]));
      const float es = ed[e] * gt[e], ys = es * y[e];
      if (live) {
        d_pre[e] = fmaf(dz[e], hn, d_pre[e]);
        d_sc[e] = fmaf(ys, wo[e], d_sc[e]);
        d_post[e] = fmaf(ys, sc[e], d_post[e]);
      }
      if constexpr (GATE) dg[e] = ys * (1.f - gt[e]) * (sc[e] * wo[e]);
      h[e] = es * (sc[e] * wo[e]);  // w_post b
      t[0] = fmaf(h[e], y[e], t[0]);
    }
    if (live) c.store(static_cast<T*>(p.dx) + at, ed);
    if constexpr (GATE)
      if (live) c.store(static_cast<T*>(p.dgate) + at, dg);
    total(t);
    const float my = t[0] * inv;
#pragma unroll
    for (int e = 0; e < BN_E; ++e) h[e] = rn * fmaf(-my, y[e], h[e]);
    if (live) c.store(static_cast<T*>(p.dy) + at, h);
  }
  // this block's sums for the weights
  float* work = p.work + (int64_t)blockIdx.x * 3 * p.D;
  auto leave = [&](float (&x)[BN_E], float* out) {
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
  leave(d_post, work);
  leave(d_pre, work + p.D);
  leave(d_sc, work + 2 * p.D);
}

// column sums of work [blocks][3 D], in a fixed order
__global__ void __launch_bounds__(1024) norm_sums_kernel(NormParams p, int blocks) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x, n = 3 * p.D;
  float s = 0.f;
  if (col < n)
    for (int i = threadIdx.y; i < blocks; i += 32) s += p.work[(int64_t)i * n + col];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < n) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[i][threadIdx.x];
    float* out = col < p.D ? p.dw_post : (col < 2 * p.D ? p.dw_pre : p.dscale);
    if (out) out[col % p.D] = s;
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
  bool wide;
};
NormLaunch norm_layout(int64_t rows, int D, int per_sm, int cap) {
  NormLaunch l;
  l.g.rows = rows;
  const int need = cdiv(D, BN_E);
  l.wide = need > 32;
  if (l.wide) {
    l.g.lanes = cdiv(need, 32) * 32;
    l.g.groups = 1;
    l.threads = l.g.lanes;
  } else {
    l.g.lanes = 1;
    while (l.g.lanes < need) l.g.lanes *= 2;
    l.g.groups = BN_THREADS / l.g.lanes;
    l.threads = BN_THREADS;
  }
  int64_t most = (int64_t)sm_count() * (per_sm * BN_THREADS / l.threads > 0
                                            ? per_sm * BN_THREADS / l.threads : 1);
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

template <typename T, int V, bool WIDE, bool GATE>
cudaError_t norm_go(const NormParams& p, bool backward, cudaStream_t s) {
  const NormLaunch l =
      norm_layout((int64_t)p.B * p.N, p.D, backward ? 3 : 6, backward ? BN_MAX_BLOCKS : 1 << 30);
  if (!backward) {
    norm_kernel<T, V, WIDE, GATE><<<l.blocks, l.threads, 0, s>>>(p, l.g);
    return cudaGetLastError();
  }
  norm_bwd_kernel<T, V, WIDE, GATE><<<l.blocks, l.threads, 0, s>>>(p, l.g);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  norm_sums_kernel<<<cdiv(3 * p.D, 32), dim3(32, 32), 0, s>>>(p, l.blocks);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t norm_pick(const NormParams& p, bool backward, cudaStream_t s) {
  const bool wide = p.D > 32 * BN_E;
  if (p.gate)
    return wide ? norm_go<T, V, true, true>(p, backward, s)
                : norm_go<T, V, false, true>(p, backward, s);
  return wide ? norm_go<T, V, true, false>(p, backward, s)
              : norm_go<T, V, false, false>(p, backward, s);
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
  return blocks * 3 * D;
}

}  // namespace tarmac
