// decay_attn.cu — attention with a decay for each head over a set of rows:
// the chunk form, by warp-level products, and the states of its segments.
//
// The row axis runs in chunks of 64. Inside a chunk, by rows i and j,
//   out_i = sum_{j <= i} l^(i-j) (a_i . b_j) c_j + l^(i+1) (a_i . S)
// and across chunks the state follows
//   S' = l^n S + sum_j l^(n-1-j) b_j c_j^T,  n the chunk's rows.
// One block takes one head of one episode, or a segment of its rows, and walks
// over the chunks with S^T in shared memory. Where episodes and heads are too
// few to fill the GPU the row axis is cut in segments: a first launch forms
// what each segment adds to the state, a second joins them to the states
// before each segment, and the rows follow.
//
// Products: bf16 rows run as bf16 with fp32 sums; the weights l^(i-j) a_i . b_j
// and the copy of S that multiplies a_i are rounded to bf16 (errors of the size
// of the output's own rounding), while the weighted rows that enter S are split
// in bf16 parts: two where S only feeds such a copy (2^-17 of each term), three,
// which is an fp32's 24 bits, where the caller gets it. fp32 rows use three tf32
// products for one. S itself is fp32.
#include "decay.cuh"
#include "head_mma.cuh"

namespace tarmac {

namespace {

constexpr int DA_THREADS = 128;
constexpr int DA_ROWS = DECAY_CHUNK;

template <typename T, int DP>
struct DaPlan {
  static constexpr int RS = hm::row_stride<T, DP>();
  static constexpr int SS = hm::row_stride<float, DP>();    // fp32 state rows
  static constexpr bool COPY = sizeof(T) == 2;              // bf16 copy of S
  static constexpr int TILE = DA_ROWS * RS * (int)sizeof(T);
  static constexpr int STATE = DP * SS * 4;
  static constexpr int STATE16 = COPY ? DP * RS * 2 : 0;
  static constexpr int NB = DP >= 32 ? 4 : 2;  // 8-column tiles of a block of columns
  static constexpr int UB = DP >= 64 ? 4 : 2;  // the same in the state's update
  static constexpr int bytes(bool rows) {
    return (rows ? 3 : 2) * TILE + STATE + (rows ? STATE16 : 0);
  }
};

// o[NB tiles of 8 columns] += P . B, B's rows RS elements apart; as
// hm::aggregate, for a block of the columns.
template <int RS, int NB, int NT>
__device__ __forceinline__ void add_product(float (&o)[NB][4], const float (&p)[NT][4],
                                            const __nv_bfloat16* sB, int lane) {
  const __nv_bfloat16* pb = sB + ((lane & 7) + ((lane >> 3) & 1) * 8) * RS + (lane >> 4) * 8;
#pragma unroll
  for (int kk = 0; kk < NT / 2; ++kk) {
    const uint32_t a[4] = {hm::pack_b16(p[2 * kk][0], p[2 * kk][1]),
                           hm::pack_b16(p[2 * kk][2], p[2 * kk][3]),
                           hm::pack_b16(p[2 * kk + 1][0], p[2 * kk + 1][1]),
                           hm::pack_b16(p[2 * kk + 1][2], p[2 * kk + 1][3])};
#pragma unroll
    for (int n = 0; n < NB; n += 2) {
      uint32_t b[4];
      hm::ldsm4t(b, pb + kk * 16 * RS + n * 8);
      hm::mma_b16(o[n], a, b[0], b[1]);
      hm::mma_b16(o[n + 1], a, b[2], b[3]);
    }
  }
}
template <int RS, int NB, int NT>
__device__ __forceinline__ void add_product(float (&o)[NB][4], const float (&p)[NT][4],
                                            const float* sB, int lane) {
  // position t and t + 4 of each 8 stand for rows 2t, 2t + 1 of B
  const float* pb = sB + 2 * (lane & 3) * RS + (lane >> 2);
  float small[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) small[n][u] = 0.f;
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    uint32_t ah[4], al[4];
    hm::split_tf32(p[k][0], ah[0], al[0]);
    hm::split_tf32(p[k][2], ah[1], al[1]);
    hm::split_tf32(p[k][1], ah[2], al[2]);
    hm::split_tf32(p[k][3], ah[3], al[3]);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      uint32_t bh[2], bl[2];
      hm::split_tf32(pb[k * 8 * RS + n * 8], bh[0], bl[0]);
      hm::split_tf32(pb[(k * 8 + 1) * RS + n * 8], bh[1], bl[1]);
      hm::mma_tf32(small[n], al, bh[0], bh[1]);
      hm::mma_tf32(o[n], ah, bh[0], bh[1]);
      hm::mma_tf32(small[n], ah, bl[0], bl[1]);
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) o[n][u] += small[n][u];
}

// rows [0, n) of a tile, zero from n on and beyond d; asynchronous where rows
// are vectors
template <typename T, int DP>
__device__ __forceinline__ void stage(T* tile, const T* src, int64_t rs, int n, int d, bool vec) {
  constexpr int RS = DaPlan<T, DP>::RS, E = 16 / (int)sizeof(T), CV = DP / E;
  if (vec) {
    for (int e = threadIdx.x; e < DA_ROWS * CV; e += DA_THREADS) {
      const int r = e / CV, c = (e % CV) * E;
      const bool ok = r < n && c < d;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       tc_smem_base(tile + r * RS + c)),
                   "l"(ok ? src + (int64_t)r * rs + c : src), "r"(ok ? 16 : 0)
                   : "memory");
    }
  } else {
    for (int e = threadIdx.x; e < DA_ROWS * DP; e += DA_THREADS) {
      const int r = e / DP, c = e % DP;
      tile[r * RS + c] = r < n && c < d ? src[(int64_t)r * rs + c] : from_f32<T>(0.f);
    }
  }
}

template <typename T, int DP, bool ROWS>
__global__ void __launch_bounds__(DA_THREADS) decay_kernel(DecayParams p) {
  using Plan = DaPlan<T, DP>;
  constexpr int RS = Plan::RS, SS = Plan::SS, NB = Plan::NB, UB = Plan::UB;
  constexpr int NT = DA_ROWS / 8;
  extern __shared__ __align__(16) unsigned char da_smem[];
  __shared__ float pw[DA_ROWS + 1];
  T* tb = reinterpret_cast<T*>(da_smem);
  T* tcol = tb + DA_ROWS * RS;
  float* S = reinterpret_cast<float*>(da_smem + 2 * Plan::TILE);  // [c columns][b columns]
  T* ta = reinterpret_cast<T*>(da_smem + 2 * Plan::TILE + Plan::STATE);
  T* S16 = ta + DA_ROWS * RS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = (int)(blockIdx.x % (unsigned)p.H);
  const int bs = (int)(blockIdx.x / (unsigned)p.H);
  const int b = bs % p.B, seg = bs / p.B;
  const int len = decay_len(p, b);
  const float rate = decay_rate(p.log_decay, h);
  for (int e = threadIdx.x; e <= DA_ROWS; e += DA_THREADS) pw[e] = expf(rate * (float)e);
  const T* A = static_cast<const T*>(p.a) + b * p.sa.b + (h / p.ga) * p.sa.h;
  const T* Bt = static_cast<const T*>(p.b) + b * p.sb.b + (h / p.gb) * p.sb.h;
  const T* Ct = static_cast<const T*>(p.c) + b * p.sc.b + (h / p.gc) * p.sc.h;
  const int dd = p.d * p.d;
  const int64_t head = ((int64_t)b * p.H + h) * dd;
  // the state before the segment
  {
    const float* src = nullptr;
    if (ROWS) {
      if (p.segs > 1)
        src = p.part + (int64_t)seg * p.B * p.H * dd + head;
      else if (p.start)
        src = p.start + head;
    }
    for (int e = threadIdx.x; e < DP * SS; e += DA_THREADS) S[e] = 0.f;
    __syncthreads();
    if (src)
      for (int e = threadIdx.x; e < dd; e += DA_THREADS) {
        const int x = e / p.d, y = e % p.d;
        S[p.transposed ? x * SS + y : y * SS + x] = src[e];
      }
  }
  const int chunks = cdiv(p.N, DA_ROWS);
  const int k0 = seg * p.seg_chunks, k1 = min(k0 + p.seg_chunks, chunks);
  for (int k = k0; k < k1; ++k) {
    const int chunk = p.reverse ? chunks - 1 - k : k;
    const int t0 = chunk * DA_ROWS;
    const int n = max(0, min(len - t0, DA_ROWS));
    if (n > 0) {
      stage<T, DP>(tb, Bt + (int64_t)t0 * p.sb.n, p.sb.n, n, p.d, p.vec);
      stage<T, DP>(tcol, Ct + (int64_t)t0 * p.sc.n, p.sc.n, n, p.d, p.vec);
      if (ROWS) stage<T, DP>(ta, A + (int64_t)t0 * p.sa.n, p.sa.n, n, p.d, p.vec);
    }
    __syncthreads();  // S is whole
    if constexpr (ROWS && Plan::COPY) {
      for (int e = threadIdx.x; e < DP * DP; e += DA_THREADS)
        S16[(e / DP) * RS + e % DP] = from_f32<T>(S[(e / DP) * SS + e % DP]);
    }
    cp_async_wait_all();
    __syncthreads();
    if constexpr (ROWS) {
      const int r0 = warp * 16 + (lane >> 2);  // this lane's rows: r0, r0 + 8
      float w[NT][4];
      if (n > 0) {
        hm::scores<DP, NT>(w, ta + warp * 16 * RS, tb, lane);
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = r0 + 8 * (u >> 1), j = 8 * x + 2 * (lane & 3) + (u & 1);
            const int e = p.reverse ? j - i : i - j;
            w[x][u] = e >= 0 ? w[x][u] * (pw[max(e, 0)] * p.in_scale) : 0.f;
          }
      }
      // the state's weight: l^(i+1), backwards l^(n-1-i)
      float first[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = r0 + 8 * u;
        first[u] = pw[max(0, p.reverse ? n - 1 - i : i + 1)];
      }
#pragma unroll 1
      for (int c0 = 0; c0 < DP; c0 += NB * 8) {
        float o[NB][4];
        if (n > 0) {
          if constexpr (Plan::COPY)
            hm::scores<DP, NB>(o, ta + warp * 16 * RS, S16 + c0 * RS, lane);
          else
            hm::scores<DP, NB>(o, ta + warp * 16 * RS, S + c0 * SS, lane);
#pragma unroll
          for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int u = 0; u < 4; ++u) o[x][u] *= first[u >> 1];
          add_product<RS, NB, NT>(o, w, tcol + c0, lane);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = r0 + 8 * u;
          if (t0 + i >= p.N) continue;
          const int64_t at = (((int64_t)b * p.N + t0 + i) * p.H + h) * p.d;
#pragma unroll
          for (int x = 0; x < NB; ++x) {
            const int c = c0 + 8 * x + 2 * (lane & 3);
            const float y0 = i < n ? o[x][2 * u] * p.out_scale : 0.f;
            const float y1 = i < n ? o[x][2 * u + 1] * p.out_scale : 0.f;
            if (p.out_f32) {
              float* dst = static_cast<float*>(p.out) + at + c;
              if (c < p.d) dst[0] = y0;
              if (c + 1 < p.d) dst[1] = y1;
            } else {
              T* dst = static_cast<T*>(p.out) + at + c;
              if (c < p.d) dst[0] = from_f32<T>(y0);
              if (c + 1 < p.d) dst[1] = from_f32<T>(y1);
            }
          }
        }
      }
      __syncthreads();  // S has been read
    }
    if (n > 0 && (k + 1 < k1 || !ROWS || p.last)) {
      // S' = l^n S + sum_j (weight c_j) b_j^T: the weighted columns are the
      // A operand, its rows the columns of c
      const float all = pw[n];
      constexpr int MT = DP / 16, NU = DP / 8 / UB;
      for (int unit = warp; unit < MT * NU; unit += DA_THREADS / 32) {
        const int m0 = (unit / NU) * 16, c0 = (unit % NU) * UB * 8;
        float o[UB][4];
#pragma unroll
        for (int x = 0; x < UB; ++x)
#pragma unroll
          for (int u = 0; u < 4; ++u) o[x][u] = 0.f;
        float w[NT][4];
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int j = 8 * x + 2 * (lane & 3) + (u & 1);
            const int e = p.reverse ? j + 1 : n - 1 - j;  // j >= n: the row is zero
            w[x][u] = to_f32<T>(tcol[j * RS + m0 + (lane >> 2) + 8 * (u >> 1)]) *
                      (pw[max(0, e)] * p.in_scale);
          }
        add_product<RS, UB, NT>(o, w, tb + c0, lane);
        if constexpr (Plan::COPY) {
          for (int part = 1; part < p.planes; ++part) {
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
              for (int u = 0; u < 4; ++u) w[x][u] -= to_f32<T>(from_f32<T>(w[x][u]));
            add_product<RS, UB, NT>(o, w, tb + c0, lane);
          }
        }
#pragma unroll
        for (int x = 0; x < UB; ++x)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            float* s = S + (m0 + (lane >> 2) + 8 * (u >> 1)) * SS + c0 + 8 * x + 2 * (lane & 3) +
                       (u & 1);
            *s = fmaf(all, *s, o[x][u]);
          }
      }
      __syncthreads();  // the tiles are free again
    }
  }
  float* dst = nullptr;
  if (!ROWS)
    dst = p.part + (int64_t)seg * p.B * p.H * dd + head;
  else if (p.last && seg == p.segs - 1)
    dst = p.last + head;
  if (dst) {
    __syncthreads();
    for (int e = threadIdx.x; e < dd; e += DA_THREADS) {
      const int x = e / p.d, y = e % p.d;
      dst[e] = S[p.transposed ? x * SS + y : y * SS + x];
    }
  }
}

// part[s] (what segment s adds) becomes the state before segment s:
//   X_0 = start, X_(s+1) = l^(rows of s) X_s + part[s];
// p.last, where given, the state after the last one.
__global__ void __launch_bounds__(256) decay_join_kernel(DecayParams p, int64_t stride, int rows) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= stride) return;
  const int dd = p.d * p.d;
  const int bh = (int)(e / dd), b = bh / p.H;
  const int len = decay_len(p, b), chunk_rows = p.seg_chunks * rows;
  const int chunks = cdiv(p.N, rows), parts = p.last ? p.segs : p.segs - 1;
  const float rate = decay_rate(p.log_decay, bh % p.H);
  float x = p.start ? p.start[e] : 0.f;
  float* at = p.part + e;
  for (int s0 = 0; s0 < p.segs; s0 += 8) {
    float add[8];  // eight loads in flight
#pragma unroll
    for (int u = 0; u < 8; ++u) add[u] = s0 + u < parts ? at[(s0 + u) * stride] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u;
      if (s >= p.segs) break;
      at[s * stride] = x;
      // rows [t0, t1) of segment s
      const int t0 = p.reverse ? max(0, chunks - (s + 1) * p.seg_chunks) * rows : s * chunk_rows;
      const int t1 = p.reverse ? (chunks - s * p.seg_chunks) * rows : t0 + chunk_rows;
      const int n = max(0, min(len, t1) - t0);
      x = fmaf(expf(rate * (float)n), x, add[u]);
    }
  }
  if (p.last) p.last[e] = x;
}

template <typename T>
__global__ void __launch_bounds__(256)
    decay_share_kernel(const float* x, T* out, int64_t n, int G, int d) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  const int64_t row = e / d;  // [B, N, Hk]
  const float* src = x + row * G * d + e % d;
  float s = 0.f;
  for (int g = 0; g < G; ++g) s += src[(int64_t)g * d];
  out[e] = from_f32<T>(s);
}

template <typename T, int DP, bool ROWS>
cudaError_t decay_go(const DecayParams& p, cudaStream_t s) {
  constexpr int SMEM = DaPlan<T, DP>::bytes(ROWS);
  const void* fn = reinterpret_cast<const void*>(&decay_kernel<T, DP, ROWS>);
  const cudaError_t e = raise_smem_limit(fn, SMEM);
  if (e != cudaSuccess) return e;
  // the last segment's share of the state is nobody's start
  const int64_t blocks = (int64_t)p.B * p.H * (ROWS ? p.segs : p.segs - 1);
  decay_kernel<T, DP, ROWS><<<(unsigned)blocks, DA_THREADS, SMEM, s>>>(p);
  return cudaGetLastError();
}
template <typename T, bool ROWS>
cudaError_t decay_width(const DecayParams& p, cudaStream_t s) {
  if (p.d <= 16) return decay_go<T, 16, ROWS>(p, s);
  if (p.d <= 32) return decay_go<T, 32, ROWS>(p, s);
  if (p.d <= 64) return decay_go<T, 64, ROWS>(p, s);
  return decay_go<T, 128, ROWS>(p, s);
}

}  // namespace

DecayPlan decay_plan(int B, int N, int H, int d, bool tc) {
  if (B < 1 || N < 1) return DecayPlan{1, 1};
  if (tc) return decay_plan_tc(B, N, H, d);
  const int chunks = cdiv(N, DECAY_CHUNK);
  const int64_t heads = (int64_t)B * H;
  int64_t segs = heads >= 296 ? 1 : (592 + heads - 1) / heads;
  if (segs > chunks / 2) segs = chunks / 2;
  if (segs < 1) segs = 1;
  DecayPlan g;
  g.seg_chunks = cdiv(chunks, (int)segs);
  g.segs = cdiv(chunks, g.seg_chunks);
  return g;
}

bool decay_tc_sizes(int B, int N, int H, int d, bool bf16) {
  return bf16 && d > 32 && d % 8 == 0 && N > 64;
}

cudaError_t launch_decay_states(const DecayParams& p, bool bf16, cudaStream_t s) {
  if (!decay_uses_part(DecayPlan{p.segs, p.seg_chunks}, p.tc, p.last)) return cudaSuccess;
  DecayParams q = p;
  if (!p.tc) q.last = nullptr;
  const cudaError_t e = p.tc ? launch_decay_states_tc(p, s)
                        : bf16 ? decay_width<__nv_bfloat16, false>(p, s)
                               : decay_width<float, false>(p, s);
  if (e != cudaSuccess) return e;
  const int64_t stride = (int64_t)p.B * p.H * p.d * p.d;
  decay_join_kernel<<<(unsigned)((stride + 255) / 256), 256, 0, s>>>(
      q, stride, p.tc ? DECAY_TC_CHUNK : DECAY_CHUNK);
  return cudaGetLastError();
}

cudaError_t launch_decay_rows(const DecayParams& p, bool bf16, cudaStream_t s) {
  if (p.tc) return launch_decay_rows_tc(p, s);
  return bf16 ? decay_width<__nv_bfloat16, true>(p, s) : decay_width<float, true>(p, s);
}

cudaError_t launch_decay_share(const float* x, void* out, int64_t rows, int Hk, int G, int d,
                               bool bf16, cudaStream_t s) {
  const int64_t n = rows * Hk * d;
  const unsigned blocks = (unsigned)((n + 255) / 256);
  if (bf16)
    decay_share_kernel<<<blocks, 256, 0, s>>>(x, static_cast<__nv_bfloat16*>(out), n, G, d);
  else
    decay_share_kernel<<<blocks, 256, 0, s>>>(x, static_cast<float*>(out), n, G, d);
  return cudaGetLastError();
}

}  // namespace tarmac
