// decay_step.cu — attention with a decay for each head over few rows: the
// recurrent form, one row after the other.
//
//   S = l S + k v^T,  out = scale S^T q
// for each row, with S in registers between them. Bound by memory: a call on
// one row reads and writes the state, 8 d^2 bytes a head, and little else.
// A thread holds four neighbouring columns of RPT of S's rows; the lanes of a
// row are neighbours, so a warp moves whole 16-byte vectors of consecutive
// rows. Only the sum over S's rows crosses threads: by shuffles in the warp,
// then through shared memory. A state that is renewed row by row, call after call,
// must not gather the rounding of l: 600 rows of slow decays were 8e-6 of the norm
// off 64 bits with l in one fp32 number, 6e-7 with l as 1 + m (DecayPower). The
// state may be renewed in place: a block reads its head's state before it writes
// it. 512 x 16 heads of 128 columns: 201 us with L2 flushed, 5.4 TB/s (82 % of the
// copy rate), 173-180 us a call when calls follow one another; 1024 x 8 heads of 64:
// 49 us; 256 x 4 heads of 16: 3.4 us, latency.
#include "decay.cuh"

namespace tarmac {

namespace {

constexpr int DS_ROWS = 8;  // the most that a call has here

// DP columns, CB of them a block: LPR lanes a row, RG rows a warp at once, WARPS
// warps a head. A block of all 128 columns holds 64 KB at once and was slower
// (512 x 16 heads: 231 us).
template <int DP>
struct DsPlan {
  static constexpr int CB = DP == 128 ? 64 : DP;
  static constexpr int LPR = CB / 4, RG = 32 / LPR;
  static constexpr int WARPS = DP == 128 ? 8 : (DP == 64 ? 4 : 1);
  static constexpr int RPT = DP / (RG * WARPS);
  static constexpr int HEADS = WARPS == 1 ? 4 : 1;  // heads of a block
  static constexpr int THREADS = WARPS * HEADS * 32;
};

template <typename T>
__device__ __forceinline__ float4 columns(const T* p, int c, int d, bool vec) {
  if (vec) return c < d ? load4(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 x;
  x.x = c < d ? to_f32<T>(p[c]) : 0.f;
  x.y = c + 1 < d ? to_f32<T>(p[c + 1]) : 0.f;
  x.z = c + 2 < d ? to_f32<T>(p[c + 2]) : 0.f;
  x.w = c + 3 < d ? to_f32<T>(p[c + 3]) : 0.f;
  return x;
}

// four columns of a row of S, streamed past the caches' reuse
__device__ __forceinline__ float4 load_state(const float* src, int c, int d, bool vec) {
  if (vec) return c < d ? __ldcs(reinterpret_cast<const float4*>(src + c))
                        : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 x;
  x.x = c < d ? src[c] : 0.f;
  x.y = c + 1 < d ? src[c + 1] : 0.f;
  x.z = c + 2 < d ? src[c + 2] : 0.f;
  x.w = c + 3 < d ? src[c + 3] : 0.f;
  return x;
}
__device__ __forceinline__ void store_state(float* dst, float4 x, int c, int d, bool vec) {
  if (vec) {
    if (c < d) __stcs(reinterpret_cast<float4*>(dst + c), x);
    return;
  }
  if (c < d) dst[c] = x.x;
  if (c + 1 < d) dst[c + 1] = x.y;
  if (c + 2 < d) dst[c + 2] = x.z;
  if (c + 3 < d) dst[c + 3] = x.w;
}

// ONE: a single row. With several, the rows' values are staged first, all
// loads in flight together, and their sums over S's rows meet at the end.
template <typename T, int DP, bool ONE>
__global__ void __launch_bounds__(DsPlan<DP>::THREADS) decay_step_kernel(DecayParams p,
                                                                         int vec_state) {
  using Plan = DsPlan<DP>;
  constexpr int RPT = Plan::RPT, WARPS = Plan::WARPS, RG = Plan::RG, LPR = Plan::LPR;
  constexpr int CB = Plan::CB, ROWS = ONE ? 1 : DS_ROWS, HEADS = Plan::HEADS;
  __shared__ float4 sums[WARPS > 1 ? ROWS : 1][WARPS > 1 ? WARPS : 1][LPR];
  __shared__ float qk[ONE ? 1 : HEADS][ONE ? 1 : 2 * ROWS][DP];
  __shared__ float4 vs[ONE ? 1 : HEADS][ROWS][LPR];
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS;
  const int own = (threadIdx.x >> 5) / WARPS;  // head of the block
  const int tid = threadIdx.x % (WARPS * 32);
  constexpr int PARTS = DP / CB;  // neighbouring blocks share a head
  const int64_t bh = (int64_t)(blockIdx.x / PARTS) * HEADS + own;
  if (bh >= (int64_t)p.B * p.H) return;  // whole warps; such blocks have no barriers
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int c0 = (int)(blockIdx.x % PARTS) * CB, c = c0 + (lane % LPR) * 4;
  const int row0 = warp * RG + lane / LPR;  // rows row0 + i RG WARPS
  const int len = decay_len(p, b);
  const DecayPower l(decay_rate(p.log_decay, h), 1.f);
  const int64_t base = bh * p.d * p.d;
  float4 S[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = row0 + i * RG * WARPS;
    S[i] = p.start && r < p.d ? load_state(p.start + base + (int64_t)r * p.d, c, p.d, vec_state)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const T* q = static_cast<const T*>(p.a) + b * p.sa.b + (h / p.ga) * p.sa.h;
  const T* k = static_cast<const T*>(p.b) + b * p.sb.b + (h / p.gb) * p.sb.h;
  const T* v = static_cast<const T*>(p.c) + b * p.sc.b + (h / p.gc) * p.sc.h;
  T* out = static_cast<T*>(p.out) + ((int64_t)b * p.N * p.H + h) * p.d;
  auto meet = [] {
    if constexpr (WARPS > 1)
      __syncthreads();
    else
      __syncwarp();
  };
  if constexpr (!ONE) {
    for (int e = tid; e < len * DP; e += WARPS * 32) {
      const int t = e / DP, r = e % DP;
      qk[own][2 * t][r] = r < p.d ? to_f32<T>(q[t * p.sa.n + r]) : 0.f;
      qk[own][2 * t + 1][r] = r < p.d ? to_f32<T>(k[t * p.sb.n + r]) : 0.f;
    }
    for (int e = tid; e < len * LPR; e += WARPS * 32)
      vs[own][e / LPR][e % LPR] =
          columns<T>(v + e / LPR * p.sc.n, c0 + e % LPR * 4, p.d, p.vec);
    meet();
  }
  auto write = [&](int t, int slot, float4 o) {
    const float y[4] = {o.x * p.out_scale, o.y * p.out_scale, o.z * p.out_scale,
                        o.w * p.out_scale};
    T* dst = out + (int64_t)t * p.H * p.d + c0 + slot * 4;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c0 + slot * 4 + u < p.d) dst[u] = from_f32<T>(y[u]);
  };
  // k and q ahead of the sums, where the compiler leaves their loads behind the
  // state's (2048 x 8 heads of 32 fp32 columns: 26.5 us, 30.4 without; elsewhere
  // the registers cost more)
  constexpr bool AHEAD = ONE && DP == 32 && sizeof(T) == 4;
  float ks[AHEAD ? RPT : 1], qs[AHEAD ? RPT : 1];
  if constexpr (AHEAD)
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = row0 + i * RG * WARPS;
      ks[i] = r < p.d ? to_f32<T>(k[r]) : 0.f;
      qs[i] = r < p.d ? to_f32<T>(q[r]) : 0.f;
    }
  const int rows = ONE ? 1 : p.N;
  for (int t = 0; t < rows; ++t) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t < len) {
      const float4 vv = ONE ? columns<T>(v, c, p.d, p.vec) : vs[ONE ? 0 : own][t][lane % LPR];
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = row0 + i * RG * WARPS;
        float kk, qq;
        if constexpr (AHEAD) {
          kk = ks[i];
          qq = qs[i];
        } else if constexpr (ONE) {
          kk = r < p.d ? to_f32<T>(k[r]) : 0.f;
          qq = r < p.d ? to_f32<T>(q[r]) : 0.f;
        } else {
          qq = qk[own][2 * t][r];
          kk = qk[own][2 * t + 1][r];
        }
        S[i].x = fmaf(kk, vv.x, l.times(S[i].x));
        S[i].y = fmaf(kk, vv.y, l.times(S[i].y));
        S[i].z = fmaf(kk, vv.z, l.times(S[i].z));
        S[i].w = fmaf(kk, vv.w, l.times(S[i].w));
        if (r < p.d) {  // rows beyond d are not there, even times an infinity
          o.x = fmaf(qq, S[i].x, o.x);
          o.y = fmaf(qq, S[i].y, o.y);
          o.z = fmaf(qq, S[i].z, o.z);
          o.w = fmaf(qq, S[i].w, o.w);
        }
      }
    }
    if (p.last && t + 1 == rows) {
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = row0 + i * RG * WARPS;
        if (r < p.d) store_state(p.last + base + (int64_t)r * p.d, S[i], c, p.d, vec_state);
      }
    }
#pragma unroll
    for (int s = LPR; s < 32; s <<= 1) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, s);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, s);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, s);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, s);
    }
    if (lane < LPR) {
      if constexpr (WARPS > 1)
        sums[t][warp][lane] = o;
      else
        write(t, lane, o);
    }
  }
  if constexpr (WARPS > 1) {
    __syncthreads();
    for (int e = tid; e < rows * LPR; e += WARPS * 32) {
      const int t = e / LPR, slot = e % LPR;
      float4 o = sums[t][0][slot];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) {
        const float4 x = sums[t][w][slot];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
      }
      write(t, slot, o);
    }
  }
}

template <typename T, int DP>
cudaError_t step_go(const DecayParams& p, cudaStream_t s) {
  using Plan = DsPlan<DP>;
  const int64_t heads = (int64_t)p.B * p.H;
  const unsigned blocks = (unsigned)((heads + Plan::HEADS - 1) / Plan::HEADS) * (DP / Plan::CB);
  const int vec_state = p.d % 4 == 0 && (uintptr_t)p.start % 16 == 0 && (uintptr_t)p.last % 16 == 0;
  if (p.N == 1)
    decay_step_kernel<T, DP, true><<<blocks, Plan::THREADS, 0, s>>>(p, vec_state);
  else
    decay_step_kernel<T, DP, false><<<blocks, Plan::THREADS, 0, s>>>(p, vec_state);
  return cudaGetLastError();
}
template <typename T>
cudaError_t step_width(const DecayParams& p, cudaStream_t s) {
  if (p.d <= 16) return step_go<T, 16>(p, s);
  if (p.d <= 32) return step_go<T, 32>(p, s);
  if (p.d <= 64) return step_go<T, 64>(p, s);
  return step_go<T, 128>(p, s);
}

}  // namespace

bool decay_step_takes(int N) { return N <= DS_ROWS; }

cudaError_t launch_decay_step(const DecayParams& p, bool bf16, cudaStream_t s) {
  return bf16 ? step_width<__nv_bfloat16>(p, s) : step_width<float>(p, s);
}

}  // namespace tarmac
