// decay_step.cu — attention with a decay for each head over few rows: the
// recurrent form, one row after the other.
//
//   S = l S + k v^T,  out = scale S^T q
// for each row, with S in registers between them. Bound by memory: a call on
// one row reads and writes the state, 8 d^2 bytes a head, and little else.
// A thread holds four neighbouring columns of RPT of S's rows; the lanes of a
// row are neighbours, so a warp moves whole 16-byte vectors of consecutive
// rows. Only the sum over S's rows crosses threads: by shuffles in the warp,
// then through shared memory. The state may be renewed in place: a block reads
// its head's state before it writes it.
#include "decay.cuh"

namespace tarmac {

namespace {

// DP columns: LPR lanes a row, RG rows a warp at once, WARPS warps a head
template <int DP>
struct DsPlan {
  static constexpr int LPR = DP / 4, RG = 32 / LPR;
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

template <typename T, int DP>
__global__ void __launch_bounds__(DsPlan<DP>::THREADS) decay_step_kernel(DecayParams p,
                                                                         int vec_state) {
  using Plan = DsPlan<DP>;
  constexpr int RPT = Plan::RPT, WARPS = Plan::WARPS, RG = Plan::RG, LPR = Plan::LPR;
  __shared__ float4 sums[WARPS > 1 ? WARPS : 1][LPR];
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WARPS;
  const int64_t bh = (int64_t)blockIdx.x * Plan::HEADS + (threadIdx.x >> 5) / WARPS;
  if (bh >= (int64_t)p.B * p.H) return;  // whole warps; such blocks have no barriers
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int c = (lane % LPR) * 4, row0 = warp * RG + lane / LPR;  // rows row0 + i RG WARPS
  const int len = decay_len(p, b);
  const float l = expf(decay_rate(p.log_decay, h));
  const int64_t base = bh * p.d * p.d;
  float4 S[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = row0 + i * RG * WARPS;
    S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.start && r < p.d) {
      const float* src = p.start + base + (int64_t)r * p.d;
      if (vec_state) {
        if (c < p.d) S[i] = *reinterpret_cast<const float4*>(src + c);
      } else {
        if (c < p.d) S[i].x = src[c];
        if (c + 1 < p.d) S[i].y = src[c + 1];
        if (c + 2 < p.d) S[i].z = src[c + 2];
        if (c + 3 < p.d) S[i].w = src[c + 3];
      }
    }
  }
  const T* q = static_cast<const T*>(p.a) + b * p.sa.b + (h / p.ga) * p.sa.h;
  const T* k = static_cast<const T*>(p.b) + b * p.sb.b + (h / p.gb) * p.sb.h;
  const T* v = static_cast<const T*>(p.c) + b * p.sc.b + (h / p.gc) * p.sc.h;
  T* out = static_cast<T*>(p.out) + ((int64_t)b * p.N * p.H + h) * p.d;
  for (int t = 0; t < p.N; ++t, q += p.sa.n, k += p.sb.n, v += p.sc.n,
           out += (int64_t)p.H * p.d) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t < len) {
      const float4 vv = columns<T>(v, c, p.d, p.vec);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = row0 + i * RG * WARPS;
        const float kk = r < p.d ? to_f32<T>(k[r]) : 0.f, qq = r < p.d ? to_f32<T>(q[r]) : 0.f;
        S[i].x = fmaf(l, S[i].x, kk * vv.x);
        S[i].y = fmaf(l, S[i].y, kk * vv.y);
        S[i].z = fmaf(l, S[i].z, kk * vv.z);
        S[i].w = fmaf(l, S[i].w, kk * vv.w);
        if (r < p.d) {
          o.x = fmaf(qq, S[i].x, o.x);
          o.y = fmaf(qq, S[i].y, o.y);
          o.z = fmaf(qq, S[i].z, o.z);
          o.w = fmaf(qq, S[i].w, o.w);
        }
      }
    }
#pragma unroll
    for (int s = LPR; s < 32; s <<= 1) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, s);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, s);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, s);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, s);
    }
    if constexpr (WARPS > 1) {
      if (t > 0) __syncthreads();  // the sums of the row before have been read
      if (lane < LPR) sums[warp][lane] = o;
      __syncthreads();
      if (warp == 0 && lane < LPR) {
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
          const float4 x = sums[w][lane];
          o.x += x.x;
          o.y += x.y;
          o.z += x.z;
          o.w += x.w;
        }
      }
    }
    if (warp == 0 && lane < LPR) {
      const float y[4] = {o.x * p.out_scale, o.y * p.out_scale, o.z * p.out_scale,
                          o.w * p.out_scale};
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u < p.d) out[c + u] = from_f32<T>(y[u]);
    }
  }
  if (!p.last) return;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = row0 + i * RG * WARPS;
    if (r >= p.d) continue;
    float* dst = p.last + base + (int64_t)r * p.d;
    if (vec_state) {
      if (c < p.d) *reinterpret_cast<float4*>(dst + c) = S[i];
    } else {
      if (c < p.d) dst[c] = S[i].x;
      if (c + 1 < p.d) dst[c + 1] = S[i].y;
      if (c + 2 < p.d) dst[c + 2] = S[i].z;
      if (c + 3 < p.d) dst[c + 3] = S[i].w;
    }
  }
}

template <typename T, int DP>
cudaError_t step_go(const DecayParams& p, cudaStream_t s) {
  using Plan = DsPlan<DP>;
  const int64_t heads = (int64_t)p.B * p.H;
  const unsigned blocks = (unsigned)((heads + Plan::HEADS - 1) / Plan::HEADS);
  const int vec_state = p.d % 4 == 0 && (uintptr_t)p.start % 16 == 0 && (uintptr_t)p.last % 16 == 0;
  decay_step_kernel<T, DP><<<blocks, Plan::THREADS, 0, s>>>(p, vec_state);
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

bool decay_step_takes(int N) { return N <= 8; }

cudaError_t launch_decay_step(const DecayParams& p, bool bf16, cudaStream_t s) {
  return bf16 ? step_width<__nv_bfloat16>(p, s) : step_width<float>(p, s);
}

}  // namespace tarmac
