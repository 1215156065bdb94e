// Entry to the tensor-memory attention kernels alone, for the test builds that
// let a role of theirs give up (test_heads_give_up_gpu.py). bf16, contiguous
// [B, N, heads, d], every key visible; `delta` holds the row statistics.
#include "heads.cuh"

namespace tarmac {

cudaError_t raise_smem_limit(const void* fn, size_t bytes) {
  return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}
cudaError_t launch_head_fwd_tc(const HeadAttnParams& p, cudaStream_t s, bool* done);
cudaError_t launch_head_bwd_tc(const HeadAttnParams& p, int64_t nqp, cudaStream_t s, bool* done);

}  // namespace tarmac

using namespace tarmac;

static HeadAttnParams params(const void* q, const void* k, const void* v, int B, int N, int H,
                             int d, float scale) {
  HeadAttnParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.sq = p.sk = p.sv = p.so = p.sg = HeadStrides{(int64_t)N * H * d, (int64_t)H * d, d};
  p.bits_w = (N + 31) / 32;
  p.B = B;
  p.Nq = p.Nk = N;
  p.H = p.Hk = H;
  p.G = 1;
  p.d = d;
  p.peers = PEERS_ALL;
  p.scale = scale;
  p.vec = 1;
  p.splits = 1;
  return p;
}

#define ENTRY extern "C" __attribute__((visibility("default"))) int

// 0: launched; -1: not a call these kernels take; else a CUDA error
ENTRY forward(const void* q, const void* k, const void* v, void* out, float* lse, int B, int N,
              int H, int d, float scale, void* stream) {
  HeadAttnParams p = params(q, k, v, B, N, H, d, scale);
  p.o = out;
  p.lse = lse;
  bool done;
  const cudaError_t e = launch_head_fwd_tc(p, (cudaStream_t)stream, &done);
  return e != cudaSuccess ? (int)e : (done ? 0 : -1);
}

ENTRY backward(const void* q, const void* k, const void* v, const void* dout, float* delta,
               void* dq, void* dk, void* dv, int B, int N, int H, int d, float scale,
               void* stream) {
  HeadAttnParams p = params(q, k, v, B, N, H, d, scale);
  p.g = dout;
  p.delta = delta;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  bool done;
  const cudaError_t e = launch_head_bwd_tc(p, head_padded_rows(N), (cudaStream_t)stream, &done);
  return e != cudaSuccess ? (int)e : (done ? 0 : -1);
}
