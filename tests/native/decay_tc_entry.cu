// Entry to the tensor-memory kernels of attention with a decay alone, for the
// test builds that let a role of theirs give up (test_decay_give_up_gpu.py).
// bf16, contiguous [B, N, H, d], one segment.
#include "decay.cuh"

namespace tarmac {

cudaError_t raise_smem_limit(const void* fn, size_t bytes) {
  return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

}  // namespace tarmac

using namespace tarmac;

#define ENTRY extern "C" __attribute__((visibility("default"))) int

static DecayParams params(const void* a, const void* b, const void* c, const float* log_decay,
                          int B, int N, int H, int d) {
  DecayParams p = {};
  p.a = a;
  p.b = b;
  p.c = c;
  p.sa = p.sb = p.sc = HeadStrides{(int64_t)N * H * d, (int64_t)H * d, d};
  p.ga = p.gb = p.gc = 1;
  p.log_decay = log_decay;
  p.B = B;
  p.N = N;
  p.H = H;
  p.d = d;
  p.segs = 1;
  p.seg_chunks = cdiv(N, DECAY_TC_CHUNK);
  p.in_scale = p.out_scale = 1.f;
  p.tc = p.vec = p.planes = 1;
  return p;
}

ENTRY rows(const void* a, const void* b, const void* c, const float* log_decay, void* out, int B,
           int N, int H, int d, void* stream) {
  DecayParams p = params(a, b, c, log_decay, B, N, H, d);
  p.out = out;
  return (int)launch_decay_rows_tc(&p, 1, (cudaStream_t)stream);
}

// what the rows add to the state
ENTRY states(const void* b, const void* c, const float* log_decay, float* part, int B, int N,
             int H, int d, void* stream) {
  DecayParams p = params(b, b, c, log_decay, B, N, H, d);
  p.part = p.last = part;  // p.last: the last segment counts
  return (int)launch_decay_states_tc(p, (cudaStream_t)stream);
}
