// heads.cuh — parameters of the multi-head operators: head norms with the
// position rotation (head_rotate.cu) and masked attention with heads
// (head_attn.cu and the tensor-memory kernels beside it).
//
// Tensors are [B, N, h, d] with unit innermost stride and any batch, row and
// head strides (in elements, 64-bit: a long history passes 2^31 elements).
#pragma once

#include "common.cuh"

namespace tarmac {

// batch, row and head stride of one [B, N, h, d] tensor, in elements
struct HeadStrides {
  int64_t b, n, h;
};

struct RotateParams {
  const void *q, *k;    // inputs
  const void *gq, *gk;  // backward: gradients of the outputs
  void *oq, *ok;        // outputs (forward) or input gradients, contiguous
  HeadStrides sq, sk, sgq, sgk;
  const float *wq, *wk;       // [d] or NULL (ones)
  const float *cos, *sin;     // [Bt, N, r / 2]
  int64_t table_b;            // batch stride of the tables (0: one for all)
  float *dwq, *dwk;           // [d] or NULL
  float* work;                // backward: rows of d sums
  int B, N, H, Hk, d, r;
  float eps;
  int interleaved;
};

cudaError_t launch_rotate(const RotateParams& p, bool bf16, cudaStream_t s);
cudaError_t launch_rotate_bwd(const RotateParams& p, bool bf16, cudaStream_t s);
// floats of `work` that the backward call needs at most
int64_t rotate_bwd_work(int64_t tokens, int H, int Hk, int d);

// who a row may see (beside key_len and the visibility words)
enum HeadPeers { PEERS_ALL = 0, PEERS_OTHERS = 1, PEERS_PAST = 2 };

struct HeadAttnParams {
  const void *q, *k, *v;
  void* o;                    // forward output / backward: the forward's output
  float* lse;                 // [B, H, Nq], natural log
  const void* g;              // backward: dL/dout
  void *dq, *dk, *dv;         // backward: contiguous, the inputs' type
  HeadStrides sq, sk, sv, so, sg;
  const int32_t* key_len;     // [B] or NULL
  const int32_t* q_start;     // [B] or NULL (then Nk - Nq for all)
  const uint32_t* bits;       // visibility words [Bv, Nq, bits_w] or NULL
  int64_t bits_b;             // their batch stride in words (0: one for all)
  int bits_w;                 // words per row, ceil(Nk / 32)
  int B, Nq, Nk, H, Hk, G, d; // G = H / Hk
  int peers;
  float scale;
  int vec;                    // 16-byte rows everywhere
  int splits;                 // forward: parts of the key axis
  float* part_o;              // [splits, B, Nq, H, d]
  float* part_lse;            // [splits, B, H, Nq]
  float* delta;               // backward: row statistics (head_attn.cu)
};

// rows of the backward's statistics per head: whole 128-row tiles
__host__ __device__ constexpr int head_padded_rows(int Nq) { return cdiv(Nq, 128) * 128; }

}  // namespace tarmac
