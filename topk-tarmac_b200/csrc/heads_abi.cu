// heads_abi.cu — the extern "C" entry points of the multi-head operators
// declared in include/tarmac_b200.h: argument checks, parameters, launch.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "heads.cuh"

namespace tarmac {

cudaError_t launch_head_fwd(const HeadAttnParams& p, bool bf16, cudaStream_t s);
cudaError_t launch_head_bwd(const HeadAttnParams& p, bool bf16, cudaStream_t s);
int64_t head_fwd_tc_items(const HeadAttnParams& p);
bool head_bwd_tc_takes(const HeadAttnParams& p);
int head_splits(int B, int Nq, int Nk, int H, int Hk);
cudaError_t launch_pack_bits(const void* v, int64_t sb, int64_t sn, int B, int Nq, int Nk,
                             uint32_t* out, cudaStream_t s);

namespace {

constexpr int MAX_D = 128;

bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
int status(cudaError_t e) { return e == cudaSuccess ? TARMAC_OK : TARMAC_ERR_LAUNCH; }
int64_t round16(int64_t bytes) { return (bytes + 15) & ~(int64_t)15; }

// strides of tensor i (three int64 each), or those of a contiguous
// [B, N, h, d] tensor
HeadStrides stride_of(const int64_t* strides, int i, int64_t N, int64_t h, int64_t d) {
  if (strides) return HeadStrides{strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
  return HeadStrides{N * h * d, h * d, d};
}

int check_rotate(const void* q, const void* k, const float* cs, const float* sn, int B, int N,
                 int H, int Hk, int d, int r, int dtype, float eps) {
  if (dtype != TARMAC_F32 && dtype != TARMAC_BF16) return TARMAC_ERR_DTYPE;
  if (B < 0 || N < 0 || d < 1 || d > MAX_D) return TARMAC_ERR_SHAPE;
  if (H < 1 || Hk < 1 || r < 0 || r > d || (r & 1)) return TARMAC_ERR_HEADS;
  if (!(eps >= 0.f) || isinf(eps)) return TARMAC_ERR_SHAPE;
  if ((int64_t)B * N == 0) return TARMAC_OK;
  if ((int64_t)B * N > 0x7fffffff) return TARMAC_ERR_N_TOO_LARGE;  // rows in 31 bits
  if (!q || !k || (r > 0 && (!cs || !sn))) return TARMAC_ERR_NULL;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  if (!aligned(q, es) || !aligned(k, es) || !aligned(cs, 4) || !aligned(sn, 4))
    return TARMAC_ERR_ALIGN;
  return TARMAC_OK;
}

// Checks shared by both directions; fills everything but the strides.
int fill_attn(HeadAttnParams& p, const void* q, const void* k, const void* v,
              const int32_t* key_len, const int32_t* q_start, const uint32_t* bits,
              int64_t bits_b, int B, int Nq, int Nk, int H, int Hk, int d, int dtype, int peers,
              float scale) {
  if (dtype != TARMAC_F32 && dtype != TARMAC_BF16) return TARMAC_ERR_DTYPE;
  if (B < 0 || Nq < 0 || Nk < 0 || d < 1 || d > MAX_D) return TARMAC_ERR_SHAPE;
  // row and key counts stay below 2^29 (position arithmetic in 32 bits), rows
  // times heads of an episode below 2^31
  if (Nk > (1 << 29) || Nq > (1 << 29)) return TARMAC_ERR_N_TOO_LARGE;
  if (H < 1 || Hk < 1 || H % Hk) return TARMAC_ERR_HEADS;
  if ((int64_t)head_padded_rows(Nq) * H > 0x7fffff00) return TARMAC_ERR_N_TOO_LARGE;
  if (peers < PEERS_ALL || peers > PEERS_PAST) return TARMAC_ERR_MODE;
  if (!(scale > 0.f) || isinf(scale)) return TARMAC_ERR_SHAPE;
  if (!aligned(key_len, 4) || !aligned(q_start, 4) || !aligned(bits, 4)) return TARMAC_ERR_ALIGN;
  const int64_t nq = (int64_t)B * Nq, nk = (int64_t)B * Nk;
  if ((nq && !q) || (nk && (!k || !v))) return TARMAC_ERR_NULL;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es)) return TARMAC_ERR_ALIGN;
  p = HeadAttnParams{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.key_len = key_len;
  p.q_start = q_start;
  p.bits = bits;
  p.bits_b = bits_b;
  p.bits_w = cdiv(Nk, 32);
  p.B = B;
  p.Nq = Nq;
  p.Nk = Nk;
  p.H = H;
  p.Hk = Hk;
  p.G = H / Hk;
  p.d = d;
  p.peers = peers;
  p.scale = scale;
  p.splits = 1;
  return TARMAC_OK;
}

// may rows of this tensor be moved 16 bytes at a time?
bool vec_ok(const void* ptr, const HeadStrides& s, int es) {
  const int e = 16 / es;
  return aligned(ptr, 16) && s.b % e == 0 && s.n % e == 0 && s.h % e == 0;
}

}  // namespace
}  // namespace tarmac

using namespace tarmac;

extern "C" {

int tarmac_qk_norm_rotate(const void* q, const void* k, void* q_out, void* k_out,
                          const int64_t* strides, const float* wq, const float* wk,
                          const float* cos, const float* sin, int64_t table_b, int B, int N,
                          int H, int Hk, int d, int r, int dtype, float eps, int interleaved,
                          void* stream) {
  const int st = check_rotate(q, k, cos, sin, B, N, H, Hk, d, r, dtype, eps);
  if (st != TARMAC_OK || (int64_t)B * N == 0) return st;
  if (!q_out || !k_out) return TARMAC_ERR_NULL;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  if (!aligned(q_out, es) || !aligned(k_out, es) || !aligned(wq, 4) || !aligned(wk, 4))
    return TARMAC_ERR_ALIGN;
  RotateParams p = {};
  p.q = q;
  p.k = k;
  p.oq = q_out;
  p.ok = k_out;
  p.sq = stride_of(strides, 0, N, H, d);
  p.sk = stride_of(strides, 1, N, Hk, d);
  p.wq = wq;
  p.wk = wk;
  p.cos = cos;
  p.sin = sin;
  p.table_b = table_b;
  p.B = B;
  p.N = N;
  p.H = H;
  p.Hk = Hk;
  p.d = d;
  p.r = r;
  p.eps = eps;
  p.interleaved = interleaved != 0;
  return status(launch_rotate(p, dtype == TARMAC_BF16, (cudaStream_t)stream));
}

int64_t tarmac_qk_norm_rotate_workspace(int B, int N, int H, int Hk, int d) {
  if (B < 1 || N < 1 || H < 1 || Hk < 1 || d < 1 || d > MAX_D) return 0;
  return rotate_bwd_work((int64_t)B * N, H, Hk, d) * 4;
}

int tarmac_qk_norm_rotate_backward(const void* q, const void* k, const void* dq_out,
                                   const void* dk_out, const int64_t* strides, const float* wq,
                                   const float* wk, const float* cos, const float* sin,
                                   int64_t table_b, int B, int N, int H, int Hk, int d, int r,
                                   int dtype, float eps, int interleaved, void* dq, void* dk,
                                   float* dwq, float* dwk, void* work, void* stream) {
  const int st = check_rotate(q, k, cos, sin, B, N, H, Hk, d, r, dtype, eps);
  if (st != TARMAC_OK) return st;
  if (!aligned(dwq, 4) || !aligned(dwk, 4)) return TARMAC_ERR_ALIGN;
  cudaStream_t s = (cudaStream_t)stream;
  if ((int64_t)B * N == 0) {  // no rows: the weights' gradients are zero
    cudaError_t e = cudaSuccess;
    if (dwq) e = cudaMemsetAsync(dwq, 0, (size_t)d * 4, s);
    if (e == cudaSuccess && dwk) e = cudaMemsetAsync(dwk, 0, (size_t)d * 4, s);
    return status(e);
  }
  if (!dq_out || !dk_out || !dq || !dk || !work) return TARMAC_ERR_NULL;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  const void* el[4] = {dq_out, dk_out, dq, dk};
  for (const void* ptr : el)
    if (!aligned(ptr, es)) return TARMAC_ERR_ALIGN;
  if (!aligned(wq, 4) || !aligned(wk, 4) || !aligned(work, 16)) return TARMAC_ERR_ALIGN;
  RotateParams p = {};
  p.q = q;
  p.k = k;
  p.gq = dq_out;
  p.gk = dk_out;
  p.oq = dq;
  p.ok = dk;
  p.sq = stride_of(strides, 0, N, H, d);
  p.sk = stride_of(strides, 1, N, Hk, d);
  p.sgq = stride_of(strides, 2, N, H, d);
  p.sgk = stride_of(strides, 3, N, Hk, d);
  p.wq = wq;
  p.wk = wk;
  p.cos = cos;
  p.sin = sin;
  p.table_b = table_b;
  p.dwq = dwq;
  p.dwk = dwk;
  p.work = static_cast<float*>(work);
  p.B = B;
  p.N = N;
  p.H = H;
  p.Hk = Hk;
  p.d = d;
  p.r = r;
  p.eps = eps;
  p.interleaved = interleaved != 0;
  return status(launch_rotate_bwd(p, dtype == TARMAC_BF16, s));
}

int tarmac_pack_visibility(const void* visible, int64_t stride_b, int64_t stride_n, int B, int Nq,
                           int Nk, void* bits, void* stream) {
  if (B < 0 || Nq < 0 || Nk < 0) return TARMAC_ERR_SHAPE;
  if ((int64_t)B * Nq * Nk == 0) return TARMAC_OK;
  if (!visible || !bits) return TARMAC_ERR_NULL;
  if (!aligned(bits, 4)) return TARMAC_ERR_ALIGN;
  return status(launch_pack_bits(visible, stride_b, stride_n, B, Nq, Nk,
                                 static_cast<uint32_t*>(bits), (cudaStream_t)stream));
}

int64_t tarmac_head_attention_workspace(int B, int Nq, int Nk, int H, int Hk, int d) {
  if (B < 1 || Nq < 1 || Nk < 1 || Hk < 1 || H < Hk || H % Hk || d < 1 || d > MAX_D) return 0;
  const int splits = head_splits(B, Nq, Nk, H, Hk);
  if (splits == 1) return 0;
  const int64_t rows = (int64_t)B * Nq * H;
  return round16(splits * rows * d * 4) + round16(splits * rows * 4);
}

int tarmac_head_attention(const void* q, const void* k, const void* v, void* out, float* lse,
                          const int64_t* strides, const int32_t* key_len, const int32_t* q_start,
                          const void* bits, int64_t bits_b, int B, int Nq, int Nk, int H, int Hk,
                          int d, int dtype, int peers, float scale, void* work, void* stream) {
  HeadAttnParams p;
  const int st = fill_attn(p, q, k, v, key_len, q_start, static_cast<const uint32_t*>(bits),
                           bits_b, B, Nq, Nk, H, Hk, d, dtype, peers, scale);
  if (st != TARMAC_OK || (int64_t)B * Nq == 0) return st;
  if (!out) return TARMAC_ERR_NULL;
  if (!aligned(out, 16) || !aligned(lse, 4) || !aligned(work, 16)) return TARMAC_ERR_ALIGN;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  p.o = out;
  p.lse = lse;
  p.sq = stride_of(strides, 0, Nq, H, d);
  p.sk = stride_of(strides, 1, Nk, Hk, d);
  p.sv = stride_of(strides, 2, Nk, Hk, d);
  p.vec = d * es % 16 == 0 && vec_ok(q, p.sq, es) && vec_ok(k, p.sk, es) && vec_ok(v, p.sv, es);
  if (Nk > 0) p.splits = head_splits(B, Nq, Nk, H, Hk);
  if (p.splits > 1) {
    if (!work) return TARMAC_ERR_NULL;
    const int64_t rows = (int64_t)B * Nq * H;
    p.part_o = static_cast<float*>(work);
    p.part_lse = reinterpret_cast<float*>(static_cast<char*>(work) +
                                          round16(p.splits * rows * d * 4));
  }
  return status(launch_head_fwd(p, dtype == TARMAC_BF16, (cudaStream_t)stream));
}

int64_t tarmac_head_attention_backward_workspace(int B, int Nq, int H) {
  return B < 1 || Nq < 1 || H < 1 ? 0 : (int64_t)2 * B * head_padded_rows(Nq) * H * 4;
}

int tarmac_head_attention_backward(const void* q, const void* k, const void* v, const void* out,
                                   const float* lse, const void* dout, const int64_t* strides,
                                   const int32_t* key_len, const int32_t* q_start,
                                   const void* bits, int64_t bits_b, int B, int Nq, int Nk, int H,
                                   int Hk, int d, int dtype, int peers, float scale, void* dq,
                                   void* dk, void* dv, void* work, void* stream) {
  HeadAttnParams p;
  const int st = fill_attn(p, q, k, v, key_len, q_start, static_cast<const uint32_t*>(bits),
                           bits_b, B, Nq, Nk, H, Hk, d, dtype, peers, scale);
  if (st != TARMAC_OK || (int64_t)B * Nq + (int64_t)B * Nk == 0) return st;
  const int64_t nq = (int64_t)B * Nq, nk = (int64_t)B * Nk;
  if ((nq && (!out || !lse || !dout || !dq || !work)) || (nk && (!dk || !dv)))
    return TARMAC_ERR_NULL;
  if (!aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16) || !aligned(work, 16) ||
      !aligned(lse, 4))
    return TARMAC_ERR_ALIGN;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  if (!aligned(out, es) || !aligned(dout, es)) return TARMAC_ERR_ALIGN;
  p.o = const_cast<void*>(out);
  p.lse = const_cast<float*>(lse);
  p.g = dout;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.delta = static_cast<float*>(work);
  p.sq = stride_of(strides, 0, Nq, H, d);
  p.sk = stride_of(strides, 1, Nk, Hk, d);
  p.sv = stride_of(strides, 2, Nk, Hk, d);
  p.so = stride_of(strides, 3, Nq, H, d);
  p.sg = stride_of(strides, 4, Nq, H, d);
  p.vec = d * es % 16 == 0 && vec_ok(q, p.sq, es) && vec_ok(k, p.sk, es) &&
          vec_ok(v, p.sv, es) && vec_ok(out, p.so, es) && vec_ok(dout, p.sg, es);
  return status(launch_head_bwd(p, dtype == TARMAC_BF16, (cudaStream_t)stream));
}

int tarmac_head_attention_plan(int backward, const int64_t* strides, int B, int Nq, int Nk, int H,
                               int Hk, int d, int dtype, int peers, char* out, int len) {
  if (!out || len < 1) return TARMAC_ERR_NULL;
  out[0] = '\0';
  // only shapes, strides and alignment count: stand-in pointers on the grid
  const void* a = reinterpret_cast<const void*>((uintptr_t)1 << 20);
  HeadAttnParams p;
  const int st = fill_attn(p, a, a, a, nullptr, nullptr, nullptr, 0, B, Nq, Nk, H, Hk, d, dtype,
                           peers, 1.f);
  if (st != TARMAC_OK) return st;
  const bool bf16 = dtype == TARMAC_BF16;
  const int es = bf16 ? 2 : 4;
  p.sq = stride_of(strides, 0, Nq, H, d);
  p.sk = stride_of(strides, 1, Nk, Hk, d);
  p.sv = stride_of(strides, 2, Nk, Hk, d);
  p.vec = d * es % 16 == 0 && vec_ok(a, p.sq, es) && vec_ok(a, p.sk, es) && vec_ok(a, p.sv, es);
  char buf[128];
  if (backward) {
    p.so = stride_of(strides, 3, Nq, H, d);
    p.sg = stride_of(strides, 4, Nq, H, d);
    p.vec = p.vec && vec_ok(a, p.so, es) && vec_ok(a, p.sg, es);
    const bool tc = bf16 && head_bwd_tc_takes(p);
    const int tile = tc ? 128 : 64;
    const int64_t rows = tc ? (int64_t)p.H * cdiv(Nq, 128) : (int64_t)p.Hk * cdiv(Nq * p.G, 64);
    snprintf(buf, sizeof buf, "{\"kernel\": \"%s\", \"dq_items\": %lld, \"dkv_items\": %lld}",
             tc ? "head_bwd_tc" : "head_bwd", (long long)(B * rows),
             (long long)((int64_t)B * Hk * cdiv(Nk, tile)));
  } else {
    if (Nk > 0) p.splits = head_splits(B, Nq, Nk, H, Hk);
    const int64_t items = bf16 ? head_fwd_tc_items(p) : 0;
    if (items)
      snprintf(buf, sizeof buf, "{\"kernel\": \"head_fwd_tc\", \"items\": %lld}",
               (long long)items);
    else
      snprintf(buf, sizeof buf, "{\"kernel\": \"head_fwd\", \"parts\": %d}", p.splits);
  }
  const int n = (int)strlen(buf);
  if (n + 1 > len) return TARMAC_ERR_SHAPE;
  memcpy(out, buf, (size_t)n + 1);
  return TARMAC_OK;
}

}  // extern "C"
