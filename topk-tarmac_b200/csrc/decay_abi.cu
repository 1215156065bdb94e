// decay_abi.cu — the extern "C" entry points of attention with a decay for
// each head and of the norms around a block, declared in
// include/tarmac_b200.h: argument checks, parameters, launch.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "block_norm.cuh"
#include "decay.cuh"

namespace tarmac {

bool head_map_ok(const HeadStrides& s, int B, int N, int h);

namespace {

constexpr int MAX_D = 128;
constexpr int GRADIENTS = 3;  // sums of a backward call: dq, dv, dk

bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
int status(cudaError_t e) { return e == cudaSuccess ? TARMAC_OK : TARMAC_ERR_LAUNCH; }
int64_t round16(int64_t bytes) { return (bytes + 15) & ~(int64_t)15; }

HeadStrides stride_of(const int64_t* strides, int i, int64_t N, int64_t h, int64_t d) {
  if (strides) return HeadStrides{strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
  return HeadStrides{N * h * d, h * d, d};
}
bool vec_ok(const void* ptr, const HeadStrides& s, int es) {
  const int e = 16 / es;
  return aligned(ptr, 16) && s.b % e == 0 && s.n % e == 0 && s.h % e == 0;
}

int check_sizes(int B, int N, int H, int Hk, int d, int dtype) {
  if (dtype != TARMAC_F32 && dtype != TARMAC_BF16) return TARMAC_ERR_DTYPE;
  if (B < 0 || N < 0 || d < 1 || d > MAX_D) return TARMAC_ERR_SHAPE;
  if (H < 1 || Hk < 1 || H % Hk) return TARMAC_ERR_HEADS;
  // rows in 29 bits, blocks of a launch in 31
  if (N > (1 << 29) || (int64_t)B * H > (1 << 24)) return TARMAC_ERR_N_TOO_LARGE;
  return TARMAC_OK;
}

// Checks shared by both directions; fills what they share.
int fill_decay(DecayParams& p, const void* q, const void* k, const void* v,
               const float* log_decay, const float* state, const int32_t* lens, int B, int N,
               int H, int Hk, int d, int dtype, float scale) {
  const int st = check_sizes(B, N, H, Hk, d, dtype);
  if (st != TARMAC_OK) return st;
  if (!(scale > 0.f) || isinf(scale)) return TARMAC_ERR_SHAPE;
  if (!aligned(lens, 4) || !aligned(log_decay, 4) || !aligned(state, 4)) return TARMAC_ERR_ALIGN;
  if (B > 0 && (!log_decay || (N > 0 && (!q || !k || !v)))) return TARMAC_ERR_NULL;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es)) return TARMAC_ERR_ALIGN;
  p = DecayParams{};
  p.log_decay = log_decay;
  p.lens = lens;
  p.B = B;
  p.N = N;
  p.H = H;
  p.d = d;
  return TARMAC_OK;
}

void set_plan(DecayParams& p, bool tc, int jobs) {
  const DecayPlan g = decay_plan(p.B, p.N, p.H, p.d, tc, jobs);
  p.segs = g.segs;
  p.seg_chunks = g.seg_chunks;
  p.tc = tc;
}
// Does a launch of its own join the segments' states? Up to 32 columns off the
// tensor memory the rows' kernel joins few of them as it starts, in less than a
// launch takes (16 states of 16 x 16 a head: 4.8 us). On the tensor memory that
// was slower (4 of 128 x 128: 26 us more against 9).
void set_joined(DecayParams& p) {
  p.joined = !decay_one_walk(p.d, p.tc) || p.segs > 24;
}
// bytes of p.part, 0 where the call does not use it
int64_t part_bytes(int B, int N, int H, int d, bool tc, int jobs, bool last) {
  const DecayPlan g = decay_plan(B, N, H, d, tc, jobs);
  return decay_uses_part(g, tc, last) ? round16(decay_part_bytes(g, B, H, d, tc)) : 0;
}
// Up to 32 columns off the tensor memory the blocks of every segment read p.start
// and those of the last write p.last. Where the two are one, all read a copy,
// behind p.part. Its bytes, for a call that returns a state:
int64_t copy_bytes(int B, int N, int H, int d, bool tc) {
  if (!decay_one_walk(d, tc) || decay_plan(B, N, H, d, tc, 1).segs == 1) return 0;
  return round16((int64_t)B * H * d * d * 4);
}
// The gradients' scratch: states forwards at 0, backwards at `back` (on the tensor
// memory both are needed at once), the gradients of shared heads by query head,
// dv and dk, before their sum.
struct BackwardWork {
  int64_t back, dv, dk, bytes;
};
BackwardWork backward_work(int B, int N, int H, int Hk, int d, bool tc, bool dstate) {
  const int64_t ahead = part_bytes(B, N, H, d, tc, GRADIENTS, false);
  const int64_t behind = part_bytes(B, N, H, d, tc, GRADIENTS, dstate);
  const int64_t shared = H == Hk ? 0 : round16((int64_t)B * N * H * d * 4);
  BackwardWork w;
  w.back = tc ? ahead : 0;
  w.dv = w.back + behind;
  w.dk = w.dv + shared;
  w.bytes = w.dk + shared;
  return w;
}

// one operand: pointer, strides and how many heads share one of its heads
struct Operand {
  const void* ptr;
  HeadStrides s;
  int share;
  bool vec, map;  // rows are vectors; TMA can describe them
};
Operand operand(const void* ptr, const HeadStrides& s, int B, int N, int H, int share, int d,
                int es) {
  const bool vec = d * es % 16 == 0 && vec_ok(ptr, s, es);
  return Operand{ptr, s, share, vec, vec && es == 2 && head_map_ok(s, B, N, H / share)};
}
void set_operands(DecayParams& p, const Operand& a, const Operand& b, const Operand& c) {
  p.a = a.ptr;
  p.b = b.ptr;
  p.c = c.ptr;
  p.sa = a.s;
  p.sb = b.s;
  p.sc = c.s;
  p.ga = a.share;
  p.gb = b.share;
  p.gc = c.share;
  p.vec = a.vec && b.vec && c.vec;
}

void set_extra(DecayParams& p, const Operand& x) {
  p.e = x.ptr;
  p.se = x.s;
  p.ge = x.share;
  p.vec = p.vec && x.vec;
}

// a state as it is, or zero
cudaError_t carry_state(const float* from, float* to, int64_t n, cudaStream_t s) {
  if (!to || n == 0 || from == to) return cudaSuccess;
  if (!from) return cudaMemsetAsync(to, 0, (size_t)n * 4, s);
  return cudaMemcpyAsync(to, from, (size_t)n * 4, cudaMemcpyDeviceToDevice, s);
}

// episode and row stride of tensor i (two int64 each), or those of a
// contiguous [B, N, D] tensor
RowStrides rows_of(const int64_t* strides, int i, int64_t N, int64_t D) {
  if (strides) return RowStrides{strides[2 * i], strides[2 * i + 1]};
  return RowStrides{N * D, D};
}

// Checks shared by both directions; fills what they share.
int fill_norm(NormParams& p, const void* x, const void* y, const void* gate,
              const int64_t* strides, const float* w_post, const float* w_pre,
              const float* scale, int B, int N, int D, int dtype, float eps) {
  if (dtype != TARMAC_F32 && dtype != TARMAC_BF16) return TARMAC_ERR_DTYPE;
  if (B < 0 || N < 0 || D < 1 || D > NORM_MAX_D) return TARMAC_ERR_SHAPE;
  if (!(eps >= 0.f) || isinf(eps)) return TARMAC_ERR_SHAPE;
  if ((int64_t)B * N > 0x7fffffff) return TARMAC_ERR_N_TOO_LARGE;  // rows in 31 bits
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  if (!aligned(x, es) || !aligned(y, es) || !aligned(gate, es)) return TARMAC_ERR_ALIGN;
  if (!aligned(w_post, 4) || !aligned(w_pre, 4) || !aligned(scale, 4)) return TARMAC_ERR_ALIGN;
  if ((int64_t)B * N > 0 && (!x || !y)) return TARMAC_ERR_NULL;
  p = NormParams{};
  p.x = x;
  p.y = y;
  p.gate = gate;
  p.sx = rows_of(strides, 0, N, D);
  p.sy = rows_of(strides, 1, N, D);
  p.sg = rows_of(strides, 2, N, D);
  p.w_post = w_post;
  p.w_pre = w_pre;
  p.scale = scale;
  p.B = B;
  p.N = N;
  p.D = D;
  p.eps = eps;
  return TARMAC_OK;
}

}  // namespace
}  // namespace tarmac

using namespace tarmac;

extern "C" {

int64_t tarmac_decay_attention_workspace(int B, int N, int H, int d, int dtype, int state_out) {
  if (check_sizes(B, N, H, 1, d, dtype) != TARMAC_OK || B < 1 || N < 1) return 0;
  if (decay_step_takes(N)) return 0;
  int64_t bytes = 0;  // whichever kernels the rows' layout allows
  for (int tc = 0; tc <= (int)decay_tc_sizes(B, N, H, d, dtype == TARMAC_BF16); ++tc) {
    const int64_t n = part_bytes(B, N, H, d, tc != 0, 1, state_out != 0) +
                      (state_out ? copy_bytes(B, N, H, d, tc != 0) : 0);
    if (n > bytes) bytes = n;
  }
  return bytes;
}

int tarmac_decay_attention(const void* q, const void* k, const void* v, void* out,
                           const int64_t* strides, const float* log_decay, const float* state,
                           float* state_out, const int32_t* lens, int B, int N, int H, int Hk,
                           int d, int dtype, float scale, void* work, void* stream) {
  DecayParams p;
  const int st = fill_decay(p, q, k, v, log_decay, state, lens, B, N, H, Hk, d, dtype, scale);
  if (st != TARMAC_OK || B == 0) return st;
  if (!aligned(state_out, 4)) return TARMAC_ERR_ALIGN;
  cudaStream_t s = (cudaStream_t)stream;
  if (N == 0) return status(carry_state(state, state_out, (int64_t)B * H * d * d, s));
  if (!out) return TARMAC_ERR_NULL;
  const bool bf16 = dtype == TARMAC_BF16;
  const int es = bf16 ? 2 : 4, G = H / Hk;
  if (!aligned(out, 16) || !aligned(work, 16)) return TARMAC_ERR_ALIGN;
  const HeadStrides sq = stride_of(strides, 0, N, H, d), sk = stride_of(strides, 1, N, Hk, d),
                    sv = stride_of(strides, 2, N, Hk, d);
  const Operand oq = operand(q, sq, B, N, H, 1, d, es), ok = operand(k, sk, B, N, H, G, d, es),
                ov = operand(v, sv, B, N, H, G, d, es);
  p.out = out;
  p.start = state;
  p.last = state_out;
  p.in_scale = 1.f;
  p.out_scale = scale;
  set_operands(p, oq, ok, ov);
  if (decay_step_takes(N)) return status(launch_decay_step(p, bf16, s));
  set_plan(p, decay_tc_sizes(B, N, H, d, bf16) && oq.map && ok.map && ov.map, 1);
  if (decay_uses_part(DecayPlan{p.segs, p.seg_chunks}, p.tc, state_out)) {
    if (!work) return TARMAC_ERR_NULL;
    p.part = static_cast<float*>(work);
  }
  p.planes = state_out ? 3 : 1;
  set_joined(p);
  cudaError_t e = cudaSuccess;
  if (state && state == state_out && copy_bytes(B, N, H, d, p.tc)) {
    char* copy = static_cast<char*>(work) + part_bytes(B, N, H, d, p.tc, 1, true);
    p.start = reinterpret_cast<const float*>(copy);
    e = carry_state(state, reinterpret_cast<float*>(copy), (int64_t)B * H * d * d, s);
  }
  if (e == cudaSuccess) e = launch_decay_states(p, bf16, s);
  if (e == cudaSuccess) e = launch_decay_rows(p, bf16, s);
  return status(e);
}

int64_t tarmac_decay_attention_backward_workspace(int B, int N, int H, int Hk, int d, int dtype,
                                                  int dstate) {
  if (check_sizes(B, N, H, Hk, d, dtype) != TARMAC_OK || B < 1 || N < 1) return 0;
  int64_t bytes = 0;
  for (int tc = 0; tc <= (int)decay_tc_sizes(B, N, H, d, dtype == TARMAC_BF16); ++tc) {
    const int64_t n = backward_work(B, N, H, Hk, d, tc != 0, dstate != 0).bytes;
    if (n > bytes) bytes = n;
  }
  return bytes;
}

int tarmac_decay_attention_backward(const void* q, const void* k, const void* v, const void* dout,
                                    const int64_t* strides, const float* log_decay,
                                    const float* state, const float* dstate_out,
                                    const int32_t* lens, int B, int N, int H, int Hk, int d,
                                    int dtype, float scale, void* dq, void* dk, void* dv,
                                    float* dstate, void* work, void* stream) {
  DecayParams p;
  const int st = fill_decay(p, q, k, v, log_decay, state, lens, B, N, H, Hk, d, dtype, scale);
  if (st != TARMAC_OK) return st;
  // it stands in every term of R here, next to powers of up to l^-15 (2^105) on the
  // tensor memory, and the recurrence divides the state by it
  if (scale < 0x1p-60f || scale > 0x1p20f) return TARMAC_ERR_SHAPE;
  if (B == 0) return TARMAC_OK;
  if (!aligned(dstate, 4) || !aligned(dstate_out, 4)) return TARMAC_ERR_ALIGN;
  cudaStream_t s = (cudaStream_t)stream;
  if (N == 0) return status(carry_state(dstate_out, dstate, (int64_t)B * H * d * d, s));
  if (!dout || !dq || !dk || !dv) return TARMAC_ERR_NULL;
  const bool bf16 = dtype == TARMAC_BF16;
  const int es = bf16 ? 2 : 4, G = H / Hk;
  if (!aligned(dout, es) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16) ||
      !aligned(work, 16))
    return TARMAC_ERR_ALIGN;
  if (!work && tarmac_decay_attention_backward_workspace(B, N, H, Hk, d, dtype, dstate != nullptr))
    return TARMAC_ERR_NULL;
  const HeadStrides sq = stride_of(strides, 0, N, H, d), sk = stride_of(strides, 1, N, Hk, d),
                    sv = stride_of(strides, 2, N, Hk, d), sg = stride_of(strides, 3, N, H, d);
  const Operand oq = operand(q, sq, B, N, H, 1, d, es), ok = operand(k, sk, B, N, H, G, d, es),
                ov = operand(v, sv, B, N, H, G, d, es);
  const Operand og = operand(dout, sg, B, N, H, 1, d, es);
  set_plan(p, decay_tc_sizes(B, N, H, d, bf16) && oq.map && ok.map && ov.map && og.map,
           GRADIENTS);
  const DecayPlan plan = {p.segs, p.seg_chunks};
  const BackwardWork at = backward_work(B, N, H, Hk, d, p.tc, dstate != nullptr);
  char* scratch = static_cast<char*>(work);
  cudaError_t e = cudaSuccess;
  auto run = [&](cudaError_t (*launch)(const DecayParams&, bool, cudaStream_t)) {
    if (e == cudaSuccess) e = launch(p, bf16, s);
  };
  // On the tensor memory the three gradients are one launch; otherwise they
  // follow their states.
  DecayParams jobs[GRADIENTS];
  int n = 0;
  auto rows = [&] {
    if (p.tc)
      jobs[n++] = p;
    else
      run(launch_decay_rows);
  };
  const bool one_walk = decay_one_walk(d, p.tc);
  // dq_i = scale S_i dout_i, S over the rows as in the forward pass
  p.start = state;
  p.part = decay_uses_part(plan, p.tc, false) ? reinterpret_cast<float*>(scratch) : nullptr;
  p.planes = 1;
  p.in_scale = 1.f;
  p.out_scale = scale;
  set_operands(p, oq, ok, ov);
  set_joined(p);
  run(launch_decay_states);
  if (one_walk) {
    set_extra(p, og);
    p.row_out = dq;
  } else {
    set_operands(p, og, ov, ok);
    p.transposed = 1;
    p.out = dq;
  }
  rows();
  // R_i = sum over the rows from i on of scale q dout^T:
  // dv_i = R_i^T k_i, dk_i = R_i v_i
  p.start = dstate_out;
  p.last = dstate;
  p.part = decay_uses_part(plan, p.tc, dstate) ? reinterpret_cast<float*>(scratch + at.back)
                                               : nullptr;
  p.planes = dstate ? 3 : 1;
  p.reverse = 1;
  p.transposed = 0;
  p.in_scale = scale;
  p.out_scale = 1.f;
  set_operands(p, ok, oq, og);
  set_joined(p);
  run(launch_decay_states);
  p.out_f32 = G > 1;
  float* shared_v = reinterpret_cast<float*>(scratch + at.dv);
  float* shared_k = reinterpret_cast<float*>(scratch + at.dk);
  p.out = G > 1 ? shared_v : dv;
  if (one_walk) {
    set_extra(p, ov);
    p.row_out = G > 1 ? shared_k : dk;
    rows();
  } else {
    rows();
    set_operands(p, ov, og, oq);
    p.transposed = 1;
    p.last = nullptr;
    p.out = G > 1 ? shared_k : dk;
    rows();
  }
  if (n > 0 && e == cudaSuccess) e = launch_decay_rows_tc(jobs, n, s);
  if (G > 1 && e == cudaSuccess)
    e = launch_decay_share(shared_v, (at.dk - at.dv) / 4, dv, dk, (int64_t)B * N, Hk, G, d, bf16, s);
  return status(e);
}

int tarmac_decay_attention_plan(int backward, const int64_t* strides, int B, int N, int H, int Hk,
                                int d, int dtype, int state, char* out, int len) {
  if (!out || len < 1) return TARMAC_ERR_NULL;
  out[0] = '\0';
  const int st = check_sizes(B, N, H, Hk, d, dtype);
  if (st != TARMAC_OK) return st;
  const bool bf16 = dtype == TARMAC_BF16;
  const int es = bf16 ? 2 : 4, G = H / Hk;
  // only sizes, strides and alignment count: stand-in pointers on the grid
  const void* a = reinterpret_cast<const void*>((uintptr_t)1 << 20);
  char buf[128];
  if (!backward && decay_step_takes(N)) {
    snprintf(buf, sizeof buf, "{\"kernel\": \"decay_step\", \"segments\": 1}");
  } else {
    bool tc = decay_tc_sizes(B, N, H, d, bf16);
    for (int i = 0; i < 3 + (backward != 0); ++i) {
      const int share = i == 1 || i == 2 ? G : 1;
      tc = tc && operand(a, stride_of(strides, i, N, H / share, d), B, N, H, share, d, es).map;
    }
    const DecayPlan g = decay_plan(B, N, H, d, tc, backward ? GRADIENTS : 1);
    snprintf(buf, sizeof buf, "{\"kernel\": \"%s\", \"segments\": %d, \"states\": %s}",
             tc ? "decay_tc" : "decay_scan", g.segs,
             decay_uses_part(g, tc, state != 0) ? "true" : "false");
  }
  const int n = (int)strlen(buf);
  if (n + 1 > len) return TARMAC_ERR_SHAPE;
  memcpy(out, buf, (size_t)n + 1);
  return TARMAC_OK;
}

int tarmac_residual_norm(const void* x, const void* y, const void* gate, const int64_t* strides,
                         const float* w_post, const float* w_pre, const float* scale, int B,
                         int N, int D, int dtype, float eps, void* h, void* z, void* stream) {
  NormParams p;
  const int st = fill_norm(p, x, y, gate, strides, w_post, w_pre, scale, B, N, D, dtype, eps);
  if (st != TARMAC_OK || (int64_t)B * N == 0) return st;
  if (!h || !z) return TARMAC_ERR_NULL;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  if (!aligned(h, es) || !aligned(z, es)) return TARMAC_ERR_ALIGN;
  p.h = h;
  p.z = z;
  return status(launch_residual_norm(p, dtype == TARMAC_BF16, (cudaStream_t)stream));
}

int64_t tarmac_residual_norm_workspace(int B, int N, int D) {
  if (B < 1 || N < 1 || D < 1 || D > NORM_MAX_D) return 0;
  return residual_norm_bwd_work((int64_t)B * N, D) * 4;
}

int tarmac_residual_norm_backward(const void* x, const void* y, const void* gate, const void* dh,
                                  const void* dz, const int64_t* strides, const float* w_post,
                                  const float* w_pre, const float* scale, int B, int N, int D,
                                  int dtype, float eps, void* dx, void* dy, void* dgate,
                                  float* dw_post, float* dw_pre, float* dscale, void* work,
                                  void* stream) {
  NormParams p;
  const int st = fill_norm(p, x, y, gate, strides, w_post, w_pre, scale, B, N, D, dtype, eps);
  if (st != TARMAC_OK) return st;
  if (!aligned(dw_post, 4) || !aligned(dw_pre, 4) || !aligned(dscale, 4)) return TARMAC_ERR_ALIGN;
  cudaStream_t s = (cudaStream_t)stream;
  if ((int64_t)B * N == 0) {  // no rows: the weights' gradients are zero
    cudaError_t e = cudaSuccess;
    for (float* w : {dw_post, dw_pre, dscale})
      if (w && e == cudaSuccess) e = cudaMemsetAsync(w, 0, (size_t)D * 4, s);
    return status(e);
  }
  if (!dx || !dy || (gate && !dgate) || !work) return TARMAC_ERR_NULL;
  const int es = dtype == TARMAC_BF16 ? 2 : 4;
  for (const void* ptr : {dh, dz, (const void*)dx, (const void*)dy, (const void*)dgate})
    if (!aligned(ptr, es)) return TARMAC_ERR_ALIGN;
  if (!aligned(work, 16)) return TARMAC_ERR_ALIGN;
  p.dh = dh;
  p.dz = dz;
  p.sdh = rows_of(strides, 3, N, D);
  p.sdz = rows_of(strides, 4, N, D);
  p.dx = dx;
  p.dy = dy;
  p.dgate = gate ? dgate : nullptr;
  p.dw_post = dw_post;
  p.dw_pre = dw_pre;
  p.dscale = dscale;
  p.work = static_cast<float*>(work);
  return status(launch_residual_norm_bwd(p, dtype == TARMAC_BF16, s));
}

}  // extern "C"
