// decay.cuh — parameters of attention with a decay for each head
// (decay_tc.cu, decay_scan.cu, decay_step.cu) and how a call is divided.
//
// Every direction is one form over rows, with l the decay of a head:
//   out_i = sum_{j <= i} l^(i-j) (a_i . b_j) c_j + l^(i+1) a_i . S,
// S [columns of b, columns of c] the state before the first row, and
//   S' = l^n S + sum_j l^(n-1-j) b_j c_j^T
// the state after n rows. With q, k, v it is the forward pass; with dout, v, k
// the gradient of q (the state transposed); over the rows backwards, with
// k, q, dout and v, dout, q the gradients of v and k.
#pragma once

#include "heads.cuh"

namespace tarmac {

struct DecayParams {
  const void *a, *b, *c;
  const void* e;             // multiplies S from the other side (decay_one_walk)
  void* out;                 // [B, N, H, d] contiguous: S^T a
  void* row_out;             // the same: S e, or NULL
  HeadStrides sa, sb, sc, se;
  int ga, gb, gc, ge;        // heads that share one head of a, b, c, e
  int out_f32;               // out is fp32 (backwards only), else the rows' type
  const float* log_decay;    // [H]
  const int32_t* lens;       // [B] or NULL
  const float* start;        // [B, H, d, d], the state before, or NULL (zero)
  float* last;               // [B, H, d, d], the state after, or NULL
  float* part;               // [segs, B, H, d, d], or NULL (decay_uses_part)
  int B, N, H, d;
  int segs, seg_chunks;      // parts of the row axis and their chunks
  int joined;                // a launch of its own joins the segments' states
  int reverse;               // rows run from the last to the first
  int transposed;            // state tensors are [columns of c, columns of b]
  float in_scale;            // factor of every b_j c_j term
  float out_scale;           // factor of out
  int planes;                // tensor memory: bf16 parts of the weighted rows that enter S
  int tc;                    // runs on the tensor memory (decay_tc.cu)
  int vec;                   // 16-byte rows in a, b, c, e
};

// Powers of a decay: exp(rate e). A decay of zero (rate -inf) keeps l^0 = 1.
__device__ __forceinline__ float decay_rate(const float* log_decay, int h) {
  const float r = __ldg(log_decay + h);
  return r < -1e4f ? -1e4f : r;  // NaN stays
}
// The decay of n rows, l^n = exp(rate n), that is applied to a state again and
// again: by one fp32 number every application would be off by the same rounding.
struct DecayPower {
  float base, add;  // l^n = base + add
  __device__ __forceinline__ DecayPower(float rate, float n) {
    const float m = expm1f(rate * n), e = expf(rate * n);
    // slow: 1 + m, m good to 24 bits of its own. Fast, or NaN: what is rounded is
    // gone after a few applications.
    const bool slow = m > -0.5f;
    base = slow ? 1.f : 0.f;
    add = slow ? m : e;
  }
  // l^n s, rounded once
  __device__ __forceinline__ float times(float s) const { return fmaf(add, s, base * s); }
};
// The same as one factor at a time, where a product takes no second number: next()
// gives an fp32 number near l^n whose roundings are made up for by those after it,
// so that no run of them is off by more than 2^-24. `of`: what l^n itself is off
// from `hi` counts that many times.
struct DecayFactor {
  float hi, lo, left;
  __device__ __forceinline__ static DecayFactor make(float rate, float n, float of = 1.f) {
    const DecayPower l(rate, n);
    const float hi = l.base + l.add;
    // base is 1 and add in (-0.5, 0], or base is 0: the difference is exact
    return DecayFactor{hi, of * (l.add - (hi - l.base)), 0.f};
  }
  __device__ __forceinline__ float next() {
    const float want = left + lo, x = hi + want;
    left = want - (x - hi);
    return x;
  }
};
__device__ __forceinline__ int decay_len(const DecayParams& p, int b) {
  return p.lens ? max(0, min(__ldg(p.lens + b), p.N)) : p.N;
}

constexpr int DECAY_CHUNK = 16;      // rows that segments are counted in
constexpr int DECAY_TC_CHUNK = 128;  // and a chunk's on the tensor memory

struct DecayPlan {
  int segs, seg_chunks;
};
// jobs: sums over the same rows that a launch on the tensor memory takes
DecayPlan decay_plan(int B, int N, int H, int d, bool tc, int jobs);
DecayPlan decay_plan_tc(int B, int N, int H, int d, int jobs);
// may a call of these sizes run on the tensor memory?
bool decay_tc_sizes(int B, int N, int H, int d, bool bf16);
// Do the gradients take one walk each way (dq as row_out; dv and dk as out and
// row_out of one walk)? Else each is an out of its own, dq and dk with the state
// transposed.
bool decay_one_walk(int d, bool tc);
// bytes of p.part, where the call uses it
int64_t decay_part_bytes(const DecayPlan& g, int B, int H, int d, bool tc);
// Does the call keep states in p.part? (On the tensor memory the state after
// the last row comes from the segments' states, else from the rows' kernel.)
inline bool decay_uses_part(const DecayPlan& g, bool tc, bool last) {
  return g.segs > 1 || (tc && last);
}

// States of the segments into p.part: first what each adds, then, in place,
// the state before each (and p.last, on the tensor memory). Launches nothing
// where the call does not use p.part.
cudaError_t launch_decay_states(const DecayParams& p, bool bf16, cudaStream_t s);
cudaError_t launch_decay_rows(const DecayParams& p, bool bf16, cudaStream_t s);
cudaError_t launch_decay_states_tc(const DecayParams& p, cudaStream_t s);
cudaError_t launch_decay_rows_tc(const DecayParams* p, int jobs, cudaStream_t s);
// few rows, one after the other (forward only)
bool decay_step_takes(int N);
cudaError_t launch_decay_step(const DecayParams& p, bool bf16, cudaStream_t s);
// out0, out1 [rows, Hk, d] = sums over the G heads of a key head of x and of what
// stands x_step elements on, fp32 to the rows' type
cudaError_t launch_decay_share(const float* x, int64_t x_step, void* out0, void* out1,
                               int64_t rows, int Hk, int G, int d, bool bf16, cudaStream_t s);

}  // namespace tarmac
