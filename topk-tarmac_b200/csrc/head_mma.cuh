// head_mma.cuh — warp-level products of the multi-head attention kernels
// (head_attn.cu), for bf16 and fp32 rows in shared memory.
//
// A warp owns 16 rows. Two products make up every kernel:
//   scores:    C[16 x 8 NT] = A[16 x DP] . B[8 NT x DP]^T, both by rows;
//   aggregate: O[16 x DP] += P[16 x 8 NT] . B[8 NT x DP], P in C's registers.
// bf16 uses m16n8k16. fp32 uses m16n8k8 tf32 on both halves of every
// operand, x = hi + lo with hi = tf32(x) and lo = tf32(x - hi): the three
// products hi.hi + hi.lo + lo.hi leave out lo.lo and lo's own rounding, each
// below 2^-22 of |a b|, so a product is as good as an fp32 FMA's to within a
// few units of 2^-23. The tensor core chops its fp32 sum once per
// instruction; a long chain of one accumulator would drift, so aggregates
// start from zero in each tile and are added to the running sum in fp32.
// On B200 this path measured 275 TFLOP/s tf32 (92 for the three products)
// against 72 nominal for FFMA, and 550 TFLOP/s bf16.
#pragma once

#include "heads.cuh"

namespace tarmac {
namespace hm {

// shared-memory row stride in elements: 16 bytes of padding put the eight
// rows that a fragment touches into different banks (DP a multiple of 16)
template <typename T, int DP>
constexpr int row_stride() {
  return DP + 16 / (int)sizeof(T);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(tc_smem_base(p))
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(tc_smem_base(p))
               : "memory");
}
__device__ __forceinline__ void mma_b16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = to_tf32(x);
  lo = to_tf32(x - __uint_as_float(hi));
}
__device__ __forceinline__ uint32_t pack_b16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Fragment layout of C (and P): c[nt][0..1] are row lane/4, columns
// 8 nt + 2 (lane % 4) + {0, 1}; c[nt][2..3] the same columns of row + 8.

// C = A . B^T. sA: the warp's first row; sB: the tile's first row.
template <int DP, int NT>
__device__ __forceinline__ void scores(float (&c)[NT][4], const __nv_bfloat16* sA,
                                       const __nv_bfloat16* sB, int lane) {
  constexpr int RS = row_stride<__nv_bfloat16, DP>();
  static_assert(NT % 2 == 0, "two 8-column tiles per load");
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) c[n][u] = 0.f;
  const __nv_bfloat16* pa = sA + ((lane & 7) + ((lane >> 3) & 1) * 8) * RS + (lane >> 4) * 8;
  const __nv_bfloat16* pb = sB + ((lane & 7) + (lane >> 4) * 8) * RS + ((lane >> 3) & 1) * 8;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    uint32_t a[4];
    ldsm4(a, pa + ks * 16);
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t b[4];
      ldsm4(b, pb + n * 8 * RS + ks * 16);
      mma_b16(c[n], a, b[0], b[1]);
      mma_b16(c[n + 1], a, b[2], b[3]);
    }
  }
}

template <int DP, int NT>
__device__ __forceinline__ void scores(float (&c)[NT][4], const float* sA, const float* sB,
                                       int lane) {
  constexpr int RS = row_stride<float, DP>();
  float small[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) c[n][u] = small[n][u] = 0.f;
  const float* pa = sA + (lane >> 2) * RS + (lane & 3);
  const float* pb = sB + (lane >> 2) * RS + (lane & 3);
#pragma unroll
  for (int ks = 0; ks < DP / 8; ++ks) {
    uint32_t ah[4], al[4];
    split_tf32(pa[ks * 8], ah[0], al[0]);
    split_tf32(pa[ks * 8 + 8 * RS], ah[1], al[1]);
    split_tf32(pa[ks * 8 + 4], ah[2], al[2]);
    split_tf32(pa[ks * 8 + 8 * RS + 4], ah[3], al[3]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t bh[2], bl[2];
      split_tf32(pb[n * 8 * RS + ks * 8], bh[0], bl[0]);
      split_tf32(pb[n * 8 * RS + ks * 8 + 4], bh[1], bl[1]);
      mma_tf32(small[n], al, bh[0], bh[1]);
      mma_tf32(c[n], ah, bh[0], bh[1]);
      mma_tf32(small[n], ah, bl[0], bl[1]);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) c[n][u] += small[n][u];
}

// O += P . B; sB: the tile's first row. bf16 rounds P to bf16 (the type of
// its products; the row sum that divides it stays fp32).
template <int DP, int NT>
__device__ __forceinline__ void aggregate(float (&o)[DP / 8][4], const float (&p)[NT][4],
                                          const __nv_bfloat16* sB, int lane) {
  constexpr int RS = row_stride<__nv_bfloat16, DP>();
  const __nv_bfloat16* pb = sB + ((lane & 7) + ((lane >> 3) & 1) * 8) * RS + (lane >> 4) * 8;
#pragma unroll
  for (int kk = 0; kk < NT / 2; ++kk) {
    const uint32_t a[4] = {pack_b16(p[2 * kk][0], p[2 * kk][1]),
                           pack_b16(p[2 * kk][2], p[2 * kk][3]),
                           pack_b16(p[2 * kk + 1][0], p[2 * kk + 1][1]),
                           pack_b16(p[2 * kk + 1][2], p[2 * kk + 1][3])};
#pragma unroll
    for (int n = 0; n < DP / 8; n += 2) {
      uint32_t b[4];
      ldsm4t(b, pb + kk * 16 * RS + n * 8);
      mma_b16(o[n], a, b[0], b[1]);
      mma_b16(o[n + 1], a, b[2], b[3]);
    }
  }
}

// fp32: P's registers serve as the A operand when the contraction index is
// renumbered inside each 8: position t and t + 4 stand for columns 2t, 2t + 1.
template <int DP, int NT>
__device__ __forceinline__ void aggregate(float (&o)[DP / 8][4], const float (&p)[NT][4],
                                          const float* sB, int lane) {
  constexpr int RS = row_stride<float, DP>();
  uint32_t ah[NT][4], al[NT][4];
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    split_tf32(p[k][0], ah[k][0], al[k][0]);
    split_tf32(p[k][2], ah[k][1], al[k][1]);
    split_tf32(p[k][1], ah[k][2], al[k][2]);
    split_tf32(p[k][3], ah[k][3], al[k][3]);
  }
  const float* pb = sB + 2 * (lane & 3) * RS + (lane >> 2);
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    float c[4] = {0.f, 0.f, 0.f, 0.f}, x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      uint32_t bh[2], bl[2];
      split_tf32(pb[k * 8 * RS + n * 8], bh[0], bl[0]);
      split_tf32(pb[(k * 8 + 1) * RS + n * 8], bh[1], bl[1]);
      mma_tf32(c, ah[k], bh[0], bh[1]);
      mma_tf32(x, ah[k], bl[0], bl[1]);
      mma_tf32(y, al[k], bh[0], bh[1]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) o[n][u] += c[u] + (x[u] + y[u]);
  }
}

// ---- fp32 rows of up to 32 columns, split once when they are staged --------
// Split inside the products, every element is split by every warp that reads
// it, and that arithmetic bounds rows this narrow. Here a shared tile holds
// {hi, lo} pairs: element (r, k) at word r RS + ((2k) ^ (16 if r & 4)), RS =
// 2 DP + 8. The four rows of a half-warp's 64-bit loads then fall into
// different banks both for rows 0, 4, 1, 5 (score columns) and 0..3, 4..7.
// Score column c of an 8-key tile is key (c >> 1) + 4 (c & 1), so that a
// thread's two weights are the two contraction indexes of its A operand.
template <int DP>
constexpr int split_stride() {
  return 2 * DP + 8;
}
template <int DP>
__device__ __forceinline__ int split_word(int r, int k) {
  return r * split_stride<DP>() + ((2 * k) ^ ((r & 4) << 2));
}
template <int DP>
__device__ __forceinline__ void store_split(float* tile, int r, int c, float4 v) {
  uint32_t h[4], l[4];
  split_tf32(v.x, h[0], l[0]);
  split_tf32(v.y, h[1], l[1]);
  split_tf32(v.z, h[2], l[2]);
  split_tf32(v.w, h[3], l[3]);
  uint4* t = reinterpret_cast<uint4*>(tile + split_word<DP>(r, c));
  t[0] = make_uint4(h[0], l[0], h[1], l[1]);
  t[1] = make_uint4(h[2], l[2], h[3], l[3]);
}
__device__ __forceinline__ void lds_pair(uint32_t& hi, uint32_t& lo, const float* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  hi = v.x;
  lo = v.y;
}

template <int DP, int NT>
__device__ __forceinline__ void scores_split(float (&c)[NT][4], const float* sA, const float* sB,
                                             int lane) {
  constexpr int RS = split_stride<DP>();
  const int r = lane >> 2, t = lane & 3;
  const int flip_a = (r & 4) << 2;  // rows r and r + 8
  const int rb = (r >> 1) + 4 * (r & 1), flip_b = (r & 1) << 4;
  float small[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) c[n][u] = small[n][u] = 0.f;
#pragma unroll
  for (int ks = 0; ks < DP / 8; ++ks) {
    uint32_t ah[4], al[4];
    const int k0 = 2 * (ks * 8 + t), k1 = k0 + 8;
    lds_pair(ah[0], al[0], sA + r * RS + (k0 ^ flip_a));
    lds_pair(ah[1], al[1], sA + (r + 8) * RS + (k0 ^ flip_a));
    lds_pair(ah[2], al[2], sA + r * RS + (k1 ^ flip_a));
    lds_pair(ah[3], al[3], sA + (r + 8) * RS + (k1 ^ flip_a));
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t bh[2], bl[2];
      lds_pair(bh[0], bl[0], sB + (n * 8 + rb) * RS + (k0 ^ flip_b));
      lds_pair(bh[1], bl[1], sB + (n * 8 + rb) * RS + (k1 ^ flip_b));
      mma_tf32(small[n], al, bh[0], bh[1]);
      mma_tf32(c[n], ah, bh[0], bh[1]);
      mma_tf32(small[n], ah, bl[0], bl[1]);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) c[n][u] += small[n][u];
}

template <int DP, int NT>
__device__ __forceinline__ void aggregate_split(float (&o)[DP / 8][4], const float (&p)[NT][4],
                                                const float* sB, int lane) {
  constexpr int RS = split_stride<DP>();
  const int t = lane & 3, j = lane >> 2;
  float c[DP / 8][4], x[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) c[n][u] = x[n][u] = 0.f;
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    uint32_t ah[4], al[4];
    split_tf32(p[k][0], ah[0], al[0]);
    split_tf32(p[k][2], ah[1], al[1]);
    split_tf32(p[k][1], ah[2], al[2]);
    split_tf32(p[k][3], ah[3], al[3]);
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      uint32_t bh[2], bl[2];
      const int w = 2 * (n * 8 + j);
      lds_pair(bh[0], bl[0], sB + (k * 8 + t) * RS + w);
      lds_pair(bh[1], bl[1], sB + (k * 8 + t + 4) * RS + (w ^ 16));
      mma_tf32(x[n], al, bh[0], bh[1]);
      mma_tf32(c[n], ah, bh[0], bh[1]);
      mma_tf32(x[n], ah, bl[0], bl[1]);
    }
  }
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) o[n][u] += c[n][u] + x[n][u];
}

// sum / maximum over the four lanes that share a row
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

}  // namespace hm
}  // namespace tarmac
