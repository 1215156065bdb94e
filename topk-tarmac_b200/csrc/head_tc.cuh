// head_tc.cuh — helpers of the tensor-memory attention kernels
// (head_attn_tc.cu, head_bwd_tc.cu): TMA tiles of 64 columns in the 128-byte
// swizzle, their matrix descriptors, TMEM transfers and row masks.
//
// Rows of d columns run as NKS = 2, 4, 6 or 8 steps of 16 columns, zero beyond d.
// A tile is R rows of DP columns (64 or 128), held as DP / 64 halves of R rows
// of 128 bytes; TMA writes it in boxes of 64 rows x 64 columns (8 KB), zero
// beyond the tensor's rows and columns. The same bytes serve as an operand
// contracting over the columns (K-major: 16 columns are 32 bytes on) and as
// one contracting over the rows (MN-major: 16 rows are 2048 bytes on, the
// second 64 columns one half on).
#pragma once

#include <cuda.h>  // CUtensorMap; no driver library link

#include "heads.cuh"
#include "ws_common.cuh"

namespace tarmac {
namespace ht {

constexpr int width(int nks) { return nks <= 4 ? 64 : 128; }  // DP

// Test builds define TARMAC_GIVE_UP_AT, a number of a block's item, and
// TARMAC_GIVE_UP_ROLE: that role gives up there as it does when one of its
// waits runs out.
enum Role { ROLE_LOADER = 0, ROLE_WEIGHTS = 1 };
__device__ constexpr bool gives_up(Role role, int k) {
#ifdef TARMAC_GIVE_UP_AT
  return role == TARMAC_GIVE_UP_ROLE && k == TARMAC_GIVE_UP_AT;
#else
  return false;
#endif
}

constexpr uint32_t BOX_ROWS = 64;
constexpr uint32_t BOX_BYTES = 64 * 128;

// matrix descriptor in the 128-byte swizzle; sbo: 8 rows = 1024 bytes
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version for sm_100
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}

// descriptor offset (16-byte units) of K step ks (16 columns) of a K-major
// tile of `rows` rows
__device__ __forceinline__ uint64_t kstep(int ks, uint32_t rows) {
  return (uint64_t)(((uint32_t)(ks >> 2) * rows * 128u + (uint32_t)(ks & 3) * 32u) >> 4);
}

__device__ __forceinline__ void expect_tx(uint64_t* mbar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_addr(mbar)),
               "r"(bytes)
               : "memory");
}

// one box (64 rows x 64 columns) of a [B, N, h, d] tensor into shared memory
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint64_t* mbar,
                                        int col, int head, int row, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(tc::smem_addr(mbar)), "r"(col), "r"(head), "r"(row), "r"(b)
      : "memory");
}

// a tile of R rows
template <int DP, int R>
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, uint64_t* mbar,
                                         int head, int row, int b) {
#pragma unroll
  for (int h = 0; h < DP / 64; ++h)
#pragma unroll
    for (int r = 0; r < R / 64; ++r)
      tma_box(dst + (uint32_t)(h * R * 128 + r * (int)BOX_BYTES), map, mbar, h * 64, head,
              row + r * 64, b);
}

// bulk copy of `bytes` (a multiple of 16, both ends 16-byte aligned)
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes,
                                          uint64_t* mbar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, "
      "[%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(tc::smem_addr(mbar))
      : "memory");
}

// Bounded wait on the barrier at shared address `a`: one poll in line (most
// phases have completed by then), the rest out of line.
static __device__ __noinline__ bool poll_wait(uint32_t a, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t it = 0; it < WS_WAIT_LIMIT; ++it) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
    if ((it & 63) == 63 && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ bool wait_at(uint32_t a, uint32_t parity, volatile int* abort_flag) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(a), "r"(parity)
      : "memory");
  return done ? true : poll_wait(a, parity, abort_flag);
}
__device__ __forceinline__ void commit_at(uint32_t a) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(a)
      : "memory");
}
// Wait, bounded, until the last `n` of `count` copies into a ring of n slots
// have landed: shared memory must not be written after its block has ended.
// Copy c completes phase c / n of its slot.
__device__ __forceinline__ void drain_copies(uint64_t* full, uint32_t n, uint32_t count) {
  for (uint32_t c = count > n ? count - n : 0; c < count; ++c)
    tc::mbar_wait(&full[c % n], (c / n) & 1, WS_WAIT_LIMIT);
}
// The issuing warps' lanes wait each for itself. Before a loop's condition
// they agree on whether all go on: a lane that left alone would not meet the
// others' warp barriers.
__device__ __forceinline__ bool agree(bool ok) { return __all_sync(0xffffffffu, ok); }
// The same for the products that this warp's `leader` has issued, after it
// gave up: tensor memory is freed and the operands' tiles end with the block.
__device__ __forceinline__ void drain_products(uint64_t* drain, bool leader) {
  if (leader) commit_at(tc::smem_addr(drain));
  __syncwarp();
  tc::mbar_wait(drain, 0, WS_WAIT_LIMIT);
}
// One lane of a converged warp. The issuing warps run their loops with all
// lanes, so that addresses and descriptors stay in uniform registers, and
// only the products themselves are under this predicate.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(p));
  return p != 0;
}
// position in a ring of N slots: slot and phase parity
template <int N>
struct RingPos {
  uint32_t s = 0, ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1;
    }
  }
};

// Bounded wait by a whole warp: all lanes take the same result, so the warp
// stays together for its TMEM transfers.
__device__ __forceinline__ bool warp_wait(uint64_t* mbar, uint32_t parity,
                                          volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait_at(tc::smem_addr(mbar), parity, abort_flag));
}

__device__ __forceinline__ void st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 16 consecutive 32-bit columns of this thread's TMEM lane (warp-collective);
// load and wait in one statement, so no use can move ahead of the wait
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 32 consecutive 32-bit columns of this thread's TMEM lane (warp-collective);
// load and wait in one statement, so no use can move ahead of the wait
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// 64 consecutive 32-bit columns of this thread's TMEM lane (warp-collective);
// load and wait in one statement, so no use can move ahead of the wait
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
               : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]; A: lane m, column k / 2, lower k in the low half
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                       uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate));
}

// C[tmem_d] = A . B^T over NKS steps of 16 columns (A: 128 rows, B: RB rows,
// both K-major). Straight-line: no product is issued under a condition.
template <int NKS, int RB>
__device__ __forceinline__ void issue_scores(uint32_t tmem_d, uint64_t da, uint64_t db,
                                             uint32_t idesc) {
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks)
    tc::mma_bf16(tmem_d, da + kstep(ks, 128), db + kstep(ks, RB), idesc, ks > 0);
}
// C[tmem_d] (+)= P[tmem_a] . B, contracting over the RB rows of B (MN-major).
// P's columns come from groups of warps that own GC columns each: as bf16 they
// take GC / 2 TMEM columns, at every GC-th column.
template <int RB, int GC>
__device__ __forceinline__ void issue_aggregate(uint32_t tmem_d, uint32_t tmem_a, uint64_t db,
                                                uint32_t idesc, bool add) {
#pragma unroll
  for (int ks = 0; ks < RB / 16; ++ks)
    mma_ts(tmem_d, tmem_a + (ks * 16 / GC) * GC + (ks * 16 % GC) / 2,
           db + (uint64_t)((ks * 2048) >> 4), idesc, add || ks > 0);
}

// packed fp32 pairs (one issue slot for two IEEE operations)
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

// First query position of an episode. Positions beyond +-2^30 act like those
// bounds (lengths stay below 2^29), which keeps position arithmetic in 32 bits.
__device__ __forceinline__ int first_pos(const HeadAttnParams& p, int b) {
  const int s = p.q_start ? __ldg(p.q_start + b) : p.Nk - p.Nq;
  return max(-(1 << 30), min(1 << 30, s));
}
__device__ __forceinline__ int key_count(const HeadAttnParams& p, int b) {
  const int n = p.key_len ? __ldg(p.key_len + b) : p.Nk;
  return max(0, min(n, p.Nk));
}
// first key a row at `pos` does not see, from its length and the past rule
__device__ __forceinline__ int key_limit(const HeadAttnParams& p, int pos, int len) {
  return p.peers == PEERS_PAST ? max(0, min(len, pos + 1)) : len;
}

// Keys of the 32-key word at key j0 that a row may see: below jlim, not self,
// and set in `bits`.
__device__ __forceinline__ uint32_t key_word(int j0, int jlim, int self, uint32_t bits) {
  const int n = jlim - j0;
  uint32_t w = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
  const int s = self - j0;
  if (s >= 0 && s < 32) w &= ~(1u << s);
  return w & bits;
}

}  // namespace ht

// Tensor map of a [B, N, h, d] bf16 tensor with 64 x 64 boxes; false where
// TMA cannot describe it (head_attn_tc.cu). head_map_ok: do the strides allow it?
bool head_map_ok(const HeadStrides& s, int B, int N, int h);
bool head_tensor_map(CUtensorMap* map, const void* ptr, const HeadStrides& s, int B, int N, int h,
                     int d);
// The same for bf16 or fp32 with boxes of 128 bytes by `box_rows` rows.
bool head_box_map(CUtensorMap* map, const void* ptr, const HeadStrides& s, int B, int N, int h,
                  int d, bool f32, int box_rows);

}  // namespace tarmac
