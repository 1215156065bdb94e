// head_attn.cu — masked attention with heads, forward and backward, for fp32
// and bf16 rows of up to 128 columns: the kernels that take every call (the
// tensor-memory kernels in head_attn_tc.cu take large bf16 calls from them).
//
// Row i of episode b stands at position p = q_start[b] + i and sees key j when
// j < key_len[b], the peers rule holds (all; others: j != p; past: j <= p) and
// its visibility bit is set. With s = scale q.k over the visible keys,
//   out = softmax(s) v,  lse = log sum exp s   (no visible key: 0 and -inf),
//   D = dout . out,  dS = P (dout v^T - D),
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout.
// P is recomputed from lse, never stored. The G query heads of one key/value
// head are packed into its rows (row r is query r / G, head r % G), so shared
// keys are read once for all of them and the gradients of shared heads add up
// inside one block, in a fixed order and without atomics.
//
// Forward: one pass over the keys with the running maximum and sum of the
// softmax (base 2). Backward: one kernel per row tile for dq and one per key
// tile for dk and dv; P and dS are formed twice, which costs two of seven
// products and needs no order between blocks.
// With few rows the key axis is split over blocks and a second kernel joins
// the parts.
#include <type_traits>

#include "head_mma.cuh"

namespace tarmac {

constexpr int HA_THREADS = 128;
constexpr int HA_WARPS = 4;
constexpr int HA_PART = 256;  // keys of a part of the key axis, at least
constexpr float HA_LOG2E = 1.4426950408889634f;
constexpr float HA_LN2 = 0.6931471805599453f;

// rows of a streamed tile
template <typename T, int DP>
constexpr int ha_tile() {
  return sizeof(T) == 4 ? 32 : (DP > 64 ? 32 : 64);
}

// Copy rows [0, n) into padded shared rows, 16 bytes at a time; rows at or
// beyond `limit` and columns at or beyond d become zero, so what the tensors
// hold there is never read. row_ptr(r) gives row r's first element.
template <typename T, int DP, typename F>
__device__ __forceinline__ void load_tile(T* dst, int n, int limit, int d, int vec, F row_ptr) {
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int CH = DP / E;  // 16-byte pieces per row
  constexpr int RS = hm::row_stride<T, DP>();
  for (int e = threadIdx.x; e < n * CH; e += HA_THREADS) {
    const int r = e / CH, c = (e - r * CH) * E;
    T* s = dst + r * RS + c;
    if (r >= limit || c >= d) {
      *reinterpret_cast<uint4*>(s) = make_uint4(0, 0, 0, 0);
    } else if (vec) {
      cp_async16(s, row_ptr(r) + c);
    } else {
      const T* g = row_ptr(r) + c;
#pragma unroll
      for (int u = 0; u < E; ++u) s[u] = c + u < d ? g[u] : from_f32<T>(0.f);
    }
  }
}

// The same for rows a constant stride apart (neighbouring keys). Where a row's
// pieces divide the block evenly, a thread keeps its column and walks down the
// rows, which leaves an add and a compare per 16 bytes: a tile's copies are a
// third of the instructions of a call on few rows otherwise.
template <typename T, int DP>
__device__ __forceinline__ void load_keys_tile(T* dst, int n, int limit, int d, int vec,
                                               const T* first, int64_t stride) {
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int CH = DP / E;
  constexpr int RS = hm::row_stride<T, DP>();
  if constexpr (HA_THREADS % CH == 0) {
    if (vec) {
      constexpr int STEP = HA_THREADS / CH;
      const int c = (threadIdx.x % CH) * E;
      int r = threadIdx.x / CH;
      uint32_t s = tc_smem_base(dst + r * RS + c);
      const T* g = first + r * stride + c;
      const int lim = c < d ? limit : 0;
#pragma unroll
      for (int i = 0; i < 64 / STEP; ++i, r += STEP, s += STEP * RS * sizeof(T), g += STEP * stride) {
        if (r >= n) break;
        // no bytes are read where the row does not exist
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s),
                     "l"(r < lim ? g : first), "r"(r < lim ? 16 : 0)
                     : "memory");
      }
      return;
    }
  }
  load_tile<T, DP>(dst, n, limit, d, vec, [&](int r) { return first + r * stride; });
}

// Narrow fp32 rows are staged as split pairs (head_mma.cuh), up to 32 columns
// forward and 16 backward. 64 x 512 rows of 4 heads, staged so or split when
// read: forward d = 16 127 and 139 us, 32 215 and 227, 64 461 and 423; dk, dv
// d = 16 255 and 267, 32 501 and 475.
template <typename T, int DP>
constexpr bool ha_split() {
  return sizeof(T) == 4 && DP <= 32;
}

// R rows of DP fp32 columns on their way from global memory to a split tile:
// held in registers while the tile before them is used. Rows at or beyond
// `limit` and columns at or beyond d are zero.
template <int DP, int R>
struct SplitRows {
  static constexpr int C4 = DP / 4, U = R * C4 / HA_THREADS;
  static_assert(R * C4 % HA_THREADS == 0, "whole pieces per thread");
  float4 x[U];
  template <typename F>
  __device__ __forceinline__ void load(int limit, int d, int vec, F row_ptr) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * HA_THREADS, r = e / C4, c = (e % C4) * 4;
      x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r >= limit || c >= d) continue;
      const float* g = row_ptr(r) + c;
      if (vec) {
        x[u] = __ldg(reinterpret_cast<const float4*>(g));
      } else {
        x[u].x = g[0];
        if (c + 1 < d) x[u].y = g[1];
        if (c + 2 < d) x[u].z = g[2];
        if (c + 3 < d) x[u].w = g[3];
      }
    }
  }
  __device__ __forceinline__ void store(float* tile) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * HA_THREADS;
      hm::store_split<DP>(tile, e / C4, (e % C4) * 4, x[u]);
    }
  }
};

// Products on tiles of either kind.
template <bool SPLIT, typename T, int DP, int NT>
__device__ __forceinline__ void ha_scores(float (&c)[NT][4], const T* sA, const T* sB, int lane) {
  if constexpr (SPLIT)
    hm::scores_split<DP, NT>(c, sA, sB, lane);
  else
    hm::scores<DP, NT>(c, sA, sB, lane);
}
template <bool SPLIT, typename T, int DP, int NT>
__device__ __forceinline__ void ha_aggregate(float (&o)[DP / 8][4], const float (&p)[NT][4],
                                             const T* sB, int lane) {
  if constexpr (SPLIT)
    hm::aggregate_split<DP, NT>(o, p, sB, lane);
  else
    hm::aggregate<DP, NT>(o, p, sB, lane);
}
// column of score e (0 or 1) of a thread inside an 8-column tile
template <bool SPLIT>
__device__ __forceinline__ int ha_col(int lane, int e) {
  return SPLIT ? (lane & 3) + 4 * e : 2 * (lane & 3) + e;
}

// visible: does the row see key j? jlim: first key beyond key_len and, for
// past, beyond the row's position; self: the key left out, or -1.
__device__ __forceinline__ bool sees(int j, int jlim, int self, uint32_t word) {
  return j < jlim && j != self && ((word >> (j & 31)) & 1u);
}

template <typename T>
__device__ __forceinline__ void store2(T* p, float a, float b, bool pair, bool second) {
  if constexpr (sizeof(T) == 2) {
    if (pair) {
      *reinterpret_cast<uint32_t*>(p) = hm::pack_b16(a, b);
      return;
    }
  } else {
    if (pair) {
      *reinterpret_cast<float2*>(p) = make_float2(a, b);
      return;
    }
  }
  p[0] = from_f32<T>(a);
  if (second) p[1] = from_f32<T>(b);
}

// Write 16 rows of accumulators as rows of a contiguous tensor: dst(r) is row
// r's first element (or NULL).
template <typename T, int DP, typename F>
__device__ __forceinline__ void store_frag(const float (&o)[DP / 8][4], float f0, float f1, int d,
                                           int lane, F dst) {
  T* p0 = dst(lane >> 2);
  T* p1 = dst((lane >> 2) + 8);
  const bool even = (d & 1) == 0;
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    const int c = n * 8 + 2 * (lane & 3);
    if (c >= d) break;
    if (p0) store2(p0 + c, o[n][0] * f0, o[n][1] * f0, even, c + 1 < d);
    if (p1) store2(p1 + c, o[n][2] * f1, o[n][3] * f1, even, c + 1 < d);
  }
}

struct HaPlace {
  int b, hk, tile, split;
};
// block -> (episode, key head, row or key tile, part); the last tiles first,
// as they have the most work under the past rule
__device__ __forceinline__ HaPlace ha_place(int tiles, int Hk, int splits) {
  HaPlace w;
  int64_t x = blockIdx.x;
  w.split = (int)(x % splits);
  x /= splits;
  w.tile = tiles - 1 - (int)(x % tiles);
  x /= tiles;
  w.hk = (int)(x % Hk);
  w.b = (int)(x / Hk);
  return w;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// Wide: 64 rows, 16 per warp, every warp over all keys of a tile. Narrow (at
// most 16 rows: single tokens): all warps share the rows and take 16 keys
// each of every 64-key tile; their states are joined at the end.
template <typename T, int DP, bool NARROW>
struct HaFwd {
  static constexpr int ROWS = NARROW ? 16 : 64;
  static constexpr int KT = NARROW ? 64 : ha_tile<T, DP>();
  static constexpr int NT = (NARROW ? 16 : KT) / 8;
  static constexpr bool SPLIT = !NARROW && ha_split<T, DP>();
  static constexpr int RS = SPLIT ? hm::split_stride<DP>() : hm::row_stride<T, DP>();
  static constexpr int STAGES = 2;
  static constexpr size_t STAGE = (size_t)2 * KT * RS * sizeof(T);
  static constexpr size_t SMEM = (size_t)ROWS * RS * sizeof(T) + STAGES * STAGE;
};

template <typename T, int DP, bool NARROW>
__global__ void __launch_bounds__(HA_THREADS) head_fwd_kernel(HeadAttnParams p) {
  using C = HaFwd<T, DP, NARROW>;
  constexpr int RS = C::RS, KT = C::KT, NT = C::NT;
  constexpr bool SPLIT = C::SPLIT;
  extern __shared__ __align__(16) unsigned char ha_smem[];
  T* sQ = reinterpret_cast<T*>(ha_smem);
  T* ring = sQ + C::ROWS * RS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.Nq * p.G;
  const HaPlace w = ha_place(cdiv(rows, C::ROWS), p.Hk, p.splits);
  const int r0 = w.tile * C::ROWS;
  const int nrows = min(C::ROWS, rows - r0);
  const int start = p.q_start ? p.q_start[w.b] : p.Nk - p.Nq;
  int len = p.key_len ? p.key_len[w.b] : p.Nk;
  len = max(0, min(len, p.Nk));
  // keys of this block: its part, cut to what any of its rows may see
  const int64_t last_pos = (int64_t)start + (r0 + nrows - 1) / p.G;
  int kend = p.peers == PEERS_PAST ? (int)max((int64_t)0, min((int64_t)len, last_pos + 1)) : len;
  int kbeg = 0;
  if (p.splits > 1) {  // its equal share of the keys that these rows have
    const int per = max(HA_PART, cdiv(cdiv(kend, p.splits), 64) * 64);
    kbeg = (int)min((int64_t)kend, (int64_t)w.split * per);
    kend = min(kend, kbeg + per);
  }
  const int ntiles = kend > kbeg ? cdiv(kend - kbeg, KT) : 0;

  const T* Q = static_cast<const T*>(p.q) + w.b * p.sq.b + (int64_t)w.hk * p.G * p.sq.h;
  const T* K = static_cast<const T*>(p.k) + w.b * p.sk.b + w.hk * p.sk.h;
  const T* V = static_cast<const T*>(p.v) + w.b * p.sv.b + w.hk * p.sv.h;

  auto load_keys = [&](int t) {
    T* sK = ring + (t % C::STAGES) * 2 * KT * RS;
    const int k0 = kbeg + t * KT;
    load_keys_tile<T, DP>(sK, KT, kend - k0, p.d, p.vec, K + (int64_t)k0 * p.sk.n, p.sk.n);
    load_keys_tile<T, DP>(sK + KT * RS, KT, kend - k0, p.d, p.vec, V + (int64_t)k0 * p.sv.n,
                          p.sv.n);
  };
  auto q_row = [&](int r) {
    const int i = (r0 + r) / p.G, g = (r0 + r) - i * p.G;
    return Q + (int64_t)i * p.sq.n + g * p.sq.h;
  };
  // split rows: the next tile waits in registers
  SplitRows<SPLIT ? DP : 16, SPLIT ? KT : 32> nk, nv;
  auto fetch = [&](int t) {
    if constexpr (SPLIT) {
      const int k0 = kbeg + t * KT;
      nk.load(kend - k0, p.d, p.vec, [&](int r) { return K + (int64_t)(k0 + r) * p.sk.n; });
      nv.load(kend - k0, p.d, p.vec, [&](int r) { return V + (int64_t)(k0 + r) * p.sv.n; });
    }
  };
  auto put = [&](int t) {
    if constexpr (SPLIT) {
      T* sK = ring + (t & 1) * 2 * KT * RS;
      nk.store(sK);
      nv.store(sK + KT * RS);
    }
  };
  if constexpr (SPLIT) {
    SplitRows<DP, C::ROWS> q;
    q.load(nrows, p.d, p.vec, q_row);
    q.store(sQ);
    if (ntiles > 0) {
      fetch(0);
      put(0);
    }
  } else {
    load_tile<T, DP>(sQ, C::ROWS, nrows, p.d, p.vec, q_row);
    if (ntiles > 0) load_keys(0);
    cp_async_commit();
  }

  // this thread's two rows
  const int wrow = NARROW ? 0 : warp * 16;
  int jlim[2], self[2];
  const uint32_t* words[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = min(wrow + (lane >> 2) + 8 * u, nrows - 1);
    const int i = (r0 + r) / p.G;
    const int64_t pos = (int64_t)start + i;
    jlim[u] = p.peers == PEERS_PAST ? (int)max((int64_t)0, min((int64_t)kend, pos + 1)) : kend;
    self[u] = p.peers == PEERS_OTHERS && pos >= 0 && pos < p.Nk ? (int)pos : -1;
    words[u] = p.bits ? p.bits + w.b * p.bits_b + (int64_t)i * p.bits_w : nullptr;
  }
  const float c2 = p.scale * HA_LOG2E;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) o[n][u] = 0.f;

  for (int t = 0; t < ntiles; ++t) {
    if constexpr (SPLIT) {
      __syncthreads();
      if (t + 1 < ntiles) fetch(t + 1);
    } else {
      cp_async_wait<0>();
      __syncthreads();
      if (t + 1 < ntiles) load_keys(t + 1);
      cp_async_commit();
    }
    const T* sK = ring + (t % C::STAGES) * 2 * KT * RS + (NARROW ? warp * 16 * RS : 0);
    const T* sV = sK + KT * RS;
    const int k0 = kbeg + t * KT + (NARROW ? warp * 16 : 0);
    if (NARROW && k0 >= kend) continue;
    float s[NT][4];
    ha_scores<SPLIT, T, DP, NT>(s, sQ + wrow * RS, sK, lane);
    // masks: keys a row does not see become -inf
    const int kl = k0 + 8 * NT;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (kl <= jlim[u] && !words[u] && !(self[u] >= k0 && self[u] < kl)) continue;
      uint32_t word = 0xffffffffu;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int j = k0 + 8 * n;
        if (words[u] && ((n & 3) == 0)) word = (j >> 5) < p.bits_w ? __ldg(words[u] + (j >> 5)) : 0u;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (!sees(j + ha_col<SPLIT>(lane, e), jlim[u], self[u], word))
            s[n][2 * u + e] = -INFINITY;
      }
    }
    float f[2], mc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x = m[u];
#pragma unroll
      for (int n = 0; n < NT; ++n) x = max3f(x, s[n][2 * u], s[n][2 * u + 1]);
      x = hm::quad_max(x);
      const float base = x == -INFINITY ? 0.f : x;  // nothing visible so far
      mc[u] = base * c2;
      f[u] = hm::ex2(fmaf(m[u], c2, -mc[u]));
      m[u] = x;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float q = hm::ex2(fmaf(s[n][2 * u + e], c2, -mc[u]));
          s[n][2 * u + e] = q;
          sum += q;
        }
      l[u] = fmaf(l[u], f[u], sum);
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      o[n][0] *= f[0];
      o[n][1] *= f[0];
      o[n][2] *= f[1];
      o[n][3] *= f[1];
    }
    ha_aggregate<SPLIT, T, DP, NT>(o, s, sV, lane);
    // the other buffer was last read before this step's barrier
    if (t + 1 < ntiles) put(t + 1);
  }
  cp_async_wait<0>();
  l[0] = hm::quad_sum(l[0]);
  l[1] = hm::quad_sum(l[1]);

  if constexpr (NARROW) {
    // join the four warps' states: rescale each to the rows' common maximum
    // and add, in warp order
    constexpr int OS = DP + 1;
    float* sm = reinterpret_cast<float*>(ring);      // [4][16] maxima, [4][16] sums
    float* so = sm + 2 * HA_WARPS * 16;              // [4][16][OS]
    static_assert((2 * HA_WARPS * 16 + HA_WARPS * 16 * OS) * 4 <= C::STAGES * C::STAGE, "join");
    __syncthreads();
    if ((lane & 3) == 0) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sm[warp * 16 + (lane >> 2) + 8 * u] = m[u];
        sm[(HA_WARPS + warp) * 16 + (lane >> 2) + 8 * u] = l[u];
      }
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        so[(warp * 16 + (lane >> 2) + 8 * (u >> 1)) * OS + n * 8 + 2 * (lane & 3) + (u & 1)] =
            o[n][u];
    __syncthreads();
    const int r = threadIdx.x >> 3;  // 8 threads per row
    if (r < nrows) {
      float top = -INFINITY, tot = 0.f, fw[HA_WARPS];
#pragma unroll
      for (int v = 0; v < HA_WARPS; ++v) top = fmaxf(top, sm[v * 16 + r]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int v = 0; v < HA_WARPS; ++v) {
        const float mv = sm[v * 16 + r];
        fw[v] = mv == -INFINITY ? 0.f : hm::ex2((mv - base) * c2);
        tot = fmaf(sm[(HA_WARPS + v) * 16 + r], fw[v], tot);
      }
      const int i = (r0 + r) / p.G, g = (r0 + r) - i * p.G;
      const int h = w.hk * p.G + g;
      const float inv = tot == 0.f ? 0.f : 1.f / tot;
      const float lse = tot == 0.f ? -INFINITY : fmaf(base, c2, log2f(tot)) * HA_LN2;
      const int64_t row = ((int64_t)w.b * p.Nq + i) * p.H + h;
      const int64_t srow = ((int64_t)w.b * p.H + h) * p.Nq + i;
      const int64_t part = (int64_t)w.split * p.B * p.Nq * p.H;
      if ((threadIdx.x & 7) == 0) {
        if (p.splits > 1)
          p.part_lse[part + srow] = lse;
        else if (p.lse)
          p.lse[srow] = lse;
      }
      // the join skips parts that saw nothing
      for (int c = threadIdx.x & 7; c < p.d && !(p.splits > 1 && tot == 0.f); c += 8) {
        float x = 0.f;
#pragma unroll
        for (int v = 0; v < HA_WARPS; ++v) x = fmaf(so[(v * 16 + r) * OS + c], fw[v], x);
        x *= inv;
        if (p.splits > 1)
          p.part_o[(part + row) * p.d + c] = x;
        else
          static_cast<T*>(p.o)[row * p.d + c] = from_f32<T>(x);
      }
    }
  } else {
    float inv[2];
    int64_t orow[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = wrow + (lane >> 2) + 8 * u;
      inv[u] = l[u] == 0.f ? 0.f : 1.f / l[u];
      orow[u] = -1;
      if (r >= nrows) continue;
      const int i = (r0 + r) / p.G, g = (r0 + r) - i * p.G;
      const int h = w.hk * p.G + g;
      orow[u] = ((int64_t)w.b * p.Nq + i) * p.H + h;
      const float lse = l[u] == 0.f ? -INFINITY : fmaf(m[u], c2, log2f(l[u])) * HA_LN2;
      const int64_t srow = ((int64_t)w.b * p.H + h) * p.Nq + i;
      if ((lane & 3) == 0) {
        if (p.splits > 1)
          p.part_lse[(int64_t)w.split * p.B * p.Nq * p.H + srow] = lse;
        else if (p.lse)
          p.lse[srow] = lse;
      }
    }
    if (p.splits > 1) {
      float* base = p.part_o + (int64_t)w.split * p.B * p.Nq * p.H * p.d;
      store_frag<float, DP>(o, inv[0], inv[1], p.d, lane, [&](int r) -> float* {
        const int64_t x = orow[r >= 8];
        return x < 0 ? nullptr : base + x * p.d;
      });
    } else {
      store_frag<T, DP>(o, inv[0], inv[1], p.d, lane, [&](int r) -> T* {
        const int64_t x = orow[r >= 8];
        return x < 0 ? nullptr : static_cast<T*>(p.o) + x * p.d;
      });
    }
  }
}

// Join the parts of the key axis: out = sum_s w_s out_s, w_s = exp(lse_s -
// lse). One block per (episode, row, head); its warps share the parts, and
// their sums are added in order.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) head_join_kernel(HeadAttnParams p) {
  constexpr int WARPS = THREADS / 32;
  __shared__ float s_x[WARPS][128], s_top[WARPS], s_sum[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int64_t total = (int64_t)p.B * p.Nq * p.H;
  const int h = (int)(row % p.H);
  const int64_t bi = row / p.H;
  const int i = (int)(bi % p.Nq);
  const int b = (int)(bi / p.Nq);
  const int64_t srow = ((int64_t)b * p.H + h) * p.Nq + i;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < p.splits; s += THREADS)
    top = fmaxf(top, p.part_lse[s * total + srow]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_top[w]);
  float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  // warp w takes parts w, w + WARPS, ...; its lanes hold the weights of 32
  for (int s0 = warp; s0 < p.splits && top != -INFINITY; s0 += 32 * WARPS) {
    const int mine = s0 + lane * WARPS;
    const float ls = mine < p.splits ? p.part_lse[mine * total + srow] : -INFINITY;
    const float wgt = ls == -INFINITY ? 0.f : expf(ls - top);
    // parts that saw nothing wrote nothing
    uint32_t left = __ballot_sync(0xffffffffu, ls != -INFINITY);
    while (left) {
      float y[4][4], wv[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // four parts in flight
        const int s = left ? __ffs(left) - 1 : -1;
        if (s >= 0) left &= left - 1;
        wv[q] = __shfl_sync(0xffffffffu, wgt, s < 0 ? 0 : s);
        const float* o = p.part_o + ((int64_t)(s0 + (s < 0 ? 0 : s) * WARPS) * total + row) * p.d;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          y[q][u] = s >= 0 && lane + 32 * u < p.d ? o[lane + 32 * u] : 0.f;
        if (s < 0) wv[q] = 0.f;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sum += wv[q];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = fmaf(wv[q], y[q][u], x[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) s_x[warp][lane + 32 * u] = x[u];
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) sum += s_sum[w];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int c = threadIdx.x; c < p.d; c += THREADS) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) y += s_x[w][c];
    static_cast<T*>(p.o)[row * p.d + c] = from_f32<T>(y * inv);
  }
  if (threadIdx.x == 0 && p.lse) p.lse[srow] = sum == 0.f ? -INFINITY : top + logf(sum);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// Row statistics, [2][B, H, nqp] with nqp = Nq rounded up to 128: the negative
// of the base-2 lse (-inf for a row that saw nothing and for the rows of
// padding, which makes their weights exp2(s - inf) = 0) and -D = -dout . out
// (0 for padding). A group of 8 lanes per row.
template <typename T>
__global__ void __launch_bounds__(256) head_delta_kernel(HeadAttnParams p, int nqp) {
  const int64_t total = (int64_t)p.B * nqp * p.H;
  // a block's 128 (row, head) pairs are of one episode, four per lane group
  // with their loads in flight together; pairs per episode are below 2^31
  const int blocks_b = cdiv(nqp * p.H, 128);
  const int b = (int)(blockIdx.x / (uint32_t)blocks_b);
  const int pair0 = (int)(blockIdx.x - (uint32_t)b * blocks_b) * 128 + (threadIdx.x >> 3);
  const int sub = threadIdx.x & 7;
  const T *o[4], *g[4];
  int row[4], head[4];
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int pair = pair0 + 32 * u;
    row[u] = pair / p.H;
    head[u] = pair - row[u] * p.H;
    const int i = min(row[u], p.Nq - 1);
    o[u] = static_cast<const T*>(p.o) + b * p.so.b + i * p.so.n + head[u] * p.so.h;
    g[u] = static_cast<const T*>(p.g) + b * p.sg.b + i * p.sg.n + head[u] * p.sg.h;
  }
  if (p.vec) {
    constexpr int E = 16 / (int)sizeof(T);
    for (int c = sub * E; c < p.d; c += 8 * E) {
      uint4 x[4], y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[u] = y[u] = make_uint4(0, 0, 0, 0);
        if (row[u] < p.Nq) {
          x[u] = __ldg(reinterpret_cast<const uint4*>(o[u] + c));
          y[u] = __ldg(reinterpret_cast<const uint4*>(g[u] + c));
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const T* a = reinterpret_cast<const T*>(&x[u]);
        const T* bq = reinterpret_cast<const T*>(&y[u]);
#pragma unroll
        for (int e = 0; e < E; ++e) s[u] = fmaf(to_f32<T>(a[e]), to_f32<T>(bq[e]), s[u]);
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (row[u] < p.Nq)
        for (int c = sub; c < p.d; c += 8)
          s[u] = fmaf(to_f32<T>(o[u][c]), to_f32<T>(g[u][c]), s[u]);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], x);
    if (row[u] < nqp && sub == 0) {
      const int64_t hd = (int64_t)b * p.H + head[u];
      const float lse = row[u] < p.Nq ? p.lse[hd * p.Nq + row[u]] : -INFINITY;
      const int64_t srow = hd * nqp + row[u];
      p.delta[srow] = lse == -INFINITY ? -INFINITY : lse * -HA_LOG2E;
      p.delta[total + srow] = row[u] < p.Nq ? -s[u] : 0.f;
    }
  }
}

template <typename T, int DP>
struct HaBwd {
  static constexpr int RT = 64;                    // rows (or keys) a block owns
  static constexpr int TT = 32;                    // streamed rows per tile
  static constexpr int NT = TT / 8;
  static constexpr bool SPLIT = ha_split<T, DP>() && DP <= 16;
  static constexpr int RS = SPLIT ? hm::split_stride<DP>() : hm::row_stride<T, DP>();
  static constexpr size_t STAGE = (size_t)2 * TT * RS * sizeof(T);
  static constexpr size_t SMEM = (size_t)2 * RT * RS * sizeof(T) + 2 * STAGE;
};

// dq of 64 packed rows: streams K and V.
template <typename T, int DP>
__global__ void __launch_bounds__(HA_THREADS) head_dq_kernel(HeadAttnParams p) {
  using C = HaBwd<T, DP>;
  constexpr int RS = C::RS, KT = C::TT, NT = C::NT;
  constexpr bool SPLIT = C::SPLIT;
  extern __shared__ __align__(16) unsigned char ha_smem[];
  T* sQ = reinterpret_cast<T*>(ha_smem);
  T* sG = sQ + C::RT * RS;
  T* ring = sG + C::RT * RS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.Nq * p.G;
  const HaPlace w = ha_place(cdiv(rows, C::RT), p.Hk, 1);
  const int r0 = w.tile * C::RT;
  const int nrows = min(C::RT, rows - r0);
  const int start = p.q_start ? p.q_start[w.b] : p.Nk - p.Nq;
  int len = p.key_len ? p.key_len[w.b] : p.Nk;
  len = max(0, min(len, p.Nk));
  const int64_t last_pos = (int64_t)start + (r0 + nrows - 1) / p.G;
  const int kend =
      p.peers == PEERS_PAST ? (int)max((int64_t)0, min((int64_t)len, last_pos + 1)) : len;
  const int ntiles = cdiv(kend, KT);
  const T* Q = static_cast<const T*>(p.q) + w.b * p.sq.b + (int64_t)w.hk * p.G * p.sq.h;
  const T* Gr = static_cast<const T*>(p.g) + w.b * p.sg.b + (int64_t)w.hk * p.G * p.sg.h;
  const T* K = static_cast<const T*>(p.k) + w.b * p.sk.b + w.hk * p.sk.h;
  const T* V = static_cast<const T*>(p.v) + w.b * p.sv.b + w.hk * p.sv.h;
  auto load_keys = [&](int t) {
    T* sK = ring + (t & 1) * 2 * KT * RS;
    const int k0 = t * KT;
    load_keys_tile<T, DP>(sK, KT, kend - k0, p.d, p.vec, K + (int64_t)k0 * p.sk.n, p.sk.n);
    load_keys_tile<T, DP>(sK + KT * RS, KT, kend - k0, p.d, p.vec, V + (int64_t)k0 * p.sv.n,
                          p.sv.n);
  };
  auto row_of = [&](const T* base, const HeadStrides& s, int r) {
    const int i = (r0 + r) / p.G, g = (r0 + r) - i * p.G;
    return base + (int64_t)i * s.n + g * s.h;
  };
  auto q_row = [&](int r) { return row_of(Q, p.sq, r); };
  auto g_row = [&](int r) { return row_of(Gr, p.sg, r); };
  SplitRows<SPLIT ? DP : 16, KT> nk, nv;  // split rows: the next tile
  auto fetch = [&](int t) {
    if constexpr (SPLIT) {
      const int k0 = t * KT;
      nk.load(kend - k0, p.d, p.vec, [&](int r) { return K + (int64_t)(k0 + r) * p.sk.n; });
      nv.load(kend - k0, p.d, p.vec, [&](int r) { return V + (int64_t)(k0 + r) * p.sv.n; });
    }
  };
  auto put = [&](int t) {
    if constexpr (SPLIT) {
      T* sK = ring + (t & 1) * 2 * KT * RS;
      nk.store(sK);
      nv.store(sK + KT * RS);
    }
  };
  if constexpr (SPLIT) {
    SplitRows<DP, C::RT> x;
    x.load(nrows, p.d, p.vec, q_row);
    x.store(sQ);
    x.load(nrows, p.d, p.vec, g_row);
    x.store(sG);
    if (ntiles > 0) {
      fetch(0);
      put(0);
    }
  } else {
    load_tile<T, DP>(sQ, C::RT, nrows, p.d, p.vec, q_row);
    load_tile<T, DP>(sG, C::RT, nrows, p.d, p.vec, g_row);
    if (ntiles > 0) load_keys(0);
    cp_async_commit();
  }

  int jlim[2], self[2];
  float nlse[2], ndelta[2];
  const uint32_t* words[2];
  int64_t orow[2];
  const int nqp = head_padded_rows(p.Nq);
  const int64_t total = (int64_t)p.B * nqp * p.H;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int rr = warp * 16 + (lane >> 2) + 8 * u;
    const int r = min(rr, nrows - 1);
    const int i = (r0 + r) / p.G, g = (r0 + r) - i * p.G;
    const int h = w.hk * p.G + g;
    const int64_t pos = (int64_t)start + i;
    jlim[u] = p.peers == PEERS_PAST ? (int)max((int64_t)0, min((int64_t)kend, pos + 1)) : kend;
    self[u] = p.peers == PEERS_OTHERS && pos >= 0 && pos < p.Nk ? (int)pos : -1;
    words[u] = p.bits ? p.bits + w.b * p.bits_b + (int64_t)i * p.bits_w : nullptr;
    const int64_t srow = ((int64_t)w.b * p.H + h) * nqp + i;
    nlse[u] = p.delta[srow];
    ndelta[u] = p.delta[total + srow];
    orow[u] = rr < nrows ? ((int64_t)w.b * p.Nq + i) * p.H + h : -1;
  }
  const float c2 = p.scale * HA_LOG2E;
  float dq[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) dq[n][u] = 0.f;

  for (int t = 0; t < ntiles; ++t) {
    if constexpr (SPLIT) {
      __syncthreads();
      if (t + 1 < ntiles) fetch(t + 1);
    } else {
      cp_async_wait<0>();
      __syncthreads();
      if (t + 1 < ntiles) load_keys(t + 1);
      cp_async_commit();
    }
    const T* sK = ring + (t & 1) * 2 * KT * RS;
    const T* sV = sK + KT * RS;
    const int k0 = t * KT, kl = k0 + KT;
    float s[NT][4], dp[NT][4];
    ha_scores<SPLIT, T, DP, NT>(s, sQ + warp * 16 * RS, sK, lane);
    ha_scores<SPLIT, T, DP, NT>(dp, sG + warp * 16 * RS, sV, lane);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool edge = kl > jlim[u] || words[u] || (self[u] >= k0 && self[u] < kl);
      const uint32_t word =
          words[u] && (k0 >> 5) < p.bits_w ? __ldg(words[u] + (k0 >> 5)) : 0xffffffffu;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = k0 + 8 * n + ha_col<SPLIT>(lane, e);
          float x = hm::ex2(fmaf(s[n][2 * u + e], c2, nlse[u])) * (dp[n][2 * u + e] + ndelta[u]);
          if (edge && !sees(j, jlim[u], self[u], word)) x = 0.f;
          s[n][2 * u + e] = x;
        }
    }
    ha_aggregate<SPLIT, T, DP, NT>(dq, s, sK, lane);
    if (t + 1 < ntiles) put(t + 1);
  }
  cp_async_wait<0>();
  store_frag<T, DP>(dq, p.scale, p.scale, p.d, lane, [&](int r) -> T* {
    const int64_t x = orow[r >= 8];
    return x < 0 ? nullptr : static_cast<T*>(p.dq) + x * p.d;
  });
}

// dk and dv of 64 keys: streams the packed rows of Q and dout.
template <typename T, int DP>
__global__ void __launch_bounds__(HA_THREADS) head_dkv_kernel(HeadAttnParams p) {
  using C = HaBwd<T, DP>;
  constexpr int RS = C::RS, QT = C::TT, NT = C::NT;
  constexpr bool SPLIT = C::SPLIT;
  extern __shared__ __align__(16) unsigned char ha_smem[];
  __shared__ float s_lse[2][QT], s_delta[2][QT];
  __shared__ int s_lim[2][QT], s_self[2][QT];
  __shared__ uint32_t s_word[2][2][QT];
  T* sK = reinterpret_cast<T*>(ha_smem);
  T* sV = sK + C::RT * RS;
  T* ring = sV + C::RT * RS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.Nq * p.G;
  // first tiles first: under the past rule they have the most rows
  HaPlace w = ha_place(cdiv(p.Nk, C::RT), p.Hk, 1);
  w.tile = cdiv(p.Nk, C::RT) - 1 - w.tile;
  const int k0 = w.tile * C::RT;
  const int start = p.q_start ? p.q_start[w.b] : p.Nk - p.Nq;
  int len = p.key_len ? p.key_len[w.b] : p.Nk;
  len = max(0, min(len, p.Nk));
  const int nkeys = min(C::RT, len - k0);  // <= 0: nothing sees these keys
  // under the past rule query i sees key j from i = j - start on
  int i0 = 0;
  if (p.peers == PEERS_PAST) i0 = (int)max((int64_t)0, min((int64_t)p.Nq, (int64_t)k0 - start));
  const int rbeg = (int)(((int64_t)i0 * p.G) / QT) * QT;
  const int ntiles = nkeys > 0 && i0 < p.Nq ? cdiv(rows - rbeg, QT) : 0;
  const T* Q = static_cast<const T*>(p.q) + w.b * p.sq.b + (int64_t)w.hk * p.G * p.sq.h;
  const T* Gr = static_cast<const T*>(p.g) + w.b * p.sg.b + (int64_t)w.hk * p.G * p.sg.h;
  const T* K = static_cast<const T*>(p.k) + w.b * p.sk.b + w.hk * p.sk.h;
  const T* V = static_cast<const T*>(p.v) + w.b * p.sv.b + w.hk * p.sv.h;
  const int nqp = head_padded_rows(p.Nq);
  const int64_t total = (int64_t)p.B * nqp * p.H;
  SplitRows<SPLIT ? DP : 16, QT> nq, ng;  // split rows: the next tile
  auto put = [&](int t) {
    if constexpr (SPLIT) {
      T* sQ = ring + (t & 1) * 2 * QT * RS;
      nq.store(sQ);
      ng.store(sQ + QT * RS);
    }
  };
  auto load_rows = [&](int t) {
    const int q0 = rbeg + t * QT;
    T* sQ = ring + (t & 1) * 2 * QT * RS;
    auto row_of = [&](const T* base, const HeadStrides& s, int r) {
      const int i = (q0 + r) / p.G, g = (q0 + r) - i * p.G;
      return base + (int64_t)i * s.n + g * s.h;
    };
    if constexpr (SPLIT) {
      nq.load(rows - q0, p.d, p.vec, [&](int r) { return row_of(Q, p.sq, r); });
      ng.load(rows - q0, p.d, p.vec, [&](int r) { return row_of(Gr, p.sg, r); });
    } else if (p.G == 1) {
      load_keys_tile<T, DP>(sQ, QT, rows - q0, p.d, p.vec, Q + (int64_t)q0 * p.sq.n, p.sq.n);
      load_keys_tile<T, DP>(sQ + QT * RS, QT, rows - q0, p.d, p.vec, Gr + (int64_t)q0 * p.sg.n,
                            p.sg.n);
    } else {
      load_tile<T, DP>(sQ, QT, rows - q0, p.d, p.vec, [&](int r) { return row_of(Q, p.sq, r); });
      load_tile<T, DP>(sQ + QT * RS, QT, rows - q0, p.d, p.vec,
                       [&](int r) { return row_of(Gr, p.sg, r); });
    }
    if (threadIdx.x < QT) {
      const int r = q0 + threadIdx.x, x = threadIdx.x, st = t & 1;
      s_lse[st][x] = -INFINITY;
      s_delta[st][x] = 0.f;
      s_lim[st][x] = 0;
      s_self[st][x] = -1;
      s_word[st][0][x] = s_word[st][1][x] = 0xffffffffu;
      if (r < rows) {
        const int i = r / p.G, g = r - i * p.G;
        const int64_t srow = ((int64_t)w.b * p.H + w.hk * p.G + g) * nqp + i;
        s_lse[st][x] = p.delta[srow];
        s_delta[st][x] = p.delta[total + srow];
        const int64_t pos = (int64_t)start + i;
        s_lim[st][x] =
            p.peers == PEERS_PAST ? (int)max((int64_t)0, min((int64_t)len, pos + 1)) : len;
        s_self[st][x] = p.peers == PEERS_OTHERS && pos >= 0 && pos < p.Nk ? (int)pos : -1;
        if (p.bits) {
          const uint32_t* b = p.bits + w.b * p.bits_b + (int64_t)i * p.bits_w + (k0 >> 5);
          s_word[st][0][x] = __ldg(b);
          if ((k0 >> 5) + 1 < p.bits_w) s_word[st][1][x] = __ldg(b + 1);
        }
      }
    }
  };
  auto k_row = [&](int r) { return K + (int64_t)(k0 + r) * p.sk.n; };
  auto v_row = [&](int r) { return V + (int64_t)(k0 + r) * p.sv.n; };
  if constexpr (SPLIT) {
    SplitRows<DP, C::RT> x;
    x.load(nkeys, p.d, p.vec, k_row);
    x.store(sK);
    x.load(nkeys, p.d, p.vec, v_row);
    x.store(sV);
  } else {
    load_tile<T, DP>(sK, C::RT, nkeys, p.d, p.vec, k_row);
    load_tile<T, DP>(sV, C::RT, nkeys, p.d, p.vec, v_row);
  }
  if (ntiles > 0) {
    load_rows(0);
    put(0);
  }
  cp_async_commit();
  const float c2 = p.scale * HA_LOG2E;
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) dk[n][u] = dv[n][u] = 0.f;
  const int j0 = k0 + warp * 16 + (lane >> 2);  // this thread's keys: j0, j0 + 8
  for (int t = 0; t < ntiles; ++t) {
    cp_async_wait<0>();
    __syncthreads();
    if (t + 1 < ntiles) load_rows(t + 1);
    cp_async_commit();
    const int st = t & 1;
    const T* sQ = ring + st * 2 * QT * RS;
    const T* sG = sQ + QT * RS;
    float s[NT][4], dp[NT][4];
    ha_scores<SPLIT, T, DP, NT>(s, sK + warp * 16 * RS, sQ, lane);
    ha_scores<SPLIT, T, DP, NT>(dp, sV + warp * 16 * RS, sG, lane);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int x = n * 8 + ha_col<SPLIT>(lane, e);  // query column
        const float ls = s_lse[st][x], de = s_delta[st][x];
        const int lim = s_lim[st][x], self = s_self[st][x];
        const uint32_t word = s_word[st][warp >> 1][x];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float pr = sees(j0 + 8 * u, lim, self, word)
                               ? hm::ex2(fmaf(s[n][2 * u + e], c2, ls))
                               : 0.f;
          s[n][2 * u + e] = pr;
          dp[n][2 * u + e] = pr == 0.f ? 0.f : pr * (dp[n][2 * u + e] + de);
        }
      }
    ha_aggregate<SPLIT, T, DP, NT>(dv, s, sG, lane);
    ha_aggregate<SPLIT, T, DP, NT>(dk, dp, sQ, lane);
    if (t + 1 < ntiles) put(t + 1);
  }
  cp_async_wait<0>();
  auto place = [&](void* base, int r) -> T* {
    const int j = k0 + warp * 16 + r;
    return j < p.Nk ? static_cast<T*>(base) + (((int64_t)w.b * p.Nk + j) * p.Hk + w.hk) * p.d
                    : nullptr;
  };
  store_frag<T, DP>(dk, p.scale, p.scale, p.d, lane, [&](int r) { return place(p.dk, r); });
  store_frag<T, DP>(dv, 1.f, 1.f, p.d, lane, [&](int r) { return place(p.dv, r); });
}

// ---------------------------------------------------------------------------
// visibility words
// ---------------------------------------------------------------------------
// 32 truth values (bytes) to one word, lowest key in the lowest bit.
__global__ void __launch_bounds__(256) pack_bits_kernel(const unsigned char* v, int64_t sb,
                                                        int64_t sn, int B, int Nq, int Nk, int W,
                                                        int vec, uint32_t* out) {
  const int64_t total = (int64_t)B * Nq * W;
  if (vec) {  // rows of whole 16-byte pieces: a thread packs one word
    const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (x >= total) return;
    const int wd = (int)(x % W);
    const int64_t row = x / W;
    const int i = (int)(row % Nq);
    const unsigned char* src = v + (row / Nq) * sb + (int64_t)i * sn + (int64_t)wd * 32;
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (wd * 32 + u * 16 >= Nk) break;
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(src) + u);
      const uint32_t y[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // four 0/1 bytes to four bits: byte t lands on bit 24 + t
        const uint32_t one = __vminu4(y[e], 0x01010101u);
        bits |= (((one * 0x01020408u) >> 24) & 0xfu) << (16 * u + 4 * e);
      }
    }
    out[x] = bits;
    return;
  }
  // any alignment: a warp walks along a row, reads 32 neighbouring bytes and
  // votes; lane u keeps the u-th word of 32
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (int64_t)B * Nq) return;
  const unsigned char* src = v + (row / Nq) * sb + (row % Nq) * sn;
  for (int w0 = 0; w0 < W; w0 += 32) {
    uint32_t mine = 0;
#pragma unroll 8
    for (int u = 0; u < 32; ++u) {
      const int j = (w0 + u) * 32 + lane;
      if ((w0 + u) * 32 >= Nk) break;
      const uint32_t word = __ballot_sync(0xffffffffu, j < Nk && src[j] != 0);
      if (lane == u) mine = word;
    }
    if (w0 + lane < W) out[row * W + w0 + lane] = mine;
  }
}

cudaError_t launch_pack_bits(const void* v, int64_t sb, int64_t sn, int B, int Nq, int Nk,
                             uint32_t* out, cudaStream_t s) {
  const int W = cdiv(Nk, 32);
  const int vec = ((uintptr_t)v % 16 == 0) && sb % 16 == 0 && sn % 16 == 0 && Nk % 16 == 0;
  const int64_t blocks =
      vec ? ((int64_t)B * Nq * W + 255) / 256 : ((int64_t)B * Nq + 7) / 8;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  pack_bits_kernel<<<(unsigned)blocks, 256, 0, s>>>(static_cast<const unsigned char*>(v), sb, sn,
                                                    B, Nq, Nk, W, vec, out);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
constexpr int HA_SMS = 148;
// Up to 16 packed rows a block owns one tile of 16 and its warps share the
// keys; else 64 rows, 16 a warp. One token, 32 x 16384 keys, 16 heads on 2, d =
// 128, bf16: 98 us with 16-row blocks, 144 with 64; 256 episodes of 16 agents,
// 8 heads, d = 64: 20 and 27 us; of 6 agents, 4 heads, d = 16, fp32: 8 and 11.
constexpr int HA_NARROW_ROWS = 16;

// Parts of the key axis: with fewer blocks than the GPU holds at once, split
// until there are about six per SM, each of at least 256 keys. A part is an
// equal share of what its rows may see, so ragged lengths leave no block idle.
// One token, 32 episodes of 16 heads on 2, d = 128, bf16: 16384 keys with four
// parts per SM 106 us, six 95 (5.6 TB/s), eight 98; up to 16384 keys 56, 58
// and 57 (parts of equal length, half of them empty: 63).
int head_splits(int B, int Nq, int Nk, int H, int Hk) {
  const int64_t rows = (int64_t)Nq * (H / Hk);
  const int tile = rows <= HA_NARROW_ROWS ? 16 : 64;
  const int64_t base = (int64_t)B * Hk * ((rows + tile - 1) / tile);
  if (base >= 2 * HA_SMS || Nk < 2 * HA_PART) return 1;
  const int64_t n = (6 * HA_SMS + base - 1) / base;
  return (int)(n < Nk / HA_PART ? n : Nk / HA_PART);
}

template <typename T, int DP, bool NARROW>
static cudaError_t fwd_go(const HeadAttnParams& p, cudaStream_t s) {
  using C = HaFwd<T, DP, NARROW>;
  const int64_t blocks = (int64_t)p.B * p.Hk * cdiv(p.Nq * p.G, C::ROWS) * p.splits;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const void* fn = reinterpret_cast<const void*>(&head_fwd_kernel<T, DP, NARROW>);
  cudaError_t e = raise_smem_limit(fn, C::SMEM);
  if (e != cudaSuccess) return e;
  head_fwd_kernel<T, DP, NARROW><<<(unsigned)blocks, HA_THREADS, C::SMEM, s>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  const int64_t rows = (int64_t)p.B * p.Nq * p.H;
  // few rows: more warps for each. 16 rows of 256 parts: 6.3 us with 256
  // threads, 9.4 with 128; 4096 rows of 8 parts: 6.6 us with 64, 9.7 with 128.
  if (rows <= 4 * HA_SMS)
    head_join_kernel<T, 256><<<(unsigned)rows, 256, 0, s>>>(p);
  else
    head_join_kernel<T, 64><<<(unsigned)rows, 64, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int DP>
static cudaError_t bwd_go(const HeadAttnParams& p, cudaStream_t s) {
  using C = HaBwd<T, DP>;
  const int64_t bq = (int64_t)p.B * p.Hk * cdiv(p.Nq * p.G, C::RT);
  const int64_t bk = (int64_t)p.B * p.Hk * cdiv(p.Nk, C::RT);
  if (bq > 0x7fffffff || bk > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaError_t e = raise_smem_limit(reinterpret_cast<const void*>(&head_dq_kernel<T, DP>), C::SMEM);
  if (e == cudaSuccess)
    e = raise_smem_limit(reinterpret_cast<const void*>(&head_dkv_kernel<T, DP>), C::SMEM);
  if (e != cudaSuccess) return e;
  if (bk) head_dkv_kernel<T, DP><<<(unsigned)bk, HA_THREADS, C::SMEM, s>>>(p);
  if (bq) head_dq_kernel<T, DP><<<(unsigned)bq, HA_THREADS, C::SMEM, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t fwd_any(const HeadAttnParams& p, cudaStream_t s) {
  const bool narrow = (int64_t)p.Nq * p.G <= HA_NARROW_ROWS;
  auto go = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    return narrow ? fwd_go<T, DP, true>(p, s) : fwd_go<T, DP, false>(p, s);
  };
  if (p.d <= 16) return go(std::integral_constant<int, 16>());
  if (p.d <= 32) return go(std::integral_constant<int, 32>());
  if (p.d <= 64) return go(std::integral_constant<int, 64>());
  if (p.d <= 96) return go(std::integral_constant<int, 96>());
  return go(std::integral_constant<int, 128>());
}

cudaError_t launch_head_bwd_tc(const HeadAttnParams& p, int64_t nqp, cudaStream_t s, bool* done);

template <typename T>
static cudaError_t bwd_any(const HeadAttnParams& p, cudaStream_t s) {
  const int nqp = head_padded_rows(p.Nq);
  const int64_t blocks = (int64_t)p.B * cdiv((int)((int64_t)nqp * p.H), 128);
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (blocks) head_delta_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(p, nqp);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if constexpr (sizeof(T) == 2) {
    bool done;
    e = launch_head_bwd_tc(p, nqp, s, &done);
    if (done || e != cudaSuccess) return e;
  }
  if (p.d <= 16) return bwd_go<T, 16>(p, s);
  if (p.d <= 32) return bwd_go<T, 32>(p, s);
  if (p.d <= 64) return bwd_go<T, 64>(p, s);
  if (p.d <= 96) return bwd_go<T, 96>(p, s);
  return bwd_go<T, 128>(p, s);
}

cudaError_t launch_head_fwd_tc(const HeadAttnParams& p, cudaStream_t s, bool* done);

cudaError_t launch_head_fwd(const HeadAttnParams& p, bool bf16, cudaStream_t s) {
  if (bf16) {
    bool done;
    const cudaError_t e = launch_head_fwd_tc(p, s, &done);
    if (done || e != cudaSuccess) return e;
  }
  return bf16 ? fwd_any<__nv_bfloat16>(p, s) : fwd_any<float>(p, s);
}
cudaError_t launch_head_bwd(const HeadAttnParams& p, bool bf16, cudaStream_t s) {
  return bf16 ? bwd_any<__nv_bfloat16>(p, s) : bwd_any<float>(p, s);
}

}  // namespace tarmac
