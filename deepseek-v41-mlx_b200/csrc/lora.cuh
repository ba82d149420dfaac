// lora.cuh -- low-rank adapters of many requests beside one shared projection.
//
// Forward, with i = ids[t] (a negative id: no adapter):
//   h[t, r] = sum_k x[t, k] A_i[r, k]                      A [n, R, K] bf16
//   y[t, c] = base[t, c] + s_i sum_r h[t, r] B_i[c, r]     B [n, N, R] bf16
// Backward, given dy:
//   g[t, r]     = s_i sum_c dy[t, c] B_i[c, r]
//   dx[t, k]    = base[t, k] + sum_r g[t, r] A_i[r, k]
//   dA_i[r, k]  = sum_{t: ids[t] = i} g[t, r] x[t, k]
//   dB_i[c, r]  = s_i sum_{t: ids[t] = i} dy[t, c] h[t, r]
// Three products, each used in both directions:
//   shrink  [tokens x long] . [long x R]      k_lora_shrink   (h, g)
//   expand  [tokens x R] . [R x long]         k_lora_expand   (y, dx)
//   wgrad   [long x tokens] . [tokens x R]    k_lora_wgrad    (dA, dB)
// Every one streams a long activation matrix once against a small operand, so the bound is
// HBM.  All sums are fp32; h and g stay fp32 in memory.  Where h or g is an operand of a
// bf16 tensor-core product it goes in as a sum of bf16 parts (v = p0 + p1 + ..., each the
// rounding of what the earlier ones leave): two parts keep 17 bits or more, below the rounding of a
// bf16 result, three keep all 24 for an fp32 result.
//
// k_lora_plan sorts the tokens by adapter first (a stable counting sort), so that a tile of
// 128 token rows belongs to one adapter; tokens without one come last.
#pragma once
#include "aqgemm.cuh"
#include "bsgemm.cuh"
#include "common.cuh"

namespace dsv41 {

constexpr int LR_TILE = 128;        // token rows of a tile
constexpr int LR_KB = 64;           // contraction length of a stage

// ------------------------------------------------------------------ plan
struct LoraPlan {
  int *perm;       // [T] token of sorted position p
  int2 *tiles;     // {adapter (n: none), tile of that adapter}
  int *n_tiles;    // [1]
  int *off;        // [n + 2] first position of each adapter (n: none), then T
  int *stages;     // [n + 1] 64-token stages of the adapters before this one (wgrad's work)
  int *tickets;    // zeroed here: wgrad's joins
  int n_tickets;
};

// The bin of token t: its adapter in [0, n), or n.  Ids at or past n raise the bad-index status.
__device__ __forceinline__ int lora_bin(int id, int n) {
  if (id >= n) dev_flag(DSV41_DEVST_BAD_INDEX);
  return (id < 0 || id >= n) ? n : id;
}

// Inclusive scan of three values over the block's 1024 threads; tot = the block's sums.
__device__ __forceinline__ void block_scan3(int (&v)[3], int (&tot)[3], int (*wsum)[3]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] += u;
    }
  __syncthreads();
  if (lane == 31)
    for (int i = 0; i < 3; ++i) wsum[warp][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int w = wsum[lane][i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    tot[i] = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    if (warp) v[i] += before;
  }
}

// One cluster of 1024-thread CTAs, each on a contiguous slice of the tokens: histogram in
// shared memory, the other CTAs' histograms over distributed shared memory, one scan over the
// adapters, then the stable scatter (warps of a 1024-token batch in order).  One launch of
// about 4-6 us up to 8192 tokens; sorting in global memory would take three.
__global__ void __launch_bounds__(1024, 1)
    k_lora_plan(const int32_t *__restrict__ ids, int T, int n, LoraPlan p) {
  extern __shared__ int lp_smem[];
  int *cnt = lp_smem, *pos = cnt + (n + 1), *tile0 = pos + (n + 1);   // [n + 1] each
  __shared__ int wsum[32][3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = gridDim.x, rank = blockIdx.x;
  const int per = (((T + C - 1) / C) + 1023) & ~1023;
  const int t0 = min(int64_t(rank) * per, int64_t(T)), t1 = min(int64_t(t0) + per, int64_t(T));
  for (int i = tid; i <= n; i += 1024) cnt[i] = 0;
  __syncthreads();
  for (int t = t0 + tid; t < t1; t += 1024) atomicAdd(&cnt[lora_bin(ids[t], n)], 1);
  cluster_sync();
  int run[3] = {0, 0, 0};                       // tokens, tiles, stages before this batch
  for (int b0 = 0; b0 <= n; b0 += 1024) {
    const int b = b0 + tid;
    int total = 0, before = 0;
    if (b <= n)
      for (int c = 0; c < C; ++c) {
        const int v = ld_cluster_s32(mapa_rank(&cnt[b], c));
        if (c < rank) before += v;
        total += v;
      }
    const int nt = (total + LR_TILE - 1) / LR_TILE, ns = (total + LR_KB - 1) / LR_KB;
    int v[3] = {total, nt, ns}, tot[3];
    block_scan3(v, tot, wsum);
    if (b <= n) {
      const int first = run[0] + v[0] - total;
      pos[b] = first + before;
      tile0[b] = run[1] + v[1] - nt;
      if (rank == 0) {
        p.off[b] = first;
        p.stages[b] = run[2] + v[2] - ns;
        if (b == n) p.off[n + 1] = T;
      }
    }
    for (int i = 0; i < 3; ++i) run[i] += tot[i];
  }
  cluster_sync();                               // everyone has read the histograms
  for (int i = rank * 1024 + tid; i < p.n_tickets; i += C * 1024) p.tickets[i] = 0;
  if (rank == 0 && tid == 0) *p.n_tiles = run[1];
  // scatter: batches of 1024 tokens, their warps one after another
  for (int b0 = t0; b0 < t1; b0 += 1024) {
    const int t = b0 + tid;
    const int bin = t < t1 ? lora_bin(ids[t], n) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, bin);
    const int before = __popc(same & ((1u << lane) - 1));
    const int warps = min(32, (t1 - b0 + 31) >> 5);
    int start = 0;
    for (int w = 0; w < warps; ++w) {
      if (w == warp && before == 0 && bin >= 0) {
        start = pos[bin];
        pos[bin] = start + __popc(same);
      }
      __syncthreads();
    }
    start = __shfl_sync(0xffffffffu, start, __ffs(same) - 1);
    if (bin >= 0) p.perm[start + before] = t;
  }
  // tiles: adapter by binary search over the first tiles
  for (int i = rank * 1024 + tid; i < run[1]; i += C * 1024) {
    int lo = 0, hi = n;                         // last b with tile0[b] <= i (and tiles of its own)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tile0[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    p.tiles[i] = make_int2(lo, i - tile0[lo]);
  }
}

// The rows of tile i: adapter, first sorted position, row count.
struct LoraTile {
  int adapter, p0, rows;
};
__device__ __forceinline__ LoraTile lora_tile(const LoraPlan &p, int i) {
  const int2 v = p.tiles[i];
  const int a = p.off[v.x], b = p.off[v.x + 1];
  const int p0 = a + v.y * LR_TILE;
  return LoraTile{v.x, p0, min(LR_TILE, b - p0)};
}

// ------------------------------------------------------------------ operand staging
// kind::f16 instruction descriptor: fp32 accumulator, bf16 operands, M = 128; mn = 1: that
// operand is stored with its M (or N) index contiguous.
__device__ __forceinline__ uint32_t idesc_lora(uint32_t n, uint32_t a_mn, uint32_t b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) |
         (8u << 24);
}
// Shared-memory descriptor with explicit strides: lbo / sbo in bytes, swz 0 (none) or 2 (128 B).
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lbo, uint32_t sbo,
                                          uint32_t swz) {
  return uint64_t((saddr >> 4) & 0x3FFF) | (uint64_t(lbo >> 4) << 16) |
         (uint64_t(sbo >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(swz) << 61);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(src_bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}
// Eight bf16 values of a row to shared memory, zeros past `valid` of them (valid <= 0: none is
// read).  VEC: the row is 16-byte aligned and valid is 0 or >= 8 (one asynchronous copy);
// otherwise (rows of a length that is no multiple of 8) element loads.
template <bool VEC>
__device__ __forceinline__ void stage8(uint32_t dst, const __nv_bfloat16 *src, int64_t valid) {
  if constexpr (VEC) {
    cp_async16(dst, src, valid > 0 ? 16u : 0u);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
    const uint16_t *s = reinterpret_cast<const uint16_t *>(src);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) w[e >> 1] |= uint32_t(__ldg(s + e)) << (16 * (e & 1));
    st_shared16(dst, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// ------------------------------------------------------------------ shrink
struct LoraShrink {
  const __nv_bfloat16 *x;      // [T, K]
  int64_t K;                   // contraction length
  const __nv_bfloat16 *w;      // [n][R][K], or [n][K][R] (WMN)
  int R, Rp, n;                // Rp: R rounded up to 16
  const float *scaling;        // NULL: 1
  float *out;                  // [T, R]
  LoraPlan plan;
  uint32_t w_bytes;            // staged bytes of w in a stage
};

constexpr int LS_THREADS = 160;
constexpr int LS_X_BYTES = LR_TILE * LR_KB * 2;     // 16 KB
constexpr int LS_MN_LD = LR_KB * 16 + 16;           // bytes between 8-wide r groups (WMN)

// D[128 tokens x Rp] in TMEM: tcgen05.mma kind::f16, M = 128, N = Rp.  A cluster of C CTAs
// takes one tile, each CTA a C-th of the contraction; the partial sums meet in distributed
// shared memory and are added in rank order.  Warps 0-3 gather the token rows (64 values of
// 128 rows a stage) and the adapter's values with 16-byte asynchronous copies, several stages
// ahead; warp 4 issues the MMAs.  Rows past the tile's are zeros, so nothing that other tokens
// hold can reach it.
template <bool WMN, bool VEC, int S>
__global__ void __launch_bounds__(LS_THREADS, 2) k_lora_shrink(const LoraShrink a) {
  extern __shared__ uint8_t ls_raw[];
  uint8_t *smem = ls_raw + ((1024u - (smem_u32(ls_raw) & 1023u)) & 1023u);
  const uint32_t sx = smem_u32(smem), sw = sx + S * LS_X_BYTES;
  __shared__ uint64_t full[S], empty[S], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int rows_s[LR_TILE];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = int(cluster_nctas()), rank = int(cluster_rank());
  const uint32_t cols = a.Rp <= 32 ? 32u : a.Rp <= 64 ? 64u : 128u;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 4);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    fence_barrier_init();
  }
  if (warp == 4) {
    tmem_alloc(&tmem_slot, cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int nkb = int((a.K + LR_KB - 1) / LR_KB);
  const int kb0 = int(int64_t(nkb) * rank / C), kb1 = int(int64_t(nkb) * (rank + 1) / C);
  const int ntiles = *a.plan.n_tiles;
  int it = 0, done = 0;                   // stages and tiles so far (barrier parities)
  bool ok = true;                         // no wait of this thread has run out
  for (int i = int(cluster_id_x()); i < ntiles; i += int(ncluster_x())) {
    const LoraTile tl = lora_tile(a.plan, i);
    if (tl.adapter == a.n) {              // no adapter: h = 0
      if (rank == 0)
        for (int e = tid; e < tl.rows * a.R; e += LS_THREADS)
          a.out[int64_t(a.plan.perm[tl.p0 + e / a.R]) * a.R + e % a.R] = 0.0f;
      continue;
    }
    if (tid < LR_TILE) rows_s[tid] = tid < tl.rows ? a.plan.perm[tl.p0 + tid] : -1;
    __syncthreads();
    if (warp < 4) {
      // ------------------------------------------------------------ producers
      const int c = tid & 7, r0 = tid >> 3;          // 16-byte chunk, rows r0 + 16 j
      int tok[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) tok[j] = rows_s[r0 + 16 * j];
      const __nv_bfloat16 *wi = a.w + int64_t(tl.adapter) * a.R * a.K;
      int jt = it;
      for (int kb = kb0; kb < kb1 && ok; ++kb, ++jt) {
        const int s = jt % S;
        if (!mbar_wait(&empty[s], (uint32_t(jt / S) & 1u) ^ 1u)) {
          ok = false;
          break;
        }
        const int64_t k = int64_t(kb) * LR_KB + c * 8;
        const uint32_t dx = sx + s * LS_X_BYTES + r0 * 128 + ((c ^ (r0 & 7)) << 4);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          stage8<VEC>(dx + j * 2048, tok[j] < 0 ? a.x : a.x + int64_t(tok[j]) * a.K + k,
                      tok[j] < 0 ? 0 : a.K - k);
        const uint32_t dw = sw + s * a.w_bytes;
        if constexpr (!WMN) {
          for (int r = r0; r < a.Rp; r += 16)
            cp_async16(dw + r * 128 + ((c ^ (r & 7)) << 4), r < a.R && k < a.K ? wi + r * a.K + k : wi,
                       r < a.R && k < a.K ? 16u : 0u);
        } else {
          const int rc = a.Rp >> 3;
          for (int e = tid; e < rc * LR_KB; e += 128) {
            const int g = e % rc, kk = e / rc;
            const int64_t kr = int64_t(kb) * LR_KB + kk;
            const bool in = g * 8 < a.R && kr < a.K;
            cp_async16(dw + g * LS_MN_LD + kk * 16, in ? wi + kr * a.R + g * 8 : wi, in ? 16u : 0u);
          }
        }
        cp_async_commit();
        if (kb - kb0 >= S - 2) {                     // the stage issued S - 2 ago has landed
          cp_async_wait<S - 2>();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[(jt - (S - 2)) % S]);
        }
      }
      cp_async_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && ok)
        for (int e = max(it, jt - (S - 2)); e < jt; ++e) mbar_arrive(&full[e % S]);
    } else {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t id = idesc_lora(a.Rp, 0, WMN ? 1 : 0);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        const int jt = it + kb - kb0, s = jt % S;
        if (!warp_wait(&full[s], uint32_t(jt / S) & 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t da = sdesc_sw128(sx + s * LS_X_BYTES);
        const uint32_t bw = sw + s * a.w_bytes;
        const uint64_t db = WMN ? sdesc(bw, 128, LS_MN_LD, 0) : sdesc_sw128(bw);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma_bf16_el(tmem, da + uint64_t(2 * k), db + uint64_t((WMN ? 16 : 2) * k), id,
                         (kb > kb0 || k) ? 1u : 0u);
        tc_commit_el(&empty[s]);
      }
      if (ok) tc_commit_el(&acc_full);
      __syncwarp();
    }
    it += kb1 - kb0;
    // ------------------------------------------------------------ the C partial sums
    float *red = reinterpret_cast<float *>(smem);
    const int ld = a.Rp + 4;
    if (warp < 4) {
      if (ok) ok = warp_wait(&acc_full, uint32_t(done) & 1u);
      tc_fence_after();
      for (int c0 = 0; c0 < a.Rp; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(tmem + (uint32_t(32 * warp) << 16) + c0, v);
        float *dst = red + tid * ld + c0;
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          if (c0 + e < a.Rp)
            *reinterpret_cast<uint4 *>(dst + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
      }
      tc_fence_before();
    }
    ++done;
    cluster_sync();
    tc_fence_after();
    const float sc = a.scaling ? a.scaling[tl.adapter] : 1.0f;
    const int q4 = a.R >> 2, row_a = LR_TILE * rank / C, row_b = LR_TILE * (rank + 1) / C;
    for (int e = tid; e < (row_b - row_a) * q4; e += LS_THREADS) {
      const int row = row_a + e / q4, c4 = (e % q4) * 4;
      if (row >= tl.rows) break;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < C; ++q) {
        float4 v;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                     : "r"(mapa_rank(red + row * ld + c4, q))
                     : "memory");
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      *reinterpret_cast<float4 *>(a.out + int64_t(rows_s[row]) * a.R + c4) =
          make_float4(s.x * sc, s.y * sc, s.z * sc, s.w * sc);
    }
    cluster_sync();                       // before the stages are written again
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// ------------------------------------------------------------------ few tokens
struct LoraDecode {
  const __nv_bfloat16 *x, *a, *b;
  int64_t K, N;
  int R, n;
  const float *scaling;
  const int32_t *ids;
  const void *base;
  void *y;
  float *h;                    // NULL: not kept
};

// 8 bf16 products added to acc
__device__ __forceinline__ float dot8(uint4 u, uint4 v, float acc) {
  const uint32_t a[4] = {u.x, u.y, u.z, u.w}, b[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(b[i] << 16), acc);
    acc = fmaf(__uint_as_float(a[i] & 0xFFFF0000u), __uint_as_float(b[i] & 0xFFFF0000u), acc);
  }
  return acc;
}

constexpr int LD_THREADS = 256, LD_WARPS = 8;

// Both products of a token in one launch, no plan: a cluster per token.  Each CTA takes a slice
// of K (its warps R / 8 ranks each), the partial h meet in distributed shared memory in rank
// order, then each CTA takes a slice of the columns, a row of B per group of LPR lanes.  The
// first rows of B are requested before the cluster meets.  Bound by the latency of one pass
// over an adapter (360 KB at K 7168, N 4096, R 16), which tokens on the same adapter find in L2.
// RW: ranks a warp; LPR: lanes a row of B, the power of two at or above R / 8.
template <typename OT, int RW, int LPR>
__global__ void __launch_bounds__(LD_THREADS) k_lora_decode(const LoraDecode p) {
  constexpr int COLS = LD_THREADS / LPR;            // columns a pass
  constexpr int PF = 8;                             // passes requested ahead
  __shared__ float part[LD_WARPS * RW];
  __shared__ float hs[LD_WARPS * RW];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = int(cluster_nctas()), rank = int(cluster_rank());
  const int64_t t = cluster_id_x();
  const OT *base = static_cast<const OT *>(p.base);
  OT *y = static_cast<OT *>(p.y) + t * p.N;
  const int i = lora_bin(p.ids[t], p.n);
  const int64_t c0 = p.N * rank / C, c1 = p.N * (rank + 1) / C;
  if (i == p.n) {                                   // uniform over the cluster
    for (int64_t c = c0 + tid; c < c1; c += LD_THREADS)
      y[c] = base ? base[t * p.N + c] : OT(0.0f);
    if (p.h && rank == 0)
      for (int r = tid; r < p.R; r += LD_THREADS) p.h[t * p.R + r] = 0.0f;
    return;
  }
  const uint4 z = make_uint4(0, 0, 0, 0);
  const int ln = tid % LPR, cg = tid / LPR;
  const __nv_bfloat16 *bi = p.b + int64_t(i) * p.N * p.R + ln * 8;
  uint4 bv[PF];
#pragma unroll
  for (int u = 0; u < PF; ++u) {
    const int64_t c = c0 + u * COLS + cg;
    bv[u] = (c < c1 && ln * 8 < p.R) ? __ldg(reinterpret_cast<const uint4 *>(bi + c * p.R)) : z;
  }
  {
    const int64_t nk = p.K >> 3, k0 = nk * rank / C, k1 = nk * (rank + 1) / C;
    const uint4 *xr = reinterpret_cast<const uint4 *>(p.x + t * p.K);
    const uint4 *ar = reinterpret_cast<const uint4 *>(p.a + int64_t(i) * p.R * p.K);
    float acc[RW] = {};
#pragma unroll 2
    for (int64_t k = k0 + lane; k < k1; k += 32) {
      const uint4 xv = __ldg(xr + k);
      uint4 av[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r)
        av[r] = warp * RW + r < p.R ? __ldg(ar + (warp * RW + r) * nk + k) : z;
#pragma unroll
      for (int r = 0; r < RW; ++r) acc[r] = dot8(xv, av[r], acc[r]);
    }
#pragma unroll
    for (int r = 0; r < RW; ++r) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
      if (lane == 0) part[warp * RW + r] = acc[r];
    }
  }
  cluster_sync();
  if (tid < LD_WARPS * RW) {
    float s = 0.0f;
    for (int q = 0; q < C; ++q)
      s += __int_as_float(ld_cluster_s32(mapa_rank(part + tid, q)));
    if (p.h && rank == 0 && tid < p.R) p.h[t * p.R + tid] = s;
    hs[tid] = tid < p.R ? s * (p.scaling ? p.scaling[i] : 1.0f) : 0.0f;
  }
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");      // part has been read
  float hv[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) hv[e] = ln * 8 + e < p.R ? hs[ln * 8 + e] : 0.0f;
  for (int64_t cb = c0; cb < c1; cb += PF * COLS) {
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      const int64_t c = cb + u * COLS + cg;
      const uint32_t w[4] = {bv[u].x, bv[u].y, bv[u].z, bv[u].w};
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s = fmaf(hv[2 * e], __uint_as_float(w[e] << 16), s);
        s = fmaf(hv[2 * e + 1], __uint_as_float(w[e] & 0xFFFF0000u), s);
      }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (ln == 0 && c < c1) y[c] = OT((base ? float(base[t * p.N + c]) : 0.0f) + s);
      const int64_t cn = c + PF * COLS;
      bv[u] = (cn < c1 && ln * 8 < p.R) ? __ldg(reinterpret_cast<const uint4 *>(bi + cn * p.R)) : z;
    }
  }
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// ------------------------------------------------------------------ expand
struct LoraExpand {
  const float *h;              // [T, R]
  const __nv_bfloat16 *w;      // [n][N][R], or [n][R][N] (WMN)
  int64_t N;
  int R, n;
  const float *scaling;        // NULL: 1
  const void *base;            // [T, N] or NULL
  void *y;                     // [T, N]
  LoraPlan plan;
  int ncb, cpu;                // 256-column blocks, and how many of them a work item takes
  int vec;                     // rows of base and y are 16-byte aligned
};

// v as bf16 parts; the rest after each part is exact in fp32 (and zero after an infinity or NaN).
template <int NS>
__device__ __forceinline__ void split_bf16(float v, uint16_t (&p)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    p[i] = f2bf_bits(v);
    v = (p[i] & 0x7F80) == 0x7F80 ? 0.0f : v - bf_bits2f(p[i]);
  }
}

// A CTA of 8 warps takes a tile's 128 token rows and 256 output columns at a time, a warp 32
// columns: the warp's piece of W stays in registers for all 128 rows (mma.sync m16n8k16), the
// split rows of h are in shared memory.  Output columns are dealt to the MMA's n indices so
// that a lane's four accumulator pairs are 8 neighbouring columns (and k indices so that a
// lane's operand values are 4 neighbouring r): base and y move as 16-byte pieces straight from
// registers, no transposition.  KJ = ceil(R / 16) rounded up to 1, 2, 4 or 8.
template <bool WMN, typename OT, int KJ>
__global__ void __launch_bounds__(256) k_lora_expand(const LoraExpand a) {
  constexpr int NS = sizeof(OT) == 4 ? 3 : 2;
  extern __shared__ uint2 le_h[];                 // [NS][KJ][128 rows][4 lanes] pairs of bf16x2
  __shared__ int rows_s[LR_TILE];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const OT *base = static_cast<const OT *>(a.base);
  OT *y = static_cast<OT *>(a.y);
  const int per_tile = (a.ncb + a.cpu - 1) / a.cpu;
  const int64_t items = int64_t(*a.plan.n_tiles) * per_tile;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const LoraTile tl = lora_tile(a.plan, int(item / per_tile));
    const bool live = tl.adapter < a.n;
    const int cb0 = int(item % per_tile) * a.cpu, cb1 = min(cb0 + a.cpu, a.ncb);
    __syncthreads();
    if (tid < LR_TILE) rows_s[tid] = tid < tl.rows ? a.plan.perm[tl.p0 + tid] : -1;
    __syncthreads();
    if (live) {
      const float sc = a.scaling ? a.scaling[tl.adapter] : 1.0f;
      for (int e = tid; e < KJ * LR_TILE * 4; e += 256) {
        const int row = (e >> 2) / KJ, r = ((e >> 2) % KJ) * 16 + (e & 3) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (rows_s[row] >= 0 && r < a.R)
          v = *reinterpret_cast<const float4 *>(a.h + int64_t(rows_s[row]) * a.R + r);
        uint16_t p0[NS], p1[NS], p2[NS], p3[NS];
        split_bf16<NS>(v.x * sc, p0);
        split_bf16<NS>(v.y * sc, p1);
        split_bf16<NS>(v.z * sc, p2);
        split_bf16<NS>(v.w * sc, p3);
#pragma unroll
        for (int i = 0; i < NS; ++i)
          le_h[((i * KJ + (r >> 4)) * LR_TILE + row) * 4 + (e & 3)] = make_uint2(
              uint32_t(p0[i]) | (uint32_t(p1[i]) << 16), uint32_t(p2[i]) | (uint32_t(p3[i]) << 16));
      }
    }
    __syncthreads();
    for (int cb = cb0; cb < cb1; ++cb) {
      const int64_t c0 = int64_t(cb) * 256 + warp * 32;
      if (c0 >= a.N) break;
      // W of this warp's 32 columns: b[j][q] = the k16 step j of n index g = column
      // c0 + 8 (g >> 1) + 2 q + (g & 1), values r = 16 j + 4 t .. + 3
      uint2 b[KJ][4];
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) b[j][q] = make_uint2(0u, 0u);
      if (live) {
        if constexpr (!WMN) {
          const __nv_bfloat16 *wi = a.w + int64_t(tl.adapter) * a.R * a.N;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int64_t col = c0 + 8 * (g >> 1) + 2 * q + (g & 1);
#pragma unroll
            for (int j = 0; j < KJ; ++j)
              if (col < a.N && 16 * j + 4 * t < a.R)
                b[j][q] = __ldg(reinterpret_cast<const uint2 *>(wi + col * a.R + 16 * j + 4 * t));
          }
        } else {
          const __nv_bfloat16 *wi = a.w + int64_t(tl.adapter) * a.R * a.N;
          const int64_t col = c0 + 8 * (g >> 1);          // N % 8 == 0: 8 columns or none
#pragma unroll
          for (int j = 0; j < KJ; ++j) {
            const int r = 16 * j + 4 * t;
            if (col < a.N && r < a.R) {
              uint4 v[4];
#pragma unroll
              for (int u = 0; u < 4; ++u)
                v[u] = __ldg(reinterpret_cast<const uint4 *>(wi + int64_t(r + u) * a.N + col));
              const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;   // this lane's column of each pair
              b[j][0] = make_uint2(__byte_perm(v[0].x, v[1].x, sel), __byte_perm(v[2].x, v[3].x, sel));
              b[j][1] = make_uint2(__byte_perm(v[0].y, v[1].y, sel), __byte_perm(v[2].y, v[3].y, sel));
              b[j][2] = make_uint2(__byte_perm(v[0].z, v[1].z, sel), __byte_perm(v[2].z, v[3].z, sel));
              b[j][3] = make_uint2(__byte_perm(v[0].w, v[1].w, sel), __byte_perm(v[2].w, v[3].w, sel));
            }
          }
        }
      }
      const int64_t col = c0 + 8 * t;                      // this lane's 8 output columns
      for (int m0 = 0; m0 < tl.rows; m0 += 16) {
        const int row[2] = {rows_s[m0 + g], rows_s[m0 + g + 8]};
        float d[4][4];
        if (a.vec && col < a.N) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (base && row[u] >= 0) {
              const OT *src = base + int64_t(row[u]) * a.N + col;
              if constexpr (sizeof(OT) == 4) {
                const float4 v0 = *reinterpret_cast<const float4 *>(src);
                const float4 v1 = *reinterpret_cast<const float4 *>(src + 4);
                f[0] = v0.x; f[1] = v0.y; f[2] = v0.z; f[3] = v0.w;
                f[4] = v1.x; f[5] = v1.y; f[6] = v1.z; f[7] = v1.w;
              } else {
                const uint4 v = *reinterpret_cast<const uint4 *>(src);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  f[2 * q] = bf_bits2f(uint16_t(w[q]));
                  f[2 * q + 1] = bf_bits2f(uint16_t(w[q] >> 16));
                }
              }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              d[q][2 * u] = f[2 * q];
              d[q][2 * u + 1] = f[2 * q + 1];
            }
          }
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              d[e >> 1][2 * u + (e & 1)] =
                  (base && row[u] >= 0 && col + e < a.N)
                      ? float(base[int64_t(row[u]) * a.N + col + e]) : 0.0f;
        }
        if (live) {
          float acc[4][4] = {};
#pragma unroll
          for (int i = NS - 1; i >= 0; --i)                // the smallest parts first
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
              const uint2 *hp = le_h + ((i * KJ + j) * LR_TILE + m0) * 4;
              const uint2 lo = hp[g * 4 + t], hi = hp[(g + 8) * 4 + t];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                mma_bf16(acc[q], lo.x, hi.x, lo.y, hi.y, b[j][q].x, b[j][q].y);
            }
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[q][e] += acc[q][e];
        }
        if (a.vec && col < a.N) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (row[u] < 0) continue;
            OT *dst = y + int64_t(row[u]) * a.N + col;
            if constexpr (sizeof(OT) == 4) {
              *reinterpret_cast<float4 *>(dst) =
                  make_float4(d[0][2 * u], d[0][2 * u + 1], d[1][2 * u], d[1][2 * u + 1]);
              *reinterpret_cast<float4 *>(dst + 4) =
                  make_float4(d[2][2 * u], d[2][2 * u + 1], d[3][2 * u], d[3][2 * u + 1]);
            } else {
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                w[q] = uint32_t(f2bf_bits(d[q][2 * u])) | (uint32_t(f2bf_bits(d[q][2 * u + 1])) << 16);
              *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (row[u] >= 0 && col + e < a.N)
                y[int64_t(row[u]) * a.N + col + e] = OT(d[e >> 1][2 * u + (e & 1)]);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ wgrad
struct LoraGradSide {
  const __nv_bfloat16 *v;      // [T, C] long side: x (dA) or dy (dB)
  const float *u;              // [T, R] rank side: g (dA) or h (dB)
  int64_t C;
  int ncb;                     // 256-column blocks
  const float *scaling;        // multiplies u (NULL: 1)
  void *out;                   // [n, R, C] (r_major) or [n, C, R]
  int r_major;
  int vec;                     // v's rows are 16-byte aligned
};
struct LoraWgrad {
  LoraGradSide side[2];
  int R, Rp, n;
  LoraPlan plan;
  float *part;                 // [2 * grid][Rp][256] partial sums
  uint32_t u_bytes;            // one bf16 part of a stage of u: (Rp / 8) * LG_MN_LD
};

constexpr int LG_THREADS = 416;
constexpr int LG_COLS = 256;
constexpr int LG_X_BYTES = LR_KB * LG_COLS * 2;     // 32 KB: 4 pieces of [64 tokens x 128 B]
constexpr int LG_MN_LD = LR_KB * 16 + 16;
__host__ __device__ __forceinline__ constexpr uint32_t lg_tmem_cols(int Rp) {
  return Rp <= 32 ? 128u : Rp <= 64 ? 256u : 512u;   // two buffers of two accumulators
}

// One piece of work of a CTA: stages [s0, s1) of one (side, adapter, column block).
struct LoraSeg {
  int side, adapter, cb;
  int first, count;            // 64-token stages of the adapter: first, how many
  int total;                   // stages of the whole item
  int64_t item0;               // the item's first stage in the launch's work
};

__device__ __forceinline__ LoraSeg lora_seg(const LoraWgrad &a, int64_t s, int64_t s_end) {
  LoraSeg g;
  const int64_t tot = a.plan.stages[a.n];           // stages of all adapters
  g.side = s >= tot * a.side[0].ncb ? 1 : 0;
  const int64_t base = g.side ? tot * a.side[0].ncb : 0;
  const int ncb = a.side[g.side].ncb;
  const int64_t q = s - base;
  int lo = 0, hi = a.n - 1;                         // last adapter with stages * ncb <= q
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (int64_t(a.plan.stages[mid]) * ncb <= q) lo = mid;
    else hi = mid - 1;
  }
  g.adapter = lo;
  const int64_t a0 = int64_t(a.plan.stages[lo]) * ncb;
  g.total = a.plan.stages[lo + 1] - a.plan.stages[lo];
  g.cb = int((q - a0) / g.total);
  g.first = int((q - a0) % g.total);
  g.item0 = s - g.first;
  g.count = int(min(int64_t(g.total - g.first), s_end - s));
  return g;
}

// D[256 columns x Rp] = sum over an adapter's tokens, two M = 128 accumulators in TMEM; both
// operands have the token index as their rows in memory, which is the MMA's contraction
// index: v as 128-byte-swizzled pieces of 64 columns, u (its bf16 parts) as unswizzled groups
// of 8.  The work of both gradients (every adapter's 64-token stages times the column blocks)
// is one line that the CTAs cut into equal pieces: an item that one CTA covers is written at
// once, one that a cut divides is written as fp32 partial sums (at most two per CTA) and the
// last CTA to arrive adds them in order.  Warps 0-3 copy v, 4-7 split u, 8 issues the MMAs,
// 9-12 read TMEM; accumulators are double-buffered, so an item's stores overlap the next one.
template <typename OT, int S>
__global__ void __launch_bounds__(LG_THREADS, S == 3 ? 2 : 1) k_lora_wgrad(const LoraWgrad a) {
  constexpr int NS = sizeof(OT) == 4 ? 3 : 2;
  extern __shared__ uint8_t lg_raw[];
  uint8_t *smem = lg_raw + ((1024u - (smem_u32(lg_raw) & 1023u)) & 1023u);
  const uint32_t sx = smem_u32(smem), su = sx + S * LG_X_BYTES;
  const uint32_t u_stage = NS * a.u_bytes;
  __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2], mma_done;
  __shared__ uint32_t tmem_slot;
  __shared__ int last_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t cols = lg_tmem_cols(a.Rp), acc_cols = cols / 2, half_cols = cols / 4;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 8);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    mbar_init(&mma_done, 1);
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(&tmem_slot, cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int64_t all = int64_t(a.plan.stages[a.n]) * (a.side[0].ncb + a.side[1].ncb);
  const int64_t per = (all + gridDim.x - 1) / gridDim.x;
  const int64_t w0 = min(int64_t(blockIdx.x) * per, all), w1 = min(w0 + per, all);

  if (warp < 8) {
    // -------------------------------------------------------------- producers
    int it = 0;
    bool ok = true;
    for (int64_t s = w0; s < w1 && ok;) {
      const LoraSeg sg = lora_seg(a, s, w1);
      const LoraGradSide &sd = a.side[sg.side];
      const int p0 = a.plan.off[sg.adapter], pn = a.plan.off[sg.adapter + 1];
      const float sc = sd.scaling ? sd.scaling[sg.adapter] : 1.0f;
      for (int q = 0; q < sg.count; ++q, ++it) {
        const int st = it % S;
        if (!mbar_wait(&empty[st], (uint32_t(it / S) & 1u) ^ 1u)) {
          ok = false;
          break;
        }
        const int pos = p0 + (sg.first + q) * LR_KB;       // sorted position of the stage's row 0
        if (warp < 4) {
          // 64 rows x 32 chunks of 16 bytes: a warp's 32 lanes take one row
          const int64_t c = int64_t(sg.cb) * LG_COLS + lane * 8;
          const uint32_t d0 = sx + st * LG_X_BYTES + (lane >> 3) * 8192;
          // the token indices of this warp's 16 rows, one load a lane
          const int mine = pos + warp * 16 + (lane & 15);
          const int tok_l = mine < pn ? a.plan.perm[mine] : -1;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int row = warp * 16 + j;
            const int tok = __shfl_sync(0xffffffffu, tok_l, j);
            const uint32_t d = d0 + row * 128 + (((lane & 7) ^ (row & 7)) << 4);
            const bool in = tok >= 0 && c < sd.C;
            const __nv_bfloat16 *src = in ? sd.v + int64_t(tok) * sd.C + c : sd.v;
            if (sd.vec) stage8<true>(d, src, in ? 8 : 0);
            else stage8<false>(d, src, in ? sd.C - c : 0);
          }
          cp_async_commit();
          if (it >= S - 2) {
            cp_async_wait<S - 2>();
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[(it - (S - 2)) % S]);
          }
        } else {
          const int e = tid - 128, row = e & 63;
          const int tok = pos + row < pn ? a.plan.perm[pos + row] : -1;
          const uint32_t d = su + st * u_stage + row * 16;
          for (int g = e >> 6; g < (a.Rp >> 3); g += 2) {
            float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (tok >= 0 && g * 8 < a.R) {
              const float4 *src = reinterpret_cast<const float4 *>(sd.u + int64_t(tok) * a.R + g * 8);
              const float4 v0 = __ldg(src), v1 = __ldg(src + 1);
              f[0] = v0.x * sc; f[1] = v0.y * sc; f[2] = v0.z * sc; f[3] = v0.w * sc;
              f[4] = v1.x * sc; f[5] = v1.y * sc; f[6] = v1.z * sc; f[7] = v1.w * sc;
            }
            uint32_t w[NS][4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint16_t plo[NS], phi[NS];
              split_bf16<NS>(f[2 * x], plo);
              split_bf16<NS>(f[2 * x + 1], phi);
#pragma unroll
              for (int i = 0; i < NS; ++i) w[i][x] = uint32_t(plo[i]) | (uint32_t(phi[i]) << 16);
            }
#pragma unroll
            for (int i = 0; i < NS; ++i)
              st_shared16(d + i * a.u_bytes + g * LG_MN_LD,
                          make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[st]);
        }
      }
      s += sg.count;
    }
    if (warp < 4) {
      cp_async_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && ok)
        for (int e = max(0, it - (S - 2)); e < it; ++e) mbar_arrive(&full[e % S]);
    }
  } else if (warp == 8) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t id = idesc_lora(a.Rp, 1, 1);
    int it = 0, seg = 0;
    bool ok = true;
    for (int64_t s = w0; s < w1 && ok; ++seg) {
      const LoraSeg sg = lora_seg(a, s, w1);
      if (!warp_wait(&acc_empty[seg & 1], (uint32_t(seg >> 1) & 1u) ^ 1u)) break;
      tc_fence_after();
      const uint32_t acc = tmem + uint32_t(seg & 1) * acc_cols;
      for (int q = 0; q < sg.count; ++q, ++it) {
        const int st = it % S;
        if (!warp_wait(&full[st], uint32_t(it / S) & 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t dv = sdesc(sx + st * LG_X_BYTES, 8192, 1024, 2);
        const uint64_t du = sdesc(su + st * u_stage, 128, LG_MN_LD, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k)                 // 16 tokens an MMA
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
              tc_mma_bf16_el(acc + hf * half_cols, dv + uint64_t(128 * k + 1024 * hf),
                             du + uint64_t(16 * k) + uint64_t(i * (a.u_bytes >> 4)), id,
                             (q || k || i) ? 1u : 0u);
        tc_commit_el(&empty[st]);
      }
      if (!ok) break;
      tc_commit_el(&acc_full[seg & 1]);
      s += sg.count;
    }
    tc_commit_el(&mma_done);
    warp_wait(&mma_done, 0);
    __syncwarp();
  } else {
    // -------------------------------------------------------------- epilogue
    const int e4 = tid - 288;                       // 0 .. 127
    const int q4 = warp & 3;                        // TMEM lanes 32 q4 .. + 31
    int seg = 0;
    bool ok = true;
    for (int64_t s = w0; s < w1; ++seg) {
      const LoraSeg sg = lora_seg(a, s, w1);
      const LoraGradSide &sd = a.side[sg.side];
      // a warp whose wait ran out goes on without waiting: the others meet it at the barriers
      if (ok) ok = warp_wait(&acc_full[seg & 1], uint32_t(seg >> 1) & 1u);
      tc_fence_after();
      const uint32_t acc = tmem + uint32_t(seg & 1) * acc_cols + (uint32_t(32 * q4) << 16);
      const int64_t f = sg.item0 / per, l = (sg.item0 + sg.total - 1) / per;   // CTAs of the item
      const int col = 32 * q4 + lane;               // this thread's column in each half
      OT *out = static_cast<OT *>(sd.out) + int64_t(sg.adapter) * a.R * sd.C;
      const int slot = 2 * int(blockIdx.x) + (s == w0 ? 0 : 1);
      float *mine = a.part + int64_t(slot) * a.Rp * LG_COLS;
      bool join = f == l;
      if (f != l) {
        for (int hf = 0; hf < 2; ++hf)
          for (int c0 = 0; c0 < a.Rp; c0 += 32) {
            uint32_t v[32];
            tmem_ld32(acc + hf * half_cols + c0, v);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (c0 + x < a.R) mine[(c0 + x) * LG_COLS + hf * 128 + col] = __uint_as_float(v[x]);
          }
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (e4 == 0) last_s = atomicAdd(a.plan.tickets + f, 1) == int(l - f);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        join = last_s != 0;
        if (join) __threadfence();
      }
      if (join) {
        for (int hf = 0; hf < 2; ++hf) {
          const int64_t c = int64_t(sg.cb) * LG_COLS + hf * 128 + col;
          for (int c0 = 0; c0 < a.Rp; c0 += 32) {
            uint32_t v[32];
            if (f == l) {
              tmem_ld32(acc + hf * half_cols + c0, v);
            } else {
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] = 0u;
              for (int64_t k = f; k <= l; ++k) {
                const int sl = 2 * int(k) + (k == f && sg.item0 > f * per ? 1 : 0);
                const float *src = a.part + int64_t(sl) * a.Rp * LG_COLS + hf * 128 + col;
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (c0 + x < a.R)
                    v[x] = __float_as_uint(__uint_as_float(v[x]) + __ldcg(src + (c0 + x) * LG_COLS));
              }
            }
            if (c < sd.C) {
              if (sd.r_major) {
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (c0 + x < a.R) out[int64_t(c0 + x) * sd.C + c] = OT(__uint_as_float(v[x]));
              } else {
#pragma unroll
                for (int x = 0; x < 32; x += 8)
                  if (c0 + x < a.R) {
                    OT *dst = out + c * a.R + c0 + x;
                    if constexpr (sizeof(OT) == 4) {
                      *reinterpret_cast<uint4 *>(dst) = make_uint4(v[x], v[x + 1], v[x + 2], v[x + 3]);
                      *reinterpret_cast<uint4 *>(dst + 4) =
                          make_uint4(v[x + 4], v[x + 5], v[x + 6], v[x + 7]);
                    } else {
                      uint32_t w[4];
#pragma unroll
                      for (int y = 0; y < 4; ++y)
                        w[y] = uint32_t(f2bf_bits(__uint_as_float(v[x + 2 * y]))) |
                               (uint32_t(f2bf_bits(__uint_as_float(v[x + 2 * y + 1]))) << 16);
                      *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                  }
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[seg & 1]);
      s += sg.count;
    }
    // adapters without tokens: zero gradients, 16 bytes a store
    for (int i = 0; i < a.n; ++i) {
      if (a.plan.off[i] != a.plan.off[i + 1]) continue;
      for (int z = 0; z < 2; ++z) {
        const int64_t nz = int64_t(a.R) * a.side[z].C * int64_t(sizeof(OT)) / 16;
        uint4 *o = reinterpret_cast<uint4 *>(static_cast<OT *>(a.side[z].out) +
                                             int64_t(i) * a.R * a.side[z].C);
        for (int64_t x = int64_t(blockIdx.x) * 128 + e4; x < nz; x += int64_t(gridDim.x) * 128)
          o[x] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

}  // namespace dsv41
