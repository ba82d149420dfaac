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
// HBM.  All sums are fp32.  Where h or g is an operand of a bf16 tensor-core product it goes in
// as a sum of bf16 parts (v = p0 + p1 + ..., each the rounding of what the earlier ones leave):
// two parts keep 17 bits or more, below the rounding of a bf16 result, three keep all 24 for an
// fp32 result.  Shrink writes the parts, in sorted order, for both consumers.
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
  int4 *tiles;     // {adapter (n: none), first position, rows, 0}
  int *head;       // [2] tiles, adapters with tokens
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
// adapters, then the stable scatter (warps of a 1024-token batch in order).  One launch; sorting
// through global memory would take three.
constexpr int LP_MAX_CTAS = 8;
__global__ void __launch_bounds__(1024, 1)
    k_lora_plan(const int32_t *__restrict__ ids, int T, int n, LoraPlan p) {
  extern __shared__ int lp_smem[];                                    // [n + 1] each
  int *cnt = lp_smem, *pos = cnt + (n + 1), *tile0 = pos + (n + 1), *first = tile0 + (n + 1);
  __shared__ int wsum[32][3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = gridDim.x, rank = blockIdx.x;
  const int per = (((T + C - 1) / C) + 1023) & ~1023;
  const int t0 = int(min(int64_t(rank) * per, int64_t(T)));
  const int t1 = int(min(int64_t(t0) + per, int64_t(T)));
  for (int i = tid; i <= n; i += 1024) cnt[i] = 0;
  __syncthreads();
  for (int b0 = t0; b0 < t1; b0 += 1024) {
    const int bin = b0 + tid < t1 ? lora_bin(ids[b0 + tid], n) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, bin);         // runs: one add a warp
    if (bin >= 0 && lane == __ffs(same) - 1) atomicAdd(&cnt[bin], __popc(same));
  }
  cluster_sync();
  int run[3] = {0, 0, 0}, used = 0;             // tokens, tiles, stages before this batch
  for (int b0 = 0; b0 <= n; b0 += 1024) {
    const int b = b0 + tid;
    int total = 0, before = 0;
    if (b <= n) {
      int v[LP_MAX_CTAS];                       // all requests in flight at once
#pragma unroll
      for (int c = 0; c < LP_MAX_CTAS; ++c) v[c] = c < C ? ld_cluster_s32(mapa_rank(&cnt[b], c)) : 0;
#pragma unroll
      for (int c = 0; c < LP_MAX_CTAS; ++c) {
        if (c < rank) before += v[c];
        total += v[c];
      }
    }
    const int nt = (total + LR_TILE - 1) / LR_TILE, ns = (total + LR_KB - 1) / LR_KB;
    int v[3] = {total, nt, ns}, tot[3];
    block_scan3(v, tot, wsum);
    if (b <= n) {
      first[b] = run[0] + v[0] - total;
      pos[b] = first[b] + before;
      tile0[b] = run[1] + v[1] - nt;
      if (rank == 0) {
        p.off[b] = first[b];
        p.stages[b] = run[2] + v[2] - ns;
        if (b == n) p.off[n + 1] = T;
      }
    }
    used += __syncthreads_count(b < n && total > 0);
    for (int i = 0; i < 3; ++i) run[i] += tot[i];
  }
  for (int i = rank * 1024 + tid; i < p.n_tickets; i += C * 1024) p.tickets[i] = 0;
  if (rank == 0 && tid == 0) {
    p.head[0] = run[1];
    p.head[1] = used;
  }
  // tiles: the adapter by binary search over the first tiles
  for (int i = rank * 1024 + tid; i < run[1]; i += C * 1024) {
    int lo = 0, hi = n;                         // last b with tile0[b] <= i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tile0[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    const int p0 = first[lo] + (i - tile0[lo]) * LR_TILE;
    p.tiles[i] = make_int4(lo, p0, min(LR_TILE, (lo == n ? T : first[lo + 1]) - p0), 0);
  }
  // scatter: batches of 1024 tokens, their warps one after another
  for (int b0 = t0; b0 < t1; b0 += 1024) {
    const int t = b0 + tid, bin0 = lora_bin(ids[b0], n);
    const int bin = t < t1 ? lora_bin(ids[t], n) : -1;
    if (__syncthreads_and(bin < 0 || bin == bin0)) {                  // a run on one adapter
      if (bin >= 0) p.perm[pos[bin0] + tid] = t;
      __syncthreads();
      if (tid == 0) pos[bin0] += min(1024, t1 - b0);
    } else {
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
    __syncthreads();
  }
  cluster_sync();                               // the others have read this histogram
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
// the same, asking L2 for the 256 bytes around it: rows are walked 128 bytes a stage
__device__ __forceinline__ void cp_async16_256(uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(src_bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}
// This thread's part of a stage is on its way: its arrival on `full` follows its copies.  The
// MMA warp fences the proxies once it has seen the barrier.  Element stores are fenced and released
// by the thread itself.
template <bool VEC> __device__ __forceinline__ void stage_arrive(uint64_t *full) {
  if constexpr (VEC) {
    cp_async_arrive_noinc(full);
  } else {
    cp_async_wait_all();
    fence_proxy_async_smem();
    mbar_arrive(full);
  }
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}
// Items e = tid + 128 i of a [major][minor] grid, without a division an item.
struct GridWalk {
  int major, minor, dmajor, dminor, n;
  __device__ __forceinline__ GridWalk(int e, int n_minor)
      : major(e / n_minor), minor(e % n_minor), dmajor(128 / n_minor), dminor(128 % n_minor),
        n(n_minor) {}
  __device__ __forceinline__ void next() {
    major += dmajor;
    minor += dminor;
    if (minor >= n) {
      minor -= n;
      ++major;
    }
  }
};
// Eight bf16 values of a row to shared memory, zeros past `valid` of them (valid <= 0: none is
// read).  VEC: the row is 16-byte aligned and valid is 0 or >= 8 (one asynchronous copy);
// otherwise (rows of a length that is no multiple of 8) element loads.
template <bool VEC>
__device__ __forceinline__ void stage8(uint32_t dst, const __nv_bfloat16 *src, int64_t valid) {
  if constexpr (VEC) {
    cp_async16_256(dst, src, valid > 0 ? 16u : 0u);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
    const uint16_t *s = reinterpret_cast<const uint16_t *>(src);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) w[e >> 1] |= uint32_t(__ldg(s + e)) << (16 * (e & 1));
    st_shared16(dst, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// v as bf16 parts; the rest after each part is exact in fp32 (and zero after an infinity or NaN).
template <int NS>
__device__ __forceinline__ void split_bf16(float v, uint16_t (&p)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    p[i] = f2bf_bits(v);
    v = (p[i] & 0x7F80) == 0x7F80 ? 0.0f : v - bf_bits2f(p[i]);
  }
}

// Four values times sc to their parts: LR_PARTS planes of [T][Rp], `plane` apart.
constexpr int LR_PARTS = 3;
__device__ __forceinline__ void store_parts(__nv_bfloat16 *dst, int64_t plane, float4 v, float sc) {
  uint16_t p[4][LR_PARTS];
  split_bf16<LR_PARTS>(v.x * sc, p[0]);
  split_bf16<LR_PARTS>(v.y * sc, p[1]);
  split_bf16<LR_PARTS>(v.z * sc, p[2]);
  split_bf16<LR_PARTS>(v.w * sc, p[3]);
#pragma unroll
  for (int i = 0; i < LR_PARTS; ++i)
    *reinterpret_cast<uint2 *>(dst + i * plane) = make_uint2(
        uint32_t(p[0][i]) | (uint32_t(p[1][i]) << 16), uint32_t(p[2][i]) | (uint32_t(p[3][i]) << 16));
}

// ------------------------------------------------------------------ shrink
struct LoraTile {
  int adapter, p0, rows;       // n: none; first sorted position; rows <= LR_TILE
};
struct LoraShrink {
  const __nv_bfloat16 *x;      // [T, K]
  int64_t K;                   // contraction length
  const __nv_bfloat16 *w;      // [n][R][K], or [n][K][R] (WMN)
  int R, Rp, n;                // Rp: R rounded up to 16
  const float *scaling;        // NULL: 1
  float *out;                  // [T, R] the product as it is, or NULL
  __nv_bfloat16 *parts;        // [LR_PARTS][T][Rp] the product times scaling, sorted order
  const float *h;              // [T, R] or NULL: a second value to scale and split the same way
  __nv_bfloat16 *h_parts;
  int64_t plane;               // T * Rp
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
      mbar_init(&full[s], 128);
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
  const int ntiles = a.plan.head[0];
  int it = 0, done = 0;                   // stages and tiles so far (barrier parities)
  bool ok = true;                         // no wait of this thread has run out
  for (int i = int(cluster_id_x()); i < ntiles; i += int(ncluster_x())) {
    const int4 tv = a.plan.tiles[i];
    const LoraTile tl{tv.x, tv.y, tv.z};
    if (tl.adapter == a.n) {              // no adapter: h = 0
      if (rank == 0 && a.out)
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
      const GridWalk w0(tid, a.Rp >> 3);             // WMN: 8-wide groups of r, contraction rows
      const uint32_t swz = uint32_t(c ^ (r0 & 7)) << 4;
      int jt = it;
      for (int kb = kb0; kb < kb1 && ok; ++kb, ++jt) {
        const int s = jt % S;
        if (!mbar_wait(&empty[s], (uint32_t(jt / S) & 1u) ^ 1u)) {
          ok = false;
          break;
        }
        const int64_t k = int64_t(kb) * LR_KB + c * 8;
        const uint32_t dx = sx + s * LS_X_BYTES + r0 * 128 + swz;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          stage8<VEC>(dx + j * 2048, tok[j] < 0 ? a.x : a.x + int64_t(tok[j]) * a.K + k,
                      tok[j] < 0 ? 0 : a.K - k);
        const uint32_t dw = sw + s * a.w_bytes;
        if constexpr (!WMN) {
          for (int r = r0; r < a.Rp; r += 16)
            cp_async16(dw + r * 128 + swz, r < a.R && k < a.K ? wi + r * a.K + k : wi,
                       r < a.R && k < a.K ? 16u : 0u);
        } else {
          const __nv_bfloat16 *wk = wi + int64_t(kb) * LR_KB * a.R;
          const int rows = int(min(int64_t(LR_KB), a.K - int64_t(kb) * LR_KB));
#pragma unroll 4
          for (GridWalk w = w0; w.major < LR_KB; w.next()) {
            const bool in = w.minor * 8 < a.R && w.major < rows;
            cp_async16(dw + w.minor * LS_MN_LD + w.major * 16,
                       in ? wk + w.major * a.R + w.minor * 8 : wi, in ? 16u : 0u);
          }
        }
        stage_arrive<VEC>(&full[s]);
      }
    } else {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t id = idesc_lora(a.Rp, 0, WMN ? 1 : 0);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        const int jt = it + kb - kb0, s = jt % S;
        if (!warp_wait(&full[s], uint32_t(jt / S) & 1u)) {
          ok = false;
          break;
        }
        fence_proxy_async_smem();
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
    const int q4 = a.Rp >> 2, row_a = LR_TILE * rank / C, row_b = LR_TILE * (rank + 1) / C;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int e = tid; e < (row_b - row_a) * q4; e += LS_THREADS) {
      const int row = row_a + e / q4, c4 = (e % q4) * 4;
      if (row >= tl.rows) break;
      const bool in = c4 < a.R;                    // the padding of Rp: zeros
      const int64_t tok = rows_s[row], at = int64_t(tl.p0 + row) * a.Rp + c4;
      float4 v[8], s = zero;                       // all requests in flight, added in rank order
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        v[q] = zero;
        if (in && q < C)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[q].x), "=f"(v[q].y), "=f"(v[q].z), "=f"(v[q].w)
                       : "r"(mapa_rank(red + row * ld + c4, q))
                       : "memory");
      }
      const float4 h = in && a.h ? __ldg(reinterpret_cast<const float4 *>(a.h + tok * a.R + c4)) : zero;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        s.x += v[q].x;
        s.y += v[q].y;
        s.z += v[q].z;
        s.w += v[q].w;
      }
      if (a.out && in) *reinterpret_cast<float4 *>(a.out + tok * a.R + c4) = s;
      store_parts(a.parts + at, a.plane, s, sc);
      if (a.h) store_parts(a.h_parts + at, a.plane, h, sc);
    }
    cluster_sync();                       // before the stages are written again
  }
  cp_async_wait_all();
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
  const __nv_bfloat16 *parts;  // [LR_PARTS][T][Rp] h times scaling, sorted order
  int64_t plane;
  const __nv_bfloat16 *w;      // [n][N][R], or [n][R][N] (WMN)
  int64_t N;
  int R, Rp, n;
  const void *base;            // [T, N] or NULL
  void *y;                     // [T, N]
  LoraPlan plan;
  int ncb, cpu;                // 128-column blocks, and how many of them a work item takes
  int vec;                     // rows of base and y are 16-byte aligned
  uint32_t a_bytes, w_bytes;   // staged bytes of the parts and of a column block of W
};

constexpr int LE_COLS = 128;
constexpr int LE_THREADS = 13 * 32;
constexpr int LE_LD = 128 * 16 + 16;              // bytes between 8-wide k groups of 128 rows
constexpr int LE_EPI_LD = 36;                     // floats of a transposition row
constexpr int LE_EPI_BYTES = 8 * 32 * LE_EPI_LD * 4;

// D[128 tokens x 128 columns] in TMEM (tcgen05.mma kind::f16, double-buffered): the tile's
// parts are the A operand, contraction NS * Rp, staged once for a work item's column blocks; a
// block of W is the B operand, double-buffered, in its own order in memory (rows of r for B,
// columns contiguous for A: the MMA takes either).  Warps 0-3 stage, 4 issues the MMAs, 5-12
// read TMEM, turn 32 x 32 pieces through shared memory and move base and y in 64- or 128-byte
// pieces of a row.  mma.sync with its accumulators stored straight from registers took 185 us
// at T 8192, N 14336, R 32 (two CTAs an SM at 122 registers, too few loads in flight).
template <bool WMN, typename OT>
__global__ void __launch_bounds__(LE_THREADS, 2) k_lora_expand(const LoraExpand a) {
  constexpr int NS = sizeof(OT) == 4 ? 3 : 2;
  extern __shared__ __align__(128) uint8_t le_smem[];
  const uint32_t sa = smem_u32(le_smem), sw = sa + a.a_bytes;
  float *epi = reinterpret_cast<float *>(le_smem + a.a_bytes + 2 * a.w_bytes);
  __shared__ uint64_t a_empty, w_full[2], w_empty[2], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&a_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&w_full[i], 128);
      mbar_init(&w_empty[i], 1);
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);
    }
    fence_barrier_init();
  }
  if (warp == 4) {
    tmem_alloc(&tmem_slot, 2 * LE_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int per_tile = (a.ncb + a.cpu - 1) / a.cpu, rg = a.Rp >> 3;
  const int64_t items = int64_t(a.plan.head[0]) * per_tile;
  bool ok = true;
  int blk = 0, live = 0;                          // column blocks and live items so far
  if (warp < 4) {
    // -------------------------------------------------------------- staging
    const GridWalk w0(tid, rg);
    for (int64_t item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const int4 tl = a.plan.tiles[item / per_tile];
      if (tl.x >= a.n) continue;
      const int cb0 = int(item % per_tile) * a.cpu, cb1 = min(cb0 + a.cpu, a.ncb);
      const __nv_bfloat16 *wi = a.w + int64_t(tl.x) * a.R * a.N;
      if (!(ok = mbar_wait(&a_empty, (uint32_t(live) & 1u) ^ 1u))) break;
      ++live;
      const __nv_bfloat16 *pt = a.parts + int64_t(tl.y) * a.Rp;
#pragma unroll 2
      for (GridWalk w = w0; w.major < LR_TILE; w.next()) {
        const bool in = w.major < tl.z;
        const __nv_bfloat16 *src = in ? pt + w.major * a.Rp + w.minor * 8 : a.parts;
#pragma unroll
        for (int i = 0; i < NS; ++i)
          cp_async16(sa + uint32_t(i * rg + w.minor) * LE_LD + w.major * 16,
                     src + (in ? i * a.plane : 0), in ? 16u : 0u);
      }
      for (int cb = cb0; cb < cb1 && ok; ++cb, ++blk) {
        const int b = blk & 1;
        if (!(ok = mbar_wait(&w_empty[b], (uint32_t(blk >> 1) & 1u) ^ 1u))) break;
        const int64_t c0 = int64_t(cb) * LE_COLS;
        const uint32_t dw = sw + b * a.w_bytes;
        if constexpr (!WMN) {
          const __nv_bfloat16 *wc = wi + c0 * a.R;
          const int n_cols = int(min(int64_t(LE_COLS), a.N - c0));
#pragma unroll 4
          for (GridWalk w = w0; w.major < LE_COLS; w.next()) {
            const bool in = w.major < n_cols && w.minor * 8 < a.R;
            cp_async16(dw + uint32_t(w.minor) * LE_LD + w.major * 16,
                       in ? wc + w.major * a.R + w.minor * 8 : wi, in ? 16u : 0u);
          }
        } else {
          const int g = tid & 15;                  // 8 columns; rows r = tid / 16 + 8 i
          const bool cin = c0 + g * 8 < a.N;
          const __nv_bfloat16 *wc = wi + c0 + g * 8;
          const uint32_t dg = dw + uint32_t(g) * (a.Rp * 16 + 16);
#pragma unroll 4
          for (int r = tid >> 4; r < a.Rp; r += 8) {
            const bool in = cin && r < a.R;
            cp_async16(dg + r * 16, in ? wc + int64_t(r) * a.N : wi, in ? 16u : 0u);
          }
        }
        stage_arrive<true>(&w_full[b]);
      }
    }
    cp_async_wait_all();
  } else if (warp == 4) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t id = idesc_lora(LE_COLS, 0, WMN ? 1 : 0);
    for (int64_t item = blockIdx.x; item < items && ok; item += gridDim.x) {
      if (a.plan.tiles[item / per_tile].x >= a.n) continue;
      const int cb0 = int(item % per_tile) * a.cpu, cb1 = min(cb0 + a.cpu, a.ncb);
      for (int cb = cb0; cb < cb1; ++cb, ++blk) {
        const int b = blk & 1;
        const uint32_t ph = uint32_t(blk >> 1) & 1u;
        if (!warp_wait(&acc_empty[b], ph ^ 1u) || !warp_wait(&w_full[b], ph)) {
          ok = false;
          break;
        }
        fence_proxy_async_smem();
        tc_fence_after();
        const uint64_t da = sdesc(sa, LE_LD, 128, 0);
        const uint32_t bw = sw + b * a.w_bytes;
        const uint64_t db = WMN ? sdesc(bw, 128, a.Rp * 16 + 16, 0) : sdesc(bw, LE_LD, 128, 0);
        const uint32_t bstep = WMN ? 256 : 2 * LE_LD;            // 16 contraction indices
        for (int i = NS - 1; i >= 0; --i)                        // the smallest parts first
          for (int k = 0; k < a.Rp / 16; ++k)
            tc_mma_bf16_el(tmem + b * LE_COLS,
                           da + uint64_t(uint32_t(i * rg + 2 * k) * (LE_LD >> 4)),
                           db + uint64_t(k * (bstep >> 4)), id, (i < NS - 1 || k) ? 1u : 0u);
        tc_commit_el(&w_empty[b]);
        tc_commit_el(&acc_full[b]);
      }
      if (ok) tc_commit_el(&a_empty);
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- epilogue
    const OT *base = static_cast<const OT *>(a.base);
    OT *y = static_cast<OT *>(a.y);
    const int w8 = warp - 5, q4 = warp & 3, half = w8 >> 2;     // TMEM lanes 32 q4 .., 64 columns
    float *tp = epi + w8 * 32 * LE_EPI_LD;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
      const int4 tl = a.plan.tiles[item / per_tile];
      const bool has = tl.x < a.n;
      const int cb0 = int(item % per_tile) * a.cpu, cb1 = min(cb0 + a.cpu, a.ncb);
      // vec: rows 32 q4 + 8 j + lane / 4; else the tokens of all 32 rows, a lane each
      int tok[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 32 * q4 + 8 * j + (lane >> 2);
        tok[j] = row < tl.z ? a.plan.perm[tl.y + row] : -1;
      }
      const int row_l = 32 * q4 + lane;
      const int tok_l = row_l < tl.z ? a.plan.perm[tl.y + row_l] : -1;
      for (int cb = cb0; cb < cb1; ++cb) {
        const int b = blk & 1;
#pragma unroll 1
        for (int ch = 0; ch < 2; ++ch) {
          const int64_t c0 = int64_t(cb) * LE_COLS + half * 64 + ch * 32;
          const int64_t c = c0 + (lane & 3) * 8;
          uint4 in[4][sizeof(OT) / 2];
          if (a.vec && base && c < a.N) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (tok[j] >= 0) {
                const uint4 *src = reinterpret_cast<const uint4 *>(base + int64_t(tok[j]) * a.N + c);
#pragma unroll
                for (int u = 0; u < int(sizeof(OT) / 2); ++u) in[j][u] = src[u];
              }
          }
          if (has && ch == 0) {
            // a warp whose wait ran out goes on without waiting
            if (ok) ok = warp_wait(&acc_full[b], uint32_t(blk >> 1) & 1u);
            tc_fence_after();
          }
          if (has) {
            uint32_t v[32];
            tmem_ld32(tmem + (uint32_t(32 * q4) << 16) + b * LE_COLS + half * 64 + ch * 32, v);
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4 *>(tp + lane * LE_EPI_LD + e) =
                  make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            __syncwarp();
          }
          if (a.vec) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
              if (has) {
                const float4 *src = reinterpret_cast<const float4 *>(
                    tp + (8 * j + (lane >> 2)) * LE_EPI_LD + (lane & 3) * 8);
                const float4 v0 = src[0], v1 = src[1];
                f[0] = v0.x; f[1] = v0.y; f[2] = v0.z; f[3] = v0.w;
                f[4] = v1.x; f[5] = v1.y; f[6] = v1.z; f[7] = v1.w;
              }
              if (tok[j] < 0 || c >= a.N) continue;
              uint4 *dst = reinterpret_cast<uint4 *>(y + int64_t(tok[j]) * a.N + c);
              if constexpr (sizeof(OT) == 4) {
                if (base) {
                  const uint32_t *s = reinterpret_cast<const uint32_t *>(in[j]);
#pragma unroll
                  for (int e = 0; e < 8; ++e) f[e] += __uint_as_float(s[e]);
                }
                dst[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]),
                                    __float_as_uint(f[2]), __float_as_uint(f[3]));
                dst[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]),
                                    __float_as_uint(f[6]), __float_as_uint(f[7]));
              } else {
                const uint32_t s[4] = {in[j][0].x, in[j][0].y, in[j][0].z, in[j][0].w};
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if (base) {
                    f[2 * e] += bf_bits2f(uint16_t(s[e]));
                    f[2 * e + 1] += bf_bits2f(uint16_t(s[e] >> 16));
                  }
                  o[e] = uint32_t(f2bf_bits(f[2 * e])) | (uint32_t(f2bf_bits(f[2 * e + 1])) << 16);
                }
                dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
          } else {
            // rows that start anywhere: a row a step, a lane per column
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
              const int tk = __shfl_sync(0xffffffffu, tok_l, r);
              if (tk < 0 || c0 + lane >= a.N) continue;
              const int64_t at = int64_t(tk) * a.N + c0 + lane;
              float f = has ? tp[r * LE_EPI_LD + lane] : 0.0f;
              if (base) f += float(base[at]);
              y[at] = OT(f);
            }
          }
          __syncwarp();
        }
        if (has) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[b]);
          ++blk;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * LE_COLS);
  }
}

// ------------------------------------------------------------------ wgrad
struct LoraGradSide {
  const __nv_bfloat16 *v;      // [T, C] long side: x (dA) or dy (dB)
  const __nv_bfloat16 *u;      // [LR_PARTS][T][Rp] rank side, sorted: g (dA) or h (dB), scaled
  int64_t C;
  int ncb;                     // 128-column blocks
  void *out;                   // [n, R, C] (r_major) or [n, C, R]
  int r_major;
  int vec;                     // v's rows are 16-byte aligned
};
struct LoraWgrad {
  LoraGradSide side[2];
  int R, Rp, n;
  int64_t plane;               // T * Rp
  LoraPlan plan;
  float *part;                 // [2 * grid][Rp][128] partial sums
  uint32_t u_bytes;            // one bf16 part of a stage of u: (Rp / 8) * LG_MN_LD
};

constexpr int LG_THREADS = 416;
constexpr int LG_COLS = 128;
constexpr int LG_X_BYTES = LR_KB * LG_COLS * 2;     // 16 KB: 2 pieces of [64 tokens x 128 B]
constexpr int LG_MIN_STAGES = 8;                    // a CTA's least share, see k_lora_wgrad
constexpr int LG_MN_LD = LR_KB * 16 + 16;
__host__ __device__ __forceinline__ constexpr uint32_t lg_tmem_cols(int Rp) {
  return Rp <= 32 ? 64u : Rp <= 64 ? 128u : 256u;   // two accumulators
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

// D[128 columns x Rp] = sum over an adapter's tokens, in TMEM; both operands have the token
// index as their rows in memory, which is the MMA's contraction index: v as 128-byte-swizzled
// pieces of 64 columns, u (its bf16 parts) as unswizzled groups of 8.  The work of both
// gradients (every adapter's 64-token stages times the column blocks) is one line that the CTAs
// cut into equal pieces: an item that one CTA covers is written at once, one that a cut divides
// is written as fp32 partial sums (at most two per CTA) and the last CTA to arrive adds them in
// order.  A piece is at least min(8, the average item's) stages: cutting a few microseconds of
// loads costs more in the join than it saves.  Warps 0-3 copy v, 4-7 u, 8 issues the MMAs, 9-12
// read TMEM; accumulators are double-buffered, so an item's stores overlap the next one.
template <typename OT, int S>
__global__ void __launch_bounds__(LG_THREADS, S == 6 || S == 3 ? 1 : 2) k_lora_wgrad(const LoraWgrad a) {
  constexpr int NS = sizeof(OT) == 4 ? 3 : 2;
  extern __shared__ uint8_t lg_raw[];
  uint8_t *smem = lg_raw + ((1024u - (smem_u32(lg_raw) & 1023u)) & 1023u);
  const uint32_t sx = smem_u32(smem), su = sx + S * LG_X_BYTES;
  const uint32_t u_stage = NS * a.u_bytes;
  __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2], mma_done;
  __shared__ uint32_t tmem_slot;
  __shared__ int last_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t cols = lg_tmem_cols(a.Rp), acc_cols = cols / 2;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 256);
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
  const int64_t stages = a.plan.stages[a.n], all = stages * (a.side[0].ncb + a.side[1].ncb);
  const int used = max(1, a.plan.head[1]);
  const int64_t per = max((all + gridDim.x - 1) / gridDim.x,
                          min(int64_t(LG_MIN_STAGES), (stages + used - 1) / used));
  const int64_t w0 = min(int64_t(blockIdx.x) * per, all), w1 = min(w0 + per, all);

  if (warp < 8) {
    // -------------------------------------------------------------- producers
    int it = 0;
    bool ok = true;
    for (int64_t s = w0; s < w1 && ok;) {
      const LoraSeg sg = lora_seg(a, s, w1);
      const LoraGradSide &sd = a.side[sg.side];
      const int p0 = a.plan.off[sg.adapter] + sg.first * LR_KB, pn = a.plan.off[sg.adapter + 1];
      if (warp < 4) {
        // 64 rows x 16 chunks of 16 bytes: a warp's half takes a row, 8 steps for its 16 rows
        // (fields of sd in registers: the copies' memory clobbers would have them read again)
        const int64_t c = int64_t(sg.cb) * LG_COLS + (lane & 15) * 8, C = sd.C;
        const bool cin = c < C, vec = sd.vec != 0;
        const __nv_bfloat16 *v0 = sd.v, *vc = v0 + c;
        const uint32_t d0 = sx + ((lane & 15) >> 3) * 8192 + (warp * 16 + (lane >> 4)) * 128;
        const int r16 = warp * 16 + (lane & 15);
        int tok_n = p0 + r16 < pn ? a.plan.perm[p0 + r16] : -1;    // one stage ahead
        for (int q = 0; q < sg.count; ++q, ++it) {
          const int st = it % S;
          const int tok_l = tok_n, nx = p0 + (q + 1) * LR_KB + r16;
          tok_n = q + 1 < sg.count && nx < pn ? a.plan.perm[nx] : -1;
          if (!(ok = mbar_wait(&empty[st], (uint32_t(it / S) & 1u) ^ 1u))) break;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int row8 = (2 * j + (lane >> 4)) & 7;
            const int tok = __shfl_sync(0xffffffffu, tok_l, 2 * j + (lane >> 4));
            const uint32_t d = d0 + st * LG_X_BYTES + j * 256 + (((lane & 7) ^ row8) << 4);
            const bool in = tok >= 0 && cin;
            const __nv_bfloat16 *src = in ? vc + int64_t(tok) * C : v0;
            if (vec) stage8<true>(d, src, in ? 8 : 0);
            else stage8<false>(d, src, in ? C - c : 0);
          }
          if (vec) stage_arrive<true>(&full[st]);
          else stage_arrive<false>(&full[st]);
        }
      } else {
        const GridWalk u0(tid - 128, a.Rp >> 3);
        const __nv_bfloat16 *ub = sd.u;
        for (int q = 0; q < sg.count; ++q, ++it) {
          const int st = it % S;
          if (!(ok = mbar_wait(&empty[st], (uint32_t(it / S) & 1u) ^ 1u))) break;
          const int pos = p0 + q * LR_KB;
          const __nv_bfloat16 *up = ub + int64_t(pos) * a.Rp;
#pragma unroll 4
          for (GridWalk w = u0; w.major < LR_KB; w.next()) {
            const bool in = pos + w.major < pn;
            const __nv_bfloat16 *src = in ? up + w.major * a.Rp + w.minor * 8 : ub;
            const uint32_t d = su + st * u_stage + w.minor * LG_MN_LD + w.major * 16;
#pragma unroll
            for (int i = 0; i < NS; ++i)
              cp_async16(d + i * a.u_bytes, src + (in ? i * a.plane : 0), in ? 16u : 0u);
          }
          stage_arrive<true>(&full[st]);
        }
      }
      s += sg.count;
    }
    cp_async_wait_all();
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
        fence_proxy_async_smem();
        tc_fence_after();
        const uint64_t dv = sdesc(sx + st * LG_X_BYTES, 8192, 1024, 2);
        const uint64_t du = sdesc(su + st * u_stage, 128, LG_MN_LD, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k)                 // 16 tokens an MMA
#pragma unroll
          for (int i = 0; i < NS; ++i)
            tc_mma_bf16_el(acc, dv + uint64_t(128 * k),
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
    const int col = 32 * (warp & 3) + lane;         // this thread's TMEM lane and column
    int seg = 0;
    bool ok = true;
    for (int64_t s = w0; s < w1; ++seg) {
      const LoraSeg sg = lora_seg(a, s, w1);
      const LoraGradSide &sd = a.side[sg.side];
      // a warp whose wait ran out goes on without waiting: the others meet it at the barriers
      if (ok) ok = warp_wait(&acc_full[seg & 1], uint32_t(seg >> 1) & 1u);
      tc_fence_after();
      const uint32_t acc = tmem + uint32_t(seg & 1) * acc_cols + (uint32_t(32 * (warp & 3)) << 16);
      const int64_t f = sg.item0 / per, l = (sg.item0 + sg.total - 1) / per;   // CTAs of the item
      OT *out = static_cast<OT *>(sd.out) + int64_t(sg.adapter) * a.R * sd.C;
      bool join = f == l;
      if (f != l) {
        float *mine = a.part + int64_t(2 * int(blockIdx.x) + (s == w0 ? 0 : 1)) * a.Rp * LG_COLS;
        for (int c0 = 0; c0 < a.Rp; c0 += 32) {
          uint32_t v[32];
          tmem_ld32(acc + c0, v);
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (c0 + x < a.R) __stcg(mine + (c0 + x) * LG_COLS + col, __uint_as_float(v[x]));
        }
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (e4 == 0) last_s = atomicAdd(a.plan.tickets + f, 1) == int(l - f);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        join = last_s != 0;
        if (join) __threadfence();
      }
      if (join) {
        const int64_t c = int64_t(sg.cb) * LG_COLS + col;
        for (int c0 = 0; c0 < a.Rp; c0 += 32) {
          uint32_t v[32];
          if (f == l) {
            tmem_ld32(acc + c0, v);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) v[x] = 0u;
#pragma unroll 2
            for (int64_t k = f; k <= l; ++k) {
              const int sl = 2 * int(k) + (k == f && sg.item0 > f * per ? 1 : 0);
              const float *src = a.part + int64_t(sl) * a.Rp * LG_COLS + col;
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
