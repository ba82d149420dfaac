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
// fp32 result.  Shrink writes the parts, in sorted order, for both consumers.  (Parts may differ in
// sign or be zero, so an infinite weight, x or dy that they meet gives NaN where one factor would give
// an infinity; both stay in the elements whose sums it enters.)
//
// k_lora_plan sorts the tokens by adapter first (a stable counting sort), so that a tile of
// 128 token rows belongs to one adapter; tokens without one come last.
#pragma once
#include "aqgemm.cuh"
#include "bsgemm.cuh"
#include "common.cuh"
#include <type_traits>

namespace dsv41 {

constexpr int LR_TILE = 128;        // token rows of a tile
constexpr int LR_KB = 64;           // contraction length of a stage

// ------------------------------------------------------------------ plan
struct LoraPlan {
  int *perm;       // [T] token of sorted position p
  int4 *tiles;     // {adapter (n: none), first position, rows, first 64-row block of the parts}
  int *head;       // [2] tiles, adapters with tokens
  int *off;        // [n + 2] first position of each adapter (n: none), then T
  int *stages;     // [n + 1] 64-row blocks of the adapters before this one: where an adapter's
                   // parts begin, and wgrad's work
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
// through global memory would take three.  6 to 8 us for 500 to 8192 tokens, a chain of latencies:
// ids, the cluster's meeting, scan, scatter.
constexpr int LP_MAX_CTAS = 8;
__global__ void __launch_bounds__(1024, 1)
    k_lora_plan(const int32_t *__restrict__ ids, int T, int n, LoraPlan p) {
  extern __shared__ int lp_smem[];                                    // [n + 1] each
  int *cnt = lp_smem, *pos = cnt + (n + 1), *tile0 = pos + (n + 1), *first = tile0 + (n + 1),
      *block0 = first + (n + 1);
  __shared__ int wsum[32][3], bin_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = gridDim.x, rank = blockIdx.x;
  pdl_trigger();
  const int per = (((T + C - 1) / C) + 1023) & ~1023;
  const int t0 = int(min(int64_t(rank) * per, int64_t(T)));
  const int t1 = int(min(int64_t(t0) + per, int64_t(T)));
  int bin_1 = t0 + tid < t1 ? lora_bin(ids[t0 + tid], n) : -1;        // of the first batch
  for (int i = tid; i <= n; i += 1024) cnt[i] = 0;
  __syncthreads();
  for (int b0 = t0; b0 < t1; b0 += 1024) {
    const int bin = b0 == t0 ? bin_1 : b0 + tid < t1 ? lora_bin(ids[b0 + tid], n) : -1;
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
      block0[b] = run[2] + v[2] - ns;
      if (rank == 0) {
        p.off[b] = first[b];
        p.stages[b] = block0[b];
        if (b == n) p.off[n + 1] = T;
      }
    }
    used += __syncthreads_count(b < n && total > 0);
    for (int i = 0; i < 3; ++i) run[i] += tot[i];
  }
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");      // histograms read
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
    p.tiles[i] = make_int4(lo, p0, min(LR_TILE, (lo == n ? T : first[lo + 1]) - p0),
                           block0[lo] + (i - tile0[lo]) * (LR_TILE / LR_KB));
  }
  // scatter: batches of 1024 tokens, their warps one after another
  for (int b0 = t0; b0 < t1; b0 += 1024) {
    const int t = b0 + tid;
    const int bin = b0 == t0 ? bin_1 : t < t1 ? lora_bin(ids[t], n) : -1;
    if (tid == 0) bin_s = bin;
    __syncthreads();
    const int bin0 = bin_s;
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
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
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
// Four rows of a [rows][columns] tensor map whose box is 128 bytes of one row, by row index: 512
// bytes, 128-byte swizzle.  A converged warp runs it, one elected lane issues.
__device__ __forceinline__ void tma_gather4_el(uint32_t dst, const CUtensorMap *map, uint64_t *bar,
                                               int32_t x, int4 rows) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z),
      "r"(rows.w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_el(uint32_t dst, const CUtensorMap *map, uint64_t *bar,
                                               int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_rows_el(uint32_t dst, const CUtensorMap *map, uint64_t *bar,
                                            int32_t x, int32_t y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// The other direction; completion by bulk groups of the elected lane (elect.sync picks the same
// lane of a full warp every time).
__device__ __forceinline__ void tma_scatter4_el(const CUtensorMap *map, uint32_t src, int32_t x,
                                                int4 rows) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.global.shared::cta.tile::scatter4.bulk_group"
      " [%0, {%1, %2, %3, %4, %5}], [%6];\n\t}" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(src)
      : "memory");
}
__device__ __forceinline__ void tma_store_rows_el(const CUtensorMap *map, uint32_t src, int32_t x,
                                                  int32_t y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\t}" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(y), "r"(src)
      : "memory");
}
__device__ __forceinline__ void bulk_commit_el() {
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
               "@e cp.async.bulk.commit_group;\n\t}" ::: "memory");
}
// every bulk store of the elected lane has read its shared memory / is complete
__device__ __forceinline__ void bulk_wait_read_el() {
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
               "@e cp.async.bulk.wait_group.read 0;\n\t}" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void bulk_wait_el() {
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
               "@e cp.async.bulk.wait_group 0;\n\t}" ::: "memory");
  __syncwarp();
}

// The 16 token rows of a group, as a warp holds them: lane l's tok is the token of row l & 15
// (missing rows repeat the last one).  Sorting is stable, so tokens ascend: the group is one run
// of rows if its last and first are as far apart as their places.
constexpr int LR_GROUP = 16;
struct LoraRows {
  CUtensorMap gather, run;     // boxes of 128 bytes of one row / of LR_GROUP rows
};
// 128 bytes of each of the group's first `rows` rows to shared memory (the rest of the group may
// be filled too): one TMA instruction for a run of rows, else one for every four.
__device__ __forceinline__ uint32_t lora_rows_bytes(bool run, int rows) {
  return run ? LR_GROUP * 128 : uint32_t((rows + 3) >> 2) * 512;
}
__device__ __forceinline__ void lora_rows_load(uint32_t dst, const LoraRows &m, uint64_t *bar, int x,
                                               int tok, bool run, int rows) {
  if (run) {
    tma_rows_el(dst, &m.run, bar, x, __shfl_sync(0xffffffffu, tok, 0));
    return;
  }
  for (int j = 0; 4 * j < rows; ++j)
    tma_gather4_el(dst + j * 512, &m.gather, bar, x,
                   make_int4(__shfl_sync(0xffffffffu, tok, 4 * j), __shfl_sync(0xffffffffu, tok, 4 * j + 1),
                             __shfl_sync(0xffffffffu, tok, 4 * j + 2),
                             __shfl_sync(0xffffffffu, tok, 4 * j + 3)));
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}
// Eight bf16 values of a row that starts anywhere (rows of a length that is no multiple of 8) to
// shared memory, zeros past `valid` of them (<= 0: nothing is read): the one or two aligned
// 16-byte words that hold them, shifted.  `end`: the tensor's end, past which no word is read.
__device__ __forceinline__ void stage8_any(uint32_t dst, const __nv_bfloat16 *src, int64_t valid,
                                           const __nv_bfloat16 *end) {
  uint4 o = make_uint4(0, 0, 0, 0);
  if (valid > 0) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(src), lo = at & ~uintptr_t(15);
    const int sh = int(at & 15) >> 1;                       // elements before src in its word
    const int n = valid < 8 ? int(valid) : 8;
    if (lo + 32 <= reinterpret_cast<uintptr_t>(end)) {
      const uint4 u = __ldg(reinterpret_cast<const uint4 *>(lo));
      const uint4 v = sh + n > 8 ? __ldg(reinterpret_cast<const uint4 *>(lo) + 1) : o;
      const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q == (sh >> 1)) {
            a = w[i + q];
            b = w[i + q + 1 < 8 ? i + q + 1 : 7];
          }
        r[i] = (sh & 1) ? __funnelshift_r(a, b, 16) : a;
        const int left = n - 2 * i;
        r[i] &= left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u;
      }
      o = make_uint4(r[0], r[1], r[2], r[3]);
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
      const uint16_t *s = reinterpret_cast<const uint16_t *>(src);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) w[e >> 1] |= uint32_t(__ldg(s + e)) << (16 * (e & 1));
      o = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  st_shared16(dst, o);
}

// A bank's matrix [rows][R] (contiguous in r) comes to shared memory in pieces of pw values of
// r, pw the largest of 64, 32, 16, 8 that divides R: rows of 2 pw bytes under the swizzle of that
// width (none for 8), which is the tensor core's canonical layout with either index contracted.
struct LoraPieces {
  uint32_t swz, rb;            // descriptor's layout type; bytes of a row of a piece
  __device__ __forceinline__ explicit LoraPieces(int pw)
      : swz(pw == 64 ? 2u : pw == 32 ? 4u : pw == 16 ? 6u : 0u), rb(uint32_t(pw) * 2) {}
  // r is not contracted (rows are), `rows` of them staged
  __device__ __forceinline__ uint64_t desc_mn(uint32_t at, uint32_t rows) const {
    return swz ? sdesc(at, rows * rb, 8 * rb, swz) : sdesc(at, 128, rows * 16, 0);
  }
  // r is contracted
  __device__ __forceinline__ uint64_t desc_k(uint32_t at, uint32_t rows) const {
    return swz ? sdesc(at, 16, 8 * rb, swz) : sdesc(at, rows * 16, 128, 0);
  }
};
// Byte offset of the k-th MMA's 16 contraction indices in a staged operand (shifts only: the
// issuing warp's address arithmetic is what an MMA of this size costs).
struct LoraSteps {
  uint32_t shift, mask, big;
  __device__ __forceinline__ LoraSteps(uint32_t sh, uint32_t b) : shift(sh), mask((1u << sh) - 1), big(b) {}
  static __device__ __forceinline__ LoraSteps mn(const LoraPieces &p) { return LoraSteps(0, 16 * p.rb); }
  static __device__ __forceinline__ LoraSteps k(const LoraPieces &p, uint32_t rows) {
    return p.swz ? LoraSteps(p.rb == 128 ? 2 : p.rb == 64 ? 1 : 0, rows * p.rb) : LoraSteps(0, rows * 32);
  }
  __device__ __forceinline__ uint32_t at(uint32_t i) const { return (i >> shift) * big + (i & mask) * 32; }
};

// v as bf16 parts; the rest after each part is exact in fp32 (and zero after an infinity or NaN).
// A finite value that would round to an infinity gets the largest bf16 and its rest.
template <int NS>
__device__ __forceinline__ void split_bf16(float v, uint16_t (&p)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    p[i] = f2bf_bits(v);
    if ((p[i] & 0x7F80) == 0x7F80 && fabsf(v) < INFINITY) p[i] -= 1;
    v = (p[i] & 0x7F80) == 0x7F80 ? 0.0f : v - bf_bits2f(p[i]);
  }
}

// The parts in memory: blocks of 64 sorted rows of one adapter (its last block padded with zero
// rows), [block][part][Rp / 8][64 rows][8]: the order in which a tensor core takes a 64-row (or,
// two blocks, 128-row) operand without swizzle, so that a block is one or a few bulk copies.
constexpr int LR_PARTS = 3;
__device__ __forceinline__ void store_parts(__nv_bfloat16 *parts, int np, int Rp, int block, int row,
                                            int c4, float4 v, float sc) {
  uint16_t p[4][LR_PARTS];
  split_bf16<LR_PARTS>(v.x * sc, p[0]);
  split_bf16<LR_PARTS>(v.y * sc, p[1]);
  split_bf16<LR_PARTS>(v.z * sc, p[2]);
  split_bf16<LR_PARTS>(v.w * sc, p[3]);
  __nv_bfloat16 *dst = parts + int64_t(block + (row >> 6)) * np * Rp * 64 + (c4 >> 3) * 512 +
                       (row & 63) * 8 + (c4 & 7);
#pragma unroll
  for (int i = 0; i < LR_PARTS; ++i)
    if (i < np)
      *reinterpret_cast<uint2 *>(dst + i * Rp * 64) = make_uint2(
          uint32_t(p[0][i]) | (uint32_t(p[1][i]) << 16),
          uint32_t(p[2][i]) | (uint32_t(p[3][i]) << 16));
}

// ------------------------------------------------------------------ shrink
struct LoraTile {
  int adapter, p0, rows, block;     // n: none; first sorted position; rows <= LR_TILE
};
struct LoraShrink {
  const __nv_bfloat16 *x;      // [T, K]
  int64_t T;
  int64_t K;                   // contraction length
  const __nv_bfloat16 *w;      // [n][R][K], or [n][K][R] (WMN)
  int R, Rp, n;                // Rp: R rounded up to 16
  const float *scaling;        // NULL: 1
  float *out;                  // [T, R] the product as it is, or NULL
  __nv_bfloat16 *parts;        // the product times scaling, np parts
  const float *h;              // [T, R] or NULL: a second value to scale and split the same way
  __nv_bfloat16 *h_parts;
  int np;
  LoraPlan plan;
  int pw;                      // WMN: see LoraPieces
};
struct LoraShrinkMaps {
  LoraRows x;
  CUtensorMap w;               // [n][R][K], box 64 k x R; WMN: [n][K][R], box pw x 64 k
};

constexpr int LS_THREADS = 160;
constexpr int LS_BATCH = 2;
constexpr int LS_X_BYTES = LR_TILE * LR_KB * 2;     // 16 KB

// D[128 tokens x Rp] in TMEM: tcgen05.mma kind::f16, M = 128, N = Rp.  A cluster of C CTAs
// takes one tile, each CTA a C-th of the contraction; the partial sums meet in distributed
// shared memory and are added in rank order.  Warps 0-3 fetch 32 token rows each, 64 values a
// stage, warp 0 also the adapter's values, all by TMA; warp 4 issues the MMAs.  (Both went
// through cp.async first: 512 bytes cost about 20 shared-memory cycles that way, which all but
// caps an SM at its share of HBM.)  T 8192, K 7168, R 32: 27 us, 4.3 TB/s, of which some 7 are the
// start behind the plan and the join.  What stands in the rows past the tile's only reaches
// accumulator rows that nobody reads.  Rows that TMA cannot address, of odd lengths, are staged
// by the threads.
template <bool WMN, bool VEC, int S>
__global__ void __launch_bounds__(LS_THREADS, 2)
    k_lora_shrink(const __grid_constant__ LoraShrinkMaps maps, const LoraShrink a) {
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
    prefetch_tmap(&maps.w);
    prefetch_tmap(&maps.x.run);
    prefetch_tmap(&maps.x.gather);
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
  pdl_wait();                             // the plan
  pdl_trigger();
  const int nkb = int((a.K + LR_KB - 1) / LR_KB);
  const int kb0 = int(int64_t(nkb) * rank / C), kb1 = int(int64_t(nkb) * (rank + 1) / C);
  const int ntiles = a.plan.head[0];
  int it = 0, done = 0;                   // stages and tiles so far (barrier parities)
  int sent = 0;                           // stages that this warp's copies were issued for
  bool ok = true;                         // no wait of this thread has run out
  for (int i = int(cluster_id_x()); i < ntiles; i += int(ncluster_x())) {
    const int4 tv = a.plan.tiles[i];
    const LoraTile tl{tv.x, tv.y, tv.z, tv.w};
    if (tl.adapter == a.n) {              // no adapter: h = 0
      if (rank == 0 && a.out)
        for (int e = tid; e < tl.rows * a.R; e += LS_THREADS)
          a.out[int64_t(a.plan.perm[tl.p0 + e / a.R]) * a.R + e % a.R] = 0.0f;
      continue;
    }
    if (tid < LR_TILE) rows_s[tid] = a.plan.perm[tl.p0 + min(tid, tl.rows - 1)];
    __syncthreads();
    if (warp < 4) {
      // ------------------------------------------------------------ producers
      int tok[2], rows[2];                           // this warp's two groups of 16 rows
      bool run[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = warp * 32 + h * LR_GROUP;
        tok[h] = rows_s[r + (lane & 15)];
        rows[h] = max(0, min(LR_GROUP, tl.rows - r));
        run[h] = rows[h] > 0 && rows_s[r + rows[h] - 1] - rows_s[r] == rows[h] - 1;
      }
      uint32_t tx = warp == 0 ? uint32_t(a.R) * 128 : 0u;
      if (VEC) tx += lora_rows_bytes(run[0], rows[0]) + lora_rows_bytes(run[1], rows[1]);
      int jt = it;
      for (int kb = kb0; kb < kb1 && ok; ++kb, ++jt) {
        const int s = jt % S;
        if (!(ok = warp_wait(&empty[s], (uint32_t(jt / S) & 1u) ^ 1u))) break;
        const uint32_t dx = sx + s * LS_X_BYTES + warp * 4096, dw = sw + s * (a.Rp * 128);
        if constexpr (!VEC) {
          const int64_t k = int64_t(kb) * LR_KB + (lane & 7) * 8;
#pragma unroll 4
          for (int j = 0; j < 8; ++j) {              // 8 lanes a row
            const int row = j * 4 + (lane >> 3);
            stage8_any(dx + row * 128 + (((lane & 7) ^ (row & 7)) << 4),
                       a.x + int64_t(rows_s[warp * 32 + row]) * a.K + k, a.K - k, a.x + a.T * a.K);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[s], tx);
        __syncwarp();
        if constexpr (VEC) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (rows[h] > 0)
              lora_rows_load(dx + h * 2048, maps.x, &full[s], kb * LR_KB, tok[h], run[h], rows[h]);
        }
        if (warp == 0) {
          if constexpr (!WMN) {
            tma_load_3d_el(dw, &maps.w, &full[s], kb * LR_KB, 0, tl.adapter);
          } else {
            for (int r = 0; r < a.R; r += a.pw)
              tma_load_3d_el(dw + r * 128, &maps.w, &full[s], r, kb * LR_KB, tl.adapter);
          }
        }
        sent = jt + 1;
      }
    } else {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t id = idesc_lora(a.Rp, 0, WMN ? 1 : 0);
      const LoraPieces pc(WMN ? a.pw : 64);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        const int jt = it + kb - kb0, s = jt % S;
        if (!warp_wait(&full[s], uint32_t(jt / S) & 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t da = sdesc_sw128(sx + s * LS_X_BYTES);
        const uint32_t bw = sw + s * (a.Rp * 128);
        const uint64_t db = WMN ? pc.desc_mn(bw, LR_KB) : sdesc_sw128(bw);
        const uint32_t step = WMN ? pc.rb : 2;        // 16 rows, or 32 bytes
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma_bf16_el(tmem, da + uint64_t(2 * k), db + uint64_t(step * k), id,
                         (kb > kb0 || k) ? 1u : 0u);
        tc_commit_el(&empty[s]);
      }
      tc_commit_el(&acc_full);            // (after a wait that ran out too: TMEM outlives the MMAs)
      __syncwarp();
    }
    it += kb1 - kb0;
    // ------------------------------------------------------------ the C partial sums: each CTA
    // adds 128 / C rows, which it reads from the others' shared memories, neighbouring lanes along
    // a row.  (Rows sent to their adder straight from TMEM, a lane a row, took 10 us at R 128.)
    float *red = reinterpret_cast<float *>(smem);
    const int ld = a.Rp + 4, own = LR_TILE / C;
    const int q4 = a.Rp >> 2;
    const float sc = a.scaling ? a.scaling[tl.adapter] : 1.0f;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    // this thread's next pieces of h, requested ahead of the waits
    float4 hv[LS_BATCH];
    auto load_h = [&](int e0) {
#pragma unroll
      for (int u = 0; u < LS_BATCH; ++u) {
        const int e = e0 + u * LS_THREADS, row = rank * own + e / q4, c4 = (e % q4) * 4;
        hv[u] = zero;
        if (a.h && e < own * q4 && c4 < a.R && row < tl.rows)
          hv[u] = __ldg(reinterpret_cast<const float4 *>(a.h + int64_t(rows_s[row]) * a.R + c4));
      }
    };
    load_h(tid);
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
#pragma unroll 1
    for (int e0 = tid; e0 < own * q4; e0 += LS_BATCH * LS_THREADS) {
      if (e0 != tid) load_h(e0);
      float4 v[LS_BATCH][8];                         // all requests in flight
#pragma unroll
      for (int u = 0; u < LS_BATCH; ++u) {
        const int e = e0 + u * LS_THREADS, row = rank * own + e / q4, c4 = (e % q4) * 4;
        const bool in = e < own * q4 && c4 < a.R && row < tl.rows;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          v[u][q] = zero;
          if (in && q < C)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[u][q].x), "=f"(v[u][q].y), "=f"(v[u][q].z), "=f"(v[u][q].w)
                         : "r"(mapa_rank(red + row * ld + c4, q))
                         : "memory");
        }
      }
#pragma unroll
      for (int u = 0; u < LS_BATCH; ++u) {
        const int e = e0 + u * LS_THREADS, row = rank * own + e / q4, c4 = (e % q4) * 4;
        if (e >= own * q4 || row >= ((tl.rows + 63) & ~63)) break;
        const bool in = c4 < a.R && row < tl.rows;   // the padding of Rp and of the block: zeros
        float4 s = zero;
#pragma unroll
        for (int q = 0; q < 8; ++q) {                // in rank order
          s.x += v[u][q].x;
          s.y += v[u][q].y;
          s.z += v[u][q].z;
          s.w += v[u][q].w;
        }
        if (a.out && in) *reinterpret_cast<float4 *>(a.out + int64_t(rows_s[row]) * a.R + c4) = s;
        // (zeros are not scaled: an infinite scaling would make them NaN)
        store_parts(a.parts, a.np, a.Rp, tl.block, row, c4, s, in ? sc : 1.0f);
        if (a.h) store_parts(a.h_parts, a.np, a.Rp, tl.block, row, c4, hv[u], in ? sc : 1.0f);
      }
    }
    cluster_sync();                       // the others have read; before the stages are written again
    fence_proxy_async_smem();
  }
  // the last copies have landed before the CTA can end, after a wait that ran out too (bounded)
  for (int e = max(0, sent - S); e < sent; ++e) warp_wait(&full[e % S], uint32_t(e / S) & 1u);
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

// Both products of a token in one launch, no plan: a cluster per token.  Each CTA takes a slice
// of K (its warps R / 8 ranks each), the partial h meet in distributed shared memory in rank
// order, then each CTA takes a slice of the columns, a row of B per group of LPR lanes.  The
// first rows of B are requested before the cluster meets.  Bound by the latency of one pass
// over an adapter (360 KB at K 7168, N 4096, R 16: 7 us for one token, 10 us for 64 where L2 holds
// the bank, 13 and 18 us where it has to be read), which tokens on the same adapter find in L2.
// TH threads; RW: ranks a warp; LPR: lanes a row of B, the power of two at or above R / 8.
template <typename OT, int TH, int RW, int LPR>
__global__ void __launch_bounds__(TH) k_lora_decode(const LoraDecode p) {
  constexpr int LD_WARPS = TH / 32;
  constexpr int COLS = TH / LPR;                    // columns a pass
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
    for (int64_t c = c0 + tid; c < c1; c += TH)
      y[c] = base ? base[t * p.N + c] : OT(0.0f);
    if (p.h && rank == 0)
      for (int r = tid; r < p.R; r += TH) p.h[t * p.R + r] = 0.0f;
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
// The MMAs of one block, NS parts (the smallest first) times KS steps: unrolled, about 42 cycles
// an MMA to issue against 75 in a loop.
template <int NS, int KS>
__device__ __forceinline__ void lora_issue(uint32_t acc, uint64_t da, uint64_t db, uint32_t id,
                                           const LoraSteps &steps, int rg) {
#pragma unroll
  for (int i = NS - 1; i >= 0; --i)
#pragma unroll
    for (int k = 0; k < KS; ++k)
      tc_mma_bf16_el(acc, da + uint64_t(uint32_t(i * rg + 2 * k) * 128),
                     db + uint64_t(steps.at(k) >> 4), id, (i < NS - 1 || k) ? 1u : 0u);
}

struct LoraExpand {
  const __nv_bfloat16 *parts;  // the parts of h times scaling (np of them)
  const __nv_bfloat16 *w;      // [n][N][R], or [n][R][N] (WMN)
  int64_t N;
  int R, Rp, n, np;
  const void *base;            // [T, N] or NULL
  void *y;                     // [T, N]
  LoraPlan plan;
  int ncb;                     // column blocks of 128 bytes of a row; an MMA takes a pair
  int ring;                    // tiles of 128 rows x 128 bytes in shared memory (of LE_GROUPS)
  int abuf, wbuf;              // buffers of the parts and of W's column blocks
  int pw;                      // !WMN: see LoraPieces
};

// The work is one line, tile after tile, a tile's pairs of column blocks in order.  The CTAs go
// along it in rounds of `turn` neighbouring pairs each; the last round shares what is left.  A
// CTA's whole share at once, far from the other CTAs', reads DRAM worse; one pair at a time reloads
// the parts for each: the square root of the share has the least of both.  (T 8192, N 14336, R 32,
// 49 pairs a CTA: 115 us the call, 141 with 1, 124 with 49; T 4096, N 7168, R 128, 13 pairs: 47, 55
// and 47 us.)  next() gives a CTA's stretches: column blocks [cb0, cb1) of one tile.
struct LoraWalk {
  int64_t work, at, end, round;
  int ncb, turn, tile, cb0, cb1;
  __device__ __forceinline__ explicit LoraWalk(const LoraExpand &a)
      : work(int64_t(a.plan.head[0]) * ((a.ncb + 1) >> 1)), at(0), end(0), round(0), ncb(a.ncb) {
    turn = max(1, int(rintf(sqrtf(float((work + gridDim.x - 1) / gridDim.x)))));
  }
  __device__ __forceinline__ bool next() {
    while (at >= end) {
      if (round >= work) return false;
      const int64_t n = min(int64_t(turn), (work - round + gridDim.x - 1) / gridDim.x);
      at = round + blockIdx.x * n;
      end = min(at + n, work);
      round += gridDim.x * n;
    }
    const int pairs = (ncb + 1) >> 1;
    tile = int(at / pairs);
    const int p = int(at - int64_t(tile) * pairs), q = int(min(int64_t(pairs), p + end - at));
    cb0 = 2 * p;
    cb1 = min(2 * q, ncb);
    at += q - p;
    return true;
  }
  __device__ __forceinline__ int pairs() const { return (cb1 - cb0 + 1) >> 1; }
};
struct LoraExpandMaps {
  LoraRows base, y;
  CUtensorMap w;               // [n][N][R], box pw x MB columns; WMN: [n][R][N], box CB columns x R
  CUtensorMap parts;           // [np Rp / 8][blocks][1 KB], box of a part's groups of two blocks
};

constexpr int LE_GROUPS = 3;                      // epilogues of four warps that take turns
constexpr int LE_THREADS = (6 + 4 * LE_GROUPS) * 32;
constexpr int LE_BUF = 4;                         // accumulators (and at most as many blocks of W)
constexpr int LE_TILE_BYTES = LR_TILE * 128;      // 16 KB
constexpr int LE_RING_MAX = 9;
constexpr int LE_EPI_LD = 36;                     // floats of a transposition row (odd rows only)

// D[128 tokens x MB columns] in TMEM (tcgen05.mma kind::f16; MB = 2 CB columns, CB are 128 bytes
// of a row of y; with CB alone the MMAs of R = 128, which read the parts from shared memory every
// time, took longer than the stores): the tile's parts are the A operand, contraction NS * Rp,
// staged once for a stretch of column blocks; a block of W is the B operand, in its own order in
// memory (rows of r for B, columns contiguous for A: the MMA takes either).  base comes in through
// a ring of 16 KB tiles, the epilogue adds the accumulators to it in place, a thread a row, and
// the tile goes out the same way (128-byte swizzle: no bank conflicts); rows that follow one
// another move 16 an instruction, others four.  Warps 0-3 fetch base, 4 issues the MMAs, 5 fetches
// W and the parts, the others are three epilogues that take turns (one's turn is about 2500 cycles
// a tile: two fell behind HBM).  Row-wise plain loads and stores, through a transposition in shared
// memory, kept the load/store pipe busy for twice the time that HBM needs (135 us at T 8192, N
// 14336, R 32, against 77 us now: 6.1 TB/s).  Rows that TMA cannot address (VEC false: odd lengths)
// are still moved that way, by a kernel of their own (in one kernel its rows pushed the hot loop
// out of the instruction cache).
template <bool WMN, typename OT, bool VEC>
__global__ void __launch_bounds__(LE_THREADS, 1)
    k_lora_expand(const __grid_constant__ LoraExpandMaps maps, const LoraExpand a) {
  constexpr int NS = sizeof(OT) == 4 ? 3 : 2;
  constexpr int CB = 128 / int(sizeof(OT)), MB = 2 * CB;       // columns of a block, of an MMA
  extern __shared__ uint8_t le_raw[];
  uint8_t *smem = le_raw + ((1024u - (smem_u32(le_raw) & 1023u)) & 1023u);
  const uint32_t w_bytes = uint32_t(MB) * a.Rp * 2;
  const uint32_t s_ring = smem_u32(smem), sw = s_ring + a.ring * LE_TILE_BYTES,
                 sa = sw + a.wbuf * w_bytes, a_bytes = uint32_t(NS) * a.Rp * 256;
  __shared__ uint64_t a_full[2], a_empty[2], w_full[LE_BUF], w_empty[LE_BUF], acc_full[LE_BUF],
      acc_empty[LE_BUF], b_full[LE_RING_MAX], b_empty[LE_RING_MAX], mma_done;
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    prefetch_tmap(&maps.w);
    prefetch_tmap(&maps.parts);
    prefetch_tmap(&maps.base.run);
    prefetch_tmap(&maps.y.run);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&a_full[i], 1);
      mbar_init(&a_empty[i], 1);
    }
    for (int i = 0; i < LE_BUF; ++i) {
      mbar_init(&w_full[i], 1);
      mbar_init(&w_empty[i], 1);
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);
    }
    for (int i = 0; i < a.ring; ++i) {
      mbar_init(&b_full[i], 4);
      mbar_init(&b_empty[i], 4);
    }
    mbar_init(&mma_done, 1);
    fence_barrier_init();
  }
  if (warp == 4) {
    tmem_alloc(&tmem_slot, LE_BUF * MB);
    tmem_relinquish();
  }
  if (a.Rp > a.R) {               // the contraction's padding: zero for good, no copy writes it
    // (WMN: in each of the two pieces of CB columns)
    constexpr int PC = WMN ? CB : MB;
    for (int e = tid; e < a.wbuf * MB; e += LE_THREADS)
      st_shared16(sw + e / MB * w_bytes + e % MB / PC * (PC * a.Rp * 2) + uint32_t(a.R) * PC * 2 +
                      e % PC * 16,
                  make_uint4(0, 0, 0, 0));
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();                             // the parts
  pdl_trigger();
  const int rg = a.Rp >> 3;
  LoraWalk st(a);
  bool ok = true;
  int blk = 0, live = 0;          // column blocks (warps 4, 5: MMA blocks of live tiles), live stretches
  if (warp < 4) {
    // -------------------------------------------------------------- base, 32 rows a warp
    if (VEC && a.base) {
      while (ok && st.next()) {
        const int4 tl = a.plan.tiles[st.tile];
        int tok[2], rows[2];
        bool run[2];
        uint32_t tx = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = warp * 32 + h * LR_GROUP;
          tok[h] = a.plan.perm[tl.y + min(r + (lane & 15), tl.z - 1)];
          rows[h] = max(0, min(LR_GROUP, tl.z - r));
          const int last = __shfl_sync(0xffffffffu, tok[h], max(0, rows[h] - 1));
          run[h] = rows[h] > 0 && last - __shfl_sync(0xffffffffu, tok[h], 0) == rows[h] - 1;
          tx += lora_rows_bytes(run[h], rows[h]);
        }
        for (int cb = st.cb0; cb < st.cb1; ++cb, ++blk) {
          const int s = blk % a.ring;
          if (!(ok = warp_wait(&b_empty[s], (uint32_t(blk / a.ring) & 1u) ^ 1u))) break;
          if (lane == 0) mbar_arrive_expect_tx(&b_full[s], tx);
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (rows[h] > 0)
              lora_rows_load(s_ring + s * LE_TILE_BYTES + warp * 4096 + h * 2048, maps.base,
                             &b_full[s], cb * CB, tok[h], run[h], rows[h]);
        }
      }
      for (int e = max(0, blk - a.ring); e < blk; ++e)
        warp_wait(&b_full[e % a.ring], uint32_t(e / a.ring) & 1u);
    }
  } else if (warp == 4) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t id = idesc_lora(MB, 0, WMN ? 1 : 0);
    const LoraPieces pc(WMN ? CB : a.pw);
    const LoraSteps steps = WMN ? LoraSteps::mn(pc) : LoraSteps::k(pc, MB);
    while (ok && st.next()) {
      if (a.plan.tiles[st.tile].x >= a.n) continue;
      const int ab = live % a.abuf;
      if (!(ok = warp_wait(&a_full[ab], uint32_t(live / a.abuf) & 1u))) break;
      ++live;
      const uint64_t da = sdesc(sa + ab * a_bytes, 2048, 128, 0);
      for (int cb = st.cb0; cb < st.cb1; cb += 2, ++blk) {
        const int b = blk % LE_BUF, wb = blk % a.wbuf;
        if (!warp_wait(&acc_empty[b], (uint32_t(blk / LE_BUF) & 1u) ^ 1u) ||
            !warp_wait(&w_full[wb], uint32_t(blk / a.wbuf) & 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t bw = sw + wb * w_bytes;
        const uint64_t db = WMN ? pc.desc_mn(bw, a.Rp) : pc.desc_k(bw, MB);
        switch (a.Rp) {
          case 16: lora_issue<NS, 1>(tmem + b * MB, da, db, id, steps, rg); break;
          case 32: lora_issue<NS, 2>(tmem + b * MB, da, db, id, steps, rg); break;
          case 64: lora_issue<NS, 4>(tmem + b * MB, da, db, id, steps, rg); break;
          case 128: lora_issue<NS, 8>(tmem + b * MB, da, db, id, steps, rg); break;
          default:
            for (int i = NS - 1; i >= 0; --i)
              for (int k = 0; k < a.Rp / 16; ++k)
                tc_mma_bf16_el(tmem + b * MB, da + uint64_t(uint32_t(i * rg + 2 * k) * 128),
                               db + uint64_t(steps.at(k) >> 4), id, (i < NS - 1 || k) ? 1u : 0u);
        }
        tc_commit_el(&w_empty[wb]);
        tc_commit_el(&acc_full[b]);
      }
      if (ok) tc_commit_el(&a_empty[ab]);
    }
    if (!ok) {                            // TMEM and the operands outlive the MMAs (bounded)
      tc_commit_el(&mma_done);
      warp_wait(&mma_done, 0);
    }
    __syncwarp();
  } else if (warp == 5) {
    // -------------------------------------------------------------- W and the parts
    while (ok && st.next()) {
      const int4 tl = a.plan.tiles[st.tile];
      if (tl.x >= a.n) continue;
      // two 64-row blocks of parts (the second may be another adapter's: its rows reach only
      // accumulator rows that nobody reads)
      const int ab = live % a.abuf;
      if (!(ok = warp_wait(&a_empty[ab], (uint32_t(live / a.abuf) & 1u) ^ 1u))) break;
      ++live;
      if (lane == 0) mbar_arrive_expect_tx(&a_full[ab], a_bytes);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < NS; ++i)
        tma_load_3d_el(sa + ab * a_bytes + i * a.Rp * 256, &maps.parts, &a_full[ab], 0, tl.w, i * rg);
      for (int cb = st.cb0; cb < st.cb1; cb += 2, ++blk) {
        const int b = blk % a.wbuf;
        if (!(ok = warp_wait(&w_empty[b], (uint32_t(blk / a.wbuf) & 1u) ^ 1u))) break;
        const uint32_t dw = sw + b * w_bytes;
        if (lane == 0) mbar_arrive_expect_tx(&w_full[b], uint32_t(MB) * a.R * 2);
        __syncwarp();
        if constexpr (WMN) {
          tma_load_3d_el(dw, &maps.w, &w_full[b], cb * CB, 0, tl.x);
          tma_load_3d_el(dw + CB * a.Rp * 2, &maps.w, &w_full[b], cb * CB + CB, 0, tl.x);
        } else {
          for (int r = 0; r < a.R; r += a.pw)
            tma_load_3d_el(dw + uint32_t(r) * MB * 2, &maps.w, &w_full[b], r, cb * CB, tl.x);
        }
      }
    }
    // the last copies have landed before the CTA can end (bounded)
    for (int e = max(0, live - a.abuf); e < live; ++e)
      warp_wait(&a_full[e % a.abuf], uint32_t(e / a.abuf) & 1u);
    for (int e = max(0, blk - a.wbuf); e < blk; ++e)
      warp_wait(&w_full[e % a.wbuf], uint32_t(e / a.wbuf) & 1u);
  } else {
    // -------------------------------------------------------------- epilogue
    const OT *base = static_cast<const OT *>(a.base);
    OT *y = static_cast<OT *>(a.y);
    const int grp = (warp - 6) >> 2, q4 = warp & 3;      // TMEM lanes 32 q4 .. + 31
    const int row = 32 * q4 + lane;                      // this thread's row of the tile
    float *tp = reinterpret_cast<float *>(smem) + (warp - 6) * 32 * LE_EPI_LD;
    int all = 0, turn = 0, prev = -1;                    // blocks so far; the tile last stored
    while (st.next()) {
      const int4 tl = a.plan.tiles[st.tile];
      const bool has = tl.x < a.n;
      const int cb0 = st.cb0, cb1 = st.cb1;
      const int tok = row < tl.z ? a.plan.perm[tl.y + row] : -1;
      for (int cb = cb0; cb < cb1; ++cb, ++all, turn = turn == LE_GROUPS - 1 ? 0 : turn + 1) {
        if (turn != grp) continue;
        const int mb = blk + ((cb - cb0) >> 1), b = mb % LE_BUF, s = all % a.ring;
        const uint32_t tacc = tmem + (uint32_t(32 * q4) << 16) + b * MB + ((cb - cb0) & 1) * CB;
        // the accumulator is free when both its halves have been read; a missing half counts too
        const bool lone = cb == cb1 - 1 && ((cb - cb0) & 1) == 0;
        if constexpr (VEC) {
          // the tile of this warp's last turn has been read: the fetch may refill it
          if (prev >= 0) {
            bulk_wait_read_el();
            if (base && lane == 0) mbar_arrive(&b_empty[prev]);
            __syncwarp();
          }
          // a warp whose wait ran out goes on without waiting
          if (base && ok) ok = warp_wait(&b_full[s], uint32_t(all / a.ring) & 1u);
        }
        // odd rows: 16 rows of 32 columns at a time, a lane a column, the first ones of base ahead
        // of the wait
        using Bits = std::conditional_t<sizeof(OT) == 4, uint32_t, uint16_t>;
        Bits odd[VEC ? 1 : 16];
        const int64_t col = int64_t(cb) * CB + lane;
        auto load_odd = [&](int64_t c, int r0) {           // (missing rows and columns read others')
          const Bits *from = reinterpret_cast<const Bits *>(base) + min(c, a.N - 1);
          const int any = __shfl_sync(0xffffffffu, tok, 0);
          if (base && any >= 0) {
#pragma unroll
            for (int r = 0; r < (VEC ? 1 : 16); ++r)
              odd[r] = from[int64_t(max(__shfl_sync(0xffffffffu, tok, r0 + r), any)) * a.N];
          }
        };
        if (!VEC) load_odd(col, 0);
        if (has) {
          if (ok) ok = warp_wait(&acc_full[b], uint32_t(mb / LE_BUF) & 1u);
          tc_fence_after();
        }
        if constexpr (VEC) {
          // (no adapter: the tile of base goes out as it came, every bit of it, or zeros)
          uint8_t *trow = smem + s * LE_TILE_BYTES + row * 128;
          if (!has && !base) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              *reinterpret_cast<uint4 *>(trow + ((k ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int h = 0; h < CB; h += 32) {
            if (!has) break;
            uint32_t v[32];
            tmem_ld32(tacc + h, v);
            if constexpr (sizeof(OT) == 4) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                float4 *at = reinterpret_cast<float4 *>(trow + ((k ^ (row & 7)) << 4));
                float4 o = base ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                o.x += __uint_as_float(v[4 * k]);
                o.y += __uint_as_float(v[4 * k + 1]);
                o.z += __uint_as_float(v[4 * k + 2]);
                o.w += __uint_as_float(v[4 * k + 3]);
                *at = o;
              }
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint4 *at = reinterpret_cast<uint4 *>(trow + (((h / 8 + k) ^ (row & 7)) << 4));
                const uint4 in = base ? *at : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {in.x, in.y, in.z, in.w};
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float lo = __uint_as_float(w[e] << 16) + __uint_as_float(v[8 * k + 2 * e]);
                  const float hi = __uint_as_float(w[e] & 0xFFFF0000u) +
                                   __uint_as_float(v[8 * k + 2 * e + 1]);
                  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
                  o[e] = *reinterpret_cast<const uint32_t *>(&p);
                }
                *at = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
          }
          if (has) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&acc_empty[b]);
              if (lone) mbar_arrive(&acc_empty[b]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) {                    // this warp's two groups of 16 rows
            const int r0 = 32 * q4 + h * LR_GROUP, rows = min(LR_GROUP, tl.z - r0);
            const uint32_t tile = s_ring + s * LE_TILE_BYTES + r0 * 128;
            const int t0 = __shfl_sync(0xffffffffu, tok, h * LR_GROUP);
            if (rows == LR_GROUP &&
                __shfl_sync(0xffffffffu, tok, h * LR_GROUP + LR_GROUP - 1) - t0 == LR_GROUP - 1) {
              tma_store_rows_el(&maps.y.run, tile, cb * CB, t0);
              continue;
            }
            for (int j = 0; 4 * j < rows; ++j) {
              const int4 r = make_int4(__shfl_sync(0xffffffffu, tok, h * LR_GROUP + 4 * j),
                                       __shfl_sync(0xffffffffu, tok, h * LR_GROUP + 4 * j + 1),
                                       __shfl_sync(0xffffffffu, tok, h * LR_GROUP + 4 * j + 2),
                                       __shfl_sync(0xffffffffu, tok, h * LR_GROUP + 4 * j + 3));
              if (4 * j + 4 <= rows) {
                tma_scatter4_el(&maps.y.gather, tile + j * 512, cb * CB, r);
              } else {
                // the tile's last one to three rows: 8 lanes a row
                const int rr = 4 * j + (lane >> 3), k = lane & 7;
                const int64_t c = int64_t(cb) * CB + k * (16 / int(sizeof(OT)));
                const int t4 = lane >> 3 == 0 ? r.x : lane >> 3 == 1 ? r.y : r.z;
                if (rr < rows && c < a.N)
                  *reinterpret_cast<uint4 *>(y + int64_t(t4) * a.N + c) =
                      *reinterpret_cast<const uint4 *>(smem + s * LE_TILE_BYTES + (r0 + rr) * 128 +
                                                       ((k ^ (rr & 7)) << 4));
              }
            }
          }
          bulk_commit_el();
          prev = s;
        } else {
          // rows that start anywhere: 32 x 32 pieces turned in shared memory.  (Loads without a
          // condition, 16 in flight, in loops that stay small: unrolled over all rows, each load
          // behind a test, T 4000, N 5884 took 172 us, now 71.)
          const int rows = min(32, tl.z - 32 * q4);
#pragma unroll 1
          for (int h = 0; h < CB; h += 32) {
            if (has) {
              uint32_t v[32];
              tmem_ld32(tacc + h, v);
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<uint4 *>(tp + lane * LE_EPI_LD + e) =
                    make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
            __syncwarp();
            const int64_t c = col + h;
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += 16) {
              float f[16];
              // (no adapter: base's bits alone, or zeros)
#pragma unroll
              for (int r = 0; r < 16; ++r) f[r] = has ? tp[(r0 + r) * LE_EPI_LD + lane] : 0.0f;
              if (base) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  const uint32_t in = odd[VEC ? 0 : r];
                  const float o = __uint_as_float(sizeof(OT) == 4 ? in : in << 16);
                  f[r] = has ? f[r] + o : o;
                }
              }
              if (r0 == 0 && rows > 16) load_odd(c, 16);
              else if (h + 32 < CB && r0 + 16 >= rows) load_odd(c + 32, 0);
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int tk = __shfl_sync(0xffffffffu, tok, r0 + r);
                const Bits raw = Bits(__float_as_uint(f[r]) >> (32 - 8 * sizeof(OT)));
                const OT o = OT(f[r]);
                if (tk >= 0 && c < a.N)
                  reinterpret_cast<Bits *>(y)[int64_t(tk) * a.N + c] =
                      has ? *reinterpret_cast<const Bits *>(&o) : raw;
              }
              if (r0 + 16 >= rows) break;
            }
            __syncwarp();
          }
          if (has) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&acc_empty[b]);
              if (lone) mbar_arrive(&acc_empty[b]);
            }
          }
        }
      }
      if (has) blk += st.pairs();
    }
    bulk_wait_el();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, LE_BUF * MB);
  }
}

// ------------------------------------------------------------------ wgrad
struct LoraGradSide {
  const __nv_bfloat16 *v;      // [T, C] long side: x (dA) or dy (dB)
  const __nv_bfloat16 *u;      // rank side, the parts of g (dA) or h (dB)
  int64_t C;
  int ncb;                     // 128-column blocks
  void *out;                   // [n, R, C] (r_major) or [n, C, R]
  int r_major;
  int vec;                     // v's rows are 16-byte aligned: TMA reads them
};
struct LoraWgrad {
  LoraGradSide side[2];
  int R, Rp, n, np;
  int64_t T;
  LoraPlan plan;
  float *part;                 // [2 * grid][R][128] partial sums
  int grid;
};
struct LoraWgradMaps {
  LoraRows v[2];               // the long sides
};

constexpr int LG_THREADS = 288;
constexpr int LG_COLS = 128;
constexpr int LG_X_BYTES = LR_KB * LG_COLS * 2;     // 16 KB: 2 pieces of [64 tokens x 128 B]
constexpr int LG_MIN_STAGES = 8;                    // a CTA's least share, see k_lora_wgrad
// Two accumulators of the MMA's N columns (at least 32: the epilogue reads 32 at a time).
__host__ __device__ __forceinline__ constexpr uint32_t lg_acc_cols(int n) {
  return n <= 32 ? 32u : n <= 64 ? 64u : n <= 128 ? 128u : 256u;
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

// How the CTAs cut the line of work: `per` stages each.  A piece is at least min(8, the average
// item's) stages: cutting a few microseconds of loads costs more in the join than it saves.
struct LoraCut {
  int64_t all, per;
  __device__ __forceinline__ explicit LoraCut(const LoraWgrad &a) {
    const int64_t stages = a.plan.stages[a.n];
    const int used = max(1, a.plan.head[1]);
    all = stages * (a.side[0].ncb + a.side[1].ncb);
    per = max((all + a.grid - 1) / a.grid, min(int64_t(LG_MIN_STAGES), (stages + used - 1) / used));
    per = max(per, int64_t(1));
  }
};

// One value per r of 32 from c0 on, for column c of the item: rounded and written
template <typename OT>
__device__ __forceinline__ void lora_wgrad_store(const LoraGradSide &sd, OT *out, int R, int64_t c,
                                                 int c0, int count, const float *v) {
  if (c >= sd.C) return;
  if (sd.r_major) {
#pragma unroll
    for (int x = 0; x < 32; ++x)
      if (x < count && c0 + x < R) out[int64_t(c0 + x) * sd.C + c] = OT(v[x]);
    return;
  }
#pragma unroll
  for (int x = 0; x < 32; x += 8)
    if (x < count && c0 + x < R) {
      OT *dst = out + c * R + c0 + x;
      if constexpr (sizeof(OT) == 4) {
        *reinterpret_cast<float4 *>(dst) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
        *reinterpret_cast<float4 *>(dst + 4) = make_float4(v[x + 4], v[x + 5], v[x + 6], v[x + 7]);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
          w[y] = uint32_t(f2bf_bits(v[x + 2 * y])) | (uint32_t(f2bf_bits(v[x + 2 * y + 1])) << 16);
        *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
}

// D[128 columns x Rp] = sum over an adapter's tokens, in TMEM; both operands have the token
// index as their rows in memory, which is the MMA's contraction index: v as 128-byte-swizzled
// pieces of 64 columns, u as unswizzled groups of 8.  u's bf16 parts stand side by side as NS Rp
// columns of one MMA where 256 columns hold them (v is then read once for all of them) and the
// epilogue adds them; else they are accumulated one after another.  The work of both gradients
// (every adapter's 64-token stages times the column blocks) is one line that the CTAs cut into
// equal pieces: an item that one CTA covers is written at once, one that a cut divides is written
// as fp32 partial sums, at most two per CTA, which k_lora_join adds in order (the last CTA to
// arrive did that first: 17 us of one CTA's time behind 41 us of work at T 8192, R 64).  Warps
// 0-3 fetch v's rows (missing ones repeat one of the adapter's own, against zero rows of u) and
// u's block, the stages dealt in turn to four of them, or to three where the ring has three stages
// (see P); 4 issues the MMAs, 5-8 read TMEM; accumulators are
// double-buffered, so an item's stores overlap the next one.  T 8192, K 7168, N 4096, R 64: 39 us,
// 4.7 TB/s (pieces of 256 bytes a row, and u once for every 128 columns), and 7 us the join.
template <typename OT, int S>
__global__ void __launch_bounds__(LG_THREADS, S == 6 || S == 3 ? 1 : 2) k_lora_wgrad(
    const __grid_constant__ LoraWgradMaps maps, const LoraWgrad a) {
  constexpr int NS = sizeof(OT) == 4 ? 3 : 2;
  // Warps that deal the stages.  A dealer goes from stage i to stage i + P, whose slot it may have
  // once stage i + P - S is released.  The wait's one-bit parity tells that release from the slot's
  // previous one, stage i + P - 2 S, only if that one is known to be over: it is, since the dealer
  // has waited for stage i - S and releases come in order, as long as P <= S.
  constexpr int P = S < 4 ? S : 4;
  static_assert(P <= S, "the parities of the ring's waits would be ambiguous");
  extern __shared__ uint8_t lg_raw[];
  uint8_t *smem = lg_raw + ((1024u - (smem_u32(lg_raw) & 1023u)) & 1023u);
  const uint32_t sx = smem_u32(smem), su = sx + S * LG_X_BYTES;
  const uint32_t u_bytes = uint32_t(a.Rp) * 128, u_stage = NS * u_bytes;   // a part, all parts
  __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2], mma_done;
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool wide = NS * a.Rp <= 256;
  const uint32_t mma_n = wide ? NS * a.Rp : a.Rp;
  const uint32_t acc_cols = lg_acc_cols(int(mma_n)), cols = 2 * acc_cols;
  if (tid == 0) {
    prefetch_tmap(&maps.v[0].run);
    prefetch_tmap(&maps.v[1].run);
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    mbar_init(&mma_done, 1);
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
  pdl_wait();                             // the parts
  pdl_trigger();
  const LoraCut cut(a);
  const int64_t w0 = min(int64_t(blockIdx.x) * cut.per, cut.all), w1 = min(w0 + cut.per, cut.all);

  if (warp < 4) {
    // -------------------------------------------------------------- producers
    int it = 0;
    bool ok = true;
    for (int64_t s = w0; s < w1 && ok;) {
      const LoraSeg sg = lora_seg(a, s, w1);
      const LoraGradSide &sd = a.side[sg.side];
      const LoraRows &map = maps.v[sg.side];
      const int p0 = a.plan.off[sg.adapter] + sg.first * LR_KB, pn = a.plan.off[sg.adapter + 1];
      // (fields of sd in registers: the copies' memory clobbers would have them read again)
      const bool vec = sd.vec != 0;
      const __nv_bfloat16 *v = sd.v, *v_end = v + a.T * sd.C;
      const int64_t C = sd.C;
      const __nv_bfloat16 *u = sd.u + int64_t(a.plan.stages[sg.adapter] + sg.first) * a.np * a.Rp * 64;
      const int c0 = sg.cb * LG_COLS;
      // every P-th stage is this warp's; its 64 rows as two tokens a lane, one turn ahead
      int q = warp < P ? (warp + P - it % P) % P : sg.count;
      int tn0 = a.plan.perm[min(p0 + q * LR_KB + lane, pn - 1)];
      int tn1 = a.plan.perm[min(p0 + q * LR_KB + 32 + lane, pn - 1)];
      for (; q < sg.count; q += P) {
        const int i = it + q, st = i % S;
        const int tok[2] = {tn0, tn1};
        tn0 = a.plan.perm[min(p0 + (q + P) * LR_KB + lane, pn - 1)];
        tn1 = a.plan.perm[min(p0 + (q + P) * LR_KB + 32 + lane, pn - 1)];
        if (!(ok = warp_wait(&empty[st], (uint32_t(i / S) & 1u) ^ 1u))) break;
        const uint32_t dv = sx + st * LG_X_BYTES;
        const int left = pn - p0 - q * LR_KB;              // rows of the adapter from here on
        if (vec) {
          if (lane == 0) mbar_arrive_expect_tx(&full[st], LG_X_BYTES + u_stage);
          __syncwarp();
          bulk_load_el(su + st * u_stage, u + int64_t(q) * a.np * a.Rp * 64, u_stage, &full[st]);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            // (only rows of the stage itself: what u's zero rows meet must be the adapter's own)
            const int tg = __shfl_sync(0xffffffffu, tok[g >> 1], (g & 1) * 16 + (lane & 15));
            const bool run = left >= (g + 1) * LR_GROUP &&
                             __shfl_sync(0xffffffffu, tg, 15) - __shfl_sync(0xffffffffu, tg, 0) == 15;
            lora_rows_load(dv + g * 2048, map, &full[st], c0, tg, run, LR_GROUP);
            lora_rows_load(dv + g * 2048 + 8192, map, &full[st], c0 + 64, tg, run, LR_GROUP);
          }
        } else {
#pragma unroll 4
          for (int j = 0; j < 32; ++j) {           // half a warp takes a row, 16 chunks
            const int row = 2 * j + (lane >> 4), k8 = lane & 15;
            const int tk = __shfl_sync(0xffffffffu, j < 16 ? tok[0] : tok[1], row & 31);
            stage8_any(dv + (k8 >> 3) * 8192 + row * 128 + (((k8 & 7) ^ (row & 7)) << 4),
                       v + int64_t(tk) * C + c0 + k8 * 8, C - c0 - k8 * 8, v_end);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(&full[st], u_stage);
          __syncwarp();
          bulk_load_el(su + st * u_stage, u + int64_t(q) * a.np * a.Rp * 64, u_stage, &full[st]);
        }
      }
      it += sg.count;
      s += sg.count;
    }
    // the last stages' copies have landed before the CTA can end (bounded)
    for (int e = max(0, it - S); e < it; ++e) warp_wait(&full[e % S], uint32_t(e / S) & 1u);
  } else if (warp == 4) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t id = idesc_lora(mma_n, 1, 1);
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
        const uint64_t du = sdesc(su + st * u_stage, 128, 1024, 0);
        if (wide) {
#pragma unroll
          for (int k = 0; k < 4; ++k)               // 16 tokens an MMA
            tc_mma_bf16_el(acc, dv + uint64_t(128 * k), du + uint64_t(16 * k), id, (q || k) ? 1u : 0u);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = NS - 1; i >= 0; --i)
              tc_mma_bf16_el(acc, dv + uint64_t(128 * k),
                             du + uint64_t(16 * k) + uint64_t(i * (u_bytes >> 4)), id,
                             (q || k || i < NS - 1) ? 1u : 0u);
        }
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
    const int e4 = tid - 160;                       // 0 .. 127
    const int col = 32 * (warp & 3) + lane;         // this thread's TMEM lane and column
    int seg = 0;
    bool ok = true;
    for (int64_t s = w0; s < w1; ++seg) {
      const LoraSeg sg = lora_seg(a, s, w1);
      const LoraGradSide &sd = a.side[sg.side];
      if (ok) ok = warp_wait(&acc_full[seg & 1], uint32_t(seg >> 1) & 1u);
      tc_fence_after();
      const uint32_t acc = tmem + uint32_t(seg & 1) * acc_cols + (uint32_t(32 * (warp & 3)) << 16);
      const bool whole = sg.count == sg.total;
      float *mine = a.part + int64_t(2 * int(blockIdx.x) + (s == w0 ? 0 : 1)) * a.R * LG_COLS + col;
      for (int c0 = 0; c0 < a.R; c0 += 32) {
        float v[32];
        if (wide) {
#pragma unroll
          for (int i = NS - 1; i >= 0; --i) {        // the smallest parts first
            uint32_t w[32];
            tmem_ld32(acc + min(i * a.Rp + c0, int(acc_cols) - 32), w);
            // (a part that ends less than 32 columns before the accumulator's end is read from
            // further left)
            const int back = max(0, i * a.Rp + c0 + 32 - int(acc_cols));
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              const uint32_t at = back == 0 ? w[x] : x + 16 < 32 ? w[x + 16] : 0u;
              v[x] = i == NS - 1 ? __uint_as_float(at) : v[x] + __uint_as_float(at);
            }
          }
        } else {
          uint32_t w[32];
          tmem_ld32(acc + c0, w);
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(w[x]);
        }
        if (whole) {
          lora_wgrad_store<OT>(sd, static_cast<OT *>(sd.out) + int64_t(sg.adapter) * a.R * sd.C, a.R,
                               int64_t(sg.cb) * LG_COLS + col, c0, 32, v);
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (c0 + x < a.R) mine[(c0 + x) * LG_COLS] = v[x];
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
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// The items that a cut divides: block x adds those that begin in CTA x's piece and end in a later
// one, eight r's a block; the partial sums in the order of the tokens.
template <typename OT>
__global__ void __launch_bounds__(LG_COLS) k_lora_join(const LoraWgrad a) {
  pdl_wait();
  const LoraCut cut(a);
  const int64_t f = blockIdx.x, end = min((f + 1) * cut.per, cut.all);
  if (f * cut.per >= end) return;
  const LoraSeg sg = lora_seg(a, end - 1, end);
  const int64_t item_end = sg.item0 + sg.total;
  if (item_end <= end || sg.item0 < f * cut.per) return;
  const int64_t l = (item_end - 1) / cut.per;
  const LoraGradSide &sd = a.side[sg.side];
  const int c0 = blockIdx.y * 8;
  float v[32] = {};
#pragma unroll 4
  for (int64_t k = f; k <= l; ++k) {
    // CTA k's piece of the item is its first one (place 0) unless the item begins inside it
    const int64_t slot = 2 * k + (k == f && sg.item0 > f * cut.per ? 1 : 0);
    const float *src = a.part + slot * a.R * LG_COLS + threadIdx.x;
    // (not __ldg: this grid starts while k_lora_wgrad still writes, so the sums are not read-only)
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] += __ldcg(src + (c0 + x) * LG_COLS);
  }
  lora_wgrad_store<OT>(sd, static_cast<OT *>(sd.out) + int64_t(sg.adapter) * a.R * sd.C, a.R,
                       int64_t(sg.cb) * LG_COLS + threadIdx.x, c0, 8, v);
}

}  // namespace dsv41
