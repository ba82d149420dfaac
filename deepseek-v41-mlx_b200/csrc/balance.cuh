// balance.cuh -- the router's training pass: per-sequence balance loss, per-expert counts, and
// the gradient of that loss and of the routing weights to the router's logits.
//
// With z the logits of a token, s = f(z / temp) the router's scores (router.cuh), Z = sum_e s_e
// + 1e-20, p = s / Z, c_e the number of times expert e was chosen in the token's sequence and m
// the sequence's live tokens (k choices each):
//   loss_q = sum_e f_e P_e,  f_e = E c_e / (k m),  P_e = sum_t p_te / m
//          = E / (k m^2) sum_t sum_e c_e p_te                        (c is held constant)
//   dloss_q / ds_te = E / (k m^2) (c_e - sum_j c_j p_tj) / Z
// and the routing weights w_j = s_ij / (sum_l s_il + 1e-20) * scale (normalised when k > 1) give
//   ds_ij += scale / (sum_l s_il + 1e-20) (dw_j - sum_l dw_l w_l / scale).
// The counts come first (they need the choices alone); then sum_e c_e p_te serves the loss and
// the gradient alike, so one pass over the logits gives both: each row is read once and, with a
// gradient, written once, and the bound is HBM.  Sums over a sequence's tokens are doubles.
#pragma once
#include "bsgemm.cuh"
#include "common.cuh"

namespace dsv41 {

constexpr int BL_WARPS = 8;             // warps of a CTA, a token each at a time
constexpr int BL_SMALL_INTS = 12288;    // shared-memory counters (S * E) of the one-launch form
constexpr int BL_COUNT_INTS = 28672;    // and of the counting cluster

struct BalArgs {
  const void *logits;          // [T, E] fp32 or bf16
  int64_t T;
  int E, topk, S, func;
  const int32_t *indices, *offsets;
  const uint8_t *mask;
  float inv_temp;
  const float *grad_loss, *dweights;
  int norm;
  float route_scale;
  float *loss;
  int32_t *counts;
  void *dlogits;
  int *live;                   // [S] live tokens (and one ticket behind them)
  double *part;                // [runs + S] sum of c . p over a run's tokens of one sequence
  int run;                     // tokens of a run: a warp's contiguous tokens
};

// The sequence of token t, the last q with offsets[q] <= t < offsets[q + 1], or -1; [a, b) the
// tokens up to the next change.
struct BalSeq {
  int q;
  int64_t a, b;
};
__device__ __forceinline__ BalSeq balance_seq(const BalArgs &p, int64_t t) {
  if (!p.offsets) return BalSeq{0, 0, p.T};
  int lo = 0, hi = p.S + 1;            // first i with offsets[i] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.offsets + mid) > t) hi = mid;
    else lo = mid + 1;
  }
  const int64_t a = lo > 0 ? __ldg(p.offsets + lo - 1) : 0;
  const int64_t b = lo <= p.S ? __ldg(p.offsets + lo) : p.T;
  return BalSeq{lo == 0 || lo > p.S ? -1 : lo - 1, a, b < p.T ? b : p.T};
}

// e^x to about 2 units in the last place: the rounding of x log2(e) is carried along.
__device__ __forceinline__ float exp_acc(float x) {
  const float hi = x * 1.44269504f;
  const float lo = fmaf(x, 1.44269504f, -hi) + x * 1.92596300e-8f;   // log2(e) - float(log2(e))
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(hi));
  return x < -150.0f ? 0.0f : fmaf(e, lo * 0.693147181f, e);     // lo is NaN for x = -inf
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// sqrt(softplus(z)) and its derivative sigmoid(z) / (2 s).  softplus = max(z, 0) + log1p(u), u =
// e^-|z| in (0, 1], with log1p(u) / u by a Chebyshev interpolant of degree 8 (relative error
// 2e-7): the library's log1pf, sqrtf and divisions would bound the pass by issue slots (448 us
// at T = 65536, E = 384 in the one-thread-a-value form against 31 us of HBM time).
__device__ __forceinline__ void score_sqrtsoftplus(float z, float &s, float &ds) {
  const float u = exp_acc(-fabsf(z));
  float p = 5.126101896e-3f;
  p = fmaf(p, u, -2.907406539e-2f);
  p = fmaf(p, u, 7.751608640e-2f);
  p = fmaf(p, u, -1.360224783e-1f);
  p = fmaf(p, u, 1.907688081e-1f);
  p = fmaf(p, u, -2.483539879e-1f);
  p = fmaf(p, u, 3.331812024e-1f);
  p = fmaf(p, u, -4.999944568e-1f);
  p = fmaf(p, u, 9.999999404e-1f);
  const float sp = fmaf(p, u, fmaxf(z, 0.0f));
  const float r = rsqrt_approx(sp), d = rcp_approx(1.0f + u);
  s = sp * r;
  ds = 0.5f * r * (z < 0.0f ? u * d : d);
  if (z < -80.0f) {                    // softplus(z) = e^z leaves fp32's normal range
    s = exp_acc(0.5f * z);
    ds = 0.5f * s;
  }
}
// 1 - s from the same exponential: s (1 - s) = u / (1 + u)^2 keeps its digits at both ends.
__device__ __forceinline__ void score_sigmoid(float z, float &s, float &ds) {
  const float u = exp_acc(-fabsf(z)), d = rcp_approx(1.0f + u);
  s = z < 0.0f ? u * d : d;
  ds = u * d * d;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float bal_ld(const float *p) { return __ldg(p); }
__device__ __forceinline__ float bal_ld(const __nv_bfloat16 *p) {
  return bf_bits2f(__ldg(reinterpret_cast<const uint16_t *>(p)));
}

// A row's values as lane l holds them: VEC = 4: elements 4 (32 j + l) + v (E % 4 == 0, aligned
// rows); VEC = 1: elements 32 j + l.
template <typename IT, int NV, int VEC> struct BalRow;
template <int NV> struct BalRow<float, NV, 4> {
  float4 r[NV];
  __device__ __forceinline__ void load(const float *row, int E, int lane) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (4 * (32 * j + lane) < E) r[j] = __ldg(reinterpret_cast<const float4 *>(row) + 32 * j + lane);
  }
  __device__ __forceinline__ float at(int j, int v) const { return (&r[j].x)[v]; }
};
template <int NV> struct BalRow<__nv_bfloat16, NV, 4> {
  uint2 r[NV];
  __device__ __forceinline__ void load(const __nv_bfloat16 *row, int E, int lane) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (4 * (32 * j + lane) < E) r[j] = __ldg(reinterpret_cast<const uint2 *>(row) + 32 * j + lane);
  }
  __device__ __forceinline__ float at(int j, int v) const {
    const uint32_t w = v < 2 ? r[j].x : r[j].y;
    return bf_bits2f(uint16_t(v & 1 ? w >> 16 : w));
  }
};
template <typename IT, int NV> struct BalRow<IT, NV, 1> {
  float r[NV];
  __device__ __forceinline__ void load(const IT *row, int E, int lane) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (32 * j + lane < E) r[j] = bal_ld(row + 32 * j + lane);
  }
  __device__ __forceinline__ float at(int j, int) const { return r[j]; }
};

template <typename IT, int VEC>
__device__ __forceinline__ void bal_store(IT *row, int j, int lane, const float *v) {
  if constexpr (VEC == 1) {
    row[32 * j + lane] = IT(v[0]);
  } else if constexpr (sizeof(IT) == 4) {
    reinterpret_cast<float4 *>(row)[32 * j + lane] = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    reinterpret_cast<uint2 *>(row)[32 * j + lane] =
        make_uint2(uint32_t(f2bf_bits(v[0])) | (uint32_t(f2bf_bits(v[1])) << 16),
                   uint32_t(f2bf_bits(v[2])) | (uint32_t(f2bf_bits(v[3])) << 16));
  }
}

// A warp's tokens [t0, t1), in order.  cnt / live: the sequences' counters (global or shared
// memory).  add: this warp's row of E floats in shared memory, zero between tokens (the routing
// weights' gradients on their way to the lanes that own the experts).  done(t, q, dot) takes
// c . p of token t; it is also called with 0 at the first token of each sequence.
template <typename IT, int NV, int VEC, bool GRAD, typename Done>
__device__ __forceinline__ void balance_tokens(const BalArgs &p, int64_t t0, int64_t t1,
                                               const int *cnt, const int *live, float *add,
                                               Done &&done) {
  const int lane = threadIdx.x & 31;
  const int E = p.E, k = p.topk;
  const IT *logits = static_cast<const IT *>(p.logits);
  IT *dl = static_cast<IT *>(p.dlogits);
  BalSeq sq{-1, 0, t0};
  float c[NV][VEC], coef = 0.0f;
  BalRow<IT, NV, VEC> nx;
  if (t0 < t1 && !(p.mask && !p.mask[t0])) nx.load(logits + t0 * E, E, lane);
  for (int64_t t = t0; t < t1; ++t) {
    BalRow<IT, NV, VEC> row = nx;
    if (t + 1 < t1 && !(p.mask && !p.mask[t + 1])) nx.load(logits + (t + 1) * E, E, lane);
    if (t >= sq.b) {
      sq = balance_seq(p, t);
      if (sq.q >= 0) {
        done(t, sq.q, 0.0f);
        const float m = float(live[sq.q]);
        coef = (GRAD && p.grad_loss ? p.grad_loss[sq.q] : 0.0f) * (float(E) / (float(k) * m * m));
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            const int e = VEC * (32 * j + lane) + v;
            c[j][v] = e < E ? float(cnt[int64_t(sq.q) * E + e]) : 0.0f;
          }
      }
    }
    if (sq.q < 0 || (p.mask && !p.mask[t])) {
      if constexpr (GRAD) {
        const float z4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (VEC * (32 * j + lane) < E) bal_store<IT, VEC>(dl + t * E, j, lane, z4);
      }
      continue;
    }
    // the chosen experts' logits, read again while the row is in the cache
    int idx[2] = {-1, -1};
    float dw[2] = {0.f, 0.f}, zs[2] = {0.f, 0.f};
    const bool routed = GRAD && p.dweights;
    if (routed) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (lane + 32 * u < k) {
          const int i = p.indices[t * k + lane + 32 * u];
          if (i >= 0 && i < E) {
            idx[u] = i;
            dw[u] = p.dweights[t * k + lane + 32 * u];
            zs[u] = bal_ld(logits + t * E + i) * p.inv_temp;
          }
        }
    }
    float s[NV][VEC], d[NV][VEC];                    // scores and their derivatives
    float sum = 0.0f, cs = 0.0f, mx = 0.0f, rs = 0.0f;
    if (p.func == DSV41_SCORE_SOFTMAX) {
      mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (VEC * (32 * j + lane) < E)
#pragma unroll
          for (int v = 0; v < VEC; ++v) mx = fmaxf(mx, row.at(j, v));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mx *= p.inv_temp;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const bool in = VEC * (32 * j + lane) < E && mx > -INFINITY;
          s[j][v] = in ? exp_acc(row.at(j, v) * p.inv_temp - mx) : 0.0f;
          sum += s[j][v];
        }
      sum = warp_sum(sum);
      rs = mx > -INFINITY ? __fdividef(1.0f, sum) : 0.0f;
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < VEC; ++v) s[j][v] *= rs;
    } else if (p.func == DSV41_SCORE_SIGMOID) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          s[j][v] = d[j][v] = 0.0f;
          if (VEC * (32 * j + lane) < E) score_sigmoid(row.at(j, v) * p.inv_temp, s[j][v], d[j][v]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          s[j][v] = d[j][v] = 0.0f;
          if (VEC * (32 * j + lane) < E)
            score_sqrtsoftplus(row.at(j, v) * p.inv_temp, s[j][v], d[j][v]);
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        sum += s[j][v];
        cs = fmaf(c[j][v], s[j][v], cs);
      }
    sum = warp_sum(sum);
    cs = warp_sum(cs);
    const float rz = __fdividef(1.0f, sum + 1e-20f), dot = cs * rz;
    done(t, sq.q, dot);
    if constexpr (GRAD) {
      const float ca = coef * rz;
      float R = 0.0f;
      if (routed) {
        float ss[2], dd[2], sel = 0.0f, dws = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ss[u] = dd[u] = 0.0f;
          if (idx[u] >= 0) {
            if (p.func == DSV41_SCORE_SOFTMAX) ss[u] = dd[u] = mx > -INFINITY ? exp_acc(zs[u] - mx) * rs : 0.0f;
            else if (p.func == DSV41_SCORE_SIGMOID) score_sigmoid(zs[u], ss[u], dd[u]);
            else score_sqrtsoftplus(zs[u], ss[u], dd[u]);
          }
          sel += ss[u];
          dws = fmaf(dw[u], ss[u], dws);
        }
        const bool nrm = p.norm && k > 1;
        float rsel = 1.0f, mean = 0.0f;
        if (nrm) {
          rsel = __fdividef(1.0f, warp_sum(sel) + 1e-20f);
          mean = warp_sum(dws) * rsel;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (u && k <= 32) break;
          const float g = p.route_scale * (dw[u] - mean) * rsel;
          R += idx[u] >= 0 ? g * ss[u] : 0.0f;
          // the same expert twice: one after another, in lane order
          const unsigned same = __match_any_sync(0xffffffffu, idx[u] >= 0 ? idx[u] : -1 - lane);
          const int turn = __popc(same & ((1u << lane) - 1));
          for (int o = 0; __any_sync(0xffffffffu, turn >= o); ++o) {
            if (turn == o && idx[u] >= 0) add[idx[u]] += g * dd[u] * p.inv_temp;
            __syncwarp();
          }
        }
        if (p.func == DSV41_SCORE_SOFTMAX) R = warp_sum(R);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (VEC * (32 * j + lane) < E) {
          float o[VEC];
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            const float g = ca * (c[j][v] - dot);
            o[v] = (p.func == DSV41_SCORE_SOFTMAX ? s[j][v] * (g - R) : g * d[j][v]) * p.inv_temp;
          }
          if (routed) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] += add[VEC * (32 * j + lane) + v];
          }
          bal_store<IT, VEC>(dl + t * E, j, lane, o);
        }
      if (routed) {
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (idx[u] >= 0) add[idx[u]] = 0.0f;
        __syncwarp();
      }
    }
  }
}

// ------------------------------------------------------------------ counts
// This thread's choices of the tokens [t0, t1), counted into hist (shared, [S][E]) and live
// (shared, [S]); rows strided over the block.
__device__ __forceinline__ void balance_count_shared(const BalArgs &p, int64_t t0, int64_t t1,
                                                     int *hist, int *live) {
  BalSeq sq{-1, 0, 0};
  for (int64_t t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
    if (p.mask && !p.mask[t]) continue;
    if (t < sq.a || t >= sq.b) sq = balance_seq(p, t);
    if (sq.q < 0) continue;
    atomicAdd(live + sq.q, 1);
    for (int j = 0; j < p.topk; ++j) {
      const int e = __ldg(p.indices + t * p.topk + j);
      if (e >= p.E) dev_flag(DSV41_DEVST_BAD_INDEX);
      else if (e >= 0) atomicAdd(hist + sq.q * p.E + e, 1);
    }
  }
}

// One cluster: every CTA counts a slice of the tokens in shared memory, then sums a slice of
// the counters over the cluster's shared memories: no counter has to be zeroed in memory first.
__global__ void __launch_bounds__(1024, 1) k_balance_count(const BalArgs p) {
  extern __shared__ int bc_smem[];
  int *hist = bc_smem, *live = bc_smem + p.S * p.E;
  const int C = gridDim.x, rank = blockIdx.x, n = p.S * p.E + p.S;
  for (int i = threadIdx.x; i < n; i += 1024) hist[i] = 0;
  __syncthreads();
  balance_count_shared(p, p.T * rank / C, p.T * (rank + 1) / C, hist, live);
  cluster_sync();
  for (int i = rank * 1024 + threadIdx.x; i < n; i += C * 1024) {
    int v = 0;
    for (int c = 0; c < C; ++c) v += ld_cluster_s32(mapa_rank(hist + i, c));
    if (i < p.S * p.E) p.counts[i] = v;
    else p.live[i - p.S * p.E] = v;
  }
  if (rank == 0 && threadIdx.x == 0) p.live[p.S] = 0;      // the ticket of k_balance
  cluster_sync();
}

// More counters than a CTA's shared memory holds: straight to memory (zeroed before).
__global__ void __launch_bounds__(256) k_balance_count_global(const BalArgs p) {
  const int64_t t = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (t >= p.T || (p.mask && !p.mask[t])) return;
  const BalSeq sq = balance_seq(p, t);
  if (sq.q < 0) return;
  atomicAdd(p.live + sq.q, 1);
  for (int j = 0; j < p.topk; ++j) {
    const int e = p.indices[t * p.topk + j];
    if (e >= p.E) dev_flag(DSV41_DEVST_BAD_INDEX);
    else if (e >= 0) atomicAdd(p.counts + int64_t(sq.q) * p.E + e, 1);
  }
}

// ------------------------------------------------------------------ loss and gradient
// loss = E / (k m^2) sum of the tokens' c . p
__device__ __forceinline__ float balance_scale(const BalArgs &p, double sum, int m) {
  return m ? float(sum * double(p.E) / (double(p.topk) * double(m) * double(m))) : 0.0f;
}

// A run of tokens a warp, its row of the next token in flight while it works on one.  The sum
// of a run's tokens of sequence q goes to part[run index + q]: runs and sequences both ascend
// with the tokens, so no two share a place.  The last CTA adds each sequence's places in order.
template <typename IT, int NV, int VEC, bool GRAD>
__global__ void __launch_bounds__(32 * BL_WARPS) k_balance(const BalArgs p) {
  extern __shared__ float bl_add[];                // [BL_WARPS][E], with routing weights
  __shared__ int last_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *add = bl_add + warp * p.E;
  if (GRAD && p.dweights) {
    for (int e = lane; e < p.E; e += 32) add[e] = 0.0f;
    __syncwarp();
  }
  const int64_t r = blockIdx.x * (int64_t)BL_WARPS + warp;
  const int64_t t0 = min(r * p.run, p.T), t1 = min(t0 + p.run, p.T);
  double sum = 0.0;
  int cur = -1;
  balance_tokens<IT, NV, VEC, GRAD>(p, t0, t1, p.counts, p.live, add,
                                    [&](int64_t, int q, float dot) {
    if (q != cur) {
      if (cur >= 0 && lane == 0) p.part[r + cur] = sum;
      cur = q;
      sum = 0.0;
    }
    sum += double(dot);
  });
  if (cur >= 0 && lane == 0) p.part[r + cur] = sum;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_s = atomicAdd(p.live + p.S, 1) == int(gridDim.x) - 1;
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  // places of q: the runs that hold tokens of it
  for (int q = warp; q < p.S; q += BL_WARPS) {
    int64_t a = p.offsets ? p.offsets[q] : 0, b = p.offsets ? p.offsets[q + 1] : p.T;
    a = a < 0 ? 0 : a;
    b = b > p.T ? p.T : b;
    double v = 0.0;
    if (a < b)
      for (int64_t i = a / p.run + lane; i <= (b - 1) / p.run; i += 32) v += __ldcg(p.part + i + q);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) p.loss[q] = balance_scale(p, v, p.live[q]);
  }
}

// The whole pass in one launch, for few tokens: one cluster whose CTAs each count all choices in
// shared memory and take a share of the rows; the rows' c . p meet in rank 0's shared memory.
template <typename IT, int NV, int VEC, bool GRAD>
__global__ void __launch_bounds__(32 * BL_WARPS) k_balance_small(const BalArgs p) {
  extern __shared__ int bs_smem[];
  const int C = gridDim.x, rank = blockIdx.x, n = p.S * p.E;
  int *hist = bs_smem, *live = hist + n;
  float *dots = reinterpret_cast<float *>(live + p.S);         // [T], rank 0's is used
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *add = dots + p.T + warp * p.E;
  for (int i = threadIdx.x; i < n + p.S; i += blockDim.x) hist[i] = 0;
  for (int i = threadIdx.x; i < p.T; i += blockDim.x) dots[i] = 0.0f;
  if (GRAD && p.dweights)
    for (int e = lane; e < p.E; e += 32) add[e] = 0.0f;
  cluster_sync();                                              // rank 0's dots are zero
  balance_count_shared(p, 0, p.T, hist, live);
  __syncthreads();
  for (int i = rank * blockDim.x + threadIdx.x; i < n; i += C * blockDim.x) p.counts[i] = hist[i];
  const int64_t w = rank * BL_WARPS + warp, W = C * BL_WARPS;
  const uint32_t dots0 = mapa_rank(dots, 0);
  balance_tokens<IT, NV, VEC, GRAD>(p, p.T * w / W, p.T * (w + 1) / W, hist, live, add,
                                    [&](int64_t t, int, float dot) {
    if (lane == 0)
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dots0 + uint32_t(t) * 4), "f"(dot)
                   : "memory");
  });
  cluster_sync();
  if (rank) return;
  for (int q = warp; q < p.S; q += BL_WARPS) {
    int64_t a = p.offsets ? p.offsets[q] : 0, b = p.offsets ? p.offsets[q + 1] : p.T;
    a = a < 0 ? 0 : a;
    b = b > p.T ? p.T : b;
    double v = 0.0;
    for (int64_t t = a + lane; t < b; t += 32) v += double(dots[t]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) p.loss[q] = balance_scale(p, v, live[q]);
  }
}

}  // namespace dsv41
