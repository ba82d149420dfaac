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
// gradient, written once.  Sums over a sequence's tokens are doubles.
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
// 2e-7): the library's log1pf, sqrtf and divisions would bound the pass by issue slots.
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
// The same for two values at once, |z| <= 16 where z < 0: packed fp32 pairs halve the polynomial,
// and the exponential needs no correction there (its argument's rounding costs |z| half steps).
// temp_l2e = -log2(e) / temp.  (At T 65536, E 384 with routing weights: 107 us with the scalar
// form above, bound by issue slots.)
__device__ __forceinline__ void score2_sqrtsoftplus(float z0, float z1, float inv_temp,
                                                    float temp_l2e, uint64_t &s, uint64_t &ds) {
  float u0, u1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(u0) : "f"(fabsf(z0) * temp_l2e));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(u1) : "f"(fabsf(z1) * temp_l2e));
  const uint64_t u = f32x2(u0, u1);
  uint64_t p = f32x2(5.126101896e-3f, 5.126101896e-3f);
  p = f32x2_fma(p, u, f32x2(-2.907406539e-2f, -2.907406539e-2f));
  p = f32x2_fma(p, u, f32x2(7.751608640e-2f, 7.751608640e-2f));
  p = f32x2_fma(p, u, f32x2(-1.360224783e-1f, -1.360224783e-1f));
  p = f32x2_fma(p, u, f32x2(1.907688081e-1f, 1.907688081e-1f));
  p = f32x2_fma(p, u, f32x2(-2.483539879e-1f, -2.483539879e-1f));
  p = f32x2_fma(p, u, f32x2(3.331812024e-1f, 3.331812024e-1f));
  p = f32x2_fma(p, u, f32x2(-4.999944568e-1f, -4.999944568e-1f));
  p = f32x2_fma(p, u, f32x2(9.999999404e-1f, 9.999999404e-1f));
  const uint64_t m = f32x2_mul(f32x2(fmaxf(z0, 0.0f), fmaxf(z1, 0.0f)), f32x2(inv_temp, inv_temp));
  const uint64_t sp = f32x2_fma(p, u, m), w = f32x2_add(u, f32x2(1.0f, 1.0f));
  const uint64_t r = f32x2(rsqrt_approx(f32x2_lo(sp)), rsqrt_approx(f32x2_hi(sp)));
  const uint64_t d = f32x2(rcp_approx(f32x2_lo(w)), rcp_approx(f32x2_hi(w)));
  s = f32x2_mul(sp, r);
  const uint64_t h = f32x2_mul(r, f32x2(z0 < 0.0f ? 0.5f * u0 : 0.5f, z1 < 0.0f ? 0.5f * u1 : 0.5f));
  ds = f32x2_mul(h, d);
}
// 1 - s from the same exponential: s (1 - s) = u / (1 + u)^2 keeps its digits at both ends.
__device__ __forceinline__ void score_sigmoid(float z, float &s, float &ds) {
  const float u = exp_acc(-fabsf(z)), d = rcp_approx(1.0f + u);
  s = z < 0.0f ? u * d : d;
  ds = u * d * d;
}

// The warp's sums of two values in 7 shuffles: half the lanes go on with one, half with the other.
__device__ __forceinline__ void warp_sum2(float &a, float &b) {
  const bool h = threadIdx.x & 16;
  float v = (h ? b : a) + __shfl_xor_sync(0xffffffffu, h ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  a = __shfl_sync(0xffffffffu, v, 0);
  b = __shfl_sync(0xffffffffu, v, 16);
}

__device__ __forceinline__ float bal_ld(const float *p) { return __ldg(p); }
__device__ __forceinline__ float bal_ld(const __nv_bfloat16 *p) {
  return bf_bits2f(__ldg(reinterpret_cast<const uint16_t *>(p)));
}

// A row's values as lane l holds them, in NP pairs: VEC = 4 (E % 4 == 0, aligned rows): pairs 2 j
// and 2 j + 1 are elements 4 (32 j + l) .. + 3; VEC = 1: pair j is elements 64 j + l and + 32.
template <typename IT, int NP, int VEC> struct BalRow;
template <int NP> struct BalRow<float, NP, 4> {
  float4 r[NP / 2];
  __device__ __forceinline__ void load(const float *row, int E, int lane) {
#pragma unroll
    for (int j = 0; j < NP / 2; ++j)
      if (4 * (32 * j + lane) < E) r[j] = __ldg(reinterpret_cast<const float4 *>(row) + 32 * j + lane);
  }
  __device__ __forceinline__ float at(int p, int h) const { return (&r[p >> 1].x)[2 * (p & 1) + h]; }
};
template <int NP> struct BalRow<__nv_bfloat16, NP, 4> {
  uint2 r[NP / 2];
  __device__ __forceinline__ void load(const __nv_bfloat16 *row, int E, int lane) {
#pragma unroll
    for (int j = 0; j < NP / 2; ++j)
      if (4 * (32 * j + lane) < E) r[j] = __ldg(reinterpret_cast<const uint2 *>(row) + 32 * j + lane);
  }
  __device__ __forceinline__ float at(int p, int h) const {
    const uint32_t w = p & 1 ? r[p >> 1].y : r[p >> 1].x;
    return __uint_as_float(h ? w & 0xFFFF0000u : w << 16);
  }
};
template <typename IT, int NP> struct BalRow<IT, NP, 1> {
  float r[2 * NP];
  __device__ __forceinline__ void load(const IT *row, int E, int lane) {
#pragma unroll
    for (int j = 0; j < 2 * NP; ++j) r[j] = 32 * j + lane < E ? bal_ld(row + 32 * j + lane) : 0.0f;
  }
  __device__ __forceinline__ float at(int p, int h) const { return r[2 * p + h]; }
};
// Element h of pair p of lane l, and whether the row has it (VEC = 4: both or neither).
template <int VEC> __device__ __forceinline__ int bal_elem(int p, int h, int lane) {
  return VEC == 4 ? 4 * (32 * (p >> 1) + lane) + 2 * (p & 1) + h : 64 * p + 32 * h + lane;
}
// Pairs 2 j and 2 j + 1 (VEC = 4) or pair p (VEC = 1) of a row
template <typename IT, int NP, int VEC>
__device__ __forceinline__ void bal_store(IT *row, int E, int lane, const uint64_t (&v)[NP]) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if (bal_elem<1>(p, 0, lane) < E) row[bal_elem<1>(p, 0, lane)] = IT(f32x2_lo(v[p]));
      if (bal_elem<1>(p, 1, lane) < E) row[bal_elem<1>(p, 1, lane)] = IT(f32x2_hi(v[p]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < NP / 2; ++j)
      if (4 * (32 * j + lane) < E) {
        const uint64_t a = v[2 * j], b = v[2 * j + 1];
        if constexpr (sizeof(IT) == 4) {
          reinterpret_cast<float4 *>(row)[32 * j + lane] =
              make_float4(f32x2_lo(a), f32x2_hi(a), f32x2_lo(b), f32x2_hi(b));
        } else {
          const __nv_bfloat162 x = __floats2bfloat162_rn(f32x2_lo(a), f32x2_hi(a));
          const __nv_bfloat162 y = __floats2bfloat162_rn(f32x2_lo(b), f32x2_hi(b));
          reinterpret_cast<uint2 *>(row)[32 * j + lane] = make_uint2(
              *reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
        }
      }
  }
}

// The routing weights' side of 32 / k tokens at once, a lane a choice (k <= 32): what a token's
// choices need of one another is summed here, and a choice of an expert that an earlier lane of
// the same token has chosen too is left to that lane.  (One token at a time, most lanes idle, was a
// third of the pass: 28 of 83 us at T 65536, E 384, k 6.)
template <typename IT, int FUNC> struct BalChoices {
  int seg, idx;                // token of the batch, expert (-1: none here)
  float dw, n, e, d, sum, dsum, top;
  // idx_in, dw_in: this lane's choice; z: the tokens' rows from the batch's first on
  __device__ __forceinline__ void make(const BalArgs &p, const IT *z, int k, int idx_in, float dw_in) {
    const int lane = threadIdx.x & 31;
    idx = idx_in < p.E ? idx_in : -1;
    dw = idx >= 0 ? dw_in : 0.0f;
    const float zs = idx >= 0 ? bal_ld(z + int64_t(seg) * p.E + idx) * p.inv_temp : -INFINITY;
    e = d = top = 0.0f;
    const int first = min(seg * k, 32 - k);          // (idle lanes read a token that exists)
    if constexpr (FUNC == DSV41_SCORE_SOFTMAX) {
      top = -INFINITY;
      for (int j = 0; j < k; ++j) top = fmaxf(top, __shfl_sync(0xffffffffu, zs, first + j));
      if (idx >= 0) e = d = top > -INFINITY ? exp_acc(zs - top) : 0.0f;
    } else if (idx >= 0) {
      if (FUNC == DSV41_SCORE_SIGMOID) score_sigmoid(zs, e, d);
      else score_sqrtsoftplus(zs, e, d);
    }
    sum = dsum = 0.0f;
    for (int j = 0; j < k; ++j) {
      sum += __shfl_sync(0xffffffffu, e, first + j);
      dsum += __shfl_sync(0xffffffffu, dw * e, first + j);
    }
    n = 1.0f;
    const unsigned same = __match_any_sync(0xffffffffu, idx >= 0 ? (seg << 16) | idx : -1 - lane);
    if (__any_sync(0xffffffffu, __popc(same) > 1)) {
      float all = 0.0f;
      for (int j = 0; j < 32; ++j) {
        const float v = __shfl_sync(0xffffffffu, dw, j);
        if (same >> j & 1) all += v;
      }
      dw = all;
      n = float(__popc(same));
      if (lane != __ffs(same) - 1) idx = -1;
    }
  }
};

// A warp's tokens [t0, t1), in order.  cnt / live: the sequences' counters (global or shared
// memory), ready after `ready()`.  add: this warp's row of E floats in shared memory, zero between
// tokens (the routing weights' gradients on their way to the lanes that own the experts).
// done(t, q, dot) takes c . p of token t; it is also called with 0 at the first token of each
// sequence.  The next token's row, choices and weights' gradients are requested a token ahead.
// NP pairs a lane; FUNC: the score function.
template <typename IT, int NP, int VEC, bool GRAD, int FUNC, typename Ready, typename Done>
__device__ __forceinline__ void balance_tokens(const BalArgs &p, int64_t t0, int64_t t1,
                                               const int *cnt, const int *live, float *add,
                                               Ready &&ready, Done &&done) {
  const int lane = threadIdx.x & 31;
  const int E = p.E, k = p.topk;
  const IT *z = static_cast<const IT *>(p.logits) + t0 * E;     // this token's row, choices, ...
  IT *dl = static_cast<IT *>(p.dlogits) + t0 * E;
  const int32_t *ip = p.indices + t0 * k;
  const float *wp = p.dweights + (p.dweights ? t0 * k : 0);
  const uint8_t *mp = p.mask + (p.mask ? t0 : 0);
  const bool routed = GRAD && p.dweights, nrm = p.norm && k > 1, wide = k > 32;
  const float temp_l2e = -1.44269504f * p.inv_temp;
  BalSeq sq{-1, 0, t0};
  uint64_t c[NP];
  float coef = 0.0f;
  BalRow<IT, NP, VEC> nx;
  bool on_n = false;
  const int G = wide ? 1 : 32 / k;                  // tokens of a batch of choices
  BalChoices<IT, FUNC> bc;
  bc.seg = wide ? 0 : lane / k;
  int at = G - 1, ch_idx = -1;                      // token of the batch; the next batch's choices
  float ch_dw = 0.0f;
  auto fetch = [&](const IT *zr, const uint8_t *mr) {
    on_n = !p.mask || *mr;
    if (on_n) nx.load(zr, E, lane);
  };
  // this lane's choice of the batch that begins at token t (ip, wp, mp: that token's)
  auto fetch_choices = [&](int64_t t) {
    ch_idx = -1;
    if (bc.seg < G && t + bc.seg < t1 && (!p.mask || mp[bc.seg])) {
      ch_idx = __ldg(ip + lane);
      ch_dw = __ldg(wp + lane);
    }
  };
  if (t0 < t1) fetch(z, mp);
  if (routed && !wide) fetch_choices(t0);
  ready();
#pragma unroll 1
  for (int64_t t = t0; t < t1; ++t, z += E, dl += E) {
    const BalRow<IT, NP, VEC> row = nx;
    const bool on = on_n;
    if (routed && !wide && ++at >= G) {
      const int ci = ch_idx;
      const float cw = ch_dw;
      const int64_t left = t1 - t;
      at = 0;
      // ip, wp and mp run a batch ahead of z
      ip += G * k;
      wp += G * k;
      mp += G;
      if (left > G) fetch_choices(t + G);
      bc.make(p, z, k, ci, cw);
    }
    if (t + 1 < t1) fetch(z + E, p.mask + (p.mask ? t + 1 : 0));
    if (t >= sq.b) {
      sq = balance_seq(p, t);
      if (sq.q >= 0) {
        done(t, sq.q, 0.0f);
        const float m = float(live[sq.q]);
        coef = (GRAD && p.grad_loss ? p.grad_loss[sq.q] : 0.0f) * (float(E) / (float(k) * m * m));
        const int *cq = cnt + int64_t(sq.q) * E;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int e0 = bal_elem<VEC>(i, 0, lane), e1 = bal_elem<VEC>(i, 1, lane);
          c[i] = f32x2(e0 < E ? float(cq[e0]) : 0.0f, e1 < E ? float(cq[e1]) : 0.0f);
        }
      }
    }
    if (sq.q < 0 || !on) {
      if constexpr (GRAD) {
        const uint64_t zero[NP] = {};
        bal_store<IT, NP, VEC>(dl, E, lane, zero);
      }
      continue;
    }
    uint64_t s[NP], d[NP];                           // scores and their derivatives
    float mx = 0.0f;
    if constexpr (FUNC == DSV41_SCORE_SOFTMAX) {
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (bal_elem<VEC>(i, h, lane) < E) mx = fmaxf(mx, row.at(i, h));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (mx == -INFINITY) {                         // (fmaxf passes over NaN: a row of nothing else)
        bool nan = false;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (bal_elem<VEC>(i, h, lane) < E) nan |= isnan(row.at(i, h));
        if (__any_sync(0xffffffffu, nan)) mx = __int_as_float(0x7FFFFFFF);
      }
      mx *= p.inv_temp;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        float e[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          e[h] = bal_elem<VEC>(i, h, lane) < E && mx > -INFINITY ? exp_acc(row.at(i, h) * p.inv_temp - mx)
                                                                 : 0.0f;
        s[i] = d[i] = f32x2(e[0], e[1]);
      }
    } else {
      bool fast = false;
      if constexpr (FUNC == DSV41_SCORE_SQRTSOFTPLUS && VEC == 4) {
        float mn = 0.0f;
#pragma unroll
        for (int i = 0; i < NP; ++i)
          if (bal_elem<VEC>(i, 0, lane) < E) mn = fminf(mn, fminf(row.at(i, 0), row.at(i, 1)));
        fast = !__any_sync(0xffffffffu, mn * p.inv_temp < -16.0f);
        if (fast) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            s[i] = d[i] = 0;
            if (bal_elem<VEC>(i, 0, lane) < E)
              score2_sqrtsoftplus(row.at(i, 0), row.at(i, 1), p.inv_temp, temp_l2e, s[i], d[i]);
          }
        }
      }
      if (!fast) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          float e[2] = {0.f, 0.f}, f[2] = {0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (bal_elem<VEC>(i, h, lane) < E) {
              if (FUNC == DSV41_SCORE_SIGMOID) score_sigmoid(row.at(i, h) * p.inv_temp, e[h], f[h]);
              else score_sqrtsoftplus(row.at(i, h) * p.inv_temp, e[h], f[h]);
            }
          s[i] = f32x2(e[0], e[1]);
          d[i] = f32x2(f[0], f[1]);
        }
      }
    }
    uint64_t sum2 = s[0], cs2 = f32x2_mul(c[0], s[0]);
#pragma unroll
    for (int i = 1; i < NP; ++i) {
      sum2 = f32x2_add(sum2, s[i]);
      cs2 = f32x2_fma(c[i], s[i], cs2);
    }
    float sum = f32x2_lo(sum2) + f32x2_hi(sum2), cs = f32x2_lo(cs2) + f32x2_hi(cs2);
    warp_sum2(sum, cs);
    float rs = 1.0f, rz;                             // 1 / sum of the exponentials, of the scores
    if constexpr (FUNC == DSV41_SCORE_SOFTMAX) {
      // s and d still lack the factor rs (a row of -inf: zeros; NaN stays NaN)
      rs = mx > -INFINITY ? __fdividef(1.0f, sum) : (mx == -INFINITY ? 0.0f : mx);
      rz = 1.0f;
      cs *= rs;
    } else {
      rz = __fdividef(1.0f, sum + 1e-20f);
    }
    const float dot = cs * rz;
    done(t, sq.q, dot);
    if constexpr (GRAD) {
      // the routing weights: with S = sum s and D = sum dw s over the choices, a choice adds scale
      // (dw - D / S) / S ds/dz (not normalised: scale dw ds/dz); softmax also takes R = sum ds s
      // off every element.  Its e are scaled to the choices' largest: s = phi e.
      float R = 0.0f;
      if (routed && !wide) {
        float phi = 1.0f, S = bc.sum, D = bc.dsum;
        if constexpr (FUNC == DSV41_SCORE_SOFTMAX) {
          const int from = at * k;
          S = __shfl_sync(0xffffffffu, bc.sum, from);
          D = __shfl_sync(0xffffffffu, bc.dsum, from);
          const float top = __shfl_sync(0xffffffffu, bc.top, from);
          phi = top > -INFINITY ? exp_acc(top - mx) * rs : 0.0f;
        }
        const float w = nrm ? __fdividef(phi, fmaf(phi, S, 1e-20f)) : phi, mean = nrm ? D * w : 0.0f;
        if (FUNC == DSV41_SCORE_SOFTMAX) R = p.route_scale * w * (nrm ? fmaf(-mean, S, D) : D);
        if (bc.seg == at && bc.idx >= 0)
          add[bc.idx] = p.route_scale * w * fmaf(-bc.n, mean, bc.dw) * bc.d * p.inv_temp;
        __syncwarp();
      } else if (routed) {
        // more than 32 choices: two a lane, added one after another
        float e[2], f[2], w[2], S = 0.0f, D = 0.0f;
        int id[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          e[u] = f[u] = w[u] = 0.0f;
          id[u] = lane + 32 * u < k ? p.indices[t * k + lane + 32 * u] : -1;
          if (id[u] >= E) id[u] = -1;
          if (id[u] >= 0) {
            const float zi = bal_ld(z + id[u]) * p.inv_temp;
            w[u] = p.dweights[t * k + lane + 32 * u];
            if (FUNC == DSV41_SCORE_SOFTMAX) e[u] = f[u] = mx > -INFINITY ? exp_acc(zi - mx) * rs : 0.0f;
            else if (FUNC == DSV41_SCORE_SIGMOID) score_sigmoid(zi, e[u], f[u]);
            else score_sqrtsoftplus(zi, e[u], f[u]);
          }
          S += e[u];
          D = fmaf(w[u], e[u], D);
        }
        warp_sum2(S, D);
        const float r = nrm ? __fdividef(1.0f, S + 1e-20f) : 1.0f, mean = nrm ? D * r : 0.0f;
        if (FUNC == DSV41_SCORE_SOFTMAX) R = p.route_scale * r * fmaf(-mean, S, D);
        for (int j = 0; j < k; ++j) {
          const int u = j >> 5;
          const float g = p.route_scale * r * ((u ? w[1] : w[0]) - mean) * (u ? f[1] : f[0]) * p.inv_temp;
          if (lane == (j & 31) && (u ? id[1] : id[0]) >= 0) add[u ? id[1] : id[0]] += g;
          __syncwarp();
        }
      }
      // d loss / d s = ca (c - dot); times the derivative (softmax: s (ds - sum ds s), whose loss
      // part has no sum: sum_e p_e (c_e - dot) = 0)
      const float ca = coef * rz * p.inv_temp * rs;
      const float cb = -dot * ca - (FUNC == DSV41_SCORE_SOFTMAX ? R * p.inv_temp * rs : 0.0f);
      uint64_t o[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i)
        o[i] = f32x2_mul(f32x2_fma(c[i], f32x2(ca, ca), f32x2(cb, cb)), d[i]);
      if (routed) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int e0 = bal_elem<VEC>(i, 0, lane), e1 = bal_elem<VEC>(i, 1, lane);
          if constexpr (VEC == 4) {
            if (e0 < E) {
              const uint4 *at = reinterpret_cast<const uint4 *>(add + (e0 & ~3));
              o[i] = f32x2_add(o[i], i & 1 ? (uint64_t(at->w) << 32) | at->z : (uint64_t(at->y) << 32) | at->x);
            }
          } else {
            o[i] = f32x2_add(o[i], f32x2(e0 < E ? add[e0] : 0.0f, e1 < E ? add[e1] : 0.0f));
          }
        }
      }
      bal_store<IT, NP, VEC>(dl, E, lane, o);
      if (routed) {
        __syncwarp();
        if (!wide) {
          if (bc.seg == at && bc.idx >= 0) add[bc.idx] = 0.0f;
        } else {
          for (int e = lane; e < E; e += 32) add[e] = 0.0f;
        }
        __syncwarp();
      }
    }
  }
}

// ------------------------------------------------------------------ counts
// This block's choices of the tokens [t0, t1), counted into hist ([S][E]) and live ([S]).
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
      else if (e >= 0) atomicAdd(hist + int64_t(sq.q) * p.E + e, 1);
    }
  }
}

// One cluster: every CTA counts a slice of the tokens in shared memory, then sums a slice of
// the counters over the cluster's shared memories: no counter has to be zeroed in memory first.
__global__ void __launch_bounds__(1024, 1) k_balance_count(const BalArgs p) {
  extern __shared__ int bc_smem[];
  pdl_trigger();
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

// Many choices: every SM counts a slice of the tokens and adds what it counted to counters in
// memory (zeroed by k_balance_zero).  Counted in shared memory first where all counters fit (straight
// to memory took 45 us more at T 65536: a sequence's choices meet in a few cache lines).
__global__ void __launch_bounds__(256) k_balance_zero(const BalArgs p) {
  pdl_trigger();
  const int64_t n = int64_t(p.S) * p.E, step = int64_t(gridDim.x) * 256;
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += step) p.counts[i] = 0;
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i <= p.S; i += step) p.live[i] = 0;
}
__global__ void __launch_bounds__(256) k_balance_count_wide(const BalArgs p, int shared) {
  extern __shared__ int bc_smem[];
  const int64_t t0 = p.T * blockIdx.x / gridDim.x, t1 = p.T * (blockIdx.x + 1) / gridDim.x;
  const int n = shared ? p.S * p.E + p.S : 0;
  int *hist = bc_smem, *live = bc_smem + p.S * p.E;
  for (int i = threadIdx.x; i < n; i += 256) hist[i] = 0;
  __syncthreads();
  if (shared) {
    balance_count_shared(p, t0, t1, hist, live);
    __syncthreads();
  }
  pdl_wait();                                       // the zeros
  pdl_trigger();
  if (!shared) {
    balance_count_shared(p, t0, t1, p.counts, p.live);
    return;
  }
  for (int i = threadIdx.x; i < n; i += 256)
    if (hist[i]) atomicAdd(i < p.S * p.E ? p.counts + i : p.live + (i - p.S * p.E), hist[i]);
}

// ------------------------------------------------------------------ loss and gradient
// loss = E / (k m^2) sum of the tokens' c . p
__device__ __forceinline__ float balance_scale(const BalArgs &p, double sum, int m) {
  return m ? float(sum * double(p.E) / (double(p.topk) * double(m) * double(m))) : 0.0f;
}

// A run of tokens a warp, its row of the next token in flight while it works on one.  The sum
// of a run's tokens of sequence q goes to part[run index + q]: runs and sequences both ascend
// with the tokens, so no two share a place.  The last CTA adds each sequence's places in order.
// T 65536, E 384, k 6, fp32 with both gradients: 72 us, 2.8 TB/s, bound by instructions (an
// element takes about 50, three of them special functions; 56% of the issue slots) and their latency.
template <typename IT, int NP, int VEC, bool GRAD, int FUNC>
__global__ void __launch_bounds__(32 * BL_WARPS, NP <= 4 ? 3 : NP <= 8 ? 2 : 1)
    k_balance(const BalArgs p) {
  extern __shared__ __align__(16) float bl_add[];  // [BL_WARPS][E], with routing weights
  __shared__ int last_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *add = bl_add + warp * ((p.E + 3) & ~3);
  if (GRAD && p.dweights) {
    for (int e = lane; e < p.E; e += 32) add[e] = 0.0f;
    __syncwarp();
  }
  const int64_t r = blockIdx.x * (int64_t)BL_WARPS + warp;
  const int64_t t0 = min(r * p.run, p.T), t1 = min(t0 + p.run, p.T);
  double sum = 0.0;
  int cur = -1;
  balance_tokens<IT, NP, VEC, GRAD, FUNC>(p, t0, t1, p.counts, p.live, add, [] { pdl_wait(); },
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
  // places of q: the runs that hold tokens of it.  A warp a sequence; the long ones, where there are
  // few sequences, by the whole CTA (one warp took 20 us for the 3500 runs of one sequence).
  __shared__ double sums[BL_WARPS];
  __shared__ int4 far[64];                       // {sequence, first run, end}
  __shared__ int n_far;
  if (threadIdx.x == 0) n_far = 0;
  __syncthreads();
  auto add_runs = [&](int q, int i0, int i1, int step) {
    double v = 0.0;
#pragma unroll 4
    for (int i = i0; i < i1; i += step) v += __ldcg(p.part + int64_t(i) + q);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  for (int q = warp; q < p.S; q += BL_WARPS) {
    int a = p.offsets ? p.offsets[q] : 0;
    const int b = int(min(p.offsets ? int64_t(p.offsets[q + 1]) : p.T, p.T));
    a = max(a, 0);
    const int i0 = a / p.run, i1 = a < b ? (b - 1) / p.run + 1 : i0;
    if (p.S <= 64 && i1 - i0 > 256) {
      if (lane == 0) far[atomicAdd(&n_far, 1)] = make_int4(q, i0, i1, 0);
      continue;
    }
    const double v = add_runs(q, i0 + lane, i1, 32);
    if (lane == 0) p.loss[q] = balance_scale(p, v, p.live[q]);
  }
  __syncthreads();
  for (int f = 0; f < n_far; ++f) {
    const int4 w = far[f];
    double v = add_runs(w.x, w.y + threadIdx.x, w.z, 32 * BL_WARPS);
    if (lane == 0) sums[warp] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
      v = 0.0;
      for (int i = 0; i < BL_WARPS; ++i) v += sums[i];
      p.loss[w.x] = balance_scale(p, v, p.live[w.x]);
    }
    __syncthreads();
  }
}

// The whole pass in one launch, for few tokens: one cluster whose CTAs each count all choices in
// shared memory and take a share of the rows; the rows' c . p meet in rank 0's shared memory.
template <typename IT, int NP, int VEC, bool GRAD, int FUNC>
__global__ void __launch_bounds__(32 * BL_WARPS) k_balance_small(const BalArgs p) {
  extern __shared__ __align__(16) int bs_smem[];
  const int C = gridDim.x, rank = blockIdx.x, n = p.S * p.E;
  int *hist = bs_smem, *live = hist + ((n + 3) & ~3);
  float *dots = reinterpret_cast<float *>(live + ((p.S + 3) & ~3));    // [T], rank 0's is used
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *add = dots + ((p.T + 3) & ~3) + warp * ((p.E + 3) & ~3);
  for (int i = threadIdx.x; i < n; i += blockDim.x) hist[i] = 0;
  for (int i = threadIdx.x; i < p.S; i += blockDim.x) live[i] = 0;
  for (int i = threadIdx.x; i < p.T; i += blockDim.x) dots[i] = 0.0f;
  if (GRAD && p.dweights)
    for (int e = lane; e < p.E; e += 32) add[e] = 0.0f;
  cluster_sync();                                              // rank 0's dots are zero
  balance_count_shared(p, 0, p.T, hist, live);
  __syncthreads();
  for (int i = rank * blockDim.x + threadIdx.x; i < n; i += C * blockDim.x) p.counts[i] = hist[i];
  const int64_t w = rank * BL_WARPS + warp, W = C * BL_WARPS;
  const uint32_t dots0 = mapa_rank(dots, 0);
  balance_tokens<IT, NP, VEC, GRAD, FUNC>(p, p.T * w / W, p.T * (w + 1) / W, hist, live, add, [] {},
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
