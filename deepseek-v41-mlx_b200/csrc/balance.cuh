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
// The counts come first (they need the choices alone), so one pass over the logits gives the
// loss and the gradient: each row is read once and, with a gradient, written once.
#pragma once
#include "common.cuh"

namespace dsv41 {

// The sequence of token t: the last q with offsets[q] <= t < offsets[q + 1], or -1.
__device__ __forceinline__ int balance_seq(const int32_t *offsets, int S, int64_t t) {
  if (!offsets) return 0;
  int lo = 0, hi = S + 1;              // first q with offsets[q] > t lies in [lo, hi]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] > t) hi = mid;
    else lo = mid + 1;
  }
  return (lo == 0 || lo == S + 1) ? -1 : lo - 1;
}

__global__ void k_balance_count(const int32_t *__restrict__ indices, int64_t T, int topk, int E,
                                const int32_t *__restrict__ offsets, int S,
                                const uint8_t *__restrict__ mask, int32_t *__restrict__ counts,
                                int *__restrict__ live) {
  const int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (t >= T || (mask && !mask[t])) return;
  const int q = balance_seq(offsets, S, t);
  if (q < 0) return;
  atomicAdd(live + q, 1);
  for (int j = 0; j < topk; ++j) {
    const int e = indices[t * topk + j];
    if (e >= E) dev_flag(DSV41_DEVST_BAD_INDEX);
    else if (e >= 0) atomicAdd(counts + (int64_t)q * E + e, 1);
  }
}

template <typename T> __device__ __forceinline__ float ld_f(const T *p) { return float(*p); }

// A CTA per token; the row's sums by block reduction.  tok_dot[t] = sum_e c_e p_te.
template <typename IT>
__global__ void k_balance_row(const IT *__restrict__ logits, int64_t T, int E,
                              const int32_t *__restrict__ indices, int topk,
                              const int32_t *__restrict__ offsets, int S,
                              const uint8_t *__restrict__ mask, int score_func, float gate_temp,
                              const float *__restrict__ grad_loss,
                              const float *__restrict__ dweights, int norm, float route_scale,
                              const int32_t *__restrict__ counts, const int *__restrict__ live,
                              float *__restrict__ tok_dot, IT *__restrict__ dlogits) {
  __shared__ float red[32], ws[64], wd[64];
  __shared__ float add[1024];
  const int64_t t = blockIdx.x;
  const int e = threadIdx.x;
  const bool in = e < E;
  const int q = (mask && !mask[t]) ? -1 : balance_seq(offsets, S, t);
  if (q < 0) {
    if (e == 0) tok_dot[t] = 0.0f;
    if (in && dlogits) dlogits[t * E + e] = IT(0.0f);
    return;
  }
  const float z = in ? ld_f(logits + t * E + e) / gate_temp : -INFINITY;
  float s, ds_dz = 0.0f;
  if (score_func == DSV41_SCORE_SOFTMAX) {
    const float m = block_reduce_max(z, red);
    const float ex = (in && m > -INFINITY) ? expf(z - m) : 0.0f;
    const float sum = block_reduce_sum(ex, red);
    s = sum > 0.0f || isnan(sum) ? ex / sum : 0.0f;
  } else if (score_func == DSV41_SCORE_SIGMOID) {
    // 1 - s from the same exponential: s (1 - s) = u / (1 + u)^2 keeps its digits at both ends
    const float u = expf(-fabsf(z)), d = 1.0f / (1.0f + u);
    s = in ? (z < 0.0f ? u * d : d) : 0.0f;
    ds_dz = u * d * d;
  } else if (z < -40.0f) {
    s = expf(0.5f * z);                    // softplus(z) = e^z to fp32
    ds_dz = 0.5f * s;
  } else {
    s = sqrtf(fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z))));
    ds_dz = 1.0f / (1.0f + expf(-z)) / (2.0f * s);
  }
  const float c = in ? float(counts[(int64_t)q * E + e]) : 0.0f;
  const float Z = block_reduce_sum(s, red) + 1e-20f;
  const float dot = block_reduce_sum(c * s, red) / Z;
  if (e == 0) tok_dot[t] = dot;
  if (!dlogits) return;
  const float m = float(live[q]);
  float ds = grad_loss ? grad_loss[q] * float(E) / (float(topk) * m * m) * (c - dot) / Z : 0.0f;
  if (dweights) {
    __shared__ float row[1024];
    row[e] = s;
    add[e] = 0.0f;
    __syncthreads();
    if (e == 0) {
      float sum = 1e-20f, dw_w = 0.0f;
      for (int j = 0; j < topk; ++j) {
        const int i = indices[t * topk + j];
        ws[j] = (i >= 0 && i < E) ? row[i] : 0.0f;
        wd[j] = (i >= 0 && i < E) ? dweights[t * topk + j] : 0.0f;
        sum += ws[j];
        dw_w += wd[j] * ws[j];
      }
      for (int j = 0; j < topk; ++j) {
        const int i = indices[t * topk + j];
        if (i < 0 || i >= E) continue;
        const float d = (norm && topk > 1) ? (wd[j] - dw_w / sum) / sum : wd[j];
        add[i] += route_scale * d;
      }
    }
    __syncthreads();
    ds += add[e];
  }
  float dz;
  if (score_func == DSV41_SCORE_SOFTMAX) dz = s * (ds - block_reduce_sum(in ? ds * s : 0.0f, red));
  else dz = ds * ds_dz;
  if (in) dlogits[t * E + e] = IT(dz / gate_temp);
}

// loss[q] = E / (k m^2) sum_t tok_dot[t], a CTA of 256 threads per sequence, fixed order
__global__ void k_balance_loss(const float *__restrict__ tok_dot, int64_t T, int E, int topk,
                               const int32_t *__restrict__ offsets,
                               const int *__restrict__ live, float *__restrict__ loss) {
  __shared__ double part[256];
  const int q = blockIdx.x;
  int64_t a = offsets ? offsets[q] : 0, b = offsets ? offsets[q + 1] : T;
  a = a < 0 ? 0 : a;
  b = b > T ? T : b;
  double s = 0.0;
  for (int64_t t = a + threadIdx.x; t < b; t += 256) s += double(tok_dot[t]);
  part[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double m = double(live[q]);
    loss[q] = live[q] ? float(part[0] * double(E) / (double(topk) * m * m)) : 0.0f;
  }
}

}  // namespace dsv41
