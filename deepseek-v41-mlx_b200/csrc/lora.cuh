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
// All sums are fp32; h and g stay fp32 between the products.
#pragma once
#include "common.cuh"

namespace dsv41 {

// The adapter of token t: in [0, n), or -1 (ids at or past n raise the bad-index status).
__device__ __forceinline__ int lora_id(const int32_t *ids, int64_t t, int64_t n) {
  const int i = ids[t];
  if (i >= n) {
    dev_flag(DSV41_DEVST_BAD_INDEX);
    return -1;
  }
  return i < 0 ? -1 : i;
}

// out[t, r] = s_i sum_k x[t, k] W_i[r * wr + k * wk], a warp per (t, r)
__global__ void k_lora_shrink(const __nv_bfloat16 *__restrict__ x, int64_t T, int64_t K,
                              const __nv_bfloat16 *__restrict__ w, int64_t wr, int64_t wk,
                              int64_t n, int R, const int32_t *__restrict__ ids,
                              const float *__restrict__ scaling, float *__restrict__ out) {
  const int64_t gw = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (gw >= T * R) return;
  const int64_t t = gw / R;
  const int r = int(gw % R);
  const int i = lora_id(ids, t, n);
  float s = 0.0f;
  if (i >= 0) {
    const __nv_bfloat16 *wi = w + i * (int64_t)R * K + r * wr;
    for (int64_t k = lane; k < K; k += 32)
      s += __bfloat162float(x[t * K + k]) * __bfloat162float(wi[k * wk]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (scaling) s *= scaling[i];
  }
  if (lane == 0) out[gw] = s;
}

// y[t, c] = base[t, c] + s_i sum_r h[t, r] W_i[c * wc + r * wr], a thread per (t, c)
template <typename OT>
__global__ void k_lora_expand(const float *__restrict__ h, int64_t T, int64_t N,
                              const __nv_bfloat16 *__restrict__ w, int64_t wc, int64_t wr,
                              int64_t n, int R, const int32_t *__restrict__ ids,
                              const float *__restrict__ scaling, const OT *base, OT *y) {
  const int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (e >= T * N) return;
  const int64_t t = e / N, c = e % N;
  const int i = lora_id(ids, t, n);
  float s = 0.0f;
  if (i >= 0) {
    const __nv_bfloat16 *wi = w + i * (int64_t)R * N + c * wc;
    for (int r = 0; r < R; ++r) s += h[t * R + r] * __bfloat162float(wi[r * wr]);
    if (scaling) s *= scaling[i];
  }
  if (base) s += float(base[e]);
  y[e] = OT(s);
}

// d[i][r * dr + c * dc] = s_i sum_{t: ids[t] = i} u[t, r] v[t, c], a thread per (i, r, c)
template <typename OT>
__global__ void k_lora_wgrad(const float *__restrict__ u, const __nv_bfloat16 *__restrict__ v,
                             int64_t T, int64_t C, int64_t n, int R,
                             const int32_t *__restrict__ ids, const float *__restrict__ scaling,
                             int64_t dr, int64_t dc, OT *__restrict__ d) {
  const int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (e >= n * R * C) return;
  const int64_t c = e % C, ir = e / C;
  const int r = int(ir % R);
  const int64_t i = ir / R;
  float s = 0.0f;
  bool any = false;
  for (int64_t t = 0; t < T; ++t)
    if (ids[t] == i) {
      s += u[t * R + r] * __bfloat162float(v[t * C + c]);
      any = true;
    }
  if (scaling && any) s *= scaling[i];
  d[i * R * C + r * dr + c * dc] = OT(s);
}

}  // namespace dsv41
