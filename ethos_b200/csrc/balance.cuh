// Balance loss over the router's choices, and per-expert counts.
//
// For the selections (t, h, j) of the tokens with mask m[t] (all when there is
// no mask), n such tokens, expert ids id and routing weights w (the softmax
// weights of model.py:234):
//   c[e] = number of selections of e,   f[e] = c[e] / (n H k),
//   P[e] = sum of their weights / (n H),
//   L = N sum_e f[e] P[e] = C sum_{t,h,j} m[t] w c[id],  C = N / (n^2 H^2 k),
// which is 1 when experts are chosen evenly and grows as choices crowd.  The
// counts carry no gradient: dL/dw = m[t] C c[id].  Written per selection the
// loss needs no per-expert sums of weights: the counts are integers, whose
// atomics give the same result in any order, and the weighted sum has a fixed
// order.
#pragma once

#include <cuda_bf16.h>

#include "sm100.cuh"

namespace ethos {

constexpr int BAL_THREADS = 256;
constexpr int BAL_MAX_BLOCKS = 1184;  // 8 per SM of a B200

// scratch of one call, after the counts
struct BalScratch {
  int tokens;     // unmasked tokens
  unsigned done;  // blocks of k_balance_loss that have added their part
  double part[BAL_MAX_BLOCKS];
};

template <class I>
__global__ void __launch_bounds__(BAL_THREADS) k_balance_count(const I* __restrict__ ids,
                                                               const uint8_t* __restrict__ mask, int64_t tokens,
                                                               int per_token, int64_t experts,
                                                               int* __restrict__ counts, BalScratch* __restrict__ s,
                                                               int* err) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t n = tokens * per_token;
  const int64_t nt = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = tid; i < n; i += nt) {
    if (mask != nullptr && !mask[i / per_token]) continue;
    const int64_t e = static_cast<int64_t>(__ldg(ids + i));
    if (e < 0 || e >= experts) record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
    else atomicAdd(counts + e, 1);
  }
  if (mask != nullptr) {
    int live = 0;
    for (int64_t t = tid; t < tokens; t += nt) live += mask[t] ? 1 : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) live += __shfl_xor_sync(0xffffffffu, live, o);
    if ((threadIdx.x & 31) == 0 && live) atomicAdd(&s->tokens, live);
  } else if (tid == 0) {
    s->tokens = static_cast<int>(tokens);
  }
}

// C = N / (n^2 H^2 k), 0 without tokens
__device__ __forceinline__ double balance_coef(int live, int64_t experts, int heads, int k) {
  if (live <= 0) return 0.0;
  const double nh = static_cast<double>(live) * heads;
  return static_cast<double>(experts) / (nh * nh * k);
}

template <class I, class W>
__global__ void __launch_bounds__(BAL_THREADS) k_balance_loss(const I* __restrict__ ids, const W* __restrict__ w,
                                                              const uint8_t* __restrict__ mask, int64_t tokens,
                                                              int heads, int k, int64_t experts,
                                                              const int* __restrict__ counts,
                                                              BalScratch* __restrict__ s, float* __restrict__ loss) {
  __shared__ double red[BAL_THREADS];
  __shared__ bool last;
  pdl_launch_dependents();
  pdl_wait();
  const int per_token = heads * k;
  const int64_t n = tokens * per_token;
  const int64_t nt = static_cast<int64_t>(gridDim.x) * blockDim.x;
  double acc = 0.0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += nt) {
    if (mask != nullptr && !mask[i / per_token]) continue;
    const int64_t e = static_cast<int64_t>(__ldg(ids + i));
    if (e >= 0 && e < experts) acc += static_cast<double>(static_cast<float>(w[i]) * static_cast<float>(counts[e]));
  }
  red[threadIdx.x] = acc;
  __syncthreads();
  for (int o = BAL_THREADS / 2; o > 0; o >>= 1) {
    if (static_cast<int>(threadIdx.x) < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    s->part[blockIdx.x] = red[0];
    __threadfence();
    last = atomicAdd(&s->done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  // the last block adds the parts in block order
  __threadfence();
  acc = 0.0;
  for (int b = threadIdx.x; b < static_cast<int>(gridDim.x); b += BAL_THREADS)
    acc += *static_cast<volatile double*>(&s->part[b]);
  red[threadIdx.x] = acc;
  __syncthreads();
  for (int o = BAL_THREADS / 2; o > 0; o >>= 1) {
    if (static_cast<int>(threadIdx.x) < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = static_cast<float>(red[0] * balance_coef(s->tokens, experts, heads, k));
}

template <class I, class W>
__global__ void __launch_bounds__(BAL_THREADS) k_balance_bwd(const I* __restrict__ ids,
                                                             const uint8_t* __restrict__ mask, int64_t tokens,
                                                             int heads, int k, int64_t experts,
                                                             const int* __restrict__ counts,
                                                             const BalScratch* __restrict__ s,
                                                             const float* __restrict__ grad, W* __restrict__ dw) {
  pdl_launch_dependents();
  pdl_wait();
  const float c = static_cast<float>(balance_coef(s->tokens, experts, heads, k) * static_cast<double>(*grad));
  const int per_token = heads * k;
  const int64_t n = tokens * per_token;
  const int64_t nt = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += nt) {
    float v = 0.0f;
    if (mask == nullptr || mask[i / per_token]) {
      const int64_t e = static_cast<int64_t>(__ldg(ids + i));
      if (e >= 0 && e < experts) v = c * static_cast<float>(counts[e]);
    }
    dw[i] = static_cast<W>(v);
  }
}

}  // namespace ethos
