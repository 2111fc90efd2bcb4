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
//
// Counting.  Popular experts make atomics on one address queue up in L2: 2.1 M
// selections that crowd (density ~ id^-1/2 of 262 144 experts) took 41 us.  So
// with many selections each block counts one class of experts in shared memory
// over its part of the selections, and adds its counters to the global counts,
// or stores them for a pass that adds them up.  Classes interleave groups of 8
// experts: crowded neighbours are spread over the blocks (with whole ranges the
// block of the popular one took 65 us at 8.4 M selections), and the 8 counts of
// a group still go out together.  The ids are read once per class (L2 to SM);
// 16-bit counters make that 4 classes for 262 144 experts.  What bounds it is
// shared-memory atomics, about one lane a cycle and SM: 30 of the count's 52 us
// at 8.4 M selections of 262 144 experts.
#pragma once

#include <cuda_bf16.h>

#include "sm100.cuh"

namespace ethos {

constexpr int BAL_THREADS = 256;
constexpr int BAL_MAX_BLOCKS = 1184;   // 8 per SM of a B200
constexpr int BAL_COUNT_THREADS = 1024;
constexpr int BAL_CLASS = 102400;      // most experts counted by one block (200 KB of shared memory)
// 16-bit counters: before each window of selections what a counter holds in
// multiples of 4096 moves to the global count, so none can pass 65 535.
constexpr unsigned BAL_MOVED = 0xf000f000u;
constexpr int BAL_WINDOW = 65535 - 4095;

// Scratch of one call: the header, then sel [tokens * H * k] fp32, the count of
// each selection's expert (0 for a selection left out), for the backward.
struct BalScratch {
  int tokens;     // unmasked tokens
  unsigned done;  // blocks of k_balance_loss that have added their part
  int live[BAL_MAX_BLOCKS];
  double part[BAL_MAX_BLOCKS];
};

// 16 bytes read once: not kept in L1, which is left to the counts
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// 4 consecutive ids (16-byte loads) as unsigned 32-bit numbers; an id that does
// not fit (negative, or 2^31 and more) becomes one that no table has
__device__ __forceinline__ void load_ids4(const int32_t* p, unsigned (&e)[4]) {
  const uint4 v = load_once(p);
  e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
}
__device__ __forceinline__ void load_ids4(const int64_t* p, unsigned (&e)[4]) {
  const uint4 a = load_once(p), b = load_once(p + 2);
  e[0] = a.y ? ~0u : a.x; e[1] = a.w ? ~0u : a.z; e[2] = b.y ? ~0u : b.x; e[3] = b.w ? ~0u : b.z;
}
__device__ __forceinline__ unsigned load_id(const int32_t* p) { return static_cast<unsigned>(*p); }
__device__ __forceinline__ unsigned load_id(const int64_t* p) {
  const uint64_t x = static_cast<uint64_t>(*p);
  return (x >> 32) ? ~0u : static_cast<unsigned>(x);
}

// Calls f(id) for the selections [i0, i1) of unmasked tokens, threads of the
// block in turn, four at a time where addresses allow.
template <bool kMask, class I, class F>
__device__ __forceinline__ void each_selection(const I* __restrict__ ids, const uint8_t* __restrict__ mask,
                                               unsigned per_token, bool quads, unsigned i0, unsigned i1, F f) {
  if (quads) {  // per_token % 4 == 0, ids 16-byte aligned: a quad is of one token
    constexpr unsigned U = 4;  // quads in flight
    const unsigned step = 4 * blockDim.x;
    unsigned i = i0 + 4 * threadIdx.x;
    for (; i + (U - 1) * step < i1; i += U * step) {
      unsigned e[U][4];
      uint8_t in[U];
#pragma unroll
      for (unsigned u = 0; u < U; ++u) {
        load_ids4(ids + i + u * step, e[u]);
        if (kMask) in[u] = mask[(i + u * step) / per_token];
      }
#pragma unroll
      for (unsigned u = 0; u < U; ++u) {
        if (kMask && !in[u]) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) f(e[u][j]);
      }
    }
    for (; i < i1; i += step) {
      unsigned e[4];
      load_ids4(ids + i, e);
      if (kMask && !mask[i / per_token]) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) f(e[j]);
    }
  } else {
    for (unsigned i = i0 + threadIdx.x; i < i1; i += blockDim.x) {
      if (kMask && !mask[i / per_token]) continue;
      f(load_id(ids + i));
    }
  }
}
template <class I, class F>
__device__ __forceinline__ void each_selection(const I* __restrict__ ids, const uint8_t* __restrict__ mask,
                                               int per_token, bool quads, int64_t i0, int64_t i1, F f) {
  if (i0 >= i1) return;
  if (mask != nullptr)
    each_selection<true>(ids, mask, per_token, quads, static_cast<unsigned>(i0), static_cast<unsigned>(i1), f);
  else
    each_selection<false>(ids, mask, per_token, quads, static_cast<unsigned>(i0), static_cast<unsigned>(i1), f);
}

// Unmasked tokens of part b of `parts`, into live[b] (thread 0 of the block).
__device__ __forceinline__ void count_live(const uint8_t* __restrict__ mask, int tokens, int b, int parts,
                                           BalScratch* __restrict__ s) {
  __shared__ int sum;
  const int per = (tokens + parts - 1) / parts;
  const int t0 = min(tokens, b * per), t1 = min(tokens, t0 + per);
  if (threadIdx.x == 0) {
    sum = 0;
    if (b == 0) s->done = 0;
  }
  __syncthreads();
  int n = mask == nullptr && threadIdx.x == 0 ? t1 - t0 : 0;
  if (mask != nullptr)
    for (int t = t0 + static_cast<int>(threadIdx.x); t < t1; t += static_cast<int>(blockDim.x)) n += mask[t] ? 1 : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if ((threadIdx.x & 31) == 0 && n) atomicAdd(&sum, n);
  __syncthreads();
  if (threadIdx.x == 0) s->live[b] = sum;
}

// Few selections: atomics on the global counts.
template <class I>
__global__ void __launch_bounds__(BAL_THREADS) k_balance_count(const I* __restrict__ ids,
                                                               const uint8_t* __restrict__ mask, int tokens,
                                                               int per_token, int experts, bool quads,
                                                               int* __restrict__ counts,
                                                               BalScratch* __restrict__ s) {
  pdl_launch_dependents();
  pdl_wait();
  const int n = tokens * per_token, b = blockIdx.x, parts = gridDim.x;
  const int per = ((n + parts - 1) / parts + 3) / 4 * 4;
  const int64_t i0 = static_cast<int64_t>(b) * per;
  each_selection(ids, mask, per_token, quads, i0, i0 + per < n ? i0 + per : n, [&](unsigned e) {
    if (e < static_cast<unsigned>(experts)) atomicAdd(counts + e, 1);
  });
  count_live(mask, tokens, b, parts, s);
}

// Many: block b counts class r = b mod 2^shift, the experts whose group of 8
// is r modulo 2^shift, over part b / 2^shift of the selections.  Counter l of
// the class is expert 8 ((l / 8) 2^shift + r) + l % 8; two counters a word,
// `words` of them.
//
// `part` null: the counters are added to the counts.  Else they go, as they
// are, to part[blockIdx.x], and k_balance_join adds them up.
template <class I>
__global__ void __launch_bounds__(BAL_COUNT_THREADS) k_balance_count_classes(const I* __restrict__ ids,
                                                                             const uint8_t* __restrict__ mask,
                                                                             int tokens, int per_token, int experts,
                                                                             bool quads, int shift, int words,
                                                                             int* __restrict__ counts,
                                                                             uint4* __restrict__ part,
                                                                             BalScratch* __restrict__ s) {
  extern __shared__ uint4 mine4[];
  unsigned* mine = reinterpret_cast<unsigned*>(mine4);
  pdl_launch_dependents();
  const unsigned classes = 1u << shift, r = blockIdx.x & (classes - 1);
  const int b = blockIdx.x >> shift, parts = gridDim.x >> shift;
  for (int i = threadIdx.x; i < words / 4; i += BAL_COUNT_THREADS) mine4[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  pdl_wait();
  const int n = tokens * per_token;
  const int per = ((n + parts - 1) / parts + 3) / 4 * 4;
  const int64_t i0 = static_cast<int64_t>(b) * per, i1 = i0 + per < n ? i0 + per : n;
  // adds what `bits` of word i holds to the counts
  auto add = [&](int i, unsigned bits) {
    int* at = counts + ((((static_cast<unsigned>(i) >> 2) << shift) + r) << 3) + 2 * (i & 3);
    if (bits & 0xffffu) atomicAdd(at, static_cast<int>(bits & 0xffffu));
    if (bits >> 16) atomicAdd(at + 1, static_cast<int>(bits >> 16));
  };
  for (int64_t a = i0; a < i1; a += BAL_WINDOW) {
    if (a > i0) {
      for (int i = threadIdx.x; i < words; i += BAL_COUNT_THREADS) {
        const unsigned c = mine[i] & BAL_MOVED;
        if (c) {
          mine[i] -= c;
          add(i, c);
        }
      }
      __syncthreads();
    }
    each_selection(ids, mask, per_token, quads, a, a + BAL_WINDOW < i1 ? a + BAL_WINDOW : i1, [&](unsigned e) {
      if (((e >> 3) & (classes - 1)) == r && e < static_cast<unsigned>(experts))
        atomicAdd(mine + ((e >> (3 + shift)) << 2) + ((e & 7) >> 1), 1u << (16 * (e & 1)));
    });
    __syncthreads();
  }
  if (part != nullptr) {
    uint4* out = part + static_cast<size_t>(blockIdx.x) * (words / 4);
    for (int i = threadIdx.x; i < words / 4; i += BAL_COUNT_THREADS) out[i] = mine4[i];
  } else {
    for (int i = threadIdx.x; i < words; i += BAL_COUNT_THREADS)
      if (mine[i]) add(i, mine[i]);
  }
  if (r == 0) count_live(mask, tokens, b, parts, s);
}

// Adds the blocks' counters to the counts: 32 groups of 8 experts (neighbours
// within a class) a block, warp by warp over the parts.
__global__ void __launch_bounds__(BAL_THREADS) k_balance_join(const uint4* __restrict__ part, int parts, int shift,
                                                              int words, int experts, int* __restrict__ counts) {
  __shared__ int sum[BAL_THREADS / 32][8][32];
  pdl_launch_dependents();
  pdl_wait();
  const int quads = words / 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = blockIdx.x * 32 + lane;  // of quads << shift
  const int r = g / quads, l = g - r * quads;
  int c[8] = {};
  if (g < quads << shift) {
#pragma unroll 4
    for (int p = warp; p < parts; p += BAL_THREADS / 32) {
      const uint4 v = part[static_cast<size_t>((p << shift) + r) * quads + l];
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[2 * j] += static_cast<int>(w[j] & 0xffffu);
        c[2 * j + 1] += static_cast<int>(w[j] >> 16);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[warp][j][lane] = c[j];
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int v = 0; v < BAL_THREADS / 32; ++v) t += sum[v][warp][lane];
  // expert `warp` of this lane's group
  const int e = (((l << shift) + r) << 3) + warp;
  if (g < quads << shift && e < experts && t) counts[e] += t;
}

// C = N / (n^2 H^2 k), 0 without tokens
__device__ __forceinline__ double balance_coef(int live, int64_t experts, int heads, int k) {
  if (live <= 0) return 0.0;
  const double nh = static_cast<double>(live) * heads;
  return static_cast<double>(experts) / (nh * nh * k);
}

__device__ __forceinline__ void load_w4(const float* p, float (&v)[4]) {
  const uint4 a = load_once(p);
  v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
}
__device__ __forceinline__ void load_w4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ void store_w4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_w4(__nv_bfloat16* p, const float (&v)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Sums w c[id] and leaves c[id] in sel; an id outside [0, experts) is recorded
// and left out, as the count kernels leave it out.  Thread by thread the terms
// are fixed, blocks add in fp64, and the last block adds the blocks in order.
template <class I, class W>
__global__ void __launch_bounds__(BAL_THREADS) k_balance_loss(const I* __restrict__ ids, const W* __restrict__ w,
                                                              const uint8_t* __restrict__ mask, int tokens, int heads,
                                                              int k, int experts, bool quads, int live_parts,
                                                              const int* __restrict__ counts,
                                                              BalScratch* __restrict__ s, float* __restrict__ sel,
                                                              float* __restrict__ loss, int* err) {
  __shared__ double red[BAL_THREADS];
  __shared__ bool last;
  pdl_launch_dependents();
  pdl_wait();
  const int per_token = heads * k;
  const int n = tokens * per_token;
  const int nt = gridDim.x * BAL_THREADS, tid = blockIdx.x * BAL_THREADS + threadIdx.x;
  double acc = 0.0;
  // c of one selection
  auto count_of = [&](unsigned e, bool in) {
    if (!in) return 0.0f;
    if (e >= static_cast<unsigned>(experts)) {
      record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
      return 0.0f;
    }
    return static_cast<float>(__ldg(counts + e));
  };
  if (quads) {
    constexpr int U = 1;
    for (int64_t i = 4ll * tid; i < n; i += 4ll * U * nt) {
      unsigned e[U][4];
      float x[U][4], c[U][4];
      bool in[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = i + 4ll * u * nt;
        in[u] = at < n;
        if (in[u]) {
          load_ids4(ids + at, e[u]);
          load_w4(w + at, x[u]);
          if (mask != nullptr) in[u] = mask[static_cast<unsigned>(at) / static_cast<unsigned>(per_token)] != 0;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) c[u][j] = count_of(e[u][j], in[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = i + 4ll * u * nt;
        if (at < n) store_w4(sel + at, c[u]);
        // a weight left out is not read into the sum (it may be NaN)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc += static_cast<double>(c[u][j] != 0.0f ? x[u][j] * c[u][j] : 0.0f);
      }
    }
  } else {
    for (int64_t i = tid; i < n; i += nt) {
      const bool in = mask == nullptr || mask[static_cast<unsigned>(i) / static_cast<unsigned>(per_token)];
      const float c = count_of(load_id(ids + i), in);
      sel[i] = c;
      acc += static_cast<double>(c != 0.0f ? static_cast<float>(w[i]) * c : 0.0f);
    }
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
  __threadfence();
  __shared__ int live;
  if (threadIdx.x == 0) live = 0;
  acc = 0.0;
  for (int b = threadIdx.x; b < static_cast<int>(gridDim.x); b += BAL_THREADS)
    acc += *static_cast<volatile double*>(&s->part[b]);
  int l = 0;
  for (int b = threadIdx.x; b < live_parts; b += BAL_THREADS) l += s->live[b];
  red[threadIdx.x] = acc;
  __syncthreads();
  if (l) atomicAdd(&live, l);
  for (int o = BAL_THREADS / 2; o > 0; o >>= 1) {
    if (static_cast<int>(threadIdx.x) < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    s->tokens = live;
    *loss = static_cast<float>(red[0] * balance_coef(live, experts, heads, k));
  }
}

// dw = grad C sel
template <class W>
__global__ void __launch_bounds__(BAL_THREADS) k_balance_bwd(int n, int heads, int k, int experts, bool quads,
                                                             const BalScratch* __restrict__ s,
                                                             const float* __restrict__ sel,
                                                             const float* __restrict__ grad, W* __restrict__ dw) {
  pdl_launch_dependents();
  pdl_wait();
  const float c = static_cast<float>(balance_coef(s->tokens, experts, heads, k) * static_cast<double>(*grad));
  const int nt = gridDim.x * BAL_THREADS, tid = blockIdx.x * BAL_THREADS + threadIdx.x;
  if (quads) {
#pragma unroll 4
    for (int64_t i = 4ll * tid; i < n; i += 4ll * nt) {
      float x[4];
      load_w4(sel + i, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= c;
      store_w4(dw + i, x);
    }
  } else {
    for (int64_t i = tid; i < n; i += nt) dw[i] = static_cast<W>(sel[i] * c);
  }
}

}  // namespace ethos
