// Token embedding with scaling, and its gradient (model.py:374, nn.Embedding;
// the table is tied to the output head, model.py:385).
//
//   forward   y[t] = s W[id[t]]
//   backward  dW[v] = s sum_{t : id[t] = v} dy[t]
//
// The gradient is dense in v.  It is computed without atomics on floating
// point values, so it is the same in every run: tokens are sorted by id
// (stable, so each row sums its tokens in token order), the sorted list is cut
// into chunks of EMB_CHUNK tokens that are summed independently (a frequent
// token then occupies many SMs), rows that lie inside one chunk are written
// directly, and the pieces of rows that cross chunks are joined in chunk
// order.  Sums are fp32; each row is rounded once.
#pragma once

#include <cuda_bf16.h>
#include <type_traits>

#include "sm100.cuh"

namespace ethos {

constexpr int EMB_SORT_THREADS = 512;
constexpr int EMB_SORT_WARPS = EMB_SORT_THREADS / 32;
constexpr int EMB_MAX_RANGE = 1024;  // ids owned by one block of the sort
constexpr int EMB_CHUNK = 32;        // sorted tokens summed by one unit
constexpr int64_t EMB_NO_PADDING = INT64_MIN;

template <class T>
struct Vec16;  // 16-byte vector of T as fp32 values
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Vec16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
  }
};
// N consecutive elements of a row: one 16-byte access, or (kVec false, a row
// pitch or base that is not 16-byte aligned) one element
template <class T, bool kVec>
struct RowAccess {
  static constexpr int N = kVec ? Vec16<T>::N : 1;
  static __device__ __forceinline__ void load(const T* p, float (&v)[N]) {
    if constexpr (kVec) {
      Vec16<T>::load(p, v);
    } else {
      v[0] = static_cast<float>(*p);
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[N]) {
    if constexpr (kVec) {
      Vec16<T>::store(p, v);
    } else if constexpr (std::is_same<T, float>::value) {
      *p = v[0];
    } else {
      *p = __float2bfloat16_rn(v[0]);
    }
  }
};

// ---------------------------------------------------------------- forward --
// One thread per row piece (a 16-byte piece or one element); the grid covers
// tokens * pieces.  An id outside [0, V) is recorded and its row is zero.
template <class T, class I, bool kVec>
__global__ void __launch_bounds__(256) k_embed_fwd(const I* __restrict__ ids, const T* __restrict__ w, int64_t ldw,
                                                   int64_t tokens, int d, int64_t vocab, float scale,
                                                   T* __restrict__ y, int* err) {
  using A = RowAccess<T, kVec>;
  pdl_launch_dependents();
  pdl_wait();
  const int pieces = d / A::N;
  const int64_t total = tokens * pieces;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = i / pieces;
    const int c = static_cast<int>(i - t * pieces) * A::N;
    const int64_t id = static_cast<int64_t>(__ldg(ids + t));
    float v[A::N];
    if (id < 0 || id >= vocab) {
      record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
#pragma unroll
      for (int j = 0; j < A::N; ++j) v[j] = 0.0f;
    } else {
      A::load(w + id * ldw + c, v);
#pragma unroll
      for (int j = 0; j < A::N; ++j) v[j] *= scale;
    }
    A::store(y + t * d + c, v);
  }
}

// ------------------------------------------------------------------- sort --
// Block b owns the ids [b * range, (b + 1) * range).  Every block reads all
// ids: it counts those below its range, which is where its part of the sorted
// list begins, so that blocks need nothing from one another.  Within the
// block, warp w takes the w-th contiguous part of the tokens, counts its ids,
// and after a scan over (id, warp) places its tokens in order.  Ids that are
// out of range, or equal to `padding` (no gradient; EMB_NO_PADDING: no such
// id), take no place.  `count`, if given, is the number of tokens on the device
// (at most `tokens`).
//   offs [V + 1]  first place of each id (offs[V] = places in use)
//   perm [tokens] token at each place;  sid [tokens] its id
template <class I>
__global__ void __launch_bounds__(EMB_SORT_THREADS) k_embed_sort(const I* __restrict__ ids, int tokens,
                                                                 const int* __restrict__ count, int64_t vocab,
                                                                 int64_t padding, int range, int* __restrict__ offs,
                                                                 int* __restrict__ perm, int* __restrict__ sid,
                                                                 int* err) {
  extern __shared__ int cnt[];  // [EMB_SORT_WARPS][range]
  __shared__ int warp_sum[EMB_SORT_WARPS];
  __shared__ int below_sum[EMB_SORT_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (count != nullptr) tokens = min(tokens, *count);
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * range;
  const int n = static_cast<int>(lo + range < vocab ? range : vocab - lo);  // ids owned
  for (int i = threadIdx.x; i < EMB_SORT_WARPS * range; i += EMB_SORT_THREADS) cnt[i] = 0;
  __syncthreads();
  int* mine = cnt + warp * range;
  const int part = ((tokens + EMB_SORT_WARPS * 32 - 1) / (EMB_SORT_WARPS * 32)) * 32;
  const int64_t t0 = static_cast<int64_t>(warp) * part;
  const int64_t t1 = t0 + part < tokens ? t0 + part : tokens;
  int below = 0;
#pragma unroll 4
  for (int64_t t = t0 + lane; t < t1; t += 32) {
    const int64_t id = static_cast<int64_t>(__ldg(ids + t));
    if (id == padding) continue;
    if (id < 0 || id >= vocab) {
      if (blockIdx.x == 0) record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
    } else if (id < lo) {
      ++below;
    } else if (id < lo + n) {
      atomicAdd(mine + static_cast<int>(id - lo), 1);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0) below_sum[warp] = below;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < EMB_SORT_WARPS; ++w) base += below_sum[w];
  // exclusive scan over the ids (two per thread), then over the warps of each id
  static_assert(EMB_MAX_RANGE <= 2 * EMB_SORT_THREADS, "two ids per thread");
  int tot[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 2 * static_cast<int>(threadIdx.x) + j;
    if (r < n)
      for (int w = 0; w < EMB_SORT_WARPS; ++w) tot[j] += cnt[w * range + r];
  }
  int incl = tot[0] + tot[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int run = base + incl - (tot[0] + tot[1]);
  for (int w = 0; w < warp; ++w) run += warp_sum[w];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 2 * static_cast<int>(threadIdx.x) + j;
    if (r < n) {
      offs[lo + r] = run;
      int at = run;
      for (int w = 0; w < EMB_SORT_WARPS; ++w) {
        const int c = cnt[w * range + r];
        cnt[w * range + r] = at;
        at += c;
      }
      run = at;
      if (lo + r == vocab - 1) offs[vocab] = at;
    }
  }
  __syncthreads();
  // placement in token order: lanes of one id rank by lane number
  for (int64_t tb = t0; tb < t1; tb += 32) {
    const int64_t t = tb + lane;
    int r = -1;
    if (t < t1) {
      const int64_t id = static_cast<int64_t>(__ldg(ids + t));
      if (id != padding && id >= lo && id < lo + n) r = static_cast<int>(id - lo);
    }
    const unsigned in = __ballot_sync(0xffffffffu, r >= 0);
    if (in == 0) continue;
    if (r >= 0) {
      const unsigned same = __match_any_sync(in, r);
      const int rank = __popc(same & ((1u << lane) - 1u));
      const int at = mine[r] + rank;
      __syncwarp(in);
      if (rank == 0) mine[r] = at + __popc(same);
      perm[at] = static_cast<int>(t);
      sid[at] = static_cast<int>(lo + r);
    }
    __syncwarp();
  }
}

// --------------------------------------------------------------- row sums --
// N fp32 values to N elements of O (16-byte stores with kVec)
template <class O, bool kVec, int N>
__device__ __forceinline__ void store_row(O* p, const float (&v)[N]) {
  if constexpr (!kVec) {
    RowAccess<O, false>::store(p, v);
  } else if constexpr (std::is_same<O, float>::value) {
#pragma unroll
    for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  } else {
    Vec16<O>::store(p, v);
  }
}

// Blocks [0, sum_blocks): chunks of EMB_CHUNK places, `ty` chunks per block,
// tx threads along the columns.  Token t contributes row t of dy (pitch ldy)
// times row_scale[t], if given.  part [chunks][2][d] fp32 receives the piece
// of the row that continues from the previous chunk (0) and of the row that
// continues into the next (1); a chunk inside one row uses slot 0.
// Sums go to row id of dw, or (kByPlace) to row offs[id]: the rows of ids in
// use, without the others.  Remaining blocks: zero rows of ids that no token
// holds.
template <class T, bool kVec, class O, bool kByPlace>
__global__ void __launch_bounds__(256) k_embed_rows(const T* __restrict__ dy, int64_t ldy,
                                                    const float* __restrict__ row_scale, int d, int64_t vocab,
                                                    float scale, const int* __restrict__ offs,
                                                    const int* __restrict__ perm, const int* __restrict__ sid,
                                                    int chunk_blocks, int col_blocks, float* __restrict__ part,
                                                    O* __restrict__ dw) {
  using A = RowAccess<T, kVec>;
  constexpr int N = A::N;
  constexpr int U = 4;  // rows in flight per thread
  pdl_launch_dependents();
  pdl_wait();
  const int places = offs[vocab];
  const int sum_blocks = chunk_blocks * col_blocks;
  if (static_cast<int>(blockIdx.x) < sum_blocks) {
    const int cb = blockIdx.x % col_blocks;
    const int64_t chunk = static_cast<int64_t>(blockIdx.x / col_blocks) * blockDim.y + threadIdx.y;
    const int c = (cb * blockDim.x + threadIdx.x) * N;
    const int64_t p0 = chunk * EMB_CHUNK;
    if (c >= d || p0 >= places) return;
    const int64_t p1 = p0 + EMB_CHUNK < places ? p0 + EMB_CHUNK : places;
    const bool from_prev = p0 > 0 && sid[p0 - 1] == sid[p0];
    const bool into_next = p1 < places && sid[p1] == sid[p1 - 1];
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.0f;
    int cur = sid[p0];
    bool first = true;
    for (int64_t p = p0; p < p1; p += U) {
      float v[U][N];
      int id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        id[u] = -1;
        if (p + u < p1) {
          const int t = perm[p + u];
          id[u] = sid[p + u];
          A::load(dy + t * ldy + c, v[u]);
          if (row_scale != nullptr) {
            const float f = row_scale[t];
#pragma unroll
            for (int j = 0; j < N; ++j) v[u][j] *= f;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (id[u] < 0) continue;
        if (id[u] != cur) {  // the row `cur` ends here
          if (first && from_prev) {
#pragma unroll
            for (int j = 0; j < N; ++j) part[(chunk * 2) * d + c + j] = acc[j];
          } else {
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] *= scale;
            store_row<O, kVec>(dw + static_cast<int64_t>(kByPlace ? offs[cur] : cur) * d + c, acc);
          }
          first = false;
          cur = id[u];
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += v[u][j];
      }
    }
    const bool head = first && from_prev;
    if (head || into_next) {
#pragma unroll
      for (int j = 0; j < N; ++j) part[(chunk * 2 + (head ? 0 : 1)) * d + c + j] = acc[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] *= scale;
      store_row<O, kVec>(dw + static_cast<int64_t>(kByPlace ? offs[cur] : cur) * d + c, acc);
    }
    return;
  }
  // rows without a token
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int lane = tid & 31;
  const int64_t nw = static_cast<int64_t>(gridDim.x - sum_blocks) * 8;
  float z[N];
#pragma unroll
  for (int j = 0; j < N; ++j) z[j] = 0.0f;
  for (int64_t v = static_cast<int64_t>(blockIdx.x - sum_blocks) * 8 + (tid >> 5); v < vocab; v += nw) {
    if (offs[v] != offs[v + 1]) continue;
    for (int c = lane * N; c < d; c += 32 * N) store_row<O, kVec>(dw + v * d + c, z);
  }
}

// Rows that cross chunks: the chunk in which such a row begins adds its own
// piece and the pieces of the following chunks, in order, and writes the row.
template <class T, bool kVec, class O, bool kByPlace>
__global__ void __launch_bounds__(256) k_embed_join(int d, int64_t vocab, float scale, const int* __restrict__ offs,
                                                    const int* __restrict__ sid, int col_blocks,
                                                    const float* __restrict__ part, O* __restrict__ dw) {
  constexpr int N = RowAccess<T, kVec>::N;
  pdl_launch_dependents();
  pdl_wait();
  const int places = offs[vocab];
  const int cb = blockIdx.x % col_blocks;
  const int64_t chunk = static_cast<int64_t>(blockIdx.x / col_blocks) * blockDim.y + threadIdx.y;
  const int c = (cb * blockDim.x + threadIdx.x) * N;
  const int64_t p0 = chunk * EMB_CHUNK, p1 = p0 + EMB_CHUNK;
  if (c >= d || p1 >= places) return;
  const int cur = sid[p1 - 1];
  if (sid[p1] != cur) return;                                     // does not continue
  if (p0 > 0 && sid[p0] == cur && sid[p0 - 1] == cur) return;     // began in an earlier chunk
  const int64_t last = (static_cast<int64_t>(offs[cur + 1]) - 1) / EMB_CHUNK;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = part[(chunk * 2 + 1) * d + c + j];
#pragma unroll 4
  for (int64_t k = chunk + 1; k <= last; ++k) {
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += part[(k * 2) * d + c + j];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] *= scale;
  store_row<O, kVec>(dw + static_cast<int64_t>(kByPlace ? offs[cur] : cur) * d + c, acc);
}

}  // namespace ethos
