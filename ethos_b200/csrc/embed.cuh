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

constexpr int EMB_SORT_THREADS = 1024;
constexpr int EMB_SORT_WARPS = EMB_SORT_THREADS / 32;
constexpr int EMB_MAX_RANGE = 1024;  // ids owned by one block of the sort
constexpr int EMB_CHUNK = 32;        // sorted tokens summed by one unit
constexpr int EMB_FILL = 8;          // ids checked together for rows without a token
constexpr int64_t EMB_NO_PADDING = INT64_MIN;

// N consecutive elements of a row as fp32 values: one 16-byte access, or
// (kVec false, a row pitch or base that is not 16-byte aligned) one element.
// Raw is what a load leaves in registers until it is used.
template <class T, bool kVec>
struct RowAccess {  // one element
  static constexpr int N = 1;
  using Raw = T;
  static __device__ __forceinline__ Raw load_raw(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[1]) { v[0] = static_cast<float>(r); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[1]) {
    if constexpr (std::is_same<T, float>::value) *p = v[0];
    else *p = __float2bfloat16_rn(v[0]);
  }
};
template <>
struct RowAccess<float, true> {
  static constexpr int N = 4;
  using Raw = float4;
  static __device__ __forceinline__ Raw load_raw(const float* p) { return *reinterpret_cast<const float4*>(p); }
  static __device__ __forceinline__ void unpack(const Raw& a, float (&v)[4]) {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct RowAccess<__nv_bfloat16, true> {
  static constexpr int N = 8;
  using Raw = uint4;
  static __device__ __forceinline__ Raw load_raw(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void unpack(const Raw& u, float (&v)[8]) {
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
template <class T>
struct Vec16 : RowAccess<T, true> {
  using A = RowAccess<T, true>;
  static __device__ __forceinline__ void load(const T* p, float (&v)[A::N]) { A::unpack(A::load_raw(p), v); }
};

// ---------------------------------------------------------------- forward --
// Threads (tx along a row's pieces of 16 bytes or one element, ty tokens); each
// takes EMB_FWD_ROWS tokens with their loads in flight together (65 536 rows
// of 2 KB, caches cold: 57, 53, 59 and 65 us with 1, 2, 4 and 8, 268 MB at up
// to 5.1 TB/s).  An id outside [0, V) is recorded and its row is zero.
constexpr int EMB_FWD_ROWS = 2;
template <class T, class I, bool kVec>
__global__ void __launch_bounds__(256) k_embed_fwd(const I* __restrict__ ids, const T* __restrict__ w, int64_t ldw,
                                                   int64_t tokens, int d, int64_t vocab, float scale,
                                                   T* __restrict__ y, int* err) {
  using A = RowAccess<T, kVec>;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (EMB_FWD_ROWS * blockDim.y) + threadIdx.y;
  int64_t id[EMB_FWD_ROWS];
#pragma unroll
  for (int k = 0; k < EMB_FWD_ROWS; ++k) {
    const int64_t t = t0 + k * blockDim.y;
    id[k] = t < tokens ? static_cast<int64_t>(__ldg(ids + t)) : 0;
    if (id[k] < 0 || id[k] >= vocab) {
      record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
      id[k] = -1;
    }
  }
  for (int c = threadIdx.x * A::N; c < d; c += blockDim.x * A::N) {
    typename A::Raw raw[EMB_FWD_ROWS];
#pragma unroll
    for (int k = 0; k < EMB_FWD_ROWS; ++k)
      if (t0 + k * blockDim.y < tokens && id[k] >= 0) raw[k] = A::load_raw(w + id[k] * ldw + c);
#pragma unroll
    for (int k = 0; k < EMB_FWD_ROWS; ++k) {
      const int64_t t = t0 + k * blockDim.y;
      if (t >= tokens) continue;
      float v[A::N];
      if (id[k] >= 0) {
        A::unpack(raw[k], v);
#pragma unroll
        for (int j = 0; j < A::N; ++j) v[j] *= scale;
      } else {
#pragma unroll
        for (int j = 0; j < A::N; ++j) v[j] = 0.0f;
      }
      A::store(y + t * d + c, v);
    }
  }
}

// ------------------------------------------------------------------- sort --
// Groups the tokens by id, in token order within an id.  Block b owns the ids
// that are b modulo the number of blocks (2^shift): frequent ids are low ids in practice,
// and blocks that owned ranges left one with most of the tokens (26 us against
// 20 at 16 384 Zipf-distributed tokens of 100 277 ids, caches cold).  Every block reads
// all ids: it counts those of lower blocks, which is where its part of the
// list begins, so that blocks need nothing from one another.  Within the
// block, warp w takes the w-th contiguous part of the tokens, counts its ids,
// and after a scan over (id, warp) places its tokens in order.  Ids that are
// out of range, or equal to `padding` (no gradient; EMB_NO_PADDING: no such
// id), take no place.  `count`, if given, is the number of tokens on the device
// (at most `tokens`).
//   span [V]  first place of each id and the place after its last;
//   span[V].x places in use
//   perm [tokens] token at each place;  sid [tokens] its id
template <class I>
__global__ void __launch_bounds__(EMB_SORT_THREADS) k_embed_sort(const I* __restrict__ ids, int tokens,
                                                                 const int* __restrict__ count, int64_t vocab,
                                                                 int64_t padding, int range, int shift,
                                                                 int2* __restrict__ span,
                                                                 int* __restrict__ perm, int* __restrict__ sid,
                                                                 int* err) {
  extern __shared__ int cnt[];  // [EMB_SORT_WARPS][range]
  __shared__ int warp_sum[EMB_SORT_WARPS];
  __shared__ int below_sum[EMB_SORT_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned owner = blockIdx.x, owners = gridDim.x;
  for (int i = threadIdx.x; i < EMB_SORT_WARPS * range; i += EMB_SORT_THREADS) cnt[i] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  if (count != nullptr) tokens = min(tokens, *count);
  // local number of an id owned here, -1 for others, -2 for those of lower blocks
  auto local = [&](int64_t t, bool report) {
    const int64_t id = static_cast<int64_t>(__ldg(ids + t));
    if (id == padding) return -1;
    if (id < 0 || id >= vocab) {
      if (report && owner == 0) record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
      return -1;
    }
    const unsigned u = static_cast<unsigned>(id), o = u & (owners - 1);
    return o == owner ? static_cast<int>(u >> shift) : (o < owner ? -2 : -1);
  };
  int* mine = cnt + warp * range;
  const int part = ((tokens + EMB_SORT_WARPS * 32 - 1) / (EMB_SORT_WARPS * 32)) * 32;
  const int64_t t0 = static_cast<int64_t>(warp) * part;
  const int64_t t1 = t0 + part < tokens ? t0 + part : tokens;
  int below = 0;
#pragma unroll 8
  for (int64_t t = t0 + lane; t < t1; t += 32) {
    const int l = local(t, true);
    if (l >= 0) atomicAdd(mine + l, 1);
    below += l == -2;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0) below_sum[warp] = below;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < EMB_SORT_WARPS; ++w) base += below_sum[w];
  // exclusive scan over the ids (one per thread), then over the warps of each id
  static_assert(EMB_MAX_RANGE <= EMB_SORT_THREADS, "one id per thread");
  const int r = threadIdx.x;
  const int64_t id = static_cast<int64_t>(r) * owners + owner;
  const bool own = r < range && id < vocab;
  int tot = 0;
  if (own)
    for (int w = 0; w < EMB_SORT_WARPS; ++w) tot += cnt[w * range + r];
  int incl = tot;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int at0 = base + incl - tot;
#pragma unroll
  for (int w = 0; w < EMB_SORT_WARPS; ++w)
    if (w < warp) at0 += warp_sum[w];
  if (own) {
    span[id] = make_int2(at0, at0 + tot);
    if (tot > 0)
      for (int w = 0; w < EMB_SORT_WARPS; ++w) {
        const int c = cnt[w * range + r];
        cnt[w * range + r] = at0;
        at0 += c;
      }
  }
  if (threadIdx.x == EMB_SORT_THREADS - 1 && owner == owners - 1) {
    int all = base;
    for (int w = 0; w < EMB_SORT_WARPS; ++w) all += warp_sum[w];
    span[vocab] = make_int2(all, 0);
  }
  __syncthreads();
  // placement in token order: lanes of one id rank by lane number; ids of
  // several rounds are loaded ahead
  constexpr int AHEAD = 4;
  for (int64_t tb = t0; tb < t1; tb += 32 * AHEAD) {
    int l[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int64_t t = tb + 32 * a + lane;
      l[a] = t < t1 ? local(t, false) : -1;
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const unsigned in = __ballot_sync(0xffffffffu, l[a] >= 0);
      if (in == 0) continue;
      if (l[a] >= 0) {
        const unsigned same = __match_any_sync(in, l[a]);
        const int rank = __popc(same & ((1u << lane) - 1u));
        const int at = mine[l[a]] + rank;
        __syncwarp(in);
        if (rank == 0) mine[l[a]] = at + __popc(same);
        perm[at] = static_cast<int>(tb + 32 * a + lane);
        sid[at] = l[a] * static_cast<int>(owners) + static_cast<int>(owner);
      }
      __syncwarp();
    }
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
    RowAccess<O, true>::store(p, v);
  }
}

// Blocks [0, sum_blocks): chunks of EMB_CHUNK places, `ty` chunks per block,
// tx threads along the columns.  Token t contributes row t of dy (pitch ldy)
// times row_scale[t], if given.  part [chunks][2][d] fp32 receives the piece
// of the row that continues from the previous chunk (0) and of the row that
// continues into the next (1); a chunk inside one row uses slot 0.
// Sums go to row id of dw, or (kByPlace) to row span[id].x: the rows of ids in
// use, without the others.  Remaining blocks: zero rows of ids that no token
// holds.
template <class T, bool kVec, class O, bool kByPlace>
__global__ void __launch_bounds__(256) k_embed_rows(const T* __restrict__ dy, int64_t ldy,
                                                    const float* __restrict__ row_scale, int d, int64_t vocab,
                                                    float scale, const int2* __restrict__ span,
                                                    const int* __restrict__ perm, const int* __restrict__ sid,
                                                    int chunk_blocks, int col_blocks, float* __restrict__ part,
                                                    O* __restrict__ dw) {
  using A = RowAccess<T, kVec>;
  constexpr int N = A::N;
  constexpr int U = 8;  // rows in flight per thread
  static_assert(EMB_CHUNK % U == 0, "whole batches");
  __shared__ int s_sid[32][EMB_CHUNK + 2];  // with the neighbours' ids at both ends
  __shared__ int s_tok[32][EMB_CHUNK];
  __shared__ float s_f[32][EMB_CHUNK];
  pdl_launch_dependents();
  pdl_wait();
  const int places = span[vocab].x;
  const int sum_blocks = chunk_blocks * col_blocks;
  if (static_cast<int>(blockIdx.x) < sum_blocks) {
    const int cb = blockIdx.x % col_blocks, ty = threadIdx.y;
    const int64_t chunk = static_cast<int64_t>(blockIdx.x / col_blocks) * blockDim.y + ty;
    const int64_t p0 = chunk * EMB_CHUNK;
    for (int i = threadIdx.x; i < EMB_CHUNK + 2; i += blockDim.x) {
      const int64_t p = p0 - 1 + i;
      s_sid[ty][i] = p >= 0 && p < places ? sid[p] : -1;
    }
    for (int i = threadIdx.x; i < EMB_CHUNK; i += blockDim.x) {
      const int t = p0 + i < places ? perm[p0 + i] : 0;
      s_tok[ty][i] = t;
      if (row_scale != nullptr) s_f[ty][i] = p0 + i < places ? row_scale[t] : 0.0f;
    }
    __syncthreads();
    const int c = (cb * blockDim.x + threadIdx.x) * N;
    if (c >= d || p0 >= places) return;
    const int cnt = static_cast<int>(places - p0 < EMB_CHUNK ? places - p0 : EMB_CHUNK);
    const int* id = s_sid[ty] + 1;
    const bool from_prev = id[-1] == id[0];
    const bool into_next = cnt == EMB_CHUNK && id[cnt] == id[cnt - 1];
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.0f;
    int cur = id[0], begin = 0;  // the row being summed, its first place in the chunk
    auto flush = [&](bool open_end) {
      const bool head = begin == 0 && from_prev;
      if (head || open_end) {
#pragma unroll
        for (int j = 0; j < N; ++j) part[(chunk * 2 + (head ? 0 : 1)) * d + c + j] = acc[j];
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] *= scale;
        store_row<O, kVec>(dw + (kByPlace ? p0 + begin : static_cast<int64_t>(cur)) * d + c, acc);
      }
    };
    for (int i0 = 0; i0 < cnt; i0 += U) {
      typename A::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < cnt) raw[u] = A::load_raw(dy + s_tok[ty][i0 + u] * ldy + c);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u;
        if (i >= cnt) continue;
        if (id[i] != cur) {  // the row `cur` ends here
          flush(false);
          cur = id[i];
          begin = i;
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        }
        float v[N];
        A::unpack(raw[u], v);
        if (row_scale != nullptr) {
          const float f = s_f[ty][i];
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] = fmaf(v[j], f, acc[j]);
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += v[j];
        }
      }
    }
    flush(into_next);
    return;
  }
  // rows without a token, EMB_FILL ids of a warp at a time
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int lane = tid & 31;
  const int64_t nw = static_cast<int64_t>(gridDim.x - sum_blocks) * 8;
  float z[N];
#pragma unroll
  for (int j = 0; j < N; ++j) z[j] = 0.0f;
  for (int64_t v0 = (static_cast<int64_t>(blockIdx.x - sum_blocks) * 8 + (tid >> 5)) * EMB_FILL; v0 < vocab;
       v0 += nw * EMB_FILL) {
    const int64_t v = v0 + lane;
    int2 sp = make_int2(0, 1);
    if (lane < EMB_FILL && v < vocab) sp = span[v];
    unsigned empty = __ballot_sync(0xffffffffu, sp.x == sp.y);
    while (empty) {
      const int64_t row = v0 + __ffs(empty) - 1;
      empty &= empty - 1;
      for (int c = lane * N; c < d; c += 32 * N) store_row<O, kVec>(dw + row * d + c, z);
    }
  }
}

// Rows that cross chunks: block of the chunk in which such a row begins; its
// ty threads per column take contiguous parts of the following chunks' pieces,
// and their sums are added in order.
constexpr int EMB_JOIN_THREADS = 1024;
template <class T, bool kVec, class O, bool kByPlace>
__global__ void __launch_bounds__(EMB_JOIN_THREADS) k_embed_join(int d, int64_t vocab, float scale,
                                                                 const int2* __restrict__ span,
                                                                 const int* __restrict__ sid, int col_blocks,
                                                                 const float* __restrict__ part, O* __restrict__ dw) {
  constexpr int N = RowAccess<T, kVec>::N;
  __shared__ float sums[EMB_JOIN_THREADS * N];
  pdl_launch_dependents();
  pdl_wait();
  const int places = span[vocab].x;
  const int cb = blockIdx.x % col_blocks, tx = threadIdx.x, ty = threadIdx.y;
  const int64_t chunk = blockIdx.x / col_blocks;
  const int64_t p0 = chunk * EMB_CHUNK, p1 = p0 + EMB_CHUNK;
  if (p1 >= places) return;
  const int cur = sid[p1 - 1];
  if (sid[p1] != cur) return;                                     // does not continue
  const int2 sp = span[cur];
  const int64_t start = sp.x;
  if (start < p0) return;                                         // began in an earlier chunk
  const int64_t last = (static_cast<int64_t>(sp.y) - 1) / EMB_CHUNK;
  const int c = (cb * blockDim.x + tx) * N;
  const int64_t per = (last - chunk + blockDim.y - 1) / blockDim.y;
  const int64_t k0 = chunk + 1 + ty * per, k1 = k0 + per - 1 < last ? k0 + per - 1 : last;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.0f;
  if (c < d) {
    if (ty == 0) {
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = part[(chunk * 2 + 1) * d + c + j];
    }
#pragma unroll 8
    for (int64_t k = k0; k <= k1; ++k) {
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] += part[(k * 2) * d + c + j];
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) sums[(ty * blockDim.x + tx) * N + j] = acc[j];
  __syncthreads();
  if (ty != 0 || c >= d) return;
  for (int y = 1; y < static_cast<int>(blockDim.y); ++y)
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += sums[(y * blockDim.x + tx) * N + j];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] *= scale;
  store_row<O, kVec>(dw + (kByPlace ? start : static_cast<int64_t>(cur)) * d + c, acc);
}

}  // namespace ethos
