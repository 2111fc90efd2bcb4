// Cross entropy of the output head (model.py:385, train.py:200) without its
// logits in memory:
//
//   l[t, v] = h[t] . W[v],   lse[t] = log sum_v exp l[t, v],
//   loss[t] = lse[t] - l[t, y[t]]                       (0 for ignored tokens)
//   dl[t, v] = g[t] (exp(l[t, v] - lse[t]) - [v = y[t]])
//   dh = dl W,   dW = dl^T h
//
// The label's column stays out of the exponentials: c = l[t, y] is a dot
// product in fp32, and with S = sum_{v != y} exp(l[t, v] - c)
//   loss = log(1 + S),  1 - p[y] = S / (1 + S),
// so that a confident token's loss and gradient are not differences of nearly
// equal numbers.
//
// Two ways, by what the caller needs:
//
//  keep    (bf16; loss and gradients in one call, for a gradient of the loss
//          that is one number).  The GEMM's epilogue writes E = exp(l - c) of
//          every other column as bf16 while it adds up S.  With r = 1/(1 + S)
//          a row of p is r E, and the two products read E as it is:
//            dh = r (E W) + (p[y] - 1) W[y],   dW = E^T (r h) + label rows,
//          where row v of the label rows is the sum of (p[y] - 1) h[t] over the
//          tokens with label v, in fp32, by the sort of embed.cuh.  Three
//          products of 2 T V d FLOPs.  A row whose logits pass c by more than
//          XE_KEEP_RANGE is done again with its largest logit for c.
//  piece   (everything else).  The forward keeps, for each row, the running
//          maximum and sum over the tiles it sees.  The backward forms the
//          logits again, one piece of the vocabulary after another; their
//          gradient goes to a [tokens, piece] bf16 buffer straight from the
//          accumulators, and one launch computes both products with it.  Four
//          products.  The label's own entry, the largest of a row, is not
//          among them for bf16: its terms are added in fp32 as the keep way
//          adds them (rounded with the rest, the gradients were off by 2.4e-3
//          in the norm, where the output's rounding alone is 1.7e-3).
//
// Both are bounded by the tensor cores.
//
// Rows.  With more than XE_ROWS_IN_PLACE tokens the tokens that are not ignored
// are packed first (their number stays on the device), so ignored tokens cost
// nothing after that; fewer fit one row tile and keep their places.
//
// Types.  bf16: operands as they are; E (or dl) and r h are rounded to bf16,
// the operand type of the products; sums are fp32.  fp32: operands, and dl, are
// carried as three bf16 planes whose sum is the fp32 value, and each product is
// six plane products.  The accumulator of the matrix unit loses about half an
// ulp of the running sum per step of 16, so each K block of 64 (24 steps, the
// smallest products first) has a fresh accumulator and the blocks are added up
// in fp32 registers.  The six products read each plane from shared memory,
// where it comes once: loaded for each product anew, the feed from L2 bound
// the kernel (815 us against 513 for the gradient products of 2047 tokens,
// 32 003 x 512).
//
// GEMM: k_xent_gemm runs on SM pairs as k_gemm2sm does (each CTA staging 128
// rows of A and of each 256 of B, cta_group::2 MMA, no multicast loads), with
// row counts read from the device, ragged M, N and K, and units grouped so that
// the operand shared by concurrent pairs stays in L2.  bf16 tiles are 256 x
// 512: both accumulators of the pair read one A tile, a quarter fewer operand
// bytes per product than 256 x 256, whose feed from L2 bounded it.
#pragma once

#include "embed.cuh"
#include "gemm2sm.cuh"

namespace ethos {

constexpr int XE_ROWS_IN_PLACE = 256;  // tokens that keep their places (one row tile)
constexpr int XE_TILE = 256;         // rows of a pair's tile; columns of one accumulator
constexpr int XE_GROUP_M = 64;       // row tiles walked before the next column tile
constexpr int XE_NO_ROW = 1 << 29;   // beyond any operand's rows
constexpr float XE_LOG2E = 1.4426950408889634f;
constexpr float XE_KEEP_RANGE = 60.0f;  // e^60 times any sum over a vocabulary is finite in fp32 and bf16

enum XeMode { XE_STATS, XE_KEEP, XE_DLOGITS, XE_GRADS };

// What the forward leaves for the backward, at the start of the save buffer.
struct XeMeta {
  int rows;       // rows of the packed problem
  int valid;      // tokens that are not ignored
  unsigned done;  // blocks of k_xent_loss that have added their part
  int redo;       // KEEP: some row's shift was too low
};

// Row index, compacted: pos[t] = row of token t or -1, idx[r] = token of row
// r, yc[r] = its label (-1: an ignored token that kept its place).
struct XeRows {
  XeMeta* meta;
  int* pos;
  int* idx;
  int* yc;
  float* lab;  // the label's logit
  float* c;    // KEEP: shift of the row's exponents
  float* lse;
  float* q;    // p[y] - 1
  float* r;    // KEEP: 1 / sum of exp(l - c)
};

template <class I>
__global__ void __launch_bounds__(1024) k_xent_index(const I* __restrict__ labels, int tokens, int64_t vocab,
                                                     int64_t ignore, bool compact, XeRows rw,
                                                     float* __restrict__ loss_rows, int* __restrict__ redo_tile,
                                                     int* err) {
  __shared__ int warp_sum[32];
  pdl_launch_dependents();
  pdl_wait();
  if (redo_tile != nullptr)
    for (int i = threadIdx.x; i < (tokens + XE_TILE - 1) / XE_TILE; i += 1024) redo_tile[i] = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int base = 0;
  for (int t0 = 0; t0 < tokens; t0 += 1024) {
    const int t = t0 + static_cast<int>(threadIdx.x);
    int64_t y = -1;
    if (t < tokens) {
      y = static_cast<int64_t>(__ldg(labels + t));
      if (y == ignore) {
        y = -1;
      } else if (y < 0 || y >= vocab) {
        record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
        y = -1;
      }
    }
    const unsigned live = __ballot_sync(0xffffffffu, y >= 0);
    if (lane == 0) warp_sum[warp] = __popc(live);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    __syncthreads();
    if (t < tokens) {
      const int at = compact ? base + before + __popc(live & ((1u << lane) - 1u)) : t;
      if (y >= 0 || !compact) {
        rw.idx[at] = t;
        rw.yc[at] = static_cast<int>(y);
      }
      rw.pos[t] = y >= 0 ? at : -1;
      if (y < 0 && loss_rows != nullptr) loss_rows[t] = 0.0f;
    }
    base += all;
  }
  if (threadIdx.x == 0) {
    rw.meta->rows = compact ? base : tokens;
    rw.meta->valid = base;
    rw.meta->done = 0;
    rw.meta->redo = 0;
  }
}

// ------------------------------------------------------------------- pack --
// 8 consecutive elements of a row as fp32 (columns from d on are zero)
template <class S>
__device__ __forceinline__ void load8(const S* s, int c, int d, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= d) {
    if constexpr (sizeof(S) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(s + c), b = *reinterpret_cast<const float4*>(s + c + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(s + c);
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(h[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < d ? static_cast<float>(s[c + j]) : 0.0f;
  }
}
// the leading bf16 part of 8 values, which is taken off them
__device__ __forceinline__ uint4 take_plane(float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    w[j] = *reinterpret_cast<const uint32_t*>(&h);
    const float2 f = __bfloat1622float2(h);
    v[2 * j] -= f.x;
    v[2 * j + 1] -= f.y;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <class S>
__device__ __forceinline__ bool rows_vec(const S* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % static_cast<int64_t>(16 / sizeof(S)) == 0;
}

// dst [PLANES][plane_rows][ldd] bf16 <- rows of src (the vocabulary): plane 0 =
// bf16(v), plane 1 = bf16(v - plane 0), plane 2 the rest; columns d..ldd and
// rows count..plane_rows are zero.
template <class S, int PLANES>
__global__ void __launch_bounds__(256) k_xent_pack(const S* __restrict__ src, int64_t lds, int d, int64_t count,
                                                   __nv_bfloat16* __restrict__ dst, int64_t plane_rows, int ldd) {
  pdl_launch_dependents();
  pdl_wait();
  const int pieces = ldd / 8;
  const int64_t total = plane_rows * pieces;
  const bool vec = rows_vec(src, lds);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / pieces;
    const int c = static_cast<int>(i - r * pieces) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < count) load8(src + r * lds, c, d, vec, v);
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
      *reinterpret_cast<uint4*>(dst + (p * plane_rows + r) * ldd + c) = take_plane(v);
  }
}

// One warp per row of the packed problem: the label's logit in fp32, and the
// row's planes; ignored rows, and rows up to the next multiple of XE_TILE, are
// zero.
template <class S, int PLANES>
__global__ void __launch_bounds__(256) k_xent_rows(const S* __restrict__ hidden, int64_t ldh,
                                                   const S* __restrict__ weight, int64_t ldw, int64_t vocab, int d,
                                                   XeRows rw, __nv_bfloat16* __restrict__ dst, int64_t plane_rows,
                                                   int ldd) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int rows = rw.meta->rows;
  const int upto = (rows + XE_TILE - 1) / XE_TILE * XE_TILE;
  const bool hvec = rows_vec(hidden, ldh), wvec = rows_vec(weight, ldw);
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < upto; r += gridDim.x * 8) {
    const bool in = r < rows;
    const S* h = hidden + (in ? static_cast<int64_t>(rw.idx[r]) : 0) * ldh;
    int y = in ? rw.yc[r] : -1;
    if (y >= vocab) y = -1;  // a save buffer of a larger table's forward
    const S* w = weight + static_cast<int64_t>(y < 0 ? 0 : y) * ldw;
    float dot = 0.0f;
#pragma unroll 2
    for (int c = lane * 8; c < ldd; c += 256) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (y >= 0) {  // rows of ignored tokens are zero whatever they hold
        float x[8];
        load8(h, c, d, hvec, v);
        load8(w, c, d, wvec, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(v[j], x[j], dot);
      }
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
        *reinterpret_cast<uint4*>(dst + (p * plane_rows + r) * ldd + c) = take_plane(v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (in && lane == 0) {
      rw.lab[r] = dot;
      rw.c[r] = dot;
    }
  }
}

// joins two (maximum, sum of exponentials relative to it) pairs
__device__ __forceinline__ void lse_join(float& m, float& s, float m2, float s2) {
  const float hi = fmaxf(m, m2);
  if (hi == -INFINITY) {  // nothing seen yet, or logits of -inf (or NaN) only
    s += s2;
    return;
  }
  s = s * exp2f((m - hi) * XE_LOG2E) + s2 * exp2f((m2 - hi) * XE_LOG2E);
  m = hi;
}

// ------------------------------------------------------------- few tokens --
// The forward for few tokens: one pass over the vocabulary on the fp32 units,
// bounded by its bytes for one token (the table of 100 277 x 1024 bf16, 205 MB,
// in 46 to 50 us, 4.1 to 4.4 TB/s) and by its products and their reduction for
// more.  A warp takes 32 / TT rows of the vocabulary
// at a time, lanes along the columns, TT >= tokens accumulators for each; the
// 32 sums are transposed and reduced over the lanes so that lane l holds the
// logit of row l / TT and token l % TT, and keeps a running (maximum, sum)
// of its token.  The token's label is left out of the sum and its logit kept.
// Block 0 also writes the row index that k_xent_index writes otherwise.
//
// Most tokens that take it rather than the matrix units' row tile of 256.  The
// whole forward in us, caches cold, for 1, 2, 4 and 8 tokens this way and for 9
// the other: bf16, 100 277 x 1024: 62, 69, 81, 130 and 82; 32 003 x 512: 24, 26,
// 28, 36 and 35; 32 003 x 515 (one element at a time): 32, 40, 56, 83 and 47.
// fp32, 100 277 x 1024: 95, 101, 118, 175 and 399; 32 003 x 515: 40, 48, 67, 97
// and 100.
template <class S, bool kVec>
constexpr int xe_few() {
  return sizeof(S) == 4 ? 8 : (kVec ? 4 : 2);
}
constexpr int XE_FEW_BLOCKS = 148;    // pieces of each row's sum
constexpr int XE_FEW_SMEM = 128 * 1024;  // the tokens' states in fp32

template <class S, bool kVec, int TT>
__global__ void __launch_bounds__(256, 1) k_xent_few(const S* __restrict__ hidden, int64_t ldh,
                                                     const S* __restrict__ weight, int64_t ldw, int d, int vocab,
                                                     int tokens, const void* __restrict__ labels, bool labels_i64,
                                                     int64_t ignore, XeRows rw, float* __restrict__ loss_rows,
                                                     float2* __restrict__ part, int64_t part_ld, int* err) {
  using A = RowAccess<S, kVec>;
  constexpr int N = A::N, R = 32 / TT;
  extern __shared__ float hs[];  // [TT][ld], zero beyond the tokens and columns
  __shared__ float2 wp[8][TT];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ld = (d + 32 * N - 1) / (32 * N) * (32 * N);
  for (int i = threadIdx.x; i < TT * ld; i += 256) {
    const int t = i / ld, c = i - t * ld;
    hs[i] = t < tokens && c < d ? static_cast<float>(hidden[t * ldh + c]) : 0.0f;
  }
  // this lane's token and its label (-1: ignored, -2: no token)
  const int t = lane % TT;
  int64_t y = -2;
  if (t < tokens) {
    y = labels_i64 ? static_cast<const int64_t*>(labels)[t] : static_cast<const int32_t*>(labels)[t];
    if (y == ignore) {
      y = -1;
    } else if (y < 0 || y >= vocab) {
      if (blockIdx.x == 0) record_error(err, ETHOS_ERR_ID_OUT_OF_RANGE);
      y = -1;
    }
  }
  if (blockIdx.x == 0 && warp == 0) {
    const unsigned valid = __ballot_sync(0xffffffffu, lane < TT && y >= 0);
    if (lane < TT && lane < tokens) {
      rw.idx[lane] = lane;
      rw.yc[lane] = static_cast<int>(y);
      rw.pos[lane] = y >= 0 ? lane : -1;
      if (y < 0) {
        rw.lab[lane] = 0.0f;
        if (loss_rows != nullptr) loss_rows[lane] = 0.0f;
      }
    }
    if (lane == 0) {
      rw.meta->rows = tokens;
      rw.meta->valid = __popc(valid);
      rw.meta->done = 0;
      rw.meta->redo = 0;
    }
  }
  __syncthreads();
  float m = -INFINITY, s = 0.0f;
  // contiguous shares of the rows, the last group of each cut short
  const int64_t me = blockIdx.x * 8 + warp, all = gridDim.x * 8;
  const int begin = static_cast<int>(me * vocab / all), end = static_cast<int>((me + 1) * vocab / all);
  for (int v0 = begin; v0 < end; v0 += R) {
    float acc[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.0f;
    for (int c = lane * N; c < ld; c += 32 * N) {
      typename A::Raw raw[R];
      const S* w = weight + static_cast<int64_t>(v0) * ldw + c;
      if (c < d) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (v0 + r < end) raw[r] = A::load_raw(w + r * ldw);
      }
      float h[TT][N];
#pragma unroll
      for (int k = 0; k < TT; ++k) {
        if constexpr (N == 1) {
          h[k][0] = hs[k * ld + c];
        } else {
#pragma unroll
          for (int j = 0; j < N; j += 4) {
            const float4 x = *reinterpret_cast<const float4*>(hs + k * ld + c + j);
            h[k][j] = x.x; h[k][j + 1] = x.y; h[k][j + 2] = x.z; h[k][j + 3] = x.w;
          }
        }
      }
      if (c < d) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (v0 + r >= end) continue;
          float x[N];
          A::unpack(raw[r], x);
#pragma unroll
          for (int k = 0; k < TT; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) acc[r * TT + k] = fmaf(x[j], h[k][j], acc[r * TT + k]);
        }
      }
    }
    const float l = warp_transpose_reduce32(acc, lane);
    const int v = v0 + lane / TT;
    if (v < end && t < tokens) {
      if (v == y) rw.lab[t] = l;
      else lse_join(m, s, l, l != l ? l : 1.0f);  // NaN stays in the sum
    }
  }
#pragma unroll
  for (int o = 16; o >= TT; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    lse_join(m, s, m2, s2);
  }
  if (lane < TT) wp[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < tokens) {
    m = wp[0][threadIdx.x].x;
    s = wp[0][threadIdx.x].y;
    for (int w = 1; w < 8; ++w) lse_join(m, s, wp[w][threadIdx.x].x, wp[w][threadIdx.x].y);
    part[blockIdx.x * part_ld + threadIdx.x] = make_float2(m, s);
  }
}

// ------------------------------------------------------------------- loss --
// Joins the (maximum, sum) pieces of each row and writes its loss: 8 rows per
// block, 32 threads along a row's pieces.  Sums over tokens have a fixed
// order: block sums (fp64), added by the last block in block order.
constexpr int XE_LOSS_ROWS = 8;
enum XeReduction { XE_NONE, XE_SUM, XE_MEAN };

// (maximum, sum) of one row over all its pieces (without the label's column):
// valid in threads 0..7, which hold rows blockIdx.x * 8 + threadIdx.x
template <class Join>
__device__ __forceinline__ void join_parts(const float2* __restrict__ part, int parts, int64_t part_ld, int rows,
                                           float& m, float& s, Join join) {
  __shared__ float2 wp[8][XE_LOSS_ROWS];
  const int row = blockIdx.x * XE_LOSS_ROWS + (threadIdx.x & (XE_LOSS_ROWS - 1));
  m = -INFINITY;
  s = 0.0f;
  if (row < rows) {
#pragma unroll 8
    for (int p = threadIdx.x / XE_LOSS_ROWS; p < parts; p += 32) {
      const float2 v = part[p * part_ld + row];
      join(m, s, v.x, v.y);
    }
  }
  // lanes of a warp hold 4 pieces of each of 8 rows; then over the 8 warps
#pragma unroll
  for (int o = 16; o >= XE_LOSS_ROWS; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, m2, s2);
  }
  if ((threadIdx.x & 31) < XE_LOSS_ROWS) wp[threadIdx.x >> 5][threadIdx.x & 31] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < XE_LOSS_ROWS)
    for (int w = 1; w < 8; ++w) join(m, s, wp[w][threadIdx.x].x, wp[w][threadIdx.x].y);
}
struct JoinMax {  // KEEP: sums share the row's shift
  __device__ __forceinline__ void operator()(float& m, float& s, float m2, float s2) const {
    m = fmaxf(m, m2);
    s += s2;
  }
};
struct JoinLse {
  __device__ __forceinline__ void operator()(float& m, float& s, float m2, float s2) const { lse_join(m, s, m2, s2); }
};

// Losses, and what the gradients need of each row.
// KEEP: rows whose logits pass the shift by more than XE_KEEP_RANGE take their
// maximum for it; redo_tile marks their row tiles, which k_xent_gemm then does
// again, and a second launch of this kernel (again = true) with it; both end at
// once when no row is marked.  hr receives the rows r h of the packed rows hp,
// rounded to bf16 (the second operand of dW).
__global__ void __launch_bounds__(256) k_xent_loss(XeRows rw, const float2* __restrict__ part, int parts,
                                                   int64_t part_ld, bool keep, bool again,
                                                   int* __restrict__ redo_tile, int reduction,
                                                   float* __restrict__ loss, double* __restrict__ block_sum,
                                                   const __nv_bfloat16* __restrict__ hp,
                                                   __nv_bfloat16* __restrict__ hr, int ldd) {
  __shared__ double red[256];
  __shared__ float row_r[XE_LOSS_ROWS];
  __shared__ bool last;
  pdl_launch_dependents();
  pdl_wait();
  if (again && rw.meta->redo == 0) return;
  const int rows = rw.meta->rows;
  float m, s;
  if (keep) join_parts(part, parts, part_ld, rows, m, s, JoinMax());
  else join_parts(part, parts, part_ld, rows, m, s, JoinLse());
  const int row0 = blockIdx.x * XE_LOSS_ROWS;
  const int row = row0 + threadIdx.x;
  double mine = 0.0;
  if (threadIdx.x < XE_LOSS_ROWS) {
    float r = 0.0f;
    if (row < rows) {
      const float l = rw.lab[row];
      const bool live = rw.yc[row] >= 0;
      float c = keep ? rw.c[row] : fmaxf(m, l);
      if (keep && live && m - c > XE_KEEP_RANGE) {
        rw.c[row] = m;
        redo_tile[row / XE_TILE] = 1;  // any writer writes the same
        rw.meta->redo = 1;
      }
      // s: sum of exp(l[v] - c) over the other columns; b: the label's own
      if (!keep && m != c) s *= expf(m - c);  // m < c = l (m is -inf when there is no other column)
      const float b = c == l ? 1.0f : expf(l - c);
      const float above = c == l ? log1pf(s) : logf(s + b);  // logsumexp - c
      const float v = c == l ? above : (c - l) + above;
      r = live ? 1.0f / (s + b) : 0.0f;
      rw.lse[row] = c + above;  // not l + v: two large numbers where the label is hopeless
      rw.q[row] = -s / (s + b);
      rw.r[row] = r;
      if (live) {
        if (reduction == XE_NONE) loss[rw.idx[row]] = v;
        mine = static_cast<double>(v);
      }
    }
    row_r[threadIdx.x] = r;
  }
  red[threadIdx.x] = mine;
  __syncthreads();
  if (hr != nullptr) {
    const int upto = (rows + XE_TILE - 1) / XE_TILE * XE_TILE;
    const int pieces = ldd / 8;
    for (int i = threadIdx.x; i < XE_LOSS_ROWS * pieces; i += 256) {
      const int k = i / pieces;
      if (row0 + k >= upto) break;
      const int64_t at = static_cast<int64_t>(row0 + k) * ldd + static_cast<int64_t>(i - k * pieces) * 8;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const float f = row_r[k];
      if (f != 0.0f) {  // ignored and padding rows stay zero whatever they hold
        Vec16<__nv_bfloat16>::load(hp + at, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= f;
      }
      Vec16<__nv_bfloat16>::store(hr + at, x);
    }
  }
  if (reduction == XE_NONE) return;
  if (threadIdx.x == 0) {
    double b = 0.0;
    for (int i = 0; i < XE_LOSS_ROWS; ++i) b += red[i];
    block_sum[blockIdx.x] = b;
    __threadfence();
    last = atomicAdd(&rw.meta->done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double acc = 0.0;
  for (int b = threadIdx.x; b < static_cast<int>(gridDim.x); b += 256)
    acc += *static_cast<volatile double*>(&block_sum[b]);
  red[threadIdx.x] = acc;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (static_cast<int>(threadIdx.x) < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    rw.meta->done = 0;
    // no token left: 0 for the sum, NaN for the mean
    *loss = static_cast<float>(reduction == XE_MEAN ? red[0] / rw.meta->valid : red[0]);
  }
}

// -------------------------------------------------------------- dh output --
// The loss's gradient as a factor of the rows' gradients (NONE: in dl already)
__device__ __forceinline__ float xe_scale(const XeRows& rw, const float* grad, int reduction) {
  if (reduction == XE_NONE) return 1.0f;
  const float g = grad != nullptr ? *grad : 1.0f;
  const int valid = rw.meta->valid;
  return reduction == XE_SUM ? g : (valid > 0 ? g / valid : 0.0f);
}

// d_hidden[t] = scale * (f sum over slots of acc[slot][pos[t]] + e W[y]), zero
// for an ignored token.  KEEP: f = r, e = p[y] - 1; pieces: f = 1 (null),
// e = g (p[y] - 1) for bf16 and 0 (null) for fp32, whose sum has the label's.
template <class D>
__global__ void __launch_bounds__(256) k_xent_dhidden(const float* __restrict__ acc, int slots, int64_t slot_size,
                                                      int64_t lda, XeRows rw, const float* __restrict__ grad,
                                                      int reduction, const float* __restrict__ f_rows,
                                                      const float* __restrict__ e_rows,
                                                      const D* __restrict__ weight, int64_t ldw, int64_t vocab,
                                                      int64_t tokens, int d, D* __restrict__ out) {
  pdl_launch_dependents();
  pdl_wait();
  const float scale = xe_scale(rw, grad, reduction);
  const int pieces = (d + 7) / 8;
  const int64_t total = tokens * pieces;
  const bool vec = d % 8 == 0 && rows_vec(out, d);
  const bool wvec = rows_vec(weight, ldw);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = i / pieces;
    const int c = static_cast<int>(i - t * pieces) * 8;
    const int r = rw.pos[t];
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r >= 0) {
      const float* a = acc + static_cast<int64_t>(r) * lda + c;
#pragma unroll 8
      for (int s = 0; s < slots; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(a + s * slot_size);
        const float4 y = *reinterpret_cast<const float4*>(a + s * slot_size + 4);
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      }
      if (e_rows != nullptr && rw.yc[r] < vocab) {
        const float f = f_rows != nullptr ? f_rows[r] : 1.0f, e = e_rows[r];
        float w[8];
        load8(weight + static_cast<int64_t>(rw.yc[r]) * ldw, c, d, wvec, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fmaf(v[j], f, e * w[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= scale;
    }
    D* o = out + t * d + c;
    if (vec) {
      store_row<D, true>(o, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e[1] = {v[j]};
        if (c + j < d) RowAccess<D, false>::store(o + j, e);
      }
    }
  }
}

// dst [rows][d] <- src [rows][lds], bf16, eight consecutive elements of dst a
// thread (dst rows of an odd width have no alignment of their own).
__global__ void __launch_bounds__(256) k_xent_unpad(const __nv_bfloat16* __restrict__ src, int64_t lds, int d,
                                                    int64_t total, __nv_bfloat16* __restrict__ dst) {
  pdl_launch_dependents();
  pdl_wait();
  const bool vec = (reinterpret_cast<uintptr_t>(dst) & 15u) == 0;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 8; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x * 8) {
    int64_t r = i / d;
    int c = static_cast<int>(i - r * d);
    __align__(16) __nv_bfloat16 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i + j < total) v[j] = src[r * lds + c];
      if (++c == d) {
        c = 0;
        ++r;
      }
    }
    if (vec && i + 8 <= total) {
      *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < total) dst[i + j] = v[j];
    }
  }
}

// x *= *factor and y *= *factor, unless it is 1 (the gradients of the KEEP way are those of a
// loss whose own gradient is 1).  They were rounded to D when they were computed
// and are rounded again here, which a power of two leaves exact: held in fp32
// until then, dW would take twice its memory between the calls.
template <class D>
__global__ void __launch_bounds__(256) k_xent_scale(const float* __restrict__ factor, D* __restrict__ x, int64_t nx,
                                                    D* __restrict__ y, int64_t ny) {
  pdl_launch_dependents();
  pdl_wait();
  const float f = *factor;
  if (f == 1.0f) return;
  constexpr int N = Vec16<D>::N;
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t nt = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int t = 0; t < 2; ++t) {
    D* p = t == 0 ? x : y;
    const int64_t n = t == 0 ? nx : ny;
    const int64_t nv = (reinterpret_cast<uintptr_t>(p) & 15u) == 0 ? n / N : 0;
    for (int64_t i = tid; i < nv; i += nt) {
      float v[N];
      Vec16<D>::load(p + i * N, v);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] *= f;
      Vec16<D>::store(p + i * N, v);
    }
    for (int64_t i = nv * N + tid; i < n; i += nt) {
      const float v[1] = {static_cast<float>(p[i]) * f};
      RowAccess<D, false>::store(p + i, v);
    }
  }
}

// ------------------------------------------------------------------- GEMM --
// One product of a launch: A rows (M) x B rows (N) over K.
struct XeProduct {
  int a_plane_rows, b_plane_rows;  // y offset between planes of an operand
  int M;                           // host bound of the rows
  int N, K;
};

__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

struct XeArgs {
  XeRows rw;
  XeProduct p[2];  // STATS, KEEP, DLOGITS: p[0]; GRADS: p[0] = dh, p[1] = dW
  // STATS, KEEP: (maximum, sum) of each row over a unit's columns
  int run;  // column tiles per unit
  float2* part;
  int64_t part_ld;
  const int* redo_tile;  // KEEP, second launch: only the row tiles marked here
  // KEEP: E; DLOGITS: gradient of the logits of columns [v0, v0 + N);
  // [PLANES][dl_plane_rows][ldl], columns up to a multiple of 64 written
  int v0;
  const float* grad;
  int reduction;
  __nv_bfloat16* dl;
  int64_t dl_plane_rows;
  int64_t ldl;
  float* label_grad;   // DLOGITS, bf16: g (p[y] - 1) of each row, by the units of the first column tile
  // GRADS
  int dh_slots;        // K slices of dh, each with a buffer of its own
  int dh_accumulate;   // add to dh_acc (pieces after the first)
  float* dh_acc;       // [slots][rows][dh_ld]
  int64_t dh_slot_size;
  int64_t dh_ld;
  void* dw;            // rows of this piece, [N rows][d]; the padded rows where those are what is read
  int64_t dw_ld;
  int dw_bf16;
  int dw_tma;          // dW through the tensor map tmC (16-byte rows)
  const float* label_rows;  // added to dW before scaling: row v's is label_rows[label_span[v].x],
  const int2* label_span;   // where that span is not empty
  int do_dh, do_dw;
};

template <int PLANES>
struct XeCfg {
  // bf16: two accumulators side by side read one A tile; fp32: one, so that
  // the epilogue can add up accumulations in registers
  static constexpr int kHalves = PLANES == 1 ? 2 : 1;
  static constexpr int kTileN = XE_TILE * kHalves;
  // fp32: all planes of a K block in one stage, for its six products
  static constexpr int kStageBytes = PLANES * G2_A_BYTES + (PLANES == 1 ? kHalves : PLANES) * G2_B_BYTES;
  static constexpr int kStages = PLANES == 1 ? 4 : 2;
  // blocks by which the second accumulator's MMAs follow the first's at the
  // end of a tile and the start of the next: while one accumulator works the
  // epilogue empties the other.  In between they go together, so that the
  // ring's stages are free for the copies.
  static constexpr int kLag = 2;
  static constexpr int kBOff = PLANES * G2_A_BYTES;  // B within a stage
  // K blocks of dh that take as long as a tile of dW at the least (5 to 7 us,
  // its loads, accumulator hand-over and stores).  Gradients of 120, 256 and 600
  // tokens of 100 277 x 1024, in us: 282, 302, 450 with 6 (bf16), 257, 275, 429
  // with 13, 259, 275, 422 with 16, 263, 280, 425 with 20; of 300 x 32 000 x
  // 512: 170, 146, 137, 135.  An fp32 K block has six products.
  static constexpr int kStoreKb = PLANES == 1 ? 16 : 6;
};
struct XeCtl {
  uint64_t full[6];
  uint64_t empty[6];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
// Warps 0 (copies), 1 (MMA), 2 and 3 (idle), 4.. (epilogue).  The epilogue
// holds 128 accumulator columns per lane, more than an even split of the
// registers allows, so the first four warps give registers up: the launch's
// 384 x 168 are divided 128 x 88 + 256 x 208, the same sum (the host checks that
// the kernel was compiled for XE_LAUNCH_REGS before it launches it).
constexpr int XE_EPI_WARPS = 8;
constexpr int XE_EPI_WARP0 = 4;
constexpr int XE_THREADS = 32 * (XE_EPI_WARP0 + XE_EPI_WARPS);
constexpr int XE_LAUNCH_REGS = 168, XE_LEAN_REGS = 88, XE_EPI_REGS = 208;
static_assert(XE_EPI_WARP0 * XE_LEAN_REGS + XE_EPI_WARPS * XE_EPI_REGS <=
                  (XE_EPI_WARP0 + XE_EPI_WARPS) * XE_LAUNCH_REGS,
              "register split");

// mbar_wait, expanded in place (a kernel that moves registers between its
// warps makes no calls)
__device__ __forceinline__ bool xe_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int site) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  const uint64_t limit = *static_cast<volatile unsigned long long*>(&g_wait_limit_ns);
#pragma unroll 1
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0u) {
      if (abort != nullptr && *abort) return false;
      if (global_timer_ns() - t0 > limit) {
        if (abort != nullptr) *abort = 1;
        record_error(err, ETHOS_ERR_TIMEOUT_BASE + site);
        return false;
      }
    }
  }
}
// bf16 outputs (E, dl, dW) leave through TMA stores of each warp's staged 32 x 64
// block: written from the lanes, whose rows are far apart, dW of 1000 tokens
// (100 277 x 1024) took 235 us instead of 210
constexpr int XE_STG_WARP_BYTES = 32 * 128;
template <int PLANES>
constexpr int xe_smem() {
  return XeCfg<PLANES>::kStages * XeCfg<PLANES>::kStageBytes + XE_EPI_WARPS * XE_STG_WARP_BYTES + 1024 +
         static_cast<int>(sizeof(XeCtl));
}
static_assert(xe_smem<1>() <= 227 * 1024 && xe_smem<3>() <= 227 * 1024, "shared memory");

// One accumulation: tile at (m0, n0) of product `prod`, K blocks [kb0, kb1)
// over all plane products.
struct XeStep {
  int prod, m0, n0, kb0, kb1;
  bool first, last;      // of its unit
  bool kfirst, klast;    // of its tile
  bool second;           // the tile has columns in the second accumulator
  int slot;
};

// The units of a pair, as a sequence of accumulations; every role of both
// CTAs walks the same sequence.
template <int MODE, int PLANES>
struct XeWalk {
  static constexpr int TN = XeCfg<PLANES>::kTileN;
  const XeArgs& a;
  int num_m, num_n, nkb, pair, pairs;
  int u;           // unit (its number among the pair's units in GRADS)
  int units;       // units of the launch (of the pair in GRADS)
  int c, j;        // column tile and accumulation within the unit
  int cols;        // STATS, KEEP: units along the columns; DLOGITS: column tiles
  int kb_w;        // GRADS: K blocks of dW
  int kb_slot;     // GRADS: K blocks of dh per slot
  int long_units, my_long;     // GRADS: dh units of the launch, of this pair
  int na, diff, extra;         // GRADS: see below
  __device__ XeWalk(const XeArgs& args, int rows, int pair_, int pairs_) : a(args), pair(pair_), pairs(pairs_) {
    num_m = (rows + XE_TILE - 1) / XE_TILE;
    num_n = (a.p[0].N + TN - 1) / TN;
    nkb = (a.p[0].K + G2_BK - 1) / G2_BK;
    c = j = 0;
    if (MODE != XE_GRADS) {
      cols = MODE == XE_DLOGITS ? num_n : (num_n + a.run - 1) / a.run;
      u = pair;
      units = num_m * cols;
      return;
    }
    // dh units (long_units of them, kb_slot blocks each) in turn, so that the
    // pairs below `extra` have one more than the others.  Then dW tiles (kb_w
    // blocks each): na each, `diff` more to the others (the dW tiles that one
    // dh unit is worth; writing a tile takes about as long as kStoreKb
    // blocks, so short contractions do not make it cheaper), and what is left
    // one by one, the others first.
    kb_slot = (nkb + a.dh_slots - 1) / a.dh_slots;
    long_units = a.do_dh ? num_m * num_n * a.dh_slots : 0;
    kb_w = (rows + G2_BK - 1) / G2_BK;
    const int n2 = a.do_dw ? (a.p[1].M + XE_TILE - 1) / XE_TILE * num_n : 0;
    extra = long_units % pairs;
    const int others = pairs - extra;
    my_long = long_units / pairs + (pair < extra ? 1 : 0);
    constexpr int least = XeCfg<PLANES>::kStoreKb;
    diff = (max(kb_slot, least) + max(kb_w, least) / 2) / max(kb_w, least);
    na = (n2 - diff * others) / pairs;
    if (n2 < diff * others) {
      na = 0;
      diff = n2 / others;
    }
    const int rem = n2 - na * pairs - diff * others;
    u = 0;
    units = my_long + na + (pair >= extra ? diff : 0) + ((pair - extra + pairs) % pairs < rem ? 1 : 0);
  }
  // the next accumulation; false when the pair's units are done
  __device__ bool next(XeStep& s) {
    while (true) {
      if (u >= units) return false;
      int steps = 1, ntiles = 1;
      s.slot = 0;
      s.prod = 0;
      int kb0 = 0, kb1 = nkb;
      if (MODE != XE_GRADS) {
        // row tiles in groups of XE_GROUP_M, all columns of a group before the
        // next: A's group and one column tile of B (or a run of them) in L2
        const int per_group = XE_GROUP_M * cols;
        const int g = u / per_group;
        const int gm = min(XE_GROUP_M, num_m - g * XE_GROUP_M);
        const int v = u - g * per_group;
        const int cu = v / gm;
        const int mt = g * XE_GROUP_M + v % gm;
        if (MODE == XE_KEEP && a.redo_tile != nullptr && !a.redo_tile[mt]) {
          u += pairs;
          continue;
        }
        s.m0 = mt * XE_TILE;
        if (MODE == XE_DLOGITS) {
          s.n0 = cu * TN;
        } else {
          ntiles = min(a.run, num_n - cu * a.run);
          s.n0 = (cu * a.run + c) * TN;
          s.slot = cu;
        }
      } else if (u < my_long) {
        const int l = pair + u * pairs;
        const int t = l % (num_m * num_n);
        s.slot = l / (num_m * num_n);
        s.m0 = (t / num_n) * XE_TILE;
        s.n0 = (t % num_n) * TN;
        kb0 = s.slot * kb_slot;
        kb1 = min(nkb, kb0 + kb_slot);
      } else {
        const int i = u - my_long, others = pairs - extra;
        const int t = i < na ? i * pairs + pair
                      : pair >= extra && i < na + diff
                          ? na * pairs + (i - na) * others + pair - extra
                          : na * pairs + diff * others + (pair - extra + pairs) % pairs;
        s.prod = 1;
        s.m0 = (t / num_n) * XE_TILE;
        s.n0 = (t % num_n) * TN;
        kb1 = kb_w;
      }
      const int fl = PLANES == 1 ? (1 << 28) : 1;  // K blocks per accumulation
      steps = max(1, (kb1 - kb0 + fl - 1) / fl);
      s.kb0 = kb0 + j * fl;
      s.kb1 = min(kb1, s.kb0 + fl);
      s.kfirst = j == 0;
      s.klast = j + 1 >= steps;
      s.first = j == 0 && c == 0;
      s.last = s.klast && c + 1 >= ntiles;
      s.second = PLANES == 1 && s.n0 + XE_TILE < a.p[s.prod].N;
      if (!s.klast) {
        ++j;
      } else {
        j = 0;
        if (!s.last) {
          ++c;
        } else {
          c = 0;
          u += MODE == XE_GRADS ? 1 : pairs;
        }
      }
      return true;
    }
  }
};

// Plane pairs of a product, smallest first: A = 0, 2, 1, 1, 0, 0 and
// B = 2, 0, 1, 0, 1, 0 (0 the leading plane).
__device__ __forceinline__ int xe_plane_a(int seg) { return (0x058 >> (2 * seg)) & 3; }
__device__ __forceinline__ int xe_plane_b(int seg) { return (0x112 >> (2 * seg)) & 3; }

__device__ __forceinline__ void st_v8(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f,
                                      uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e),
               "r"(f), "r"(g), "r"(h)
               : "memory");
}

// 32 columns of this lane's row from `col` on, of a matrix with `cols`
// columns: bf16 rows that TMA stores cannot take (dW at an odd address), and
// fp32 ones (32-byte stores, whole sectors; `align`: the byte alignment that
// every row start shares, 32, 16 or less; `acc`: added to what is there)
__device__ __forceinline__ void row_store_bf16(__nv_bfloat16* row, int col, int cols, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (col + j < cols) row[col + j] = __float2bfloat16_rn(v[j]);
}
__device__ __forceinline__ void row_store_f32(float* row, int col, int cols, int align, float (&v)[32], bool acc) {
  if (align >= 16 && col + 32 <= cols) {
    float* p = row + col;
    if (acc) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 o = *reinterpret_cast<const float4*>(p + 4 * j);
        v[4 * j] += o.x; v[4 * j + 1] += o.y; v[4 * j + 2] += o.z; v[4 * j + 3] += o.w;
      }
    }
    if (align >= 32) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        st_v8(p + 8 * j, __float_as_uint(v[8 * j]), __float_as_uint(v[8 * j + 1]), __float_as_uint(v[8 * j + 2]),
              __float_as_uint(v[8 * j + 3]), __float_as_uint(v[8 * j + 4]), __float_as_uint(v[8 * j + 5]),
              __float_as_uint(v[8 * j + 6]), __float_as_uint(v[8 * j + 7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float4*>(p + 4 * j) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col + j < cols) row[col + j] = acc ? row[col + j] + v[j] : v[j];
  }
}
// a when kFirst, else b (arrays of which the other one has no elements to speak of)
template <bool kFirst, class A, class B>
__device__ __forceinline__ auto& pick(A& a, B& b) {
  if constexpr (kFirst) return a;
  else return b;
}
// 64 bf16 columns of the warp's 32 rows (v0, v1: this lane's row) at (col, row0)
// of the matrix behind tm, through the warp's staging block
__device__ __forceinline__ void block_store_bf16(const CUtensorMap* tm, uint8_t* stg, int lane, const float (&v0)[32],
                                                 const float (&v1)[32], int col, int row0) {
  if (lane == 0) bulk_wait_read<0>();  // the block's last store has read it
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* x = (c == 0 ? v0 : v1) + 8 * j;
      w[j] = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                        pack_bf16x2(x[6], x[7]));
    }
    stage_row_sw128(stg, lane, c, w);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(tm, stg, col, row0);
    bulk_commit();
  }
}
__device__ __forceinline__ int byte_align(const void* p, int64_t pitch_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(pitch_bytes);
  return (x & 31u) == 0 ? 32 : ((x & 15u) == 0 ? 16 : 1);
}

// One lane of a converged warp.  The copy and MMA warps run their loops whole
// and only issue from one lane, so that addresses and descriptors stay in
// uniform registers: with the loops on a single lane, issue bound the MMA warp
// (about 1750 cycles for the eight MMAs of a block that take 1024, with or
// without copies).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
// The 128-byte-swizzle descriptors of umma_desc_sw128 (K-major) and
// umma_desc_sw128_mn (LBO 8192): constant high word, low word of the address.
constexpr uint32_t XE_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t xe_desc_lo(uint32_t smem_addr, bool mn) {
  return ((smem_addr & 0x3FFFFu) >> 4) | (mn ? (8192u >> 4) << 16 : 1u << 16);
}
__device__ __forceinline__ void xe_mma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(XE_DESC_HI), "r"(accumulate)
      : "memory");
}

template <int MODE, int PLANES>
__global__ void __launch_bounds__(XE_THREADS, 1)
    k_xent_gemm(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmB0,
                const __grid_constant__ CUtensorMap tmA1, const __grid_constant__ CUtensorMap tmB1,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ XeArgs args, int* err) {
  using Cfg = XeCfg<PLANES>;
  constexpr int HALVES = Cfg::kHalves;
  constexpr int STAGES = Cfg::kStages;
  constexpr int STAGE_BYTES = Cfg::kStageBytes;
  constexpr int CHUNKS = (XE_TILE / 32) / (XE_EPI_WARPS / 4);  // 32-column chunks per epilogue warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t* stg_s = smem + STAGES * STAGE_BYTES;
  XeCtl* ctl = reinterpret_cast<XeCtl*>(stg_s + XE_EPI_WARPS * XE_STG_WARP_BYTES);
  const int warp = warp_id();
  const int lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(blockIdx.x) >> 1;
  const int pairs = static_cast<int>(gridDim.x) >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ctl->acc_full[b], 1);
      mbar_init(&ctl->acc_empty[b], 2 * XE_EPI_WARPS);
    }
    mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&ctl->tmem_base, 2 * XE_TILE);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers initialised before any remote arrive or commit
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  pdl_launch_dependents();
  pdl_wait();  // set-up above touched only shared memory, TMEM and parameters
  int rows = *static_cast<const volatile int*>(&args.rw.meta->rows);
  if (MODE == XE_KEEP && args.redo_tile != nullptr && *static_cast<const volatile int*>(&args.rw.meta->redo) == 0)
    rows = 0;  // no row to do again
  volatile int* abort = &ctl->abort;

  if (warp < XE_EPI_WARP0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XE_LEAN_REGS));
    if (warp == 0) {
      XeWalk<MODE, PLANES> walk(args, rows, pair, pairs);
      XeStep st;
      RingPos rp;
      bool ok = true;
      while (ok && walk.next(st)) {
        const int m0 = st.m0 + static_cast<int>(rank) * G2_BM;
        // a half tile of rows past the last is filled with zeros (a coordinate
        // out of range), which reads no memory
        const int a_row = m0 < rows ? m0 : XE_NO_ROW;
        const int n0 = st.n0 + static_cast<int>(rank) * (XE_TILE / 2);
        const uint32_t bytes = 2u * (PLANES * G2_A_BYTES + (PLANES == 1 ? (st.second ? 2 : 1) : PLANES) * G2_B_BYTES);
        const CUtensorMap* ta = st.prod == 0 ? &tmA0 : &tmA1;
        const CUtensorMap* tb = st.prod == 0 ? &tmB0 : &tmB1;
        const XeProduct& p = args.p[st.prod];
        for (int kb = st.kb0; kb < st.kb1; ++kb) {
          ok = __all_sync(0xffffffffu, xe_wait(&ctl->empty[rp.stage], rp.phase ^ 1u, abort, err, 1));
          if (!ok) break;
          uint8_t* sa = smem + rp.stage * STAGE_BYTES;
          uint8_t* sb = sa + Cfg::kBOff;
          const uint32_t fb = cluster_map(smem_u32(&ctl->full[rp.stage]), 0);
          if (elect_one()) {
            if (leader) mbar_arrive_expect_tx(&ctl->full[rp.stage], bytes);
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl) {
              const int ya = pl * p.a_plane_rows, yb = pl * p.b_plane_rows;
              uint8_t* da = sa + pl * G2_A_BYTES;
              uint8_t* db = sb + pl * G2_B_BYTES;
              if (MODE == XE_GRADS && st.prod == 1) {
                tma_load_2d_pair(da, ta, fb, m0, ya + kb * G2_BK);
                tma_load_2d_pair(da + 8192, ta, fb, m0 + 64, ya + kb * G2_BK);
              } else {
                tma_load_2d_pair(da, ta, fb, kb * G2_BK, ya + a_row);
              }
              if (MODE == XE_GRADS) {
                tma_load_2d_pair(db, tb, fb, n0, yb + kb * G2_BK);
                tma_load_2d_pair(db + 8192, tb, fb, n0 + 64, yb + kb * G2_BK);
              } else {
                tma_load_2d_pair(db, tb, fb, kb * G2_BK, yb + n0);
              }
            }
            if (PLANES == 1 && st.second) {  // the second accumulator's columns
              if (MODE == XE_GRADS) {
                tma_load_2d_pair(sb + G2_B_BYTES, tb, fb, n0 + XE_TILE, kb * G2_BK);
                tma_load_2d_pair(sb + G2_B_BYTES + 8192, tb, fb, n0 + XE_TILE + 64, kb * G2_BK);
              } else {
                tma_load_2d_pair(sb + G2_B_BYTES, tb, fb, kb * G2_BK, n0 + XE_TILE);
              }
            }
          }
          __syncwarp();
          rp.advance(STAGES);
        }
      }
      if (!ok) {
        // as in k_gemm2sm: both CTAs' copies complete on the leader's
        // barriers; the peer waits a bounded 100 us for its own to land
        if (leader) {
          int sg = rp.stage;
          uint32_t ph = rp.phase;
          for (int i = 0; i < STAGES && i < rp.issued; ++i) {
            if (sg == 0) {
              sg = STAGES - 1;
              ph ^= 1u;
            } else {
              --sg;
            }
            xe_wait(&ctl->full[sg], ph, nullptr, err, 5);
          }
        } else {
          const uint64_t t0 = global_timer_ns();
          while (global_timer_ns() - t0 < 100000ull) {
          }
        }
      }
  } else if (warp == 1) {
    if (leader) {
      // One stream of K blocks per accumulator.  With two, the second follows
      // kLag blocks behind the first and releases the ring's stages.
      XeWalk<MODE, PLANES> w0(args, rows, pair, pairs), w1(args, rows, pair, pairs);
      XeStep s0, s1;
      int stage0 = 0, stage1 = 0;
      uint32_t phase0 = 0;
      int it0 = 0, it1 = 0;          // accumulations begun, per accumulator stream
      int b0 = 0, n0 = 0;            // block of stream 0's step, and their number
      int b1 = 0, n1 = 0;
      int ahead = 0;                 // blocks of stream 0 that stream 1 has yet to do
      int begun0 = 0, done1 = 0;     // tiles begun by stream 0, finished by stream 1
      bool more0 = true, more1 = HALVES == 2;
      bool ok = true;
      const uint32_t smem0 = smem_u32(smem);
      auto mma_block = [&](const XeStep& st, int stage, int half, uint32_t d, bool first) {
        const bool a_mn = MODE == XE_GRADS && st.prod == 1;
        constexpr bool b_mn = MODE == XE_GRADS;
        const uint32_t idesc = umma_idesc_bf16_f32_major(2 * G2_BM, XE_TILE, a_mn, b_mn);
        const uint32_t a_base = smem0 + static_cast<uint32_t>(stage * STAGE_BYTES);
        const uint32_t a_lo = xe_desc_lo(a_base, a_mn);
        const uint32_t b_lo = xe_desc_lo(a_base + static_cast<uint32_t>(Cfg::kBOff + half * G2_B_BYTES), b_mn);
        const uint32_t a_step = a_mn ? 2048u >> 4 : 32u >> 4;
        constexpr uint32_t b_step = b_mn ? 2048u >> 4 : 32u >> 4;
        if (elect_one()) {
#pragma unroll
          for (int seg = 0; seg < (PLANES == 1 ? 1 : 6); ++seg) {
            const uint32_t ao = PLANES == 1 ? 0u : static_cast<uint32_t>(xe_plane_a(seg) * (G2_A_BYTES >> 4));
            const uint32_t bo = PLANES == 1 ? 0u : static_cast<uint32_t>(xe_plane_b(seg) * (G2_B_BYTES >> 4));
#pragma unroll
            for (int k = 0; k < G2_BK / 16; ++k)
              xe_mma(d, a_lo + ao + k * a_step, b_lo + bo + k * b_step, idesc,
                     (!first || seg > 0 || k > 0) ? 1u : 0u);
          }
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit_pair_mc(bar, 0x3);
        __syncwarp();
      };
      while (ok && (more0 || more1)) {
        // stream 0 may begin tile j once stream 1 is through tile j - 2: the
        // epilogue takes the accumulators in the order of the tiles
        const bool go0 = more0 && (HALVES == 1 || b0 != n0 || begun0 <= done1 + 1);
        if (go0) {
          if (b0 == n0) {  // next step with blocks
            b0 = n0 = 0;
            while (n0 == 0 && (more0 = w0.next(s0))) n0 = max(0, s0.kb1 - s0.kb0);
          }
          if (more0) {
            const int buf = HALVES == 2 ? 0 : it0 & 1;
            const uint32_t par = static_cast<uint32_t>(HALVES == 2 ? it0 : it0 >> 1) & 1u;
            if (b0 == 0) {
              ++begun0;
              ok = __all_sync(0xffffffffu, xe_wait(&ctl->acc_empty[buf], par ^ 1u, abort, err, 2));
              if (!ok) break;
            }
            ok = __all_sync(0xffffffffu, xe_wait(&ctl->full[stage0], phase0, abort, err, 3));
            if (!ok) break;
            tc_fence_after();
            mma_block(s0, stage0, 0, tmem + static_cast<uint32_t>(buf * XE_TILE), b0 == 0);
            if (HALVES == 1) commit(&ctl->empty[stage0]);
            if (++b0 == n0) {
              commit(&ctl->acc_full[buf]);
              ++it0;
            }
            if (++stage0 == STAGES) {
              stage0 = 0;
              phase0 ^= 1u;
            }
            ++ahead;
          }
        }
        // b0: blocks of the current tile that stream 0 has done (n0 at its end)
        const int lag = more0 && go0 && (b0 <= Cfg::kLag || n0 - b0 <= Cfg::kLag) ? Cfg::kLag : 0;
        while (HALVES == 2 && more1 && (ahead > lag || !more0 || !go0)) {
          if (b1 == n1) {
            b1 = n1 = 0;
            while (n1 == 0 && (more1 = w1.next(s1))) n1 = max(0, s1.kb1 - s1.kb0);
          }
          if (more1) {
            if (s1.second) {
              if (b1 == 0) {
                ok = __all_sync(0xffffffffu, xe_wait(&ctl->acc_empty[1], (static_cast<uint32_t>(it1) & 1u) ^ 1u, abort,
                                                     err, 2));
                if (!ok) break;
                tc_fence_after();
              }
              mma_block(s1, stage1, 1, tmem + static_cast<uint32_t>(XE_TILE), b1 == 0);
            }
            commit(&ctl->empty[stage1]);
            if (++b1 == n1) {
              ++done1;
              if (s1.second) {
                commit(&ctl->acc_full[1]);
                ++it1;
              }
            }
            if (++stage1 == STAGES) stage1 = 0;
            --ahead;
            if (!go0 && begun0 <= done1 + 1) break;  // stream 0 may go on
          }
        }
      }
      if (!__all_sync(0xffffffffu, ok && !*abort)) {
        // drain: every MMA of the pair done before the memory goes away (the
        // same lane issued them all)
        if (elect_one()) umma_commit_pair(&ctl->drain);
        __syncwarp();
        xe_wait(&ctl->drain, 0, nullptr, err, 6);
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(XE_EPI_REGS));
    // Epilogue warps never leave the walk early: after an abort they skip the
    // work but still arrive on every acc_empty phase.  A warp takes its 128
    // columns of an accumulator into registers and releases it before it
    // works on them.
    XeWalk<MODE, PLANES> walk(args, rows, pair, pairs);
    XeStep st;
    const int q = warp & 3;
    const int ch = (warp - XE_EPI_WARP0) >> 2;  // column half of an accumulator
    uint8_t* stg = stg_s + (warp - XE_EPI_WARP0) * XE_STG_WARP_BYTES;
    const uint32_t acc_empty0 = cluster_map(smem_u32(&ctl->acc_empty[0]), 0);
    const uint32_t acc_empty1 = cluster_map(smem_u32(&ctl->acc_empty[1]), 0);
    int it0 = 0, it1 = 0;  // accumulations taken (HALVES 1: all in it0)
    bool ok = true;
    // per-row state (this lane's row of the tile)
    int y = -1;
    bool live = false, all_live = false;
    float run_m = -INFINITY, run_s = 0.0f;  // STATS, KEEP
    float c2 = 0.0f;                        // KEEP: shift, DLOGITS: logsumexp, in units of log 2
    float g = 1.0f, at_label = 0.0f;        // DLOGITS
    const float scale = MODE == XE_GRADS ? xe_scale(args.rw, args.grad, args.reduction) : 1.0f;
    float sum[HALVES == 1 ? CHUNKS : 1][32];  // fp32: accumulations added up
    while (walk.next(st)) {
      const bool any = st.kb0 < st.kb1;
      const int row = st.m0 + static_cast<int>(rank) * G2_BM + q * 32 + lane;
      // bf16 KEEP, DLOGITS: dW reads whole K blocks of rows, dh's rows past the
      // last go nowhere (300 tokens of which 120 have labels: 298 -> 292 us)
      const bool stored = PLANES != 1 || row - lane < (rows + G2_BK - 1) / G2_BK * G2_BK;
      if ((MODE == XE_STATS || MODE == XE_KEEP) && st.first) {
        live = row < rows;
        y = live ? args.rw.yc[row] : -1;
        if (MODE == XE_KEEP) {
          live = y >= 0;
          c2 = live ? args.rw.c[row] * XE_LOG2E : 0.0f;
        }
        all_live = __all_sync(0xffffffffu, live);
        run_m = -INFINITY;
        run_s = 0.0f;
      }
      if (MODE == XE_DLOGITS && st.kfirst) {
        y = row < rows ? args.rw.yc[row] : -1;
        live = y >= 0;
        c2 = live ? args.rw.lse[row] * XE_LOG2E : 0.0f;
        at_label = live ? args.rw.q[row] : 0.0f;
        g = args.reduction == XE_NONE && live ? args.grad[args.rw.idx[row]] : 1.0f;
        if (PLANES == 1) {  // the label's entry goes its own way, in fp32
          if (args.label_grad != nullptr && st.n0 == 0 && ch == 0 && row < rows) args.label_grad[row] = at_label * g;
          at_label = 0.0f;
        }
      }
      // GRADS: this row's label row, looked up and on its way before the wait
      // (loads of it afterwards, by one lane of few warps, took 9 of 146 us of
      // the gradients of 120 tokens of 100 277 x 1024)
      const float* extra = nullptr;
      if (MODE == XE_GRADS && st.prod == 1 && args.label_rows != nullptr && row < args.p[1].M) {
        const int2 sp = args.label_span[row];
        if (sp.x < sp.y) {
          extra = args.label_rows + static_cast<int64_t>(sp.x) * args.p[1].N;
#pragma unroll
          for (int half = 0; half < HALVES; ++half)
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
              const int col = st.n0 + half * XE_TILE + (ch * CHUNKS + k) * 32;
              if (col < args.p[1].N) prefetch_l1(extra + col);
            }
        }
      }
#pragma unroll 1
      for (int half = 0; half < (st.second ? 2 : 1); ++half) {
        const int col0 = st.n0 + half * XE_TILE + ch * CHUNKS * 32;
        if (!any) {  // no rows to add up: zeros
          if (MODE == XE_GRADS && st.prod == 1 && row < args.p[1].M) {
            const int d = args.p[1].N;
            for (int c = col0; c < min(d, col0 + CHUNKS * 32); ++c) {
              if (args.dw_bf16) static_cast<__nv_bfloat16*>(args.dw)[row * args.dw_ld + c] = __float2bfloat16_rn(0.0f);
              else static_cast<float*>(args.dw)[row * args.dw_ld + c] = 0.0f;
            }
          }
          continue;
        }
        const int buf = HALVES == 2 ? half : it0 & 1;
        const int n = HALVES == 2 ? (half ? it1 : it0) : it0 >> 1;
        if (ok) ok = __all_sync(0xffffffffu, xe_wait(&ctl->acc_full[buf], static_cast<uint32_t>(n) & 1u, abort, err, 4));
        if (half) ++it1;
        else ++it0;
        tc_fence_after();
        float fresh[HALVES == 2 ? CHUNKS : 1][32];
        float(&v)[CHUNKS][32] = pick<HALVES == 1>(sum, fresh);
        if (ok) {
          const uint32_t ta = tmem_addr(tmem, q * 32, buf * XE_TILE + ch * CHUNKS * 32);
          if constexpr (HALVES == 2) {
#pragma unroll
            for (int k = 0; k < CHUNKS; k += 2) {
              float x[64];
              tmem_ld64(ta + 32 * k, x);
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                v[k][i] = x[i];
                v[k + 1][i] = x[32 + i];
              }
            }
          } else {
            if (st.kfirst) {
#pragma unroll
              for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int i = 0; i < 32; ++i) v[k][i] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
              float x[32];
              tmem_ld32(ta + 32 * k, x);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[k][i] += x[i];
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(buf ? acc_empty1 : acc_empty0);
        if (!ok || !st.klast) continue;
        if (MODE == XE_STATS || MODE == XE_KEEP) {
          const int N = args.p[0].N;
#pragma unroll
          for (int k = 0; k < CHUNKS; ++k) {
            const int col = col0 + k * 32;
            if (col + 32 > N) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i >= N) v[k][i] = -INFINITY;
            }
            // the label's column is not among the others
            if (__any_sync(0xffffffffu, y >= col && y < col + 32)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (y == col + i) v[k][i] = -INFINITY;
            }
          }
          float m = run_m;
#pragma unroll
          for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int i = 0; i < 32; i += 2) m = fmaxf(m, fmaxf(v[k][i], v[k][i + 1]));
          // exponentials in pairs: one packed fma and one packed add for two
          unsigned long long sum2 = pk2(0.0f, 0.0f);
          const unsigned long long l2 = pk2(XE_LOG2E, XE_LOG2E);
          float s0, s1;
          if (MODE == XE_KEEP) {
            const unsigned long long mc = pk2(-c2, -c2);
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float t0, t1;
                upk2(ffma2(pk2(v[k][i], v[k][i + 1]), l2, mc), t0, t1);
                v[k][i] = ex2_approx(t0);
                v[k][i + 1] = ex2_approx(t1);
              }
              if (!all_live) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[k][i] = live ? v[k][i] : 0.0f;
              }
#pragma unroll
              for (int i = 0; i < 32; i += 2) sum2 = fadd2(sum2, pk2(v[k][i], v[k][i + 1]));
              if (k % 2 == 1 && stored && col0 + (k - 1) * 32 < args.ldl)
                block_store_bf16(&tmC, stg, lane, v[k - 1], v[k], col0 + (k - 1) * 32, row - lane);
            }
            upk2(sum2, s0, s1);
            run_s += s0 + s1;
          } else if (m > -INFINITY) {
            const float m2 = m * XE_LOG2E;
            const unsigned long long mm = pk2(-m2, -m2);
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float t0, t1;
                upk2(ffma2(pk2(v[k][i], v[k][i + 1]), l2, mm), t0, t1);
                sum2 = fadd2(sum2, pk2(ex2_approx(t0), ex2_approx(t1)));
              }
            upk2(sum2, s0, s1);
            run_s = fmaf(run_s, ex2_approx(fmaf(run_m, XE_LOG2E, -m2)), s0 + s1);
          } else {  // -inf or NaN only: NaN is carried into the sum
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (isnan(v[k][i])) run_s = v[k][i];
          }
          run_m = m;
        } else if (MODE == XE_DLOGITS) {
          const int N = args.p[0].N;
#pragma unroll
          for (int k = 0; k < CHUNKS; ++k) {
            const int col = col0 + k * 32;
            const int gc = args.v0 + col;  // column in the vocabulary
#pragma unroll
            for (int i = 0; i < 32; ++i) v[k][i] = ex2_approx(fmaf(v[k][i], XE_LOG2E, -c2));
            if (__any_sync(0xffffffffu, y >= gc && y < gc + 32)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (y == gc + i) v[k][i] = at_label;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[k][i] = live ? v[k][i] * g : 0.0f;
            if (col + 32 > N) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i >= N) v[k][i] = 0.0f;
            }
            if (k % 2 == 1 && stored && col0 + (k - 1) * 32 < args.ldl) {
#pragma unroll
              for (int pl = 0; pl < PLANES; ++pl) {
                block_store_bf16(&tmC, stg, lane, v[k - 1], v[k], col0 + (k - 1) * 32,
                                 pl * static_cast<int>(args.dl_plane_rows) + row - lane);
                if (pl + 1 < PLANES) {
#pragma unroll
                  for (int i = 0; i < 32; ++i) {
                    v[k - 1][i] -= __bfloat162float(__float2bfloat16_rn(v[k - 1][i]));
                    v[k][i] -= __bfloat162float(__float2bfloat16_rn(v[k][i]));
                  }
                }
              }
            }
          }
        } else if (st.prod == 0) {
          if (row < rows) {
            float* o = args.dh_acc + st.slot * args.dh_slot_size + row * args.dh_ld;
            const int align = byte_align(args.dh_acc, args.dh_ld * 4);  // a slot is whole rows
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
              row_store_f32(o, col0 + k * 32, static_cast<int>(args.dh_ld), align, v[k], args.dh_accumulate != 0);
          }
        } else {
          const int d = args.p[1].N;
          const bool in = row < args.p[1].M;
          const int esz = args.dw_bf16 ? 2 : 4;
          const int align = byte_align(args.dw, args.dw_ld * esz);
#pragma unroll
          for (int k = 0; k < CHUNKS; ++k) {
            const int col = col0 + k * 32;
            if (extra != nullptr) {
              if (d % 4 == 0 && col + 32 <= d) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const float4 e = *reinterpret_cast<const float4*>(extra + col + i);
                  v[k][i] += e.x; v[k][i + 1] += e.y; v[k][i + 2] += e.z; v[k][i + 3] += e.w;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (col + i < d) v[k][i] += extra[col + i];
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[k][i] *= scale;
            if (PLANES == 1 && args.dw_tma) {
              if (k % 2 == 1 && col0 + (k - 1) * 32 < d)
                block_store_bf16(&tmC, stg, lane, v[k - 1], v[k], col0 + (k - 1) * 32, row - lane);
            } else if (in) {
              if (args.dw_bf16)
                row_store_bf16(static_cast<__nv_bfloat16*>(args.dw) + row * args.dw_ld, col, d, v[k]);
              else
                row_store_f32(static_cast<float*>(args.dw) + row * args.dw_ld, col, d, align, v[k], false);
            }
          }
        }
      }
      if ((MODE == XE_STATS || MODE == XE_KEEP) && st.last && ok && row < rows)
        args.part[(st.slot * 2 + ch) * args.part_ld + row] = make_float2(run_m, run_s);
    }
    if (lane == 0) bulk_wait<0>();  // the stores have read their blocks and written
  }

  // Teardown as in k_gemm2sm: every accumulator was consumed (or the roles
  // gave up and drained); both CTAs stay until the other is done.
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * XE_TILE);
  }
}

}  // namespace ethos
