// Cross entropy of the output head (model.py:385, train.py:200) without its
// logits in memory:
//
//   l[t, v] = h[t] . W[v],   lse[t] = log sum_v exp l[t, v],
//   loss[t] = lse[t] - l[t, y[t]]                       (0 for ignored tokens)
//   dl[t, v] = g[t] (exp(l[t, v] - lse[t]) - [v = y[t]])
//   dh = dl W,   dW = dl^T h
//
// forward: one GEMM whose epilogue keeps, for each row, the running maximum and
// the sum of exponentials over the tiles it sees, and picks the label's logit;
// a second kernel joins the pieces of each row.  backward: for one piece of
// the vocabulary after another, the logits are formed again, their gradient
// goes to a [tokens, piece] bf16 buffer straight from the accumulators, and
// one launch computes both products with it.  Four products of 2 T V d FLOPs,
// bounded by the tensor cores; memory beyond inputs and outputs is one piece.
//
// Rows.  With more than XE_ROWS_DIRECT tokens the tokens that are not ignored
// are packed first (their number stays on the device), so ignored tokens cost
// nothing after that; fewer fit one row tile and keep their places.
//
// Types.  bf16: operands as they are; dl is rounded to bf16 (the operand type
// of the two products), sums are fp32.  fp32: operands, and dl, are carried
// as three bf16 planes whose sum is the fp32 value, and each product is six
// plane products, the smallest first, with a fresh accumulator every
// XE_FLUSH_KB blocks of 64 (the accumulator of the matrix unit loses about
// half an ulp of the running sum per step), added up in fp32.
//
// GEMM: k_xent_gemm runs on SM pairs as k_gemm2sm does (256 x 256 tile, each
// CTA staging 128 rows of A and of B, cta_group::2 MMA, two accumulators in
// TMEM, no multicast loads), with row counts read from the device, ragged M,
// N and K, and units grouped so that the operand shared by concurrent pairs
// stays in L2.
#pragma once

#include "gemm2sm.cuh"

namespace ethos {

constexpr int XE_ROWS_DIRECT = 256;  // tokens that keep their places (one row tile)
constexpr int XE_TILE = 256;         // tile rows and columns of an SM pair
constexpr int XE_GROUP_M = 64;       // row tiles walked before the next column tile
constexpr int XE_FLUSH_KB = 8;       // fp32: K blocks of 64 per accumulator in the gradient products
constexpr int XE_STG_WARP_BYTES = 32 * 64;
constexpr float XE_LOG2E = 1.4426950408889634f;

enum XeMode { XE_STATS, XE_DLOGITS, XE_GRADS };

// What the forward leaves for the backward, at the start of the save buffer.
struct XeMeta {
  int rows;       // rows of the packed problem
  int valid;      // tokens that are not ignored
  unsigned done;  // blocks of k_xent_loss that have added their part
};

// Row index, compacted: pos[t] = row of token t or -1, idx[r] = token of row
// r, yc[r] = its label (-1: an ignored token that kept its place).
struct XeRows {
  XeMeta* meta;
  int* pos;
  int* idx;
  int* yc;
  float* lse;
  float* lab;  // the label's logit
};

template <class I>
__global__ void __launch_bounds__(1024) k_xent_index(const I* __restrict__ labels, int tokens, int64_t vocab,
                                                     int64_t ignore, bool compact, XeRows rw,
                                                     float* __restrict__ loss_rows, int* err) {
  __shared__ int warp_sum[32];
  pdl_launch_dependents();
  pdl_wait();
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
  }
}

// ------------------------------------------------------------------- pack --
// dst [PLANES][plane_rows][ldd] bf16 <- rows of src: plane 0 = bf16(v), plane
// 1 = bf16(v - plane 0), plane 2 the rest.  With idx, row r is src[idx[r]] for
// r < *rows, and rows up to the next multiple of XE_TILE are zero; without,
// rows 0..count-1 and zeros up to plane_rows.  Columns d..ldd are zero.
template <class S, int PLANES>
__global__ void __launch_bounds__(256) k_xent_pack(const S* __restrict__ src, int64_t lds, int d,
                                                   const int* __restrict__ idx, const int* __restrict__ rows,
                                                   int64_t count, __nv_bfloat16* __restrict__ dst, int64_t plane_rows,
                                                   int ldd) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t n = rows != nullptr ? *rows : count;
  const int64_t n_pad = rows != nullptr ? (n + XE_TILE - 1) / XE_TILE * XE_TILE : plane_rows;
  const int pieces = ldd / 8;
  const int64_t total = n_pad * pieces;
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 && lds % (16 / sizeof(S)) == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / pieces;
    const int c = static_cast<int>(i - r * pieces) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (r < n) {
      const S* s = src + (idx != nullptr ? static_cast<int64_t>(idx[r]) : r) * lds + c;
      if (vec && c + 8 <= d) {
        if constexpr (sizeof(S) == 4) {
          const float4 a = reinterpret_cast<const float4*>(s)[0], b = reinterpret_cast<const float4*>(s)[1];
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(s);
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
        for (int j = 0; j < 8; ++j)
          if (c + j < d) v[j] = static_cast<float>(s[j]);
      }
    }
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
        const float2 f = __bfloat1622float2(h);
        v[2 * j] -= f.x;
        v[2 * j + 1] -= f.y;
      }
      *reinterpret_cast<uint4*>(dst + (p * plane_rows + r) * ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ------------------------------------------------------------------- loss --
// Joins the (maximum, sum) pieces of each row and writes its loss: 8 rows per
// block, 32 threads along a row's pieces.  Sums over tokens have a fixed
// order: block sums (fp64), added by the last block in block order.
constexpr int XE_LOSS_ROWS = 8;
enum XeReduction { XE_NONE, XE_SUM, XE_MEAN };

__device__ __forceinline__ void lse_join(float& m, float& s, float m2, float s2) {
  const float hi = fmaxf(m, m2);
  if (hi == -INFINITY) {  // nothing seen yet, or logits of -inf (or NaN) only
    s += s2;
    return;
  }
  s = s * exp2f((m - hi) * XE_LOG2E) + s2 * exp2f((m2 - hi) * XE_LOG2E);
  m = hi;
}

__global__ void __launch_bounds__(256) k_xent_loss(XeRows rw, const float2* __restrict__ part, int parts,
                                                   int64_t part_ld, int reduction, float* __restrict__ loss,
                                                   double* __restrict__ block_sum) {
  __shared__ double red[256];
  __shared__ bool last;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x * XE_LOSS_ROWS + (threadIdx.x & (XE_LOSS_ROWS - 1));
  const int py = threadIdx.x / XE_LOSS_ROWS;  // 0..31
  const int rows = rw.meta->rows;
  float m = -INFINITY, s = 0.0f;
  if (row < rows) {
#pragma unroll 4
    for (int p = py; p < parts; p += 32) {
      const float2 v = part[p * part_ld + row];
      lse_join(m, s, v.x, v.y);
    }
  }
  // lanes of a warp hold 4 pieces of each of 8 rows; then over the 8 warps
#pragma unroll
  for (int o = 16; o >= XE_LOSS_ROWS; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    lse_join(m, s, m2, s2);
  }
  __shared__ float2 wp[8][XE_LOSS_ROWS];
  if ((threadIdx.x & 31) < XE_LOSS_ROWS) wp[threadIdx.x >> 5][threadIdx.x & 31] = make_float2(m, s);
  __syncthreads();
  double mine = 0.0;
  if (threadIdx.x < XE_LOSS_ROWS && row < rows) {
    for (int w = 1; w < 8; ++w) lse_join(m, s, wp[w][threadIdx.x].x, wp[w][threadIdx.x].y);
    const float lse = m + logf(s);
    rw.lse[row] = lse;
    if (rw.yc[row] >= 0) {
      const float l = lse - rw.lab[row];
      if (reduction == XE_NONE) loss[rw.idx[row]] = l;
      mine = static_cast<double>(l);
    }
  }
  if (reduction == XE_NONE) return;
  red[threadIdx.x] = mine;
  __syncthreads();
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
  // no token left: 0 for the sum, NaN for the mean
  if (threadIdx.x == 0) *loss = static_cast<float>(reduction == XE_MEAN ? red[0] / rw.meta->valid : red[0]);
}

// -------------------------------------------------------------- dh output --
// d_hidden[t] = scale * (sum over slots of acc[slot][pos[t]]), zero for an
// ignored token.
template <class D>
__global__ void __launch_bounds__(256) k_xent_dhidden(const float* __restrict__ acc, int slots, int64_t slot_size,
                                                      int64_t lda, XeRows rw, const float* __restrict__ grad,
                                                      int reduction, int64_t tokens, int d, D* __restrict__ out) {
  pdl_launch_dependents();
  pdl_wait();
  const float scale = reduction == XE_NONE ? 1.0f : (reduction == XE_SUM ? *grad : *grad / rw.meta->valid);
  const int pieces = (d + 3) / 4;
  const int64_t total = tokens * pieces;
  const bool vec = d % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = i / pieces;
    const int c = static_cast<int>(i - t * pieces) * 4;
    const int r = rw.pos[t];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r >= 0) {
      const float* a = acc + static_cast<int64_t>(r) * lda + c;
#pragma unroll 4
      for (int s = 0; s < slots; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(a + s * slot_size);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      v.x *= scale; v.y *= scale; v.z *= scale; v.w *= scale;
    }
    D* o = out + t * d + c;
    if (vec) {
      if constexpr (sizeof(D) == 4) {
        *reinterpret_cast<float4*>(o) = v;
      } else {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      }
    } else {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < d) {
          if constexpr (sizeof(D) == 4) o[j] = e[j];
          else o[j] = __float2bfloat16_rn(e[j]);
        }
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

struct XeArgs {
  XeRows rw;
  XeProduct p[2];  // STATS, DLOGITS: p[0]; GRADS: p[0] = dh, p[1] = dW
  // STATS
  int run;  // column tiles per unit
  float2* part;
  int64_t part_ld;
  // DLOGITS: gradient of the logits of columns [v0, v0 + N) into
  // dl [PLANES][dl_plane_rows][ldl]
  int v0;
  const float* grad;
  int reduction;
  __nv_bfloat16* dl;
  int64_t dl_plane_rows;
  int64_t ldl;
  // GRADS
  int dh_slots;        // K slices of dh, each with a buffer of its own
  int dh_accumulate;   // add to dh_acc (pieces after the first)
  float* dh_acc;       // [slots][rows][dh_ld]
  int64_t dh_slot_size;
  int64_t dh_ld;
  void* dw;            // rows of this piece, [N rows][d] with pitch d
  int dw_bf16;
  int do_dh, do_dw;
};

struct XeCtl {
  uint64_t full[G2_STAGES];
  uint64_t empty[G2_STAGES];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
constexpr int XE_EPI_WARPS = 8;
constexpr int XE_THREADS = 64 + 32 * XE_EPI_WARPS;
constexpr int XE_SMEM = G2_STAGES * G2_STAGE_BYTES + XE_EPI_WARPS * XE_STG_WARP_BYTES + 1024 +
                        static_cast<int>(sizeof(XeCtl));
static_assert(XE_SMEM <= 227 * 1024, "shared memory");

// One accumulation: tile at (m0, n0) of product `prod`, K blocks [kb0, kb1)
// over all plane products.
struct XeStep {
  int prod, m0, n0, kb0, kb1;
  bool first, last;  // of its unit
  int slot;
};

// The units of a pair, as a sequence of accumulations; every role of both
// CTAs walks the same sequence.
template <int MODE, int PLANES>
struct XeWalk {
  const XeArgs& a;
  int rows, num_m, num_n, nkb, units0, units, u, stride;
  int j;           // accumulation within the unit
  int mt_w, kb_w;  // GRADS: row tiles and K blocks of dW
  int kb_slot;     // GRADS: K blocks of dh per slot
  __device__ XeWalk(const XeArgs& args, int rows_, int pair, int pairs)
      : a(args), rows(rows_), u(pair), stride(pairs), j(0) {
    num_m = (rows + XE_TILE - 1) / XE_TILE;
    num_n = (a.p[0].N + XE_TILE - 1) / XE_TILE;
    nkb = (a.p[0].K + G2_BK - 1) / G2_BK;
    mt_w = kb_w = kb_slot = 0;
    if (MODE == XE_STATS) {
      units0 = units = num_m * ((num_n + a.run - 1) / a.run);
    } else if (MODE == XE_DLOGITS) {
      units0 = units = num_m * num_n;
    } else {
      kb_slot = (nkb + a.dh_slots - 1) / a.dh_slots;
      units0 = a.do_dh ? num_m * num_n * a.dh_slots : 0;
      mt_w = (a.p[1].M + XE_TILE - 1) / XE_TILE;
      kb_w = (rows + G2_BK - 1) / G2_BK;
      units = units0 + (a.do_dw ? mt_w * num_n : 0);
    }
  }
  // the next accumulation; false when the pair's units are done
  __device__ bool next(XeStep& s) {
    if (u >= units) return false;
    int steps;
    s.slot = 0;
    if (MODE == XE_STATS || MODE == XE_DLOGITS) {
      // row tiles in groups of XE_GROUP_M, all columns of a group before the
      // next: A's group and one column tile of B (or a run of them) in L2
      const int cols = MODE == XE_STATS ? (num_n + a.run - 1) / a.run : num_n;
      const int per_group = XE_GROUP_M * cols;
      const int g = u / per_group;
      const int gm = min(XE_GROUP_M, num_m - g * XE_GROUP_M);
      const int v = u - g * per_group;
      const int c = v / gm;
      s.prod = 0;
      s.m0 = (g * XE_GROUP_M + v % gm) * XE_TILE;
      s.kb0 = 0;
      s.kb1 = nkb;
      if (MODE == XE_STATS) {
        steps = min(a.run, num_n - c * a.run);
        s.n0 = (c * a.run + j) * XE_TILE;
        s.slot = c;
      } else {
        steps = 1;
        s.n0 = c * XE_TILE;
      }
    } else {
      int kb0, kb1;
      if (u < units0) {
        const int t = u % (num_m * num_n);
        s.slot = u / (num_m * num_n);
        s.prod = 0;
        s.m0 = (t / num_n) * XE_TILE;
        s.n0 = (t % num_n) * XE_TILE;
        kb0 = s.slot * kb_slot;
        kb1 = min(nkb, kb0 + kb_slot);
      } else {
        const int t = u - units0;
        s.prod = 1;
        s.m0 = (t / num_n) * XE_TILE;
        s.n0 = (t % num_n) * XE_TILE;
        kb0 = 0;
        kb1 = kb_w;
      }
      const int fl = PLANES == 1 ? (1 << 28) : XE_FLUSH_KB;
      steps = max(1, (kb1 - kb0 + fl - 1) / fl);
      s.kb0 = kb0 + j * fl;
      s.kb1 = min(kb1, s.kb0 + fl);
    }
    s.first = j == 0;
    s.last = j + 1 >= steps;
    if (s.last) {
      j = 0;
      u += stride;
    } else {
      ++j;
    }
    return true;
  }
};

// Plane pairs of a product, smallest first: A = 0, 2, 1, 1, 0, 0 and
// B = 2, 0, 1, 0, 1, 0 (0 the leading plane).
__device__ __forceinline__ int xe_plane_a(int seg) { return (0x058 >> (2 * seg)) & 3; }
__device__ __forceinline__ int xe_plane_b(int seg) { return (0x112 >> (2 * seg)) & 3; }

// 32 rows x 32 columns of fp32 accumulators to a row-major matrix of `cols`
// columns, coalesced through the warp's staging block (two halves of 16
// columns); `acc` adds to what is there.  Rows >= nrows are skipped.
__device__ __forceinline__ void xe_store_f32(uint8_t* stg, int lane, int nrows, const float (&v)[32], float* dst,
                                             int64_t ld, int col, int cols, bool vec, bool acc) {
  const int sw = (lane >> 1) & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4*>(stg + lane * 64 + ((j ^ sw) << 4)) =
          make_float4(v[16 * h + 4 * j], v[16 * h + 4 * j + 1], v[16 * h + 4 * j + 2], v[16 * h + 4 * j + 3]);
    __syncwarp();
    if (vec) {
      const int piece = lane & 3;
      const int c = col + 16 * h + 4 * piece;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 8 * k + (lane >> 2);
        float4 u = *reinterpret_cast<const float4*>(stg + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
        if (r < nrows && c < cols) {
          float4* o = reinterpret_cast<float4*>(dst + r * ld + c);
          if (acc) {
            const float4 p = *o;
            u.x += p.x; u.y += p.y; u.z += p.z; u.w += p.w;
          }
          *o = u;
        }
      }
    } else {
      const int e = lane & 15;
      const int c = col + 16 * h + e;
      for (int r = lane >> 4; r < nrows; r += 2) {
        const float u = *reinterpret_cast<const float*>(stg + r * 64 + (((e >> 2) ^ ((r >> 1) & 3)) << 4) + (e & 3) * 4);
        if (c < cols) dst[r * ld + c] = acc ? dst[r * ld + c] + u : u;
      }
    }
    __syncwarp();
  }
}
// the same, rounded to bf16 (no accumulation)
__device__ __forceinline__ void xe_store_bf16(uint8_t* stg, int lane, int nrows, const float (&v)[32],
                                              __nv_bfloat16* dst, int64_t ld, int col, int cols, bool vec) {
  const int sw = (lane >> 1) & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(stg + lane * 64 + ((j ^ sw) << 4)) =
        make_uint4(pack_bf16x2(v[8 * j], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                   pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
  __syncwarp();
  if (vec) {
    const int piece = lane & 3;
    const int c = col + 8 * piece;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = 8 * k + (lane >> 2);
      const uint4 u = *reinterpret_cast<const uint4*>(stg + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
      if (r < nrows && c < cols) *reinterpret_cast<uint4*>(dst + r * ld + c) = u;
    }
  } else {
    const int c = col + lane;
    for (int r = 0; r < nrows; ++r) {
      const __nv_bfloat16 u =
          *reinterpret_cast<const __nv_bfloat16*>(stg + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
      if (c < cols) dst[r * ld + c] = u;
    }
  }
  __syncwarp();
}

template <int MODE, int PLANES>
__global__ void __launch_bounds__(XE_THREADS, 1)
    k_xent_gemm(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmB0,
                const __grid_constant__ CUtensorMap tmA1, const __grid_constant__ CUtensorMap tmB1,
                const __grid_constant__ XeArgs args, int* err) {
  constexpr int SEGS = PLANES == 1 ? 1 : 6;
  constexpr int CHUNKS = (XE_TILE / 32) / (XE_EPI_WARPS / 4);  // 32-column chunks per epilogue warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t* stg_s = smem + G2_STAGES * G2_STAGE_BYTES;
  XeCtl* ctl = reinterpret_cast<XeCtl*>(stg_s + XE_EPI_WARPS * XE_STG_WARP_BYTES);
  const int warp = warp_id();
  const int lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(blockIdx.x) >> 1;
  const int pairs = static_cast<int>(gridDim.x) >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G2_STAGES; ++s) {
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
  const int rows = *static_cast<const volatile int*>(&args.rw.meta->rows);
  volatile int* abort = &ctl->abort;
  XeWalk<MODE, PLANES> walk(args, rows, pair, pairs);
  XeStep st;

  if (warp == 0) {
    if (lane == 0) {
      RingPos rp;
      bool ok = true;
      while (ok && walk.next(st)) {
        const int m0 = st.m0 + static_cast<int>(rank) * G2_BM;
        const int n0 = st.n0 + static_cast<int>(rank) * (XE_TILE / 2);
        const CUtensorMap* ta = st.prod == 0 ? &tmA0 : &tmA1;
        const CUtensorMap* tb = st.prod == 0 ? &tmB0 : &tmB1;
        const XeProduct& p = args.p[st.prod];
        for (int seg = 0; ok && seg < SEGS; ++seg) {
          const int ya = SEGS == 1 ? 0 : xe_plane_a(seg) * p.a_plane_rows;
          const int yb = SEGS == 1 ? 0 : xe_plane_b(seg) * p.b_plane_rows;
          for (int kb = st.kb0; kb < st.kb1; ++kb) {
            if (!mbar_wait(&ctl->empty[rp.stage], rp.phase ^ 1u, abort, err, 1)) {
              ok = false;
              break;
            }
            uint8_t* sa = smem + rp.stage * G2_STAGE_BYTES;
            uint8_t* sb = sa + G2_A_BYTES;
            if (leader) mbar_arrive_expect_tx(&ctl->full[rp.stage], 2 * G2_STAGE_BYTES);
            const uint32_t fb = cluster_map(smem_u32(&ctl->full[rp.stage]), 0);
            if (MODE == XE_GRADS && st.prod == 1) {
              tma_load_2d_pair(sa, ta, fb, m0, ya + kb * G2_BK);
              tma_load_2d_pair(sa + 8192, ta, fb, m0 + 64, ya + kb * G2_BK);
            } else {
              tma_load_2d_pair(sa, ta, fb, kb * G2_BK, ya + m0);
            }
            if (MODE == XE_GRADS) {
              tma_load_2d_pair(sb, tb, fb, n0, yb + kb * G2_BK);
              tma_load_2d_pair(sb + 8192, tb, fb, n0 + 64, yb + kb * G2_BK);
            } else {
              tma_load_2d_pair(sb, tb, fb, kb * G2_BK, yb + n0);
            }
            rp.advance(G2_STAGES);
          }
        }
      }
      if (!ok) {
        // as in k_gemm2sm: both CTAs' copies complete on the leader's
        // barriers; the peer waits a bounded 100 us for its own to land
        if (leader) {
          rp.drain(ctl->full, G2_STAGES, err, 5);
        } else {
          const uint64_t t0 = global_timer_ns();
          while (global_timer_ns() - t0 < 100000ull) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      while (ok && walk.next(st)) {
        if (st.kb0 >= st.kb1) continue;  // nothing to add up (no rows)
        const bool a_mn = MODE == XE_GRADS && st.prod == 1;
        const uint32_t idesc = umma_idesc_bf16_f32_major(2 * G2_BM, XE_TILE, a_mn, MODE == XE_GRADS);
        const int buf = it & 1;
        const uint32_t acc_phase = static_cast<uint32_t>(it >> 1) & 1u;
        ++it;
        if (!mbar_wait(&ctl->acc_empty[buf], acc_phase ^ 1u, abort, err, 2)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(buf * XE_TILE);
        const int blocks = SEGS * (st.kb1 - st.kb0);
        for (int b = 0; b < blocks; ++b) {
          if (!mbar_wait(&ctl->full[stage], phase, abort, err, 3)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_base = smem_u32(smem + stage * G2_STAGE_BYTES);
          const uint32_t b_base = a_base + G2_A_BYTES;
#pragma unroll
          for (int k = 0; k < G2_BK / 16; ++k) {
            const uint64_t ad = a_mn ? umma_desc_sw128_mn(a_base + k * 2048, 8192) : umma_desc_sw128(a_base + k * 32);
            const uint64_t bd =
                MODE == XE_GRADS ? umma_desc_sw128_mn(b_base + k * 2048, 8192) : umma_desc_sw128(b_base + k * 32);
            umma_bf16_pair(d, ad, bd, idesc, (b > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit_pair_mc(&ctl->empty[stage], 0x3);
          if (++stage == G2_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair_mc(&ctl->acc_full[buf], 0x3);
      }
      if (!ok || *abort) {
        umma_commit_pair(&ctl->drain);
        mbar_wait(&ctl->drain, 0, nullptr, err, 6);
      }
    }
  } else {
    // Epilogue warps never leave the walk early: after an abort they skip the
    // work but still arrive on every acc_empty phase.
    const int q = warp & 3;
    const int ch = (warp - 2) >> 2;  // column half of the tile
    uint8_t* stg = stg_s + (warp - 2) * XE_STG_WARP_BYTES;
    const uint32_t acc_empty0 = cluster_map(smem_u32(&ctl->acc_empty[0]), 0);
    const uint32_t acc_empty1 = cluster_map(smem_u32(&ctl->acc_empty[1]), 0);
    int it = 0;
    bool ok = true;
    // per-row state (this lane's row of the tile)
    int y = -1;
    float run_m = -INFINITY, run_s = 0.0f;       // STATS
    float lse2 = 0.0f, lse = 0.0f, g = 0.0f;      // DLOGITS
    float scale = 1.0f;                           // GRADS: dW
    if (MODE == XE_GRADS && args.reduction != XE_NONE) {
      scale = *args.grad;
      if (args.reduction == XE_MEAN) {
        const int valid = args.rw.meta->valid;
        scale = valid > 0 ? scale / valid : 0.0f;
      }
    }
    while (walk.next(st)) {
      const bool any = st.kb0 < st.kb1;
      const int row0 = st.m0 + static_cast<int>(rank) * G2_BM + q * 32;
      const int row = row0 + lane;
      if (MODE == XE_STATS && st.first) {
        y = row < rows ? args.rw.yc[row] : -1;
        run_m = -INFINITY;
        run_s = 0.0f;
      }
      if (MODE == XE_DLOGITS) {
        y = row < rows ? args.rw.yc[row] : -1;
        lse = row < rows ? args.rw.lse[row] : 0.0f;
        lse2 = lse * XE_LOG2E;
        g = 1.0f;
        if (args.reduction == XE_NONE && y >= 0) g = args.grad[args.rw.idx[row]];
      }
      const int buf = it & 1;
      const uint32_t acc_phase = static_cast<uint32_t>(it >> 1) & 1u;
      if (any) {
        ++it;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&ctl->acc_full[buf], acc_phase, abort, err, 4));
        tc_fence_after();
      }
      if (ok) {
#pragma unroll 1
        for (int c = ch * CHUNKS; c < (ch + 1) * CHUNKS; ++c) {
          float v[32];
          if (any) {
            tmem_ld32(tmem_addr(tmem, q * 32, buf * XE_TILE + c * 32), v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.0f;
          }
          const int col = st.n0 + c * 32;
          if (MODE == XE_STATS) {
            const int N = args.p[0].N;
            if (col + 32 > N) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i >= N) v[i] = -INFINITY;
            }
            if (__any_sync(0xffffffffu, y >= col && y < col + 32)) {
              float l = 0.0f;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (y == col + i) l = v[i];
              if (y >= col && y < col + 32) args.rw.lab[row] = l;
            }
            float m = run_m;
#pragma unroll
            for (int i = 0; i < 32; ++i) m = fmaxf(m, v[i]);
            if (m > -INFINITY) {
              const float m2 = m * XE_LOG2E;
              float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                s0 += ex2_approx(fmaf(v[i], XE_LOG2E, -m2));
                s1 += ex2_approx(fmaf(v[i + 1], XE_LOG2E, -m2));
              }
              run_s = fmaf(run_s, ex2_approx(fmaf(run_m, XE_LOG2E, -m2)), s0 + s1);
              run_m = m;
            } else {  // -inf or NaN only: NaN is carried into the sum
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (isnan(v[i])) run_s = v[i];
            }
          } else if (MODE == XE_DLOGITS) {
            const bool live = y >= 0;
            const int gc = args.v0 + col;  // column in the vocabulary
            const int N = args.p[0].N;
            // p - 1 at the label, without the cancellation
            const bool label = live && y >= gc && y < gc + 32;
            const bool any_label = __any_sync(0xffffffffu, label);
            float at_label = 0.0f;
            if (any_label) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (y == gc + i) at_label = v[i];
              at_label = expm1f(at_label - lse);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = ex2_approx(fmaf(v[i], XE_LOG2E, -lse2));
            if (any_label) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (y == gc + i) v[i] = at_label;
            }
            if (args.reduction == XE_NONE) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= g;
            }
            if (!live) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.0f;
            }
            if (col + 32 > N) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i >= N) v[i] = 0.0f;
            }
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl) {
              xe_store_bf16(stg, lane, 32, v,
                            args.dl + (pl * args.dl_plane_rows + row0) * args.ldl, args.ldl, col,
                            static_cast<int>(args.ldl), true);
              if (pl + 1 < PLANES) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] -= __bfloat162float(__float2bfloat16_rn(v[i]));
              }
            }
          } else if (st.prod == 0) {
            xe_store_f32(stg, lane, min(32, rows - row0), v,
                         args.dh_acc + st.slot * args.dh_slot_size + row0 * args.dh_ld, args.dh_ld, col,
                         static_cast<int>(args.dh_ld), true, args.dh_accumulate != 0 || !st.first);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= scale;
            const int d = args.p[1].N;
            const int nr = min(32, args.p[1].M - row0);
            if (args.dw_bf16) {
              __nv_bfloat16* o = static_cast<__nv_bfloat16*>(args.dw) + static_cast<int64_t>(row0) * d;
              xe_store_bf16(stg, lane, nr, v, o, d, col, d,
                            d % 8 == 0 && (reinterpret_cast<uintptr_t>(args.dw) & 15u) == 0);
            } else {
              float* o = static_cast<float*>(args.dw) + static_cast<int64_t>(row0) * d;
              xe_store_f32(stg, lane, nr, v, o, d, col, d,
                           d % 4 == 0 && (reinterpret_cast<uintptr_t>(args.dw) & 15u) == 0, !st.first);
            }
          }
        }
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(buf ? acc_empty1 : acc_empty0);
      }
      if (MODE == XE_STATS && st.last && ok && row < rows)
        args.part[(st.slot * 2 + ch) * args.part_ld + row] = make_float2(run_m, run_s);
    }
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
