// C ABI of the training operators around the expert layers (declared in
// include/ethos_b200.h): token embedding, routing balance loss.
// Host-side orchestration only, as in capi.cu.
#include <cuda.h>
#include <cuda_runtime.h>

#include "ethos_b200.h"
#include "host.cuh"
#include "balance.cuh"
#include "embed.cuh"

using namespace ethos;

namespace ethos {
int training_set_wait_limit(unsigned long long limit_ns) {
  return cudaMemcpyToSymbol(g_wait_limit_ns, &limit_ns, sizeof(limit_ns)) == cudaSuccess ? ETHOS_OK : ETHOS_ERR_CUDA;
}
}  // namespace ethos

namespace {

bool known_dtype(int dtype) { return dtype == ETHOS_F32 || dtype == ETHOS_BF16; }

// -------------------------------------------------------------- embedding --
template <class T, class I, bool kVec>
int embed_fwd(const void* ids, const void* w, int64_t ldw, int64_t tokens, int64_t vocab, int d, float scale, void* out,
              int* err, cudaStream_t sm, const DeviceInfo& dev) {
  const int64_t pieces = tokens * (d / RowAccess<T, kVec>::N);
  int64_t blocks = (pieces + 255) / 256;
  const int64_t most = 16ll * dev.sm_count;
  if (blocks > most) blocks = most;
  return launch_pdl(k_embed_fwd<T, I, kVec>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, sm,
                    static_cast<const I*>(ids), static_cast<const T*>(w), ldw, tokens, d, vocab, scale,
                    static_cast<T*>(out), err);
}

template <class T>
int embed_fwd_ids(const void* ids, int ids_i64, const void* w, int64_t ldw, int64_t tokens, int64_t vocab, int d,
                  float scale, void* out, int* err, cudaStream_t sm, const DeviceInfo& dev) {
  constexpr int N = Vec16<T>::N;
  const bool vec = d % N == 0 && ldw % N == 0 && aligned16(w) && aligned16(out);
  if (ids_i64)
    return vec ? embed_fwd<T, int64_t, true>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm, dev)
               : embed_fwd<T, int64_t, false>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm, dev);
  return vec ? embed_fwd<T, int32_t, true>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm, dev)
             : embed_fwd<T, int32_t, false>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm, dev);
}

struct EmbedScratch {
  int *offs, *perm, *sid;
  float* part;
};
void carve_embed(Carve& c, int64_t tokens, int64_t vocab, int64_t dim, EmbedScratch* s) {
  s->offs = c.take<int>(static_cast<size_t>(vocab + 1));
  s->perm = c.take<int>(static_cast<size_t>(tokens));
  s->sid = c.take<int>(static_cast<size_t>(tokens));
  s->part = c.take<float>(static_cast<size_t>((tokens + EMB_CHUNK - 1) / EMB_CHUNK * 2 * dim));
}

template <class T, bool kVec>
int embed_rows(const EmbedScratch& s, const void* dy, int64_t tokens, int64_t vocab, int d, float scale, void* dw,
               cudaStream_t sm, const DeviceInfo& dev) {
  const int pieces = d / RowAccess<T, kVec>::N;
  int tx = 8;
  while (tx < pieces && tx < 256) tx *= 2;
  const int ty = 256 / tx;
  const int col_blocks = (pieces + tx - 1) / tx;
  const int chunks = static_cast<int>((tokens + EMB_CHUNK - 1) / EMB_CHUNK);
  const int chunk_blocks = (chunks + ty - 1) / ty;
  const int64_t fill_most = (vocab + 7) / 8;
  const int fill = static_cast<int>(fill_most < 4 * dev.sm_count ? fill_most : 4 * dev.sm_count);
  const int64_t grid = static_cast<int64_t>(chunk_blocks) * col_blocks;
  if (grid + fill > (int64_t(1) << 31) - 1) return ETHOS_ERR_UNSUPPORTED_SHAPE;
  int st = launch_pdl(k_embed_rows<T, kVec>, dim3(static_cast<unsigned>(grid + fill)), dim3(tx, ty), 0, sm,
                      static_cast<const T*>(dy), d, vocab, scale, static_cast<const int*>(s.offs),
                      static_cast<const int*>(s.perm), static_cast<const int*>(s.sid), chunk_blocks, col_blocks,
                      s.part, static_cast<T*>(dw));
  if (st != ETHOS_OK || chunks < 2) return st;
  return launch_pdl(k_embed_join<T, kVec>, dim3(static_cast<unsigned>(grid)), dim3(tx, ty), 0, sm, d, vocab, scale,
                    static_cast<const int*>(s.offs), static_cast<const int*>(s.sid), col_blocks,
                    static_cast<const float*>(s.part), static_cast<T*>(dw));
}

template <class I>
int embed_sort(const EmbedScratch& s, const void* ids, int64_t tokens, int64_t vocab, int64_t padding, int* err,
               cudaStream_t sm, const DeviceInfo& dev) {
  // one block per SM, more when a block would own over EMB_MAX_RANGE ids
  int64_t blocks = dev.sm_count;
  if (blocks * EMB_MAX_RANGE < vocab) blocks = (vocab + EMB_MAX_RANGE - 1) / EMB_MAX_RANGE;
  const int range = static_cast<int>((vocab + blocks - 1) / blocks);
  blocks = (vocab + range - 1) / range;
  const int smem = EMB_SORT_WARPS * range * static_cast<int>(sizeof(int));
  auto kern = k_embed_sort<I>;
  const int st = smem_attr_once(reinterpret_cast<const void*>(kern),
                                EMB_SORT_WARPS * EMB_MAX_RANGE * static_cast<int>(sizeof(int)));
  if (st != ETHOS_OK) return st;
  return launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(EMB_SORT_THREADS), static_cast<size_t>(smem), sm,
                    static_cast<const I*>(ids), static_cast<int>(tokens), vocab, padding, range, s.offs, s.perm,
                    s.sid, err);
}

// ---------------------------------------------------------------- balance --
int balance_blocks(int64_t n, const DeviceInfo& dev) {
  int64_t b = (n + BAL_THREADS - 1) / BAL_THREADS;
  const int64_t most = 8ll * dev.sm_count < BAL_MAX_BLOCKS ? 8ll * dev.sm_count : BAL_MAX_BLOCKS;
  return static_cast<int>(b < 1 ? 1 : (b < most ? b : most));
}

template <class I, class W>
int balance_forward(const void* ids, const void* weights, const uint8_t* mask, int64_t tokens, int heads, int k,
                    int64_t experts, int32_t* counts, float* loss, BalScratch* s, int* err, cudaStream_t sm,
                    const DeviceInfo& dev) {
  const int blocks = balance_blocks(tokens * heads * k, dev);
  int st = launch_pdl(k_balance_count<I>, dim3(blocks), dim3(BAL_THREADS), 0, sm, static_cast<const I*>(ids), mask,
                      tokens, heads * k, experts, counts, s, err);
  if (st != ETHOS_OK) return st;
  return launch_pdl(k_balance_loss<I, W>, dim3(blocks), dim3(BAL_THREADS), 0, sm, static_cast<const I*>(ids),
                    static_cast<const W*>(weights), mask, tokens, heads, k, experts,
                    static_cast<const int*>(counts), s, loss);
}

template <class I, class W>
int balance_backward(const void* ids, const uint8_t* mask, int64_t tokens, int heads, int k, int64_t experts,
                     const int32_t* counts, const BalScratch* s, const float* grad, void* dw, cudaStream_t sm,
                     const DeviceInfo& dev) {
  const int blocks = balance_blocks(tokens * heads * k, dev);
  return launch_pdl(k_balance_bwd<I, W>, dim3(blocks), dim3(BAL_THREADS), 0, sm, static_cast<const I*>(ids), mask,
                    tokens, heads, k, experts, static_cast<const int*>(counts), s, grad, static_cast<W*>(dw));
}

int balance_check(const void* ids, int dtype, int64_t tokens, int64_t heads, int64_t k, int64_t experts) {
  if ((!ids && tokens > 0) || tokens < 0 || heads < 1 || k < 1 || experts < 1) return ETHOS_ERR_INVALID_ARG;
  if (!known_dtype(dtype)) return ETHOS_ERR_INVALID_ARG;
  // counts are int32
  if (heads > (1 << 20) || k > (1 << 20) || tokens > ((int64_t(1) << 31) - 1) / (heads * k))
    return ETHOS_ERR_UNSUPPORTED_SHAPE;
  return ETHOS_OK;
}

}  // namespace

extern "C" {

int ethos_embedding_forward(const void* ids, int ids_i64, const void* weight, int64_t ldw, int dtype, int64_t tokens,
                            int64_t vocab, int64_t dim, float scale, void* out, int* dev_err, void* stream) {
  if (tokens < 0 || vocab < 1 || dim < 1 || ldw < dim || !known_dtype(dtype)) return ETHOS_ERR_INVALID_ARG;
  if (dim > (1 << 24)) return ETHOS_ERR_UNSUPPORTED_SHAPE;
  if (tokens == 0) return ETHOS_OK;
  if (!ids || !weight || !out || !dev_err) return ETHOS_ERR_INVALID_ARG;
  DeviceInfo* dev = nullptr;
  const int st = base_device_info(&dev);
  if (st != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  const int d = static_cast<int>(dim);
  return dtype == ETHOS_BF16
             ? embed_fwd_ids<__nv_bfloat16>(ids, ids_i64, weight, ldw, tokens, vocab, d, scale, out, dev_err, sm, *dev)
             : embed_fwd_ids<float>(ids, ids_i64, weight, ldw, tokens, vocab, d, scale, out, dev_err, sm, *dev);
}

size_t ethos_embedding_backward_workspace_size(int64_t tokens, int64_t vocab, int64_t dim) {
  if (tokens < 0 || vocab < 1 || dim < 1) return 0;
  Carve c{nullptr, 0, 0};
  EmbedScratch s;
  carve_embed(c, tokens, vocab, dim, &s);
  return c.off + 256;
}

int ethos_embedding_backward(const void* ids, int ids_i64, const void* dy, int dtype, int64_t tokens, int64_t vocab,
                             int64_t dim, int64_t padding, float scale, void* d_weight, void* workspace,
                             size_t workspace_bytes, int* dev_err, void* stream) {
  if (tokens < 0 || vocab < 1 || dim < 1 || !known_dtype(dtype) || !d_weight || !dev_err)
    return ETHOS_ERR_INVALID_ARG;
  if (tokens >= (1 << 30) || vocab >= (1 << 30) || dim > (1 << 24)) return ETHOS_ERR_UNSUPPORTED_SHAPE;
  if (tokens > 0 && (!ids || !dy)) return ETHOS_ERR_INVALID_ARG;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  if (tokens == 0) {
    const size_t bytes = static_cast<size_t>(vocab) * dim * (dtype == ETHOS_BF16 ? 2 : 4);
    return cudaMemsetAsync(d_weight, 0, bytes, sm) == cudaSuccess ? ETHOS_OK : ETHOS_ERR_CUDA;
  }
  Carve c{static_cast<char*>(workspace), 0, workspace_bytes};
  EmbedScratch s;
  carve_embed(c, tokens, vocab, dim, &s);
  if (!workspace || c.off > workspace_bytes) return ETHOS_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return ETHOS_ERR_ALIGNMENT;
  DeviceInfo* dev = nullptr;
  int st = base_device_info(&dev);
  if (st != ETHOS_OK) return st;
  st = ids_i64 ? embed_sort<int64_t>(s, ids, tokens, vocab, padding, dev_err, sm, *dev)
               : embed_sort<int32_t>(s, ids, tokens, vocab, padding, dev_err, sm, *dev);
  if (st != ETHOS_OK) return st;
  const int d = static_cast<int>(dim);
  const bool al = aligned16(dy) && aligned16(d_weight);
  if (dtype == ETHOS_BF16)
    return al && d % 8 == 0 ? embed_rows<__nv_bfloat16, true>(s, dy, tokens, vocab, d, scale, d_weight, sm, *dev)
                            : embed_rows<__nv_bfloat16, false>(s, dy, tokens, vocab, d, scale, d_weight, sm, *dev);
  return al && d % 4 == 0 ? embed_rows<float, true>(s, dy, tokens, vocab, d, scale, d_weight, sm, *dev)
                          : embed_rows<float, false>(s, dy, tokens, vocab, d, scale, d_weight, sm, *dev);
}

size_t ethos_balance_scratch_size(void) { return sizeof(BalScratch); }

int ethos_balance_forward(const void* ids, int ids_i64, const void* weights, int dtype, const uint8_t* mask,
                          int64_t tokens, int64_t heads, int64_t k, int64_t experts, int32_t* counts, float* loss,
                          void* scratch, int* dev_err, void* stream) {
  int st = balance_check(ids, dtype, tokens, heads, k, experts);
  if (st != ETHOS_OK) return st;
  if ((!weights && tokens > 0) || !counts || !loss || !scratch || !dev_err) return ETHOS_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(scratch) & 15u) != 0) return ETHOS_ERR_ALIGNMENT;
  DeviceInfo* dev = nullptr;
  if ((st = base_device_info(&dev)) != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  BalScratch* s = static_cast<BalScratch*>(scratch);
  if (cudaMemsetAsync(counts, 0, sizeof(int32_t) * static_cast<size_t>(experts), sm) != cudaSuccess)
    return ETHOS_ERR_CUDA;
  if (cudaMemsetAsync(s, 0, offsetof(BalScratch, part), sm) != cudaSuccess) return ETHOS_ERR_CUDA;
  const int H = static_cast<int>(heads), K = static_cast<int>(k);
  if (ids_i64)
    return dtype == ETHOS_BF16
               ? balance_forward<int64_t, __nv_bfloat16>(ids, weights, mask, tokens, H, K, experts, counts, loss, s,
                                                         dev_err, sm, *dev)
               : balance_forward<int64_t, float>(ids, weights, mask, tokens, H, K, experts, counts, loss, s, dev_err,
                                                 sm, *dev);
  return dtype == ETHOS_BF16
             ? balance_forward<int32_t, __nv_bfloat16>(ids, weights, mask, tokens, H, K, experts, counts, loss, s,
                                                       dev_err, sm, *dev)
             : balance_forward<int32_t, float>(ids, weights, mask, tokens, H, K, experts, counts, loss, s, dev_err,
                                               sm, *dev);
}

int ethos_balance_backward(const void* ids, int ids_i64, int dtype, const uint8_t* mask, int64_t tokens,
                           int64_t heads, int64_t k, int64_t experts, const int32_t* counts, const void* scratch,
                           const float* grad, void* d_weights, void* stream) {
  int st = balance_check(ids, dtype, tokens, heads, k, experts);
  if (st != ETHOS_OK) return st;
  if (tokens == 0) return ETHOS_OK;
  if (!counts || !scratch || !grad || !d_weights) return ETHOS_ERR_INVALID_ARG;
  DeviceInfo* dev = nullptr;
  if ((st = base_device_info(&dev)) != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  const BalScratch* s = static_cast<const BalScratch*>(scratch);
  const int H = static_cast<int>(heads), K = static_cast<int>(k);
  if (ids_i64)
    return dtype == ETHOS_BF16
               ? balance_backward<int64_t, __nv_bfloat16>(ids, mask, tokens, H, K, experts, counts, s, grad,
                                                          d_weights, sm, *dev)
               : balance_backward<int64_t, float>(ids, mask, tokens, H, K, experts, counts, s, grad, d_weights, sm,
                                                  *dev);
  return dtype == ETHOS_BF16 ? balance_backward<int32_t, __nv_bfloat16>(ids, mask, tokens, H, K, experts, counts, s,
                                                                        grad, d_weights, sm, *dev)
                             : balance_backward<int32_t, float>(ids, mask, tokens, H, K, experts, counts, s, grad,
                                                                d_weights, sm, *dev);
}

}  // extern "C"
