// C ABI of the training operators around the expert layers (declared in
// include/ethos_b200.h): token embedding, routing balance loss, cross
// entropy of the output head.
// Host-side orchestration only, as in capi.cu.
#include <cuda.h>
#include <cuda_runtime.h>

#include "ethos_b200.h"
#include "host.cuh"
#include "balance.cuh"
#include "embed.cuh"
#include "xent.cuh"

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
              int* err, cudaStream_t sm) {
  const int pieces = d / RowAccess<T, kVec>::N;
  int tx = 8;
  while (tx < pieces && tx < 256) tx *= 2;
  const int ty = 256 / tx;
  const int64_t blocks = (tokens + EMB_FWD_ROWS * ty - 1) / (EMB_FWD_ROWS * ty);
  if (blocks > (int64_t(1) << 31) - 1) return ETHOS_ERR_UNSUPPORTED_SHAPE;
  return launch_pdl(k_embed_fwd<T, I, kVec>, dim3(static_cast<unsigned>(blocks)), dim3(tx, ty), 0, sm,
                    static_cast<const I*>(ids), static_cast<const T*>(w), ldw, tokens, d, vocab, scale,
                    static_cast<T*>(out), err);
}

template <class T>
int embed_fwd_ids(const void* ids, int ids_i64, const void* w, int64_t ldw, int64_t tokens, int64_t vocab, int d,
                  float scale, void* out, int* err, cudaStream_t sm) {
  constexpr int N = Vec16<T>::N;
  const bool vec = d % N == 0 && ldw % N == 0 && aligned16(w) && aligned16(out);
  if (ids_i64)
    return vec ? embed_fwd<T, int64_t, true>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm)
               : embed_fwd<T, int64_t, false>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm);
  return vec ? embed_fwd<T, int32_t, true>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm)
             : embed_fwd<T, int32_t, false>(ids, w, ldw, tokens, vocab, d, scale, out, err, sm);
}

struct EmbedScratch {
  int2* span;
  int *perm, *sid;
  float* part;
};
void carve_embed(Carve& c, int64_t tokens, int64_t vocab, int64_t dim, EmbedScratch* s) {
  s->span = c.take<int2>(static_cast<size_t>(vocab + 1));
  s->perm = c.take<int>(static_cast<size_t>(tokens));
  s->sid = c.take<int>(static_cast<size_t>(tokens));
  s->part = c.take<float>(static_cast<size_t>((tokens + EMB_CHUNK - 1) / EMB_CHUNK * 2 * dim));
}

// Row sums of the sorted tokens (k_embed_rows, k_embed_join).  kByPlace: the
// rows in use only; otherwise every row of the table.
template <class T, bool kVec, class O, bool kByPlace>
int embed_rows(const EmbedScratch& s, const void* dy, int64_t ldy, const float* row_scale, int64_t tokens,
               int64_t vocab, int d, float scale, O* dw, cudaStream_t sm, const DeviceInfo& dev) {
  const int pieces = d / RowAccess<T, kVec>::N;
  int tx = 8;
  while (tx < pieces && tx < 256) tx *= 2;
  const int ty = 256 / tx;
  const int col_blocks = (pieces + tx - 1) / tx;
  const int chunks = static_cast<int>((tokens + EMB_CHUNK - 1) / EMB_CHUNK);
  const int chunk_blocks = (chunks + ty - 1) / ty;
  const int64_t fill_most = kByPlace ? 0 : (vocab + 8 * EMB_FILL - 1) / (8 * EMB_FILL);
  const int fill = static_cast<int>(fill_most < 4 * dev.sm_count ? fill_most : 4 * dev.sm_count);
  const int64_t grid = static_cast<int64_t>(chunk_blocks) * col_blocks;
  if (grid + fill > (int64_t(1) << 31) - 1) return ETHOS_ERR_UNSUPPORTED_SHAPE;
  int st = launch_pdl(k_embed_rows<T, kVec, O, kByPlace>, dim3(static_cast<unsigned>(grid + fill)), dim3(tx, ty), 0,
                      sm, static_cast<const T*>(dy), ldy, row_scale, d, vocab, scale, static_cast<const int2*>(s.span),
                      static_cast<const int*>(s.perm), static_cast<const int*>(s.sid), chunk_blocks, col_blocks,
                      s.part, dw);
  if (st != ETHOS_OK || chunks < 2) return st;
  return launch_pdl(k_embed_join<T, kVec, O, kByPlace>, dim3(static_cast<unsigned>(chunks) * col_blocks),
                    dim3(tx, EMB_JOIN_THREADS / tx), 0, sm, d,
                    vocab, scale, static_cast<const int2*>(s.span), static_cast<const int*>(s.sid), col_blocks,
                    static_cast<const float*>(s.part), dw);
}

template <class I>
int embed_sort(const EmbedScratch& s, const void* ids, int64_t tokens, const int* count, int64_t vocab,
               int64_t padding, int* err, cudaStream_t sm, const DeviceInfo& dev) {
  // a power of two of blocks, so that owner and local number are bits of the
  // id: 128 (of 148 SMs), more when a block would own over EMB_MAX_RANGE ids
  int shift = 7;
  while ((vocab >> shift) >= EMB_MAX_RANGE) ++shift;
  const int64_t blocks = int64_t(1) << shift;
  const int range = static_cast<int>((vocab + blocks - 1) >> shift);
  const int smem = EMB_SORT_WARPS * range * static_cast<int>(sizeof(int));
  auto kern = k_embed_sort<I>;
  const int st = smem_attr_once(reinterpret_cast<const void*>(kern),
                                EMB_SORT_WARPS * EMB_MAX_RANGE * static_cast<int>(sizeof(int)));
  if (st != ETHOS_OK) return st;
  return launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(EMB_SORT_THREADS), static_cast<size_t>(smem), sm,
                    static_cast<const I*>(ids), static_cast<int>(tokens), count, vocab, padding, range, shift, s.span,
                    s.perm, s.sid, err);
}

template <class T>
int embed_table_grad(const EmbedScratch& s, const void* dy, int64_t tokens, int64_t vocab, int d, float scale,
                     void* dw, cudaStream_t sm, const DeviceInfo& dev) {
  T* o = static_cast<T*>(dw);
  return d % Vec16<T>::N == 0 && aligned16(dy) && aligned16(dw)
             ? embed_rows<T, true, T, false>(s, dy, d, nullptr, tokens, vocab, d, scale, o, sm, dev)
             : embed_rows<T, false, T, false>(s, dy, d, nullptr, tokens, vocab, d, scale, o, sm, dev);
}

// ---------------------------------------------------------------- balance --
// Selections from which counting by classes in shared memory is taken over
// global atomics.  With the loss pass, 262 144 selections took 20-26 us by
// classes whatever the ids, and 18 (even) to 58 us (crowded on few experts) by
// atomics; 131 072 took 21-27 against 18-35.
constexpr int64_t kBalanceClasses = 200000;
// Words of counters, over all blocks, from which storing them and adding them
// up in a pass of its own beats atomics on the counts: 8.4 M selections took,
// with the loss pass, 39 against 33 us for 4096 experts (0.3 M words, mostly
// full: few atomics), 58 against 67 us for 65 536 (4.8 M words of mostly one
// or two selections) and 94 against 104 us for 262 144.
constexpr int64_t kBalanceJoin = 2000000;

struct BalScratchAll {
  BalScratch* head;
  float* sel;
};
void carve_balance(Carve& c, int64_t n, BalScratchAll* s) {
  s->head = c.take<BalScratch>(1);
  s->sel = c.take<float>(static_cast<size_t>(n));
}

int balance_blocks(int64_t n, const DeviceInfo& dev) {
  int64_t b = (n / 4 + BAL_THREADS) / BAL_THREADS;
  const int64_t most = 8ll * dev.sm_count < BAL_MAX_BLOCKS ? 8ll * dev.sm_count : BAL_MAX_BLOCKS;
  return static_cast<int>(b < most ? b : most);
}

template <class I, class W>
int balance_forward(const void* ids_, const void* weights, const uint8_t* mask, int64_t tokens, int heads, int k,
                    int experts, int32_t* counts, float* loss, const BalScratchAll& s, int* err, cudaStream_t sm,
                    const DeviceInfo& dev) {
  const I* ids = static_cast<const I*>(ids_);
  const int T = static_cast<int>(tokens), per = heads * k;
  const int64_t n = tokens * per;
  const bool quads = per % 4 == 0 && aligned16(ids) && aligned16(weights);
  const int blocks = balance_blocks(n, dev);
  int shift = 0;  // log2 of the classes: groups of 8 experts, shared evenly
  const int groups = (experts + 7) / 8;
  while (((groups + (1 << shift) - 1) >> shift) * 8 > BAL_CLASS) ++shift;
  int st, live_parts;
  if (n >= kBalanceClasses && (1 << shift) <= dev.sm_count) {
    auto kern = k_balance_count_classes<I>;
    if ((st = smem_attr_once(reinterpret_cast<const void*>(kern), BAL_CLASS * 2)) != ETHOS_OK) return st;
    const int words = ((groups + (1 << shift) - 1) >> shift) * 4;
    live_parts = dev.sm_count >> shift;
    const int count_blocks = live_parts << shift;
    // the counters lie where the loss pass will write, if they fit
    const int64_t all = static_cast<int64_t>(count_blocks) * words;
    uint4* part = all >= kBalanceJoin && all <= n ? reinterpret_cast<uint4*>(s.sel) : nullptr;
    st = launch_pdl(kern, dim3(static_cast<unsigned>(count_blocks)), dim3(BAL_COUNT_THREADS),
                    static_cast<size_t>(words) * 4, sm, ids, mask, T, per, experts, quads, shift, words, counts, part,
                    s.head);
    if (st == ETHOS_OK && part != nullptr)
      st = launch_pdl(k_balance_join, dim3(static_cast<unsigned>(((words / 4 << shift) + 31) / 32)),
                      dim3(BAL_THREADS), 0, sm, static_cast<const uint4*>(part), live_parts, shift, words, experts,
                      counts);
  } else {
    live_parts = blocks;
    st = launch_pdl(k_balance_count<I>, dim3(blocks), dim3(BAL_THREADS), 0, sm, ids, mask, T, per, experts, quads,
                    counts, s.head);
  }
  if (st != ETHOS_OK) return st;
  return launch_pdl(k_balance_loss<I, W>, dim3(blocks), dim3(BAL_THREADS), 0, sm, ids,
                    static_cast<const W*>(weights), mask, T, heads, k, experts, quads, live_parts,
                    static_cast<const int*>(counts), s.head, s.sel, loss, err);
}

template <class W>
int balance_backward(int64_t n, int heads, int k, int experts, const BalScratchAll& s, const float* grad, void* dw,
                     cudaStream_t sm, const DeviceInfo& dev) {
  return launch_pdl(k_balance_bwd<W>, dim3(balance_blocks(n, dev)), dim3(BAL_THREADS), 0, sm, static_cast<int>(n),
                    heads, k, experts, n % 4 == 0 && aligned16(dw), static_cast<const BalScratch*>(s.head),
                    static_cast<const float*>(s.sel), grad, static_cast<W*>(dw));
}

int balance_check(int dtype, int64_t tokens, int64_t heads, int64_t k, int64_t experts) {
  if (tokens < 0 || heads < 1 || k < 1 || experts < 1 || !known_dtype(dtype)) return ETHOS_ERR_INVALID_ARG;
  // selections are numbered, and counted, in int32
  if (experts >= (1 << 30) || heads > (1 << 20) || k > (1 << 20) || tokens > (int64_t(1) << 30) / (heads * k))
    return ETHOS_ERR_UNSUPPORTED_SHAPE;
  return ETHOS_OK;
}

// ---------------------------------------------------------- cross entropy --
// Layout of one problem.  The unit counts assume 74 SM pairs (a B200); the
// kernels are right for any number.
constexpr int64_t kPairs = 74;
// one piece's gradient of the logits; at least XE_MIN_PIECE columns
constexpr int64_t kPieceBytes = int64_t(1) << 30;
constexpr int64_t kMinPiece = 8192;
// largest E of the keep way: 16 384 tokens of a 100 277-word vocabulary take
// 3.3 GB of the GPU's 180 for the length of the call
constexpr int64_t kKeepBytes = int64_t(4) << 30;

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct XentPlan {
  int64_t T, V, d;
  int planes;
  int tile_n;              // columns of a GEMM tile
  bool keep;               // the keep way is open
  bool pack_w;             // the table is read through bf16 planes
  bool pad_dw;             // bf16 dW of an odd width goes through padded rows
  int64_t ldd;             // columns of a plane
  int64_t t_pad, v_pad;    // rows of a plane
  int run, runs;           // STATS: column tiles per unit, units along the vocabulary
  int64_t piece;           // DLOGITS, GRADS: columns of a piece
  int slots, slots_piece;  // K slices of dh: keep way, piece way
  int64_t dh_ld;
};

XentPlan xent_plan(int64_t T, int64_t V, int64_t d, int dtype) {
  XentPlan p;
  p.T = T;
  p.V = V;
  p.d = d;
  p.planes = dtype == ETHOS_F32 ? 3 : 1;
  p.tile_n = p.planes == 1 ? XeCfg<1>::kTileN : XeCfg<3>::kTileN;
  p.pack_w = dtype == ETHOS_F32 || d % 8 != 0;
  p.pad_dw = dtype == ETHOS_BF16 && d % 8 != 0;
  p.ldd = up(d, 8);
  p.t_pad = up(T, XE_TILE);
  p.v_pad = up(V, XE_TILE);
  p.keep = p.planes == 1 && p.t_pad * up(V, 64) * 2 <= kKeepBytes;
  const int64_t num_m = p.t_pad / XE_TILE, num_n = (V + p.tile_n - 1) / p.tile_n;
  // a unit's columns: the most (up to 4096) that leave the last round of units
  // as full as any choice does, within a percent; one tile where six rounds
  // are not reached (how many rows there are is known on the device only)
  auto rounds = [&](int64_t run) { return (num_m * ((num_n + run - 1) / run) + kPairs - 1) / kPairs * run; };
  int64_t best = rounds(1);
  for (int64_t run = 2; run <= 4096 / p.tile_n; ++run) best = rounds(run) < best ? rounds(run) : best;
  p.run = 1;
  for (int64_t run = 2; run <= 4096 / p.tile_n; ++run)
    if (num_m * ((num_n + run - 1) / run) >= 6 * kPairs && 100 * rounds(run) <= 101 * best)
      p.run = static_cast<int>(run);
  p.runs = static_cast<int>((num_n + p.run - 1) / p.run);
  int64_t most = kPieceBytes / (p.t_pad * 2 * p.planes) / XE_TILE * XE_TILE;
  if (most < kMinPiece) most = kMinPiece;
  const int64_t pieces = (V + most - 1) / most;
  p.piece = up((V + pieces - 1) / pieces, XE_TILE);
  p.dh_ld = up(d, 8);
  if (pieces > 1 && !p.keep) {
    p.slots = 1;
  } else {
    // few row tiles and a long contraction: cut dh's K so that a tile's slice
    // is at most about half of a pair's share of the whole work (gradients of
    // 120, 256 and 600 tokens of 100 277 x 1024, in us: 258, 275, 425 with a
    // third, 250, 263, 414 with half, 268, 275, 400 with the whole of it)
    const int64_t nt = (d + p.tile_n - 1) / p.tile_n;
    const int64_t kb_h = (V + G2_BK - 1) / G2_BK, kb_w = (T + G2_BK - 1) / G2_BK;
    const int64_t least = p.planes == 1 ? XeCfg<1>::kStoreKb : XeCfg<3>::kStoreKb;
    const int64_t cost_w = kb_w > least ? kb_w : least;
    const int64_t share = (num_m * nt * kb_h + p.v_pad / XE_TILE * nt * cost_w) / (kPairs * 2);
    const int64_t target = share > 8 ? share : 8;
    int64_t s = (kb_h + target - 1) / target;
    if (s > 64) s = 64;
    const int64_t per = (kb_h + s - 1) / s;
    p.slots = static_cast<int>((kb_h + per - 1) / per);
  }
  p.slots_piece = pieces == 1 ? p.slots : 1;
  return p;
}

struct XentSave {
  XeRows rw;
  __nv_bfloat16* hp;  // packed rows of hidden, [planes][t_pad][ldd]
};
void carve_save(Carve& c, const XentPlan& p, XentSave* s) {
  s->rw.meta = c.take<XeMeta>(1);
  s->rw.pos = c.take<int>(static_cast<size_t>(p.T));
  s->rw.idx = c.take<int>(static_cast<size_t>(p.t_pad));
  s->rw.yc = c.take<int>(static_cast<size_t>(p.t_pad));
  s->rw.lab = c.take<float>(static_cast<size_t>(p.t_pad));
  s->rw.c = c.take<float>(static_cast<size_t>(p.t_pad));
  s->rw.lse = c.take<float>(static_cast<size_t>(p.t_pad));
  s->rw.q = c.take<float>(static_cast<size_t>(p.t_pad));
  s->rw.r = c.take<float>(static_cast<size_t>(p.t_pad));
  s->hp = c.take<__nv_bfloat16>(static_cast<size_t>(p.planes * p.t_pad * p.ldd));
}
struct XentFwd {
  __nv_bfloat16* wp;
  float2* part;
  double* block_sum;
};
void carve_xent_fwd(Carve& c, const XentPlan& p, XentFwd* s) {
  s->wp = p.pack_w ? c.take<__nv_bfloat16>(static_cast<size_t>(p.planes * p.v_pad * p.ldd)) : nullptr;
  const int64_t parts = 2 * p.runs > XE_FEW_BLOCKS ? 2 * p.runs : XE_FEW_BLOCKS;
  s->part = c.take<float2>(static_cast<size_t>(parts * p.t_pad));
  s->block_sum = c.take<double>(static_cast<size_t>(p.t_pad / XE_LOSS_ROWS));
}
struct XentBwd {
  __nv_bfloat16* wp;
  __nv_bfloat16* dl;
  float* dh;
  __nv_bfloat16* dwp;  // rows of dW at a pitch of whole 16-byte pieces
  // bf16: the label's terms, as in the keep way
  float* label_grad;
  EmbedScratch sort;
  float* label_rows;
};
void carve_xent_bwd(Carve& c, const XentPlan& p, XentBwd* s) {
  s->wp = p.pack_w ? c.take<__nv_bfloat16>(static_cast<size_t>(p.planes * p.v_pad * p.ldd)) : nullptr;
  s->dl = c.take<__nv_bfloat16>(static_cast<size_t>(p.planes * p.t_pad * p.piece));
  s->dh = c.take<float>(static_cast<size_t>(p.slots_piece * p.t_pad * p.dh_ld));
  s->dwp = p.pad_dw ? c.take<__nv_bfloat16>(static_cast<size_t>(p.piece * p.ldd)) : nullptr;
  s->label_grad = s->label_rows = nullptr;
  if (p.planes != 1) return;
  s->label_grad = c.take<float>(static_cast<size_t>(p.t_pad));
  carve_embed(c, p.t_pad, p.V, p.d, &s->sort);
  s->label_rows = c.take<float>(static_cast<size_t>(p.t_pad * p.d));
}
struct XentKeep {
  XentFwd f;
  int* redo_tile;
  __nv_bfloat16* e;     // [t_pad][lde]
  int64_t lde;
  __nv_bfloat16* hr;    // rows r h
  float* dh;
  EmbedScratch sort;
  float* label_rows;
  __nv_bfloat16* dwp;
};
void carve_xent_keep(Carve& c, const XentPlan& p, XentKeep* s) {
  carve_xent_fwd(c, p, &s->f);
  s->lde = up(p.V, 64);
  s->redo_tile = c.take<int>(static_cast<size_t>(p.t_pad / XE_TILE));
  s->e = c.take<__nv_bfloat16>(static_cast<size_t>(p.t_pad * s->lde));
  s->hr = c.take<__nv_bfloat16>(static_cast<size_t>(p.t_pad * p.ldd));
  s->dh = c.take<float>(static_cast<size_t>(p.slots * p.t_pad * p.dh_ld));
  carve_embed(c, p.t_pad, p.V, p.d, &s->sort);
  s->label_rows = c.take<float>(static_cast<size_t>(p.t_pad * p.d));
  s->dwp = p.pad_dw ? c.take<__nv_bfloat16>(static_cast<size_t>(p.v_pad * p.ldd)) : nullptr;
}

int xent_pack_w(const XentPlan& p, int dtype, const void* weight, int64_t ldw, __nv_bfloat16* wp, cudaStream_t sm,
                const DeviceInfo& dev) {
  int64_t blocks = (p.v_pad * (p.ldd / 8) + 255) / 256;
  if (blocks > 16ll * dev.sm_count) blocks = 16ll * dev.sm_count;
  const dim3 grid(static_cast<unsigned>(blocks));
  const int d = static_cast<int>(p.d), ldd = static_cast<int>(p.ldd);
  return dtype == ETHOS_BF16
             ? launch_pdl(k_xent_pack<__nv_bfloat16, 1>, grid, dim3(256), 0, sm,
                          static_cast<const __nv_bfloat16*>(weight), ldw, d, p.V, wp, p.v_pad, ldd)
             : launch_pdl(k_xent_pack<float, 3>, grid, dim3(256), 0, sm, static_cast<const float*>(weight), ldw, d,
                          p.V, wp, p.v_pad, ldd);
}

// The packed rows and the labels' logits.
int xent_rows_pass(const XentPlan& p, const XentSave& sv, const void* hidden, int64_t ldh, const void* weight,
                   int64_t ldw, int dtype, cudaStream_t sm, const DeviceInfo& dev) {
  int64_t blocks = (p.t_pad + 7) / 8;
  if (blocks > 8ll * dev.sm_count) blocks = 8ll * dev.sm_count;
  const dim3 grid(static_cast<unsigned>(blocks));
  const int d = static_cast<int>(p.d), ldd = static_cast<int>(p.ldd);
  return dtype == ETHOS_BF16
             ? launch_pdl(k_xent_rows<__nv_bfloat16, 1>, grid, dim3(256), 0, sm,
                          static_cast<const __nv_bfloat16*>(hidden), ldh, static_cast<const __nv_bfloat16*>(weight),
                          ldw, p.V, d, sv.rw, sv.hp, p.t_pad, ldd)
             : launch_pdl(k_xent_rows<float, 3>, grid, dim3(256), 0, sm, static_cast<const float*>(hidden), ldh,
                          static_cast<const float*>(weight), ldw, p.V, d, sv.rw, sv.hp, p.t_pad, ldd);
}

int xent_index(const XentPlan& p, const XentSave& sv, const void* labels, int labels_i64, int64_t ignore_index,
               float* loss_rows, int* redo_tile, int* err, cudaStream_t sm) {
  const bool compact = p.T > XE_ROWS_IN_PLACE;
  const int T = static_cast<int>(p.T);
  return labels_i64 ? launch_pdl(k_xent_index<int64_t>, dim3(1), dim3(1024), 0, sm,
                                 static_cast<const int64_t*>(labels), T, p.V, ignore_index, compact, sv.rw, loss_rows,
                                 redo_tile, err)
                    : launch_pdl(k_xent_index<int32_t>, dim3(1), dim3(1024), 0, sm,
                                 static_cast<const int32_t*>(labels), T, p.V, ignore_index, compact, sv.rw, loss_rows,
                                 redo_tile, err);
}

template <int MODE, int PLANES>
int launch_xent(const CUtensorMap& a0, const CUtensorMap& b0, const CUtensorMap& a1, const CUtensorMap& b1,
                const CUtensorMap& c, const XeArgs& args, int64_t units, int* err, cudaStream_t sm, const DeviceInfo& dev) {
  auto kern = k_xent_gemm<MODE, PLANES>;
  int st = smem_attr_once(reinterpret_cast<const void*>(kern), xe_smem<PLANES>());
  if (st != ETHOS_OK) return st;
  // the kernel divides its registers anew and would wait for ever for more
  // than the launch has
  static const bool regs_ok = [] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, k_xent_gemm<MODE, PLANES>) == cudaSuccess && fa.numRegs == XE_LAUNCH_REGS;
  }();
  if (!regs_ok) return ETHOS_ERR_CUDA;
  int64_t pairs = max_pair_clusters(reinterpret_cast<const void*>(kern), XE_THREADS, xe_smem<PLANES>(), dev);
  if (pairs <= 0) return ETHOS_ERR_CUDA;
  if (pairs > units) pairs = units;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(static_cast<unsigned>(XE_THREADS));
  cfg.dynamicSmemBytes = static_cast<size_t>(xe_smem<PLANES>());
  cfg.stream = sm;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launch();
  if (cudaLaunchKernelEx(&cfg, kern, a0, b0, a1, b1, c, args, err) != cudaSuccess) return ETHOS_ERR_CUDA;
  return launch_status();
}
template <int MODE>
int launch_xent_planes(int planes, const CUtensorMap& a0, const CUtensorMap& b0, const CUtensorMap& a1,
                       const CUtensorMap& b1, const CUtensorMap& c, const XeArgs& args, int64_t units, int* err,
                       cudaStream_t sm, const DeviceInfo& dev) {
  return planes == 1 ? launch_xent<MODE, 1>(a0, b0, a1, b1, c, args, units, err, sm, dev)
                     : launch_xent<MODE, 3>(a0, b0, a1, b1, c, args, units, err, sm, dev);
}

// The logits' GEMM over the whole vocabulary: row statistics, and E (KEEP).
template <int MODE>
int xent_logits(const XentPlan& p, const XentSave& sv, const void* weight, int64_t ldw, const XentFwd& ws,
                __nv_bfloat16* e, int64_t lde, const int* redo_tile, int* err, cudaStream_t sm,
                const DeviceInfo& dev) {
  CUtensorMap ta, tb;
  int st;
  if ((st = make_tmap_bf16(&ta, sv.hp, p.planes * p.t_pad, p.ldd, G2_BM, p.ldd)) != ETHOS_OK) return st;
  st = p.pack_w ? make_tmap_bf16(&tb, ws.wp, p.planes * p.v_pad, p.ldd, G2_BM, p.ldd)
                : make_tmap_bf16(&tb, weight, p.V, p.d, G2_BM, ldw);
  if (st != ETHOS_OK) return st;
  XeArgs a = {};
  a.rw = sv.rw;
  a.p[0] = XeProduct{static_cast<int>(p.t_pad), static_cast<int>(p.v_pad), static_cast<int>(p.T),
                     static_cast<int>(p.V), static_cast<int>(p.d)};
  a.run = p.run;
  a.part = ws.part;
  a.part_ld = p.t_pad;
  a.redo_tile = redo_tile;
  a.dl = e;
  a.ldl = lde;
  const int64_t units = p.t_pad / XE_TILE * p.runs;
  if constexpr (MODE == XE_KEEP) {
    CUtensorMap tc;
    if ((st = make_tmap_bf16(&tc, e, p.t_pad, lde, 32, lde)) != ETHOS_OK) return st;
    return launch_xent<MODE, 1>(ta, tb, ta, tb, tc, a, units, err, sm, dev);
  } else {
    return launch_xent_planes<MODE>(p.planes, ta, tb, ta, tb, ta, a, units, err, sm, dev);
  }
}

int xent_loss(const XentPlan& p, const XentSave& sv, const XentFwd& ws, int reduction, float* loss, cudaStream_t sm,
              int parts, bool keep = false, bool again = false, int* redo_tile = nullptr, __nv_bfloat16* hr = nullptr) {
  const int64_t rows = hr ? p.t_pad : p.T;
  return launch_pdl(k_xent_loss, dim3(static_cast<unsigned>((rows + XE_LOSS_ROWS - 1) / XE_LOSS_ROWS)), dim3(256), 0,
                    sm, sv.rw, static_cast<const float2*>(ws.part), parts, p.t_pad, keep, again, redo_tile,
                    reduction, loss, ws.block_sum, static_cast<const __nv_bfloat16*>(sv.hp), hr,
                    static_cast<int>(p.ldd));
}

// Where the products leave dW, and its tensor map: its own rows [rows][d], or
// the padded rows dwp, as 16-byte pieces (bf16); any map where it has neither.
int xent_dw_out(CUtensorMap* m, const CUtensorMap& other, XeArgs* g, void* dw, int64_t rows, int64_t d,
                __nv_bfloat16* dwp, int64_t ldd) {
  g->do_dw = dw != nullptr;
  g->dw = dw != nullptr && dwp != nullptr ? dwp : dw;
  g->dw_ld = dwp != nullptr ? ldd : d;
  g->dw_tma = g->do_dw && g->dw_bf16 && aligned16(g->dw);
  if (g->dw_tma) return make_tmap_bf16(m, g->dw, rows, g->dw_ld, 32, g->dw_ld);
  *m = other;
  return ETHOS_OK;
}
int xent_unpad(const __nv_bfloat16* dwp, int64_t ldd, int64_t rows, int64_t d, void* dw, cudaStream_t sm,
               const DeviceInfo& dev) {
  int64_t blocks = (rows * d / 8 + 256) / 256;
  if (blocks > 16ll * dev.sm_count) blocks = 16ll * dev.sm_count;
  return launch_pdl(k_xent_unpad, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, sm, dwp, ldd,
                    static_cast<int>(d), rows * d, static_cast<__nv_bfloat16*>(dw));
}

// The forward of few tokens (xent_is_few).
template <class S, bool kVec>
int xent_few_t(const XentPlan& p, const XentSave& sv, const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
               const void* labels, int labels_i64, int64_t ignore, float* loss_rows, const XentFwd& ws, int* err,
               cudaStream_t sm) {
  const S* h = static_cast<const S*>(hidden);
  const S* w = static_cast<const S*>(weight);
  const int tt = p.T <= 1 ? 1 : (p.T <= 2 ? 2 : (p.T <= 4 ? 4 : 8));
  const int step = 32 * RowAccess<S, kVec>::N;
  const size_t smem = static_cast<size_t>(tt) * up(p.d, step) * sizeof(float);
  auto go = [&](auto kern) {
    const int st = smem_attr_once(reinterpret_cast<const void*>(kern), XE_FEW_SMEM);
    if (st != ETHOS_OK) return st;
    return launch_pdl(kern, dim3(XE_FEW_BLOCKS), dim3(256), smem, sm, h, ldh, w, ldw, static_cast<int>(p.d),
                      static_cast<int>(p.V), static_cast<int>(p.T), labels, labels_i64 != 0, ignore, sv.rw, loss_rows,
                      ws.part, p.t_pad, err);
  };
  if (tt == 1) return go(k_xent_few<S, kVec, 1>);
  if constexpr (xe_few<S, kVec>() >= 2) {
    if (tt == 2) return go(k_xent_few<S, kVec, 2>);
  }
  if constexpr (xe_few<S, kVec>() >= 4) {
    if (tt == 4) return go(k_xent_few<S, kVec, 4>);
  }
  if constexpr (xe_few<S, kVec>() >= 8) {
    if (tt == 8) return go(k_xent_few<S, kVec, 8>);
  }
  return ETHOS_ERR_UNSUPPORTED_SHAPE;
}
// By width, not by address: the backward asks again and has to find the same.
// (bf16 tables of whole 16-byte rows at other addresses are refused before.)
bool xent_is_few(const XentPlan& p) {
  const int most = p.planes == 3 ? xe_few<float, true>()
                                 : (p.pack_w ? xe_few<__nv_bfloat16, false>() : xe_few<__nv_bfloat16, true>());
  return p.T <= most && up(p.T, 8) * up(p.d, 256) * 4 <= XE_FEW_SMEM;
}
int xent_few(const XentPlan& p, const XentSave& sv, const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
             int dtype, const void* labels, int labels_i64, int64_t ignore, float* loss_rows, const XentFwd& ws,
             int* err, cudaStream_t sm) {
  const int esz = dtype == ETHOS_BF16 ? 2 : 4;
  const bool vec = p.d * esz % 16 == 0 && ldw * esz % 16 == 0 && aligned16(weight);
  if (dtype == ETHOS_BF16)
    return vec ? xent_few_t<__nv_bfloat16, true>(p, sv, hidden, ldh, weight, ldw, labels, labels_i64, ignore, loss_rows,
                                                 ws, err, sm)
               : xent_few_t<__nv_bfloat16, false>(p, sv, hidden, ldh, weight, ldw, labels, labels_i64, ignore,
                                                  loss_rows, ws, err, sm);
  return vec ? xent_few_t<float, true>(p, sv, hidden, ldh, weight, ldw, labels, labels_i64, ignore, loss_rows, ws, err,
                                       sm)
             : xent_few_t<float, false>(p, sv, hidden, ldh, weight, ldw, labels, labels_i64, ignore, loss_rows, ws,
                                        err, sm);
}

int64_t xent_grad_units(const XentPlan& p, int64_t n, int slots, const XeArgs& g) {
  const int64_t nt = (p.d + p.tile_n - 1) / p.tile_n;
  return (g.do_dh ? p.t_pad / XE_TILE * nt * slots : 0) + (g.do_dw ? (n + XE_TILE - 1) / XE_TILE * nt : 0);
}

// Label rows of dW (bf16): e[t] h[t] summed by label.
int xent_label_rows(const XentPlan& p, const XentSave& sv, const EmbedScratch& sort, const float* e, float* label_rows,
                    int* err, cudaStream_t sm, const DeviceInfo& dev) {
  const int st = embed_sort<int32_t>(sort, sv.rw.yc, p.t_pad, &sv.rw.meta->rows, p.V, -1, err, sm, dev);
  if (st != ETHOS_OK) return st;
  const int d = static_cast<int>(p.d);
  return d % 8 == 0 ? embed_rows<__nv_bfloat16, true, float, true>(sort, sv.hp, p.ldd, e, p.t_pad, p.V, d, 1.0f,
                                                                   label_rows, sm, dev)
                    : embed_rows<__nv_bfloat16, false, float, true>(sort, sv.hp, p.ldd, e, p.t_pad, p.V, d, 1.0f,
                                                                    label_rows, sm, dev);
}

template <class D>
int xent_dhidden(const XentPlan& p, const XentSave& sv, const float* acc, int slots, const float* grad, int reduction,
                 const float* f_rows, const float* e_rows, const void* weight, int64_t ldw, void* out,
                 cudaStream_t sm, const DeviceInfo& dev) {
  int64_t blocks = (p.T * ((p.d + 7) / 8) + 255) / 256;
  if (blocks > 16ll * dev.sm_count) blocks = 16ll * dev.sm_count;
  return launch_pdl(k_xent_dhidden<D>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, sm, acc, slots,
                    p.t_pad * p.dh_ld, p.dh_ld, sv.rw, grad, reduction, f_rows, e_rows, static_cast<const D*>(weight),
                    ldw, p.V, p.T, static_cast<int>(p.d), static_cast<D*>(out));
}

int xent_check(int64_t tokens, int64_t vocab, int64_t dim, int64_t ldh, int64_t ldw, int dtype, int reduction) {
  if (tokens < 1 || vocab < 1 || dim < 1 || ldh < dim || ldw < dim || !known_dtype(dtype)) return ETHOS_ERR_INVALID_ARG;
  if (reduction < XE_NONE || reduction > XE_MEAN) return ETHOS_ERR_INVALID_ARG;
  if (tokens > (1 << 24) || vocab > (1 << 24) || dim > (1 << 16)) return ETHOS_ERR_UNSUPPORTED_SHAPE;
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
             ? embed_fwd_ids<__nv_bfloat16>(ids, ids_i64, weight, ldw, tokens, vocab, d, scale, out, dev_err, sm)
             : embed_fwd_ids<float>(ids, ids_i64, weight, ldw, tokens, vocab, d, scale, out, dev_err, sm);
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
  if (padding < 0) padding = EMB_NO_PADDING;
  st = ids_i64 ? embed_sort<int64_t>(s, ids, tokens, nullptr, vocab, padding, dev_err, sm, *dev)
               : embed_sort<int32_t>(s, ids, tokens, nullptr, vocab, padding, dev_err, sm, *dev);
  if (st != ETHOS_OK) return st;
  const int d = static_cast<int>(dim);
  return dtype == ETHOS_BF16 ? embed_table_grad<__nv_bfloat16>(s, dy, tokens, vocab, d, scale, d_weight, sm, *dev)
                             : embed_table_grad<float>(s, dy, tokens, vocab, d, scale, d_weight, sm, *dev);
}

size_t ethos_balance_scratch_size(int64_t tokens, int64_t heads, int64_t k) {
  if (balance_check(ETHOS_F32, tokens, heads, k, 1) != ETHOS_OK) return 0;
  Carve c{nullptr, 0, 0};
  BalScratchAll s;
  carve_balance(c, tokens * heads * k, &s);
  return c.off + 256;
}

int ethos_balance_forward(const void* ids, int ids_i64, const void* weights, int dtype, const uint8_t* mask,
                          int64_t tokens, int64_t heads, int64_t k, int64_t experts, int32_t* counts, float* loss,
                          void* scratch, size_t scratch_bytes, int* dev_err, void* stream) {
  int st = balance_check(dtype, tokens, heads, k, experts);
  if (st != ETHOS_OK) return st;
  if ((tokens > 0 && (!ids || !weights)) || !counts || !loss || !dev_err) return ETHOS_ERR_INVALID_ARG;
  Carve c{static_cast<char*>(scratch), 0, scratch_bytes};
  BalScratchAll s;
  carve_balance(c, tokens * heads * k, &s);
  if (!scratch || c.off > scratch_bytes) return ETHOS_ERR_WORKSPACE;
  if (!aligned16(scratch)) return ETHOS_ERR_ALIGNMENT;
  DeviceInfo* dev = nullptr;
  if ((st = base_device_info(&dev)) != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  if (cudaMemsetAsync(counts, 0, sizeof(int32_t) * static_cast<size_t>(experts), sm) != cudaSuccess)
    return ETHOS_ERR_CUDA;
  const int H = static_cast<int>(heads), K = static_cast<int>(k), N = static_cast<int>(experts);
  if (ids_i64)
    return dtype == ETHOS_BF16 ? balance_forward<int64_t, __nv_bfloat16>(ids, weights, mask, tokens, H, K, N, counts,
                                                                         loss, s, dev_err, sm, *dev)
                               : balance_forward<int64_t, float>(ids, weights, mask, tokens, H, K, N, counts, loss, s,
                                                                 dev_err, sm, *dev);
  return dtype == ETHOS_BF16 ? balance_forward<int32_t, __nv_bfloat16>(ids, weights, mask, tokens, H, K, N, counts,
                                                                       loss, s, dev_err, sm, *dev)
                             : balance_forward<int32_t, float>(ids, weights, mask, tokens, H, K, N, counts, loss, s,
                                                               dev_err, sm, *dev);
}

int ethos_balance_backward(int dtype, int64_t tokens, int64_t heads, int64_t k, int64_t experts,
                           const void* scratch, size_t scratch_bytes, const float* grad, void* d_weights,
                           void* stream) {
  int st = balance_check(dtype, tokens, heads, k, experts);
  if (st != ETHOS_OK) return st;
  if (tokens == 0) return ETHOS_OK;
  if (!grad || !d_weights) return ETHOS_ERR_INVALID_ARG;
  Carve c{static_cast<char*>(const_cast<void*>(scratch)), 0, scratch_bytes};
  BalScratchAll s;
  carve_balance(c, tokens * heads * k, &s);
  if (!scratch || c.off > scratch_bytes) return ETHOS_ERR_WORKSPACE;
  if (!aligned16(scratch)) return ETHOS_ERR_ALIGNMENT;
  DeviceInfo* dev = nullptr;
  if ((st = base_device_info(&dev)) != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  const int H = static_cast<int>(heads), K = static_cast<int>(k), N = static_cast<int>(experts);
  return dtype == ETHOS_BF16
             ? balance_backward<__nv_bfloat16>(tokens * heads * k, H, K, N, s, grad, d_weights, sm, *dev)
             : balance_backward<float>(tokens * heads * k, H, K, N, s, grad, d_weights, sm, *dev);
}

size_t ethos_xent_save_size(int64_t tokens, int64_t vocab, int64_t dim, int dtype) {
  if (xent_check(tokens, vocab, dim, dim, dim, dtype, 0) != ETHOS_OK) return 0;
  Carve c{nullptr, 0, 0};
  XentSave s;
  carve_save(c, xent_plan(tokens, vocab, dim, dtype), &s);
  return c.off + 256;
}

size_t ethos_xent_forward_workspace_size(int64_t tokens, int64_t vocab, int64_t dim, int dtype) {
  if (xent_check(tokens, vocab, dim, dim, dim, dtype, 0) != ETHOS_OK) return 0;
  Carve c{nullptr, 0, 0};
  XentFwd s;
  carve_xent_fwd(c, xent_plan(tokens, vocab, dim, dtype), &s);
  return c.off + 256;
}

size_t ethos_xent_backward_workspace_size(int64_t tokens, int64_t vocab, int64_t dim, int dtype) {
  if (xent_check(tokens, vocab, dim, dim, dim, dtype, 0) != ETHOS_OK) return 0;
  Carve c{nullptr, 0, 0};
  XentBwd s;
  carve_xent_bwd(c, xent_plan(tokens, vocab, dim, dtype), &s);
  return c.off + 256;
}

int ethos_xent_forward(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, int dtype,
                       const void* labels, int labels_i64, int64_t ignore_index, int reduction, int64_t tokens,
                       int64_t vocab, int64_t dim, float* loss, void* save, size_t save_bytes, void* workspace,
                       size_t workspace_bytes, int* dev_err, void* stream) {
  int st = xent_check(tokens, vocab, dim, ldh, ldw, dtype, reduction);
  if (st != ETHOS_OK) return st;
  if (!hidden || !weight || !labels || !loss || !dev_err) return ETHOS_ERR_INVALID_ARG;
  const XentPlan p = xent_plan(tokens, vocab, dim, dtype);
  Carve cs{static_cast<char*>(save), 0, save_bytes}, cw{static_cast<char*>(workspace), 0, workspace_bytes};
  XentSave sv;
  XentFwd ws;
  carve_save(cs, p, &sv);
  carve_xent_fwd(cw, p, &ws);
  if (!save || !workspace || cs.off > save_bytes || cw.off > workspace_bytes) return ETHOS_ERR_WORKSPACE;
  if (!aligned16(save) || !aligned16(workspace)) return ETHOS_ERR_ALIGNMENT;
  if (!p.pack_w && (ldw % 8 != 0 || !aligned16(weight))) return ETHOS_ERR_ALIGNMENT;
  DeviceInfo* dev = nullptr;
  if ((st = base_device_info(&dev)) != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  float* loss_rows = reduction == XE_NONE ? loss : nullptr;
  if (xent_is_few(p)) {
    if ((st = xent_few(p, sv, hidden, ldh, weight, ldw, dtype, labels, labels_i64, ignore_index, loss_rows, ws,
                       dev_err, sm)) != ETHOS_OK)
      return st;
    return xent_loss(p, sv, ws, reduction, loss, sm, XE_FEW_BLOCKS);
  }
  if ((st = xent_index(p, sv, labels, labels_i64, ignore_index, loss_rows, nullptr, dev_err, sm)) != ETHOS_OK)
    return st;
  if ((st = xent_rows_pass(p, sv, hidden, ldh, weight, ldw, dtype, sm, *dev)) != ETHOS_OK) return st;
  if (p.pack_w && (st = xent_pack_w(p, dtype, weight, ldw, ws.wp, sm, *dev)) != ETHOS_OK) return st;
  if ((st = xent_logits<XE_STATS>(p, sv, weight, ldw, ws, nullptr, 0, nullptr, dev_err, sm, *dev)) != ETHOS_OK)
    return st;
  return xent_loss(p, sv, ws, reduction, loss, sm, 2 * p.runs);
}

size_t ethos_xent_forward_backward_workspace_size(int64_t tokens, int64_t vocab, int64_t dim, int dtype) {
  if (xent_check(tokens, vocab, dim, dim, dim, dtype, 0) != ETHOS_OK) return 0;
  const XentPlan p = xent_plan(tokens, vocab, dim, dtype);
  if (!p.keep) return 0;
  Carve c{nullptr, 0, 0};
  XentKeep s;
  carve_xent_keep(c, p, &s);
  return c.off + 256;
}

int ethos_xent_forward_backward(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, int dtype,
                                const void* labels, int labels_i64, int64_t ignore_index, int reduction,
                                int64_t tokens, int64_t vocab, int64_t dim, float* loss, void* save,
                                size_t save_bytes, void* d_hidden, void* d_weight, void* workspace,
                                size_t workspace_bytes, int* dev_err, void* stream) {
  int st = xent_check(tokens, vocab, dim, ldh, ldw, dtype, reduction);
  if (st != ETHOS_OK) return st;
  if (!hidden || !weight || !labels || !loss || !dev_err || reduction == XE_NONE) return ETHOS_ERR_INVALID_ARG;
  const XentPlan p = xent_plan(tokens, vocab, dim, dtype);
  if (!p.keep) return ETHOS_ERR_UNSUPPORTED_SHAPE;
  Carve cs{static_cast<char*>(save), 0, save_bytes}, cw{static_cast<char*>(workspace), 0, workspace_bytes};
  XentSave sv;
  XentKeep ws;
  carve_save(cs, p, &sv);
  carve_xent_keep(cw, p, &ws);
  if (!save || !workspace || cs.off > save_bytes || cw.off > workspace_bytes) return ETHOS_ERR_WORKSPACE;
  if (!aligned16(save) || !aligned16(workspace)) return ETHOS_ERR_ALIGNMENT;
  if (!p.pack_w && (ldw % 8 != 0 || !aligned16(weight))) return ETHOS_ERR_ALIGNMENT;
  DeviceInfo* dev = nullptr;
  if ((st = base_device_info(&dev)) != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  const int D = static_cast<int>(dim);
  if ((st = xent_index(p, sv, labels, labels_i64, ignore_index, nullptr, ws.redo_tile, dev_err, sm)) != ETHOS_OK)
    return st;
  if ((st = xent_rows_pass(p, sv, hidden, ldh, weight, ldw, dtype, sm, *dev)) != ETHOS_OK) return st;
  if (p.pack_w && (st = xent_pack_w(p, dtype, weight, ldw, ws.f.wp, sm, *dev)) != ETHOS_OK) return st;
  // E and the sums; rows whose shift was too low once more with their maximum
  if ((st = xent_logits<XE_KEEP>(p, sv, weight, ldw, ws.f, ws.e, ws.lde, nullptr, dev_err, sm, *dev)) != ETHOS_OK)
    return st;
  __nv_bfloat16* hr = d_weight ? ws.hr : nullptr;
  if ((st = xent_loss(p, sv, ws.f, reduction, loss, sm, 2 * p.runs, true, false, ws.redo_tile, hr)) != ETHOS_OK) return st;
  if ((st = xent_logits<XE_KEEP>(p, sv, weight, ldw, ws.f, ws.e, ws.lde, ws.redo_tile, dev_err, sm, *dev)) !=
      ETHOS_OK)
    return st;
  if ((st = xent_loss(p, sv, ws.f, reduction, loss, sm, 2 * p.runs, true, true, ws.redo_tile, hr)) != ETHOS_OK) return st;
  if (!d_hidden && !d_weight) return ETHOS_OK;
  if (d_weight) {
    if ((st = xent_label_rows(p, sv, ws.sort, sv.rw.q, ws.label_rows, dev_err, sm, *dev)) != ETHOS_OK) return st;
  }
  const void* wptr = p.pack_w ? static_cast<const void*>(ws.f.wp) : weight;
  const int64_t wld = p.pack_w ? p.ldd : ldw;
  CUtensorMap ek, em, wk, hb;
  if ((st = make_tmap_bf16(&ek, ws.e, p.t_pad, ws.lde, G2_BM, ws.lde)) != ETHOS_OK) return st;
  if ((st = make_tmap_bf16(&em, ws.e, p.t_pad, ws.lde, G2_BK, ws.lde)) != ETHOS_OK) return st;
  if ((st = make_tmap_bf16(&wk, wptr, p.pack_w ? p.v_pad : vocab, p.pack_w ? p.ldd : dim, G2_BK, wld)) != ETHOS_OK)
    return st;
  if ((st = make_tmap_bf16(&hb, ws.hr, p.t_pad, p.ldd, G2_BK, p.ldd)) != ETHOS_OK) return st;
  const int T = static_cast<int>(tokens), V = static_cast<int>(vocab);
  XeArgs g = {};
  g.rw = sv.rw;
  g.reduction = reduction;
  g.p[0] = XeProduct{0, 0, T, D, V};
  g.p[1] = XeProduct{0, 0, V, D, T};
  g.dh_slots = p.slots;
  g.dh_acc = ws.dh;
  g.dh_slot_size = p.t_pad * p.dh_ld;
  g.dh_ld = p.dh_ld;
  g.dw_bf16 = 1;
  g.label_rows = ws.label_rows;
  g.label_span = ws.sort.span;
  g.do_dh = d_hidden != nullptr;
  CUtensorMap wc;
  if ((st = xent_dw_out(&wc, ek, &g, d_weight, vocab, dim, ws.dwp, p.ldd)) != ETHOS_OK) return st;
  if ((st = launch_xent<XE_GRADS, 1>(ek, wk, em, hb, wc, g, xent_grad_units(p, vocab, p.slots, g), dev_err, sm,
                                     *dev)) != ETHOS_OK)
    return st;
  if (d_weight && p.pad_dw && (st = xent_unpad(ws.dwp, p.ldd, vocab, dim, d_weight, sm, *dev)) != ETHOS_OK) return st;
  if (!d_hidden) return ETHOS_OK;
  return xent_dhidden<__nv_bfloat16>(p, sv, ws.dh, p.slots, nullptr, reduction, sv.rw.r, sv.rw.q, weight, ldw,
                                     d_hidden, sm, *dev);
}

int ethos_xent_scale(const float* factor, void* x, int64_t nx, void* y, int64_t ny, int dtype, void* stream) {
  if (nx < 0 || ny < 0 || !known_dtype(dtype)) return ETHOS_ERR_INVALID_ARG;
  if (nx + ny == 0) return ETHOS_OK;
  if (!factor || (nx > 0 && !x) || (ny > 0 && !y)) return ETHOS_ERR_INVALID_ARG;
  DeviceInfo* dev = nullptr;
  const int st = base_device_info(&dev);
  if (st != ETHOS_OK) return st;
  int64_t blocks = ((nx + ny) / 8 + 256) / 256;
  if (blocks > 8ll * dev->sm_count) blocks = 8ll * dev->sm_count;
  const dim3 grid(static_cast<unsigned>(blocks));
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  return dtype == ETHOS_BF16 ? launch_pdl(k_xent_scale<__nv_bfloat16>, grid, dim3(256), 0, sm, factor,
                                          static_cast<__nv_bfloat16*>(x), nx, static_cast<__nv_bfloat16*>(y), ny)
                             : launch_pdl(k_xent_scale<float>, grid, dim3(256), 0, sm, factor,
                                          static_cast<float*>(x), nx, static_cast<float*>(y), ny);
}

int ethos_xent_backward(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, int dtype, int reduction,
                        int64_t tokens, int64_t vocab, int64_t dim, const float* grad, const void* save,
                        size_t save_bytes, void* d_hidden, void* d_weight, void* workspace, size_t workspace_bytes,
                        int* dev_err, void* stream) {
  int st = xent_check(tokens, vocab, dim, ldh, ldw, dtype, reduction);
  if (st != ETHOS_OK) return st;
  if (!hidden || !weight || !grad || !dev_err) return ETHOS_ERR_INVALID_ARG;
  const XentPlan p = xent_plan(tokens, vocab, dim, dtype);
  Carve cs{static_cast<char*>(const_cast<void*>(save)), 0, save_bytes},
      cw{static_cast<char*>(workspace), 0, workspace_bytes};
  XentSave sv;
  XentBwd ws;
  carve_save(cs, p, &sv);
  carve_xent_bwd(cw, p, &ws);
  if (!save || !workspace || cs.off > save_bytes || cw.off > workspace_bytes) return ETHOS_ERR_WORKSPACE;
  if (!aligned16(save) || !aligned16(workspace)) return ETHOS_ERR_ALIGNMENT;
  if (!p.pack_w && (ldw % 8 != 0 || !aligned16(weight))) return ETHOS_ERR_ALIGNMENT;
  if (!d_hidden && !d_weight) return ETHOS_OK;
  DeviceInfo* dev = nullptr;
  if ((st = base_device_info(&dev)) != ETHOS_OK) return st;
  cudaStream_t sm = static_cast<cudaStream_t>(stream);
  // the forward of few tokens has not packed them
  if (xent_is_few(p) && (st = xent_rows_pass(p, sv, hidden, ldh, weight, ldw, dtype, sm, *dev)) != ETHOS_OK) return st;
  if (p.pack_w && (st = xent_pack_w(p, dtype, weight, ldw, ws.wp, sm, *dev)) != ETHOS_OK) return st;
  const int T = static_cast<int>(tokens), D = static_cast<int>(dim);
  const int64_t num_m = p.t_pad / XE_TILE;
  const int esz = dtype == ETHOS_BF16 ? 2 : 4;
  CUtensorMap ha, hb;  // rows of hidden, K-major (A of the logits) and MN-major (B of dW)
  if ((st = make_tmap_bf16(&ha, sv.hp, p.planes * p.t_pad, p.ldd, G2_BM, p.ldd)) != ETHOS_OK) return st;
  if ((st = make_tmap_bf16(&hb, sv.hp, p.planes * p.t_pad, p.ldd, G2_BK, p.ldd)) != ETHOS_OK) return st;
  for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
    const int64_t n = vocab - v0 < p.piece ? vocab - v0 : p.piece;
    const void* wptr = p.pack_w ? static_cast<const void*>(ws.wp + v0 * p.ldd)
                                : static_cast<const void*>(static_cast<const __nv_bfloat16*>(weight) + v0 * ldw);
    const int64_t wrows = p.pack_w ? p.planes * p.v_pad - v0 : n;
    const int64_t wcols = p.pack_w ? p.ldd : dim, wld = p.pack_w ? p.ldd : ldw;
    CUtensorMap wb, wk, dk, dm;
    if ((st = make_tmap_bf16(&wb, wptr, wrows, wcols, G2_BM, wld)) != ETHOS_OK) return st;
    if ((st = make_tmap_bf16(&wk, wptr, wrows, wcols, G2_BK, wld)) != ETHOS_OK) return st;
    if ((st = make_tmap_bf16(&dk, ws.dl, p.planes * p.t_pad, p.piece, G2_BM, p.piece)) != ETHOS_OK) return st;
    if ((st = make_tmap_bf16(&dm, ws.dl, p.planes * p.t_pad, p.piece, G2_BK, p.piece)) != ETHOS_OK) return st;
    XeArgs a = {};
    a.rw = sv.rw;
    a.p[0] = XeProduct{static_cast<int>(p.t_pad), static_cast<int>(p.v_pad), T, static_cast<int>(n), D};
    a.v0 = static_cast<int>(v0);
    a.grad = grad;
    a.reduction = reduction;
    a.dl = ws.dl;
    a.dl_plane_rows = p.t_pad;
    a.ldl = p.piece;
    a.label_grad = v0 == 0 ? ws.label_grad : nullptr;
    CUtensorMap dc;
    if ((st = make_tmap_bf16(&dc, ws.dl, p.planes * p.t_pad, p.piece, 32, p.piece)) != ETHOS_OK) return st;
    if ((st = launch_xent_planes<XE_DLOGITS>(p.planes, ha, wb, ha, wb, dc, a, num_m * ((n + p.tile_n - 1) / p.tile_n),
                                             dev_err, sm, *dev)) != ETHOS_OK)
      return st;
    if (v0 == 0 && d_weight && p.planes == 1 &&
        (st = xent_label_rows(p, sv, ws.sort, ws.label_grad, ws.label_rows, dev_err, sm, *dev)) != ETHOS_OK)
      return st;
    XeArgs g = {};
    g.rw = sv.rw;
    g.grad = grad;
    g.reduction = reduction;
    g.p[0] = XeProduct{static_cast<int>(p.t_pad), static_cast<int>(p.v_pad), T, D, static_cast<int>(n)};
    g.p[1] = XeProduct{static_cast<int>(p.t_pad), static_cast<int>(p.t_pad), static_cast<int>(n), D, T};
    g.dh_slots = p.slots_piece;
    g.dh_accumulate = v0 > 0;
    g.dh_acc = ws.dh;
    g.dh_slot_size = p.t_pad * p.dh_ld;
    g.dh_ld = p.dh_ld;
    void* dw = d_weight ? static_cast<char*>(d_weight) + v0 * dim * esz : nullptr;
    g.dw_bf16 = dtype == ETHOS_BF16;
    g.label_rows = ws.label_rows;
    g.label_span = p.planes == 1 ? ws.sort.span + v0 : nullptr;
    g.do_dh = d_hidden != nullptr;
    CUtensorMap wc;
    if ((st = xent_dw_out(&wc, dk, &g, dw, n, dim, ws.dwp, p.ldd)) != ETHOS_OK) return st;
    const int64_t units = xent_grad_units(p, n, p.slots_piece, g);
    if ((st = launch_xent_planes<XE_GRADS>(p.planes, dk, wk, dm, hb, wc, g, units, dev_err, sm, *dev)) != ETHOS_OK)
      return st;
    if (d_weight && p.pad_dw && (st = xent_unpad(ws.dwp, p.ldd, n, dim, dw, sm, *dev)) != ETHOS_OK) return st;
  }
  if (!d_hidden) return ETHOS_OK;
  return dtype == ETHOS_BF16 ? xent_dhidden<__nv_bfloat16>(p, sv, ws.dh, p.slots_piece, grad, reduction, nullptr,
                                                           ws.label_grad, weight, ldw, d_hidden, sm, *dev)
                             : xent_dhidden<float>(p, sv, ws.dh, p.slots_piece, grad, reduction, nullptr, nullptr,
                                                   weight, ldw, d_hidden, sm, *dev);
}

}  // extern "C"
