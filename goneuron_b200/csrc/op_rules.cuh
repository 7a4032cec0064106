// op_rules.cuh -- operators on device memory: what a call's arguments must be, and how its work is cut.  Plain C++ (tested on the CPU).
// The checks return null, or what is wrong.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <initializer_list>

#include "../../include/goneuron_cuda.h"

namespace gn {

constexpr int64_t OP_MAX_ROWS = 0x7fffffff;                          // tokens, rows, vocabulary
inline int dtype_size(int dtype) { return dtype == GN_F32 ? 4 : dtype == GN_F16 || dtype == GN_BF16 ? 2 : 0; }
inline bool aligned_to(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }
inline const char* check_dtype(int dtype, const void* p) {
  if (!dtype_size(dtype)) return "dtype is none of GN_F32, GN_F16, GN_BF16";
  return aligned_to(p, dtype_size(dtype)) ? nullptr : "a pointer is not aligned to its type";
}
inline const char* check_index(int index_type, const void* p) {
  if (index_type != GN_I32 && index_type != GN_I64) return "index_type is neither GN_I32 nor GN_I64";
  return aligned_to(p, index_type == GN_I64 ? 8 : 4) ? nullptr : "an index pointer is not aligned to its type";
}

// ------------------------------------------------------------------ norm of queries and keys with the rotation
struct QkArgs {
  int dtype; int64_t tokens; int head_size, rotated; float eps; const gn_heads *q, *k; const float *gain_q, *gain_k;
  const void* positions; int index_type; const double* frequencies;
};
inline const char* check_heads(const QkArgs& a, const gn_heads* h, int heads, bool written) {
  if (!h || h->heads != heads) return "tensors of the same heads are needed for every input and output";
  if (a.tokens && heads && !h->data) return "a data pointer is null";
  if (const char* e = check_dtype(a.dtype, h->data)) return e;
  if (h->token_stride < 0 || h->head_stride < 0) return "a stride is negative";
  if (written) {                                                     // rows lie side by side within the smaller stride, and all of those within the larger one
    const bool many_t = a.tokens > 1, many_h = heads > 1;
    if ((many_t && h->token_stride < a.head_size) || (many_h && h->head_stride < a.head_size)) return "an output's rows overlap";
    if (many_t && many_h) {
      const bool tokens_inside = h->token_stride < h->head_stride;
      const int64_t inner = tokens_inside ? h->token_stride : h->head_stride, n = tokens_inside ? a.tokens : heads, outer = tokens_inside ? h->head_stride : h->token_stride;
      if ((outer - a.head_size) / inner < n - 1) return "an output's rows overlap";
    }
  }
  return nullptr;
}
inline const char* check_qk(const QkArgs& a) {
  if (!dtype_size(a.dtype)) return "dtype is none of GN_F32, GN_F16, GN_BF16";
  if (a.tokens < 0 || a.tokens > OP_MAX_ROWS) return "tokens out of range";
  if (a.head_size < 1 || a.head_size > 1024) return "head_size is not in [1, 1024]";
  if (a.rotated < 0 || a.rotated > a.head_size || a.rotated % 2) return "rotated is not an even number of at most head_size elements";
  if (!(a.eps >= 0.f) || std::isinf(a.eps)) return "eps is negative or not finite";
  if (!a.q) return "q is null";
  if (a.q->heads < 0 || a.q->heads > 65536 || (a.k && (a.k->heads < 0 || a.k->heads > 65536))) return "the number of heads is not in [0, 65536]";
  if (!aligned_to(a.gain_q, 4) || !aligned_to(a.gain_k, 4) || !aligned_to(a.frequencies, 8)) return "a pointer is not aligned to its type";
  if (a.rotated && a.tokens && (!a.positions || !a.frequencies)) return "positions and frequencies are needed for a rotation";
  if (a.rotated) if (const char* e = check_index(a.index_type, a.positions)) return e;
  if (const char* e = check_heads(a, a.q, a.q->heads, false)) return e;
  return a.k ? check_heads(a, a.k, a.k->heads, false) : nullptr;
}
// In place, a row has to be written where it was read.
inline const char* check_in_place(const gn_heads* in, const gn_heads* out) {
  return in && out && in->data && in->data == out->data && (in->token_stride != out->token_stride || in->head_stride != out->head_stride) ? "in place, both tensors' strides have to be the same" : nullptr;
}
// A tensor that is written may be its own input, but not the other one's, nor the other one that is written: blocks of queries and of keys do not wait for each other.
inline const char* check_apart(const gn_heads* written, const gn_heads* other) {
  return written && other && written->data && written->data == other->data && written->heads && other->heads ? "an output of the queries lies on a tensor of the keys, or the other way round" : nullptr;
}
// Groups of lanes: a lane has two pieces of a row, 16 bytes each, or 8 where 16 do not fit and the type has 16 bits; a row's lanes are neighbours, 2 to 32 of them.  0: the
// pieces do not fit (sizes, strides or pointers, pairs that end inside one, rows of more than 64 pieces); a row that neither fits goes element by element.
inline int qk_group(int dtype, int head_size, int rotated, bool interleaved, const gn_heads* const* t, int n, int piece = 16) {
  const int vec = piece / dtype_size(dtype), pieces = head_size / vec;
  if (head_size % vec || pieces > 64 || (!interleaved && rotated % (2 * vec))) return 0;
  for (int i = 0; i < n; i++)
    if (t[i] && (!aligned_to(t[i]->data, piece) || t[i]->token_stride % vec || t[i]->head_stride % vec)) return 0;
  int g = 2;
  while (2 * g < pieces) g *= 2;
  return g;
}
// Work of the queries and of the keys goes to blocks of their own.  A block takes as many tokens at a time as its groups of lanes fill, where that leaves work for all blocks, and at most
// 32 KB of cosines and sines.
constexpr int QK_ROW_WARPS = 16;                                      // of a block that goes element by element, a row each
constexpr int QK_PER_SM = 2, QK_HEADS_FWD = 4, QK_HEADS_BWD = 2;     // heads of a token that a group of lanes takes at a time
inline int qk_tokens(int64_t tokens, int sms, int group, int heads, int heads_at_a_time, int rotated) {
  const int64_t per_token = group ? std::max<int64_t>(1, ceil_div(heads, heads_at_a_time)) : heads, groups = group ? 256 / group : QK_ROW_WARPS;
  int64_t n = std::max<int64_t>(1, groups / std::max<int64_t>(1, per_token));
  n = std::min(n, std::max<int64_t>(1, ceil_div(tokens, (int64_t)sms * QK_PER_SM)));
  return (int)std::min<int64_t>(n, rotated ? std::max(1, 8192 / rotated) : 256);
}
// Shared memory of a block that goes element by element, at most: cosines and sines, frequencies, a row of sums for every warp.
constexpr int QK_ROWS_SMEM_MOST = (8192 + 1024 + QK_ROW_WARPS * 1024) * 4;
// All blocks are resident at once, so that a gradient leaves no more partial sums than those.
inline int64_t qk_blocks(int64_t tokens, int sms, int tokens_at_a_time) { return std::max<int64_t>(1, std::min<int64_t>(ceil_div(tokens, tokens_at_a_time), (int64_t)sms * QK_PER_SM)); }
inline int64_t qk_workspace(int64_t tokens, int head_size, int sms) { return qk_blocks(tokens, sms, 1) * 2 * head_size * 4; }

// ------------------------------------------------------------------ distillation
constexpr int DISTILL_THREADS = 480, DISTILL_PART = 104 * 1024, DISTILL_PART_MOST = 176 * 1024;
// Beside its part of a row a block has the teacher's entries in shared memory: three rows of them, what one row needs while it is worked on, and a table of ids.
constexpr int DISTILL_TOP = 1024, TEACHER_TABLE = 2048;
constexpr int teacher_smem(int top) { return (top + 15) / 16 * 16 * 40 + 2 * TEACHER_TABLE; }
constexpr int DISTILL_SMEM_MOST = DISTILL_PART_MOST + teacher_smem(DISTILL_TOP);
inline const char* check_distill(int dtype, int64_t rows, int64_t vocab, int top, float temperature, const void* logits, int64_t row_stride, const void* top_ids, int index_type,
                                 const float* top_logits, const float* weight, const float* loss, const void* dlogits, int64_t drow_stride) {
  if (rows < 0 || rows > OP_MAX_ROWS) return "rows out of range";
  if (vocab < 1 || vocab > OP_MAX_ROWS) return "vocab out of range";
  if (top < 0 || top > DISTILL_TOP) return "top is not in [0, 1024]";
  if (!(temperature > 0.f) || std::isinf(temperature)) return "temperature is not positive and finite";
  if (rows && (!logits || !loss || (top && (!top_ids || !top_logits)))) return "a data pointer is null";
  if (const char* e = check_dtype(dtype, logits)) return e;
  if (const char* e = check_dtype(dtype, dlogits)) return e;
  if (const char* e = check_index(index_type, top_ids)) return e;
  if (!aligned_to(top_logits, 4) || !aligned_to(weight, 4) || !aligned_to(loss, 4)) return "a pointer is not aligned to its type";
  if (row_stride < 0 || (rows > 1 && dlogits && drow_stride < vocab)) return "rows overlap, or a stride is negative";
  if (dlogits && dlogits == logits && rows > 1 && row_stride != drow_stride) return "in place, both strides have to be the same";
  if (dlogits && dlogits != logits && (rows == 1 || row_stride == drow_stride)) {      // rows of one may lie partly on rows of the other: those nearest to each other, t rows apart
    const int64_t d = (int64_t)(reinterpret_cast<intptr_t>(dlogits) - reinterpret_cast<intptr_t>(logits)) / dtype_size(dtype), down = rows == 1 ? 0 : d / row_stride;
    for (int64_t t = down - 1; t <= down + 1; t++)
      if (std::llabs(t) < rows && std::llabs(d - t * row_stride) < vocab) return "dlogits lies partly on logits";
  }
  return nullptr;
}
// Beside dynamic shared memory a block takes up to 2 KB of its own and 1 KB that is set apart; a multiprocessor has 228 KB.
constexpr int DISTILL_FIXED = 3 * 1024, DISTILL_SM_SMEM = 228 * 1024;
// A row is kept in the shared memory of `cluster` blocks, `per` 16-byte pieces in each, some eight of them a thread.  cluster 0: it does not fit and is read again instead.  Parts of up to 104 KB, less where
// the teacher has more than 64 entries, leave room for two blocks on a multiprocessor, which overlap each other's phases (4096 rows of 50257, bf16, 256 entries: one block a row and multiprocessor 682 us, two
// blocks a row 564; 53000 with 64 entries, two blocks a multiprocessor instead of one: 238 and 191); a cluster's barrier costs more than that gives, so that four and eight blocks are taken only where two cannot
// hold the row (515 rows of 100003, f16: one block 66 us, two 61, four 80; 2000 rows of 130000, bf16: two 291, four 330), and four again only where their parts leave room for two on a multiprocessor
// (512 rows of 128000, f32: four 216 us, eight 166; of 250000, bf16: 256 and 180).  Few rows are cut further, so that they fill the multiprocessors, down to two
// thousand elements per block.
struct DistillPlan { int cluster, threads, per; };
inline DistillPlan distill_plan(int64_t rows, int64_t vocab, int size, int sms, int top = 0) {
  const int64_t part = std::min(DISTILL_PART, DISTILL_SM_SMEM / 2 - DISTILL_FIXED - teacher_smem(top));
  const int64_t v = 16 / size, pieces = ceil_div(vocab + v - 1, v);  // (a row may begin inside a piece)
  int c = 1;
  while (c < 8 && ceil_div(pieces, c) * 16 > (c == 2 ? DISTILL_PART_MOST : part)) c *= 2;
  if (ceil_div(pieces, c) * 16 > DISTILL_PART_MOST) return {0, 1024, 0};
  while (c < 8 && rows * c * 2 <= sms && vocab >= 4096L * c) c *= 2;
  const int64_t per = ceil_div(pieces, c);
  return {c, (int)std::min<int64_t>(DISTILL_THREADS, std::max<int64_t>(64, round_up(ceil_div(per, 8), 32))), (int)per};
}

// ------------------------------------------------------------------ embedding
inline const char* check_embedding(int dtype, int64_t tokens, int64_t vocab, int dim, float scale, const void* rows_in, int64_t in_stride, int64_t in_rows, const void* ids, int index_type,
                                   const void* out, int64_t out_stride, int64_t out_rows) {
  if (tokens < 0 || tokens > OP_MAX_ROWS) return "tokens out of range";
  if (vocab < 1 || vocab >= OP_MAX_ROWS) return "vocab out of range";
  if (dim < 1) return "dim out of range";
  if (!(std::fabs(scale) <= 3.4028235e38f)) return "scale is not finite";
  if ((in_rows && !rows_in) || (tokens && !ids) || (out_rows && !out)) return "a data pointer is null";
  if (const char* e = check_dtype(dtype, rows_in)) return e;
  if (const char* e = check_index(index_type, ids)) return e;
  if (in_stride < 0 || (out_rows > 1 && out_stride < dim)) return "rows overlap, or a stride is negative";
  return nullptr;
}
// The tokens' order by id, then sums of it in pieces of `chunk` neighbouring places.  Up to SORT_SMALL tokens places are counted directly, with the
// square of the tokens' number; above, passes of 8 bits over tiles of SORT_TILE tokens (gradient of 300 elements and 5000 ids, f32: counted, 17 us for
// 4500 tokens, 22 for 6000, 30 for 8192; in passes 29 for 8192).
constexpr int SORT_SMALL = 7168, SORT_TILE = 2048, SORT_BITS = 8, SORT_SCAN_TILES = 128;      // SCAN_TILES: up to so many tiles add up the others' counts themselves
struct EmbeddingPlan {
  bool small; int bits, passes, chunk; int64_t tiles, chunks;
  int64_t keys, order, keys2, order2, hist, partial, bytes;          // places in the workspace, in bytes
};
inline EmbeddingPlan embedding_plan(int64_t tokens, int64_t vocab, int dim, int sms) {
  EmbeddingPlan p{};
  p.small = tokens <= SORT_SMALL;
  p.bits = 1;
  while (((int64_t)1 << p.bits) <= vocab) p.bits++;                  // keys 0 .. vocab (padding)
  p.passes = (int)ceil_div(p.bits, SORT_BITS);
  p.chunk = 4;                                                       // places of a piece: some eight pieces for each multiprocessor, 64 at most
  while (p.chunk < 64 && tokens > (int64_t)p.chunk * 8 * sms) p.chunk *= 2;
  p.tiles = ceil_div(tokens, SORT_TILE); p.chunks = ceil_div(tokens, p.chunk);
  int64_t at = 0; auto take = [&](int64_t bytes) { const int64_t a = at; at += round_up(bytes, 256); return a; };
  p.keys = take(4 * tokens); p.order = take(4 * tokens);
  p.keys2 = take(p.small ? 0 : 4 * tokens); p.order2 = take(p.small ? 0 : 4 * tokens);
  p.hist = take(p.small ? 0 : 4 * (p.tiles << SORT_BITS));
  p.partial = take(p.chunks * 2 * (int64_t)dim * 4);                 // a piece's first and last sum may go on in its neighbours
  p.bytes = at; return p;
}

// ------------------------------------------------------------------ gated feed-forward block
inline const char* check_ffn_sizes(int64_t tokens, int dim, int ff) {
  if (tokens < 0 || tokens > OP_MAX_ROWS - 1024) return "tokens out of range";
  if (dim < 8 || ff < 8 || dim % 8 || ff % 8 || dim > (1 << 24) || ff > (1 << 24)) return "dim and ff have to be multiples of 8, at most 2^24";
  return nullptr;
}
inline const char* check_ffn_strides(int64_t tokens, int dim, std::initializer_list<int64_t> strides) {
  if (tokens > 1) for (int64_t s : strides) if (s < dim || s % 8 || s >= (1LL << 38)) return "a row stride is below dim, no multiple of 8 or too large";
  return nullptr;
}
inline const char* check_ffn(int dtype, int activation, int64_t tokens, int dim, int ff, std::initializer_list<const void*> pointers, std::initializer_list<int64_t> strides) {
  if (dtype != GN_F16 && dtype != GN_BF16) return "dtype is neither GN_F16 nor GN_BF16";
  if (activation != GN_ACT_SILU && activation != GN_ACT_GELU && activation != GN_ACT_RELU) return "activation is none of GN_ACT_SILU, GN_ACT_GELU, GN_ACT_RELU";
  if (const char* e = check_ffn_sizes(tokens, dim, ff)) return e;
  for (const void* p : pointers) {
    if (tokens && !p) return "a data pointer is null";
    if (!aligned_to(p, 16)) return "a pointer is not 16-byte aligned";
  }
  return check_ffn_strides(tokens, dim, strides);
}
// Pairs of blocks that share a tile of 256 rows.
inline int ffn_pairs(int sms) { return std::max(1, sms / 2); }
// Width of the output tiles (256 x bn) and slices of the contraction of a plain product.
struct FfnCut { int bn, splits; };
// Left-over tiles of a last round that would keep at most half of the pairs busy: they run as two halves each.
inline int64_t ffn_tail(int64_t items, int pairs) { const int64_t left = items % pairs; return items > pairs && 2 * left <= pairs ? left : 0; }
// The cheapest cut by a count of tensor-core cycles: a block of 64 indices takes 540 in a tile 256 wide and 400 in one 128 wide (256 of arithmetic; shared memory bounds it), a tile 4000
// around its main loop in the first round; slices cost a launch (4000) and the float32 partial sums' way to memory and back.
struct FfnShape { int64_t M, N; };
inline FfnCut ffn_cut(std::initializer_list<FfnShape> shapes, int64_t kb, int sms) {
  FfnCut best{256, 1}; double least = 1e300; const int pairs = ffn_pairs(sms);
  for (int bn : {256, 128}) {
    int64_t tiles = 0;
    for (const FfnShape& s : shapes) tiles += ceil_div(s.M, 256) * ceil_div(s.N, bn);
    for (int splits = 1; splits <= 32 && splits <= kb; splits++) {
      if (splits > 1 && (tiles * splits > 4 * pairs || kb / splits < 2)) break;
      const int64_t items = tiles * splits; double rounds = (double)ceil_div(items, pairs);
      if (splits == 1 && bn == 256 && ffn_tail(items, pairs)) rounds -= 0.4;
      double cost = rounds * (double)ceil_div(kb, splits) * (bn == 256 ? 540 : 400) + 4000;
      if (splits > 1) cost += 4000 + (double)items * 256 * bn * 8 / (2500.0 * sms / 148);      // 4 bytes written, 4 read; some 2500 bytes a cycle
      if (cost < least) { least = cost; best = FfnCut{bn, splits}; }
    }
  }
  return best;
}
inline int64_t ffn_partial(std::initializer_list<FfnShape> shapes, const FfnCut& c) {
  int64_t tiles = 0;
  for (const FfnShape& s : shapes) tiles += ceil_div(s.M, 256) * ceil_div(s.N, c.bn);
  return c.splits > 1 ? tiles * c.splits * 256 * c.bn * 4 : 0;
}
constexpr int FFN_FEW_TOKENS = 16;                                   // up to so many, without a gradient, go through kernels of their own, up to half of that in blocks of eight
// Places, in bytes, in what the forward pass saves (g and u in blocks of 32 x 16, 24 bits each, then h) and in the workspaces.
struct FfnPlan { FfnCut y, dx, dw; int64_t saved_h, saved, fwd_h, fwd_partial, fwd, bwd_dg, bwd_du, bwd_partial, bwd; };
inline FfnPlan ffn_make_plan(int64_t M, int64_t D, int64_t F, int sms) {
  FfnPlan p{};
  const int64_t kf = ceil_div(F, 64), h = round_up(2 * M * F, 256);
  p.y = ffn_cut({{M, D}}, kf, sms); p.dx = ffn_cut({{M, D}}, 2 * kf, sms); p.dw = ffn_cut({{F, D}, {F, D}, {D, F}}, std::max<int64_t>(1, ceil_div(M, 64)), sms);
  p.saved_h = ceil_div(M, 32) * ceil_div(F, 16) * (32 * 16 * 6); p.saved = p.saved_h + h;
  p.fwd_h = 0; p.fwd_partial = M <= FFN_FEW_TOKENS / 2 ? round_up(4 * M * F, 256) : h; p.fwd = p.fwd_partial + ffn_partial({{M, D}}, p.y);      // (few tokens: two planes)
  p.bwd_dg = 0; p.bwd_du = h; p.bwd_partial = 2 * h; p.bwd = 2 * h + std::max(ffn_partial({{M, D}}, p.dx), ffn_partial({{F, D}, {F, D}, {D, F}}, p.dw));
  return p;
}
// The last sizes' plan is kept by the thread: a call asks for it up to three times, and some hundred cuts are compared for it.
inline const FfnPlan& ffn_plan(int64_t M, int64_t D, int64_t F, int sms) {
  thread_local int64_t m = -1, d = -1, f = -1, s = -1; thread_local FfnPlan p;
  if (m != M || d != D || f != F || s != sms) { p = ffn_make_plan(M, D, F, sms); m = M; d = D; f = F; s = sms; }
  return p;
}
// Few tokens: blocks of a cluster that share the contraction of 16 rows, until there are blocks for every multiprocessor.
inline int ffn_few_cluster(int64_t N, int64_t K, int sms) {
  int c = 1;
  while (c < 8 && ceil_div(N, 16) * c < sms && K >= 512L * c) c *= 2;
  return c;
}

}  // namespace gn
