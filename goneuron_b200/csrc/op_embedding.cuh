// op_embedding.cuh -- embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale table[id_i],      dtable[v] = scale sum over i with id_i = v of dout[i]
//
// The gradient sorts the tokens' places by id (stable: equal ids keep their order), cuts the sorted list into pieces of `chunk` neighbouring places, whatever ids
// they hold, and lets a block sum each piece run by run.  Frequent tokens are thereby spread over many blocks and rare ones share one.  A run that lies within its
// piece is written where it belongs; a run that crosses pieces leaves its parts in the workspace and a second launch adds them in order.  Rows that no token names
// are zeroed by blocks of the same launch.  No atomics on values: the order of every sum follows from the sizes.
#pragma once
#include "device_ops.cuh"

namespace gn {

// ------------------------------------------------------------------ lookup
// A warp per token.  V: elements of an access (16 bytes, or one where sizes, strides or pointers do not allow that).
template <class T, int V>
__global__ void __launch_bounds__(256) embedding_kernel(const T* table, long table_stride, const void* ids, int index_type, long tokens, long vocab, int dim, float scale,
                                                        T* out, long out_stride) {
  op_begin();
  const int lane = threadIdx.x & 31; const long warps = (long)gridDim.x * 8;
  for (long i = (long)blockIdx.x * 8 + (threadIdx.x >> 5); i < tokens; i += warps) {
    const int64_t id = load_index(ids, index_type, i); const bool there = id >= 0 && id < vocab;
    if (!there && id != -1 && lane == 0) op_report(OP_BAD_INDEX);
    const T* src = table + (there ? id : 0) * table_stride; T* dst = out + i * out_stride;
    if constexpr (V == 1) {
      for (int e = lane; e < dim; e += 32) dst[e] = there ? from_f32<T>(to_f32(src[e]) * scale) : from_f32<T>(0.f);
    } else {
      constexpr int U = 4;                                           // four accesses of a lane under way
      const int n = dim / V;
      for (int e0 = lane; e0 < n; e0 += 32 * U) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; j++) { u[j] = make_uint4(0, 0, 0, 0); if (there && e0 + 32 * j < n) u[j] = ld(reinterpret_cast<const uint4*>(src) + e0 + 32 * j); }
#pragma unroll
        for (int j = 0; j < U; j++) {
          float v[Vec<T>::N]; unpack<T>(u[j], v);
#pragma unroll
          for (int k = 0; k < Vec<T>::N; k++) v[k] = there ? v[k] * scale : 0.f;
          if (e0 + 32 * j < n) __stcs(reinterpret_cast<uint4*>(dst) + e0 + 32 * j, pack<T>(v));      // (the table's rows are read again, these are not)
        }
      }
    }
  }
}

// ------------------------------------------------------------------ order of the tokens by id
// Key of a token: its id, or `vocab` (behind every row) for padding.
__device__ __forceinline__ unsigned token_key(const void* ids, int index_type, long i, long vocab) {
  const int64_t id = load_index(ids, index_type, i);
  if (id >= 0 && id < vocab) return (unsigned)id;
  if (id != -1) op_report(OP_BAD_INDEX);
  return (unsigned)vocab;
}
// One pass of a stable sort over one tile of shared counters: `cnt` is [warps][256].  Every warp owns a run of neighbouring places, `per` rows of 32.  First each warp
// counts its digits, then a digit's counts become the places where the warps' own begin, then every warp walks its rows again.
struct TileDigit {
  // places of the 32 lanes' digits among equal ones of the warp's earlier rows (in `c`) and lower lanes; moves the counters on
  static __device__ __forceinline__ unsigned place(unsigned* c, unsigned digit, bool on, int lane) {
    const unsigned same = __match_any_sync(0xffffffffu, on ? digit : 256u + lane);
    const unsigned before = __popc(same & ((1u << lane) - 1));
    unsigned at = 0;
    if (on) at = c[digit] + before;
    __syncwarp();
    if (on && before == 0) c[digit] += __popc(same);
    __syncwarp();
    return at;
  }
};

// Few tokens: a token's place is the number of keys below its own, and of equal ones before it.  A warp counts for four neighbouring tokens at a time, all keys in every block's shared memory: 9
// million comparisons for 3001 tokens, spread over all multiprocessors.  (One block that sorted them in shared memory took 10 us.)
constexpr int RANK_THREADS = 1024, RANK_TOKENS = 4;
__global__ void __launch_bounds__(RANK_THREADS) sort_rank_kernel(const void* ids, int index_type, int tokens, long vocab, unsigned* keys, int* order) {
  op_begin();
  __shared__ __align__(16) unsigned all[SORT_SMALL];
  const int lane = threadIdx.x & 31, padded = (tokens + 127) & ~127;
  for (int i = threadIdx.x; i < padded; i += RANK_THREADS) all[i] = i < tokens ? token_key(ids, index_type, i, vocab) : 0xffffffffu;
  __syncthreads();
  for (int i = ((threadIdx.x >> 5) * gridDim.x + blockIdx.x) * RANK_TOKENS; i < tokens; i += gridDim.x * (RANK_THREADS / 32) * RANK_TOKENS) {
    const uint4 own = *reinterpret_cast<const uint4*>(all + i); const unsigned key[RANK_TOKENS] = {own.x, own.y, own.z, own.w};
    int n[RANK_TOKENS] = {};
#pragma unroll 2
    for (int j = lane * 4; j < padded; j += 128) {
      const uint4 k = *reinterpret_cast<const uint4*>(all + j); const unsigned before = j < i;      // (four keys all before the four tokens, all behind them or they themselves; keys are below 2^31)
#pragma unroll
      for (int t = 0; t < RANK_TOKENS; t++) { const unsigned to = key[t] + before; n[t] += (k.x < to) + (k.y < to) + (k.z < to) + (k.w < to); }
    }
#pragma unroll
    for (int t = 0; t < RANK_TOKENS; t++) {
      n[t] = __reduce_add_sync(0xffffffffu, n[t]);
#pragma unroll
      for (int e = 0; e < t; e++) n[t] += key[e] == key[t];
      if (lane == t && i + t < tokens) { keys[n[t]] = key[t]; order[n[t]] = i + t; }
    }
  }
}

// Many tokens: per pass the digits of every tile are counted, the counts of all tiles become places (digit by digit, within a digit tile by tile), and every tile
// moves its tokens there.  FIRST: keys come from the ids and places are the tokens' own.
constexpr int SORT_THREADS = 256;
template <bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const void* ids, int index_type, const unsigned* keys, long tokens, long vocab, int shift, bool by_tile, unsigned* hist) {
  op_begin();
  __shared__ unsigned cnt[256];
  cnt[threadIdx.x] = 0;
  __syncthreads();
  const long base = (long)blockIdx.x * SORT_TILE;
#pragma unroll
  for (int j = 0; j < SORT_TILE / SORT_THREADS; j++) {
    const long i = base + j * SORT_THREADS + threadIdx.x;
    if (i < tokens) atomicAdd(&cnt[((FIRST ? token_key(ids, index_type, i, vocab) : ld(keys + i)) >> shift) & 255], 1u);
  }
  __syncthreads();
  hist[by_tile ? blockIdx.x * 256L + threadIdx.x : (long)threadIdx.x * gridDim.x + blockIdx.x] = cnt[threadIdx.x];      // digit by digit for the scan
}
// In place: every count becomes the sum of those before it.  One block.
__global__ void __launch_bounds__(1024) sort_scan_kernel(unsigned* hist, long n) {
  op_begin();
  __shared__ unsigned sums[32];
  __shared__ unsigned carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (long base = 0; base < n; base += 4096) {                      // (n is a multiple of 256)
    const long i = base + 4L * threadIdx.x; const bool on = i < n;
    const uint4 u = on ? *reinterpret_cast<const uint4*>(hist + i) : make_uint4(0, 0, 0, 0);
    const unsigned own = u.x + u.y + u.z + u.w; unsigned s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned v = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += v; }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    unsigned before = carry, total = 0;
    { const unsigned v = sums[lane]; unsigned a = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const unsigned t = __shfl_up_sync(0xffffffffu, a, o); if (lane >= o) a += t; }
      total = __shfl_sync(0xffffffffu, a, 31); before += __shfl_sync(0xffffffffu, a - v, warp); }
    unsigned at = before + s - own;
    if (on) *reinterpret_cast<uint4*>(hist + i) = make_uint4(at, at + u.x, at + u.x + u.y, at + u.x + u.y + u.z);
    __syncthreads();
    if (threadIdx.x == 0) carry += total;
    __syncthreads();
  }
}
// SCAN: the counts are as sort_count_kernel left them, and every tile adds up what lies before its own (few tiles: a launch less a pass).
template <bool FIRST, bool SCAN>
__global__ void __launch_bounds__(SORT_THREADS) sort_move_kernel(const void* ids, int index_type, const unsigned* keys, const int* order, long tokens, long vocab, int shift,
                                                                 const unsigned* hist, unsigned* keys_out, int* order_out) {
  constexpr int W = SORT_THREADS / 32, PER = SORT_TILE / SORT_THREADS;      // rows of 32 places of a warp
  op_begin();
  __shared__ unsigned cnt[W * 256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long first = (long)blockIdx.x * SORT_TILE + warp * (PER * 32);
  unsigned key[PER]; int val[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const long i = first + j * 32 + lane; const bool on = i < tokens;
    key[j] = !on ? 0u : FIRST ? token_key(ids, index_type, i, vocab) : ld(keys + i);
    val[j] = !on ? 0 : FIRST ? (int)i : ld(order + i);
  }
  for (int e = tid; e < W * 256; e += SORT_THREADS) cnt[e] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; j++) if (first + j * 32 + lane < tokens) atomicAdd(&cnt[warp * 256 + ((key[j] >> shift) & 255)], 1u);
  __syncthreads();
  unsigned at0;                                                      // thread = digit: where this tile's begin
  if constexpr (SCAN) {
    __shared__ unsigned sums[W];
    unsigned before = 0, total = 0;
#pragma unroll 32
    for (int t = 0; t < (int)gridDim.x; t++) { const unsigned c = ld(hist + t * 256 + tid); if (t < (int)blockIdx.x) before += c; total += c; }
    unsigned s = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned u = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += u; }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    for (int w = 0; w < warp; w++) s += sums[w];
    at0 = s - total + before;
  } else at0 = ld(hist + (long)tid * gridDim.x + blockIdx.x);
#pragma unroll
  for (int w = 0; w < W; w++) { const unsigned c = cnt[w * 256 + tid]; cnt[w * 256 + tid] = at0; at0 += c; }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const bool on = first + j * 32 + lane < tokens;
    const unsigned at = TileDigit::place(cnt + warp * 256, (key[j] >> shift) & 255, on, lane);
    if (on) { keys_out[at] = key[j]; order_out[at] = val[j]; }
  }
}

// ------------------------------------------------------------------ sums
// First place of the sorted keys that is not below `key`.
__device__ __forceinline__ long first_place(const unsigned* keys, long n, unsigned key) {
  long lo = 0, hi = n;
  while (lo < hi) { const long mid = (lo + hi) >> 1; if (ld(keys + mid) < key) lo = mid + 1; else hi = mid; }
  return lo;
}
constexpr int EMB_THREADS = 128, EMB_ZERO_ROWS = 32;
// Columns of a block: EMB_THREADS accesses of V elements; blockIdx.y counts those.  Blocks below `chunks` sum a piece each, the others zero the rows among
// EMB_ZERO_ROWS that no token names.
template <class T, int V>
__global__ void __launch_bounds__(EMB_THREADS) embedding_sum_kernel(const T* dout, long stride, const unsigned* keys, const int* order, long tokens, long vocab, int dim,
                                                                    float scale, int chunk, long chunks, float* dtable, float* partial) {
  op_begin();
  const long col = ((long)blockIdx.y * EMB_THREADS + threadIdx.x) * V; const bool in = col < dim;
  auto put = [&](float* row, const float (&v)[V]) {
    if (!in) return;
    if constexpr (V == 1) row[col] = v[0];
    else {
#pragma unroll
      for (int j = 0; j < V; j += 4) *reinterpret_cast<float4*>(row + col + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
  };
  if (blockIdx.x >= chunks) {
    const long v0 = (blockIdx.x - chunks) * EMB_ZERO_ROWS; const int lane = threadIdx.x & 31;
    const long v = v0 + lane; bool absent = false;
    if (v < vocab) { const long at = first_place(keys, tokens, (unsigned)v); absent = at >= tokens || ld(keys + at) != (unsigned)v; }
    unsigned todo = __ballot_sync(0xffffffffu, absent);
    float zero[V];
#pragma unroll
    for (int j = 0; j < V; j++) zero[j] = 0.f;
    while (todo) { const int r = __ffs(todo) - 1; todo &= todo - 1; put(dtable + (v0 + r) * dim, zero); }
    return;
  }
  const long first = (long)blockIdx.x * chunk, last = min(tokens, first + chunk);
  __shared__ unsigned ks[64 + 2]; __shared__ int os[64];
  for (int e = threadIdx.x; e < (int)(last - first); e += EMB_THREADS) { ks[e + 1] = ld(keys + first + e); os[e] = ld(order + first + e); }
  if (threadIdx.x == 0) ks[0] = first > 0 ? ld(keys + first - 1) : 0xffffffffu;
  if (threadIdx.x == 1) ks[last - first + 1] = last < tokens ? ld(keys + last) : 0xffffffffu;
  __syncthreads();
  const int n = (int)(last - first);
  constexpr int U = 8;                                               // rows under way
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; j++) sum[j] = 0.f;
  int begin = 0;                                                     // where the run under way begins
  for (int i0 = 0; i0 < n; i0 += U) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool on = in && i0 + u < n && ks[i0 + u + 1] < (unsigned)vocab;
      const T* src = dout + (long)(on ? os[i0 + u] : 0) * stride + col;
      if constexpr (V == 1) x[u][0] = on ? to_f32(*src) : 0.f;
      else {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (on) w = __ldcs(reinterpret_cast<const uint4*>(src));
        unpack<T>(w, x[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u;
      if (i >= n) break;
#pragma unroll
      for (int j = 0; j < V; j++) sum[j] += x[u][j];
      const unsigned key = ks[i + 1];
      const bool ends = key != ks[i + 2];
      if (ends || i == n - 1) {                                      // the run ends, or the piece does
        const bool came = begin == 0 && first > 0 && ks[0] == key, goes = !ends;
#pragma unroll
        for (int j = 0; j < V; j++) sum[j] *= scale;
        if (key < (unsigned)vocab) put(came ? partial + (2L * blockIdx.x) * dim : goes ? partial + (2L * blockIdx.x + 1) * dim : dtable + (long)key * dim, sum);
#pragma unroll
        for (int j = 0; j < V; j++) sum[j] = 0.f;
        begin = i + 1;
      }
    }
  }
}
// A run that goes on over the end of the piece where it began: that piece's last sum, then the first sums of the pieces behind it up to the one where the run ends.  Most runs end in the next piece:
// two warps look at a piece and add a run's parts, V columns a lane, in order; a run of more than JOIN_LONG pieces is left to the whole block, a quarter of its pieces to each two warps.  (A block for every
// piece: 18 us for 131072 tokens of 1024; looking the run's end up by bisection and 32 columns at a time: 127.)
constexpr int JOIN_COLS = 64, JOIN_GROUPS = 4, JOIN_LONG = 32;
template <int V>
__global__ void __launch_bounds__(JOIN_GROUPS * JOIN_COLS) embedding_join_kernel(const unsigned* keys, long tokens, long vocab, int dim, int chunk, long chunks, const float* partial, float* dtable) {
  op_begin();
  __shared__ float red[JOIN_GROUPS - 1][JOIN_COLS * V];
  __shared__ long length[JOIN_GROUPS]; __shared__ unsigned key_of[JOIN_GROUPS];
  const int w = threadIdx.x / JOIN_COLS, lane = threadIdx.x % JOIN_COLS; const long col = ((long)blockIdx.y * JOIN_COLS + lane) * V; const bool in = col < dim;
  const long c0 = (long)blockIdx.x * JOIN_GROUPS, c = c0 + w;
  long m = 0;                                                        // pieces behind this one that begin within a run which began here
  unsigned key = 0;
  if (c + 1 < chunks) {                                              // (a last piece has nothing behind it)
    key = ld(keys + (c + 1) * chunk - 1);
    const unsigned next = ld(keys + (c + 1) * chunk), begin = ld(keys + c * chunk), before = c > 0 ? ld(keys + c * chunk - 1) : 0xffffffffu;
    if (key < (unsigned)vocab && next == key && !(begin == key && before == key))
      for (long i0 = c + 2;; i0 += 32) {                             // the first piece behind that does not begin within the run
        const long i = i0 + (threadIdx.x & 31);
        const unsigned other = __ballot_sync(0xffffffffu, i >= chunks || ld(keys + i * chunk) != key);
        if (other) { m = i0 + __ffs(other) - 1 - c - 1; break; }
      }
  }
  auto add = [&](float (&v)[V], const float* row) {
    if constexpr (V == 1) v[0] += ld(row + col);
    else { const float4 u = ld(reinterpret_cast<const float4*>(row + col)); v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w; }
  };
  auto put = [&](const float (&v)[V], unsigned k) {
    float* out = dtable + (long)k * dim + col;
    if constexpr (V == 1) *out = v[0]; else *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
  };
  if (m > 0 && m <= JOIN_LONG && in) {
    float v[V] = {};
    add(v, partial + (2 * c + 1) * dim);
#pragma unroll 4
    for (long i = 0; i < m; i++) add(v, partial + 2 * (c + 1 + i) * dim);
    put(v, key);
  }
  if (lane == 0) { length[w] = m; key_of[w] = key; }
  if (!__syncthreads_or(m > JOIN_LONG)) return;
  for (int g = 0; g < JOIN_GROUPS; g++) {
    const long n = length[g], p = c0 + g, per = (n + JOIN_GROUPS - 1) / JOIN_GROUPS;
    if (n <= JOIN_LONG) continue;
    float v[V] = {};
    if (in) {
      if (w == 0) add(v, partial + (2 * p + 1) * dim);
#pragma unroll 8
      for (long i = w * per; i < min(n, (w + 1) * per); i++) add(v, partial + 2 * (p + 1 + i) * dim);
    }
    if (w > 0) {
#pragma unroll
      for (int j = 0; j < V; j++) red[w - 1][lane * V + j] = v[j];
    }
    __syncthreads();
    if (w == 0 && in) {
#pragma unroll
      for (int j = 0; j < V; j++) for (int i = 0; i < JOIN_GROUPS - 1; i++) v[j] += red[i][lane * V + j];
      put(v, key_of[g]);
    }
    __syncthreads();
  }
}

template <class T>
inline int embedding_sums(const EmbeddingPlan& pl, const void* dout, long stride, uint8_t* ws, long tokens, long vocab, int dim, float scale, float* dtable, void* stream) {
  const unsigned* keys = reinterpret_cast<const unsigned*>(ws + pl.keys); const int* order = reinterpret_cast<const int*>(ws + pl.order);
  float* partial = reinterpret_cast<float*>(ws + pl.partial);
  constexpr int N = Vec<T>::N;
  const bool vec = dim % N == 0 && stride % N == 0 && aligned_to(dout, 16) && aligned_to(dtable, 16);
  const dim3 grid((unsigned)(pl.chunks + ceil_div(vocab, EMB_ZERO_ROWS)), (unsigned)ceil_div(dim, EMB_THREADS * (vec ? N : 1)));
  if (ceil_div(dim, JOIN_COLS) > 65535) return fail(GN_ERR_UNSUPPORTED, "op_embedding_backward: dim is too large");
  if (vec) GN_TRY(op_launch("embedding_sum", stream, embedding_sum_kernel<T, N>, grid, dim3(EMB_THREADS), 0, 0, static_cast<const T*>(dout), stride, keys, order, tokens, vocab, dim, scale, pl.chunk, (long)pl.chunks, dtable, partial));
  else GN_TRY(op_launch("embedding_sum", stream, embedding_sum_kernel<T, 1>, grid, dim3(EMB_THREADS), 0, 0, static_cast<const T*>(dout), stride, keys, order, tokens, vocab, dim, scale, pl.chunk, (long)pl.chunks, dtable, partial));
  if (pl.chunks < 2) return GN_OK;
  const bool vec4 = dim % 4 == 0 && aligned_to(dtable, 16);
  const dim3 join((unsigned)ceil_div(pl.chunks - 1, JOIN_GROUPS), (unsigned)ceil_div(dim, JOIN_COLS * (vec4 ? 4 : 1)));
  return op_launch("embedding_join", stream, vec4 ? embedding_join_kernel<4> : embedding_join_kernel<1>, join, dim3(JOIN_GROUPS * JOIN_COLS), 0, 0, keys, tokens, vocab, dim, pl.chunk, (long)pl.chunks, (const float*)partial, dtable);
}

}  // namespace gn

extern "C" {

int gn_op_embedding(gn_ctx* ctx, int dtype, int64_t tokens, int64_t vocab, int dim, float scale, const void* table, int64_t table_stride, const void* ids, int index_type, void* out, int64_t out_stride, void* stream) {
  using namespace gn;
  const char* wrong = check_embedding(dtype, tokens, vocab, dim, scale, table, table_stride, vocab, ids, index_type, out, out_stride, tokens);
  if (!wrong) wrong = check_dtype(dtype, out);
  GN_OP_BEGIN("op_embedding", wrong);
  if (tokens == 0) return GN_OK;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(tokens, 8), (int64_t)ctx->c.sm_count * 8);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t); constexpr int N = Vec<T>::N;
    const bool vec = dim % N == 0 && table_stride % N == 0 && out_stride % N == 0 && aligned_to(table, 16) && aligned_to(out, 16);
    return op_launch("embedding", stream, vec ? embedding_kernel<T, N> : embedding_kernel<T, 1>, dim3(grid), dim3(256), 0, 0, static_cast<const T*>(table), (long)table_stride, ids, index_type, (long)tokens, (long)vocab, dim, scale,
                     static_cast<T*>(out), (long)out_stride);
  });
}

int gn_op_embedding_workspace(gn_ctx* ctx, int64_t tokens, int64_t vocab, int dim, int64_t* bytes) {
  using namespace gn;
  if (!ctx || !ctx->alive || !bytes || tokens < 0 || tokens > OP_MAX_ROWS || vocab < 1 || vocab >= OP_MAX_ROWS || dim < 1) return fail(GN_ERR_INVALID_ARG, "op_embedding_workspace: bad argument");
  *bytes = tokens == 0 ? 0 : embedding_plan(tokens, vocab, dim, ctx->c.sm_count).bytes; return GN_OK;
}

int gn_op_embedding_backward(gn_ctx* ctx, int dtype, int64_t tokens, int64_t vocab, int dim, float scale, const void* dout, int64_t dout_stride, const void* ids, int index_type, float* dtable,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace gn;
  const char* wrong = check_embedding(dtype, tokens, vocab, dim, scale, dout, dout_stride, tokens, ids, index_type, dtable, dim, vocab);
  if (!wrong && !aligned_to(dtable, 4)) wrong = "a pointer is not aligned to its type";
  GN_OP_BEGIN("op_embedding_backward", wrong);
  if (tokens == 0) { GN_CUDA(cudaMemsetAsync(dtable, 0, 4UL * vocab * dim, (cudaStream_t)stream)); return GN_OK; }
  const EmbeddingPlan pl = embedding_plan(tokens, vocab, dim, ctx->c.sm_count);
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < pl.bytes) return fail(GN_ERR_INVALID_ARG, "op_embedding_backward: the workspace is too small, null or not aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto u = [&](int64_t at) { return reinterpret_cast<unsigned*>(ws + at); };
  if (pl.small) {
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(tokens, RANK_TOKENS), (int64_t)ctx->c.sm_count);
    GN_TRY(op_launch("sort_rank", stream, sort_rank_kernel, dim3(blocks), dim3(RANK_THREADS), 0, 0, ids, index_type, (int)tokens, (long)vocab, u(pl.keys), (int*)u(pl.order)));
  } else {
    const dim3 grid((unsigned)pl.tiles), block(SORT_THREADS);
    for (int pass = 0; pass < pl.passes; pass++) {                   // the last pass writes `keys` and `order`
      const bool to_first = (pl.passes - pass) % 2 == 1;
      const unsigned* kin = u(to_first ? pl.keys2 : pl.keys); const int* vin = (const int*)u(to_first ? pl.order2 : pl.order);
      unsigned* kout = u(to_first ? pl.keys : pl.keys2); int* vout = (int*)u(to_first ? pl.order : pl.order2);
      const int shift = pass * SORT_BITS; const bool scan = pl.tiles <= SORT_SCAN_TILES;
      GN_TRY(op_launch("sort_count", stream, pass == 0 ? sort_count_kernel<true> : sort_count_kernel<false>, grid, block, 0, 0, ids, index_type, kin, (long)tokens, (long)vocab, shift, scan, u(pl.hist)));
      if (!scan) GN_TRY(op_launch("sort_scan", stream, sort_scan_kernel, dim3(1), dim3(1024), 0, 0, u(pl.hist), (long)(pl.tiles << SORT_BITS)));
      GN_TRY(op_launch("sort_move", stream, pass == 0 ? (scan ? sort_move_kernel<true, true> : sort_move_kernel<true, false>) : scan ? sort_move_kernel<false, true> : sort_move_kernel<false, false>, grid, block, 0, 0, ids, index_type, kin, vin, (long)tokens, (long)vocab, shift, (const unsigned*)u(pl.hist), kout, vout));
    }
  }
  return with_type(dtype, [&](auto t) { using T = decltype(t); return embedding_sums<T>(pl, dout, (long)dout_stride, ws, (long)tokens, (long)vocab, dim, scale, dtable, stream); });
}

}  // extern "C"
