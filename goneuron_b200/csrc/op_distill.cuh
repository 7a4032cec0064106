// op_distill.cuh -- distillation from a teacher's top logits: loss and gradient from one reading of the student's logits.
//
//   p = softmax(t / T) over a row's entries, q = softmax(s / T) over the vocabulary,
//   loss = w T^2 sum_k p_k (log p_k - log q_{id_k}),      ds = w T (q - p)
//
// All exponentials are of base 2, with c = log2(e) / T: e_j = 2^((s_j - m) c) with m the largest s_j of the thread's own elements, so that no thread waits for
// another before it sums; (m, sum) pairs then meet in shuffles, in shared memory and between the blocks of a cluster, and q_j = e_j 2^((m - M) c) / S.  Differences
// come before the factor: logits at the type's lowest value stay finite.
//
// Bound by memory: a row is read once and its gradient written once.  One launch forms what the teacher's few entries come to, a warp a row, so that no long
// row waits for their chain of dependent loads; the second streams the rows.  A row stays on chip there, 32 elements a thread in registers as float32 exponentials (one exponential
// an element: with two the special-function units bound it, 2 x 11 an SM and cycle at full bandwidth against the 16 they give).  While a row is in registers the same
// thread's asynchronous copies fetch its elements of the next one, into slots of shared memory that no other thread touches, so that the only barrier
// of a row is the one at which the sums meet.  A row that is too long for 512 threads is spread over a cluster of blocks, two of which share an SM and overlap each
// other's barriers.  Each block writes q for all of its elements; where the teacher has entries q - p is written over it, behind the next row's barrier.
#pragma once
#include "device_ops.cuh"

namespace gn {

// What the teacher's entries of a row come to: l as in Norm below, r the student's largest value where the teacher has probability (0 if it has none), d = sum of
// p ((t - max t) - (s - r)); w: the row's weight, 0 where it has no entry of positive probability.
struct alignas(16) Teacher { float l, d, r, w; };
struct DistillParams {
  const void* logits; long stride; const void* ids; int index_type; const float* top_logits; const float* weight; float* loss; void* dlogits; long dstride;
  long rows, vocab; int top; float temperature;
  Teacher* teach; int* id; float* prob; float* stud;                 // workspace: [rows], and [rows][top] each (the gradient's)
};

struct MaxSum { float m, s; };                                       // of values v: m >= all v (or -inf: none), s = sum of 2^((v - m) c)
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m), r = m == -INFINITY ? 0.f : m;     // (nothing on either side)
  return MaxSum{m, a.s * ex2((a.m - r) * c) + b.s * ex2((b.m - r) * c)};
}
__device__ __forceinline__ MaxSum warp_join(MaxSum v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, MaxSum{__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o)}, c);
  return v;
}
// A row's probabilities are 2^((s - m) c - l).
struct Norm { float m, l; };
__device__ __forceinline__ Norm norm_of(MaxSum v) { return Norm{v.m, log2f(v.s)}; }

constexpr int DISTILL_TOP = 1024;
// id (-1: none) and logit of entry k
__device__ __forceinline__ int teacher_entry(const DistillParams& p, long row, int k, float& t) {
  const int64_t id = load_index(p.ids, p.index_type, row * p.top + k);
  const bool there = id >= 0 && id < p.vocab;
  if (!there && id != -1) op_report(OP_BAD_INDEX);
  t = there ? __ldg(p.top_logits + row * p.top + k) : -INFINITY;
  return there ? (int)id : -1;
}
// A warp a row.  With a gradient the entries' ids, probabilities and student values are kept for the second launch; of entries with the same id the first keeps all of their
// probability and the others become -1.  Such entries are rare and found by a table: every entry writes its number at its id's place, and whoever finds another's number there, or is found by
// another of the same id, looks through the row.
constexpr int TEACHER_WARPS = 4, TEACHER_TABLE = 2048;
inline int teacher_smem(int top) { return TEACHER_WARPS * (TEACHER_TABLE * 2 + (top + 3) / 4 * 4 * 9); }      // table, ids, probabilities, flags
template <class T, bool GRAD>
__global__ void __launch_bounds__(32 * TEACHER_WARPS) distill_teacher_kernel(const __grid_constant__ DistillParams p) {
  op_begin();
  extern __shared__ uint4 teacher_smem_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, top4 = (p.top + 3) & ~3; const float c = 1.4426950408889634f / p.temperature;
  uint8_t* own = reinterpret_cast<uint8_t*>(teacher_smem_raw) + warp * (TEACHER_TABLE * 2 + top4 * 9);
  int* id_of = reinterpret_cast<int*>(own); float* prob_of = reinterpret_cast<float*>(id_of + top4);
  unsigned short* table = reinterpret_cast<unsigned short*>(prob_of + top4); uint8_t* look = reinterpret_cast<uint8_t*>(table + TEACHER_TABLE);
  const long row = (long)blockIdx.x * TEACHER_WARPS + warp;
  if (row >= p.rows) return;
  const float w = p.weight ? __ldg(p.weight + row) : 1.f;
  Teacher out{0.f, 0.f, 0.f, 0.f};
  if (w != 0.f) {
    const T* logits = static_cast<const T*>(p.logits) + row * p.stride;
    MaxSum v{-INFINITY, 0.f};
    for (int k = lane; k < p.top; k += 32) { float t; teacher_entry(p, row, k, t); v = join(v, MaxSum{t, t == -INFINITY ? 0.f : 1.f}, c); }
    v = warp_join(v, c);
    const bool some = !(v.m == -INFINITY && v.s == 0.f); const Norm n = norm_of(v);
    float d = 0.f, r = -INFINITY, weight = 0.f;                      // d: relative to this lane's r so far; weight: the probability that it holds
    for (int k = lane; k < p.top; k += 32) {
      float t; const int id = teacher_entry(p, row, k, t);
      const float pk = !some || t == -INFINITY ? 0.f : exp2f((t - n.m) * c - n.l), s = id >= 0 ? to_f32(logits[id]) : 0.f;
      if (pk != 0.f) {                                               // (an entry without weight says nothing, whatever the student has there)
        if (s > r) { if (weight != 0.f) d += weight * (s - r); r = s; }      // sum of p (r - s) moves with r
        d += pk * ((t - n.m) - (s - (r == -INFINITY ? 0.f : r))); weight += pk;
      }
      if constexpr (GRAD) {
        p.stud[row * p.top + k] = s; id_of[k] = id; prob_of[k] = pk; look[k] = 0;
        if (id >= 0) table[id & (TEACHER_TABLE - 1)] = (unsigned short)k;
      }
    }
    const float top = warp_max(r), ref = top == -INFINITY ? 0.f : top;
    if (weight != 0.f) d += weight * (ref - (r == -INFINITY ? 0.f : r));
    out = Teacher{n.l, warp_sum(d), ref, some ? w : 0.f};
    if constexpr (GRAD) {
      __syncwarp();
      for (int k = lane; k < p.top; k += 32) {
        const int id = id_of[k];
        if (id < 0) continue;
        const int found = table[id & (TEACHER_TABLE - 1)];
        if (found != k) { look[k] = 1; if (id_of[found] == id) look[found] = 1; }
      }
      __syncwarp();
      for (int k = lane; k < p.top; k += 32) {
        int id = id_of[k]; float pk = prob_of[k];
        if (look[k]) {
          pk = 0.f;
          for (int f = 0; f < p.top; f++) if (id_of[f] == id) { if (f < k) { id = -1; break; } pk += prob_of[f]; }
        }
        p.id[row * p.top + k] = id; p.prob[row * p.top + k] = pk;
      }
    }
  }
  if (lane == 0) p.teach[row] = out;
}
// w T^2 sum of p (log p - log q), from p = 2^((t - max t) c - l_t) and q = 2^((s - M) c - l), as the p add up to 1
__device__ __forceinline__ float distill_loss(const Teacher& t, Norm n, float tau) { return t.w != 0.f ? t.w * tau * (t.d + (n.m - t.r) + tau * 0.69314718055994531f * (n.l - t.l)) : 0.f; }
// q - p where the teacher has entries of row r, over what is there, for ids in [lo, hi)
template <class T>
__device__ __forceinline__ void distill_entries(const DistillParams& p, long r, float w, Norm n, float c, long lo, long hi) {
  if (w == 0.f) return;
  T* out = static_cast<T*>(p.dlogits) + r * p.dstride;
  for (int e = threadIdx.x; e < p.top; e += blockDim.x) {
    const int id = p.id[r * p.top + e];
    if (id >= lo && id < hi && id >= 0) out[id] = from_f32<T>(w * p.temperature * (ex2((p.stud[r * p.top + e] - n.m) * c - n.l) - p.prob[r * p.top + e]));
  }
}

// Elements of a row from the 16-byte boundary at or before its first one.
template <class T> __device__ __forceinline__ int row_lead(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }

// NT threads of `cl` blocks on a row, `per` 16-byte pieces of it (counted from its 16-byte boundary) for each block; BUF rows of slots.
template <class T, int NT, bool GRAD>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_kernel(const __grid_constant__ DistillParams p, int cl, int per) {
  namespace cg = cooperative_groups;
  constexpr int V = Vec<T>::N, J = DISTILL_ITEMS / V, W = NT / 32, BUF = sizeof(T) == 2 ? 2 : 1;      // J pieces a thread; two rows under way where 16-bit elements leave room for them
  op_begin();
  extern __shared__ uint4 slots[];                                   // [BUF][J][NT]
  __shared__ MaxSum part[2][W]; __shared__ MaxSum peers[2][8];       // (rows take turns: a warp may be a row ahead of another, never two)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = (int)p.vocab;
  const int rank = cl > 1 ? (int)(blockIdx.x % cl) : 0; const long row0 = blockIdx.x / cl, step = gridDim.x / cl;
  const float c = 1.4426950408889634f / p.temperature;
  const uint32_t slot0 = (uint32_t)__cvta_generic_to_shared(slots) + tid * 16;
  const int at = rank * per;                                         // this block's pieces: [at, at + per), as far as the row goes
  auto row_of = [&](long r) { return static_cast<const T*>(p.logits) + r * p.stride; };
  auto weight_of = [&](long r) { return r < p.rows ? __ldg(&p.teach[r].w) : 0.f; };
  // copies of this thread's pieces of row r into buffer b; pieces that the row does not fill are put together element by element, -inf where it has none
  auto fetch = [&](long r, float w, int b) {
    if (w != 0.f) {
      const T* row = row_of(r); const int lead = row_lead(row);
#pragma unroll
      for (int j = 0; j < J; j++) {
        const int i = j * NT + tid, e = (at + i) * V - lead;         // e: first element
        if (i < per && e < vocab) {
          if (e >= 0 && e + V <= vocab) cp16(slot0 + (b * J + j) * NT * 16, row + e);
          else {
            T* q = reinterpret_cast<T*>(slots + (b * J + j) * NT + tid);
#pragma unroll
            for (int l = 0; l < V; l++) q[l] = e + l >= 0 && e + l < vocab ? row[e + l] : from_f32<T>(-INFINITY);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  for (int b = 0; b < BUF; b++) fetch(row0 + b * step, weight_of(row0 + b * step), b);
  float ahead = weight_of(row0 + BUF * step);                        // weight of the row that is fetched next
  int b = 0, par = 0; long done = -1; float done_w = 0.f; Norm done_n{0.f, 0.f};
  for (long r = row0; r < p.rows; r += step) {
    const T* row = row_of(r); const int lead = row_lead(row);
    const Teacher t = p.teach[r]; const bool on = t.w != 0.f;
    if constexpr (BUF == 1) asm volatile("cp.async.wait_group 0;" ::: "memory"); else asm volatile("cp.async.wait_group 1;" ::: "memory");
    float x[DISTILL_ITEMS]; float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; j++) {
      float v[V]; const int i = j * NT + tid;
      if (on && i < per && (at + i) * V - lead < vocab) unpack<T>(slots[(b * J + j) * NT + tid], v);
      else {
#pragma unroll
        for (int l = 0; l < V; l++) v[l] = -INFINITY;
      }
#pragma unroll
      for (int l = 0; l < V; l++) { x[j * V + l] = v[l]; m = fmaxf(m, v[l]); }
    }
    fetch(r + BUF * step, ahead, b);                                 // (the values have been read: m depends on them all)
    ahead = weight_of(r + (BUF + 1) * step);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < DISTILL_ITEMS; j++) { x[j] = ex2((x[j] - ref) * c); s += x[j]; }
    s = warp_sum(s);
    if (lane == 0) part[par][warp] = MaxSum{m, s};
    __syncthreads();
    auto meet = [&](MaxSum v) {
      const float top = warp_max(v.m), to = top == -INFINITY ? 0.f : top;
      return MaxSum{top, warp_sum(v.s * ex2((v.m - to) * c))};
    };
    MaxSum v = meet(lane < W ? part[par][lane] : MaxSum{-INFINITY, 0.f});
    if (cl > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      if (tid < cl) *cluster.map_shared_rank(&peers[par][rank], tid) = v;
      cluster.sync();
      v = meet(lane < cl ? peers[par][lane] : MaxSum{-INFINITY, 0.f});
    }
    const Norm n = norm_of(v);
    if (tid == 0 && rank == 0) p.loss[r] = distill_loss(t, n, p.temperature);
    if constexpr (GRAD) {
      const float f = !on || (m == -INFINITY && n.m > -INFINITY) ? 0.f : t.w * p.temperature * ex2((m - n.m) * c - n.l);
      T* out = static_cast<T*>(p.dlogits) + r * p.dstride; const bool same = row_lead(out) == lead;
#pragma unroll
      for (int j = 0; j < J; j++) {
        const int i = j * NT + tid, e = (at + i) * V - lead;
        if (i >= per || e >= vocab) continue;
        float y[V];
#pragma unroll
        for (int l = 0; l < V; l++) y[l] = on ? x[j * V + l] * f : 0.f;
        if (same && e >= 0 && e + V <= vocab) *reinterpret_cast<uint4*>(out + e) = pack<T>(y);
        else {
#pragma unroll
          for (int l = 0; l < V; l++) if (e + l >= 0 && e + l < vocab) out[e + l] = from_f32<T>(y[l]);
        }
      }
      if (done >= 0) { const int l0 = row_lead(row_of(done)); distill_entries<T>(p, done, done_w, done_n, c, (long)at * V - l0, (long)(at + per) * V - l0); }
      done = r; done_w = t.w; done_n = n;
    }
    par ^= 1; if (++b == BUF) b = 0;
  }
  if constexpr (GRAD) {
    __syncthreads();
    if (done >= 0) { const int l0 = row_lead(row_of(done)); distill_entries<T>(p, done, done_w, done_n, c, (long)at * V - l0, (long)(at + per) * V - l0); }
  }
  if (cl > 1) cg::this_cluster().sync();                             // (no block leaves while another may still write into it)
}

// A row that does not fit on chip: one block reads it twice.
template <class T, bool GRAD>
__global__ void __launch_bounds__(1024) distill_long_kernel(const __grid_constant__ DistillParams p) {
  op_begin();
  __shared__ MaxSum part[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5; const float c = 1.4426950408889634f / p.temperature;
  for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* row = static_cast<const T*>(p.logits) + r * p.stride; const Teacher t = p.teach[r]; const bool on = t.w != 0.f;
    MaxSum v{-INFINITY, 0.f};
    if (on)
      for (long e0 = tid; e0 < p.vocab; e0 += 8 * 1024) {
        float x[8]; float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; j++) { x[j] = e0 + j * 1024 < p.vocab ? to_f32(row[e0 + j * 1024]) : -INFINITY; m = fmaxf(m, x[j]); }
        const float ref = m == -INFINITY ? 0.f : m; float s = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) s += ex2((x[j] - ref) * c);
        v = join(v, MaxSum{m, s}, c);
      }
    v = warp_join(v, c);
    if (lane == 0) part[warp] = v;
    __syncthreads();
    const Norm n = norm_of(warp_join(part[lane], c));
    if (tid == 0) p.loss[r] = distill_loss(t, n, p.temperature);
    if constexpr (GRAD) {
      T* out = static_cast<T*>(p.dlogits) + r * p.dstride;
      for (long e = tid; e < p.vocab; e += 1024) out[e] = from_f32<T>(on ? t.w * p.temperature * ex2((to_f32(row[e]) - n.m) * c - n.l) : 0.f);
      __syncthreads();
      distill_entries<T>(p, r, t.w, n, c, 0, p.vocab);
    }
    __syncthreads();
  }
}

template <class T, bool GRAD>
inline int distill_launch(gn_ctx* ctx, const DistillParams& p, void* stream) {
  const int sms = ctx->c.sm_count; const DistillPlan pl = distill_plan(p.rows, p.vocab, sms);
  const int tsmem = teacher_smem(GRAD ? p.top : 0);
  if (tsmem > 48 * 1024) GN_TRY(op_smem("distill_teacher", distill_teacher_kernel<T, GRAD>, tsmem));
  GN_TRY(op_launch("distill_teacher", stream, distill_teacher_kernel<T, GRAD>, dim3(cdiv(p.rows, TEACHER_WARPS)), dim3(32 * TEACHER_WARPS), tsmem, 0, p));
  if (pl.cluster == 0) return op_launch("distill_long", stream, distill_long_kernel<T, GRAD>, dim3((unsigned)std::min<int64_t>(p.rows, 2L * sms)), dim3(1024), 0, 0, p);
  const int V = 16 / (int)sizeof(T), smem = (sizeof(T) == 2 ? 2 : 1) * pl.threads * DISTILL_ITEMS * (int)sizeof(T);      // 64 KB for 512 threads
  const int per = (int)ceil_div(ceil_div(p.vocab + V - 1, V), pl.cluster);
  const dim3 grid((unsigned)(std::min<int64_t>(p.rows, std::max<int64_t>(1, (int64_t)sms * (1024 / pl.threads) / pl.cluster)) * pl.cluster));
  auto go = [&](auto kernel) { if (smem > 48 * 1024) GN_TRY(op_smem("distill", kernel, smem)); return op_launch("distill", stream, kernel, grid, dim3(pl.threads), smem, pl.cluster, p, pl.cluster, per); };
  return pl.threads == 1024 ? go(distill_kernel<T, 1024, GRAD>) : pl.threads == 512 ? go(distill_kernel<T, 512, GRAD>) : pl.threads == 256 ? go(distill_kernel<T, 256, GRAD>) : go(distill_kernel<T, 64, GRAD>);
}

}  // namespace gn

extern "C" {

int gn_op_distill_workspace(gn_ctx* ctx, int64_t rows, int top, int gradient, int64_t* bytes) {
  using namespace gn;
  if (!ctx || !ctx->alive || !bytes || rows < 0 || rows > OP_MAX_ROWS || top < 0 || top > DISTILL_TOP) return fail(GN_ERR_INVALID_ARG, "op_distill_workspace: bad argument");
  *bytes = distill_workspace(rows, top, gradient != 0); return GN_OK;
}

int gn_op_distill(gn_ctx* ctx, int dtype, int64_t rows, int64_t vocab, int top, float temperature, const void* logits, int64_t row_stride, const void* top_ids, int index_type, const float* top_logits,
                  const float* weight, float* loss, void* dlogits, int64_t drow_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace gn;
  GN_OP_BEGIN("op_distill", check_distill(dtype, rows, vocab, top, temperature, logits, row_stride, top_ids, index_type, top_logits, weight, loss, dlogits, drow_stride));
  if (rows == 0) return GN_OK;
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < distill_workspace(rows, top, dlogits != nullptr)) return fail(GN_ERR_INVALID_ARG, "op_distill: the workspace is too small, null or not aligned");
  Teacher* teach = static_cast<Teacher*>(workspace); int* id = reinterpret_cast<int*>(teach + rows); float* prob = reinterpret_cast<float*>(id + rows * top);
  const DistillParams p{logits, (long)row_stride, top_ids, index_type, top_logits, weight, loss, dlogits, (long)drow_stride, (long)rows, (long)vocab, top, temperature, teach, id, prob, prob + rows * top};
  return with_type(dtype, [&](auto t) { using T = decltype(t); return dlogits ? distill_launch<T, true>(ctx, p, stream) : distill_launch<T, false>(ctx, p, stream); });
}

}  // extern "C"
