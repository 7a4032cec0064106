// op_distill.cuh -- distillation from a teacher's top logits: loss and gradient from one reading of the student's logits.
//
//   p = softmax(t / T) over a row's entries, q = softmax(s / T) over the vocabulary,
//   loss = w T^2 sum_k p_k (log p_k - log q_{id_k}),      ds = w T (q - p)
//
// All exponentials are of base 2, with c = log2(e) / T: e_j = 2^((s_j - m) c) with m the largest s_j of the thread's own elements, so that no thread waits for
// another before it sums; (m, sum) pairs then meet in shuffles, in shared memory and between the blocks of a cluster, and q_j = e_j 2^((m - M) c) / S.  Differences
// come before the factor: logits at the type's lowest value stay finite.
//
// Bound by memory: a row is read once and its gradient written once.  A row stays on chip, 32 elements a thread in registers as float32 exponentials (one exponential an element:
// with two the special-function units bound it, 2 x 11 an SM and cycle at full bandwidth against the 16 they give).  While a row is in registers the same
// thread's asynchronous copies fetch its elements of the next one, into slots of shared memory that no other thread touches, so that the only barrier
// of a row is the one at which the sums meet.  A row that is too long for one block is spread over a cluster of up to eight.
// Each block writes q for all of its elements; where the teacher has entries q - p is written over it, behind the next row's barrier.
#pragma once
#include "device_ops.cuh"

namespace gn {

struct DistillParams {
  const void* logits; long stride; const void* ids; int index_type; const float* top_logits; const float* weight; float* loss; void* dlogits; long dstride;
  long rows, vocab; int top; float temperature;
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

// What the teacher's entries of a row come to, formed by one warp: l as above, r the student's largest value where the teacher has probability (0 if it has none),
// d = sum of p ((t - max t) - (s - r)).
struct Teacher { float l, d, r; bool some; };
constexpr int DISTILL_TOP = 1024;
// id (-1: none) and logit of entry k
__device__ __forceinline__ int teacher_entry(const DistillParams& p, long row, int k, float& t) {
  const int64_t id = load_index(p.ids, p.index_type, row * p.top + k);
  const bool there = id >= 0 && id < p.vocab;
  if (!there && id != -1) op_report(OP_BAD_INDEX);
  t = there ? __ldg(p.top_logits + row * p.top + k) : -INFINITY;
  return there ? (int)id : -1;
}
// ids / probabilities / student values of the row's entries to `ids`, `prob`, `stud` (`keep`), and the loss's part (`loss`); one warp.
template <class T>
__device__ __forceinline__ Teacher teacher_row(const DistillParams& p, long row, const T* logits, float c, int lane, bool keep, int* ids, float* prob, float* stud, bool loss) {
  MaxSum v{-INFINITY, 0.f};
  for (int k = lane; k < p.top; k += 32) { float t; teacher_entry(p, row, k, t); v = join(v, MaxSum{t, t == -INFINITY ? 0.f : 1.f}, c); }
  v = warp_join(v, c);
  Teacher out{0.f, 0.f, 0.f, !(v.m == -INFINITY && v.s == 0.f)};
  const Norm n = norm_of(v);
  out.l = n.l;
  float d = 0.f, r = -INFINITY;                                      // d: relative to this lane's r so far
  float weight = 0.f;                                                // probability that it holds
  for (int k = lane; k < p.top; k += 32) {
    float t; const int id = teacher_entry(p, row, k, t);
    const float pk = !out.some || t == -INFINITY ? 0.f : exp2f((t - n.m) * c - n.l);
    const float s = id >= 0 && (loss || keep) ? to_f32(logits[id]) : 0.f;
    if (pk != 0.f) {                                                 // (an entry without weight says nothing, whatever the student has there)
      if (s > r) { if (weight != 0.f) d += weight * (s - r); r = s; }      // sum of p (r - s) moves with r
      d += pk * ((t - n.m) - (s - (r == -INFINITY ? 0.f : r))); weight += pk;
    }
    if (keep) { ids[k] = id; prob[k] = pk; stud[k] = s; }
  }
  const float top = warp_max(r), ref = top == -INFINITY ? 0.f : top;
  if (weight != 0.f) d += weight * (ref - (r == -INFINITY ? 0.f : r));
  out.r = ref; out.d = warp_sum(d); return out;
}
// w T^2 sum of p (log p - log q), from p = 2^((t - max t) c - l_t) and q = 2^((s - M) c - l), as the p add up to 1
__device__ __forceinline__ float distill_loss(const Teacher& t, Norm n, float tau, float w, bool on) {
  return on ? w * tau * (t.d + (n.m - t.r) + tau * 0.69314718055994531f * (n.l - t.l)) : 0.f;
}

// Elements of a row from the 16-byte boundary at or before its first one.
template <class T> __device__ __forceinline__ int row_lead(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }

// NT threads of CL blocks on a row, BUF rows of slots.
template <class T, int NT, bool GRAD>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_kernel(const __grid_constant__ DistillParams p, int cl, int buffers) {
  namespace cg = cooperative_groups;
  constexpr int V = Vec<T>::N, J = DISTILL_ITEMS / V, W = NT / 32;   // J accesses of 16 bytes a thread
  extern __shared__ uint4 slots[];                                   // [buffers][J][NT], then per row in turn of three the entries' ids, probabilities and student values
  __shared__ MaxSum part[2][W]; __shared__ MaxSum peers[2][8]; __shared__ Teacher teach[3];
  __shared__ Norm norms[3];
  // Rows take turns with what their barrier guards: two sets where it is read before the next row's barrier, three where behind it (a warp may be a row
  // ahead of another, never two).
  float* const kept = reinterpret_cast<float*>(slots + (long)buffers * J * NT);
  auto ids = [&](int t) { return reinterpret_cast<int*>(kept + t * 3 * p.top); };
  auto prob = [&](int t) { return kept + t * 3 * p.top + p.top; };
  auto stud = [&](int t) { return kept + t * 3 * p.top + 2 * p.top; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cl > 1 ? (int)(blockIdx.x % cl) : 0; const long row0 = blockIdx.x / cl, step = gridDim.x / cl;
  const float c = 1.4426950408889634f / p.temperature;
  const uint32_t slot0 = (uint32_t)__cvta_generic_to_shared(slots) + tid * 16;
  // pieces of a row: [0, n) from its 16-byte boundary on, of which this block has [at, at + own)
  struct Cut { const T* row; int lead; long n, at, own; };
  auto cut = [&](long r) {
    Cut k; k.row = static_cast<const T*>(p.logits) + r * p.stride; k.lead = row_lead(k.row);
    k.n = (k.lead + p.vocab + V - 1) / V; const long per = (k.n + cl - 1) / cl;
    k.at = min(k.n, rank * per); k.own = min(k.n, k.at + per) - k.at; return k;
  };
  auto weight_of = [&](long r) { return p.weight ? __ldg(p.weight + r) : 1.f; };
  // copies of this thread's pieces of row r into buffer b; pieces that the row does not fill are put together element by element, -inf where it has none
  auto fetch = [&](long r, int b) {
    if (r < p.rows && weight_of(r) != 0.f) {
      const Cut k = cut(r);
#pragma unroll
      for (int j = 0; j < J; j++) {
        const long i = j * NT + tid;
        if (i < k.own) {
          const long e = (k.at + i) * V - k.lead;                    // first element
          uint4* s = slots + (long)(b * J + j) * NT + tid;
          if (e >= 0 && e + V <= p.vocab) cp16(slot0 + (b * J + j) * NT * 16, k.row + e);
          else {
            T* q = reinterpret_cast<T*>(s);
#pragma unroll
            for (int l = 0; l < V; l++) q[l] = e + l >= 0 && e + l < p.vocab ? k.row[e + l] : from_f32<T>(-INFINITY);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // q - p where the teacher has entries of row r, over the q of this block's elements; equal ids: the first one writes for all
  auto entries = [&](long r, int t) {
    const float w = weight_of(r); const Norm n = norms[t];
    if (w == 0.f || !teach[t].some) return;
    const Cut k = cut(r); const long lo = k.at * V - k.lead, hi = lo + k.own * V;
    T* out = static_cast<T*>(p.dlogits) + r * p.dstride; const int* id_of = ids(t); const float* prob_of = prob(t);
    for (int e = tid; e < p.top; e += NT) {
      const int id = id_of[e];
      if (id < 0 || id < lo || id >= hi) continue;
      float sum = 0.f; bool first = true;
      for (int f = 0; f < p.top; f++) if (id_of[f] == id) { if (f < e) { first = false; break; } sum += prob_of[f]; }
      if (first) out[id] = from_f32<T>(w * p.temperature * (ex2((stud(t)[e] - n.m) * c - n.l) - sum));
    }
  };

  for (int b = 0; b < buffers; b++) fetch(row0 + b * step, b);
  int b = 0, par = 0, turn = 0; long done = -1;
  for (long r = row0; r < p.rows; r += step) {
    const Cut k = cut(r); const float w = weight_of(r); const bool live = w != 0.f;
    if (buffers == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (buffers == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
    float x[DISTILL_ITEMS]; float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; j++) {
      float v[V];
      if (live && j * NT + tid < k.own) unpack<T>(slots[(long)(b * J + j) * NT + tid], v);
      else {
#pragma unroll
        for (int l = 0; l < V; l++) v[l] = -INFINITY;
      }
#pragma unroll
      for (int l = 0; l < V; l++) { x[j * V + l] = v[l]; m = fmaxf(m, v[l]); }
    }
    fetch(r + buffers * step, b);                                    // (the values have been read: m depends on them all)
    if (warp == 0) {                                                 // the teacher's part, and the student's values there, before anything of the row is overwritten
      Teacher t{};
      if (live) t = teacher_row<T>(p, r, k.row, c, lane, GRAD, ids(turn), prob(turn), stud(turn), rank == 0);
      if (lane == 0) teach[turn] = t;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < DISTILL_ITEMS; j++) { x[j] = ex2((x[j] - ref) * c); s += x[j]; }
    MaxSum v = warp_join(MaxSum{m, s}, c);
    if (lane == 0) part[par][warp] = v;
    __syncthreads();
    v = warp_join(lane < W ? part[par][lane] : MaxSum{-INFINITY, 0.f}, c);
    if (cl > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      if (tid < cl) *cluster.map_shared_rank(&peers[par][rank], tid) = v;
      cluster.sync();
      v = warp_join(lane < cl ? peers[par][lane] : MaxSum{-INFINITY, 0.f}, c);
    }
    const Norm n = norm_of(v); const Teacher t = teach[turn]; const bool on = live && t.some;
    if (tid == 0) { norms[turn] = n; if (rank == 0) p.loss[r] = distill_loss(t, n, p.temperature, w, on); }
    if constexpr (GRAD) {
      if (done >= 0) entries(done, turn == 0 ? 2 : turn - 1);
      const float f = !on || (m == -INFINITY && n.m > -INFINITY) ? 0.f : w * p.temperature * ex2((m - n.m) * c - n.l);
      T* out = static_cast<T*>(p.dlogits) + r * p.dstride; const bool same = row_lead(out) == k.lead;
#pragma unroll
      for (int j = 0; j < J; j++) {
        const long i = j * NT + tid;
        if (i >= k.own) continue;
        const long e = (k.at + i) * V - k.lead;
        float y[V];
#pragma unroll
        for (int l = 0; l < V; l++) y[l] = on ? x[j * V + l] * f : 0.f;
        if (same && e >= 0 && e + V <= p.vocab) *reinterpret_cast<uint4*>(out + e) = pack<T>(y);
        else {
#pragma unroll
          for (int l = 0; l < V; l++) if (e + l >= 0 && e + l < p.vocab) out[e + l] = from_f32<T>(y[l]);
        }
      }
      done = r;
    }
    par ^= 1; if (++turn == 3) turn = 0; if (++b == buffers) b = 0;
  }
  if constexpr (GRAD) {
    __syncthreads();
    if (done >= 0) entries(done, turn == 0 ? 2 : turn - 1);
  }
  if (cl > 1) cg::this_cluster().sync();                             // (no block leaves while another may still write into it)
}

// A row that does not fit on chip: one block reads it twice.
template <class T, bool GRAD>
__global__ void __launch_bounds__(1024) distill_long_kernel(const __grid_constant__ DistillParams p) {
  __shared__ MaxSum part[32]; __shared__ Teacher teach;
  __shared__ int ids[DISTILL_TOP]; __shared__ float prob[DISTILL_TOP], stud[DISTILL_TOP];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5; const float c = 1.4426950408889634f / p.temperature;
  for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* row = static_cast<const T*>(p.logits) + r * p.stride; const float w = p.weight ? __ldg(p.weight + r) : 1.f; const bool live = w != 0.f;
    MaxSum v{-INFINITY, 0.f};
    if (live) {
      for (long e0 = tid; e0 < p.vocab; e0 += 8 * 1024) {
        float x[8]; float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; j++) { x[j] = e0 + j * 1024 < p.vocab ? to_f32(row[e0 + j * 1024]) : -INFINITY; m = fmaxf(m, x[j]); }
        const float ref = m == -INFINITY ? 0.f : m; float s = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) s += ex2((x[j] - ref) * c);
        v = join(v, MaxSum{m, s}, c);
      }
      if (warp == 0) { const Teacher t = teacher_row<T>(p, r, row, c, lane, true, ids, prob, stud, true); if (lane == 0) teach = t; }
    } else if (tid == 0) teach = Teacher{};
    v = warp_join(v, c);
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = warp_join(part[lane], c);
    const Norm n = norm_of(v); const Teacher t = teach; const bool on = live && t.some;
    if (tid == 0) p.loss[r] = distill_loss(t, n, p.temperature, w, on);
    if constexpr (GRAD) {
      T* out = static_cast<T*>(p.dlogits) + r * p.dstride;
      for (long e = tid; e < p.vocab; e += 1024) out[e] = from_f32<T>(on ? w * p.temperature * ex2((to_f32(row[e]) - n.m) * c - n.l) : 0.f);
      __syncthreads();
      if (on)
        for (int e = tid; e < p.top; e += 1024) {
          const int id = ids[e]; if (id < 0) continue;
          float sum = 0.f; bool first = true;
          for (int f = 0; f < p.top; f++) if (ids[f] == id) { if (f < e) { first = false; break; } sum += prob[f]; }
          if (first) out[id] = from_f32<T>(w * p.temperature * (ex2((stud[e] - n.m) * c - n.l) - sum));
        }
    }
    __syncthreads();
  }
}

template <class T, bool GRAD>
inline int distill_launch(gn_ctx* ctx, const DistillParams& p, void* stream) {
  const int sms = ctx->c.sm_count; const DistillPlan pl = distill_plan(p.rows, p.vocab, sms);
  if (pl.cluster == 0) return op_launch("distill_long", stream, distill_long_kernel<T, GRAD>, dim3((unsigned)std::min<int64_t>(p.rows, 2L * sms)), dim3(1024), 0, 0, p);
  // two rows of slots where 16-bit elements leave room for them: 128 KB for 1024 threads either way
  const int buffers = sizeof(T) == 2 ? 2 : 1, smem = buffers * pl.threads * DISTILL_ITEMS * (int)sizeof(T) + (GRAD ? 3 * 12 * p.top : 0);
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>(1024 / pl.threads, 220 * 1024 / (smem + 2048)));
  const dim3 grid((unsigned)(std::min<int64_t>(p.rows, std::max<int64_t>(1, sms * per_sm / pl.cluster)) * pl.cluster));
  auto go = [&](auto kernel) { GN_TRY(op_smem("distill", kernel, smem)); return op_launch("distill", stream, kernel, grid, dim3(pl.threads), smem, pl.cluster, p, pl.cluster, buffers); };
  return pl.threads == 1024 ? go(distill_kernel<T, 1024, GRAD>) : pl.threads == 512 ? go(distill_kernel<T, 512, GRAD>) : pl.threads == 256 ? go(distill_kernel<T, 256, GRAD>) : go(distill_kernel<T, 64, GRAD>);
}

}  // namespace gn

extern "C" int gn_op_distill(gn_ctx* ctx, int dtype, int64_t rows, int64_t vocab, int top, float temperature, const void* logits, int64_t row_stride, const void* top_ids, int index_type, const float* top_logits,
                             const float* weight, float* loss, void* dlogits, int64_t drow_stride, void* stream) {
  using namespace gn;
  GN_OP_BEGIN("op_distill", check_distill(dtype, rows, vocab, top, temperature, logits, row_stride, top_ids, index_type, top_logits, weight, loss, dlogits, drow_stride));
  if (rows == 0) return GN_OK;
  const DistillParams p{logits, (long)row_stride, top_ids, index_type, top_logits, weight, loss, dlogits, (long)drow_stride, (long)rows, (long)vocab, top, temperature};
  return with_type(dtype, [&](auto t) { using T = decltype(t); return dlogits ? distill_launch<T, true>(ctx, p, stream) : distill_launch<T, false>(ctx, p, stream); });
}
