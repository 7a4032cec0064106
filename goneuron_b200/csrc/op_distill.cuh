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
// row waits for their chain of dependent loads; the second streams the rows.  A row, or a block's part of it, lies in shared memory; every thread copies there, sums over and writes back its own
// 16-byte pieces of it, so that the only barrier of a row is the one at which the warps' sums meet, and the copies of a thread's next row are under way as soon as it has written this one.
// Blocks of an SM (three for rows of 64 KB) overlap each other's phases.  (Rows held as exponentials in registers, 1024 threads a row: 26 instructions an element, most of them per row
// and thread, 2.4 TB/s.)  A row of more than 72 KB is spread over a cluster of blocks, whose barrier is then the cluster's.
// Each block writes q for all of its elements; where the teacher has entries q - p is written over it, behind the next row's barrier.
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
// A warp a row, 128 entries of it at a time in registers.  With a gradient the entries' ids, probabilities and student values are kept for the second launch; of entries with the same id the
// first keeps all of their probability and the others become -1.  Such entries are rare and found by a table: every entry writes its number at its id's place, and whoever finds
// another's number there, or is found by another of the same id, looks through the row.
constexpr int TEACHER_WARPS = 4, TEACHER_TABLE = 2048;
inline int teacher_smem(int top) { return TEACHER_WARPS * (TEACHER_TABLE * 2 + (top + 15) / 16 * 16 * 9); }      // table, ids, probabilities, flags
template <class T, bool GRAD>
__global__ void __launch_bounds__(32 * TEACHER_WARPS) distill_teacher_kernel(const __grid_constant__ DistillParams p) {
  pdl_wait(); pdl_launch();                                          // (in this order: the launch behind fetches logits before this one has finished)
  extern __shared__ uint4 teacher_smem_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, top16 = (p.top + 15) & ~15; const float c = 1.4426950408889634f / p.temperature;
  uint8_t* own = reinterpret_cast<uint8_t*>(teacher_smem_raw) + warp * (TEACHER_TABLE * 2 + top16 * 9);
  int* id_of = reinterpret_cast<int*>(own); float* prob_of = reinterpret_cast<float*>(id_of + top16);
  unsigned short* table = reinterpret_cast<unsigned short*>(prob_of + top16); uint8_t* look = reinterpret_cast<uint8_t*>(table + TEACHER_TABLE);
  const long row = (long)blockIdx.x * TEACHER_WARPS + warp;
  if (row >= p.rows) return;
  const float w = p.weight ? __ldg(p.weight + row) : 1.f;
  Teacher out{0.f, 0.f, 0.f, 0.f};
  if (w != 0.f) {
    const T* logits = static_cast<const T*>(p.logits) + row * p.stride;
    constexpr int E = 4;
    int id[E]; float t[E];
    auto load = [&](int k0) {
#pragma unroll
      for (int e = 0; e < E; e++) { const int k = k0 + 32 * e + lane; id[e] = -1; t[e] = -INFINITY; if (k < p.top) id[e] = teacher_entry(p, row, k, t[e]); }
    };
    MaxSum v{-INFINITY, 0.f};
    for (int k0 = 0; k0 < p.top; k0 += 32 * E) {
      load(k0);
#pragma unroll
      for (int e = 0; e < E; e++) v = join(v, MaxSum{t[e], t[e] == -INFINITY ? 0.f : 1.f}, c);
    }
    v = warp_join(v, c);
    const bool some = !(v.m == -INFINITY && v.s == 0.f); const Norm n = norm_of(v);
    float d = 0.f, r = -INFINITY, weight = 0.f;                      // d: relative to this lane's r so far; weight: the probability that it holds
    for (int k0 = 0; k0 < p.top; k0 += 32 * E) {
      if (p.top > 32 * E) load(k0);
      float s[E];
#pragma unroll
      for (int e = 0; e < E; e++) s[e] = id[e] >= 0 ? to_f32(logits[id[e]]) : 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int k = k0 + 32 * e + lane;
        const float pk = !some || t[e] == -INFINITY ? 0.f : exp2f((t[e] - n.m) * c - n.l);
        if (pk != 0.f) {                                             // (an entry without weight says nothing, whatever the student has there)
          if (s[e] > r) { if (weight != 0.f) d += weight * (s[e] - r); r = s[e]; }      // sum of p (r - s) moves with r
          d += pk * ((t[e] - n.m) - (s[e] - (r == -INFINITY ? 0.f : r))); weight += pk;
        }
        if constexpr (GRAD) {
          if (k < top16) { id_of[k] = k < p.top ? id[e] : -2; prob_of[k] = pk; look[k] = 0; }
          if (k < p.top) { p.stud[row * p.top + k] = s[e]; if (id[e] >= 0) table[id[e] & (TEACHER_TABLE - 1)] = (unsigned short)k; }
        }
      }
    }
    const float top = warp_max(r), ref = top == -INFINITY ? 0.f : top;
    if (weight != 0.f) d += weight * (ref - (r == -INFINITY ? 0.f : r));
    out = Teacher{n.l, warp_sum(d), ref, some ? w : 0.f};
    if constexpr (GRAD) {
      __syncwarp();
      for (int k = lane; k < p.top; k += 32) {
        const int i = id_of[k];
        if (i < 0) continue;
        const int found = table[i & (TEACHER_TABLE - 1)];
        if (found != k) { look[k] = 1; if (id_of[found] == i) look[found] = 1; }
      }
      __syncwarp();
      for (int k = lane; k < p.top; k += 32) {
        int i = id_of[k]; float pk = prob_of[k];
        if (look[k]) {
          const int mine = i; pk = 0.f;
          for (int f = 0; f < top16; f += 4) {
            const int4 o = *reinterpret_cast<const int4*>(id_of + f);
            if (o.x != mine && o.y != mine && o.z != mine && o.w != mine) continue;
            const int q[4] = {o.x, o.y, o.z, o.w};
            for (int l = 0; l < 4; l++) if (q[l] == mine) { if (f + l < k) i = -1; pk += prob_of[f + l]; }
          }
        }
        p.id[row * p.top + k] = i; p.prob[row * p.top + k] = pk;
      }
    }
  }
  if (lane == 0) p.teach[row] = out;
}
// w T^2 sum of p (log p - log q), from p = 2^((t - max t) c - l_t) and q = 2^((s - M) c - l), as the p add up to 1
__device__ __forceinline__ float distill_loss(const Teacher& t, Norm n, float tau) { return t.w != 0.f ? t.w * tau * (t.d + (n.m - t.r) + tau * 0.69314718055994531f * (n.l - t.l)) : 0.f; }
// q - p where the teacher has entries of row r, over what is there, for ids in [lo, hi)
template <class T>
__device__ __forceinline__ void distill_entry(const DistillParams& p, T* out, int id, float prob, float stud, float w, Norm n, float c, long lo, long hi) {
  if (id >= 0 && id >= lo && id < hi) out[id] = from_f32<T>(w * p.temperature * (ex2((stud - n.m) * c - n.l) - prob));
}
template <class T>
__device__ __forceinline__ void distill_entries(const DistillParams& p, long r, int first, float w, Norm n, float c, long lo, long hi) {
  T* out = static_cast<T*>(p.dlogits) + r * p.dstride;
  for (int e = first + threadIdx.x; e < p.top; e += blockDim.x) { const long i = r * p.top + e; distill_entry<T>(p, out, p.id[i], p.prob[i], p.stud[i], w, n, c, lo, hi); }
}

// Elements of a row from the 16-byte boundary at or before its first one.
template <class T> __device__ __forceinline__ int row_lead(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
// Largest element of a piece (a NaN counts as none)
template <class T> __device__ __forceinline__ float piece_max(const uint4& u) {
  if constexpr (sizeof(T) == 4) return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto as = [](uint32_t v) { return *reinterpret_cast<const T2*>(&v); };
    const T2 m = __hmax2(__hmax2(as(u.x), as(u.y)), __hmax2(as(u.z), as(u.w)));
    return fmaxf(to_f32(m.x), to_f32(m.y));
  }
}

// two floats an instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r; asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y)); return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r; asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y)); return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r; asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y)); return r;
}
// element pairs of a piece
template <class T> __device__ __forceinline__ float2 piece_pair(const uint4& u, int i) {      // i: a constant once unrolled
  if constexpr (sizeof(T) == 4) return i == 0 ? make_float2(__uint_as_float(u.x), __uint_as_float(u.y)) : make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  else return unpack2(i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w, T());
}

// `cl` blocks on a row, `per` 16-byte pieces of it (counted from its 16-byte boundary) for each.  WHOLE: every row and its gradient begin on such a boundary and fill their pieces.
template <class T, bool GRAD, bool WHOLE>
__global__ void __launch_bounds__(DISTILL_THREADS, 3) distill_kernel(const __grid_constant__ DistillParams p, int cl, int per) {
  namespace cg = cooperative_groups;
  constexpr int V = Vec<T>::N;
  extern __shared__ uint4 slots[];                                   // [per], rounded up to whole turns of all threads: -inf behind
  __shared__ MaxSum part[2][8 * DISTILL_THREADS / 32];               // sums of all warps of the cluster (rows take turns: a warp may be a row ahead of another, never two)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x, warps = nt >> 5, vocab = (int)p.vocab;
  const int rank = cl > 1 ? (int)(blockIdx.x % cl) : 0; const long row0 = blockIdx.x / cl, step = gridDim.x / cl;
  const float c = 1.4426950408889634f / p.temperature;
  const int at = rank * per;                                         // this block's pieces: [at, at + per), as far as the row goes
  pdl_launch();
  if (cl > 1) cg::this_cluster().sync();                             // (all blocks are there before one writes into another)
  auto row_of = [&](long r) { return static_cast<const T*>(p.logits) + r * p.stride; };
  auto lead_of = [&](long r) { return WHOLE ? 0 : row_lead(row_of(r)); };
  auto count = [&](int lead) { return min(per, (lead + vocab + V - 1) / V - at); };      // pieces of this block
  const int n_whole = (per + nt - 1) / nt * nt;                      // places of all threads' turns
  auto weight_of = [&](long r) { return r >= p.rows ? 0.f : p.weight ? __ldg(p.weight + r) : 1.f; };
  // copies of this thread's pieces of row r; pieces that the row does not fill are put together element by element, -inf where it has none
  const uint32_t slot0 = (uint32_t)__cvta_generic_to_shared(slots), none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  const uint4 nothing = make_uint4(none, none, none, none);          // -inf
  auto fetch = [&](long r, float w) {
    if (w != 0.f) {
      const T* row = row_of(r); const int lead = lead_of(r), n = count(lead);
      for (int i = tid; i < (WHOLE ? n : n_whole); i += nt) {        // (WHOLE: what lies behind is the same for every row)
        const int e = (at + i) * V - lead;                           // first element
        if (!WHOLE && i >= n) slots[i] = nothing;
        else if (WHOLE || (e >= 0 && e + V <= vocab)) cp16(slot0 + i * 16, row + e);
        else {
          T* q = reinterpret_cast<T*>(slots + i);
#pragma unroll
          for (int l = 0; l < V; l++) q[l] = e + l >= 0 && e + l < vocab ? row[e + l] : from_f32<T>(-INFINITY);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  if (WHOLE) for (int i = tid; i < n_whole; i += nt) if (i >= count(0)) slots[i] = nothing;
  float w_now = weight_of(row0); fetch(row0, w_now);
  pdl_wait();                                                        // for the teacher's launch
  int turn = 0; long done = -1; float done_w = 0.f; Norm done_n{0.f, 0.f};
  for (long r = row0; r < p.rows; r += step, turn ^= 1) {
    const Teacher t = p.teach[r]; const float w_next = weight_of(r + step); const int lead = lead_of(r), n = count(lead); const bool on = t.w != 0.f;
    // the entries of the row before, one a thread
    int id = -1; float prob = 0.f, stud = 0.f;
    if constexpr (GRAD) { if (done_w != 0.f && tid < p.top) { const long i = done * p.top + tid; id = p.id[i]; prob = p.prob[i]; stud = p.stud[i]; } }
    asm volatile("cp.async.wait_all;" ::: "memory");
    float m = -INFINITY, s = 0.f;
    if (w_now != 0.f) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll 2
      for (int i = tid; i < n_whole; i += nt) {
        const uint4 u = slots[i];
        const float top = fmaxf(m, piece_max<T>(u));
        if (top > m) { const float g = ex2((m - top) * c); sum = mul2(sum, make_float2(g, g)); m = top; }      // (rarely behind the first pieces)
        const float ref = m == -INFINITY ? 0.f : m; const float2 r2 = make_float2(-ref, -ref), c2 = make_float2(c, c);
#pragma unroll
        for (int l = 0; l < V / 2; l++) { const float2 x = mul2(add2(piece_pair<T>(u, l), r2), c2); sum = add2(sum, make_float2(ex2(x.x), ex2(x.y))); }
      }
      s = sum.x + sum.y;
    }
    auto meet = [&](MaxSum v) {
      const float top = warp_max(v.m), to = top == -INFINITY ? 0.f : top;
      return MaxSum{top, warp_sum(v.s * ex2((v.m - to) * c))};
    };
    MaxSum v = meet(MaxSum{m, s});
    if (cl == 1) {
      if (lane == 0) part[turn][warp] = v;
      __syncthreads();
    } else {
      cg::cluster_group cluster = cg::this_cluster();
      if (lane < cl) *cluster.map_shared_rank(&part[turn][rank * warps + warp], lane) = v;
      cluster.sync();
    }
    v = MaxSum{-INFINITY, 0.f};
    for (int k = lane; k < cl * warps; k += 32) v = join(v, part[turn][k], c);
    const Norm nm = norm_of(meet(v));
    if (tid == 0 && rank == 0) p.loss[r] = distill_loss(t, nm, p.temperature);
    if constexpr (GRAD) {
      const float f = t.w * p.temperature;
      T* out = static_cast<T*>(p.dlogits) + r * p.dstride; const bool same = WHOLE || row_lead(out) == lead;
      auto put = [&](int i, const float (&y)[V]) {
        const int e = (at + i) * V - lead;
        if (WHOLE || (same && e >= 0 && e + V <= vocab)) *reinterpret_cast<uint4*>(out + e) = pack<T>(y);
        else {
#pragma unroll
          for (int l = 0; l < V; l++) if (e + l >= 0 && e + l < vocab) out[e + l] = from_f32<T>(y[l]);
        }
      };
      if (on) {
        const float2 m2 = make_float2(-nm.m, -nm.m), c2 = make_float2(c, c), l2 = make_float2(-nm.l, -nm.l), f2 = make_float2(f, f);
#pragma unroll 2
        for (int i = tid; i < n; i += nt) {
          const uint4 u = slots[i]; float y[V];
#pragma unroll
          for (int l = 0; l < V / 2; l++) { const float2 x = fma2(add2(piece_pair<T>(u, l), m2), c2, l2), q = mul2(make_float2(ex2(x.x), ex2(x.y)), f2); y[2 * l] = q.x; y[2 * l + 1] = q.y; }
          put(i, y);
        }
      } else {
        float y[V] = {};
        for (int i = tid; i < n; i += nt) put(i, y);
      }
    }
    fetch(r + step, w_next);                                         // (this thread has read its pieces)
    w_now = w_next;
    if constexpr (GRAD) {
      if (done_w != 0.f) {
        const long lo = (long)at * V - lead_of(done);
        distill_entry<T>(p, static_cast<T*>(p.dlogits) + done * p.dstride, id, prob, stud, done_w, done_n, c, lo, lo + (long)per * V);
        distill_entries<T>(p, done, nt, done_w, done_n, c, lo, lo + (long)per * V);
      }
      done = r; done_w = t.w; done_n = nm;
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    if (done_w != 0.f) { const long lo = (long)at * V - lead_of(done); distill_entries<T>(p, done, 0, done_w, done_n, c, lo, lo + (long)per * V); }
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
      if (on) distill_entries<T>(p, r, 0, t.w, n, c, 0, p.vocab);
    }
    __syncthreads();
  }
}

template <class T, bool GRAD>
inline int distill_launch(gn_ctx* ctx, const DistillParams& p, void* stream) {
  const int sms = ctx->c.sm_count; const DistillPlan pl = distill_plan(p.rows, p.vocab, (int)sizeof(T), sms);
  const int tsmem = teacher_smem(GRAD ? p.top : 0);
  if (tsmem > 48 * 1024) GN_TRY(op_smem("distill_teacher", distill_teacher_kernel<T, GRAD>, tsmem));
  GN_TRY(op_launch("distill_teacher", stream, distill_teacher_kernel<T, GRAD>, dim3(cdiv(p.rows, TEACHER_WARPS)), dim3(32 * TEACHER_WARPS), tsmem, 0, p));
  if (pl.cluster == 0) return op_launch("distill_long", stream, distill_long_kernel<T, GRAD>, dim3((unsigned)std::min<int64_t>(p.rows, 2L * sms)), dim3(1024), 0, 0, p);
  constexpr int V = Vec<T>::N;
  const bool whole = p.vocab % V == 0 && p.stride % V == 0 && aligned_to(p.logits, 16) && (!GRAD || (p.dstride % V == 0 && aligned_to(p.dlogits, 16)));
  const int smem = (int)round_up(pl.per, pl.threads) * 16;
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>({2048 / pl.threads, 32, 220 * 1024 / (smem + 3 * 1024)}));
  const dim3 grid((unsigned)(std::min<int64_t>(p.rows, std::max<int64_t>(1, (int64_t)sms * per_sm / pl.cluster)) * pl.cluster));
  auto go = [&](auto kernel) { if (smem > 40 * 1024) GN_TRY(op_smem("distill", kernel, smem)); return op_launch("distill", stream, kernel, grid, dim3(pl.threads), smem, pl.cluster, p, pl.cluster, pl.per); };
  return whole ? go(distill_kernel<T, GRAD, true>) : go(distill_kernel<T, GRAD, false>);
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
