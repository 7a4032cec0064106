// op_distill.cuh -- distillation from a teacher's top logits: loss and gradient from one reading of the student's logits.
//
//   p = softmax(t / T) over a row's entries, q = softmax(s / T) over the vocabulary,
//   loss = w T^2 sum_k p_k (log p_k - log q_{id_k}),      ds = w T (q - p)
//
// All exponentials are of base 2, with c = log2(e) / T: e_j = 2^((s_j - m) c) with m the largest s_j of the thread's own elements, so that no thread waits for
// another before it sums; (m, sum) pairs then meet in shuffles, in shared memory and between the blocks of a cluster, and q_j = e_j 2^((m - M) c) / S.  Differences
// come before the factor: logits at the type's lowest value stay finite.
//
// Bound by memory: a row is read once and its gradient written once.  A row, or a block's part of it, lies in shared memory; every thread copies there, sums over and writes back its own
// 16-byte pieces of it, so that the only barrier of a row is the one at which the warps' sums meet, and the copies of a thread's next row are under way as soon as it has written this one.
// Blocks of an SM (three for rows of 64 KB) overlap each other's phases.  A row of more than 104 KB (distill_plan has the rule) is spread over a cluster of blocks, whose barrier is then the cluster's.
// One more warp of every block works on the teacher's few entries, a chain of dependent loads, one row ahead of the others (a launch of its own before this one: 58 of 162 us for 4096 rows of
// 32000 with 64 entries, bf16).  The other warps write q everywhere; that warp writes q - p over it where the teacher has entries, behind the next row's barrier.
// (Rows held as exponentials in registers, 64 elements a thread, which saves one of an element's two exponentials: 121 us without the teacher's part, 102 this way; the special-function units do not
// bound it, leaving all exponentials out saves 12.)
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
// What the teacher's entries of a row come to: l as there, r the student's largest value where the teacher has probability (0 if it has none), d = sum of p ((t - max t) - (s - r)); w: the
// row's weight, 0 where it has no entry of positive probability.
struct Teacher { float l, d, r, w; };
__device__ __forceinline__ Norm norm_of(MaxSum v) { return Norm{v.m, log2f(v.s)}; }

// id (-1: none) and logit of entry k
__device__ __forceinline__ int teacher_entry(const DistillParams& p, long row, int k, float& t) {
  const int64_t id = load_index(p.ids, p.index_type, row * p.top + k);
  const bool there = id >= 0 && id < p.vocab;
  if (!there && id != -1) op_report(OP_BAD_INDEX);
  t = there ? ld(p.top_logits + row * p.top + k) : -INFINITY;
  return there ? (int)id : -1;
}
// One warp.  The entries go through shared memory, where the gradient finds their ids, probabilities and student values again; the student's values are asked for as soon as the ids are there.
// Of entries with the same id the first keeps all of their probability and the others become -1.  They are rare and found by a table: every entry writes its number at its id's place; who
// finds another's number there and not the same id tries a second place; where that is taken too, or the ids are the same, the row is looked through.
struct TeacherRow { int* id; float *prob, *stud; };                  // [top, rounded up to 16] each
struct TeacherSmem {                                                 // rows in turns of three, then what one row needs while it is worked on
  uint8_t* base; int top16;
  __device__ __forceinline__ TeacherRow row(int turn) const { int* id = reinterpret_cast<int*>(base) + turn * 3 * top16; return TeacherRow{id, reinterpret_cast<float*>(id + top16), reinterpret_cast<float*>(id + 2 * top16)}; }
  __device__ __forceinline__ float* logit() const { return reinterpret_cast<float*>(base) + 9 * top16; }
  __device__ __forceinline__ unsigned short* table() const { return reinterpret_cast<unsigned short*>(base + 40 * top16); }
};
template <class T, bool GRAD>
__device__ __forceinline__ Teacher teacher_row(const DistillParams& p, long row, float c, int lane, const TeacherSmem& sm, const TeacherRow& to) {
  const float w = p.weight ? ld(p.weight + row) : 1.f;
  if (w == 0.f) return Teacher{0.f, 0.f, 0.f, 0.f};
  const T* logits = static_cast<const T*>(p.logits) + row * p.stride; float* logit = sm.logit(); unsigned short* table = sm.table();
  float m = -INFINITY;
  for (int k0 = lane; k0 < sm.top16; k0 += 64) {
    int id[2]; float t[2], s[2];
#pragma unroll
    for (int e = 0; e < 2; e++) { id[e] = -2; t[e] = -INFINITY; if (k0 + 32 * e < p.top) id[e] = teacher_entry(p, row, k0 + 32 * e, t[e]); }
#pragma unroll
    for (int e = 0; e < 2; e++) s[e] = id[e] >= 0 ? to_f32(logits[id[e]]) : 0.f;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int k = k0 + 32 * e;
      if (k < sm.top16) { to.id[k] = id[e]; logit[k] = t[e]; to.stud[k] = s[e]; if (GRAD && id[e] >= 0) table[id[e] & (TEACHER_TABLE - 1)] = (unsigned short)k; }
      m = fmaxf(m, t[e]);
    }
  }
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m; float sum = 0.f, r = -INFINITY;
  for (int k = lane; k < p.top; k += 32) {
    const float e = exp2f((logit[k] - ref) * c);
    sum += e; to.prob[k] = e; if (e != 0.f) r = fmaxf(r, to.stud[k]);      // (an entry without weight says nothing, whatever the student has there)
  }
  sum = warp_sum(sum); r = warp_max(r);
  const bool some = sum != 0.f; const float scale = some ? 1.f / sum : 0.f; float d = 0.f;
  if (r == -INFINITY) r = 0.f;
  for (int k = lane; k < p.top; k += 32) { const float e = to.prob[k], pk = e * scale; if (e != 0.f) d += pk * ((logit[k] - ref) - (to.stud[k] - r)); to.prob[k] = pk; }
  if constexpr (GRAD) {
    __syncwarp();
    bool lost = false, look = false;
    for (int k = lane; k < p.top; k += 32) {
      const int i = to.id[k], found = i >= 0 ? table[i & (TEACHER_TABLE - 1)] : k;
      if (found != k) { lost = true; look |= to.id[found] == i; }
    }
    if (__any_sync(0xffffffffu, lost) && !__any_sync(0xffffffffu, look)) {
      auto second = [](int i) { return (unsigned)i * 2654435761u >> 21; };      // (2^32 over the golden ratio: 11 bits)
      unsigned mine = 0;                                             // this lane's entries that lost
      for (int k = lane, j = 0; k < p.top; k += 32, j++) { const int i = to.id[k]; if (i >= 0 && table[i & (TEACHER_TABLE - 1)] != k) mine |= 1u << j; }
      __syncwarp();
      for (int k = lane, j = 0; k < p.top; k += 32, j++) if (mine >> j & 1) table[second(to.id[k])] = (unsigned short)k;
      __syncwarp();
      for (int k = lane, j = 0; k < p.top; k += 32, j++) if (mine >> j & 1) look |= table[second(to.id[k])] != k;
    }
    if (__any_sync(0xffffffffu, look)) {
      // sums for the first of each id, in order; the others become -1 when all have looked
      unsigned gone = 0;
      for (int k = lane, j = 0; k - lane < p.top; k += 32, j++) {
        const int i = k < p.top ? to.id[k] : -1; float pk = 0.f; bool first = true;
        if (i >= 0)
          for (int f = 0; f < sm.top16; f += 4) {
            const int4 o = *reinterpret_cast<const int4*>(to.id + f);
            if (o.x != i && o.y != i && o.z != i && o.w != i) continue;
            const int q[4] = {o.x, o.y, o.z, o.w};
            for (int l = 0; l < 4; l++) if (q[l] == i) { if (f + l < k) first = false; pk += to.prob[f + l]; }
          }
        __syncwarp();
        if (i >= 0 && first) to.prob[k] = pk; else if (i >= 0) gone |= 1u << j;      // (an id's sum is read by nobody behind its first entry)
        __syncwarp();
      }
      for (int k = lane, j = 0; k < p.top; k += 32, j++) if (gone >> j & 1) to.id[k] = -1;
    }
    __syncwarp();
  }
  return Teacher{log2f(sum), warp_sum(d), r, some ? w : 0.f};
}
// w T^2 sum of p (log p - log q), from p = 2^((t - max t) c - l_t) and q = 2^((s - M) c - l), as the p add up to 1
__device__ __forceinline__ float distill_loss(const Teacher& t, Norm n, float tau) { return t.w != 0.f ? t.w * tau * (t.d + (n.m - t.r) + tau * 0.69314718055994531f * (n.l - t.l)) : 0.f; }
// q - p where the teacher has entries of row r, over what is there, for ids in [lo, hi); one warp
template <class T>
__device__ __forceinline__ void distill_entries(const DistillParams& p, long r, const TeacherRow& of, float w, Norm n, float c, long lo, long hi, int lane) {
  if (w == 0.f) return;
  T* out = static_cast<T*>(p.dlogits) + r * p.dstride;
  for (int e = lane; e < p.top; e += 32) { const int id = of.id[e]; if (id >= 0 && id >= lo && id < hi) out[id] = from_f32<T>(w * p.temperature * (ex2((of.stud[e] - n.m) * c - n.l) - of.prob[e])); }
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

// element pairs of a piece
template <class T> __device__ __forceinline__ float2 piece_pair(const uint4& u, int i) {      // i: a constant once unrolled
  if constexpr (sizeof(T) == 4) return i == 0 ? make_float2(__uint_as_float(u.x), __uint_as_float(u.y)) : make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  else return unpack2(i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w, T());
}

// `cl` blocks on a row, `per` 16-byte pieces of it (counted from its 16-byte boundary) for each.  WHOLE: every row and its gradient begin on such a boundary and fill their pieces.
template <class T, bool GRAD, bool WHOLE>
__global__ void __launch_bounds__(DISTILL_THREADS + 32, 3) distill_kernel(const __grid_constant__ DistillParams p, int cl, int per) {
  namespace cg = cooperative_groups;
  constexpr int V = Vec<T>::N;
  extern __shared__ uint4 slots[];                                   // [per], then the teacher's
  // Rows take turns with what their barrier guards, a warp may be a row ahead of another, never two: sums of all warps of the cluster; weights, which are written a row ahead.
  __shared__ MaxSum part[2][8 * DISTILL_THREADS / 32]; __shared__ float weight_of_turn[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x - 32, warps = nt >> 5, vocab = (int)p.vocab;
  const int rank = cl > 1 ? (int)(blockIdx.x % cl) : 0; const long row0 = blockIdx.x / cl, step = gridDim.x / cl;
  const float c = 1.4426950408889634f / p.temperature;
  const int at = rank * per;                                         // this block's pieces: [at, at + per), as far as the row goes
  op_begin();
  if (cl > 1) cg::this_cluster().sync();                             // (all blocks are there before one writes into another)
  auto row_of = [&](long r) { return static_cast<const T*>(p.logits) + r * p.stride; };
  auto lead_of = [&](long r) { return WHOLE ? 0 : row_lead(row_of(r)); };
  auto count = [&](int lead) { return min(per, (lead + vocab + V - 1) / V - at); };      // pieces of this block
  auto weight_of = [&](long r) { return r >= p.rows ? 0.f : p.weight ? ld(p.weight + r) : 1.f; };
  // copies of this thread's pieces of row r; pieces that the row does not fill are put together element by element, -inf where it has none
  const uint32_t slot0 = (uint32_t)__cvta_generic_to_shared(slots);
  auto fetch = [&](long r, float w) {
    if (w != 0.f) {
      const T* row = row_of(r); const int lead = lead_of(r), n = count(lead);
      for (int i = tid; i < n; i += nt) {
        const int e = (at + i) * V - lead;                           // first element
        if (WHOLE || (e >= 0 && e + V <= vocab)) cp16(slot0 + i * 16, row + e);
        else {
          T* q = reinterpret_cast<T*>(slots + i);
#pragma unroll
          for (int l = 0; l < V; l++) q[l] = e + l >= 0 && e + l < vocab ? row[e + l] : from_f32<T>(-INFINITY);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  auto barrier = [&]() { if (cl == 1) __syncthreads(); else cg::this_cluster().sync(); };
  auto reduce = [&](MaxSum v) {
    const float top = warp_max(v.m), to = top == -INFINITY ? 0.f : top;
    return MaxSum{top, warp_sum(v.s * ex2((v.m - to) * c))};
  };
  auto meet = [&](int turn) {                                        // behind the barrier: all warps' sums
    MaxSum v{-INFINITY, 0.f};
    for (int k = lane; k < cl * warps; k += 32) v = join(v, part[turn][k], c);
    return norm_of(reduce(v));
  };
  if (warp == warps) {                                               // the teacher's warp
    const TeacherSmem sm{reinterpret_cast<uint8_t*>(slots + per), (p.top + 15) & ~15};
    auto bounds = [&](long r, long& lo, long& hi) { lo = (long)at * V - lead_of(r); hi = lo + (long)per * V; };
    Teacher now = teacher_row<T, GRAD>(p, row0, c, lane, sm, sm.row(0)); int three = 0, turn = 0; long done = -1; float done_w = 0.f; Norm done_n{0.f, 0.f};
    if (lane == 0) weight_of_turn[0] = now.w;
    for (long r = row0; r < p.rows; r += step, turn ^= 1) {
      const int next = three == 2 ? 0 : three + 1, last = three == 0 ? 2 : three - 1;
      Teacher then{0.f, 0.f, 0.f, 0.f};
      if (r + step < p.rows) { then = teacher_row<T, GRAD>(p, r + step, c, lane, sm, sm.row(next)); if (lane == 0) weight_of_turn[next] = then.w; }
      __syncwarp();
      barrier();
      const Norm nm = meet(turn);
      if (lane == 0 && rank == 0) p.loss[r] = distill_loss(now, nm, p.temperature);
      if constexpr (GRAD) { if (done >= 0) { long lo, hi; bounds(done, lo, hi); distill_entries<T>(p, done, sm.row(last), done_w, done_n, c, lo, hi, lane); } }
      done = r; done_w = now.w; done_n = nm; now = then; three = next;
    }
    if constexpr (GRAD) {
      __syncthreads();
      long lo, hi; bounds(done, lo, hi); distill_entries<T>(p, done, sm.row(three == 0 ? 2 : three - 1), done_w, done_n, c, lo, hi, lane);
    }
    if (cl > 1) cg::this_cluster().sync();
    return;
  }

  float w_now = weight_of(row0); fetch(row0, w_now);
  int turn = 0, three = 0;
  for (long r = row0; r < p.rows; r += step, turn ^= 1) {
    const float w_next = weight_of(r + step); const int lead = lead_of(r), n = count(lead);
    asm volatile("cp.async.wait_all;" ::: "memory");
    float m = -INFINITY, s = 0.f;
    if (w_now != 0.f) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int i = tid; i < n; i += nt) {
        const uint4 u = slots[i];
        const float top = fmaxf(m, piece_max<T>(u));
        if (top > m) { const float g = ex2((m - top) * c); sum = mul2(sum, make_float2(g, g)); m = top; }      // (rarely behind the first pieces)
        const float ref = m == -INFINITY ? 0.f : m; const float2 r2 = make_float2(-ref, -ref), c2 = make_float2(c, c);
#pragma unroll
        for (int l = 0; l < V / 2; l++) { const float2 x = mul2(add2(piece_pair<T>(u, l), r2), c2); sum = add2(sum, make_float2(ex2(x.x), ex2(x.y))); }
      }
      s = sum.x + sum.y;
    }
    const MaxSum v = reduce(MaxSum{m, s});
    if (cl == 1) { if (lane == 0) part[turn][warp] = v; }
    else if (lane < cl) *cg::this_cluster().map_shared_rank(&part[turn][rank * warps + warp], lane) = v;
    __syncwarp();
    barrier();
    if constexpr (GRAD) {
      const Norm nm = meet(turn); const float f = weight_of_turn[three] * p.temperature; const bool on = f != 0.f;
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
#pragma unroll 1
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
    if (++three == 3) three = 0;
  }
  if constexpr (GRAD) __syncthreads();                               // (the last row is written)
  if (cl > 1) cg::this_cluster().sync();                             // (no block leaves while another may still write into it)
}

// A row that does not fit on chip: one block reads it twice.
template <class T, bool GRAD>
__global__ void __launch_bounds__(1024) distill_long_kernel(const __grid_constant__ DistillParams p) {
  op_begin();
  extern __shared__ uint4 slots[];
  __shared__ MaxSum part[32]; __shared__ Teacher teach;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5; const float c = 1.4426950408889634f / p.temperature;
  const TeacherSmem sm{reinterpret_cast<uint8_t*>(slots), (p.top + 15) & ~15};
  for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* row = static_cast<const T*>(p.logits) + r * p.stride;
    MaxSum v{-INFINITY, 0.f};
    if (warp == 0) { const Teacher t = teacher_row<T, GRAD>(p, r, c, lane, sm, sm.row(0)); if (lane == 0) teach = t; }
    if ((p.weight ? ld(p.weight + r) : 1.f) != 0.f)
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
    const Norm n = norm_of(warp_join(part[lane], c)); const Teacher t = teach; const bool on = t.w != 0.f;
    if (tid == 0) p.loss[r] = distill_loss(t, n, p.temperature);
    if constexpr (GRAD) {
      T* out = static_cast<T*>(p.dlogits) + r * p.dstride;
      for (long e = tid; e < p.vocab; e += 1024) out[e] = from_f32<T>(on ? t.w * p.temperature * ex2((to_f32(row[e]) - n.m) * c - n.l) : 0.f);
      __syncthreads();
      if (warp == 0) distill_entries<T>(p, r, sm.row(0), t.w, n, c, 0, p.vocab, lane);
    }
    __syncthreads();
  }
}

template <class T, bool GRAD>
inline int distill_launch(gn_ctx* ctx, const DistillParams& p, void* stream) {
  const int sms = ctx->c.sm_count; const DistillPlan pl = distill_plan(p.rows, p.vocab, (int)sizeof(T), sms, p.top);
  const int tsmem = teacher_smem(p.top);
  if (pl.cluster == 0) return op_launch("distill_long", stream, distill_long_kernel<T, GRAD>, dim3((unsigned)std::min<int64_t>(p.rows, 2L * sms)), dim3(1024), tsmem, 0, p);
  constexpr int V = Vec<T>::N;
  const bool whole = p.vocab % V == 0 && p.stride % V == 0 && aligned_to(p.logits, 16) && (!GRAD || (p.dstride % V == 0 && aligned_to(p.dlogits, 16)));
  const int smem = pl.per * 16 + tsmem; const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>({2048 / (pl.threads + 32), 32, 65536 / (40 * (pl.threads + 32)), DISTILL_SM_SMEM / (smem + DISTILL_FIXED)}));
  const dim3 grid((unsigned)(std::min<int64_t>(p.rows, std::max<int64_t>(1, (int64_t)sms * per_sm / pl.cluster)) * pl.cluster));
  auto go = [&](auto kernel) { if (smem > 40 * 1024) GN_TRY(op_smem("distill", kernel, DISTILL_SMEM_MOST)); return op_launch("distill", stream, kernel, grid, dim3(pl.threads + 32), smem, pl.cluster, p, pl.cluster, pl.per); };
  return whole ? go(distill_kernel<T, GRAD, true>) : go(distill_kernel<T, GRAD, false>);
}

}  // namespace gn

extern "C" {

int gn_op_distill(gn_ctx* ctx, int dtype, int64_t rows, int64_t vocab, int top, float temperature, const void* logits, int64_t row_stride, const void* top_ids, int index_type, const float* top_logits,
                  const float* weight, float* loss, void* dlogits, int64_t drow_stride, void* stream) {
  using namespace gn;
  GN_OP_BEGIN("op_distill", check_distill(dtype, rows, vocab, top, temperature, logits, row_stride, top_ids, index_type, top_logits, weight, loss, dlogits, drow_stride));
  if (rows == 0) return GN_OK;
  const DistillParams p{logits, (long)row_stride, top_ids, index_type, top_logits, weight, loss, dlogits, (long)drow_stride, (long)rows, (long)vocab, top, temperature};
  return with_type(dtype, [&](auto t) { using T = decltype(t); return dlogits ? distill_launch<T, true>(ctx, p, stream) : distill_launch<T, false>(ctx, p, stream); });
}

}  // extern "C"
