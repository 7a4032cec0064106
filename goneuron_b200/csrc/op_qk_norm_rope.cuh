// op_qk_norm_rope.cuh -- norm of queries and keys per head with the position rotation in the same pass, and its gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = R (g x r);     u = R^T dy,  dx = r (g u - x r^2 mean(g u x)),  dg = sum u x r
//
// R turns pairs of elements by position * frequency.  The angle is formed in 64 bits, as a fraction of a turn, so that
// a far position costs no accuracy; sine and cosine of what is left are float32, once per token and pair for all heads, in shared memory.
// Everything between reading x (and dy) and the one rounding of the result is float32.
//
// Bound by memory: a row is read once and written once.  A lane holds two pieces of a row, of 16 bytes (or 8: 32768 tokens of 16 + 4 heads of 80, 40 of them rotated, bf16: 81 us forward and 131
// backward, element by element 643 and 1310, then with 8 warps an SM), the two halves of its pairs, so that a rotation stays
// within the lane and the sums over a row are shuffles among its 2 to 32 lanes.
#pragma once
#include "device_ops.cuh"

namespace gn {

struct QkHeads { const void* in; const void* dy; void* out; long in_t, in_h, dy_t, dy_h, out_t, out_h; int heads, per_block; const float* gain; };      // per_block: tokens of a block at a time
struct QkParams {
  QkHeads t[2]; long tokens; int head, rot, inter; float eps; const void* pos; int index_type; const double* freq; float* partial;
};

// Frequencies in turns, as 64-bit fractions of one: a position times that, in wrapping arithmetic, drops whole turns without a rounding.  (The product and the whole turns in float64 for every token
// and pair were a fifth of the forward pass's time.)
__device__ __forceinline__ void qk_frequencies(const QkParams& p, unsigned long long* fx) {
  for (int i = threadIdx.x; i < p.rot >> 1; i += blockDim.x) {
    double f = ld(p.freq + i) * 0.15915494309189533577;           // 1 / (2 pi)
    f -= floor(f);
    fx[i] = (unsigned long long)(f * 18446744073709551616.0);
  }
}
// cosines and sines of the angles of n tokens from `base` on: per token the cosines of all pairs, then the sines
__device__ __forceinline__ void qk_turns(const QkParams& p, long base, int n, const unsigned long long* fx, float* cs) {
  const int half = p.rot >> 1;
  for (int e = threadIdx.x; e < n * half; e += blockDim.x) {
    const int t = e / half, i = e - t * half;
    const int turn = (int)((unsigned long long)load_index(p.pos, p.index_type, base + t) * fx[i] >> 32);      // of 2^32, from half a turn back to half a turn on
    float s, c; sincospif((float)turn * 4.656612873077392578125e-10f, &s, &c);      // 2^-31
    cs[t * p.rot + i] = c; cs[t * p.rot + half + i] = s;
  }
}
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) { const float u = a * c - b * s; b = a * s + b * c; a = u; }

// A lane's two pieces of a row: the halves of its pairs, or two neighbours behind the rotated part (interleaved: two neighbours everywhere), with the cosines and sines of
// their pairs and the gain of their elements.  The same for all heads of a token, so that they stay in registers while a lane goes through several of them.
// V: elements of a piece, of 16 or 8 bytes.  FULL: halves are rotated, all of a row, and the lanes of a group are exactly a row's, so that nothing needs asking.  Arithmetic goes two elements an instruction.
template <class T, int V, bool FULL> struct QkLane {
  static constexpr int P = V / 2;
  using Piece = typename std::conditional<V * sizeof(T) == 16, uint4, uint2>::type;
  int pa, pb; bool has_a, has_b, split;
  float2 ga[P], gb[P], c[P], s[P];                                   // cosines and sines of pairs 2 j, 2 j + 1
  __device__ __forceinline__ QkLane(const QkParams& p, int slot) {
    const int pieces = p.head / V, turned = (p.rot >> 1) / V;
    split = FULL || (!p.inter && slot < turned);
    pa = split ? slot : 2 * slot; pb = split ? slot + turned : 2 * slot + 1;
    has_a = FULL || pa < pieces; has_b = FULL || pb < pieces;
  }
  __device__ __forceinline__ void gain(const float* g) {
    auto at = [&](bool has, int e) { return g && has ? ld(reinterpret_cast<const float2*>(g + e)) : make_float2(1.f, 1.f); };
    if (reinterpret_cast<uintptr_t>(g) & 7) {                        // (a gain need only be aligned to its type)
#pragma unroll
      for (int j = 0; j < P; j++) {
        ga[j] = has_a ? make_float2(ld(g + pa * V + 2 * j), ld(g + pa * V + 2 * j + 1)) : make_float2(1.f, 1.f);
        gb[j] = has_b ? make_float2(ld(g + pb * V + 2 * j), ld(g + pb * V + 2 * j + 1)) : make_float2(1.f, 1.f);
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < P; j++) { ga[j] = at(has_a, pa * V + 2 * j); gb[j] = at(has_b, pb * V + 2 * j); }
  }
  __device__ __forceinline__ void turns(const QkParams& p, const float* cs, float sign) {      // cs: the token's
    const int half = p.rot >> 1;
    if (split) {
#pragma unroll
      for (int j = 0; j < P; j += 2) {
        const float4 u = *reinterpret_cast<const float4*>(cs + pa * V + 2 * j), w = *reinterpret_cast<const float4*>(cs + half + pa * V + 2 * j);
        c[j] = make_float2(u.x, u.y); c[j + 1] = make_float2(u.z, u.w); s[j] = make_float2(sign * w.x, sign * w.y); s[j + 1] = make_float2(sign * w.z, sign * w.w);
      }
    } else if (p.inter) {
      auto at = [&](int j) { const int i = (j < P ? pa : pb) * P + j % P; return i < half ? make_float2(cs[i], sign * cs[half + i]) : make_float2(1.f, 0.f); };
#pragma unroll
      for (int j = 0; j < P; j++) { const float2 u = at(2 * j), w = at(2 * j + 1); c[j] = make_float2(u.x, w.x); s[j] = make_float2(u.y, w.y); }
    }
  }
  __device__ __forceinline__ void turn(const QkParams& p, float2 (&a)[P], float2 (&b)[P]) const {
    if (split) {
#pragma unroll
      for (int j = 0; j < P; j++) { const float2 n = make_float2(-s[j].x, -s[j].y), u = fma2(b[j], n, mul2(a[j], c[j])); b[j] = fma2(b[j], c[j], mul2(a[j], s[j])); a[j] = u; }
    } else if (p.inter) {                                            // (elements that do not turn are left alone: 0 times an infinity is none)
#pragma unroll
      for (int j = 0; j < P; j++) {
        if (pa * V + 2 * j < p.rot) rotate(a[j].x, a[j].y, j & 1 ? c[j / 2].y : c[j / 2].x, j & 1 ? s[j / 2].y : s[j / 2].x);
        if (pb * V + 2 * j < p.rot) rotate(b[j].x, b[j].y, (P + j) & 1 ? c[(P + j) / 2].y : c[(P + j) / 2].x, (P + j) & 1 ? s[(P + j) / 2].y : s[(P + j) / 2].x);
      }
    }
  }
  __device__ __forceinline__ void load(const void* row, Piece& a, Piece& b) const {
    a = Piece{}; b = a;
    if (has_a) a = reinterpret_cast<const Piece*>(row)[pa];
    if (has_b) b = reinterpret_cast<const Piece*>(row)[pb];
  }
  __device__ __forceinline__ static void open(const Piece& u, float2 (&v)[P]) {
    if constexpr (sizeof(Piece) == 8) { v[0] = unpack2(u.x, T()); v[1] = unpack2(u.y, T()); }
    else {
      float x[V]; unpack<T>(u, x);
#pragma unroll
      for (int j = 0; j < P; j++) v[j] = make_float2(x[2 * j], x[2 * j + 1]);
    }
  }
  __device__ __forceinline__ static Piece shut(const float2 (&v)[P]) {
    if constexpr (sizeof(Piece) == 8) return make_uint2(pack2(v[0].x, v[0].y, T()), pack2(v[1].x, v[1].y, T()));
    else {
      float x[V];
#pragma unroll
      for (int j = 0; j < P; j++) { x[2 * j] = v[j].x; x[2 * j + 1] = v[j].y; }
      return pack<T>(x);
    }
  }
  __device__ __forceinline__ void store(void* row, const float2 (&a)[P], const float2 (&b)[P]) const {
    if (has_a) reinterpret_cast<Piece*>(row)[pa] = shut(a);
    if (has_b) reinterpret_cast<Piece*>(row)[pb] = shut(b);
  }
};

constexpr int QK_THREADS = 256;
// A group of G lanes takes HB heads of one token at a time.  (One head at a time, with the cosines read from shared memory for each: 129 us forward and 236 backward for 65536 tokens of 16 + 4 heads of
// 64, bf16; one element an instruction: 79 and 131.)
template <class T, int V, int G, bool BWD, bool FULL>
__global__ void __launch_bounds__(QK_THREADS, QK_PER_SM) qk_vec_kernel(const __grid_constant__ QkParams p) {
  using Lane = QkLane<T, V, FULL>; using Piece = typename Lane::Piece;
  constexpr int P = V / 2, GROUPS = QK_THREADS / G, HB = BWD ? QK_HEADS_BWD : QK_HEADS_FWD;
  op_begin();
  extern __shared__ float4 qk_smem[];
  unsigned long long* fx = reinterpret_cast<unsigned long long*>(qk_smem); float* cs = reinterpret_cast<float*>(fx) + ((p.rot + 3) & ~3);
  __shared__ float red[BWD ? QK_THREADS / 32 * G * 2 * V : 1];
  const int slot = threadIdx.x % G, g0 = threadIdx.x / G;
  Lane lane(p, slot);
  const int kind = blockIdx.y; const QkHeads& h = p.t[kind];
  if (h.heads == 0) return;
  const int per_token = (h.heads + HB - 1) / HB;
  lane.gain(h.gain);
  float2 acc[BWD ? 2 * P : 1];
  if constexpr (BWD) {
#pragma unroll
    for (int j = 0; j < 2 * P; j++) acc[j] = make_float2(0.f, 0.f);
  }
  const float inv = 1.f / p.head;
  qk_frequencies(p, fx);                                             // (seen behind the loop's first barrier)
  for (long base = (long)blockIdx.x * h.per_block; base < p.tokens; base += (long)gridDim.x * h.per_block) {
    const int n = (int)min((long)h.per_block, p.tokens - base), items = n * per_token;
    int t0 = g0 / per_token, hb0 = g0 - t0 * per_token;              // (token, block of heads) of this group's item
    for (int i0 = 0; i0 < items; i0 += GROUPS) {                     // (the same count for a whole block: barriers and shuffles want all of it)
      if (i0 > 0) { const int i = i0 + g0; t0 = i / per_token; hb0 = i - t0 * per_token; }
      const bool on = t0 < n; const int t = on ? t0 : 0, h0 = on ? hb0 * HB : 0, heads = on ? min(HB, h.heads - h0) : 0;
      const long tok = base + t;
      const T* x = static_cast<const T*>(h.in) + tok * h.in_t + h0 * h.in_h;
      Piece ua[HB], ub[HB], wa[BWD ? HB : 1], wb[BWD ? HB : 1];
#pragma unroll
      for (int q = 0; q < HB; q++) {
        ua[q] = ub[q] = Piece{};
        if (q < heads) lane.load(x + q * h.in_h, ua[q], ub[q]);
      }
      if constexpr (BWD) {
        const T* d = static_cast<const T*>(h.dy) + tok * h.dy_t + h0 * h.dy_h;
#pragma unroll
        for (int q = 0; q < HB; q++) {
          wa[q] = wb[q] = Piece{};
          if (q < heads) lane.load(d + q * h.dy_h, wa[q], wb[q]);
        }
      }
      if (i0 == 0) {                                                 // under the loads
        __syncthreads();
        qk_turns(p, base, n, fx, cs);
        __syncthreads();
      }
      lane.turns(p, cs + t * p.rot, BWD ? -1.f : 1.f);
      T* o = static_cast<T*>(h.out) + tok * h.out_t + h0 * h.out_h;
#pragma unroll
      for (int q = 0; q < HB; q++) {
        float2 a[P], b[P]; Lane::open(ua[q], a); Lane::open(ub[q], b);
        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < P; j++) { s2 = fma2(a[j], a[j], s2); s2 = fma2(b[j], b[j], s2); }
        float ss = s2.x + s2.y;
        if constexpr (!BWD) {
#pragma unroll
          for (int m = G / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
          const float rs = rsqrtf(fmaf(ss, inv, p.eps)); const float2 r2 = make_float2(rs, rs);
#pragma unroll
          for (int j = 0; j < P; j++) { a[j] = mul2(a[j], lane.ga[j]); b[j] = mul2(b[j], lane.gb[j]); }
          lane.turn(p, a, b);
#pragma unroll
          for (int j = 0; j < P; j++) { a[j] = mul2(a[j], r2); b[j] = mul2(b[j], r2); }
          if (q < heads) lane.store(o + q * h.out_h, a, b);
        } else {
          float2 ya[P], yb[P]; Lane::open(wa[q], ya); Lane::open(wb[q], yb);
          lane.turn(p, ya, yb);
          float2 x2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < P; j++) { x2 = fma2(mul2(ya[j], lane.ga[j]), a[j], x2); x2 = fma2(mul2(yb[j], lane.gb[j]), b[j], x2); }
          float sx = x2.x + x2.y;
#pragma unroll
          for (int m = G / 2; m > 0; m >>= 1) { ss += __shfl_xor_sync(0xffffffffu, ss, m); sx += __shfl_xor_sync(0xffffffffu, sx, m); }
          const float rs = q < heads ? rsqrtf(fmaf(ss, inv, p.eps)) : 0.f, m = -rs * rs * (sx * inv);      // (a row that is not there has zeros: with eps = 0 its root would be infinite)
          const float2 r2 = make_float2(rs, rs), m2 = make_float2(m, m);
#pragma unroll
          for (int j = 0; j < P; j++) {
            acc[j] = fma2(ya[j], mul2(a[j], r2), acc[j]); acc[P + j] = fma2(yb[j], mul2(b[j], r2), acc[P + j]);      // (rows that are not there have zeros)
            ya[j] = mul2(r2, fma2(a[j], m2, mul2(ya[j], lane.ga[j]))); yb[j] = mul2(r2, fma2(b[j], m2, mul2(yb[j], lane.gb[j])));
          }
          if (q < heads) lane.store(o + q * h.out_h, ya, yb);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (!p.partial) return;
#pragma unroll
    for (int m = 16; m >= G; m >>= 1) {
#pragma unroll
      for (int j = 0; j < 2 * P; j++) { acc[j].x += __shfl_xor_sync(0xffffffffu, acc[j].x, m); acc[j].y += __shfl_xor_sync(0xffffffffu, acc[j].y, m); }
    }
    const int warp = threadIdx.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) < G) {
#pragma unroll
      for (int j = 0; j < 2 * P; j++) { red[(warp * G + slot) * 2 * V + 2 * j] = acc[j].x; red[(warp * G + slot) * 2 * V + 2 * j + 1] = acc[j].y; }
    }
    __syncthreads();
    float* out = p.partial + ((long)blockIdx.x * 2 + kind) * p.head;
    for (int e = threadIdx.x; e < G * 2 * V; e += QK_THREADS) {
      const int j = e % (2 * V); const Lane of(p, e / (2 * V)); const int piece = j < V ? of.pa : of.pb;
      float v = 0.f;
      for (int w = 0; w < QK_THREADS / 32; w++) v += red[w * G * 2 * V + e];
      if (piece * V < p.head) out[piece * V + j % V] = v;
    }
  }
}

// Rows that no pieces fit: a warp per row, an element (or a pair) per lane at a time.  Bound by the latency of a row's loads and sums one after another, so that 32 warps an SM are under way
// (32768 tokens of 16 + 4 heads of 66, bf16: 344 us forward, 496 backward; with 8 warps 697 and 1323).
template <class T, bool BWD>
__global__ void __launch_bounds__(32 * QK_ROW_WARPS, QK_PER_SM) qk_rows_kernel(const __grid_constant__ QkParams p) {
  op_begin();
  extern __shared__ float4 qk_smem[];
  unsigned long long* fx = reinterpret_cast<unsigned long long*>(qk_smem); float* cs = reinterpret_cast<float*>(fx) + ((p.rot + 3) & ~3);
  const int half = p.rot >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kind = blockIdx.y; const QkHeads& h = p.t[kind];
  if (h.heads == 0) return;
  qk_frequencies(p, fx);
  float* acc = cs + h.per_block * p.rot + warp * p.head;             // this warp's share of the gain's gradient; an element belongs to one lane
  {
    auto first = [&](int i) { return p.inter ? 2 * i : i; };
    auto second = [&](int i) { return p.inter ? 2 * i + 1 : i + half; };
    auto gain = [&](int e) { return h.gain ? ld(h.gain + e) : 1.f; };
    if constexpr (BWD) {
      __syncthreads();
      for (int e = threadIdx.x; e < QK_ROW_WARPS * p.head; e += blockDim.x) acc[e - warp * p.head] = 0.f;
    }
    for (long base = (long)blockIdx.x * h.per_block; base < p.tokens; base += (long)gridDim.x * h.per_block) {
      const int n = (int)min((long)h.per_block, p.tokens - base), rows = n * h.heads;
      __syncthreads();
      qk_turns(p, base, n, fx, cs);
      __syncthreads();
      for (int r = warp; r < rows; r += QK_ROW_WARPS) {
        const int t = r / h.heads, hd = r - t * h.heads;
        const T* x = static_cast<const T*>(h.in) + (base + t) * h.in_t + hd * h.in_h;
        T* o = static_cast<T*>(h.out) + (base + t) * h.out_t + hd * h.out_h;
        const float *c = cs + t * p.rot, *s = c + half;
        float ss = 0.f;
        for (int e = lane; e < p.head; e += 32) { const float v = to_f32(x[e]); ss += v * v; }
        const float rs = rsqrtf(warp_sum(ss) / p.head + p.eps);
        if constexpr (!BWD) {
          for (int i = lane; i < half; i += 32) {
            const int e = first(i), f = second(i);
            float a = to_f32(x[e]) * rs * gain(e), b = to_f32(x[f]) * rs * gain(f);
            rotate(a, b, c[i], s[i]); o[e] = from_f32<T>(a); o[f] = from_f32<T>(b);
          }
          for (int e = p.rot + lane; e < p.head; e += 32) o[e] = from_f32<T>(to_f32(x[e]) * rs * gain(e));
        } else {
          const T* d = static_cast<const T*>(h.dy) + (base + t) * h.dy_t + hd * h.dy_h;
          float sx = 0.f;
          for (int i = lane; i < half; i += 32) {
            const int e = first(i), f = second(i);
            float a = to_f32(d[e]), b = to_f32(d[f]); rotate(a, b, c[i], -s[i]);
            sx += a * gain(e) * to_f32(x[e]) + b * gain(f) * to_f32(x[f]);
          }
          for (int e = p.rot + lane; e < p.head; e += 32) sx += to_f32(d[e]) * gain(e) * to_f32(x[e]);
          const float m = rs * rs * (warp_sum(sx) / p.head);
          auto put = [&](int e, float u) {
            const float v = to_f32(x[e]);
            acc[e] += u * (v * rs); o[e] = from_f32<T>(rs * (u * gain(e) - v * m));
          };
          for (int i = lane; i < half; i += 32) {
            const int e = first(i), f = second(i);
            float a = to_f32(d[e]), b = to_f32(d[f]); rotate(a, b, c[i], -s[i]);
            put(e, a); put(f, b);
          }
          for (int e = p.rot + lane; e < p.head; e += 32) put(e, to_f32(d[e]));
        }
      }
    }
    if constexpr (BWD) {
      __syncthreads();
      if (p.partial)
        for (int e = threadIdx.x; e < p.head; e += blockDim.x) {
          float v = 0.f;
          for (int w = 0; w < QK_ROW_WARPS; w++) v += (acc - warp * p.head)[w * p.head + e];
          p.partial[((long)blockIdx.x * 2 + kind) * p.head + e] = v;
        }
    }
  }
}

// dgain[e] = sum of the blocks' partial sums: 32 threads a column, each a run of neighbouring blocks, in order
__global__ void __launch_bounds__(1024) qk_gain_kernel(const float* partial, int blocks, int head, float* dq, float* dk) {
  op_begin();
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, per = (blocks + 31) / 32;
  float v = 0.f;
  if (col < 2 * head && (col < head ? dq : dk)) {
#pragma unroll 8
    for (int b = w * per; b < min(blocks, (w + 1) * per); b++) v += ld(partial + (long)b * 2 * head + col);
  }
  red[w][lane] = v;
  __syncthreads();
  v = warp_sum(red[lane][w]);                                        // column w of the 32
  const int out = blockIdx.x * 32 + w;
  if (lane == 0 && out < 2 * head) { float* d = out < head ? dq : dk; if (d) d[out < head ? out : out - head] = v; }
}

template <class T, int G, bool BWD>
inline int qk_launch_vec(const QkParams& p, int piece, dim3 grid, size_t turns, void* stream) {
  constexpr int V = Vec<T>::N;
  if constexpr (sizeof(T) == 2) { if (piece == 8) return op_launch("qk_vec", stream, qk_vec_kernel<T, 4, G, BWD, false>, grid, dim3(QK_THREADS), turns, 0, p); }
  const bool full = !p.inter && p.rot == p.head && p.head == 2 * G * V;
  return op_launch("qk_vec", stream, full ? qk_vec_kernel<T, V, G, BWD, true> : qk_vec_kernel<T, V, G, BWD, false>, grid, dim3(QK_THREADS), turns, 0, p);
}
// Sets the tokens of a block and launches; *blocks: partial sums that the gradient of a gain leaves.
template <class T, bool BWD>
inline int qk_launch(QkParams p, const gn_heads* const* all, int n_all, int sms, void* stream, unsigned* blocks) {
  constexpr int dtype = sizeof(T) == 4 ? GN_F32 : GN_F16;            // (only its size counts here)
  int piece = 16, group = qk_group(dtype, p.head, p.rot, p.inter, all, n_all);
  if (group == 0 && sizeof(T) == 2) { piece = 8; group = qk_group(dtype, p.head, p.rot, p.inter, all, n_all, 8); }
  int most = 0; int64_t n = 1;
  for (QkHeads& h : p.t) {
    h.per_block = qk_tokens(p.tokens, sms, group, h.heads, BWD ? QK_HEADS_BWD : QK_HEADS_FWD, p.rot);
    if (h.heads) { most = std::max(most, h.per_block); n = std::max(n, qk_blocks(p.tokens, sms, h.per_block)); }
  }
  *blocks = (unsigned)n;
  const dim3 grid((unsigned)n, p.t[1].heads ? 2 : 1);
  const size_t turns = ((size_t)most * p.rot + ((p.rot + 3) & ~3)) * sizeof(float);      // at most 36 KB
  switch (group) {
    case 0: {
      const size_t smem = turns + (BWD ? (size_t)QK_ROW_WARPS * p.head * sizeof(float) : 0);      // at most QK_ROWS_SMEM_MOST
      if (smem > 40 * 1024) GN_TRY(op_smem("qk_rows", qk_rows_kernel<T, BWD>, QK_ROWS_SMEM_MOST));
      return op_launch("qk_rows", stream, qk_rows_kernel<T, BWD>, grid, dim3(32 * QK_ROW_WARPS), smem, 0, p);
    }
    case 2: return qk_launch_vec<T, 2, BWD>(p, piece, grid, turns, stream);
    case 4: return qk_launch_vec<T, 4, BWD>(p, piece, grid, turns, stream);
    case 8: return qk_launch_vec<T, 8, BWD>(p, piece, grid, turns, stream);
    case 16: return qk_launch_vec<T, 16, BWD>(p, piece, grid, turns, stream);
    default: return qk_launch_vec<T, 32, BWD>(p, piece, grid, turns, stream);
  }
}
inline QkHeads qk_heads(const gn_heads* x, const gn_heads* dy, const gn_heads* out, const float* gain) {
  QkHeads h{};
  if (!x) return h;
  h.in = x->data; h.in_t = x->token_stride; h.in_h = x->head_stride; h.heads = x->heads; h.gain = gain;
  if (dy) { h.dy = dy->data; h.dy_t = dy->token_stride; h.dy_h = dy->head_stride; }
  h.out = out->data; h.out_t = out->token_stride; h.out_h = out->head_stride;
  return h;
}

}  // namespace gn

extern "C" {

int gn_op_qk_norm_rope(gn_ctx* ctx, int dtype, int64_t tokens, int head_size, int rotated, int interleaved, float eps, const gn_heads* q, const gn_heads* k,
                       const float* gain_q, const float* gain_k, const void* positions, int index_type, const double* frequencies,
                       const gn_heads* q_out, const gn_heads* k_out, void* stream) {
  using namespace gn;
  const QkArgs a{dtype, tokens, head_size, rotated, eps, q, k, gain_q, gain_k, positions, index_type, frequencies};
  const char* wrong = check_qk(a);
  if (!wrong) wrong = check_heads(a, q_out, q->heads, true);
  if (!wrong && k) wrong = check_heads(a, k_out, k->heads, true);
  if (!wrong) wrong = check_in_place(q, q_out);
  if (!wrong) wrong = check_in_place(k, k_out);
  if (!wrong && k && tokens) for (const char* e : {check_apart(q_out, k), check_apart(k_out, q), check_apart(q_out, k_out)}) if (e) wrong = e;
  GN_OP_BEGIN("op_qk_norm_rope", wrong);
  if (tokens == 0 || q->heads + (k ? k->heads : 0) == 0) return GN_OK;
  const int sms = ctx->c.sm_count; const gn_heads* all[] = {q, k, q_out, k ? k_out : nullptr};
  QkParams p{{qk_heads(q, nullptr, q_out, gain_q), qk_heads(k, nullptr, k_out, gain_k)}, tokens, head_size, rotated, interleaved != 0, eps, positions, index_type, frequencies, nullptr};
  unsigned blocks = 0;
  return with_type(dtype, [&](auto t) { using T = decltype(t); return qk_launch<T, false>(p, all, 4, sms, stream, &blocks); });
}

int gn_op_qk_norm_rope_workspace(gn_ctx* ctx, int64_t tokens, int q_heads, int k_heads, int head_size, int64_t* bytes) {
  using namespace gn;
  if (!ctx || !ctx->alive || !bytes || tokens < 0 || q_heads < 0 || k_heads < 0 || head_size < 1) return fail(GN_ERR_INVALID_ARG, "op_qk_norm_rope_workspace: bad argument");
  *bytes = tokens == 0 ? 0 : qk_workspace(tokens, head_size, ctx->c.sm_count); return GN_OK;
}

int gn_op_qk_norm_rope_backward(gn_ctx* ctx, int dtype, int64_t tokens, int head_size, int rotated, int interleaved, float eps, const gn_heads* q, const gn_heads* k,
                                const float* gain_q, const float* gain_k, const void* positions, int index_type, const double* frequencies,
                                const gn_heads* dq_out, const gn_heads* dk_out, const gn_heads* dq, const gn_heads* dk, float* dgain_q, float* dgain_k,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace gn;
  const QkArgs a{dtype, tokens, head_size, rotated, eps, q, k, gain_q, gain_k, positions, index_type, frequencies};
  const char* wrong = check_qk(a);
  if (!wrong) wrong = check_heads(a, dq_out, q->heads, false);
  if (!wrong) wrong = check_heads(a, dq, q->heads, true);
  if (!wrong && k) wrong = check_heads(a, dk_out, k->heads, false);
  if (!wrong && k) wrong = check_heads(a, dk, k->heads, true);
  if (!wrong) wrong = check_in_place(dq_out, dq);
  if (!wrong && k) wrong = check_in_place(dk_out, dk);
  if (!wrong && k && tokens) for (const char* e : {check_apart(dq, k), check_apart(dq, dk_out), check_apart(dk, q), check_apart(dk, dq_out), check_apart(dq, dk)}) if (e) wrong = e;
  if (!wrong && (!aligned_to(dgain_q, 4) || !aligned_to(dgain_k, 4))) wrong = "a pointer is not aligned to its type";
  if (!wrong && dgain_k && !k) wrong = "dgain_k without k";
  GN_OP_BEGIN("op_qk_norm_rope_backward", wrong);
  const int sms = ctx->c.sm_count; const bool gains = dgain_q || dgain_k;
  if (tokens == 0) {
    if (dgain_q) GN_CUDA(cudaMemsetAsync(dgain_q, 0, 4L * head_size, (cudaStream_t)stream));
    if (dgain_k) GN_CUDA(cudaMemsetAsync(dgain_k, 0, 4L * head_size, (cudaStream_t)stream));
    return GN_OK;
  }
  if (gains && (!workspace || !aligned_to(workspace, 16) || workspace_bytes < qk_workspace(tokens, head_size, sms))) return fail(GN_ERR_INVALID_ARG, "op_qk_norm_rope_backward: the workspace is too small, null or not aligned");
  const gn_heads* all[] = {q, k, dq_out, k ? dk_out : nullptr, dq, k ? dk : nullptr};
  QkParams p{{qk_heads(q, dq_out, dq, gain_q), qk_heads(k, dk_out, dk, gain_k)}, tokens, head_size, rotated, interleaved != 0, eps, positions, index_type, frequencies, gains ? (float*)workspace : nullptr};
  unsigned blocks = 0;
  if (p.t[0].heads + p.t[1].heads) GN_TRY(with_type(dtype, [&](auto t) { using T = decltype(t); return qk_launch<T, true>(p, all, 6, sms, stream, &blocks); }));
  // a tensor of no heads has left no partial sums
  if (dgain_q && !p.t[0].heads) { GN_CUDA(cudaMemsetAsync(dgain_q, 0, 4L * head_size, (cudaStream_t)stream)); dgain_q = nullptr; }
  if (dgain_k && !p.t[1].heads) { GN_CUDA(cudaMemsetAsync(dgain_k, 0, 4L * head_size, (cudaStream_t)stream)); dgain_k = nullptr; }
  if (!dgain_q && !dgain_k) return GN_OK;
  return op_launch("qk_gain", stream, qk_gain_kernel, dim3((2 * head_size + 31) / 32), dim3(1024), 0, 0, (const float*)workspace, (int)blocks, head_size, dgain_q, dgain_k);
}

}  // extern "C"
