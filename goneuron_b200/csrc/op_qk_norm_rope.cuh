// op_qk_norm_rope.cuh -- norm of queries and keys per head with the position rotation in the same pass, and its gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = R (g x r);     u = R^T dy,  dx = r (g u - x r^2 mean(g u x)),  dg = sum u x r
//
// R turns pairs of elements by position * frequency.  The angle is formed in 64 bits, in turns, and its whole turns are dropped there, so that
// a far position costs no accuracy; sine and cosine of what is left are float32, once per token and pair for all heads, in shared memory.
// Everything between reading x (and dy) and the one rounding of the result is float32.
//
// Bound by memory: a row is read once and written once.  A lane holds two 16-byte pieces of a row, the two halves of its pairs, so that a rotation stays
// within the lane and the sums over a row are shuffles among its 2 to 32 lanes.
#pragma once
#include "device_ops.cuh"

namespace gn {

struct QkHeads { const void* in; const void* dy; void* out; long in_t, in_h, dy_t, dy_h, out_t, out_h; int heads; const float* gain; };
struct QkParams {
  QkHeads t[2]; long tokens; int head, rot, inter, per_block; float eps; const void* pos; int index_type; const double* freq; float* partial;
};

// cosine and sine of the angle of (token, pair)
__device__ __forceinline__ float2 qk_turn(const QkParams& p, long token, int pair) {
  double turns = (double)load_index(p.pos, p.index_type, token) * __ldg(p.freq + pair) * 0.15915494309189533577;      // 1 / (2 pi)
  turns -= rint(turns);
  float s, c; sincospif(2.f * (float)turns, &s, &c);
  return make_float2(c, s);
}
__device__ __forceinline__ void qk_turns(const QkParams& p, long base, int n, float2* cs) {
  const int half = p.rot >> 1;
  for (int e = threadIdx.x; e < n * half; e += blockDim.x) { const int t = e / half; cs[e] = qk_turn(p, base + t, e - t * half); }
}
// sign -1: R^T
__device__ __forceinline__ void rotate(float& a, float& b, float2 cs, float sign) { const float sn = sign * cs.y, u = a * cs.x - b * sn; b = a * sn + b * cs.x; a = u; }
// a lane's two pieces: whole halves of pairs (`split`), or neighbouring elements as pairs
template <int V>
__device__ __forceinline__ void qk_turn_pieces(const QkParams& p, float (&x)[V], float (&y)[V], const float2* cs, bool split, int s, int pa, int pb, float sign) {
  if (split) {
#pragma unroll
    for (int j = 0; j < V; j++) rotate(x[j], y[j], cs[s * V + j], sign);
  } else if (p.inter) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      if (pa * V + j < p.rot) rotate(x[j], x[j + 1], cs[(pa * V + j) >> 1], sign);
      if (pb * V + j < p.rot) rotate(y[j], y[j + 1], cs[(pb * V + j) >> 1], sign);
    }
  }
}

constexpr int QK_THREADS = 256;
template <class T, int G, bool BWD>
__global__ void __launch_bounds__(QK_THREADS, BWD ? QK_PER_SM : 4) qk_vec_kernel(const __grid_constant__ QkParams p) {
  constexpr int V = Vec<T>::N, ROWS = QK_THREADS / G;
  extern __shared__ float4 qk_smem[];
  float2* cs = reinterpret_cast<float2*>(qk_smem);
  __shared__ float red[BWD ? QK_THREADS / 32 * G * 2 * V : 1];
  const int s = threadIdx.x % G, g0 = threadIdx.x / G, half = p.rot >> 1, pieces = p.head / V, turned = half / V;
  // this lane's two pieces: the halves of its pairs, or two neighbours behind the rotated part (interleaved: two neighbours everywhere)
  const int pa = p.inter ? 2 * s : s < turned ? s : 2 * s, pb = p.inter || s >= turned ? pa + 1 : s + turned;
  const bool has_a = pa < pieces, has_b = pb < pieces, split = !p.inter && s < turned;
#pragma unroll 1
  for (int kind = 0; kind < 2; kind++) {
    const QkHeads& h = p.t[kind];
    if (h.heads == 0) continue;
    float ga[V], gb[V], acc[BWD ? 2 * V : 1];
#pragma unroll
    for (int j = 0; j < V; j++) { ga[j] = h.gain && has_a ? __ldg(h.gain + pa * V + j) : 1.f; gb[j] = h.gain && has_b ? __ldg(h.gain + pb * V + j) : 1.f; }
    if constexpr (BWD) {
#pragma unroll
      for (int j = 0; j < 2 * V; j++) acc[j] = 0.f;
    }
    for (long base = (long)blockIdx.x * p.per_block; base < p.tokens; base += (long)gridDim.x * p.per_block) {
      const int n = (int)min((long)p.per_block, p.tokens - base), rows = n * h.heads;
      __syncthreads();
      qk_turns(p, base, n, cs);
      __syncthreads();
      for (int r0 = 0; r0 < rows; r0 += ROWS) {                      // (the same count for a whole block: the shuffles below want whole warps)
        const int r = r0 + g0; const bool on = r < rows;
        const int t = on ? r / h.heads : 0, hd = r - t * h.heads;
        const long tok = base + t;
        uint4 ua = make_uint4(0, 0, 0, 0), ub = ua, wa = ua, wb = ua;
        if (on) {
          const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(h.in) + tok * h.in_t + hd * h.in_h);
          if (has_a) ua = x[pa];
          if (has_b) ub = x[pb];
          if constexpr (BWD) {
            const uint4* d = reinterpret_cast<const uint4*>(static_cast<const T*>(h.dy) + tok * h.dy_t + hd * h.dy_h);
            if (has_a) wa = d[pa];
            if (has_b) wb = d[pb];
          }
        }
        float a[V], b[V]; unpack<T>(ua, a); unpack<T>(ub, b);
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) ss += a[j] * a[j] + b[j] * b[j];
        const float2* c = cs + t * half;
        float ya[V], yb[V];
        if constexpr (!BWD) {
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float rs = rsqrtf(ss / p.head + p.eps);
#pragma unroll
          for (int j = 0; j < V; j++) { ya[j] = a[j] * rs * ga[j]; yb[j] = b[j] * rs * gb[j]; }
          qk_turn_pieces<V>(p, ya, yb, c, split, s, pa, pb, 1.f);
        } else {
          unpack<T>(wa, ya); unpack<T>(wb, yb);
          qk_turn_pieces<V>(p, ya, yb, c, split, s, pa, pb, -1.f);
          float sx = 0.f;
#pragma unroll
          for (int j = 0; j < V; j++) sx += ya[j] * ga[j] * a[j] + yb[j] * gb[j] * b[j];
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) { ss += __shfl_xor_sync(0xffffffffu, ss, o); sx += __shfl_xor_sync(0xffffffffu, sx, o); }
          const float rs = rsqrtf(ss / p.head + p.eps), m = rs * rs * (sx / p.head);
#pragma unroll
          for (int j = 0; j < V; j++) {
            acc[j] += ya[j] * (a[j] * rs); acc[V + j] += yb[j] * (b[j] * rs);      // (rows that are not there have zeros)
            ya[j] = rs * (ya[j] * ga[j] - a[j] * m); yb[j] = rs * (yb[j] * gb[j] - b[j] * m);
          }
        }
        if (on) {
          uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(h.out) + tok * h.out_t + hd * h.out_h);
          if (has_a) o[pa] = pack<T>(ya);
          if (has_b) o[pb] = pack<T>(yb);
        }
      }
    }
    if constexpr (BWD) {
      if (!p.partial) continue;
#pragma unroll
      for (int o = 16; o >= G; o >>= 1) {
#pragma unroll
        for (int j = 0; j < 2 * V; j++) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
      }
      const int warp = threadIdx.x >> 5;
      __syncthreads();
      if ((threadIdx.x & 31) < G) {
#pragma unroll
        for (int j = 0; j < 2 * V; j++) red[(warp * G + s) * 2 * V + j] = acc[j];
      }
      __syncthreads();
      float* out = p.partial + ((long)blockIdx.x * 2 + kind) * p.head;
      for (int e = threadIdx.x; e < G * 2 * V; e += QK_THREADS) {
        const int ls = e / (2 * V), j = e % (2 * V);                 // lane, its element
        const int qa = p.inter ? 2 * ls : ls < turned ? ls : 2 * ls, qb = p.inter || ls >= turned ? qa + 1 : ls + turned;
        const int piece = j < V ? qa : qb;
        float v = 0.f;
        for (int w = 0; w < QK_THREADS / 32; w++) v += red[w * G * 2 * V + e];
        if (piece < pieces) out[piece * V + j % V] = v;
      }
    }
  }
}

// Rows that 16-byte pieces do not fit: a warp per row, an element (or a pair) per lane at a time.
constexpr int QK_ROW_WARPS = 4;
template <class T, bool BWD>
__global__ void __launch_bounds__(32 * QK_ROW_WARPS) qk_rows_kernel(const __grid_constant__ QkParams p) {
  extern __shared__ float4 qk_smem[];
  float2* cs = reinterpret_cast<float2*>(qk_smem);
  const int half = p.rot >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* acc = reinterpret_cast<float*>(cs + p.per_block * half) + warp * p.head;      // this warp's share of the gain's gradient; an element belongs to one lane
  for (int kind = 0; kind < 2; kind++) {
    const QkHeads& h = p.t[kind];
    if (h.heads == 0) continue;
    auto first = [&](int i) { return p.inter ? 2 * i : i; };
    auto second = [&](int i) { return p.inter ? 2 * i + 1 : i + half; };
    auto gain = [&](int e) { return h.gain ? __ldg(h.gain + e) : 1.f; };
    if constexpr (BWD) {
      __syncthreads();
      for (int e = threadIdx.x; e < QK_ROW_WARPS * p.head; e += blockDim.x) acc[e - warp * p.head] = 0.f;
    }
    for (long base = (long)blockIdx.x * p.per_block; base < p.tokens; base += (long)gridDim.x * p.per_block) {
      const int n = (int)min((long)p.per_block, p.tokens - base), rows = n * h.heads;
      __syncthreads();
      qk_turns(p, base, n, cs);
      __syncthreads();
      for (int r = warp; r < rows; r += QK_ROW_WARPS) {
        const int t = r / h.heads, hd = r - t * h.heads;
        const T* x = static_cast<const T*>(h.in) + (base + t) * h.in_t + hd * h.in_h;
        T* o = static_cast<T*>(h.out) + (base + t) * h.out_t + hd * h.out_h;
        const float2* c = cs + t * half;
        float ss = 0.f;
        for (int e = lane; e < p.head; e += 32) { const float v = to_f32(x[e]); ss += v * v; }
        const float rs = rsqrtf(warp_sum(ss) / p.head + p.eps);
        if constexpr (!BWD) {
          for (int i = lane; i < half; i += 32) {
            const int e = first(i), f = second(i);
            float a = to_f32(x[e]) * rs * gain(e), b = to_f32(x[f]) * rs * gain(f);
            rotate(a, b, c[i], 1.f); o[e] = from_f32<T>(a); o[f] = from_f32<T>(b);
          }
          for (int e = p.rot + lane; e < p.head; e += 32) o[e] = from_f32<T>(to_f32(x[e]) * rs * gain(e));
        } else {
          const T* d = static_cast<const T*>(h.dy) + (base + t) * h.dy_t + hd * h.dy_h;
          float sx = 0.f;
          for (int i = lane; i < half; i += 32) {
            const int e = first(i), f = second(i);
            float a = to_f32(d[e]), b = to_f32(d[f]); rotate(a, b, c[i], -1.f);
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
            float a = to_f32(d[e]), b = to_f32(d[f]); rotate(a, b, c[i], -1.f);
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

// dgain[e] = sum of the blocks' partial sums: eight threads a column, each a run of neighbouring blocks, in order
__global__ void __launch_bounds__(256) qk_gain_kernel(const float* __restrict__ partial, int blocks, int head, float* __restrict__ dq, float* __restrict__ dk) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, per = (blocks + 7) / 8;
  float v = 0.f;
  if (col < 2 * head && (col < head ? dq : dk))
    for (int b = w * per; b < min(blocks, (w + 1) * per); b++) v += __ldg(partial + (long)b * 2 * head + col);
  red[w][lane] = v;
  __syncthreads();
  if (w == 0 && col < 2 * head) {
    float* out = col < head ? dq : dk;
    for (int i = 1; i < 8; i++) v += red[i][lane];
    if (out) out[col < head ? col : col - head] = v;
  }
}

template <class T, bool BWD>
inline int qk_launch(QkParams& p, int group, unsigned grid, void* stream) {
  const size_t turns = (size_t)p.per_block * (p.rot / 2) * sizeof(float2);
  if (group == 0) {
    const size_t smem = turns + (BWD ? (size_t)QK_ROW_WARPS * p.head * sizeof(float) : 0);      // at most 16 + 16 KB
    return op_launch("qk_rows", stream, qk_rows_kernel<T, BWD>, grid, 32 * QK_ROW_WARPS, smem, 0, p);
  }
  switch (group) {
    case 2: return op_launch("qk_vec", stream, qk_vec_kernel<T, 2, BWD>, grid, QK_THREADS, turns, 0, p);
    case 4: return op_launch("qk_vec", stream, qk_vec_kernel<T, 4, BWD>, grid, QK_THREADS, turns, 0, p);
    case 8: return op_launch("qk_vec", stream, qk_vec_kernel<T, 8, BWD>, grid, QK_THREADS, turns, 0, p);
    case 16: return op_launch("qk_vec", stream, qk_vec_kernel<T, 16, BWD>, grid, QK_THREADS, turns, 0, p);
    default: return op_launch("qk_vec", stream, qk_vec_kernel<T, 32, BWD>, grid, QK_THREADS, turns, 0, p);
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
  GN_OP_BEGIN("op_qk_norm_rope", wrong);
  if (tokens == 0 || q->heads + (k ? k->heads : 0) == 0) return GN_OK;
  const int sms = ctx->c.sm_count; const gn_heads* all[] = {q, k, q_out, k ? k_out : nullptr};
  QkParams p{{qk_heads(q, nullptr, q_out, gain_q), qk_heads(k, nullptr, k_out, gain_k)}, tokens, head_size, rotated, interleaved != 0, qk_tokens(tokens, sms), eps, positions, index_type, frequencies, nullptr};
  const int group = qk_group(dtype, head_size, rotated, interleaved != 0, all, 4);
  const unsigned grid = (unsigned)qk_blocks(tokens, sms, 8);
  return with_type(dtype, [&](auto t) { using T = decltype(t); return qk_launch<T, false>(p, group, grid, stream); });
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
  QkParams p{{qk_heads(q, dq_out, dq, gain_q), qk_heads(k, dk_out, dk, gain_k)}, tokens, head_size, rotated, interleaved != 0, qk_tokens(tokens, sms), eps, positions, index_type, frequencies, gains ? (float*)workspace : nullptr};
  const int group = qk_group(dtype, head_size, rotated, interleaved != 0, all, 6);
  const unsigned grid = (unsigned)qk_blocks(tokens, sms, QK_PER_SM);
  if (p.t[0].heads + p.t[1].heads) GN_TRY(with_type(dtype, [&](auto t) { using T = decltype(t); return qk_launch<T, true>(p, group, grid, stream); }));
  // a tensor of no heads has left no partial sums
  if (dgain_q && !p.t[0].heads) { GN_CUDA(cudaMemsetAsync(dgain_q, 0, 4L * head_size, (cudaStream_t)stream)); dgain_q = nullptr; }
  if (dgain_k && !p.t[1].heads) { GN_CUDA(cudaMemsetAsync(dgain_k, 0, 4L * head_size, (cudaStream_t)stream)); dgain_k = nullptr; }
  if (!dgain_q && !dgain_k) return GN_OK;
  return op_launch("qk_gain", stream, qk_gain_kernel, dim3((2 * head_size + 31) / 32), dim3(256), 0, 0, (const float*)workspace, (int)grid, head_size, dgain_q, dgain_k);
}

}  // extern "C"
