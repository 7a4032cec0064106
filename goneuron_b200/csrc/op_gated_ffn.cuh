// op_gated_ffn.cuh -- gated feed-forward block in 16 bits on the 5th-generation tensor cores, forward and backward, and its form for few tokens.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// One kernel template for all six products: TMA loads of 64 contraction indices a stage -> shared memory -> tcgen05.mma (fp32 accumulators in tensor memory, two slots, so that
// a tile's epilogue runs under the next tile's main loop) -> epilogue.  Operands are read as they lie in memory, rows along the contraction (K-major) or across it (MN-major), so that no
// product needs a transposed copy.  Pairs of blocks share a tile of 256 x 256 (cta_group::2): each holds half of A's rows and half of B's, so that an MMA of 128 cycles reads 8 KB of a
// block's shared memory and TMA writes as much, the 128 bytes a cycle that there are.  (A block by itself, 128 x 256: 12 + 12 KB, the main loop at 62 % of the MMA rate, 1327 TFLOP/s
// at K = 4096.)
//   - Forward: a tile's B operand is 128 rows of Wg followed by 128 of Wu, one 256-wide MMA for both projections, and a thread of the epilogue has g and u of the same elements:
//     activation and product are formed there and only h is written (and, for the gradient, g and u).
//   - dh is not written: its epilogue reads g and u, and writes dg and du.
//   - dx is one product over 2 ff indices, the first half of them from (dg, Wg), the second from (du, Wu).
//   - The three weight gradients are one launch.
// g and u are kept as the upper 24 bits of their float32 values, in the order in which the tensor memory hands them to a warp (blocks of 32 rows x 16 columns), so that both epilogues move
// them with whole 128-byte lines.  In 16 bits their rounding would add to those of dg and du and the error of dx be 1.7 times that of its own rounding instead of 1.4; the last 8 bits of
// float32 would be a quarter of what the epilogue of dh, which memory bounds, has to read.
// h, dg and du are rounded to 16 bits because the tensor cores read them as operands: y, dx and the weights' gradients have some 1.4 times the error of their own rounding, and of one to four tokens,
// whose sums few large terms make up, 1.2 to 1.7 times.  They have that type's range as well: in float16 infinite above 65504, zero below 2^-25.  There is no scale, which would have to be known before
// the tiles of a row are: what is too large makes its row not finite, never finite and wrong.
// Few output tiles: the contraction is cut into slices whose float32 sums a second launch adds in order.
//
// Waits are bounded as in the contraction engine: a wait that gives up sets the status word, every role of the block leaves its loops, copies and MMAs in flight are waited for
// (bounded), tensor memory is released.
#pragma once
#include "device_ops.cuh"
#include "fmath.cuh"
#include "tc_ptx.cuh"

namespace gn {

constexpr int FG_BM = 256, FG_BK = 64, FG_SAVED = 192;      // FG_SAVED: 16-byte pieces of a saved block
enum FgKind { FG_PLAIN, FG_GATE, FG_GATE_BWD };
// Maps of the operands (a0, b0 for the first kb0 blocks of the contraction, a1, b1 for the others; FG_GATE: b0 and b1 side by side) and of what is written.
struct FgProblem { CUtensorMap a0, a1, b0, b1, d0, d1; int M, N, kb0, kb, tiles_n, tiles; };
struct FgParams {
  FgProblem p[3]; int problems, splits, full, n_half;                // items: `full` whole tiles (times slices), then n_half halves of the tiles behind them
  float* partial; uint8_t* saved; int saved_cols; unsigned spin_limit; uint32_t idesc, idesc_half;
};
// EW epilogue warps: what the gates compute for an element is a chain of some 40 instructions, which 16 warps overlap.
template <int BN, FgKind KIND> struct FgCfg {
  static constexpr int EW = KIND == FG_PLAIN ? 8 : 16, THREADS = 64 + 32 * EW, COLS = BN / (KIND == FG_GATE ? 2 : 1) / (EW / 4);      // COLS: output columns of a warp
  static constexpr int STG_WARP = KIND == FG_GATE ? 2048 : 4096, STG = EW * STG_WARP;      // an epilogue warp's 32 rows of 64 or 128 bytes on their way out (dh: two of 64)
  static constexpr int A_BYTES = FG_BM * 64, B_BYTES = BN * 64, STAGE = A_BYTES + B_BYTES, STAGES = (224 * 1024 - STG) / STAGE;      // of one block of the pair
  static constexpr int SMEM = STAGES * STAGE + STG + 1024 + 256, TMEM = 2 * BN;
  static_assert(TMEM <= 512 && SMEM <= 232448 && 2 * STAGES + 5 <= 30, "");
};

// Shared-memory descriptors, 128-byte swizzle, version 1.  K-major: rows of 128 bytes (64 indices), groups of eight rows 1024 bytes apart.  MN-major: blocks of 64 rows (M or N) by 64
// indices, an index a row of 128 bytes: groups of eight indices 1024 bytes apart (stride offset), blocks 8192 bytes (leading offset).
template <bool MN> __device__ __forceinline__ uint64_t fg_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(MN ? 8192 >> 4 : 1) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16: D float32, A = B = fp16 (0) or bf16 (1), bits 15 / 16 for MN-major A / B.
inline uint32_t fg_idesc(bool bf16, bool amn, bool bmn, int N) {
  const uint32_t f = bf16 ? 1 : 0;
  return (1u << 4) | (f << 7) | (f << 10) | ((amn ? 1u : 0u) << 15) | ((bmn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(FG_BM >> 4) << 24);
}

// act(g) u, and the factors of dh in dg and du.  (relu lets a NaN through, which fmaxf would not.)
__device__ __forceinline__ float fg_relu(float g) { return g < 0.f ? 0.f : g; }
__device__ __forceinline__ float fg_sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
template <int act> __device__ __forceinline__ float fg_act(float g) { return act == GN_ACT_SILU ? g * fg_sigmoid(g) : act == GN_ACT_GELU ? gelu_f(g) : fg_relu(g); }
template <int act> __device__ __forceinline__ void fg_act_grad(float g, float& a, float& da) {
  if constexpr (act == GN_ACT_SILU) { const float p = fg_sigmoid(g); a = g * p; da = p * (1.f + g * (1.f - p)); }
  else if constexpr (act == GN_ACT_GELU) {                                     // (1 + tanh z) / 2 = sigmoid(2 z) = p, 1 - tanh^2 z = 4 p (1 - p)
    const float p = fg_sigmoid(g * fmaf(0.07135481627f * g, g, 1.5957691216057308f));
    a = g * p; da = p + g * 2.f * p * (1.f - p) * fminf(fmaf(0.10703222440890925f * g, g, 0.7978845608028654f), 3e38f);      // (far out 0 times a square that may not be finite)
  } else { a = fg_relu(g); da = g > 0.f ? 1.f : 0.f; }
}

// 16 float32 values of a lane as the upper halves of two in a word, and the bytes below of four: 48 bytes.  (What comes back repeats that byte below itself: infinities and zeros stay, and so
// does a NaN of the tensor core.)
__device__ __forceinline__ void fg_pack24(const uint32_t (&v)[16], uint4 (&q)[3]) {
  uint32_t w[12];
#pragma unroll
  for (int j = 0; j < 8; j++) w[j] = __byte_perm(v[2 * j], v[2 * j + 1], 0x7632);
#pragma unroll
  for (int j = 0; j < 4; j++) w[8 + j] = __byte_perm(__byte_perm(v[4 * j], v[4 * j + 1], 0x0051), __byte_perm(v[4 * j + 2], v[4 * j + 3], 0x0051), 0x5410);
#pragma unroll
  for (int j = 0; j < 3; j++) q[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}
__device__ __forceinline__ float fg_unpack24(const uint4 (&q)[3], int i) {      // i: a constant once unrolled
  auto word = [&](int j) { const uint4& u = q[j >> 2]; return (j & 3) == 0 ? u.x : (j & 3) == 1 ? u.y : (j & 3) == 2 ? u.z : u.w; };
  const uint32_t lo = 4 + (i & 3);
  return __uint_as_float(__byte_perm(word(i >> 1), word(8 + (i >> 2)), (i & 1 ? 0x3200u : 0x1000u) | (lo << 4) | lo));
}

// ACT: the activation of the gates' kinds, a template argument because a choice inside the loop over a row's elements kept them from overlapping.  (With the pairs of blocks, both projections of
// 16384 tokens, 16-bit g and u: 259 -> 217 us; the two were measured together.)
template <class T, int BN, bool AMN, bool BMN, FgKind KIND, int ACT>
__global__ void __launch_bounds__(FgCfg<BN, KIND>::THREADS, 1) __cluster_dims__(2, 1, 1) fg_gemm_kernel(const __grid_constant__ FgParams P) {
  using Cfg = FgCfg<BN, KIND>;
  constexpr int STAGES = Cfg::STAGES, STAGE = Cfg::STAGE;
  extern __shared__ uint8_t fg_smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)fg_smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = (uint64_t*)(smem + STAGES * STAGE + Cfg::STG);    // full[S], empty[S], tfull[2], tempty[2], drain
  uint32_t* tmem_slot = (uint32_t*)(bars + 2 * STAGES + 5);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES), tfull0 = smem_u32(bars + 2 * STAGES), tempty0 = smem_u32(bars + 2 * STAGES + 2), drain = smem_u32(bars + 2 * STAGES + 4);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t smem0 = smem_u32(smem), rank = cluster_rank(), lead_full0 = cluster_address(full0, 0), lead_tempty0 = cluster_address(tempty0, 0); const unsigned limit = P.spin_limit;

  pdl_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
    for (int b = 0; b < 2; b++) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 2 * Cfg::EW); }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Cfg::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                                // the other block's barriers are there
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();                                                        // set up under the kernel before this one
  auto give_up = [&]() { op_report(OP_TIMEOUT); *abort_flag = 1; __threadfence_block(); };

  // Items of this pair, the same in every role of both blocks: its number, + the number of pairs, ...
  struct Item { int q, m0, n0, k0, k1, half, slot; };                // problem, first row and column, blocks of the contraction, half (-1: whole tile), place of the partial sums
  auto item = [&](long t, Item& w) -> bool {
    long tile = t; int z = 0; w.half = -1;
    if (t >= P.full) {
      const long h = t - P.full;
      if (h >= P.n_half) return false;
      tile = P.full + (h >> 1); w.half = (int)(h & 1);
    } else if (P.splits > 1) { z = (int)(t % P.splits); tile = t / P.splits; }
    w.q = 0; w.slot = (int)t;
    while (w.q + 1 < P.problems && tile >= P.p[w.q].tiles) { tile -= P.p[w.q].tiles; w.q++; }
    const FgProblem& p = P.p[w.q];
    const int mt = (int)tile / p.tiles_n, nt = (int)tile - mt * p.tiles_n;
    w.m0 = mt * FG_BM; w.n0 = nt * (KIND == FG_GATE ? BN / 2 : BN) + (w.half > 0 ? BN / 2 : 0);
    w.k0 = (int)((long)p.kb * z / P.splits); w.k1 = (int)((long)p.kb * (z + 1) / P.splits);
    return true;
  };
  const bool elected = elect_one();
  if (warp == 0) {
    bool ok = true; uint32_t s = 0, ph = 0, issued = 0; Item w;
    for (long t = blockIdx.x >> 1; ok && item(t, w); t += gridDim.x >> 1) {
      const FgProblem& p = P.p[w.q]; const int bn = w.half < 0 ? BN : BN / 2;
      for (int k = w.k0; k < w.k1; k++) {
        if (issued >= (uint32_t)STAGES && !mbar_wait(empty0 + 8 * s, ph ^ 1, limit, abort_flag)) { ok = false; break; }
        if (elected) {
          const uint32_t base = smem0 + s * STAGE, bar = lead_full0 + 8 * s, bb = base + Cfg::A_BYTES;
          const bool first = KIND == FG_GATE || k < p.kb0; const CUtensorMap *a = first ? &p.a0 : &p.a1, *b = KIND == FG_GATE ? (rank ? &p.b1 : &p.b0) : first ? &p.b0 : &p.b1;
          const int kc = (first ? k : k - p.kb0) * FG_BK, m0 = w.m0 + (int)rank * 128, n0 = w.n0 + (KIND == FG_GATE ? 0 : (int)rank * (bn / 2));
          if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * Cfg::A_BYTES + bn * 128);      // both blocks' bytes
          if constexpr (AMN) { tma_load_2d_pair(base, a, m0, kc, bar); tma_load_2d_pair(base + 8192, a, m0 + 64, kc, bar); }
          else tma_load_2d_pair(base, a, kc, m0, bar);
          for (int j = 0; j < bn / 128; j++) { if constexpr (BMN) tma_load_2d_pair(bb + j * 8192, b, n0 + 64 * j, kc, bar); else tma_load_2d_pair(bb + j * 8192, b, kc, n0 + 64 * j, bar); }
        }
        issued++;
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
    // The last arrivals at this block's barriers come from the other one's MMAs: they have to be there before it leaves.
    if (ok) for (int i = 0; i < STAGES && issued > 0; i++, issued--) { const uint32_t q = (issued - 1) % STAGES, use = (issued - 1) / STAGES; if (!mbar_wait(empty0 + 8 * q, use & 1, limit, abort_flag)) { ok = false; break; } }
    if (!ok && !*abort_flag) give_up();
    // Something gave up: copies in flight still write into this block's shared memory and count at the first block's barriers, which not all roles wait for any more.  They land within
    // microseconds; the pair stays for some hundred.
    if (*abort_flag) { const long long t0 = clock64(); while (clock64() - t0 < (1LL << 18)) __nanosleep(200); }
    __syncwarp();
  } else if (warp == 1) {
    bool ok = true; uint32_t s = 0, ph = 0, lt = 0; Item w;
    const uint64_t adesc0 = fg_desc<AMN>(smem0), bdesc0 = fg_desc<BMN>(smem0 + Cfg::A_BYTES);
    constexpr uint64_t ASTEP = AMN ? 2048 >> 4 : 2, BSTEP = BMN ? 2048 >> 4 : 2;      // 16 contraction indices
    if (rank == 0) for (long t = blockIdx.x >> 1; ok && item(t, w); t += gridDim.x >> 1) {      // the first block issues for both
      const uint32_t idesc = w.half < 0 ? P.idesc : P.idesc_half, slot = lt & 1, u = lt >> 1; lt++;
      if (!mbar_wait(tempty0 + 8 * slot, (u & 1) ^ 1, limit, abort_flag)) { ok = false; break; }
      tc_fence_after();
      const uint32_t acc = tmem_base + slot * BN;
      for (int k = w.k0; k < w.k1; k++) {
        if (!mbar_wait(full0 + 8 * s, ph, limit, abort_flag)) { ok = false; break; }
        tc_fence_after();
        if (elected) {
          const uint64_t a = adesc0 + (uint64_t)(s * (STAGE >> 4)), b = bdesc0 + (uint64_t)(s * (STAGE >> 4));
#pragma unroll
          for (int i = 0; i < 4; i++) tc_mma_f16_pair(acc, a + i * ASTEP, b + i * BSTEP, idesc, (k > w.k0 || i > 0) ? 1u : 0u);
          tc_commit_pair(empty0 + 8 * s);
          if (k == w.k1 - 1) tc_commit_pair(tfull0 + 8 * slot);
        }
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
    if (!ok) {
      if (!*abort_flag) give_up();
      if (elected) { tc_commit_pair(drain); mbar_wait(drain, 0, TC_DRAIN_LIMIT); }      // MMAs in flight
    }
    __syncwarp();
  } else {
    const int ew = warp - 2, quad = warp & 3, cg = ew >> 2; uint32_t lt = 0; Item w;
    uint8_t* stg = smem + STAGES * STAGE + ew * Cfg::STG_WARP; const uint32_t stg_addr = smem_u32(stg);
    // this lane's row of the staging buffer, 16-byte unit j of it, as the swizzles of the stores' maps want them
    [[maybe_unused]] auto unit = [&](int j) { return reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)); };
    [[maybe_unused]] auto unit64 = [&](int which, int j) { return reinterpret_cast<uint4*>(stg + which * 2048 + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)); };
    auto free_stage = [&]() { if (lane == 0) bulk_wait_read(); __syncwarp(); };
    // g and u of a 32 x 16 block, kept by the forward pass
    auto saved_at = [&](int row, int col) { return reinterpret_cast<uint4*>(P.saved) + ((long)(row >> 5) * P.saved_cols + (col >> 4)) * FG_SAVED + lane; };
    auto row_of = [&](const Item& i) { return i.m0 + (int)rank * 128 + quad * 32; };
    auto first_col = [&](const Item& i) { return cg * (Cfg::COLS >> (i.half >= 0)); };      // of this warp's, in the tile
    uint4 gn_[3], un_[3];                                            // dh: those of the next block
    auto fetch = [&](const Item& i, int col) {
      if (row_of(i) < P.p[i.q].M && col < P.p[i.q].N) {
        const uint4* q = saved_at(row_of(i), col);
#pragma unroll
        for (int j = 0; j < 3; j++) { gn_[j] = __ldcs(q + j * 32); un_[j] = __ldcs(q + (3 + j) * 32); }
      }
    };
    long t = blockIdx.x >> 1; Item next; bool more = item(t, next);
    if constexpr (KIND == FG_GATE_BWD) { if (more) fetch(next, next.n0 + first_col(next)); }
    while (more) {
      w = next; t += gridDim.x >> 1; more = item(t, next);
      const FgProblem& p = P.p[w.q]; const uint32_t slot = lt & 1, u = lt >> 1; lt++;
      const int row0 = row_of(w), c0 = first_col(w), c1 = c0 + (Cfg::COLS >> (w.half >= 0)); const uint32_t acc = tmem_base + slot * BN + ((uint32_t)(quad * 32) << 16);
      int got = 1;
      if (lane == 0) got = mbar_wait(tfull0 + 8 * slot, u & 1, limit, abort_flag) ? 1 : 0;
      got = __shfl_sync(0xffffffffu, got, 0);
      if (!got) { if (lane == 0 && !*abort_flag) give_up(); break; }
      tc_fence_after();
      auto release = [&]() { tc_fence_before(); __syncwarp(); if (lane == 0) mbar_arrive_cluster(lead_tempty0 + 8 * slot); };
      if constexpr (KIND == FG_PLAIN) {
        if (P.partial) {
          float4* out = reinterpret_cast<float4*>(P.partial) + (long)w.slot * (FG_BM * BN / 4) + ((rank * 4 + quad) * (BN / 32)) * 256 + lane;
#pragma unroll 1
          for (int c = c0; c < c1; c += 32) {
            uint32_t r[32]; tmem_ld32(acc + c, r);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int j = 0; j < 8; j++) out[(c >> 5) * 256 + j * 32] = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
          }
          release();
        } else {
#pragma unroll 1
          for (int c = c0; c < c1; c += 64) {
            uint32_t r[32], q[32]; tmem_ld32(acc + c, r); tmem_ld32(acc + c + 32, q);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (c + 64 >= c1) release();
            free_stage();
#pragma unroll
            for (int j = 0; j < 4; j++) {
              auto f = [](uint32_t v) { return __uint_as_float(v); };
              *unit(j) = make_uint4(pack2(f(r[8 * j]), f(r[8 * j + 1]), T()), pack2(f(r[8 * j + 2]), f(r[8 * j + 3]), T()), pack2(f(r[8 * j + 4]), f(r[8 * j + 5]), T()), pack2(f(r[8 * j + 6]), f(r[8 * j + 7]), T()));
              *unit(4 + j) = make_uint4(pack2(f(q[8 * j]), f(q[8 * j + 1]), T()), pack2(f(q[8 * j + 2]), f(q[8 * j + 3]), T()), pack2(f(q[8 * j + 4]), f(q[8 * j + 5]), T()), pack2(f(q[8 * j + 6]), f(q[8 * j + 7]), T()));
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M && w.n0 + c < p.N) { tma_store_2d(&p.d0, w.n0 + c, row0, stg_addr); bulk_commit(); }
          }
        }
      } else if constexpr (KIND == FG_GATE) {
        free_stage();
#pragma unroll
        for (int c = 0; c < Cfg::COLS; c += 16) {
          const int col = w.n0 + c0 + c;
          uint32_t g[16], v[16]; tmem_ld16(acc + c0 + c, g); tmem_ld16(acc + BN / 2 + c0 + c, v);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if (c + 16 >= Cfg::COLS) release();
          if (P.saved && row0 < p.M && col < p.N) {
            uint4 *s = saved_at(row0, col), q[3];
            fg_pack24(g, q);
#pragma unroll
            for (int j = 0; j < 3; j++) __stcs(s + j * 32, q[j]);
            fg_pack24(v, q);
#pragma unroll
            for (int j = 0; j < 3; j++) __stcs(s + (3 + j) * 32, q[j]);
          }
#pragma unroll
          for (int j = 0; j < 2; j++) {
            float h[8];
#pragma unroll
            for (int l = 0; l < 8; l++) h[l] = fg_act<ACT>(__uint_as_float(g[8 * j + l])) * __uint_as_float(v[8 * j + l]);
            *unit64(0, c / 8 + j) = make_uint4(pack2(h[0], h[1], T()), pack2(h[2], h[3], T()), pack2(h[4], h[5], T()), pack2(h[6], h[7], T()));
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0 && row0 < p.M && w.n0 + c0 < p.N) { tma_store_2d(&p.d0, w.n0 + c0, row0, stg_addr); bulk_commit(); }
      } else {
#pragma unroll 1
        for (int c = c0; c < c1; c += 16) {
          const int col = w.n0 + c; const bool odd = (c - c0) & 16;      // blocks of 32 columns go out, their halves one after the other
          uint4 g[3], v[3];
#pragma unroll
          for (int j = 0; j < 3; j++) { g[j] = gn_[j]; v[j] = un_[j]; }
          if (c + 16 < c1) fetch(w, col + 16); else if (more) fetch(next, next.n0 + first_col(next));      // on its way while this one is worked on
          uint32_t r[16]; tmem_ld16(acc + c, r);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if (c + 16 >= c1) release();
          uint32_t dg[8], du[8];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            float a[2], b[2];
#pragma unroll
            for (int l = 0; l < 2; l++) {
              float av, da; fg_act_grad<ACT>(fg_unpack24(g, 2 * j + l), av, da);
              const float d = __uint_as_float(r[2 * j + l]); a[l] = d * fg_unpack24(v, 2 * j + l) * da; b[l] = d * av;
            }
            dg[j] = pack2(a[0], a[1], T()); du[j] = pack2(b[0], b[1], T());
          }
          if (!odd) free_stage();
#pragma unroll
          for (int j = 0; j < 2; j++) {
            *unit64(0, 2 * odd + j) = make_uint4(dg[4 * j], dg[4 * j + 1], dg[4 * j + 2], dg[4 * j + 3]);
            *unit64(1, 2 * odd + j) = make_uint4(du[4 * j], du[4 * j + 1], du[4 * j + 2], du[4 * j + 3]);
          }
          if (odd) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M && col - 16 < p.N) { tma_store_2d(&p.d0, col - 16, row0, stg_addr); tma_store_2d(&p.d1, col - 16, row0, stg_addr + 2048); bulk_commit(); }
          }
        }
      }
    }
    if (lane == 0) bulk_wait();                                      // the stores read this block's shared memory
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                                // neither block's barriers are needed any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)Cfg::TMEM) : "memory");
  }
}

// Sums of the slices in order, rounded once.  A block: one tile's 32 rows x BN columns; a thread 16 columns of a row.
struct FgReduce { const float* partial; int splits, problems; struct { void* out; long ld; int M, N, tiles_n, tiles; } p[3]; };
template <class T, int BN>
__global__ void __launch_bounds__(2 * BN) fg_reduce_kernel(const __grid_constant__ FgReduce R) {
  op_begin();
  int tile = blockIdx.x >> 3, q = 0; const int quad = blockIdx.x & 7, lane = threadIdx.x & 31, c16 = threadIdx.x >> 5;
  const float4* src = reinterpret_cast<const float4*>(R.partial) + (long)tile * R.splits * (FG_BM * BN / 4) + (quad * (BN / 32) + (c16 >> 1)) * 256 + (c16 & 1) * 128 + lane;
  while (q + 1 < R.problems && tile >= R.p[q].tiles) { tile -= R.p[q].tiles; q++; }
  const int mt = tile / R.p[q].tiles_n, nt = tile - mt * R.p[q].tiles_n, row = mt * FG_BM + quad * 32 + lane, col = nt * BN + c16 * 16;
  if (row >= R.p[q].M || col >= R.p[q].N) return;
  float4 v[4] = {};
  for (int z = 0; z < R.splits; z++) {
#pragma unroll
    for (int j = 0; j < 4; j++) { const float4 x = __ldcs(src + (long)z * (FG_BM * BN / 4) + j * 32); v[j].x += x.x; v[j].y += x.y; v[j].z += x.z; v[j].w += x.w; }
  }
  uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(R.p[q].out) + (long)row * R.p[q].ld + col);
  out[0] = make_uint4(pack2(v[0].x, v[0].y, T()), pack2(v[0].z, v[0].w, T()), pack2(v[1].x, v[1].y, T()), pack2(v[1].z, v[1].w, T()));
  if (col + 8 < R.p[q].N) out[1] = make_uint4(pack2(v[2].x, v[2].y, T()), pack2(v[2].z, v[2].w, T()), pack2(v[3].x, v[3].y, T()), pack2(v[3].z, v[3].w, T()));
}

// ------------------------------------------------------------------ few tokens
// Up to 16 tokens: the weights are all there is to read.  A warp multiplies 16 rows of a weight matrix by the tokens with warp-level MMAs (m16n8k16, rows of the weights as M), straight from
// global memory: a lane's 16 bytes of a row are eight neighbouring indices, and which of them an MMA takes as which index does not matter as long as the tokens' operand is read alike.
// The warps of a block share the contraction; their sums meet in shared memory.
template <class T> __device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int FEW_WARPS = 8;
// Up to eight tokens h is kept as the sum of two 16-bit numbers, a plane of `tokens` rows for each, and the second launch multiplies by both.  Rounded to 16 bits it would make the error of y some 1.4
// times that of its own rounding, and up to 1.7 for a single token, where few terms make up the sum.  (One token, 1024 x 4096, bf16: 9.2 -> 9.9 us.  For 9 to 16 tokens, whose
// errors average out, it would be 10 to 25 % and is not done.)
// GATE: out[t][n] = act(x w0^T) (x w1^T), else x w0^T.  n in blocks of 16, `cl` blocks of a cluster share the contraction.  NB: blocks of eight tokens.
template <class T, bool GATE, int NB, int ACT>
__global__ void __launch_bounds__(32 * FEW_WARPS) fg_few_kernel(const T* x, long x_stride, const T* w0, const T* w1, int tokens, int N, int K, T* out, long out_stride, int cl) {
  namespace cg = cooperative_groups;
  constexpr int MATS = GATE ? 2 : 1;
  __shared__ float red[FEW_WARPS][MATS * NB][4][32];
  __shared__ float sums[MATS * NB * 128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = blockIdx.x % cl, n0 = (int)(blockIdx.x / cl) * 16;
  float d[MATS][NB][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  constexpr int U = NB == 1 ? 4 : 2;                                 // steps of 32 indices under way
  const int steps = (K + 31) / 32, parts = FEW_WARPS * cl, part = rank * FEW_WARPS + warp, s_end = (int)((long)steps * (part + 1) / parts);
  constexpr int PARTS = !GATE && NB == 1 ? 2 : 1;
  uint4 a[U][MATS][2], b[U][NB][PARTS];
  auto weights = [&](int s0) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int k = (s0 + i) * 32 + q * 8; const bool in = s0 + i < s_end && k < K;      // (K is a multiple of 8)
#pragma unroll
      for (int m = 0; m < MATS; m++)
#pragma unroll
        for (int r = 0; r < 2; r++) { const int n = n0 + g + 8 * r; a[i][m][r] = in && n < N ? __ldcs(reinterpret_cast<const uint4*>((m ? w1 : w0) + (long)n * K + k)) : zero; }
    }
  };
  int s0 = (int)((long)steps * part / parts);
  // The second launch fetches its first weights while the first one still runs.  Whatever wrote them has finished: the first launch lets the second in only behind its own wait.
  if constexpr (GATE) { pdl_wait(); pdl_launch(); weights(s0); } else { pdl_launch(); weights(s0); pdl_wait(); }
  for (; s0 < s_end; s0 += U) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int k = (s0 + i) * 32 + q * 8; const bool in = s0 + i < s_end && k < K;
#pragma unroll
      for (int j = 0; j < NB; j++) {
        const int t = 8 * j + g;
#pragma unroll
        for (int e = 0; e < PARTS; e++) b[i][j][e] = in && t < tokens ? *reinterpret_cast<const uint4*>(x + (t + e * tokens) * x_stride + k) : zero;
      }
    }
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
      for (int m = 0; m < MATS; m++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
          for (int e = 0; e < PARTS; e++) {
            mma_16x8x16<T>(d[m][j], a[i][m][0].x, a[i][m][1].x, a[i][m][0].y, a[i][m][1].y, b[i][j][e].x, b[i][j][e].y);
            mma_16x8x16<T>(d[m][j], a[i][m][0].z, a[i][m][1].z, a[i][m][0].w, a[i][m][1].w, b[i][j][e].z, b[i][j][e].w);
          }
    if (s0 + U < s_end) weights(s0 + U);
  }
#pragma unroll
  for (int m = 0; m < MATS; m++)
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) red[warp][m * NB + j][e][lane] = d[m][j][e];
  __syncthreads();
  for (int e = threadIdx.x; e < MATS * NB * 128; e += 32 * FEW_WARPS) {
    float v = 0.f;
    for (int w = 0; w < FEW_WARPS; w++) v += (&red[w][0][0][0])[e];
    sums[e] = v;
  }
  if (cl > 1) cg::this_cluster().sync(); else __syncthreads();
  if (rank == 0)
    for (int e = threadIdx.x; e < NB * 128; e += 32 * FEW_WARPS) {
      const int j = e / 128, i = e / 32 % 4, l = e % 32, n = n0 + (l >> 2) + (i & 2 ? 8 : 0), t = 8 * j + (l & 3) * 2 + (i & 1);      // accumulator i of lane l: row l / 4 (+ 8), column 2 (l % 4) (+ 1)
      float v[MATS];
#pragma unroll
      for (int m = 0; m < MATS; m++) {
        v[m] = sums[m * NB * 128 + e];
        for (int r = 1; r < cl; r++) v[m] += cg::this_cluster().map_shared_rank(sums, r)[m * NB * 128 + e];
      }
      if (n < N && t < tokens) {
        const float y = GATE ? fg_act<ACT>(v[0]) * v[MATS - 1] : v[0]; const T hi = from_f32<T>(y);
        out[t * out_stride + n] = hi;
        if constexpr (GATE && NB == 1) { const float r = y - to_f32(hi); out[(t + tokens) * out_stride + n] = from_f32<T>(isinf(to_f32(hi)) ? 0.f : r); }      // (what 16 bits cannot hold is infinite by itself)
      }
    }
  if (cl > 1) cg::this_cluster().sync();                             // (the others' sums have been read)
}

// ------------------------------------------------------------------ host side
typedef CUresult (*FgEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// A [rows, cols] matrix of 16-bit elements, rows `ld` apart, read or written in boxes of box_rows x box_cols.
inline int fg_map(const Ctx& c, CUtensorMap* map, bool bf16, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, int box_cols) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(rows > 1 ? ld : cols) * 2}; const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, es[2] = {1, 1};
  const CUresult r = ((FgEncode)c.encode_tiled)(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? GN_OK : fail(GN_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d (%ld x %ld, rows %ld apart)", (int)r, (long)rows, (long)cols, (long)ld);
}
struct FgMatrix { const void* p; int64_t rows, cols, ld; };
// One product of a launch: D [M, N] = A B over K, operands as they lie in memory: a K-major operand is [M or N, K], an MN-major one [K, M or N].
struct FgProduct { FgMatrix a0, a1, b0, b1, d0, d1; int64_t M, N, K; };

template <class T, int BN, bool AMN, bool BMN, FgKind KIND, int ACT>
inline int fg_launch_bn(gn_ctx* ctx, const FgProduct* pr, int n, const FfnCut& cut, FgParams& P, void* stream) {
  using Cfg = FgCfg<BN, KIND>; constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value; const Ctx& c = ctx->c;
  P.problems = n; P.splits = cut.splits; P.spin_limit = c.spin_limit;
  P.idesc = fg_idesc(bf16, AMN, BMN, BN); P.idesc_half = fg_idesc(bf16, AMN, BMN, BN / 2);
  int64_t total = 0;
  for (int i = 0; i < n; i++) {
    FgProblem& q = P.p[i]; const FgProduct& w = pr[i];
    auto operand = [&](CUtensorMap* m, const FgMatrix& x, bool mn, int box) { return x.p ? fg_map(c, m, bf16, x.p, x.rows, x.cols, x.ld, mn ? 64 : box, 64) : GN_OK; };
    GN_TRY(operand(&q.a0, w.a0, AMN, 128)); GN_TRY(operand(&q.a1, w.a1, AMN, 128)); GN_TRY(operand(&q.b0, w.b0, BMN, 64)); GN_TRY(operand(&q.b1, w.b1, BMN, 64));
    const int dbox = KIND == FG_PLAIN ? 64 : 32;
    if (w.d0.p && !P.partial) GN_TRY(fg_map(c, &q.d0, bf16, w.d0.p, w.d0.rows, w.d0.cols, w.d0.ld, 32, dbox));
    if (w.d1.p) GN_TRY(fg_map(c, &q.d1, bf16, w.d1.p, w.d1.rows, w.d1.cols, w.d1.ld, 32, dbox));
    q.M = (int)w.M; q.N = (int)w.N; q.kb0 = (int)ceil_div(w.K, FG_BK); q.kb = q.kb0 * (KIND == FG_PLAIN && w.a1.p ? 2 : 1);
    q.tiles_n = (int)ceil_div(w.N, KIND == FG_GATE ? BN / 2 : BN); q.tiles = (int)(ceil_div(w.M, FG_BM) * q.tiles_n); total += q.tiles;
  }
  const int64_t items = total * cut.splits;
  if (items > 0x7fffffff) return fail(GN_ERR_UNSUPPORTED, "gated_ffn: too many output tiles");
  P.n_half = KIND == FG_GATE || BN < 256 || P.partial ? 0 : (int)(2 * ffn_tail(items, ffn_pairs(c.sm_count))); P.full = (int)(items - P.n_half / 2);
  auto kernel = fg_gemm_kernel<T, BN, AMN, BMN, KIND, ACT>;
  GN_TRY(op_smem("gated_ffn", kernel, Cfg::SMEM));
  GN_TRY(op_launch("gated_ffn", stream, kernel, dim3((unsigned)(2 * std::min<int64_t>(P.full + P.n_half, ffn_pairs(c.sm_count)))), dim3(Cfg::THREADS), Cfg::SMEM, 0, P));
  if (!P.partial) return GN_OK;
  FgReduce R{P.partial, cut.splits, n, {}};
  for (int i = 0; i < n; i++) { R.p[i].out = const_cast<void*>(pr[i].d0.p); R.p[i].ld = pr[i].d0.ld; R.p[i].M = P.p[i].M; R.p[i].N = P.p[i].N; R.p[i].tiles_n = P.p[i].tiles_n; R.p[i].tiles = P.p[i].tiles; }
  return op_launch("gated_ffn_reduce", stream, fg_reduce_kernel<T, BN>, dim3((unsigned)(total * 8)), dim3(2 * BN), 0, 0, R);
}
// products [M, N] of one shape class, plain output
template <class T, bool AMN, bool BMN>
inline int fg_plain(gn_ctx* ctx, const FgProduct* pr, int n, const FfnCut& cut, float* partial, void* stream) {
  FgParams P{}; P.partial = cut.splits > 1 ? partial : nullptr;
  return cut.bn == 256 ? fg_launch_bn<T, 256, AMN, BMN, FG_PLAIN, GN_ACT_LINEAR>(ctx, pr, n, cut, P, stream) : fg_launch_bn<T, 128, AMN, BMN, FG_PLAIN, GN_ACT_LINEAR>(ctx, pr, n, cut, P, stream);
}

template <class T, int ACT>
inline int ffn_forward(gn_ctx* ctx, int64_t M, int D, int F, const void* x, int64_t xs, const void* wg, const void* wu, const void* wd, void* y, int64_t ys, uint8_t* saved, uint8_t* ws, void* stream) {
  const FfnPlan& pl = ffn_plan(M, D, F, ctx->c.sm_count);
  void* h = saved ? saved + pl.saved_h : ws + pl.fwd_h;
  if (!saved && M <= FFN_FEW_TOKENS) {
    auto few = [&](auto kernel, const void* in, int64_t in_s, const void* a, const void* b, int N, int K, void* out, int64_t os) {
      const int cl = ffn_few_cluster(N, K, ctx->c.sm_count);
      return op_launch("gated_ffn_few", stream, kernel, dim3((unsigned)(ceil_div(N, 16) * cl)), dim3(32 * FEW_WARPS), 0, cl, static_cast<const T*>(in), (long)in_s, static_cast<const T*>(a), static_cast<const T*>(b), (int)M, N, K, static_cast<T*>(out), (long)os, cl);
    };
    if (M <= FFN_FEW_TOKENS / 2) { GN_TRY(few(fg_few_kernel<T, true, 1, ACT>, x, xs, wg, wu, F, D, h, F)); return few(fg_few_kernel<T, false, 1, GN_ACT_LINEAR>, h, F, wd, nullptr, D, F, y, ys); }
    GN_TRY(few(fg_few_kernel<T, true, 2, ACT>, x, xs, wg, wu, F, D, h, F)); return few(fg_few_kernel<T, false, 2, GN_ACT_LINEAR>, h, F, wd, nullptr, D, F, y, ys);
  }
  const FgMatrix none{};
  FgParams P{}; P.saved = saved; P.saved_cols = (int)ceil_div(F, 16);
  const FgProduct gate{{x, M, D, xs}, none, {wg, F, D, D}, {wu, F, D, D}, {h, M, F, F}, none, M, F, D};
  GN_TRY((fg_launch_bn<T, 256, false, false, FG_GATE, ACT>(ctx, &gate, 1, FfnCut{256, 1}, P, stream)));
  const FgProduct down{{h, M, F, F}, none, {wd, D, F, F}, none, {y, M, D, ys}, none, M, D, F};
  return fg_plain<T, false, false>(ctx, &down, 1, pl.y, reinterpret_cast<float*>(ws + pl.fwd_partial), stream);
}

template <class T, int ACT>
inline int ffn_backward(gn_ctx* ctx, int64_t M, int D, int F, const void* dy, int64_t dys, const void* x, int64_t xs, const void* wg, const void* wu, const void* wd, const uint8_t* saved,
                        void* dx, int64_t dxs, void* dwg, void* dwu, void* dwd, uint8_t* ws, void* stream) {
  const FfnPlan& pl = ffn_plan(M, D, F, ctx->c.sm_count);
  void *dg = ws + pl.bwd_dg, *du = ws + pl.bwd_du; const void* h = saved + pl.saved_h; float* partial = reinterpret_cast<float*>(ws + pl.bwd_partial);
  const FgMatrix none{};
  if (dx || dwg || dwu) {
    FgParams P{}; P.saved = const_cast<uint8_t*>(saved); P.saved_cols = (int)ceil_div(F, 16);
    const FgProduct dh{{dy, M, D, dys}, none, {wd, D, F, F}, none, {dg, M, F, F}, {du, M, F, F}, M, F, D};
    GN_TRY((fg_launch_bn<T, 256, false, true, FG_GATE_BWD, ACT>(ctx, &dh, 1, FfnCut{256, 1}, P, stream)));
  }
  if (dx) {
    const FgProduct p{{dg, M, F, F}, {du, M, F, F}, {wg, F, D, D}, {wu, F, D, D}, {dx, M, D, dxs}, none, M, D, F};
    GN_TRY((fg_plain<T, false, true>(ctx, &p, 1, pl.dx, partial, stream)));
  }
  FgProduct w[3]; int n = 0;
  if (dwg) w[n++] = FgProduct{{dg, M, F, F}, none, {x, M, D, xs}, none, {dwg, F, D, D}, none, F, D, M};
  if (dwu) w[n++] = FgProduct{{du, M, F, F}, none, {x, M, D, xs}, none, {dwu, F, D, D}, none, F, D, M};
  if (dwd) w[n++] = FgProduct{{dy, M, D, dys}, none, {h, M, F, F}, none, {dwd, D, F, F}, none, D, F, M};
  return n ? fg_plain<T, true, true>(ctx, w, n, pl.dw, partial, stream) : GN_OK;
}

template <class F> inline int with_half_and_activation(int dtype, int activation, F&& f) {
  auto act = [&](auto t) {
    return activation == GN_ACT_SILU ? f(t, std::integral_constant<int, GN_ACT_SILU>()) : activation == GN_ACT_GELU ? f(t, std::integral_constant<int, GN_ACT_GELU>()) : f(t, std::integral_constant<int, GN_ACT_RELU>());
  };
  return dtype == GN_F16 ? act(__half()) : act(__nv_bfloat16());
}

}  // namespace gn

extern "C" {

int gn_op_gated_ffn_saved(gn_ctx* ctx, int64_t tokens, int dim, int ff, int64_t* bytes) {
  using namespace gn;
  if (!ctx || !ctx->alive || !bytes) return fail(GN_ERR_INVALID_ARG, "op_gated_ffn_saved: bad argument");
  if (const char* e = check_ffn_sizes(tokens, dim, ff)) return fail(GN_ERR_INVALID_ARG, "op_gated_ffn_saved: %s", e);
  *bytes = ffn_plan(tokens, dim, ff, ctx->c.sm_count).saved; return GN_OK;
}

int gn_op_gated_ffn_workspace(gn_ctx* ctx, int64_t tokens, int dim, int ff, int backward, int64_t* bytes) {
  using namespace gn;
  if (!ctx || !ctx->alive || !bytes) return fail(GN_ERR_INVALID_ARG, "op_gated_ffn_workspace: bad argument");
  if (const char* e = check_ffn_sizes(tokens, dim, ff)) return fail(GN_ERR_INVALID_ARG, "op_gated_ffn_workspace: %s", e);
  const FfnPlan& pl = ffn_plan(tokens, dim, ff, ctx->c.sm_count);
  *bytes = backward ? pl.bwd : pl.fwd; return GN_OK;
}

int gn_op_gated_ffn(gn_ctx* ctx, int dtype, int activation, int64_t tokens, int dim, int ff, const void* x, int64_t x_stride, const void* w_gate, const void* w_up, const void* w_down, void* y, int64_t y_stride, void* saved,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace gn;
  if (ctx && ctx->alive && dtype == GN_F32) return fail(GN_ERR_UNSUPPORTED, "op_gated_ffn: there is no 32-bit form, GN_F16 or GN_BF16 is needed");
  const char* wrong = check_ffn(dtype, activation, tokens, dim, ff, {x, w_gate, w_up, w_down, y}, {x_stride, y_stride});
  if (!wrong && !aligned_to(saved, 16)) wrong = "saved is not 16-byte aligned";
  GN_OP_BEGIN("op_gated_ffn", wrong);
  if (!ctx->c.tc_ok) return fail(GN_ERR_UNSUPPORTED, "op_gated_ffn: the tensor-core engine is not available on this context");
  if (tokens == 0) return GN_OK;
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < ffn_plan(tokens, dim, ff, ctx->c.sm_count).fwd) return fail(GN_ERR_INVALID_ARG, "op_gated_ffn: the workspace is too small, null or not aligned");
  uint8_t *s = static_cast<uint8_t*>(saved), *ws = static_cast<uint8_t*>(workspace);
  return with_half_and_activation(dtype, activation, [&](auto t, auto act) { using T = decltype(t); constexpr int A = decltype(act)::value; return ffn_forward<T, A>(ctx, tokens, dim, ff, x, x_stride, w_gate, w_up, w_down, y, y_stride, s, ws, stream); });
}

int gn_op_gated_ffn_backward(gn_ctx* ctx, int dtype, int activation, int64_t tokens, int dim, int ff, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* w_gate, const void* w_up, const void* w_down,
                             const void* saved, void* dx, int64_t dx_stride, void* dw_gate, void* dw_up, void* dw_down, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace gn;
  if (ctx && ctx->alive && dtype == GN_F32) return fail(GN_ERR_UNSUPPORTED, "op_gated_ffn_backward: there is no 32-bit form, GN_F16 or GN_BF16 is needed");
  const char* wrong = check_ffn(dtype, activation, tokens, dim, ff, {dy, x, w_gate, w_up, w_down, saved}, {dy_stride, x_stride});
  if (!wrong && (!aligned_to(dx, 16) || !aligned_to(dw_gate, 16) || !aligned_to(dw_up, 16) || !aligned_to(dw_down, 16))) wrong = "a pointer is not 16-byte aligned";
  if (!wrong && dx) wrong = check_ffn_strides(tokens, dim, {dx_stride});
  GN_OP_BEGIN("op_gated_ffn_backward", wrong);
  if (!ctx->c.tc_ok) return fail(GN_ERR_UNSUPPORTED, "op_gated_ffn_backward: the tensor-core engine is not available on this context");
  if (tokens == 0) {
    for (void* w : {dw_gate, dw_up, dw_down}) if (w) GN_CUDA(cudaMemsetAsync(w, 0, 2UL * dim * ff, (cudaStream_t)stream));
    return GN_OK;
  }
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < ffn_plan(tokens, dim, ff, ctx->c.sm_count).bwd) return fail(GN_ERR_INVALID_ARG, "op_gated_ffn_backward: the workspace is too small, null or not aligned");
  const uint8_t* s = static_cast<const uint8_t*>(saved); uint8_t* ws = static_cast<uint8_t*>(workspace);
  return with_half_and_activation(dtype, activation, [&](auto t, auto act) {
    using T = decltype(t); constexpr int A = decltype(act)::value;
    return ffn_backward<T, A>(ctx, tokens, dim, ff, dy, dy_stride, x, x_stride, w_gate, w_up, w_down, s, dx, dx_stride, dw_gate, dw_up, dw_down, ws, stream);
  });
}

}  // extern "C"
