"""Operators on device memory, without a GPU: the argument checks and the plans of op_rules.cuh (plain C++), and the refusals of the Python functions."""
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r'''
#include <cstdio>
#include "goneuron_b200/csrc/op_rules.cuh"
using namespace gn;
static int bad = 0;
#define OK(x) do { if (const char* e_ = (x)) { bad++; std::printf("line %d: refused: %s\n", __LINE__, e_); } } while (0)
#define NO(x) do { if (!(x)) { bad++; std::printf("line %d: not refused\n", __LINE__); } } while (0)
#define IS(x) do { if (!(x)) { bad++; std::printf("line %d: %s\n", __LINE__, #x); } } while (0)
static void* at(uintptr_t a) { return reinterpret_cast<void*>(a); }

static void qk() {
  gn_heads q{at(4096), 512, 64, 8, 0}, k{at(8192), 512, 64, 2, 0};
  const float* g = (const float*)at(256); const double* f = (const double*)at(512); const void* pos = at(1024);
  const QkArgs a{GN_F16, 10, 64, 64, 1e-5f, &q, &k, g, g, pos, GN_I64, f};
  OK(check_qk(a));
  QkArgs b = a; b.dtype = 3; NO(check_qk(b));
  b = a; b.tokens = -1; NO(check_qk(b));
  b = a; b.tokens = 1LL << 31; NO(check_qk(b));
  for (int size : {0, -1, 1025}) { b = a; b.head_size = size; b.rotated = 0; NO(check_qk(b)); }
  for (int rot : {-2, 63, 66}) { b = a; b.rotated = rot; NO(check_qk(b)); }
  b = a; b.eps = -1.f; NO(check_qk(b)); b.eps = NAN; NO(check_qk(b)); b.eps = INFINITY; NO(check_qk(b));
  b = a; b.q = nullptr; NO(check_qk(b));
  b = a; b.k = nullptr; OK(check_qk(b));
  b = a; b.positions = nullptr; NO(check_qk(b)); b.rotated = 0; OK(check_qk(b));
  b = a; b.frequencies = nullptr; NO(check_qk(b));
  b = a; b.frequencies = (const double*)at(516); NO(check_qk(b));
  b = a; b.index_type = 2; NO(check_qk(b));
  b = a; b.positions = at(1028); NO(check_qk(b)); b.index_type = GN_I32; OK(check_qk(b));
  gn_heads r = q; r.data = at(4097); b = a; b.q = &r; NO(check_qk(b));
  r = q; r.data = nullptr; NO(check_qk(b)); b.tokens = 0; OK(check_qk(b));
  r = q; r.heads = -1; b = a; b.q = &r; NO(check_qk(b));
  r = q; r.token_stride = -512; NO(check_qk(b));
  r = q; r.token_stride = 0; OK(check_qk(b)); NO(check_heads(b, &r, 8, true));      // one row for all: as an input only
  r = q; r.head_stride = 63; NO(check_heads(b, &r, 8, true));
  // heads of a token that reach into the next one's, either way round; side by side, with room between, or as a part of wider rows is fine
  r = q; r.token_stride = 64; NO(check_heads(a, &r, 8, true)); OK(check_heads(a, &r, 8, false)); r.token_stride = 511; NO(check_heads(a, &r, 8, true)); r.token_stride = 512; OK(check_heads(a, &r, 8, true));
  r.token_stride = 64; r.head_stride = 639; NO(check_heads(a, &r, 8, true)); r.head_stride = 640; OK(check_heads(a, &r, 8, true)); r.token_stride = 66; r.head_stride = 657; NO(check_heads(a, &r, 8, true));
  r.head_stride = 658; OK(check_heads(a, &r, 8, true)); r.token_stride = 1024; r.head_stride = 128; OK(check_heads(a, &r, 8, true)); r.token_stride = 960; OK(check_heads(a, &r, 8, true));
  r.token_stride = r.head_stride = INT64_MAX; NO(check_heads(a, &r, 8, true));
  b = a; b.tokens = 1; r = q; r.token_stride = 0; OK(check_heads(b, &r, 8, true)); b = a;
  gn_heads same = q, moved = q; moved.token_stride = 1024; OK(check_in_place(&q, &same)); NO(check_in_place(&q, &moved)); OK(check_in_place(nullptr, &q)); OK(check_in_place(&q, &k));
  NO(check_heads(a, &k, 8, true)); NO(check_heads(a, nullptr, 8, true));
  const gn_heads* all[] = {&q, &k, nullptr};
  IS(qk_group(GN_F16, 64, 64, false, all, 3) == 4); IS(qk_group(GN_F32, 64, 64, false, all, 3) == 8); IS(qk_group(GN_F16, 512, 512, false, all, 3) == 32);
  IS(qk_group(GN_F16, 65, 64, false, all, 3) == 0); IS(qk_group(GN_F16, 64, 24, false, all, 3) == 0); IS(qk_group(GN_F16, 64, 24, true, all, 3) == 4); IS(qk_group(GN_F16, 1024, 0, false, all, 3) == 0);
  gn_heads odd = q; odd.token_stride = 513; all[0] = &odd; IS(qk_group(GN_F16, 64, 64, false, all, 3) == 0);
  odd = q; odd.data = at(4098); IS(qk_group(GN_F16, 64, 64, false, all, 3) == 0);
  all[0] = &q; IS(qk_group(GN_F16, 80, 40, false, all, 3) == 0 && qk_group(GN_F16, 80, 40, false, all, 3, 8) == 16); IS(qk_group(GN_BF16, 80, 44, false, all, 3, 8) == 0); IS(qk_group(GN_BF16, 260, 0, false, all, 3, 8) == 0);
  odd = q; odd.token_stride = 516; all[0] = &odd; IS(qk_group(GN_F16, 64, 64, false, all, 3) == 0 && qk_group(GN_F16, 64, 64, false, all, 3, 8) == 8); odd.data = at(4100); IS(qk_group(GN_F16, 64, 64, false, all, 3, 8) == 0);
  for (long n : {1L, 7L, 1184L, 65536L, 2000000000L}) for (int sms : {1, 148}) for (int group : {0, 4, 32}) for (int heads : {0, 1, 5, 300}) for (int rot : {0, 64, 1024}) {
    const int t = qk_tokens(n, sms, group, heads, QK_HEADS_BWD, rot); const long blocks = qk_blocks(n, sms, t);
    IS(t >= 1 && (long)t * rot * 4 <= 32768); IS(blocks >= 1 && blocks <= (long)sms * QK_PER_SM && blocks <= n); IS(qk_workspace(n, 128, sms) >= blocks * 1024);
  }
}
static void distill() {
  const float *t = (const float*)at(256), *w = (const float*)at(512), *l = (const float*)at(1024); void *x = at(4096), *d = at(1 << 20), *ids = at(2048);
  OK(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, ids, GN_I64, t, w, l, d, 100)); OK(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, ids, GN_I64, t, nullptr, l, nullptr, 0));
  OK(check_distill(GN_BF16, 4, 100, 0, 1.f, x, 0, nullptr, GN_I64, nullptr, w, l, d, 100)); OK(check_distill(GN_F32, 0, 100, 8, 1.f, nullptr, 100, nullptr, GN_I32, nullptr, nullptr, nullptr, nullptr, 0));
  NO(check_distill(9, 4, 100, 8, 1.f, x, 100, ids, GN_I64, t, w, l, d, 100)); NO(check_distill(GN_BF16, -4, 100, 8, 1.f, x, 100, ids, GN_I64, t, w, l, d, 100));
  NO(check_distill(GN_BF16, 4, 0, 8, 1.f, x, 100, ids, GN_I64, t, w, l, d, 100)); NO(check_distill(GN_BF16, 4, 100, 1025, 1.f, x, 100, ids, GN_I64, t, w, l, d, 100));
  for (float tau : {0.f, -1.f, NAN, INFINITY}) NO(check_distill(GN_BF16, 4, 100, 8, tau, x, 100, ids, GN_I64, t, w, l, d, 100));
  NO(check_distill(GN_BF16, 4, 100, 8, 1.f, nullptr, 100, ids, GN_I64, t, w, l, d, 100)); NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, nullptr, GN_I64, t, w, l, d, 100));
  NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, ids, GN_I64, nullptr, w, l, d, 100)); NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, ids, GN_I64, t, w, nullptr, d, 100));
  NO(check_distill(GN_BF16, 4, 100, 8, 1.f, at(4097), 100, ids, GN_I64, t, w, l, d, 100)); NO(check_distill(GN_F32, 4, 100, 8, 1.f, x, 100, ids, GN_I64, t, w, l, at(4098), 100));
  NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, at(2052), GN_I64, t, w, l, d, 100)); NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, ids, 2, t, w, l, d, 100));
  NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, ids, GN_I64, (const float*)at(258), w, l, d, 100)); NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, -1, ids, GN_I64, t, w, l, d, 100));
  NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 100, ids, GN_I64, t, w, l, d, 99)); OK(check_distill(GN_BF16, 1, 100, 8, 1.f, x, 100, ids, GN_I64, t, w, l, d, 0));
  NO(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 104, ids, GN_I64, t, w, l, x, 100)); OK(check_distill(GN_BF16, 4, 100, 8, 1.f, x, 104, ids, GN_I64, t, w, l, x, 104));
  // the blocks' parts hold a row, wherever it begins within 16 bytes
  for (long rows : {1L, 24L, 149L, 100000L}) for (int v = 0; v < 22; v++) for (long vocab = std::max(1L, (1L << v) - 20 * (1 + v / 14)); vocab < (1L << v) + 20; vocab++)
    for (int size : {2, 4}) {
      const DistillPlan p = distill_plan(rows, vocab, size, 148);
      if (p.cluster == 0) { IS(vocab * size > 8L * DISTILL_PART_MOST - 200); continue; }
      const int V = 16 / size;
      IS(p.threads >= 64 && p.threads <= DISTILL_THREADS && p.threads % 32 == 0 && p.per * 16 <= DISTILL_PART_MOST);
      for (int lead = 0; lead < V; lead++) if (ceil_div(lead + vocab, V) > (long)p.cluster * p.per) { bad++; std::printf("vocab %ld rows %ld\n", vocab, rows); }
    }
}
static void embedding() {
  void *x = at(4096), *ids = at(2048), *out = at(1 << 20);
  OK(check_embedding(GN_F16, 5, 100, 33, 1.f, x, 33, 100, ids, GN_I32, out, 33, 5)); OK(check_embedding(GN_F16, 0, 100, 33, 1.f, x, 33, 100, nullptr, GN_I32, nullptr, 33, 0));
  NO(check_embedding(GN_F16, -1, 100, 33, 1.f, x, 33, 100, ids, GN_I32, out, 33, 5)); NO(check_embedding(GN_F16, 5, 0, 33, 1.f, x, 33, 100, ids, GN_I32, out, 33, 5));
  NO(check_embedding(GN_F16, 5, 0x7fffffff, 33, 1.f, x, 33, 100, ids, GN_I32, out, 33, 5)); NO(check_embedding(GN_F16, 5, 100, 0, 1.f, x, 33, 100, ids, GN_I32, out, 33, 5));
  NO(check_embedding(GN_F16, 5, 100, 33, NAN, x, 33, 100, ids, GN_I32, out, 33, 5)); NO(check_embedding(GN_F16, 5, 100, 33, INFINITY, x, 33, 100, ids, GN_I32, out, 33, 5));
  NO(check_embedding(GN_F16, 5, 100, 33, 1.f, nullptr, 33, 100, ids, GN_I32, out, 33, 5)); NO(check_embedding(GN_F16, 5, 100, 33, 1.f, x, 33, 100, nullptr, GN_I32, out, 33, 5));
  NO(check_embedding(GN_F16, 5, 100, 33, 1.f, x, 33, 100, ids, GN_I32, nullptr, 33, 5)); NO(check_embedding(GN_F16, 5, 100, 33, 1.f, x, 33, 100, ids, GN_I32, out, 32, 5));
  NO(check_embedding(7, 5, 100, 33, 1.f, x, 33, 100, ids, GN_I32, out, 33, 5)); NO(check_embedding(GN_F16, 5, 100, 33, 1.f, x, 33, 100, at(2049), GN_I32, out, 33, 5));
  NO(check_embedding(GN_F16, 5, 100, 33, 1.f, x, -33, 100, ids, GN_I32, out, 33, 5));
  for (long n : {1L, 8192L, 8193L, 131072L, 2147483647L}) for (long vocab : {1L, 255L, 256L, 65535L, 65536L, 2147483646L}) for (int dim : {1, 1024}) {
    const EmbeddingPlan p = embedding_plan(n, vocab, dim, 148);
    IS((1LL << p.bits) > vocab && p.passes * SORT_BITS >= p.bits && p.passes <= 4); IS(p.chunk >= 4 && p.chunk <= 64); IS(p.chunks * p.chunk >= n && (p.chunks - 1) * p.chunk < n);
    IS(p.small || p.tiles * SORT_TILE >= n); IS(p.keys % 256 == 0 && p.order >= p.keys + 4 * n && p.partial + p.chunks * 2 * dim * 4 <= p.bytes);
    if (!p.small) IS(p.keys2 >= p.order + 4 * n && p.order2 >= p.keys2 + 4 * n && p.hist >= p.order2 + 4 * n && p.partial >= p.hist + 4 * (p.tiles << SORT_BITS));
  }
}
static void ffn() {
  void *x = at(4096), *w = at(8192), *y = at(16384);
  OK(check_ffn(GN_BF16, GN_ACT_SILU, 5, 64, 128, {x, w, w, w, y}, {64, 72})); OK(check_ffn(GN_F16, GN_ACT_GELU, 1, 8, 8, {x, w, w, w, y}, {0, 1})); OK(check_ffn(GN_F16, GN_ACT_RELU, 0, 8, 8, {nullptr, w}, {0}));
  NO(check_ffn(GN_F32, GN_ACT_SILU, 5, 64, 128, {x, w}, {64})); NO(check_ffn(GN_F16, GN_ACT_TANH, 5, 64, 128, {x, w}, {64})); NO(check_ffn(GN_F16, GN_ACT_SILU, -1, 64, 128, {x, w}, {64}));
  for (int bad : {0, -8, 4, 12, 1 << 25}) { NO(check_ffn(GN_F16, GN_ACT_SILU, 5, bad, 128, {x, w}, {1 << 26})); NO(check_ffn(GN_F16, GN_ACT_SILU, 5, 64, bad, {x, w}, {64})); }
  NO(check_ffn(GN_F16, GN_ACT_SILU, 5, 64, 128, {x, nullptr}, {64})); NO(check_ffn(GN_F16, GN_ACT_SILU, 5, 64, 128, {x, at(4104)}, {64}));
  for (long bad : {0L, 56L, 65L, -64L, 1L << 38}) NO(check_ffn(GN_F16, GN_ACT_SILU, 5, 64, 128, {x, w}, {64, bad}));
  for (long m : {1L, 17L, 128L, 129L, 8192L, 16384L, 100000000L}) for (long d : {8L, 64L, 1024L, 16384L}) for (long f : {8L, 1400L, 4096L}) for (int sms : {1, 148}) {
    const FfnPlan p = ffn_plan(m, d, f, sms);
    const long kb[] = {ceil_div(f, 64), 2 * ceil_div(f, 64), ceil_div(m, 64)}; const FfnCut* cut[] = {&p.y, &p.dx, &p.dw};
    for (int i = 0; i < 3; i++) IS((cut[i]->bn == 128 || cut[i]->bn == 256) && cut[i]->splits >= 1 && cut[i]->splits <= kb[i]);      // no slice is empty
    IS(p.saved_h >= m * f * 6 && p.saved == p.saved_h + round_up(2 * m * f, 256)); IS(p.fwd_partial >= 2 * m * f && p.fwd - p.fwd_partial == ffn_partial({{m, d}}, p.y));
    IS(p.bwd_du >= 2 * m * f && p.bwd_partial >= p.bwd_du + 2 * m * f && p.bwd - p.bwd_partial >= ffn_partial({{m, d}}, p.dx) && p.bwd - p.bwd_partial >= ffn_partial({{f, d}, {f, d}, {d, f}}, p.dw));
  }
  for (int sms : {1, 148}) for (long items : {1L, 147L, 148L, 149L, 222L, 223L, 512L}) { const long h = ffn_tail(items, sms); IS(h >= 0 && 2 * h <= sms && (h == 0 || h == items % sms)); }
  for (long n : {8L, 1024L, 100000L}) for (long k : {8L, 4096L, 100000L}) { const int c = ffn_few_cluster(n, k, 148); IS(c == 1 || c == 2 || c == 4 || c == 8); }
}
int main() { qk(); distill(); embedding(); ffn(); std::printf("%d bad\n", bad); return bad != 0; }
'''


def test_checks_and_plans():
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        open(src, "w").write(SRC)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", ROOT, "-x", "c++", src, "-o", exe])
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout


class _NoDevice:
    """Stands in for a Device where a call must not get as far as the library."""
    device, handle = 0, None


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_python_refusals_need_no_gpu():
    """What a call refuses before it looks where the tensors are; a call with nothing else wrong is refused for that."""
    from goneuron_b200 import operators as ops
    dev, q, ids, freq, half, i32 = _NoDevice(), _t(6, 2, 8), _t(6, dtype=torch.int64), _t(4, dtype=torch.float64), torch.float16, torch.int32
    x, w, d = _t(5, 16, dtype=half), _t(24, 16, dtype=half), _t(16, 24, dtype=half)
    refused = [
        ("runs on cuda:0", lambda: ops.qk_norm_rope(dev, q, q, _t(8), _t(8), ids, freq)), ("runs on cuda:0", lambda: ops.distill_loss(dev, _t(4, 10), _t(4, 3, dtype=i32), _t(4, 3), 1.0, _t(4))),
        ("runs on cuda:0", lambda: ops.embedding(dev, _t(10, 4), ids)), ("runs on cuda:0", lambda: ops.embedding_backward(dev, _t(6, 4), ids, 10)), ("runs on cuda:0", lambda: ops.gated_ffn(dev, x, w, w, d)),
        ("incompatible", lambda: ops.qk_norm_rope(dev, "q", None)), (r"\[tokens, heads, size\]", lambda: ops.qk_norm_rope(dev, _t(6, 8), None)), ("is needed", lambda: ops.qk_norm_rope(dev, q.double(), None)),
        ("last dimension", lambda: ops.qk_norm_rope(dev, q.transpose(1, 2), None)), ("differ", lambda: ops.qk_norm_rope(dev, q, _t(5, 2, 8))), ("differ", lambda: ops.qk_norm_rope(dev, q, _t(6, 2, 8, dtype=half))),
        ("gain_q", lambda: ops.qk_norm_rope(dev, q, None, _t(7))), ("gain_q", lambda: ops.qk_norm_rope(dev, q, None, _t(8, dtype=half))), ("positions", lambda: ops.qk_norm_rope(dev, q, None, None, None, None, freq)),
        ("one for each token", lambda: ops.qk_norm_rope(dev, q, None, None, None, ids[:5], freq)), ("int32 or int64", lambda: ops.qk_norm_rope(dev, q, None, None, None, ids.float(), freq)),
        ("frequencies", lambda: ops.qk_norm_rope(dev, q, None, None, None, ids, freq.float())), ("make one of tokens", lambda: ops.qk_norm_rope(dev, _t(3, 2, 2, 8).transpose(0, 1), None)),
        ("on cpu", lambda: ops.qk_norm_rope(dev, q, None, out=(_t(6, 2, 7), None))), ("on cpu", lambda: ops.qk_norm_rope_backward(dev, _t(6, 1, 8), None, q, None)),
        ("top_logits", lambda: ops.distill_loss(dev, _t(4, 10), _t(4, 3, dtype=torch.int64), _t(4, 2))), ("top_logits", lambda: ops.distill_loss(dev, _t(4, 10), _t(5, 3, dtype=torch.int64), _t(5, 3))),
        ("int32 or int64", lambda: ops.distill_loss(dev, _t(4, 10), _t(4, 3), _t(4, 3))), ("top_logits", lambda: ops.distill_loss(dev, _t(4, 10), _t(4, 3, dtype=i32), _t(4, 3, dtype=half))),
        ("last dimension", lambda: ops.distill_loss(dev, _t(10, 4).t(), _t(4, 3, dtype=i32), _t(4, 3))), ("row_weight", lambda: ops.distill_loss(dev, _t(4, 10), _t(4, 3, dtype=i32), _t(4, 3), 1.0, _t(3))),
        ("out has shape", lambda: ops.distill_loss_grad(dev, _t(4, 10), _t(4, 3, dtype=i32), _t(4, 3), out=_t(4, 9))),
        ("table has shape", lambda: ops.embedding(dev, _t(10), ids)), ("int32 or int64", lambda: ops.embedding(dev, _t(10, 4), ids.float())), ("last dimension", lambda: ops.embedding(dev, _t(10, 4).t(), ids)),
        ("not contiguous", lambda: ops.embedding(dev, _t(10, 4), ids[::2])), ("a row for each id", lambda: ops.embedding_backward(dev, _t(5, 4), ids, 10)), ("is needed", lambda: ops.embedding_backward(dev, _t(6, 4, dtype=i32), ids, 10)),
        ("make one of tokens", lambda: ops.embedding_backward(dev, _t(3, 2, 4).transpose(0, 1), ids.view(2, 3), 10)), ("negative", lambda: ops.embedding_backward(dev, _t(6, 4), ids, -1)),
        ("tanh", lambda: ops.gated_ffn(dev, x, w, w, d, "tanh")), ("32-bit form", lambda: ops.gated_ffn(dev, x.float(), w.float(), w.float(), d.float())), ("w_gate", lambda: ops.gated_ffn(dev, x.bfloat16(), w, w, d)),
        ("w_up", lambda: ops.gated_ffn(dev, x, w[:8], w, d)), ("w_down", lambda: ops.gated_ffn(dev, x, w, w, w.t())), ("w_down", lambda: ops.gated_ffn(dev, x, w, w, w)), ("w_gate", lambda: ops.gated_ffn(dev, x[:, :8], w, w, d)),
        ("make one of tokens", lambda: ops.gated_ffn(dev, _t(3, 4, 32, dtype=half)[:, :, :16].transpose(0, 1), w, w, d)),
    ]
    for message, call in refused:
        with pytest.raises((ValueError, TypeError), match=message):
            call()


def test_a_closed_device_is_a_status_code():
    """Every entry point refuses a null context before anything else."""
    from goneuron_b200 import _lib, build
    build.build()
    lib = _lib.load()
    for name in (n for n in _lib.EXPORTS if n.startswith("gn_op_") and n in lib_device_operators()):
        f = getattr(lib, name)
        assert f(*[t() if t is not None else None for t in f.argtypes]) == -1, name
        assert b"context is null" in lib.gn_last_error() or b"bad argument" in lib.gn_last_error()


def lib_device_operators():
    header = open(os.path.join(ROOT, "include", "goneuron_cuda.h")).read()
    return header[header.index("operators on device memory"):]
