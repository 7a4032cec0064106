"""gn_op_embedding and its gradient against float64: token counts around every change of plan, runs that cross pieces, padding, bad ids, odd widths, views, captured."""
import pytest
import torch

from tests.operator_checks import TYPES, assert_near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def _check(dev, ids, vocab, dim, type, scale, dout=None):
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(vocab + dim)
    t = TYPES[type]
    table = torch.randn(vocab, dim, device="cuda", generator=gen).to(t)
    out = ops.embedding(dev, table, ids, scale=scale)
    flat = ids.reshape(-1).long()
    there = (flat >= 0) & (flat < vocab)
    want = torch.where(there[:, None], table.double()[flat.clamp(0, vocab - 1)] * scale, 0.0)
    assert_near(out.reshape(-1, dim), want, 2.0 ** -24 * want.abs(), "out")
    if dout is None:
        dout = torch.randn(*ids.shape, dim, device="cuda", generator=gen).to(t)
    d = ops.embedding_backward(dev, dout, ids, vocab, scale=scale)
    rows = dout.reshape(-1, dim).double()[there] * scale
    want, size = (torch.zeros(vocab, dim, dtype=torch.float64, device="cuda").index_add_(0, flat[there], r) for r in (rows, rows.abs()))
    # a row's sum: the additions of a piece of 4 to 64 places (as embedding_plan cuts them), then those of up to 32 pieces or a quarter of them all, and four more; two products
    chunk = 4
    while chunk < 64 and flat.numel() > chunk * 8 * 148:
        chunk *= 2
    longest = chunk + max(32, flat.numel() / chunk / 4) + 8
    assert_near(d, want, 2.0 ** -24 * longest * size, "dtable")
    assert torch.equal(d, ops.embedding_backward(dev, dout, ids, vocab, scale=scale))
    return out, d


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (1, 50000, 64), (2, 3, 8), (31, 17, 300), (33, 255, 64), (1000, 256, 24), (1024, 257, 33), (4737, 700, 40), (8192, 65535, 16), (8193, 65536, 16),
                                              (20000, 5, 1032), (30001, 300, 12), (70000, 32000, 8), (262144, 4000, 8), (262145, 70000, 8)])
def test_against_float64(dev, type, tokens, vocab, dim):
    gen = torch.Generator("cuda").manual_seed(tokens)
    ids = (torch.rand(tokens, device="cuda", generator=gen) ** 2 * vocab).long().clamp_(max=vocab - 1)
    ids[::7] = -1
    _check(dev, ids, vocab, dim, type, 1.75)
    if tokens < 5000:
        _check(dev, ids.int(), vocab, dim, type, 1.0)


@pytest.mark.parametrize("tokens", [5, 127, 128, 129, 130, 131, 4097, 7165, 7167, 7168, 7169])
def test_places_of_equal_ids(dev, tokens):
    """Token counts on either side of those at which places are found another way, many tokens of an id: a sum is that of every one of its tokens, once."""
    gen = torch.Generator("cuda").manual_seed(tokens)
    ids = torch.randint(-1, 40, (tokens,), device="cuda", generator=gen)
    _check(dev, ids, 40, 8, "f32", 1.0)
    _check(dev, ids.sort(descending=True).values, 40, 8, "f16", 1.0)
    _check(dev, torch.arange(tokens, device="cuda").flip(0), tokens, 8, "bf16", 1.0)


@pytest.mark.parametrize("tokens", [64, 5000, 40000])
def test_orders_that_cross_pieces(dev, tokens):
    """One token everywhere, runs of every length, nothing but padding, a token at the last row."""
    gen = torch.Generator("cuda").manual_seed(1)
    _check(dev, torch.full((tokens,), 3, device="cuda"), 9, 48, "f32", 0.5)
    _check(dev, torch.full((tokens,), -1, device="cuda"), 9, 48, "bf16", 0.5)
    runs = torch.repeat_interleave(torch.arange(400, device="cuda"), torch.arange(400, device="cuda"))[:tokens]
    _check(dev, runs[torch.randperm(runs.numel(), device="cuda", generator=gen)], 400, 20, "f32", 2.0)
    _check(dev, torch.randint(998, 1000, (tokens,), device="cuda", generator=gen), 1000, 16, "f16", 2.0)


def test_shapes_views_and_wide_rows(dev):
    gen = torch.Generator("cuda").manual_seed(2)
    ids = torch.randint(0, 50, (6, 11), device="cuda", generator=gen)
    wide = torch.randn(66, 200, device="cuda", generator=gen).bfloat16()
    _check(dev, ids, 50, 96, "bf16", 1.5, wide[:, 8:104].view(6, 11, 96))
    _check(dev, ids, 50, 96, "bf16", 1.5, wide[:, 7:103].view(6, 11, 96))      # rows that 16-byte accesses do not fit
    _check(dev, ids, 50, 96, "f32", 1.5, torch.randn(1, 1, 96, device="cuda", generator=gen).expand(66, 1, 96).view(6, 11, 96))
    _check(dev, torch.randint(0, 20, (40,), device="cuda", generator=gen), 20, 5000, "f16", 1.0)


def test_id_out_of_range_is_reported(dev):
    from goneuron_b200 import _lib, operators as ops
    table, ids = torch.randn(100, 32, device="cuda"), torch.tensor([3, 100, -1, -2, 99], device="cuda")
    out = ops.embedding(dev, table, ids)
    with pytest.raises(_lib.GoNeuronCudaError):
        ops.check(dev)
    assert float(out[[1, 2, 3]].abs().sum()) == 0 and torch.equal(out[0], table[3]) and torch.equal(out[4], table[99])
    d = ops.embedding_backward(dev, torch.ones(5, 32, device="cuda"), ids, 100)
    with pytest.raises(_lib.GoNeuronCudaError):
        ops.check(dev)
    ops.check(dev)
    assert float(d.sum()) == 64 and float(d[[3, 99]].sum()) == 64
    ops.embedding(dev, table, torch.tensor([1 << 40, (1 << 32) + 3], device="cuda"))
    with pytest.raises(_lib.GoNeuronCudaError):
        ops.check(dev)


def test_offsets_beyond_32_bits(dev):
    """A table and a gradient of more than 2^32 bytes and 2^31 elements."""
    from goneuron_b200 import operators as ops
    vocab, dim = 300000, 8192
    table = torch.zeros(vocab, dim, device="cuda", dtype=torch.float16)
    ids = torch.tensor([0, vocab - 1, 270001, vocab - 1], device="cuda")
    table[vocab - 1], table[270001] = 2.0, 3.0
    assert ops.embedding(dev, table, ids).float().mean(1).tolist() == [0.0, 2.0, 3.0, 2.0]
    del table
    d = ops.embedding_backward(dev, torch.ones(4, dim, device="cuda", dtype=torch.float16), ids, vocab)
    assert d[[0, vocab - 1, 270001, 5]].mean(1).tolist() == [1.0, 2.0, 1.0, 0.0] and float(d.sum(dtype=torch.float64)) == 4 * dim


def test_streams_and_graphs(dev):
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(3)
    for tokens in (500, 9000):
        table, dout = torch.randn(2000, 64, device="cuda", generator=gen), torch.randn(tokens, 64, device="cuda", generator=gen)
        ids = torch.randint(0, 2000, (tokens,), device="cuda", generator=gen)
        both = lambda: (ops.embedding(dev, table, ids, 2.0), ops.embedding_backward(dev, dout, ids, 2000, 2.0))
        want = both()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = both()
        s.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, other))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = both()
        ids.copy_((ids * 7 + 1) % 2000)
        g.replay()
        again = both()
        assert all(torch.equal(x, y) for x, y in zip(held, again)) and not torch.equal(held[1], want[1])


def test_no_tokens(dev):
    from goneuron_b200 import operators as ops
    ids = torch.empty(0, device="cuda", dtype=torch.int64)
    assert ops.embedding(dev, torch.randn(5, 8, device="cuda"), ids).shape == (0, 8)
    assert float(ops.embedding_backward(dev, torch.empty(0, 8, device="cuda"), ids, 5).abs().sum()) == 0
