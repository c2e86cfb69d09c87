"""Token scores (fmd_op_logprobs) against 64-bit numpy.

Tolerance: d = x - max is one rounding of f32 inputs (exact for most); each
exponential is off by 2^-22 of its value at most (the product with log2 e, half
an ulp of an exponent below 128, then one ulp), the sum S of them by another
~20 roundings (16 values a thread and tile, then joins): S (1 + 2^-18).  log1p
turns that into at most 2^-18 absolute and, where S is small, 2^-18 S -- so
|logp - want| <= 2^-18 min(1, S) + 2^-23 |want|, entropy the same with T's
weight: 2^-17 (1 + |H|).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TDT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def model(fmd):
    cfg = fmd.TextConfig(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=1,
                         num_attention_heads=2, num_key_value_heads=2, head_dim=128)
    return fmd.Qwen3(cfg, "bf16", max_len=64)


def scores(model, x, dtype, targets, top, ld=None):
    """x: the device rows (a view may have its own stride)."""
    n, v = x.shape
    t = torch.tensor(targets, dtype=torch.int32).cuda()
    logp, ent = torch.full((n + 1,), 9.0).cuda(), torch.full((n + 1,), 9.0).cuda()
    ids = torch.full((n + 1, max(top, 1)), -7, dtype=torch.int32).cuda()
    best = torch.full((n + 1, max(top, 1)), 9.0).cuda()
    torch.cuda.synchronize()
    model.op_logprobs(x.data_ptr(), dtype, n, v, t.data_ptr(), top, logp.data_ptr(), ent.data_ptr(),
                      ids.data_ptr() if top else None, best.data_ptr() if top else None, ld=ld)
    torch.cuda.synchronize()
    for o, u in ((logp, 9.0), (ent, 9.0), (ids, -7), (best, 9.0)):
        assert (o[n:] == u).all(), "rows behind the last were written"
    return [o[:n].cpu().numpy() for o in (logp, ent, ids, best)]


def expect(x, targets, top):
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.exp(x - m)
        at = np.argmax(x, -1)
        rest = e.copy()
        rest[np.arange(len(x)), at] = 0.0
        s = rest.sum(-1)
        lse = np.log1p(s)
        d = x - m
        ent = lse - np.where(e > 0, e * d, 0.0).sum(-1) / (1 + s)
        lp = d[np.arange(len(x)), targets] - lse
    order = np.argsort(-(x + 0.0), -1, kind="stable")[:, :top]
    return lp, ent, order, np.take_along_axis(d, order, -1) - lse[:, None], s


def check(model, xt, dtype, targets, top, ld=None):
    got = scores(model, xt, dtype, targets, top, ld)
    lp, ent, ids, best, s = expect(xt.double().cpu().numpy(), np.asarray(targets), top)
    small = 2.0 ** -18 * np.minimum(1.0, s)
    assert (np.abs(got[0] - lp) <= small + 2.0 ** -23 * np.abs(lp)).all()
    assert (np.abs(got[1] - ent) <= 2.0 ** -17 * (1 + ent) * np.minimum(1, s + ent)).all()
    if top:
        assert np.array_equal(got[2], ids)
        ok = np.isfinite(best)
        assert (np.abs(got[3] - best)[ok] <= (small[:, None] + 2.0 ** -23 * np.abs(best))[ok]).all()
        assert np.array_equal(got[3][~ok], best[~ok])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 7), (2, 4096, 5), (5, 4097, 32), (1, 151936, 20),
                                            (8, 151936, 5), (40, 9999, 8), (1100, 523, 3), (3, 30001, 0)])
def test_scores(model, dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(rows * 7 + vocab)
    x = (torch.randn((rows, vocab), generator=g) * 3).to(TDT[dtype])
    x[0, vocab // 2] = 25.0     # a confident row
    targets = torch.randint(0, vocab, (rows,), generator=g).tolist()
    targets[0] = vocab // 2
    targets[-1] = int(x[-1].float().argmax())
    check(model, x.cuda(), dtype, targets, top)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties_take_the_lower_id(model, dtype):
    """Equal values across threads, tiles and pieces, both zeros among them."""
    x = torch.zeros((3, 20000))
    x[0, 1::2] = -0.0
    x[1, [19999, 3, 4096, 8191, 8192]] = 2.0
    x[2] = torch.arange(20000).float().floor_divide(5000)
    check(model, x.to(TDT[dtype]).cuda(), dtype, [0, 19999, 0], 7)


def test_every_tile_brings_better_ones(model):
    """Rising and falling rows: the alternatives change with every tile, or never after the first."""
    up = torch.arange(70000).float() / 1000
    x = torch.stack([up, -up, up.flip(0)] * 400)[:1100]
    check(model, x.cuda(), "f32", [69999] * 1100, 12)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_ruled_out_tokens(model, dtype):
    g = torch.Generator().manual_seed(5)
    x = torch.randn((4, 9000), generator=g)
    x[torch.rand((4, 9000), generator=g) < 0.6] = -float("inf")
    x[1, :] = -float("inf")
    x[1, [5000, 8999]] = torch.tensor([1.0, 2.0])   # fewer tokens left than alternatives
    x[2, 1:] = -float("inf")
    x[2, 0] = -3.0
    x[:, 10] = x[:, 10].clamp(min=-2.0)
    x[1, 10] = -float("inf")
    check(model, x.to(TDT[dtype]).cuda(), dtype, [10, 5000, 0, 10], 4)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masks_of_the_lowest_value(model, dtype):
    """Tokens at the type's lowest value: scattered, the row's first or last
    thousands (whole lanes, waves and pieces), all but one, all (uniform)."""
    g = torch.Generator().manual_seed(15)
    low = torch.finfo(TDT[dtype]).min
    x = torch.randn((6, 150001), generator=g).to(TDT[dtype])
    x[0, torch.rand(150001, generator=g) < 0.6] = low
    x[1, :90000] = low
    x[2, 400:] = low
    x[3, torch.arange(150001) != 70000] = low
    x[4] = low
    x[5, ::2] = -float("inf")
    x[5, 1::2] = low
    check(model, x.cuda(), dtype, [int(x[0].float().argmax()), 149999, 3, 70000, 5, 7], 4)
    check(model, x[:, :1023].contiguous().cuda(), dtype, [0, 1, 2, 3, 4, 5], 4)


@pytest.mark.parametrize("at", [4000.0, -5000.0, 1e6, -1e6, 1e30, 3e38, -3e38])
def test_large_logits(model, at):
    """Differences of large logits are as good as those of small ones."""
    g = torch.Generator().manual_seed(16)
    x = torch.randn((3, 9000), generator=g) * 3 + at
    check(model, x.cuda(), "f32", [1, 2, 3], 5)
    check(model, x.to(torch.bfloat16).cuda(), "bf16", [1, 2, 3], 5)


def test_rows_without_a_distribution_and_ids_outside(model):
    x = torch.zeros((5, 6000))
    x[0] = -float("inf")
    x[1, 4500] = float("nan")
    x[2, 10] = float("inf")
    x[3] = float("nan")
    logp, ent, ids, best = scores(model, x.cuda(), "f32", [1, 1, 1, 1, -1], 3)
    assert np.isnan(logp).all() and np.isnan(ent[:4]).all() and np.isnan(best[:4]).all()
    assert abs(ent[4] - np.log(6000)) < 1e-5
    assert ids.tolist() == [[0, 1, 2], [0, 1, 2], [10, 0, 1], [0, 1, 2], [0, 1, 2]]
    assert np.isnan(scores(model, x.cuda()[4:], "f32", [6000], 0)[0]).all()


def test_row_stride_and_odd_addresses(model):
    """Rows inside a wider buffer that start at any element."""
    g = torch.Generator().manual_seed(6)
    wide = torch.randn((6, 5003), generator=g).to(torch.bfloat16).cuda()
    check(model, wide[:, 3:4999], "bf16", [0, 1, 2, 3, 4, 4995], 5, ld=5003)


def test_rows_beyond_32_bit_offsets(model):
    """The second row starts 2^31 elements (4 GiB) behind the first."""
    ld = (1 << 31) + 24
    buf = torch.empty(ld + 6000, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(8)
    rows = torch.randn((2, 6000), generator=g).to(torch.bfloat16).cuda()
    buf[:6000], buf[ld:] = rows[0], rows[1]
    view = torch.as_strided(buf, (2, 6000), (ld, 1))
    got, want = scores(model, view, "bf16", [5, 7], 4, ld=ld), scores(model, rows, "bf16", [5, 7], 4)
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_deterministic_and_on_a_callers_stream(model):
    g = torch.Generator().manual_seed(7)
    x = torch.randn((8, 151936), generator=g).cuda()
    a = scores(model, x, "f32", list(range(8)), 6)
    st = torch.cuda.Stream()
    model.set_stream(st.cuda_stream)
    try:
        b = scores(model, x, "f32", list(range(8)), 6)
    finally:
        model.set_stream(None)
    assert all(np.array_equal(p, q) for p, q in zip(a, b))


def test_captured_into_a_graph(model):
    """Replayed with other logits in the same buffer, eager work in between."""
    x = torch.randn((4, 20000)).cuda()
    t = torch.zeros(4, dtype=torch.int32).cuda()
    o = [torch.empty(4).cuda(), torch.empty(4).cuda(), torch.empty((4, 3), dtype=torch.int32).cuda(),
         torch.empty((4, 3)).cuda()]
    call = lambda: model.op_logprobs(x.data_ptr(), "f32", 4, 20000, t.data_ptr(), 3, *[v.data_ptr() for v in o])  # noqa: E731
    torch.cuda.synchronize()
    call()
    st = torch.cuda.Stream()
    model.set_stream(st.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call()
        for i in range(3):
            x.copy_(torch.randn((4, 20000)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = [v.cpu().numpy() for v in o]
            lp, ent, ids, best, s = expect(x.double().cpu().numpy(), np.zeros(4, int), 3)
            assert np.array_equal(got[2], ids) and np.allclose(got[0], lp, rtol=0, atol=2e-5)
            scores(model, x, "f32", [1, 2, 3, 4], 5)     # another call's workspace use
    finally:
        model.set_stream(None)


def test_first_call_is_not_captured(fmd):
    """It allocates; after a call outside a graph the same capture replays."""
    cfg = fmd.TextConfig(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=1,
                         num_attention_heads=2, num_key_value_heads=2, head_dim=128)
    m = fmd.Qwen3(cfg, "bf16", max_len=64)
    st = torch.cuda.Stream()
    m.set_stream(st.cuda_stream)
    x, ent = torch.zeros((2, 500)).cuda(), torch.zeros(2).cuda()
    torch.cuda.synchronize()

    def call():
        m.op_logprobs(x.data_ptr(), "f32", 2, 500, None, 0, None, ent.data_ptr(), None, None)

    try:
        with pytest.raises(fmd.FmdError, match="before capturing"):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                call()
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call()
        for _ in range(3):
            ent.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert np.abs(ent.cpu().numpy() - np.log(500)).max() < 1e-5
    finally:
        m.set_stream(0)


def test_refusals(fmd, model):
    x = torch.zeros((2, 100)).cuda()
    p = x.data_ptr()
    for args, text in (((p, "f32", 2, 100, None, 0, p, None, None, None), "null"),
                       ((p, "f32", 2, 100, p, 33, p, None, p, p), "alternatives"),
                       ((p, "f32", 2, 100, p, -1, p, None, p, p), "alternatives"),
                       ((p, "f32", 2, 4, p, 5, p, None, p, p), "alternatives"),
                       ((p, "f32", 2, 100, p, 3, p, None, None, p), "null"),
                       ((p, "f32", -1, 100, p, 0, p, None, None, None), "rows"),
                       ((p, "f32", 2, 0, p, 0, p, None, None, None), "vocab"),
                       ((p + 2, "f32", 2, 100, p, 0, p, None, None, None), "unaligned"),
                       ((None, "f32", 2, 100, p, 0, p, None, None, None), "null")):
        with pytest.raises(fmd.FmdError, match=text):
            model.op_logprobs(*args)
    with pytest.raises(fmd.FmdError, match="stride"):
        model.op_logprobs(p, "f32", 2, 100, p, 0, p, None, None, None, ld=99)
    model.op_logprobs(p, "f32", 0, 100, p, 0, p, None, None, None)   # no rows: nothing to do
    with pytest.raises(fmd.FmdError, match="no logits"):
        model.logprobs(3, [1, 2, 3])
