"""The decoder over the paged 4-bit cache: steps, forks, windows, generation and
graphs.

Logits of f32 models are compared with a 64-bit evaluation of the whole decoder
whose K and V are rounded to 4 bits as the cache does (tests/pkv_ref.py).  f32
products of up to 512 terms are off by at most 512 * 2^-24 = 2^-15 relative to
their terms' magnitudes, and a key next to a border may fall on its other side:
one code of one key (a step of at most 2^(e+1), in a head's score of 128) moves
a context by under 2 |q| 2^(e+1) / sqrt(128) max|v| of that key's weight.  The
bar is 2^-9 of the largest logit, which holds a handful of such codes.
"""
import importlib

import numpy as np
import pytest
import torch

from tests import pkv_ref as ref
from tests.gpu_util import tiny_cfg

pytestmark = pytest.mark.gpu
P = "model.language_model."


class Ref64:
    """The decoder in 64 bits over sequences of 4-bit K and V."""

    def __init__(self, cfg, w, window=0, sinks=0, max_len=512):
        self.cfg, self.window, self.sinks = cfg, window, sinks
        self.w = {k.removeprefix(P): np.asarray(v, dtype=np.float64) for k, v in w.items()}
        self.cos, self.sin = ref.rope_tables(max_len, cfg.rope_theta, torch.float32)

    def new(self):
        return [[np.zeros((0, self.cfg.num_key_value_heads, 128))] * 2 for _ in range(self.cfg.num_hidden_layers)]

    @staticmethod
    def fork(cache):
        return [list(c) for c in cache]

    def _rms(self, x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.cfg.rms_norm_eps) * g

    def step(self, cache, ids):
        """Appends the tokens; returns the last one's logits."""
        c, w = self.cfg, self.w
        x = w["embed_tokens.weight"][list(ids)]
        n, at = len(ids), cache[0][0].shape[0]
        pos = np.arange(at, at + n)
        cos, sin = self.cos[pos], self.sin[pos]
        for l in range(c.num_hidden_layers):
            g = lambda t: w[f"layers.{l}.{t}.weight"]  # noqa: E731
            h = self._rms(x, g("input_layernorm"))
            q = (h @ g("self_attn.q_proj").T).reshape(n, -1, 128)
            k = (h @ g("self_attn.k_proj").T).reshape(n, -1, 128)
            v = (h @ g("self_attn.v_proj").T).reshape(n, -1, 128)
            q = ref.norm_rope(q, g("self_attn.q_norm"), cos, sin, c.rms_norm_eps)
            k = ref.norm_rope(k, g("self_attn.k_norm"), cos, sin, c.rms_norm_eps)
            cache[l] = [np.concatenate([cache[l][0], ref.quantize(k, "f32")]),
                        np.concatenate([cache[l][1], ref.quantize(v, "f32")])]
            ctx = ref.attention(q, *cache[l], pos, self.window, self.sinks)
            x = x + ctx.reshape(n, -1) @ g("self_attn.o_proj").T
            h = self._rms(x, g("post_attention_layernorm"))
            a, b = h @ g("mlp.gate_proj").T, h @ g("mlp.up_proj").T
            x = x + (a / (1 + np.exp(-a)) * b) @ g("mlp.down_proj").T
        head = w.get("lm_head.weight", w["embed_tokens.weight"])
        return self._rms(x[-1], w["norm.weight"]) @ head.T


def close(got, want):
    assert np.abs(got - want).max() <= 2.0 ** -9 * np.abs(want).max(), np.abs(got - want).max()


@pytest.fixture(scope="module")
def f32(fmd):
    cfg = tiny_cfg(fmd, layers=2, vocab=512)
    w = fmd.synthetic_weights(cfg, seed=3)
    return fmd.Qwen3(cfg, "f32", max_len=512).load(w), cfg, w


def ids_of(n, seed, vocab=512):
    return np.random.default_rng(seed).integers(0, vocab, n).tolist()


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_steps_forks_and_pieces(fmd, f32, window, sinks):
    """Prompts and single tokens together, a fork that goes its own way, a
    truncation, a compaction in between: each row's logits are those of its own
    tokens."""
    m, cfg, w = f32
    r = Ref64(cfg, w, window, sinks)
    c = fmd.PagedKvCache(m, pages=24, max_seqs=4, max_rows=256, window=window, sinks=sinks)
    a, b = c.open(), c.open()
    ra, rb = r.new(), r.new()
    pa, pb = ids_of(100, 1), ids_of(9, 2)
    got = c.step([a, b], [pa, pb])
    close(got[0], r.step(ra, pa))
    close(got[1], r.step(rb, pb))
    got = c.step([b, a], [[5], [6]])           # two decode rows, in another order
    close(got[0], r.step(rb, [5]))
    close(got[1], r.step(ra, [6]))
    d = c.fork(a)
    rd = r.fork(ra)
    e = c.copy(a)
    re = r.fork(ra)
    got = c.step([a, d, e, b], [[7], [8], [9, 10, 11], ids_of(30, 3)])
    for i, (x, t) in enumerate(((ra, [7]), (rd, [8]), (re, [9, 10, 11]), (rb, ids_of(30, 3)))):
        close(got[i], r.step(x, t))
    c.free(a)
    c.truncate(e, 101)
    re = [[k[:101], v[:101]] for k, v in re]
    c.resize(24)
    got = c.step([e, d], [[1], [2]])
    close(got[0], r.step(re, [1]))
    close(got[1], r.step(rd, [2]))
    c.resize(12)                                # a smaller pool, then a larger one
    got = c.step([d, b], [[3], [4]])
    close(got[0], r.step(rd, [3]))
    close(got[1], r.step(rb, [4]))
    c.resize(40)
    got = c.step([d], [[3, 4, 5]])
    close(got[0], r.step(rd, [3, 4, 5]))


def test_step_scores_and_greedy(fmd, f32):
    m, cfg, w = f32
    c = fmd.PagedKvCache(m, pages=8, max_seqs=3, max_rows=64)
    s = [c.open() for _ in range(3)]
    lg = c.step(s, [ids_of(5, 1), ids_of(1, 2), ids_of(9, 3)])
    t = m.logprobs(3, [1, 2, 3], top=4)
    x = lg.astype(np.float64)
    lp = x - x.max(-1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(-1, keepdims=True))
    assert np.allclose(t.logp, lp[[0, 1, 2], [1, 2, 3]], atol=1e-5)
    assert np.allclose(t.entropy, -(np.exp(lp) * lp).sum(-1), atol=1e-4)
    order = np.argsort(-x, -1, kind="stable")[:, :4]
    assert np.array_equal(t.top_ids, order)
    assert np.allclose(t.top_logp, np.take_along_axis(lp, order, -1), atol=1e-5)
    nxt, emitted = m.greedy(3, 0, np.zeros(3, np.int32), eos=511)
    want = x.argmax(-1)
    assert [n for n, e in zip(nxt, emitted) if e >= 0] == [int(v) for v in want if v != 511]
    # the 16-bit cache's calls leave their logits too, and the loops none
    kv = m.new_caches(2, 64)
    lg = m.prefill(np.stack([m.embed(ids_of(6, 4)), m.embed(ids_of(6, 5))]), kv, [0, 0])
    assert np.array_equal(m.logprobs(2, top=1).top_ids[:, 0], lg.argmax(-1))
    lg = m.decode_step([1, 2], kv, [0, 0])
    assert np.array_equal(m.logprobs(2, top=1).top_ids[:, 0], lg.argmax(-1))
    m.decode_loop(kv, [1, 2], [0, 0], 3, eos=511)
    with pytest.raises(fmd.FmdError, match="no logits"):
        m.logprobs(2)


@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 5)])
def test_generation(fmd, f32, window, sinks):
    """Tokens of the 64-bit loop wherever its two best logits are apart, their
    log probabilities, rows that end early, prompts longer than a step."""
    m, cfg, w = f32
    r = Ref64(cfg, w, window, sinks)
    prompts = [ids_of(n, 20 + n) for n in (90, 3, 33)]
    want, scores, margins = [], [], []
    for p in prompts:
        cache, feed, toks, lps, mar = r.new(), p, [], [], []
        for _ in range(12):
            lg = r.step(cache, feed)
            top = np.sort(lg)[-2:]
            mar.append(top[1] - top[0])
            t = int(lg.argmax())
            toks.append(t)
            lps.append(float(lg[t] - lg.max() - np.log(np.exp(lg - lg.max()).sum())))
            feed = [t]
        want.append(toks)
        scores.append(lps)
        margins.append(mar)
    eos = want[1][4]                     # the second row ends here, others where they reach it
    c = fmd.PagedKvCache(m, pages=16, max_seqs=3, max_rows=50, window=window, sinks=sinks)
    out = fmd.generate_paged(c, prompts, 12, eos=eos, top=3)
    assert c.free_pages() == 16
    for o, toks, lps, mar in zip(out, want, scores, margins):
        stop = toks.index(eos) if eos in toks else 12
        assert o.finish_reason == (fmd.FinishReason.STOP if stop < 12 else fmd.FinishReason.LENGTH)
        sure = next((i for i, d in enumerate(mar) if d < 0.02), 12)   # near ties end the comparison
        n = min(stop, sure)
        assert o.tokens[:n] == toks[:n] and (sure < stop or len(o.tokens) == stop)
        assert np.allclose(o.logp[:n], lps[:n], atol=0.02)
        assert all(a[0] == (t, lp) for a, t, lp in zip(o.alternatives, o.tokens, o.logp))


@pytest.mark.parametrize("prec", ["bf16", "f16", "int8"])
def test_16_bit_models_follow_the_16_bit_cache(fmd, prec):
    """The logits stay near those of the 16-bit cache (what 4 bits cost is seen,
    nothing else is wrong): relative distance under 0.3 -- rounding K and V to 4
    bits alone is 0.11 rms of them -- and single tokens continue prompts."""
    cfg = tiny_cfg(fmd, layers=2, vocab=1024)
    m = fmd.Qwen3(cfg, prec, max_len=512).load(fmd.synthetic_weights(cfg, seed=5))
    prompts = [ids_of(n, n, 1024) for n in (40, 40)]
    kv = m.new_caches(2, 64)
    a = m.prefill(np.stack([m.embed(p) for p in prompts]), kv, [0, 0])
    c = fmd.PagedKvCache(m, pages=4, max_seqs=2, max_rows=128)
    s = [c.open(), c.open()]
    b = c.step(s, prompts)
    a2, b2 = m.decode_step([3, 4], kv, [0, 0]), c.step(s, [[3], [4]])
    for x, y in ((a, b), (a2, b2)):
        assert np.linalg.norm(x - y) < 0.3 * np.linalg.norm(x)
    e = c.open
    with pytest.raises(fmd.KvCacheOverflow):
        e()


def test_scores_end_with_their_logits(fmd):
    """A call that gives the logits' buffer up for a larger one leaves no logits
    to score; one that has room for them does."""
    cfg = tiny_cfg(fmd, layers=1, vocab=64)
    m = fmd.Qwen3(cfg, "f32", max_len=64).load(fmd.synthetic_weights(cfg, seed=1))
    c = fmd.PagedKvCache(m, pages=4, max_seqs=2, max_rows=8)
    s = c.open()
    want = c.step([s], [[1, 2]]).argmax(-1)
    x = torch.zeros((4, 256)).cuda()
    torch.cuda.synchronize()
    m.op_layer_decode(m.new_caches(1, 8), 0, x.data_ptr(), [0], 1)
    assert np.array_equal(m.logprobs(1, top=1).top_ids[:, 0], want)
    m.op_layer_decode(m.new_caches(4, 8), 0, x.data_ptr(), [0] * 4, 4)
    with pytest.raises(fmd.FmdError, match="no logits"):
        m.logprobs(1, top=1)
    want = c.step([s], [[3]]).argmax(-1)
    m.op_layer_decode(m.new_caches(4, 8), 0, x.data_ptr(), [0] * 4, 4)
    assert np.array_equal(m.logprobs(1, top=1).top_ids[:, 0], want)


def test_failed_steps_leave_the_sequences(fmd, f32):
    m, cfg, w = f32
    c = fmd.PagedKvCache(m, pages=2, max_seqs=2, max_rows=64)
    s, t = c.open(), c.open()
    c.step([s], [ids_of(10, 1)])
    with pytest.raises(fmd.FmdError, match="token id"):
        c.step([s], [[512]])
    with pytest.raises(fmd.KvCacheOverflow, match="pages needed"):
        c.step([s, t], [ids_of(55, 1), ids_of(9, 1)])
    with pytest.raises(fmd.FmdError, match="at a time"):
        c.step([s], [ids_of(65, 1)])
    with pytest.raises(fmd.FmdError, match="named twice"):
        c.step([s, s], [[1], [2]])
    with pytest.raises(fmd.FmdError, match="a token of every"):
        c.step([s], [[]])
    with pytest.raises(fmd.FmdError):
        c.step([], [])
    assert c.len(s) == 10 and c.len(t) == 0 and c.free_pages() == 1
    r = Ref64(cfg, w)
    cache = r.new()
    r.step(cache, ids_of(10, 1))
    close(c.step([s], [[7]])[0], r.step(cache, [7]))


def test_embeddings_and_many_sequences(fmd, f32):
    """More rows than the GEMVs take, more sequences than one launch of the head."""
    m, cfg, w = f32
    r = Ref64(cfg, w)
    n = 19
    c = fmd.PagedKvCache(m, pages=n, max_seqs=n, max_rows=200)
    s = [c.open() for _ in range(n)]
    prompts = [ids_of(1 + i % 5, i) for i in range(n)]
    counts = [len(p) for p in prompts]
    emb = m.embed(sum(prompts, []))
    got = c.step(s, embeds=emb, counts=counts)
    refs = [r.new() for _ in range(n)]
    for i in range(n):
        close(got[i], r.step(refs[i], prompts[i]))
    got = c.step(s, embeds=torch.from_numpy(m.embed(list(range(n)))).cuda(), counts=[1] * n)
    for i in range(n):
        close(got[i], r.step(refs[i], [i]))
    assert m.logprobs(n, top=1).top_ids[:, 0].tolist() == got.argmax(-1).tolist()
    with pytest.raises(fmd.FmdError, match="embeds must be"):
        c.step(s, embeds=emb[:5], counts=[1] * n)


# --- pages on the device -------------------------------------------------------


def test_copy_pages_every_layer(fmd):
    cfg = tiny_cfg(fmd, layers=3, vocab=64)
    m = fmd.Qwen3(cfg, "bf16", max_len=64)
    c = fmd.PagedKvCache(m, pages=700, max_seqs=1, max_rows=8)
    pool = c.pool()
    assert tuple(pool.shape) == (3, 700, 2 * 8704)
    pool.copy_(torch.randint(0, 256, pool.shape, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    want = pool.clone()
    perm = np.random.default_rng(1).permutation(700)
    for n in (1, 7, 320):       # one launch and several
        src, dst = perm[:n], perm[n:2 * n]
        c.copy_pages(src, dst)
        want[:, torch.from_numpy(dst).cuda()] = want[:, torch.from_numpy(src).cuda()]
        assert torch.equal(c.pool(), want)
    c.copy_pages([5, 5], [6, 7])        # one source twice
    want[:, 6], want[:, 7] = want[:, 5], want[:, 5]
    assert torch.equal(c.pool(), want)
    c.copy_pages([], [])
    for src, dst, text in (([0], [700], "outside"), ([-1], [0], "outside"), ([0, 1], [2, 2], "twice"),
                           ([0, 1], [1, 2], "source"), ([3], [3], "source")):
        with pytest.raises(fmd.FmdError, match=text):
            c.copy_pages(src, dst)
    with pytest.raises(fmd.FmdError, match="one destination"):
        c.copy_pages([1], [])
    assert torch.equal(c.pool(), want)


# --- streams and graphs --------------------------------------------------------


def test_callers_stream_and_graph_replays_follow_the_plan(fmd):
    """A captured append + attention of one token for each sequence, replayed
    over later plans whose rows need more items than the captured one, with
    eager work in between; after a fork (no plan) it leaves the buffers alone."""
    cfg = tiny_cfg(fmd, layers=1, vocab=64)
    m = fmd.Qwen3(cfg, "bf16", max_len=4096).load(fmd.synthetic_weights(cfg, seed=1))
    dt = torch.bfloat16
    st = torch.cuda.Stream()
    m.set_stream(st.cuda_stream)
    g = torch.Generator().manual_seed(2)
    qkv = torch.empty((2, (4 + 4) * 128), dtype=dt).cuda()
    q, ctx = (torch.zeros((2, 4, 128), dtype=dt).cuda() for _ in range(2))
    torch.cuda.synchronize()

    def call(c):
        c.append(0, qkv.data_ptr(), q.data_ptr())
        c.attention(0, q.data_ptr(), ctx.data_ptr())

    def fresh():
        c = fmd.PagedKvCache(m, pages=120, max_seqs=3, max_rows=3000)
        return c, [c.open(), c.open()]

    def grow(c, seqs, n, seed):
        x = (torch.randn((2 * n, 8 * 128), generator=torch.Generator().manual_seed(seed)) * 0.7).to(dt).cuda()
        big = torch.empty((2 * n, 4, 128), dtype=dt).cuda()
        torch.cuda.synchronize()
        c.plan(seqs, [n, n])
        c.append(0, x.data_ptr(), big.data_ptr())
        torch.cuda.synchronize()

    try:
        c, seqs = fresh()       # replayed
        e, eseqs = fresh()      # eager
        grow(c, seqs, 30, 5)
        grow(e, eseqs, 30, 5)
        c.plan(seqs, [1, 1])
        with pytest.raises(fmd.FmdError, match="capture"):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                c.plan(seqs, [1, 1])
        c.truncate(seqs[0], 30)
        c.truncate(seqs[1], 30)
        c.plan(seqs, [1, 1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call(c)
        for i, n in enumerate((0, 40, 0, 1300, 700)):
            if n:
                grow(c, seqs, n, 10 + i)
                grow(e, eseqs, n, 10 + i)
            if i:
                c.plan(seqs, [1, 1])
            e.plan(eseqs, [1, 1])
            qkv.copy_((torch.randn(qkv.shape, generator=g) * 0.7).to(dt))
            torch.cuda.synchronize()
            call(e)
            torch.cuda.synchronize()
            want = ctx.clone()
            ctx.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(ctx, want) and ctx.abs().sum() > 0, i
        c.fork(seqs[0])
        ctx.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (ctx == 3.0).all()
        with pytest.raises(fmd.FmdError, match="no plan"):
            call(c)
    finally:
        m.set_stream(None)


def test_refusals(fmd, f32):
    m, cfg, w = f32
    P_ = fmd.PagedKvCache
    for args, text in (((0, 1, 1), "must be > 0"), ((1, 0, 1), "must be > 0"), ((1, 1, 0), "must be > 0"),
                       ((1, 1, 1, -1), "negative"), ((1, 1, 1, 0, 4), "sinks need"), ((1, 70000, 1), "above")):
        with pytest.raises(fmd.FmdError, match=text):
            P_(m, *args)
    with pytest.raises(fmd.FmdError) as e:
        P_(m, 2_000_000_000, 1, 1)
    assert e.value.code == -4
    c = P_(m, 2, 1, 8)
    buf = torch.zeros(8 * 8 * 128).cuda()
    p = buf.data_ptr()
    with pytest.raises(fmd.FmdError, match="no plan"):
        c.attention(0, p, p)
    s = c.open()
    c.plan([s], [2])
    for fn in (c.append, c.write, c.read, c.attention):
        with pytest.raises(fmd.FmdError, match="16-byte"):
            fn(0, p + 4, p)
        with pytest.raises(fmd.FmdError, match="bad layer"):
            fn(2, p, p)
        with pytest.raises(fmd.FmdError, match="null"):
            fn(0, None, None)
    other = fmd.Qwen3(cfg, "f32", max_len=512)
    with pytest.raises(fmd.FmdError, match="another decoder"):
        importlib.import_module("fast-moss-diarization_amd.decoder")._check(fmd.lib().fmd_op_pkv_attention(other.handle, c.handle, 0, p, p))
    d = P_(other, 1, 1, 8)
    d.plan([d.open()], [1])
    with pytest.raises(fmd.FmdError, match="q_norm"):
        d.append(0, p, p)
    with pytest.raises(fmd.FmdError, match="incomplete"):
        d.step([0], [[1]])
    c.plan([s], [0])            # no rows: calls do nothing
    c.attention(0, p, p)
    c.plan([], [])
    c.append(0, p, p)
    with pytest.raises(fmd.FmdError, match="no such"):
        c.free(5)
    with pytest.raises(fmd.FmdError, match="no such"):
        c.len(5)
    assert c.pages(s) == [0]
