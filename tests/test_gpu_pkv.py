"""The paged 4-bit KV cache on the device against tests/pkv_ref.py.

Tolerances.  u is half a unit in the last place of the output's type relative to
the value: f32 2^-24, f16 2^-11, bf16 2^-8.  K and V come back exactly.  q: one rounding, after f32
arithmetic whose relative error (a sum of 128 squares, a root, a division, three
products and a sum) stays under 32 * 2^-24 of the rotated pair's length.
Context: p and the sums are f32; p meets V as a sum of two bf16 terms in decode
rows of 16-bit caches, as one bf16 or f16 value in many-token rows, as three bf16
terms in f32 caches.  With every p off by at most the factor r = 2^-16 (2^-8 of
what the first term left), 2^-8, 2^-11 or 2^-24, and l with it, a
context element moves by at most 2 r max|v|.  A score is a sum of 128 products
in four MFMAs (f32 caches: twelve) of 32: at most 9 (17) roundings on a path,
each 2^-24 of at most sum|q k| / sqrt(128) < 30 here, then the exponent's own
roundings, 3 * 2^-24 of at most 64: x < 2^-15, and p off by the factor x moves
the context by 2 x max|v|.  So
|got - want| <= (2 r + 2^-14) max|v| + u |want|.
"""
import numpy as np
import pytest
import torch

from tests import pkv_ref as ref

pytestmark = pytest.mark.gpu

TDT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.float16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "int8": 2.0 ** -11}
PRECS = ["bf16", "f16", "f32"]


def make(fmd, prec, rep=2, nkv=2, layers=1, max_len=4096, seed=0):
    cfg = fmd.TextConfig(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=layers,
                         num_attention_heads=nkv * rep, num_key_value_heads=nkv, head_dim=128, rope_theta=1e6)
    m = fmd.Qwen3(cfg, prec, max_len=max_len)
    g = torch.Generator().manual_seed(seed)
    gains = []
    for i in range(layers):
        for t in ("q_norm", "k_norm"):
            w = (1 + 0.1 * torch.randn(128, generator=g)).to(TDT[prec])
            m.set_weight(f"layers.{i}.self_attn.{t}.weight", w.cuda())
            gains.append(w.double().numpy())
    return m, cfg, gains


def randn(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def up(t):
    """On the device, and there before work on another stream starts."""
    d = t.cuda()
    torch.cuda.synchronize()
    return d


def fill(cache, layer, seqs, kv):
    """Append kv[i] = (K, V) to seqs[i] by write(), sequence by sequence."""
    for s, (k, v) in zip(seqs, kv):
        for at in range(0, k.shape[0], cache.max_rows):
            a, b = up(k[at:at + cache.max_rows].contiguous()), up(v[at:at + cache.max_rows].contiguous())
            cache.plan([s], [a.shape[0]])
            cache.write(layer, a.data_ptr(), b.data_ptr())


def ctx_bound(prec, want, vmax, decode):
    r = {"bf16": 2.0 ** -16 if decode else 2.0 ** -8, "f16": 2.0 ** -16 if decode else 2.0 ** -11,
         "f32": 2.0 ** -24}[prec]
    return (2 * r + 2.0 ** -14) * vmax + U[prec] * np.abs(want) + 1e-30


def run_attention(fmd, prec, rep, lens, counts, window=0, sinks=0, nkv=2, seed=1, kv=None, check=True):
    m, cfg, _ = make(fmd, prec, rep, nkv)
    dt = TDT[prec]
    kv = kv or [(randn((n, nkv, 128), dt, seed + 2 * i, 1.5), randn((n, nkv, 128), dt, seed + 2 * i + 1))
                for i, n in enumerate(lens)]
    pages = sum((n + 63) // 64 for n in lens) + 1
    c = fmd.PagedKvCache(m, pages=pages, max_seqs=len(lens), max_rows=max(sum(counts), 512), window=window,
                         sinks=sinks)
    seqs = [c.open() for _ in lens]
    fill(c, 0, seqs, [(k[: k.shape[0] - n], v[: v.shape[0] - n]) for (k, v), n in zip(kv, counts)])
    c.plan(seqs, counts)
    if sum(counts):
        a, b = (up(torch.cat([x[j][x[j].shape[0] - n:] for x, n in zip(kv, counts)])) for j in (0, 1))
        c.write(0, a.data_ptr(), b.data_ptr())
    rows = sum(counts)
    q = randn((rows, nkv * rep, 128), dt, seed + 99, 1.0)
    qd = up(q)
    out = up(torch.full((rows + 2, nkv * rep, 128), 7.0, dtype=dt))
    c.attention(0, qd.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    got = out.cpu()
    assert (got[rows:] == 7.0).all(), "rows behind the plan's were written"
    got = got[:rows].double().numpy()
    if not check:
        return got, q, kv
    r0 = 0
    for (k, v), n, cnt in zip(kv, lens, counts):
        if not cnt:
            continue
        kq, vq = ref.quantize(k.double().numpy(), prec), ref.quantize(v.double().numpy(), prec)
        want = ref.attention(q[r0:r0 + cnt].double().numpy(), kq, vq, np.arange(n - cnt, n), window, sinks)
        vmax = np.repeat(np.abs(vq).max((0, 2)), rep)[None, :, None]
        err = np.abs(got[r0:r0 + cnt] - want)
        bound = ctx_bound(prec, want, vmax, cnt == 1)
        assert (err <= bound).all(), (n, cnt, float((err / bound).max()))
        r0 += cnt
    return got, q, kv


# --- rows in and out ---------------------------------------------------------


@pytest.mark.parametrize("prec", PRECS)
def test_write_read_is_the_4_bit_value(fmd, prec):
    """Every code border, signs, zeros, tiny and huge blocks, ragged pages."""
    m, cfg, _ = make(fmd, prec)
    dt = TDT[prec]
    rows = 150
    k, v = randn((rows, 2, 128), torch.float32, 3), randn((rows, 2, 128), torch.float32, 4)
    k *= torch.exp2(torch.randint(-20, 12, (rows, 2, 1), generator=torch.Generator().manual_seed(5)).float())
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    k[0, 0, :32] = torch.cat([border, -border, border * 1.01, border * 0.99])
    k[1] = 0.0
    k[2, 0, :32] = 7.0
    k[2, 0, 32:64] = 7.02
    k[3] = 2.0 ** -24
    k[4] = 60000.0
    v[0, 1] = -0.0
    k, v = k.to(dt), v.to(dt)
    c = fmd.PagedKvCache(m, pages=4, max_seqs=2, max_rows=256)
    s, t = c.open(), c.open()
    c.plan([s], [37])      # content of no matter: the rows start inside a page
    c.plan([s, t], [rows - 20, 20])
    kd, vd = up(k), up(v)
    c.write(0, kd.data_ptr(), vd.data_ptr())
    ko, vo = (up(torch.full((rows + 1, 2, 128), 5.0, dtype=dt)) for _ in range(2))
    c.read(0, ko.data_ptr(), vo.data_ptr())
    torch.cuda.synchronize()
    for got, x in ((ko, k), (vo, v)):
        got = got.cpu().double().numpy()
        assert (got[rows:] == 5.0).all()
        assert np.array_equal(got[:rows], ref.quantize(x.double().numpy(), prec))


@pytest.mark.parametrize("prec", PRECS)
def test_saturation_at_the_exponent_range(fmd, prec):
    m, cfg, _ = make(fmd, prec)
    dt = TDT[prec]
    big = 65504.0 if prec == "f16" else 3e38
    small = 2.0 ** -24 if prec == "f16" else 1e-30
    k = torch.zeros((2, 2, 128))
    k[0, :, ::3], k[1, :, ::5] = big, small
    k = k.to(dt)
    c = fmd.PagedKvCache(m, pages=1, max_seqs=1, max_rows=4)
    c.plan([c.open()], [2])
    kd = up(k)
    c.write(0, kd.data_ptr(), kd.data_ptr())
    out = up(torch.empty((2, 2, 128), dtype=dt))
    c.read(0, out.data_ptr(), None)
    torch.cuda.synchronize()
    got = out.cpu().double().numpy()
    assert np.isfinite(got).all()
    assert np.array_equal(got, ref.quantize(k.double().numpy(), prec))


@pytest.mark.parametrize("prec,rep,nkv", [("bf16", 2, 8), ("f16", 1, 3), ("f32", 4, 2), ("int8", 2, 2)])
def test_append_norms_rotates_and_stores(fmd, prec, rep, nkv):
    if (rep * nkv * 128) % 256:
        nkv += 1
    m, cfg, gains = make(fmd, prec, rep, nkv, max_len=700)
    dt = TDT[prec]
    starts, counts = [0, 130, 600, 63], [65, 1, 100, 2]
    c = fmd.PagedKvCache(m, pages=40, max_seqs=4, max_rows=800)
    seqs = [c.open() for _ in starts]
    c.plan(seqs, starts)
    c.plan(seqs, counts)
    rows, nh = sum(counts), rep * nkv
    qkv = randn((rows, (nh + 2 * nkv) * 128), dt, 8, 0.7)
    qkv[3] = 0.0
    x = up(qkv)
    q, k, v = (up(torch.full((rows + 1, h, 128), 5.0, dtype=dt)) for h in (nh, nkv, nkv))
    c.append(0, x.data_ptr(), q.data_ptr())
    c.read(0, k.data_ptr(), v.data_ptr())
    torch.cuda.synchronize()
    q, k, v = (t.cpu().double().numpy() for t in (q, k, v))
    assert (q[rows:] == 5.0).all() and (k[rows:] == 5.0).all()
    pos = np.concatenate([np.arange(s, s + n) for s, n in zip(starts, counts)])
    cos, sin = (t[pos] for t in ref.rope_tables(700, 1e6, dt))
    h = qkv.double().numpy().reshape(rows, nh + 2 * nkv, 128)
    wq = ref.norm_rope(h[:, :nh], gains[0], cos, sin, 1e-6)
    pair = np.sqrt(wq[..., :64] ** 2 + wq[..., 64:] ** 2)
    bound = U[prec] * np.abs(wq) + 32 * 2.0 ** -24 * np.concatenate([pair, pair], -1) + (
        2.0 ** -25 if prec in ("f16", "int8") else 0)
    assert (np.abs(q[:rows] - wq) <= bound).all()
    wk = ref.quantize(ref.norm_rope(h[:, nh:nh + nkv], gains[1], cos, sin, 1e-6), prec)
    assert np.array_equal(k[:rows], wk)
    assert np.array_equal(v[:rows], ref.quantize(h[:, nh + nkv:], prec))


# --- attention -----------------------------------------------------------------


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rep", [1, 2, 4])
def test_decode_rows(fmd, prec, rep):
    """One new token: a first token, page borders, several items a row."""
    run_attention(fmd, prec, rep, [1, 2, 63, 64, 65, 129, 1000, 700], [1] * 8)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rep", [1, 2, 4])
def test_many_token_rows(fmd, prec, rep):
    """Prompts from their first token, pieces in a context, odd tiles."""
    run_attention(fmd, prec, rep, [2, 64, 131, 300, 1000], [2, 64, 131, 77, 140])


@pytest.mark.parametrize("prec", PRECS)
def test_mixed_rows_and_a_sequence_without_new_tokens(fmd, prec):
    run_attention(fmd, prec, 2, [500, 90, 64, 1, 200], [1, 90, 0, 1, 3])


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 0), (64, 3), (100, 70), (130, 64), (1000, 500), (64, 0),
                                          (300, 1000)])
@pytest.mark.parametrize("prec", PRECS)
def test_window_and_sinks(fmd, prec, window, sinks):
    run_attention(fmd, prec, 2, [1, 64, 333, 700, 640], [1, 1, 1, 1, 1], window, sinks)
    run_attention(fmd, prec, 2, [64, 333, 700], [64, 40, 650], window, sinks)


def test_long_row_in_many_items(fmd):
    run_attention(fmd, "bf16", 2, [4096, 3999], [1, 1], nkv=1)
    run_attention(fmd, "bf16", 2, [4096], [90], nkv=1)


def test_pages_beyond_4_gib(fmd):
    """The last pages of a pool whose byte offsets pass 32 bits: the same bits as
    from a small pool, in decode and many-token rows, and the neighbours' bytes
    stay as they are."""
    m, cfg, _ = make(fmd, "bf16", 2, 8, max_len=65536)
    dt = torch.bfloat16
    small = fmd.PagedKvCache(m, pages=16, max_seqs=2, max_rows=512)
    big = fmd.PagedKvCache(m, pages=62 * 1024 + 16, max_seqs=64, max_rows=65536)
    assert fmd.PagedKvCache.bytes(m, 62 * 1024) > 1 << 32
    for _ in range(62):
        big.plan([big.open()], [65536])      # pages taken, nothing written
    outs = []
    mark = big.pool()[0, 62 * 1024 - 1]
    mark.fill_(7)
    for c in (small, big):
        s = [c.open(), c.open()]
        kv = [(randn((n, 8, 128), dt, n), randn((n, 8, 128), dt, n + 1)) for n in (300, 90)]
        fill(c, 0, s, [(k[:-n], v[:-n]) for (k, v), n in zip(kv, (1, 70))])
        c.plan(s, [1, 70])
        a, b = (up(torch.cat([kv[0][j][-1:], kv[1][j][-70:]])) for j in (0, 1))
        c.write(0, a.data_ptr(), b.data_ptr())
        q = up(randn((71, 16, 128), dt, 5))
        out = up(torch.zeros((71, 16, 128), dtype=dt))
        c.attention(0, q.data_ptr(), out.data_ptr())
        torch.cuda.synchronize()
        outs.append(out.cpu())
    assert min(big.pages(s[0]) + big.pages(s[1])) >= 62 * 1024
    assert torch.equal(*outs) and outs[0].float().abs().sum() > 0
    assert (big.pool()[0, 62 * 1024 - 1] == 7).all()


@pytest.mark.parametrize("prec", ["bf16", "f16", "f32"])
def test_large_scores(fmd, prec):
    """One key's score far above the others', up to 2^27 in size: its V alone.
    The exponent of the largest is then off by half an ulp of 2^28, 8 at most
    (p and its sum alike)."""
    dt = TDT[prec]
    m, cfg, _ = make(fmd, prec, 2, 2)
    c = fmd.PagedKvCache(m, pages=32, max_seqs=2, max_rows=1024)
    s = [c.open(), c.open()]
    big_q, big_k = (1.25 * 2.0 ** 15, 2.0 ** 13) if prec == "f16" else (1.25 * 2.0 ** 20, 2.0 ** 10)
    lens, counts, top = (900, 700), (1, 130), 5
    k = [torch.zeros((n, 2, 128), dtype=dt) for n in lens]
    v = [randn((n, 2, 128), dt, n) for n in lens]
    for x in k:
        x[:, :, 0] = big_k / 4
        x[top, :, 0] = big_k
    fill(c, 0, s, [(a[:-n], b[:-n]) for a, b, n in zip(k, v, counts)])
    c.plan(s, counts)
    a, b = (up(torch.cat([x[i][-n:] for i, n in enumerate(counts)])) for x in (k, v))
    c.write(0, a.data_ptr(), b.data_ptr())
    q = torch.zeros((sum(counts), 4, 128), dtype=dt)
    q[:, :, 0] = big_q
    q, out = up(q), up(torch.zeros((sum(counts), 4, 128), dtype=dt))
    c.attention(0, q.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    # V of that key as it is held: written to a sequence of its own and read back
    c.free(s[0])
    t = c.open()
    for i in range(2):
        one = [up(x[i][top:top + 1].contiguous()) for x in (k, v)]
        c.plan([t], [1])
        c.write(0, *(x.data_ptr() for x in one))
        held = up(torch.zeros((1, 2, 128), dtype=dt))
        c.read(0, None, held.data_ptr())
        torch.cuda.synchronize()
        want = held.double().cpu().numpy()[0].repeat(2, axis=0)
        rows = got[:1] if i == 0 else got[1:]
        assert (np.abs(rows - want) <= ctx_bound(prec, want, np.abs(want).max(), i == 0)).all()


def test_more_rows_than_work_group_slots(fmd):
    """300 sequences: each row is an item of its own, in several rounds."""
    run_attention(fmd, "bf16", 1, [1 + (7 * i) % 200 for i in range(300)], [1] * 300)


def test_large_plans(fmd):
    """More new tokens than the plan's first upload holds, mixed with decode rows."""
    run_attention(fmd, "f16", 2, [700, 300, 1, 513], [600, 1, 1, 513])


def test_queries_with_nan_stay_in_their_rows(fmd):
    m, cfg, _ = make(fmd, "bf16")
    c = fmd.PagedKvCache(m, pages=8, max_seqs=2, max_rows=128)
    s = [c.open(), c.open()]
    kv = [(randn((n, 2, 128), torch.bfloat16, n), randn((n, 2, 128), torch.bfloat16, n + 1)) for n in (100, 60)]
    fill(c, 0, s, [(k[:-n], v[:-n]) for (k, v), n in zip(kv, (1, 33))])
    c.plan(s, [1, 33])
    a, b = (up(torch.cat([kv[0][j][-1:], kv[1][j][-33:]])) for j in (0, 1))
    c.write(0, a.data_ptr(), b.data_ptr())
    q = randn((34, 4, 128), torch.bfloat16, 5)
    out = up(torch.zeros((34, 4, 128), dtype=torch.bfloat16))
    ref_out = up(torch.zeros((34, 4, 128), dtype=torch.bfloat16))
    qd = up(q)
    c.attention(0, qd.data_ptr(), ref_out.data_ptr())
    q[0, 1, 7], q[9, 2, 0] = float("nan"), float("inf")
    qd = up(q)
    c.attention(0, qd.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    got, want = out.cpu(), ref_out.cpu()
    bad = torch.zeros((34, 4), dtype=torch.bool)
    bad[0, 1] = bad[9, 2] = True
    assert got[bad].isnan().any(-1).all()
    assert torch.equal(got[~bad], want[~bad])


def test_nan_and_infinity_stay_where_they_are_seen(fmd):
    """A token with a NaN or an infinity in K or V poisons its head's contexts
    that see it, and no other, in decode and many-token rows."""
    for counts in ([1, 1, 1], [40, 40, 40]):
        lens = [200, 200, 200]
        kv = [(randn((200, 2, 128), torch.bfloat16, 40 + i), randn((200, 2, 128), torch.bfloat16, 50 + i))
              for i in range(3)]
        kv[0][1][20, 0, 5] = float("nan")      # outside the window below
        kv[1][0][185, 1, 77] = float("inf")    # seen by the positions from 185 on
        clean = [(k.clone(), v.clone()) for k, v in kv]
        clean[0][1][20, 0], clean[1][0][185, 1], clean[1][1][185, 1] = 0.0, 0.0, 0.0
        got, q, _ = run_attention(fmd, "bf16", 2, lens, counts, window=60, kv=kv, check=False)
        n = counts[0]
        pos = np.arange(200 - n, 200)
        for i in range(3):
            k, v = (ref.quantize(t.double().numpy(), "bf16") for t in clean[i])
            want = ref.attention(q[i * n:(i + 1) * n].double().numpy(), k, v, pos, 60)
            bad = np.zeros(want.shape, bool)
            if i == 1:
                bad[pos >= 185, 2:] = True
            g = got[i * n:(i + 1) * n]
            assert np.isnan(g[bad]).all()
            bound = ctx_bound("bf16", want, np.abs(v).max(), n == 1)
            assert (np.abs(g - want)[~bad] <= bound[~bad]).all()


def test_poisoned_tokens_read_back_as_nan(fmd):
    m, cfg, _ = make(fmd, "bf16")
    k = randn((3, 2, 128), torch.bfloat16, 1)
    v = randn((3, 2, 128), torch.bfloat16, 2)
    v[1, 0, 127] = float("-inf")
    c = fmd.PagedKvCache(m, pages=1, max_seqs=1, max_rows=4)
    c.plan([c.open()], [3])
    kd, vd = up(k), up(v)
    c.write(0, kd.data_ptr(), vd.data_ptr())
    ko, vo = up(torch.zeros_like(k)), up(torch.zeros_like(k))
    c.read(0, ko.data_ptr(), vo.data_ptr())
    torch.cuda.synchronize()
    for got, x in ((ko, k), (vo, v)):
        got = got.cpu().double().numpy()
        assert np.isnan(got[1, 0]).all()
        x = x.double().numpy()
        x[1, 0] = 0.0
        want = ref.quantize(x, "bf16")
        keep = np.ones((3, 2), bool)
        keep[1, 0] = False
        assert np.array_equal(got[keep], want[keep])
