"""What the paged 4-bit cache and the token scores are measured on.

A transcription service that keeps many long recordings at once holds their
keys and values in pages of 64 tokens and 4 bits a value, and has four things
done to them:

* ``append``: a projection's q | k | v rows get the q/k norms and the rotation;
  q comes back, K and V go into the sequences' pages in 4 bits (and are read
  back here as the values they stand for).
* ``attention``: the newest tokens' queries over everything that a sequence's
  window and its first tokens (the sinks) let them see.
* ``pages``: pages are copied inside the pool, every layer at once, when a
  sequence is copied, a shared page is written to or the pool is compacted.
* ``logprobs``: the log probability of given tokens, the entropy of the
  distribution and the best alternatives, from a step's logits.

Shapes are those of the library's decoder (fmd.QWEN3_0_6B: 16 query heads, 8
KV heads of 128, 28 layers, 151,936 tokens), contexts those of its benchmark
and of recordings up to some forty minutes.

The 4 bits: blocks of 32 consecutive dims of one token and head share a power
of two 2^e, the smallest with max|x| <= 7 * 2^e (e kept in [-23, 13] for f16
activations and in [-64, 64] for the others); x / 2^e, as a 32-bit number, is
rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its sign, ties to the
value whose last bit is even, at most 6.
"""
from __future__ import annotations

import importlib
import math
import zlib

import numpy as np
import torch

own = False

DEV = "cuda"
ACT = {"bf16": torch.bfloat16, "int8": torch.float16, "f32": torch.float32}
NH, NKV, HD, REP = 16, 8, 128, 2
PAGE = 64
PAGE_BYTES = NKV * PAGE * (HD + HD // 16)  # of one layer: K and V at 4 bits, a scale byte per 32
VOCAB = 151_936
EPS = 1e-6
MAX_ROWS = 16384


# --- the cases -----------------------------------------------------------------


def listed():
    return [
        # one decode step's new tokens of a micro-batch: latency
        dict(name="append_8x1_at_4096_bf16", kind="append", prec="bf16", batch=8, lo=4096, hi=4096,
             count_lo=1, count_hi=1, lens_seed=1),
        # a micro-batch of short and medium prompts, f32 activations
        dict(name="append_4x310_1890_f32", kind="append", prec="f32", batch=4, lo=0, hi=0, count_lo=310,
             count_hi=1890, lens_seed=2),
        # a full prefill chunk of long recordings
        dict(name="append_8x1536_at_3000_bf16", kind="append", prec="bf16", batch=8, lo=1000, hi=5000,
             count_lo=1536, count_hi=1536, lens_seed=3),
        # a decode step of one 30 s request: latency
        dict(name="attention_1x450_int8", kind="attention", prec="int8", batch=1, lo=450, hi=450, count=1,
             window=0, sinks=0, lens_seed=4),
        # a decode step of the benchmark's micro-batch
        dict(name="attention_8x4096_bf16", kind="attention", prec="bf16", batch=8, lo=4096, hi=4096, count=1,
             window=0, sinks=0, lens_seed=5),
        # a decode step over ragged long recordings
        dict(name="attention_16x8000_40000_int8", kind="attention", prec="int8", batch=16, lo=8000, hi=40000,
             count=1, window=0, sinks=0, lens_seed=6),
        # a prefill chunk of eight prompts in their contexts
        dict(name="attention_8x512_at_1500_8000_bf16", kind="attention", prec="bf16", batch=8, lo=1500,
             hi=8000, count=512, window=0, sinks=0, lens_seed=7),
        # a live recording's prompt under a sliding window that keeps its first tokens
        dict(name="attention_1x9001_window2048_int8", kind="attention", prec="int8", batch=1, lo=9001, hi=9001,
             count=9001, window=2048, sinks=20, lens_seed=8),
        # eight candidates of one sequence each get their own last page
        dict(name="pages_8x28", kind="pages", layers=28, pages=8, pool=64, lens_seed=9),
        # a long recording copied whole (16,384 tokens)
        dict(name="pages_256x28", kind="pages", layers=28, pages=256, pool=600, lens_seed=10),
        # a decode step's tokens with five alternatives each
        dict(name="logprobs_8_f32_top5", kind="logprobs", dtype="f32", rows=8, vocab=VOCAB, top=5, masked=0.0),
        # a transcript's tokens scored after the fact, some of the vocabulary ruled out
        dict(name="logprobs_1000_bf16_top8", kind="logprobs", dtype="bf16", rows=1000, vocab=VOCAB, top=8,
             masked=0.3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "pages",
                       "logprobs", "logprobs"])
    seed = rng.randrange(1 << 20)
    if kind == "pages":
        n = _log_int(rng, 1, 256)
        return dict(kind=kind, layers=_log_int(rng, 1, 28), pages=n, pool=2 * n + rng.randint(0, 50), lens_seed=seed)
    if kind == "logprobs":
        vocab = _log_int(rng, 500, VOCAB)
        return dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16"]), rows=_log_int(rng, 1, 500), vocab=vocab,
                    top=rng.randint(1, 20), masked=rng.choice([0.0, 0.3, 0.9]))
    prec = rng.choice(["bf16", "bf16", "int8", "int8", "f32"])
    batch = _log_int(rng, 1, 16)
    if kind == "append":
        lo, n = rng.choice([0, rng.randint(1, 9000)]), _log_int(rng, 1, 300 if prec == "f32" else 600)
        return dict(kind=kind, prec=prec, batch=batch, lo=lo, hi=2 * lo, count_lo=n,
                    count_hi=n + rng.randint(0, n // 10), lens_seed=seed)
    window = rng.choice([0, 0, rng.randint(1, 200), _log_int(rng, 100, 8000)])
    sinks = rng.choice([0, rng.randint(1, 200)]) if window else 0
    if rng.random() < 0.5:
        lo = _log_int(rng, 1, 15000)
        return dict(kind=kind, prec=prec, batch=batch, lo=lo, hi=lo * rng.randint(1, 2), count=1, window=window,
                    sinks=sinks, lens_seed=seed)
    n = _log_int(rng, 2, (1000 if prec == "f32" else 3000) // batch)
    lo = n + rng.randint(0, 3000)
    return dict(kind=kind, prec=prec, batch=batch, lo=lo, hi=lo + rng.randint(0, 1000), count=n, window=window,
                sinks=sinks, lens_seed=seed)


# --- inputs --------------------------------------------------------------------


def _gen(seed, tag):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + zlib.crc32(tag.encode())) % (1 << 31))
    return g


def _normal(seed, tag, shape, dtype, std=1.0, mean=0.0):
    x = torch.randn(shape, generator=_gen(seed, tag), device=DEV, dtype=torch.float32)
    return (x * std + mean).to(dtype)


def _lens(case, lo="lo", hi="hi", salt=0):
    r = np.random.default_rng([case["lens_seed"], salt])
    return [int(n) for n in r.integers(case[lo], case[hi] + 1, case["batch"])]


def _cache_rows(case, seed):
    """The keys (rotated) and values of each sequence: some key channels carry
    most of a key's length, as trained models' do."""
    dt = ACT[case["prec"]]
    wide = torch.exp(_normal(seed, "wide", (1, NKV, HD), torch.float32, std=0.7))
    out = []
    for i, n in enumerate(_lens(case)):
        k = (_normal(seed, f"k{i}", (n, NKV, HD), torch.float32) * wide).to(dt)
        out.append((k, _normal(seed, f"v{i}", (n, NKV, HD), dt)))
    return out


def _queries(case, seed):
    return _normal(seed, "q", (case["batch"] * case["count"], NH, HD), ACT[case["prec"]], std=1.5)


def _append_inputs(case, seed):
    dt = ACT[case["prec"]]
    starts, counts = _lens(case), _lens(case, "count_lo", "count_hi", 1)
    qkv = _normal(seed, "qkv", (sum(counts), (NH + 2 * NKV) * HD), dt, std=0.8)
    gains = [_normal(seed, t, (HD,), dt, std=0.1, mean=1.0) for t in ("q_norm", "k_norm")]
    pos = torch.cat([torch.arange(s, s + c, device=DEV) for s, c in zip(starts, counts)])
    return starts, counts, qkv, gains, pos


def _logits(case, seed):
    n, v = case["rows"], case["vocab"]
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[case["dtype"]]
    x = _normal(seed, "logits", (n, v), torch.float32, std=2.5)
    best = torch.randint(0, v, (n,), generator=_gen(seed, "best"), device=DEV)
    rows = torch.arange(n, device=DEV)
    x[rows, best] += 6.0 + _normal(seed, "margin", (n,), torch.float32, std=3.0)
    if case["masked"]:
        x.masked_fill_(torch.rand((n, v), generator=_gen(seed, "mask"), device=DEV) < case["masked"], -math.inf)
        x[rows, best] = 14.0   # what is asked for is not ruled out
    other = torch.randint(0, v, (n,), generator=_gen(seed, "other"), device=DEV)
    x[rows, other] = x[rows, other].clamp(min=-4.0)
    pick = torch.rand((n,), generator=_gen(seed, "pick"), device=DEV) < 0.8
    return x.to(dt), torch.where(pick, best, other).to(torch.int32)


def _copy_lists(case):
    r = np.random.default_rng([case["lens_seed"], 2])
    ids = r.permutation(case["pool"])[: 2 * case["pages"]]
    return [int(i) for i in ids[: case["pages"]]], [int(i) for i in ids[case["pages"]:]]


def _pool_words(case, seed):
    return torch.randint(-(1 << 31), 1 << 31, (case["layers"], case["pool"], PAGE_BYTES // 4),
                         generator=_gen(seed, "pool"), device=DEV, dtype=torch.int32)


def _rope_tables(n, dt):
    """The model's tables: f32 angles, their cosine and sine in its activation type."""
    inv = (1.0 / (1e6 ** (torch.arange(0, HD, 2, dtype=torch.float64) / HD))).float().to(DEV)
    a = (torch.arange(n, device=DEV).float()[:, None] * inv[None]).double()
    return torch.cos(a).float().to(dt), torch.sin(a).float().to(dt)


# --- the 4 bits, in plain operations --------------------------------------------

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exponent_range(dt):
    return (-23, 13) if dt == torch.float16 else (-64, 64)


def _encode(x, dt):
    """f32 values (..., 128) -> codes 0..7 with the sign in bit 3, and an exponent per 32."""
    x = x.reshape(*x.shape[:-1], HD // 32, 32)
    m, e = torch.frexp(x.abs().amax(-1))                       # max = m 2^e, m in [0.5, 1)
    e = torch.where(m * 8 > 7, e - 2, e - 3).clamp(*_exponent_range(dt))
    t = torch.ldexp(x.abs(), -e[..., None])
    code = ((t > 0.25).to(torch.uint8) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5.0))
    return (code + 8 * (x < 0)).to(torch.uint8), e.to(torch.int8)


def _decode(code, e):
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=DEV)
    x = torch.ldexp(table[code.int()], e[..., None].int())
    return x.reshape(*x.shape[:-2], HD)


# --- what a user has in hand ------------------------------------------------------


def _model(prec, layers, max_len):
    fmd = importlib.import_module("fast-moss-diarization_amd")
    cfg = fmd.TextConfig(vocab_size=2048, hidden_size=256, intermediate_size=256, num_hidden_layers=layers,
                         num_attention_heads=NH, num_key_value_heads=NKV, head_dim=HD, rms_norm_eps=EPS,
                         rope_theta=1e6)
    m = fmd.Qwen3(cfg, prec, max_len=max_len)
    stream = torch.cuda.Stream()
    m.set_stream(stream.cuda_stream)
    return fmd, m, stream


def prepare(case, seed):
    s = dict(case=case, own=own)
    kind = case["kind"]
    if kind == "append":
        starts, counts, qkv, gains, pos = _append_inputs(case, seed)
        s.update(qkv=qkv)
        if own:
            fmd, m, s["stream"] = _model(case["prec"], 1, max(a + b for a, b in zip(starts, counts)))
            m.set_weight("layers.0.self_attn.q_norm.weight", gains[0])
            m.set_weight("layers.0.self_attn.k_norm.weight", gains[1])
            pages = sum((a + b + PAGE - 1) // PAGE for a, b in zip(starts, counts))
            c = fmd.PagedKvCache(m, pages=pages, max_seqs=case["batch"], max_rows=MAX_ROWS)
            seqs = [c.open() for _ in starts]
            for i, n in zip(seqs, starts):
                for at in range(0, n, MAX_ROWS):
                    c.plan([i], [min(MAX_ROWS, n - at)])
            c.plan(seqs, counts)
            dt, n = qkv.dtype, qkv.shape[0]
            s.update(model=m, cache=c, q=torch.empty((n, NH, HD), device=DEV, dtype=dt),
                     k=torch.empty((n, NKV, HD), device=DEV, dtype=dt),
                     v=torch.empty((n, NKV, HD), device=DEV, dtype=dt))
        else:
            tables = _rope_tables(int(pos.max()) + 1, qkv.dtype)
            s.update(gains=gains, cos=tables[0][pos], sin=tables[1][pos])
    elif kind == "attention":
        rows, count = _cache_rows(case, seed), case["count"]
        s.update(q=_queries(case, seed))
        if own:
            fmd, m, s["stream"] = _model(case["prec"], 1, max(k.shape[0] for k, _ in rows))
            pages = sum((k.shape[0] + PAGE - 1) // PAGE for k, _ in rows)
            c = fmd.PagedKvCache(m, pages=pages, max_seqs=case["batch"], max_rows=MAX_ROWS,
                                 window=case["window"], sinks=case["sinks"])
            seqs = [c.open() for _ in rows]
            with torch.cuda.stream(s["stream"]):
                s["stream"].wait_stream(torch.cuda.default_stream())
                for i, (k, v) in zip(seqs, rows):
                    for at in range(0, k.shape[0] - count, MAX_ROWS):
                        n = min(MAX_ROWS, k.shape[0] - count - at)
                        c.plan([i], [n])
                        c.write(0, k[at:].data_ptr(), v[at:].data_ptr())
                c.plan(seqs, [count] * len(rows))
                k, v = (torch.cat([r[j][-count:] for r in rows]) for j in (0, 1))
                c.write(0, k.data_ptr(), v.data_ptr())
            torch.cuda.synchronize()
            s.update(model=m, cache=c, ctx=torch.empty_like(s["q"]))
        else:
            dt = ACT[case["prec"]]
            s["kv"] = [(_encode(k.float(), dt), _encode(v.float(), dt)) for k, v in rows]
    elif kind == "pages":
        s["src"], s["dst"] = _copy_lists(case)
        pool = _pool_words(case, seed)
        if own:
            fmd, m, s["stream"] = _model("bf16", case["layers"], PAGE)
            c = fmd.PagedKvCache(m, pages=case["pool"], max_seqs=1, max_rows=PAGE)
            s.update(model=m, cache=c, pool=c.pool().view(torch.int32))
            s["pool"].copy_(pool)
            torch.cuda.synchronize()
        else:
            s.update(pool=pool, src=torch.tensor(s["src"], device=DEV), dst=torch.tensor(s["dst"], device=DEV))
    else:
        s["logits"], s["targets"] = _logits(case, seed)
        if own:
            _, m, s["stream"] = _model("bf16", 1, PAGE)
            n, top = case["rows"], case["top"]
            s.update(model=m, logp=torch.empty(n, device=DEV), entropy=torch.empty(n, device=DEV),
                     ids=torch.empty((n, top), device=DEV, dtype=torch.int32), best=torch.empty((n, top), device=DEV))
    torch.cuda.synchronize()
    return s


# --- one pass ----------------------------------------------------------------------


def run(s):
    case = s["case"]
    return {"append": _run_append, "attention": _run_attention, "pages": _run_pages,
            "logprobs": _run_logprobs}[case["kind"]](s, case)


def _run_append(s, case):
    qkv = s["qkv"]
    if s["own"]:
        s["cache"].append(0, qkv.data_ptr(), s["q"].data_ptr())
        s["cache"].read(0, s["k"].data_ptr(), s["v"].data_ptr())
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    # 64 bits up to the rounding: a key next to a border falls on its own side
    n, dt = qkv.shape[0], qkv.dtype
    x = qkv[:, : (NH + NKV) * HD].double().reshape(n, NH + NKV, HD)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    x = x * torch.cat([s["gains"][0].double().expand(NH, HD), s["gains"][1].double().expand(NKV, HD)])
    c, sn = s["cos"].double()[:, None], s["sin"].double()[:, None]
    lo, hi = x[..., : HD // 2], x[..., HD // 2:]
    x = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1)
    v = qkv[:, (NH + NKV) * HD:].float().reshape(n, NKV, HD)
    return {"q": x[:, :NH].to(dt), "k": _decode(*_encode(x[:, NH:].float(), dt)).to(dt),
            "v": _decode(*_encode(v, dt)).to(dt)}


def _visible(first, n, lo, hi, window, sinks):
    """Which of the keys lo .. hi - 1 the queries at positions first .. first + n - 1 see."""
    p = torch.arange(first, first + n, device=DEV)[:, None]
    j = torch.arange(lo, hi, device=DEV)[None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    return seen


def _run_attention(s, case):
    q = s["q"]
    if s["own"]:
        s["cache"].attention(0, q.data_ptr(), s["ctx"].data_ptr())
        return s["ctx"]
    out, count, step = torch.empty_like(q), case["count"], 1024
    for i, (k, v) in enumerate(s["kv"]):
        L = k[0].shape[0]
        k, v = _decode(*k).transpose(0, 1).contiguous(), _decode(*v).transpose(0, 1).contiguous()
        kt = k.transpose(1, 2).contiguous()
        for at in range(0, count, step):
            n = min(step, count - at)
            first, end = L - count + at, L - count + at + n
            rows = slice(i * count + at, i * count + at + n)
            x = q[rows].float().reshape(n, NKV, REP, HD).permute(1, 2, 0, 3).reshape(NKV, REP * n, HD)
            w = torch.bmm(x, kt[:, :, :end].contiguous()) * (HD ** -0.5)
            w = w.reshape(NKV, REP, n, end).masked_fill(
                ~_visible(first, n, 0, end, case["window"], case["sinks"]), -math.inf)
            w = torch.exp(w - w.amax(-1, keepdim=True))
            w = w / w.sum(-1, keepdim=True)
            o = torch.bmm(w.reshape(NKV, REP * n, end), v[:, :end].contiguous())
            out[rows] = o.reshape(NKV, REP, n, HD).permute(2, 0, 1, 3).reshape(n, NH, HD).to(q.dtype)
    return out


def _run_pages(s, case):
    if s["own"]:
        s["cache"].copy_pages(s["src"], s["dst"])
    else:
        s["pool"][:, s["dst"]] = s["pool"][:, s["src"]]
    return s["pool"]


def _run_logprobs(s, case):
    x, t, top = s["logits"], s["targets"], case["top"]
    if s["own"]:
        s["model"].op_logprobs(x.data_ptr(), case["dtype"], case["rows"], case["vocab"], t.data_ptr(), top,
                               s["logp"].data_ptr(), s["entropy"].data_ptr(), s["ids"].data_ptr(),
                               s["best"].data_ptr())
        return {"logp": s["logp"], "entropy": s["entropy"], "ids": s["ids"], "best": s["best"]}
    x = x.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.double().sum(-1)     # a sum next to 1 has its logarithm in its last bits
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, e * d, 0.0).double().sum(-1) / total
    # the order of (value, lower index first) as one integer
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) - torch.arange(x.shape[1], device=DEV)
    ids = torch.topk(key, top, -1).indices
    return {"logp": (d.gather(1, t.long()[:, None])[:, 0].double() - lse).float(), "entropy": entropy.float(),
            "ids": ids.int(), "best": (d.gather(1, ids).double() - lse[:, None]).float()}


# --- what a pass cannot do without -------------------------------------------------


def _pairs(case):
    """(query, key) pairs of one head, and the keys that any query sees."""
    pairs = keys = 0
    w, z, count = case["window"], case["sinks"], case["count"]
    for n in _lens(case):
        p = np.arange(n - count, n, dtype=np.int64)
        lo = np.maximum(0, p - w + 1) if w else np.zeros_like(p)
        pairs += int((p + 1 - lo + np.minimum(z, lo)).sum())
        keys += n - int(lo[0]) + min(z, int(lo[0]))
    return pairs, keys


def work(case):
    kind = case["kind"]
    if kind == "pages":
        return {"bytes": 2.0 * case["layers"] * case["pages"] * PAGE_BYTES, "flops": 0.0}
    if kind == "logprobs":
        n, v = case["rows"], case["vocab"]
        esz = 4 if case["dtype"] == "f32" else 2
        return {"bytes": float(n) * (v * esz + 12 + 8 * case["top"]), "flops": 6.0 * n * v}
    esz = 4 if case["prec"] == "f32" else 2
    token = PAGE_BYTES // PAGE     # bytes of a token's K and V
    if kind == "append":
        n = float(sum(_lens(case, "count_lo", "count_hi", 1)))
        return {"bytes": n * ((NH + 2 * NKV) * HD * esz + NH * HD * esz + token + 2 * NKV * HD * esz + 2 * 64 * esz),
                "flops": n * HD * (NH + NKV) * 7.0}
    pairs, keys = _pairs(case)
    rows = case["batch"] * case["count"]
    return {"bytes": float(keys) * token + 2.0 * rows * NH * HD * esz, "flops": 4.0 * HD * NH * pairs}


# --- the same in 64 bits -------------------------------------------------------------


def _nearest(x, dt):
    """The values that 4 bits keep of x (..., 128), by distance."""
    x = x.to(torch.float32).double().reshape(*x.shape[:-1], 4, 32)
    lo, hi = _exponent_range(dt)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 7.0))
    for _ in range(2):   # log2's last bit does not decide
        e = torch.where(top > 7.0 * torch.exp2(e), e + 1, torch.where(top <= 7.0 * torch.exp2(e - 1), e - 1, e))
    e = torch.where(top > 0, e, lo).clamp(lo, hi)
    t = x / torch.exp2(e)
    kept = torch.zeros_like(t)
    far = t.abs().clamp(max=6.0)
    away = far.clone()
    # even last bits (0, 1, 2, 4) first: an odd one has to be nearer to win
    for level in (1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):
        d = (far - level).abs()
        kept, away = torch.where(d < away, level, kept), torch.minimum(d, away)
    return (torch.sign(t) * kept * torch.exp2(e)).reshape(*x.shape[:-2], HD)


def _exact_append(case, seed):
    _, _, qkv, gains, pos = _append_inputs(case, seed)
    n, dt = qkv.shape[0], qkv.dtype
    cos, sin = (t.double()[pos] for t in _rope_tables(int(pos.max()) + 1, dt))

    def turned(x, g):
        x = x.double() * torch.rsqrt(x.double().pow(2).sum(-1, keepdim=True) / HD + EPS) * g.double()
        out = torch.empty_like(x)
        out[..., :64] = x[..., :64] * cos[:, None] - x[..., 64:] * sin[:, None]
        out[..., 64:] = x[..., 64:] * cos[:, None] + x[..., :64] * sin[:, None]
        return out

    q, k, v = (t.reshape(n, -1, HD) for t in qkv.split([NH * HD, NKV * HD, NKV * HD], -1))
    return {"q": turned(q, gains[0]), "k": _nearest(turned(k, gains[1]), dt), "v": _nearest(v, dt)}


def _exact_attention(case, seed):
    q, count, dt = _queries(case, seed).double(), case["count"], ACT[case["prec"]]
    out = torch.empty_like(q)
    for i, (k, v) in enumerate(_cache_rows(case, seed)):
        L = k.shape[0]
        k, v = _nearest(k, dt), _nearest(v, dt)
        for at in range(0, count, 512):
            n = min(512, count - at)
            first = L - count + at
            # under a window only the sinks and the keys from `lo` on are looked at
            w, z = case["window"], case["sinks"]
            lo = max(0, first - w + 1) if w else 0
            at_keys = torch.cat([torch.arange(0, min(z, lo), device=DEV), torch.arange(lo, first + n, device=DEV)])
            p = torch.arange(first, first + n, device=DEV)[:, None]
            hidden = at_keys[None] > p
            if w:
                hidden |= (at_keys[None] <= p - w) & (at_keys[None] >= z)
            rows = slice(i * count + at, i * count + at + n)
            for h in range(NH):
                sc = (q[rows, h] @ k[at_keys, h // REP].t()) / math.sqrt(HD)
                out[rows, h] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ v[at_keys, h // REP]
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "append":
        return _exact_append(case, seed)
    if kind == "attention":
        return _exact_attention(case, seed)
    if kind == "pages":
        return None
    x, t = _logits(case, seed)
    logp, ent, best = [], [], []
    for r in range(0, x.shape[0], 100):   # in pieces: 64 bits of the whole take gigabytes
        lp = torch.log_softmax(x[r:r + 100].double(), -1)
        logp.append(lp.gather(1, t[r:r + 100].long()[:, None])[:, 0])
        ent.append(torch.special.entr(lp.exp()).sum(-1))
        best.append(torch.topk(lp, case["top"], -1).values)
    return {"logp": torch.cat(logp), "entropy": torch.cat(ent), "ids": None, "best": torch.cat(best)}
