"""The paged cache's host side (csrc/pkv_pages.h) without a device: random
sequences of calls against a model of what each sequence's tokens are, failures
that change nothing, and plans whose items cover what each row sees exactly once
and stay inside their bounds."""
import ctypes
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
HDR = dict(ROWS=0, PAGES=3, NDEC=4, NWORK=5, NSPLIT=6, WORK=7, PITEM=8, SPLIT=9, WORDS=32, ITEMS=32 + 512)
P = 64


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = tmp_path_factory.mktemp("pkv") / "shim.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC",
                    f"-I{ROOT / 'fast-moss-diarization_amd' / 'csrc'}",
                    str(ROOT / "tests" / "pkv_pages_shim.cpp"), "-o", str(out)], check=True)
    h = ctypes.CDLL(str(out))
    I, V, PI = ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int32)
    for name, res, args in (("pages_new", V, [I] * 6), ("pages_delete", None, [V]), ("pages_error", ctypes.c_char_p, [V]),
                            ("pages_open", I, [V, PI]), ("pages_fork", I, [V, I, PI]), ("pages_copy", I, [V, I, PI]),
                            ("pages_free", I, [V, I]), ("pages_truncate", I, [V, I, I]),
                            ("pages_extend", I, [V, I, PI, PI]), ("pages_compact", I, [V, I, I]), ("copies_n", I, []),
                            ("copies_src", PI, []), ("copies_dst", PI, []), ("pages_len", I, [V, I]),
                            ("pages_n", I, [V, I]), ("pages_of", PI, [V, I]), ("pages_refs", PI, [V]),
                            ("pages_free_n", I, [V]), ("pages_plan", I, [V, I, I, I, PI, PI]), ("plan_words", PI, []), ("plan_far", I, [ctypes.POINTER(PI)]),
                            ("plan_bounds", None, [I] * 5 + [ctypes.POINTER(ctypes.c_int64)])):
        fn = getattr(h, name)
        fn.restype, fn.argtypes = res, args
    return h


def arr(v):
    return (ctypes.c_int32 * max(len(v), 1))(*v)


class Pages:
    """The tables with a content model: page id -> token names, sequence -> tokens."""

    def __init__(self, shim, pages, seqs, rows, max_len, window=0, sinks=0):
        self.h, self.pages, self.window, self.sinks = shim, pages, window, sinks
        self.p = shim.pages_new(pages, seqs, rows, max_len, window, sinks)
        self.mem = {i: [None] * P for i in range(pages)}
        self.tok = {}
        self.next = 0

    def close(self):
        self.h.pages_delete(self.p)

    def table(self, s):
        return self.h.pages_of(self.p, s)[: self.h.pages_n(self.p, s)]

    def refs(self):
        return self.h.pages_refs(self.p)[: self.pages]

    def state(self):
        return ([(s, self.h.pages_len(self.p, s), self.table(s)) for s in self.tok], self.refs(),
                self.h.pages_free_n(self.p))

    def error(self):
        return self.h.pages_error(self.p).decode()

    def copies(self, new_pool=False):
        n = self.h.copies_n()
        src, dst = self.h.copies_src()[:n], self.h.copies_dst()[:n]
        assert len(set(dst)) == n
        if not new_pool:
            assert not set(src) & set(dst), "a page is both read and written"
        old = self.mem
        if new_pool:
            self.mem = {i: [None] * P for i in range(self.pages)}
        for a, b in zip(src, dst):
            self.mem[b] = list(old[a])

    def new(self, fn, *args):
        out = ctypes.c_int32(-1)
        rc = fn(self.p, *args, ctypes.byref(out))
        return rc, out.value

    def open(self):
        rc, s = self.new(self.h.pages_open)
        if rc == 0:
            self.tok[s] = []
        return rc, s

    def fork(self, s):
        rc, t = self.new(self.h.pages_fork, s)
        if rc == 0:
            self.tok[t] = list(self.tok[s])
        return rc, t

    def copy(self, s):
        rc, t = self.new(self.h.pages_copy, s)
        if rc == 0:
            self.copies()
            self.tok[t] = list(self.tok[s])
        return rc, t

    def free(self, s):
        rc = self.h.pages_free(self.p, s)
        if rc == 0:
            del self.tok[s]
        return rc

    def truncate(self, s, n):
        rc = self.h.pages_truncate(self.p, s, n)
        if rc == 0:
            del self.tok[s][n:]
        return rc

    def extend(self, seqs, counts):
        rc = self.h.pages_extend(self.p, len(seqs), arr(seqs), arr(counts))
        if rc == 0:
            self.copies()
            for s, n in zip(seqs, counts):
                for _ in range(n):
                    at = len(self.tok[s])
                    self.tok[s].append(self.next)
                    self.mem[self.table(s)[at // P]][at % P] = self.next
                    self.next += 1
        return rc

    def compact(self, pages, new_pool):
        rc = self.h.pages_compact(self.p, pages, int(new_pool))
        if rc == 0:
            self.pages = pages
            self.copies(new_pool)
        return rc

    def check(self):
        refs = [0] * self.pages
        for s, tok in self.tok.items():
            t = self.table(s)
            assert self.h.pages_len(self.p, s) == len(tok) and len(t) == -(-len(tok) // P)
            lo = max(0, len(tok) - self.window + 1) if self.window else 0
            for i, page in enumerate(t):
                if page >= 0:
                    refs[page] += 1
                    n = min(P, len(tok) - i * P)
                    assert self.mem[page][:n] == tok[i * P:i * P + n], "a page holds another sequence's tokens"
                else:
                    assert self.window and (i + 1) * P <= lo and i * P >= self.sinks, "a visible page was released"
        assert refs == self.refs()
        assert self.h.pages_free_n(self.p) == refs.count(0)


@pytest.mark.parametrize("seed", range(12))
def test_random_calls(shim, seed):
    r = random.Random(seed)
    window = r.choice([0, 0, 1, 30, 64, 200])
    c = Pages(shim, r.randint(4, 40), 6, 700, 2000, window, r.choice([0, 5, 64, 150]) if window else 0)
    try:
        for _ in range(400):
            before = c.state()
            live = list(c.tok)
            op = r.choice(["open", "fork", "copy", "free", "truncate", "extend", "extend", "extend", "extend", "compact"])
            if op == "open" or not live:
                rc, s = c.open()
            elif op in ("fork", "copy"):
                rc, s = getattr(c, op)(r.choice(live))
            elif op == "free":
                rc = c.free(r.choice(live))
            elif op == "truncate":
                s = r.choice(live)
                rc = c.truncate(s, r.randint(0, len(c.tok[s])))
            elif op == "compact":
                n = r.choice([c.pages, c.pages, r.randint(1, 45)])
                rc = c.compact(n, n != c.pages)
            else:
                pick = r.sample(live, r.randint(1, len(live)))
                rc = c.extend(pick, [r.choice([0, 1, 1, 1, r.randint(1, 150)]) for _ in pick])
            if rc:
                assert rc in (-1, -2, -5) and c.error()
                assert c.state() == before, f"{op} failed and changed something"
            c.check()
    finally:
        c.close()


def test_shared_page_is_copied_by_all_writers_but_the_last(shim):
    c = Pages(shim, 8, 4, 700, 2000)
    _, a = c.open()
    assert c.extend([a], [70]) == 0
    _, b = c.fork(a)
    _, d = c.fork(a)
    assert c.h.pages_free_n(c.p) == 6
    assert c.extend([a, b, d], [1, 1, 1]) == 0
    assert c.h.copies_n() == 2 and c.h.pages_free_n(c.p) == 4    # d keeps the page
    c.check()
    assert c.refs()[c.table(a)[0]] == 3                          # the full page stays shared
    c.close()


def test_refusals(shim):
    c = Pages(shim, 3, 2, 100, 150)
    _, a = c.open()
    _, b = c.open()
    assert c.open()[0] == -5
    for seqs, counts, rc, text in (([a, a], [1, 1], -1, "named twice"), ([7], [1], -1, "no such sequence"),
                                   ([-1], [1], -1, "no such sequence"), ([a], [-1], -1, "negative"),
                                   ([a], [101], -1, "at a time"), ([a, b], [60, 60], -1, "at a time"),
                                   ([a, b, a], [1, 1, 1], -1, "more sequences")):
        assert c.extend(seqs, counts) == rc and text in c.error(), (seqs, counts)
    assert c.extend([a], [100]) == 0
    assert c.extend([a], [51]) == -1 and "RoPE" in c.error()
    assert c.extend([b], [65]) == -5 and "2 pages needed, 1 of 3 free" in c.error()
    assert c.truncate(a, 101) == -1 and c.truncate(a, -1) == -1
    assert c.compact(1, True) == -1 and "2 pages are in use" in c.error()
    assert c.free(b) == 0 and c.free(b) == -1
    assert c.copy(a)[0] == -5
    c.close()


def test_window_gives_pages_back_and_refuses_to_go_back(shim):
    c = Pages(shim, 5, 1, 64, 2000, window=100, sinks=10)
    _, a = c.open()
    for _ in range(25):
        assert c.extend([a], [64]) == 0      # 1600 tokens in 5 pages
        c.check()
    t = c.table(a)
    assert t[0] >= 0 and t[1] == -1 and sum(p >= 0 for p in t) <= 4
    assert c.truncate(a, 1400) == -2 and "released" in c.error()
    assert c.truncate(a, 1599) == 0
    c.close()


def _plan(c, nkv, tile, seqs, counts):
    n = c.h.pages_plan(c.p, nkv, tile, len(seqs), arr(seqs), arr(counts))
    return np.array(c.h.plan_words()[:n], dtype=np.int64)


@pytest.mark.parametrize("seed", range(60))
def test_plans_cover_what_each_row_sees_once(shim, seed):
    r = random.Random(1000 + seed)
    nkv, tile = r.choice([1, 2, 8]), r.choice([32, 64, 128])
    n_seqs, max_rows, max_len = r.randint(1, 20), r.choice([20, 700, 5000]), r.choice([300, 9000, 65536])
    window = r.choice([0, 0, r.randint(1, 300), r.randint(1, max_len)])
    sinks = r.choice([0, r.randint(1, 400)]) if window else 0
    c = Pages.__new__(Pages)
    c.h = shim
    c.p = shim.pages_new(n_seqs * (max_len // P + 1), n_seqs, max_rows, max_len, window, sinks)
    try:
        seqs, lens = [], []
        for _ in range(n_seqs):
            out = ctypes.c_int32()
            assert shim.pages_open(c.p, ctypes.byref(out)) == 0
            seqs.append(out.value)
            lens.append(0)
        style = r.choice(["decode", "many", "mixed"])
        counts = []
        room = max_rows
        for i in range(n_seqs):
            m = 1 if style == "decode" else r.choice([0, 1, r.randint(1, 64), r.randint(1, 2000)])
            counts.append(min(m, room, max_len))
            room -= counts[-1]
        # lengths before the plan
        for i, s in enumerate(seqs):
            left = r.randint(0, max_len - counts[i])
            while left:
                m = min(left, max_rows)
                assert shim.pages_extend(c.p, 1, arr([s]), arr([m])) == 0
                lens[i] += m
                left -= m
        assert shim.pages_extend(c.p, n_seqs, arr(seqs), arr(counts)) == 0
        w = _plan(c, nkv, tile, seqs, counts)
        b = (ctypes.c_int64 * 5)()
        shim.plan_bounds(nkv, n_seqs, max_rows, max_len, tile, b)
        assert len(w) <= b[3] and w[HDR["NDEC"]] <= b[0]
        rows = sum(counts)
        assert w[HDR["ROWS"]] == rows
        row0 = np.concatenate([[0], np.cumsum(counts)])
        seq_at = {int(row0[i]) + k: i for i in range(n_seqs) for k in range(counts[i])}
        far = ctypes.POINTER(ctypes.c_int32)()
        n_far = shim.plan_far(ctypes.byref(far))
        assert n_far == (2 * rows if rows > 256 else 0) and b[3] + n_far <= b[4]
        at = np.array(far[:n_far] if n_far else w[HDR["WORDS"]:][: 2 * rows]).reshape(-1, 2)
        tables = [shim.pages_of(c.p, s)[: shim.pages_n(c.p, s)] for s in seqs]
        for row, (pos, page) in enumerate(at.tolist()):
            i = seq_at[row]
            assert pos == lens[i] + row - row0[i] and page == tables[i][pos // P]
        seen_pages = {row: [] for row in range(rows)}
        slots = {}

        def walk(row, pos, n, table, sp, wp, v0, v1, slot):
            i = seq_at[row]
            assert w[table:table + len(tables[i])].tolist() == tables[i]
            assert pos == lens[i] + row - row0[i] and 0 <= v0 < v1
            pages = [v if v < sp else wp + v - sp for v in range(v0, v1)]
            for pg in pages:
                assert w[table + pg] >= 0, "an item names a released page"
            for k in range(n):
                assert seq_at[row + k] == i
                seen_pages[row + k] += pages
            return slot

        dec = w[HDR["ITEMS"]:][: 16 * w[HDR["NDEC"]]].reshape(-1, 16)
        for row, pos, table, sp, wp, v0, v1, slot, first, parts, *ids in dec.tolist():
            walk(row, pos, 1, table, sp, wp, v0, v1, slot)
            for j in range(4):
                v = min(v0 + j, v1 - 1)
                assert ids[j] == w[table + (v if v < sp else wp + v - sp)]
            assert first <= slot < first + parts and slot < b[0] and slot not in slots
            slots[slot] = (row, first, parts)
        for slot, (row, first, parts) in slots.items():
            assert all(slots[first + k] == (row, first, parts) for k in range(parts))
        slots.clear()
        work = w[w[HDR["WORK"]]:][: w[HDR["NWORK"]] + 1].tolist()
        assert work[0] == 0 and work == sorted(set(work)) and len(work) <= b[2] + 1
        pre = w[w[HDR["PITEM"]]:][: 12 * work[-1]].reshape(-1, 12)
        loads = [int((pre[x:y, 7] - pre[x:y, 6]).sum()) for x, y in zip(work, work[1:])]
        assert len(set(loads[:-1])) <= 1 and (not loads or loads[-1] <= loads[0])
        for row, pos, n, table, sp, wp, v0, v1, slot, *_ in pre.tolist():
            assert 1 <= n <= tile
            walk(row, pos, n, table, sp, wp, v0, v1, slot)
            if slot >= 0:
                assert slot < b[2] and slot not in slots
                slots[slot] = (row, n)
        for row, n, first, parts in w[w[HDR["SPLIT"]]:][: 4 * w[HDR["NSPLIT"]]].reshape(-1, 4).tolist():
            assert parts > 1 and all(slots.pop(first + k) == (row, n) for k in range(parts))
        assert not slots
        for row in range(rows):
            i = seq_at[row]
            p = lens[i] + row - int(row0[i])
            lo = max(0, p - window + 1) if window else 0
            need = set(range(lo // P, p // P + 1)) | set(range(0, -(-min(sinks, lo) // P)))
            assert len(seen_pages[row]) == len(set(seen_pages[row])), "a page is counted twice"
            assert need <= set(seen_pages[row]), (row, p)
    finally:
        shim.pages_delete(c.p)


def test_entry_points_refuse_null_handles_without_a_device(fmd):
    lib, n = fmd.lib(), ctypes.c_int32()
    h, p, z = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_size_t()
    calls = [lambda: lib.fmd_pkv_create(None, 1, 1, 1, 0, 0, ctypes.byref(h)), lambda: lib.fmd_pkv_open(None, ctypes.byref(n)),
             lambda: lib.fmd_pkv_fork(None, 0, ctypes.byref(n)), lambda: lib.fmd_pkv_copy(None, 0, ctypes.byref(n)),
             lambda: lib.fmd_pkv_free(None, 0), lambda: lib.fmd_pkv_truncate(None, 0, 0),
             lambda: lib.fmd_pkv_resize(None, 1), lambda: lib.fmd_pkv_len(None, 0), lambda: lib.fmd_pkv_free_pages(None),
             lambda: lib.fmd_pkv_pages(None, 0, None, 0, ctypes.byref(n)),
             lambda: lib.fmd_pkv_pool(None, ctypes.byref(p), ctypes.byref(z)), lambda: lib.fmd_pkv_plan(None, 0, None, None),
             lambda: lib.fmd_op_pkv_append(None, None, 0, None, None), lambda: lib.fmd_op_pkv_write(None, None, 0, None, None),
             lambda: lib.fmd_op_pkv_read(None, None, 0, None, None),
             lambda: lib.fmd_op_pkv_attention(None, None, 0, None, None),
             lambda: lib.fmd_op_pkv_copy_pages(None, 0, None, None),
             lambda: lib.fmd_dec_step(None, None, 1, None, None, None, None, 0, None),
             lambda: lib.fmd_op_logprobs(None, None, 0, 1, 1, 1, None, 0, None, None, None, None),
             lambda: lib.fmd_dec_logprobs(None, 1, None, 0, None, None, None, None)]
    for i, call in enumerate(calls):
        assert call() == -1, i
    assert lib.fmd_pkv_destroy(None) == 0
    assert lib.fmd_pkv_bytes(None, 5) == 0
