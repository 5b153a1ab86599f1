"""Penalties, biases, bans and masks on logits on the device against their
restatement (logits_ref.py), bit for bit — needs an MI355X."""
import ctypes as C

import numpy as np
import pytest

import ctbind as cb
import logits_ref as ref
from w4_ref import Mem

pytestmark = pytest.mark.gpu

PARTS = ("hist_len", "prompt_len", "repeat", "frequency", "presence", "ngram", "bias_start", "bias_id", "bias", "mask_of")


class Call:
    """A call over device copies of what logits_ref.process takes."""

    def __init__(self, hip, mem, x, out=True, ids=True, pad=(0, 0), in_place=False, **kw):
        self.hip, self.mem, self.kw, self.shape = hip, mem, kw, x.shape
        rows, vocab = x.shape
        px, py = pad
        fx = np.full((rows, vocab + px), 77.0, np.float32)
        fx[:, :vocab] = x
        self.x = mem.put(fx)
        self.ld_out = vocab + (px if in_place else py)
        self.out = self.x if in_place else mem.put(np.full((rows, self.ld_out), 55.0, np.float32)) if out else 0
        self.behind = 77.0 if in_place else 55.0
        self.id, self.score = mem.put(np.full(rows + 1, 55, np.int32)), mem.put(np.full(rows + 1, 55, np.float32))
        a = self.a = cb.BackendLogits(logits=self.x, out=self.out, ld=vocab + px, ld_out=self.ld_out if self.out else 0,
                                      rows=rows, vocab=vocab, id=self.id if ids else 0, score=self.score if ids else 0)
        for name in PARTS:
            if kw.get(name) is not None:
                v = np.asarray(kw[name])
                setattr(a, name, mem.put(v.astype(np.float32 if v.dtype.kind == "f" else np.int32)))
        if kw.get("hist") is not None:
            a.hist, a.ld_hist = mem.put(kw["hist"].astype(np.int32)), kw["hist"].shape[1]
        if kw.get("bias_id") is not None:
            a.biases = len(kw["bias_id"])
        if kw.get("mask") is not None:
            a.mask, a.masks, a.ld_mask = mem.put(kw["mask"].astype(np.uint32)), len(kw["mask"]), kw["mask"].shape[1]
        n = hip.backend_logits_work(C.byref(a))
        self.work = a.work = mem.put(np.zeros(n + 4, np.float32))
        self.n_work = n

    def launch(self):
        self.hip.backend_logits(C.byref(self.a))

    def results(self):
        rows, vocab = self.shape
        got = self.mem.get(self.out, (rows, self.ld_out), np.float32) if self.out else None
        if got is not None:
            assert np.all(got[:, vocab:] == self.behind)
            got = got[:, :vocab]
        return got, self.mem.get(self.id, (rows + 1,), np.int32), self.mem.get(self.score, (rows + 1,), np.float32)

    def check(self, want, what):
        got, ids, scores = self.results()
        if got is not None:
            assert np.array_equal(np.isnan(got), np.isnan(want[0])), what
            bad = (got != want[0]) & ~np.isnan(got)
            assert not bad.any(), (what, np.argwhere(bad)[:4], got[bad][:4], want[0][bad][:4])
        if self.a.id:
            assert ids[-1] == 55 and scores[-1] == 55, what
            assert np.array_equal(ids[:-1], want[1]), (what, ids, want[1])
            assert np.array_equal(scores[:-1], want[2]), what
        assert np.all(self.mem.get(self.work, (self.n_work,), np.uint32) == 0), what


def run(hip, x, what, **kw):
    pos = {n: kw.pop(n) for n in ("out", "ids", "pad", "in_place") if n in kw}
    c = Call(hip, Mem(hip, 1 << 24), x, **pos, **kw)
    want = ref.process(x, **kw)
    for _ in range(1 if pos.get("in_place") else 2):     # the work is fit for a second call
        c.launch()
        c.check(want, what)
    return c


def everything(rng, rows, vocab, hist, biases, masks):
    words = -(-vocab // 32)
    h = np.minimum((np.exp(rng.random((rows, max(hist, 1))) * np.log(vocab)) - 1).astype(np.int32), vocab - 1)
    if hist > 40:
        h[:, 5:20] = h[:, 25:40]
        h[0, 3:9] = [-1, vocab, 2 ** 31 - 1, -2 ** 31, vocab + 7, 0]     # no tokens of this vocabulary
    lens = rng.integers(0, hist + 1, rows)
    lens[-1] = hist
    if hist > 40 and rows > 2:
        lens[1], lens[2] = 23, hist + 1000
    many = rng.integers(0, biases + 1, rows)
    start = np.concatenate([[0], np.cumsum(many)])
    kw = dict(hist=h, hist_len=lens, prompt_len=lens // 3, repeat=(1 + rng.random(rows)).astype(np.float32),
              frequency=rng.random(rows).astype(np.float32), presence=rng.standard_normal(rows).astype(np.float32),
              ngram=rng.integers(-1, 5, rows))
    if biases:
        ids = rng.integers(0, max(1, vocab // 3), start[-1])              # many twice
        if len(ids) > 3:
            ids[:3] = [-1, vocab, 2 ** 31 - 1]
        kw |= dict(bias_start=start, bias_id=ids, bias=rng.standard_normal(start[-1]).astype(np.float32))
    if masks:
        kw |= dict(mask=rng.integers(0, 2 ** 32, (masks, words + 1), dtype=np.uint32),
                   mask_of=rng.integers(-1, masks, rows))
    return kw


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 5), (5, 31), (4, 33), (3, 4095), (2, 4096), (6, 4097), (5, 16384), (9, 8191),
                                        (3, 50001), (2, 200000)])
def test_all_parts_together(hip, rows, vocab):
    """Vocabularies around every edge, histories from nothing to long, ids out of range."""
    print(f"case: all parts {rows} {vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    for hist, biases, masks in ((0, 0, 0), (1, 3, 1), (60, 20, 3), (900, 700, 2)):
        x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
        run(hip, x, (hist, biases, masks), **everything(rng, rows, vocab, hist, biases, masks))


@pytest.mark.parametrize("name", ["repeat", "frequency", "presence", "ngram", "bias", "mask", "nothing"])
def test_each_part_alone(hip, name):
    """Every part by itself, and none (the largest logit alone), with pitched rows, in place and without a result."""
    print(f"case: alone {name}", flush=True)
    rng = np.random.default_rng(5)
    for vocab in (100, 9000):
        x = (3 * rng.standard_normal((7, vocab))).astype(np.float32)
        kw = everything(rng, 7, vocab, 300, 50, 3)
        keep = {"bias": ("bias_start", "bias_id", "bias"), "mask": ("mask", "mask_of"),
                "nothing": ()}.get(name, ("hist", "hist_len", name))
        kw = {k: v for k, v in kw.items() if k in keep}
        for form in (dict(), dict(pad=(3, 5)), dict(pad=(4, 8)), dict(in_place=True, pad=(1, 0)), dict(out=False), dict(ids=False)):
            run(hip, x, (name, vocab, form), **form, **kw)


def test_ties_and_nothing_left(hip):
    """The lowest id of equal values, zeros of either sign equal; rows of
    -infinity, of NaN, masked whole, with a mask that is not there: -1."""
    print("case: ties", flush=True)
    vocab = 12000
    x = np.full((9, vocab), -3.0, np.float32)
    x[0, [11999, 7000, 4096]] = 2.0
    x[1, 5000:] = -0.0
    x[1, 9000] = 0.0
    x[2] = -np.inf
    x[3] = np.nan
    x[4, [0, 1]] = np.nan, np.inf
    x[5, 10] = 7.0
    x[7, 11999] = np.nan
    x[8] = -np.finfo(np.float32).max
    mask = np.full((2, vocab // 32), 0xFFFFFFFF, np.uint32)
    mask[1] = 0
    kw = dict(mask=mask, mask_of=np.array([-1, 0, 0, -5, 0, 1, 2, 0, 0]))
    c = run(hip, x, "ties", **kw)
    assert list(c.results()[1][:9]) == [4096, 5000, -1, -1, 1, -1, -1, 0, 0]
    c = run(hip, x[:2], "rows' own masks", mask=mask)
    assert list(c.results()[1][:2]) == [4096, -1]


def test_special_values(hip):
    """Infinite and NaN logits under penalties, penalties of 0, below 0 and
    infinite, long runs of one token, an n-gram as long as the history."""
    print("case: special values", flush=True)
    rng = np.random.default_rng(6)
    x = rng.standard_normal((8, 500)).astype(np.float32)
    x[:, :6] = [np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-45]
    h = np.tile(np.arange(6), (8, 1)).repeat(20, 1)
    h[4:] = 7
    run(hip, x, "values", hist=h, hist_len=np.array([120, 120, 60, 119, 120, 3, 1, 120]),
        repeat=np.array([2, 0.5, 1, 3e38, 1.3, 1.1, 2, np.inf], np.float32),
        frequency=np.array([0, -1, 1e30, np.inf, 0.1, 0.2, 0, 1], np.float32),
        presence=np.array([0, 1, -1e38, 0, 0, np.inf, 1, -1], np.float32),
        ngram=np.array([120, 121, 60, 1, 2, 3, 2, 2 ** 31 - 1]), prompt_len=np.array([0, 500, -3, 60, 119, 1, 0, 2]))


def test_bias_starts_out_of_range(hip):
    """Starts that lie outside the list, or run backwards, give no bias."""
    print("case: bias starts", flush=True)
    x = np.random.default_rng(7).standard_normal((6, 50)).astype(np.float32)
    run(hip, x, "starts", bias_start=np.array([-1, 2, 1, 5, 7, 6, 3]), bias_id=np.arange(6), bias=np.full(6, 9.0, np.float32))


def test_many_rows(hip):
    """Rows past 256 and the most histories at once."""
    print("case: many rows", flush=True)
    rng = np.random.default_rng(8)
    x = rng.standard_normal((700, 4500)).astype(np.float32)
    run(hip, x, "rows", **everything(rng, 700, 4500, 90, 5, 700))


def test_rows_of_many_workgroups(hip):
    """Rows of several workgroups' tokens, many at once and again and again over
    one work: each gives its own largest, wherever it lies."""
    print("case: many workgroups", flush=True)
    rng = np.random.default_rng(10)
    rows, vocab = 150, 70000
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    mem = Mem(hip, 1 << 25)
    c = Call(hip, mem, x, out=False)
    for i in range(20):
        at = rng.integers(0, vocab, rows)
        x[np.arange(rows), at] = 10 + i
        mem.write(c.x, x)
        for _ in range(3):
            c.launch()
        c.check((None, at.astype(np.int32), np.full(rows, 10 + i, np.float32)), i)


@pytest.mark.parametrize("hist", [4095, 4096, 4097, 9000])
def test_long_histories(hip, hist):
    """Histories around what a workgroup's threads hold at once, and past it; n-grams over the edges."""
    print(f"case: history {hist}", flush=True)
    rng = np.random.default_rng(hist)
    for vocab in (30, 3000, 20000):
        x = (3 * rng.standard_normal((4, vocab))).astype(np.float32)
        h = rng.integers(0, min(vocab, 40), (4, hist))
        h[1, 1020:1030] = h[1, hist - 10:]
        h[2, 4090:4100] = h[2, hist - 10:][:len(h[2, 4090:4100])]
        run(hip, x, vocab, hist=h, hist_len=np.array([hist, hist, hist, hist - 1]), ngram=np.array([2, 8, 6, 3]),
            prompt_len=np.array([0, 1024, 4096, 5]), frequency=np.full(4, 0.01, np.float32))


def test_captured_and_replayed(hip):
    """Replays of a captured call give what an eager one gives, with the inputs
    of the moment; a call without rows leaves all as it is."""
    print("case: captured", flush=True)
    rng = np.random.default_rng(9)
    mem = Mem(hip, 1 << 24)
    xs = [rng.standard_normal((5, 9000)).astype(np.float32) for _ in range(3)]
    kw = everything(rng, 5, 9000, 100, 20, 2)
    c = Call(hip, mem, xs[0], **kw)
    c.a.rows = 0
    c.launch()
    assert np.all(c.results()[1] == 55)
    c.a.rows = 5
    assert hip.backend_graph_replay(1, 8, 8, 8) == 0
    hip.backend_graph_begin_capture(1)
    c.launch()
    hip.backend_graph_end_capture(1, 8, 8, 8)
    for i in (0, 2, 1, 1, 0):
        mem.write(c.x, xs[i])
        mem.write(c.out, np.zeros((5, 9000), np.float32))
        assert hip.backend_graph_replay(1, 8, 8, 8) == 1
        c.check(ref.process(xs[i], **kw), i)
        c.launch()
        c.check(ref.process(xs[i], **kw), i)


def test_the_most_rows(hip):
    print("case: most rows", flush=True)
    rng = np.random.default_rng(11)
    x = rng.standard_normal((65535, 33)).astype(np.float32)
    h = rng.integers(0, 33, (65535, 4))
    run(hip, x, "rows", hist=h, hist_len=rng.integers(0, 5, 65535), repeat=np.full(65535, 1.5, np.float32),
        mask=rng.integers(0, 2 ** 32, (65535, 2), dtype=np.uint32))


def test_bias_starts_far_out_of_range(hip):
    """Starts whose sum with a thread's number passes 2^31, ends before them, the
    whole list, and lists longer than a workgroup has threads: as the header says,
    starts below 0 or past the list, and those that run backwards, give no bias."""
    print("case: bias starts, far", flush=True)
    rng = np.random.default_rng(12)
    top = 2 ** 31 - 1
    for vocab, n in ((50, 6), (9000, 1500)):
        start = np.array([top, 0, top - 5, 2, top - 254, 1, top - 510, n, top, top - 511, -2 ** 31, 3, 0, n, top, n - 1, n])
        x = rng.standard_normal((len(start) - 1, vocab)).astype(np.float32)
        run(hip, x, ("starts", vocab), bias_start=start, bias_id=rng.integers(-3, vocab + 3, n), bias=rng.standard_normal(n).astype(np.float32))


@pytest.mark.parametrize("vocab", [300, 9000])
def test_history_that_ends_with_its_last_token(hip, vocab):
    """Histories that start inside their rows, the last row's last token at the end of
    the memory: only what hist_len counts is read, so the results are the tokens' alone."""
    print(f"case: history at the end {vocab}", flush=True)
    rng = np.random.default_rng(13)
    rows, ld, off = 5, 2500, 1700
    mem = Mem(hip, 1 << 22)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    full = rng.integers(0, vocab, (rows, ld)).astype(np.int32)
    full[:, off + 300:off + 310] = full[:, -10:]
    kw = dict(hist=full[:, off:], hist_len=np.full(rows, ld - off), repeat=np.full(rows, 1.3, np.float32),
              frequency=np.full(rows, 0.25, np.float32), ngram=np.full(rows, 3))
    at = mem.end - full.nbytes
    mem.write(at, full)
    c = Call(hip, mem, x, **kw)
    c.a.hist, c.a.ld_hist = at + 4 * off, ld
    want = ref.process(x, **kw)
    c.launch()
    c.check(want, vocab)


def test_overlapping_result_is_refused(hip):
    """out among the logits' rows without being them; beside them in one array it is fine."""
    print("case: overlap", flush=True)
    import subprocess
    import sys
    prog = (f"import sys; sys.path.insert(0, {cb.PKG_DIR!r}); import ctypes as C, ctbind as cb; L = cb.hip(); L.backend_init(0); "
            "l = cb.BackendLogits(logits=1 << 20, out=(1 << 20) + 400, ld=101, ld_out=150, rows=3, vocab=101); "
            "L.backend_logits(C.byref(l)); print('returned')")
    r = subprocess.run([sys.executable, "-c", prog], capture_output=True, text=True, timeout=100)
    assert r.returncode == 1 and "out overlaps the logits" in r.stderr and "returned" not in r.stdout, r.stderr
    rng = np.random.default_rng(14)
    x = rng.standard_normal((3, 202)).astype(np.float32)
    mem = Mem(hip, 1 << 20)
    at, ids = mem.put(x), mem.put(np.zeros(3, np.int32))
    a = cb.BackendLogits(logits=at, out=at + 404, ld=202, ld_out=202, rows=3, vocab=101, id=ids)
    hip.backend_logits(C.byref(a))
    assert np.array_equal(mem.get(at, (3, 202), np.float32), np.concatenate([x[:, :101]] * 2, 1))
    assert np.array_equal(mem.get(ids, (3,), np.int32), x[:, :101].argmax(1))
