"""The operators of a decode step run together as a server or a beam search uses
them: 4-bit maps, the paged 8-bit cache with common pages, logits, forks between
the steps — needs an MI355X."""
import ctypes as C

import numpy as np
import pytest

import ctbind as cb
import kv8_ref
import logits_ref
import w4_ref
from test_gpu_kv8 import check_rows
from test_gpu_kv8_shared import entries, is_apart
from test_gpu_w4 import check

pytestmark = pytest.mark.gpu

E, HEADS, KV, D, P, SEQS, FFN, VOCAB, HIST = 256, 4, 2, 64, 16, 6, 640, 1003, 96
QKV = (HEADS + 2 * KV) * D
PROMPTS = [40, 0, 0, 25, 0, 0]


class Step:
    """One layer and its head over a cache of six sequences."""

    def __init__(self, hip, rng, wide):
        self.hip = hip
        self.emb = rng.standard_normal((VOCAB, E)).astype(np.float32)
        self.bias = w4_ref.bf16_value(w4_ref.bf16_bits(rng.standard_normal(FFN).astype(np.float32)))
        width = entries(P, KV, D, SEQS) if wide else 12
        self.cache = d = kv8_ref.Dev(hip, 1, 60, P, KV, D, SEQS, width, 1 << 23)
        self.maps = {n: self.weight(rng, i, o, g) for n, i, o, g in (
            ("qkv", E, QKV, 64), ("out", HEADS * D, E, 128), ("up", E, FFN, 32), ("down", FFN, E, 64), ("head", E, VOCAB, 128))}
        n = sum(PROMPTS)
        f = lambda *s: d.put(np.zeros(s, np.float32))  # noqa: E731
        self.x, self.qkv, self.ctx, self.mid, self.logits = f(n, E), f(n, QKV), f(n, HEADS * D), f(n, FFN), f(SEQS, VOCAB)
        self.done = f(SEQS, VOCAB)
        self.share, self.add, self.id, self.score = d.ints([0] * 2 * SEQS), d.ints([1] * SEQS), d.ints([0] * SEQS), f(SEQS)
        self.hist, self.hist_len = d.put(np.zeros((SEQS, HIST), np.int32)), d.ints([0] * SEQS)
        self.biasp = d.put(w4_ref.bf16_bits(self.bias))
        self.pen = dict(repeat=np.full(SEQS, 1.2, np.float32), frequency=np.linspace(0, 1, SEQS).astype(np.float32),
                        ngram=np.array([0, 2, 3, 1, 0, 2], np.int32), prompt_len=np.array([40, 40, 40, 25, 25, 25], np.int32),
                        mask=rng.integers(0, 2 ** 32, (2, (VOCAB + 31) // 32), dtype=np.uint32),
                        mask_of=np.array([0, -1, 1, 2, -1, 0], np.int32))     # sequence 3 has none left
        self.penp = {k: d.put(v) for k, v in self.pen.items()}
        self.at = d.at

    def weight(self, rng, in_d, out_d, group):
        """A map in the cache's memory, and its values."""
        w, g = w4_ref.Weight(self.hip, self.cache, in_d, out_d, group, False), -(-in_d // group)
        codes, zeros = rng.integers(0, 16, (out_d, in_d)).astype(np.uint8), rng.integers(0, 16, (out_d, g)).astype(np.uint8)
        bits = w4_ref.bf16_bits((np.exp(0.5 * rng.standard_normal((out_d, g))) / np.sqrt(in_d) / 4).astype(np.float32))
        w.load(codes, bits, zeros)
        return w, w4_ref.values(codes, bits, zeros, group, False)

    def linear(self, name, y, x, rows, ld_y, ld_x, **kw):
        w = self.maps[name][0]
        a = cb.BackendW4Linear(y=y, x=x, ld_y=ld_y, ld_x=ld_x, rows=rows, **kw)
        self.hip.backend_linear_w4(w.h, C.byref(a))

    def attention(self, rows, max_rows):
        """The call, with work for the prompts, which is enough for the tokens after them."""
        d = self.cache
        a = cb.BackendKv8Attn(out=self.ctx, q=self.qkv, ld_out=HEADS * D, ld_q=QKV, heads=HEADS, scale=D ** -0.5, causal=1,
                              rows=d.c.rows, n_rows=sum(PROMPTS), max_rows=max(PROMPTS))
        if not hasattr(self, "work"):
            self.work = d.take(4 * self.hip.backend_kv8_attn_shared_work(d.h, C.byref(a)) + 16)
        a.n_rows, a.max_rows, a.work = rows, max_rows, self.work
        return a

    def layer(self, rows, max_rows):
        """Launches only: rows of x through the layer."""
        hip, d = self.hip, self.cache
        hip.backend_kv8_reserve(d.h, self.add)
        self.linear("qkv", self.qkv, self.x, rows, QKV, E)
        k, v = self.qkv + 4 * HEADS * D, self.qkv + 4 * (HEADS + KV) * D
        hip.backend_kv8_append(d.h, 0, k, v, QKV, 0, d.c.rows, rows)
        hip.backend_kv8_share(d.h, self.share)
        a = self.attention(rows, max_rows)
        hip.backend_kv8_attn_shared(d.h, 0, C.byref(a), self.share)

    def rest(self, rows):
        self.linear("out", self.x, self.ctx, rows, E, HEADS * D, act=cb.W4_ADD, scale=0.5)

    def ffn(self, rows):
        self.linear("up", self.mid, self.x, rows, FFN, E, act=cb.W4_SILU, bias=self.biasp)

    def down(self, rows):
        self.linear("down", self.x, self.mid, rows, E, FFN, act=cb.W4_ADD, scale=1.0)

    def pick(self):
        self.linear("head", self.logits, self.x, SEQS, VOCAB, E)
        a = cb.BackendLogits(logits=self.logits, out=self.done, ld=VOCAB, ld_out=VOCAB, rows=SEQS, vocab=VOCAB, id=self.id,
                             score=self.score, hist=self.hist, ld_hist=HIST, hist_len=self.hist_len, masks=2,
                             ld_mask=(VOCAB + 31) // 32, **self.penp)
        if not hasattr(self, "lwork"):
            self.lwork = self.cache.put(np.zeros(self.hip.backend_logits_work(C.byref(a)) + 4, np.float32))
        a.work = self.lwork
        self.hip.backend_logits(C.byref(a))

    def all(self):
        self.layer(SEQS, 1)
        self.rest(SEQS), self.ffn(SEQS), self.down(SEQS), self.pick()

    def get(self, p, *shape, dtype=np.float32):
        return self.cache.get(p, shape, dtype)

    def checked(self, rows, add):
        """The same with every operator's result held against the models, from the inputs it had."""
        d, m = self.cache, self.cache.model
        x = self.get(self.x, rows, E)
        self.layer(rows, max(add))
        m.reserve(add)
        qkv, ctx = self.get(self.qkv, rows, QKV), self.get(self.ctx, rows, HEADS * D)
        W = {n: w[1] for n, w in self.maps.items()}
        check(qkv, W["qkv"], x, False, "qkv")
        part = lambda a, n: qkv[:, a * D:(a + n) * D].reshape(rows, n, D)  # noqa: E731
        m.append(0, part(HEADS, KV), part(HEADS + KV, KV), m.rows, rows)
        d.check("append")
        check_rows(ctx.reshape(rows, HEADS, D), *m.attend(0, part(0, HEADS), HEADS, D ** -0.5, True, 0, 0, m.rows, rows, None), False,
                   "attention")
        self.rest(rows)
        h = self.get(self.x, rows, E)
        check(h, W["out"], ctx, False, "out", act=cb.W4_ADD, scale=0.5, y=x)
        self.ffn(rows)
        mid = self.get(self.mid, rows, FFN)
        check(mid, W["up"], h, False, "up", act=cb.W4_SILU, bias=self.bias)
        self.down(rows)
        y = self.get(self.x, rows, E)
        check(y, W["down"], mid, False, "down", act=cb.W4_ADD, scale=1.0, y=h)
        return y

    def checked_pick(self, y, said):
        self.pick()
        raw, ids = self.get(self.logits, SEQS, VOCAB), self.get(self.id, SEQS, dtype=np.int32)
        check(raw, self.maps["head"][1], y, False, "head")
        hist = np.zeros((SEQS, HIST), np.int32)
        for s, t in enumerate(said):
            hist[s, :len(t)] = t
        want = logits_ref.process(raw, hist=hist, hist_len=np.array([len(t) for t in said]), **self.pen)
        assert np.array_equal(self.get(self.done, SEQS, VOCAB), want[0])
        assert np.array_equal(ids, want[1]) and np.array_equal(self.get(self.score, SEQS), want[2])
        assert ids[3] == -1

    def tell(self, said):
        """The last tokens' embeddings and the histories, to the device."""
        d = self.cache
        hist = np.zeros((SEQS, HIST), np.int32)
        for s, t in enumerate(said):
            hist[s, :len(t)] = t
        d.write(self.hist, hist)
        d.write(self.hist_len, np.array([len(t) for t in said], np.int32))
        d.write(self.x, np.stack([self.emb[t[-1]] for t in said]))


def decode(hip, wide, mode):
    """What eight steps after two prompts choose and how their last logits look."""
    rng = np.random.default_rng(21)
    st = Step(hip, rng, wide)
    d, m = st.cache, st.cache.model
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in PROMPTS]
    d.write(st.x, np.concatenate([st.emb[p] for p in prompts if p]))
    d.write(st.add, np.array(PROMPTS, np.int32))
    st.checked(sum(PROMPTS), PROMPTS)
    d.write(st.add, np.ones(SEQS, np.int32))

    def fork(dst, src):
        hip.backend_kv8_fork(d.h, d.ints(dst), d.ints(src), len(dst))
        m.fork(dst, src)
        for a, b in zip(dst, src):
            said[a] = list(said[b])

    said = [list(p) for p in prompts]
    fork([1, 2, 4, 5], [0, 0, 3, 3])
    for s in range(SEQS):                     # each sequence goes on with a token of its own
        said[s].append(int(rng.integers(0, VOCAB)))
    assert is_apart(d, st.attention(SEQS, 1)) == wide
    tag, chosen = 3, []
    for i in range(8):
        st.tell(said)
        if mode == "checked":
            st.checked_pick(st.checked(SEQS, [1] * SEQS), said)
            share = st.get(st.share, 2, SEQS, dtype=np.int32)
            assert share[0].tolist() == [0, 0, 0, 3, 3, 3] and share[1, 0] >= 32 and share[1, 3] >= 16
        elif mode == "eager" or i == 0:
            st.all()
        elif not hip.backend_graph_replay(tag, 5, 5, SEQS):
            assert i == 1
            hip.backend_graph_begin_capture(tag)
            st.all()
            hip.backend_graph_end_capture(tag, 5, 5, SEQS)
        ids = st.get(st.id, SEQS, dtype=np.int32)
        chosen.append((ids.tolist(), st.get(st.done, SEQS, VOCAB).view(np.uint32).copy()))
        if mode != "checked":
            m.reserve([1] * SEQS)
        for s in range(SEQS):
            said[s].append(max(int(ids[s]), 0))
        if i == 4:                            # hypotheses 0 and 4 go on in place of 2 and 5
            fork([2, 5], [0, 4])
    assert hip.backend_kv8_status(d.h) == 0
    d.model.status = 0
    return chosen


@pytest.mark.parametrize("wide", [True, False])
def test_steps(hip, wide):
    """Prompts, forks, steps: each operator against its model; the same steps
    without looking in between, and captured and replayed, give the same bits."""
    print(f"case: decode steps wide={wide}", flush=True)
    want = decode(hip, wide, "checked")
    for mode in ("eager", "replayed"):
        got = decode(hip, wide, mode)
        for i, (a, b) in enumerate(zip(want, got)):
            assert a[0] == b[0] and np.array_equal(a[1], b[1]), (mode, i)


def test_two_threads(hip):
    """Two threads with a stream and memory each, at once: what each gets alone."""
    print("case: decode steps, two threads", flush=True)
    import threading
    alone, both = [decode(hip, wide, "eager") for wide in (True, False)], [None, None]

    def run(i):
        hip.backend_init(0)
        both[i] = [decode(hip, i == 0, "eager") for _ in range(3)]
        hip.backend_thread_cleanup()

    ts = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
    for one, three in zip(alone, both):
        for got in three:
            assert all(a[0] == b[0] and np.array_equal(a[1], b[1]) for a, b in zip(one, got))
