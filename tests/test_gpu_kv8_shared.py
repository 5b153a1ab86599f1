"""Attention over the paged 8-bit cache of sequences that share their first
pages, on the device against the 64-bit model (kv8_ref.py) — needs an MI355X.

The result is that of attention through every sequence's own table, within
kv8_ref.tolerance of it.
"""
import ctypes as C

import numpy as np
import pytest

import ctbind as cb
import kv8_ref as ref
from test_gpu_kv8 import check_rows, starts, values

pytestmark = pytest.mark.gpu


def entries(P, kv, D, seqs):
    """Table entries with which a call without max_len could read so many codes
    that common tokens are taken apart (the launch goes by the sizes alone)."""
    return int(1.05 * 192 * 2 ** 20 / (seqs * kv * 2 * D * P)) + 2


def is_apart(d, a):
    for name in ("ctk_kv8_attn_shared_need", "ctk_kv8_attn_need"):
        f = getattr(d.hip, name)
        f.argtypes, f.restype = [C.c_void_p, C.c_void_p], C.c_size_t
    return d.hip.ctk_kv8_attn_shared_need(d.h, C.byref(a)) != d.hip.ctk_kv8_attn_need(d.h, C.byref(a))


def family(hip, rng, P, kv, D, groups, layers=1, extra=1 << 25, junk=True, rows=0):
    """A cache of `groups`, each (common tokens, [a sequence's tokens in all]),
    whose sequences take turns; the pages of the common tokens are shared, the
    last one of them too where no sequence goes on past it.  What is behind the
    last tokens is NaN codes and large values.  rows: those of a call, if fewer
    than the sequences."""
    turn = [(g, i) for i in range(max(len(m) for _, m in groups)) for g, (_, m) in enumerate(groups) if i < len(m)]
    lens = [groups[g][1][i] for g, i in turn]
    width = max(max(-(-n // P) for n in lens) + 1, entries(P, kv, D, min(len(lens), rows or len(lens))))
    common = [(c // P if any(n > c for n in m) else -(-c // P)) for c, m in groups]
    used = sum(common) + sum(max(0, -(-n // P) - common[g]) for n, (g, _) in zip(lens, turn))
    d = ref.Dev(hip, layers, used + 3, P, kv, D, len(lens), width, extra)
    m = d.model
    bad = np.array([0x7F, 0xFF, 0x7E, 0xFE], np.uint8) if junk else np.zeros(1, np.uint8)
    m.k[:], m.v[:] = rng.choice(bad, m.k.shape), rng.choice(bad, m.v.shape)
    m.ks[:], m.vs[:] = 2.0 ** 5, 2.0 ** 5
    order = [int(p) for p in rng.permutation(used + 3)[:used]]
    first = [[order.pop() for _ in range(c)] for c in common]
    for s, (n, (g, _)) in enumerate(zip(lens, turn)):
        m.len[s] = n
        for j in range(-(-n // P)):
            p = first[g][j] if j < common[g] else order.pop()
            m.table[s, j] = p
            m.refs[p] += 1
            t = min(P, n - j * P)
            e = rng.integers(-9, -5, (2, layers, kv))
            m.k[:, p, :, :t] = ref.to_codes(rng.standard_normal((layers, kv, t, D)) / 2.0 ** e[0][..., None, None])
            m.v[:, p, :, :t] = ref.to_codes(rng.standard_normal((layers, kv, t, D)) / 2.0 ** e[1][..., None, None])
            m.ks[:, p], m.vs[:, p] = 2.0 ** e[0], 2.0 ** e[1]
    d.push()
    return d, lens, [g for g, _ in turn]


def model_share(m):
    """backend_kv8_share's rule."""
    seqs, pages, P = m.dims[5], m.dims[1], m.P
    key = [int(m.table[s, 0]) if m.len[s] > 0 and 0 <= m.table[s, 0] < pages else -1 - s for s in range(seqs)]
    lead = [key.index(k) for k in key]
    tokens = []
    for s in range(seqs):
        mine = [i for i in range(seqs) if lead[i] == lead[s]]
        best = 0
        if len(mine) > 1:
            best = 10 ** 9
            for i in mine:
                used = -(-int(m.len[i]) // P)
                same = 0
                while same < used and m.table[i, same] == m.table[lead[s], same]:
                    same += 1
                best = min(best, same * P, int(m.len[i]))
        tokens.append(best)
    return np.array([lead, tokens], np.int32)


def found(d):
    """What backend_kv8_share writes, after a comparison with the rule."""
    seqs = d.model.dims[5]
    p = d.ints(np.full(2 * seqs + 1, 55))
    d.hip.backend_kv8_share(d.h, p)
    got = d.get(p, (2 * seqs + 1,), np.int32)
    assert got[-1] == 55
    want = model_share(d.model)
    assert np.array_equal(got[:-1].reshape(2, seqs), want), (got, want)
    return p, want


def attend(d, layer, q, heads, share, rows, causal=True, bf16=False, pad=0, off=0, max_rows=None, max_len=0, scale=None, apart=True):
    n, D, at = q.shape[0], q.shape[2], d.at
    ld, size = heads * D + pad, 2 if bf16 else 4
    flat = np.full(off + n * ld + 8, 77.0, np.float32)
    flat[off:off + n * ld].reshape(n, ld)[:, :heads * D] = q.reshape(n, -1)
    ofl = np.full(flat.shape, 55.0, np.float32)
    qp, op = d.put(ref.bf16_bits(flat) if bf16 else flat), d.put(ref.bf16_bits(ofl) if bf16 else ofl)
    a = cb.BackendKv8Attn(out=op + off * size, q=qp + off * size, ld_out=ld, ld_q=ld, bf16=int(bf16), heads=heads,
                          scale=scale or D ** -0.5, causal=int(causal), rows=d.ints(rows), n_rows=n,
                          max_rows=max_rows or max(1, int(np.diff(rows).max())), max_len=max_len)
    assert apart is None or is_apart(d, a) == apart
    w = d.hip.backend_kv8_attn_shared_work(d.h, C.byref(a))
    work = d.put(np.full(w + 64, np.nan, np.float32))
    a.work = work
    d.hip.backend_kv8_attn_shared(d.h, layer, C.byref(a), share)
    got = d.get(op, flat.shape, np.uint16 if bf16 else np.float32)
    got = ref.bf16_value(got) if bf16 else got
    assert np.isnan(d.get(work + 4 * w, (64,), np.float32)).all(), "past the work"
    d.at = at
    body = got[off:off + n * ld].reshape(n, ld)
    assert np.all(got[:off] == 55.0) and np.all(got[off + n * ld:] == 55.0) and np.all(body[:, heads * D:] == 55.0)
    return body[:, :heads * D].reshape(n, heads, D).copy()


def run(hip, rng, P, kv, group, D, groups, n, what, layer=0, layers=1, causal=True, bf16=False, behind=0, share=None, apart=True,
        **kw):
    total = sum(len(m) for _, m in groups)
    rows = total if isinstance(n, int) else sum(min(x, y) for x, y in zip(n, [max(m) for _, m in groups for _ in m]))
    d, lens, of = family(hip, rng, P, kv, D, groups, layers, rows=rows)
    n = [n] * len(lens) if isinstance(n, int) else n
    n = [min(x, y) for x, y in zip(n, lens)]
    rows = starts(n)
    q = values(rng, int(rows[-1]) + behind, kv * group, D)
    p = found(d)[0] if share is None else d.ints(share(d, lens, of))
    want = d.model.attend(layer, q, kv * group, kw.get("scale") or D ** -0.5, causal, 0, 0, rows, len(q), kw.get("max_len"))
    got = attend(d, layer, q, kv * group, p, rows, causal, bf16, apart=apart, **kw)
    check_rows(got, *want, bf16, what)
    if "max_len" not in kw:                   # and where so few tokens are not taken apart
        got = attend(d, layer, q, kv * group, p, rows, causal, bf16, apart=None, max_len=max(lens), **kw)
        check_rows(got, *want, bf16, (what, "short"))
    return d, q, got


SHAPES = [  # P, kv, group, D
    (16, 1, 1, 64), (64, 2, 1, 128), (32, 1, 4, 128), (128, 3, 3, 64), (16, 2, 8, 128), (64, 1, 16, 64), (32, 2, 5, 64)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", SHAPES)
def test_single_tokens(hip, P, kv, group, D, bf16):
    """Groups of every size, in turn with sequences that share nothing, around the edges of pages and tiles."""
    print(f"case: shared tokens P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    rng = np.random.default_rng(P + kv + group)
    run(hip, rng, P, kv, group, D, [(300, [301, 333, 420, 520, 364]), (128, [129, 130]), (0, [77]), (260, [260 + 3 * i + 1 for i in range(18)]),
                                    (0, [1, 2])], 1, "tokens", layer=1, layers=2, bf16=bf16, behind=2)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", SHAPES)
def test_hypotheses_of_one_clip(hip, P, kv, group, D, bf16):
    """All tokens are common, the last page partly filled, every row sees all of them."""
    print(f"case: shared clip P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    rng = np.random.default_rng(P + kv + group + 1)
    groups = [(c, [c] * k) for c, k in ((376, 5), (1, 3), (33, 2), (129, 4), (31, 1))]
    run(hip, rng, P, kv, group, D, groups, 1, "clip", causal=False, bf16=bf16, behind=1)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", SHAPES)
def test_several_rows(hip, P, kv, group, D, bf16):
    """Drafts and whole pieces behind a common text; sequences without rows."""
    print(f"case: shared rows P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    rng = np.random.default_rng(P + kv + group + 2)
    run(hip, rng, P, kv, group, D, [(256, [300, 290, 270, 330]), (384, [450, 400, 390]), (0, [20, 40])],
        [7, 3, 1, 4, 0, 40, 2, 6, 9], "rows", bf16=bf16, behind=3, apart=group == 1)
    few = 64 // group                         # rows of a sequence that still count as few
    run(hip, rng, P, kv, group, D, [(256, [300, 290, 270, 330]), (384, [450, 400, 390]), (0, [20, 40])],
        [min(few, x) for x in (7, 3, 1, 4, 0, 40, 2, 6, 9)], "fewer rows", bf16=bf16, behind=3)
    run(hip, rng, P, kv, group, D, [(256, [300, 290, 270])], [40, 30, 14], "pieces", bf16=bf16, apart=group == 1)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", [(16, 2, 4, 64), (64, 8, 4, 128), (128, 1, 8, 128), (64, 4, 1, 64)])
def test_many_sequences(hip, P, kv, group, D, bf16):
    """A group whose rows fill many tiles, over a text that is split."""
    print(f"case: shared, many P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    rng = np.random.default_rng(P + 3)
    run(hip, rng, P, kv, group, D, [(1500, [1501 + 7 * i for i in range(37)]), (640, [700] * 3)], 1, "many", bf16=bf16)
    run(hip, rng, P, kv, group, D, [(1024, [1024 + 5 + i % 9 for i in range(40)])], [1 + i % 5 for i in range(40)], "drafts", bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_all_sequences_of_a_cache(hip, bf16):
    """256 sequences: one group, 128 groups of two, none."""
    print(f"case: shared, 256 sequences bf16={bf16}", flush=True)
    rng = np.random.default_rng(4)
    run(hip, rng, 16, 2, 2, 64, [(96, [97 + i % 20 for i in range(256)])], 1, "one group", bf16=bf16)
    run(hip, rng, 16, 1, 3, 64, [(48, [50, 61]) for _ in range(128)], 1, "pairs", bf16=bf16)
    run(hip, rng, 16, 1, 1, 64, [(0, [20 + i]) for i in range(256)], 1, "alone", bf16=bf16)


def short(hip, rng, P, kv, group, D, groups, n, what, bf16, max_len=None, share=None, zero=()):
    """A call that is small enough for one workgroup a group, every row seeing all tokens."""
    d, lens, of = family(hip, rng, P, kv, D, groups, rows=1)
    assert len(lens) * kv > 512
    for s in zero:
        d.model.len[s] = 0
    d.push()
    n = [min(x, max(y, 1)) for x, y in zip([n] * len(lens) if isinstance(n, int) else n, lens)]
    rows = starts(n)
    q = values(rng, int(rows[-1]) + 2, kv * group, D)
    p = found(d)[0] if share is None else d.ints(share(d))
    max_len = max_len or max(lens)
    want = d.model.attend(0, q, kv * group, D ** -0.5, False, 0, 0, rows, len(q), max_len)
    for pad, off in ((0, 0), (5, 3)):
        got = attend(d, 0, q, kv * group, p, rows, False, bf16, max_len=max_len, apart=False, pad=pad, off=off)
        check_rows(got, *want, bf16, what)
    return d, rows, q, p, max_len


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", [(16, 8, 1, 128), (64, 8, 1, 64), (32, 4, 4, 128), (16, 3, 2, 64), (128, 16, 16, 64)])
def test_whole_groups(hip, P, kv, group, D, bf16):
    """Many clips' hypotheses in one launch; beside them groups with tokens of
    their own, of too many rows for a tile, and sequences alone, empty or without rows."""
    print(f"case: whole groups P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    rng = np.random.default_rng(P + kv + 7)
    each = max(1, 16 // group)
    groups = [(c, [c] * k) for c, k in ((376, 5), (1, 3), (33, 2), (129, 4), (31, 1), (300, each), (64, each + 1), (200, 2))]
    groups += [(128, [130, 129, 140]), (256, [256, 256, 300]), (0, [77])] + [(40 + i, [40 + i] * (1 + i % 4)) for i in range(12)]
    groups += [(50, [50, 50])] * max(0, (514 // kv - sum(len(m) for _, m in groups) + 3) // 2)
    seqs = sum(len(m) for _, m in groups)
    short(hip, rng, P, kv, group, D, groups, 1, "tokens", bf16)
    short(hip, rng, P, kv, group, D, groups, 1, "capped", bf16, max_len=100)
    short(hip, rng, P, kv, group, D, groups, 1, "empty", bf16, zero=range(0, seqs, 3))
    most = [int(x) for x in rng.integers(0, 16 // group + 1, seqs)]
    short(hip, rng, P, kv, group, D, groups, most, "rows", bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_whole_groups_of_a_caller(hip, bf16):
    """Fewer common tokens than there are, leaders out of range or without tokens."""
    print(f"case: whole groups, given bf16={bf16}", flush=True)
    groups = [(96, [96] * 4)] * 20

    def given(change):
        def make(d):
            s = model_share(d.model)
            change(s)
            return s
        return make

    def tokens(t):
        def change(s):
            s[1, ::2] = t
        return change

    def leaders(l):
        def change(s):
            s[0, 3::4] = l
        return change
    for change in (tokens(95), tokens(0), tokens(-1), tokens(2 ** 31 - 1), leaders(-1), leaders(40), leaders(2 ** 31 - 1), leaders(13),
                   leaders(-2 ** 31)):
        short(hip, np.random.default_rng(12), 32, 8, 2, 64, groups, 1, "given", bf16, share=given(change))


@pytest.mark.parametrize("bf16", [False, True])
def test_whole_groups_bad_pages(hip, bf16):
    """Missing pages, NaN in K, V and q; rows out of range and more than max_rows."""
    print(f"case: whole groups, bad pages bf16={bf16}", flush=True)
    rng = np.random.default_rng(13)
    d, rows, q, p, max_len = short(hip, rng, 16, 16, 1, 64, [(200, [200] * 5), (90, [90] * 3)] * 6, 1, "fine", bf16)
    m, seqs = d.model, len(rows) - 1
    first = m.table[:, 0].copy()
    for lead in range(seqs):
        mine = np.flatnonzero(first == first[lead])
        if mine[0] == lead and lead % 2:
            m.table[mine, 2] = 10 ** 6
        if mine[0] == lead and lead % 3 == 0:
            m.v[0, m.table[lead, 1], 2, 7, 9] = 0x7F
            m.k[0, m.table[lead, 3], 5, 3, 1] = 0xFF
    d.push()
    q[1, 3, 5], q[4, 0, 0] = np.inf, np.nan
    odd = rows.copy()
    odd[5:8] = [9, 4, 60]
    for r in (rows, odd):
        want = m.attend(0, q, 16, 0.125, False, 0, 0, r, len(q), max_len)
        got = attend(d, 0, q, 16, found(d)[0], r, False, bf16, max_rows=16, max_len=max_len, apart=False)
        # odd: row 8 is both the fifth row of sequence 4 (rows 4 .. 8) and sequence 8's
        # own (8 .. 8), so either's result may stand there
        one = np.array([sum(a <= i < b for a, b in zip(r, r[1:]) if 0 <= a and b <= len(q)) < 2 for i in range(len(q))])
        assert list(np.flatnonzero(~one)) == ([8] if r is odd else [])
        check_rows(got[one], *(x[one] for x in want), bf16, r.tolist())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kw", [dict(max_len=200, apart=False), dict(max_len=33, apart=False), dict(pad=3, off=5), dict(pad=8, off=8),
                                dict(scale=3.0), dict(max_len=10 ** 9)])
def test_options(hip, kw, bf16):
    print(f"case: shared {kw} bf16={bf16}", flush=True)
    rng = np.random.default_rng(5)
    for causal in (True, False):
        run(hip, rng, 32, 2, 2, 64, [(256, [300, 290, 270, 260]), (96, [100, 130])], 1, "options", causal=causal, bf16=bf16, **kw)


@pytest.mark.parametrize("bf16,common,causal", [(False, 1100, True), (True, 700, False)])
def test_tokens_past_max_len(hip, bf16, common, causal):
    """Sequences that hold more than max_len tokens: the common ones pass it, or the others."""
    print(f"case: shared, max_len bf16={bf16}", flush=True)
    run(hip, np.random.default_rng(11), 32, 8, 1, 128, [(common, [1101 + i % 7 for i in range(112)])], 1, common, causal=causal,
        bf16=bf16, max_len=970)


@pytest.mark.parametrize("bf16", [False, True])
def test_a_callers_own_groups(hip, bf16):
    """Fewer common tokens than there are, of any number; more than some rows
    see; leaders out of range, that do not lead themselves, or have negative
    tokens: the result stays that of every sequence's own table."""
    print(f"case: shared, own groups bf16={bf16}", flush=True)
    rng = np.random.default_rng(6)
    groups = [(256, [300, 290, 257, 260]), (192, [200, 210, 193])]

    def given(tokens, lead=None):
        def make(d, lens, of):
            s = model_share(d.model)
            s[1] = np.where(s[1] > 0, tokens, 0)
            for i, l in (lead or {}).items():
                s[0, i] = l
            return s
        return make

    for tokens in (1, 31, 33, 100, 191, -5, -2 ** 31):
        run(hip, rng, 16, 2, 4, 64, groups, 1, tokens, bf16=bf16, share=given(tokens))
    for lead in ({1: -1}, {2: 7}, {2: 2 ** 31 - 1}, {2: 3}, {0: 1, 1: 0}, {0: -2 ** 31}):
        run(hip, rng, 16, 2, 4, 64, groups, 1, lead, bf16=bf16, share=given(150, lead))
    # rows inside the common tokens: they see a part of them
    run(hip, rng, 32, 2, 2, 64, [(256, [256] * 5)], [1, 30, 2, 32, 31], "rows within", bf16=bf16)
    run(hip, rng, 32, 2, 2, 64, [(256, [256] * 5)], [1, 30, 2, 100, 256], "rows within", bf16=bf16, apart=False)
    run(hip, rng, 32, 2, 2, 64, [(256, [256] * 5)], 1, "last tokens", bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_bad_pages_lengths_and_rows(hip, bf16):
    """Missing pages in the common text and past it, NaN in K, V and q, rows out
    of range, more rows than tokens, empty sequences."""
    print(f"case: shared, bad pages bf16={bf16}", flush=True)
    rng = np.random.default_rng(7)
    d, lens, of = family(hip, rng, 16, 2, 64, [(256, [300, 290, 270, 280, 261]), (128, [140, 150, 129])])
    m = d.model
    for s in [i for i, g in enumerate(of) if g == 0]:
        m.table[s, [3, 9]] = [-1, 2 ** 31 - 1]
    m.table[0, 17] = 10 ** 6
    m.v[0, m.table[0, 5], 1, 7, 9] = 0x7F           # token 87 of the first group
    m.k[0, m.table[1, 2], 0, 3, 1] = 0xFF           # token 35 of the second
    m.v[0, m.table[4, 17], 0, 1, 2] = 0x7F          # token 273 of sequence 4
    m.len[7] = 0
    d.push()
    heads = 8
    for rows in (starts([1] * 8), np.array([0, 1, 2, 2, 1, 9, 7, 8, 8]), np.array([-3, 1, 2, 20, 3, 4, 5, 6, 6])):
        q = values(rng, 8, heads, 64)
        q[1, 3, 5], q[4, 0, 0] = np.inf, np.nan
        for causal in (True, False):
            p, _ = found(d)
            got = attend(d, 0, q, heads, p, rows.astype(np.int32), causal, bf16, max_rows=16)
            check_rows(got, *m.attend(0, q, heads, 0.125, causal, 0, 0, rows, 8), bf16, (rows.tolist(), causal))


@pytest.mark.parametrize("bf16", [False, True])
def test_sequences_that_name_the_same_rows(hip, bf16):
    """Row ranges that go back, so that the sequences' rows are many more than
    there are: a row is its first sequence's, or stays where that finds no room."""
    print(f"case: shared, the same rows bf16={bf16}", flush=True)
    rng = np.random.default_rng(14)
    d, lens, of = family(hip, rng, 16, 2, 64, [(256, [300 + i for i in range(120)]), (96, [130 + i for i in range(120)])], rows=4)
    for n, heads in ((8, 2), (4, 8)):
        rows = np.array([0, n] * (len(lens) // 2) + [0], np.int32)
        q = values(rng, n, heads, 64)
        first = np.array([0, n] + [n] * (len(lens) - 1), np.int32)
        want = d.model.attend(0, q, heads, 0.125, True, 0, 0, first, n)
        got = attend(d, 0, q, heads, found(d)[0], rows, True, bf16, max_rows=n)
        left = (got == 55.0).all(axis=2)
        ok = ~left.any(axis=1)
        check_rows(got[ok], *(x[ok] for x in want), bf16, n)


@pytest.mark.parametrize("bf16", [False, True])
def test_scales_far_apart(hip, bf16):
    """Value pages of very different sizes in the common text and past it."""
    print(f"case: shared, scales bf16={bf16}", flush=True)
    rng = np.random.default_rng(8)
    d, lens, of = family(hip, rng, 16, 2, 64, [(512, [530 + i for i in range(20)])], junk=False)
    for lo, hi in ((-20, 5), (-100, 100)):
        d.model.vs[:] = 2.0 ** rng.integers(lo, hi, d.model.vs.shape)
        d.model.ks[:] = 2.0 ** rng.integers(-10, -5, d.model.ks.shape)
        d.push()
        q = values(rng, 20, 4, 64)
        got = attend(d, 0, q, 4, found(d)[0], starts([1] * 20), bf16=bf16)
        check_rows(got, *d.model.attend(0, q, 4, 0.125, True, 0, 0, starts([1] * 20), 20), bf16, (lo, hi))


def test_share_of_tables(hip):
    """Forked, grown, trimmed and emptied sequences; pages out of range; tables
    alike past what the sequences hold."""
    print("case: share", flush=True)
    rng = np.random.default_rng(9)
    d = ref.Dev(hip, 1, 120, 16, 1, 64, 12, 80)
    d.reserve([100, 40] + [0] * 10)
    d.append(0, values(rng, 140, 1, 64), values(rng, 140, 1, 64))
    found(d)

    def fork(dst, src):
        hip.backend_kv8_fork(d.h, d.ints(dst), d.ints(src), len(dst))
        d.model.fork(dst, src)
        d.check_book()

    fork([2, 3, 4, 5], [0, 0, 1, 0])
    found(d)
    d.reserve([5, 1, 30, 0, 9, 1, 16, 3, 0, 0, 0, 0])
    d.append(0, *(values(rng, int(d.model.rows[-1]), 1, 64) for _ in range(2)))
    found(d)
    fork([8, 9], [2, 7])
    _, want = found(d)
    assert want[1, 0] == 96 and want[0, 8] == 0
    m = d.model
    m.table[10], m.len[10] = m.table[7], 2                    # one token common with 7 and 9
    m.table[11], m.len[11] = 500, 30                          # pages that are not there
    m.table[6, 1] = -1
    d.push()
    found(d)
    m.len[0] = 0
    m.len[7] = -4
    d.push()
    found(d)
    hip.backend_kv8_trim(d.h, 20, 3)
    m.trim(20, 3)
    found(d)


def test_share_of_long_tables(hip):
    """Tables that are alike for many entries, in more than one wavefront's step, and end a page apart."""
    print("case: share, long", flush=True)
    d = ref.Dev(hip, 1, 800, 16, 1, 64, 6, 700)
    m = d.model
    m.table[:] = np.arange(700)
    m.len[:] = [11200, 11195, 9000, 1024, 8200, 4000]
    m.table[4, 512] = 750
    d.push()
    assert found(d)[1][1, 0] == 1024
    m.len[3], m.len[5] = 0, 0
    d.push()
    assert found(d)[1][1, 0] == 8192


@pytest.mark.parametrize("bf16", [False, True])
def test_the_same_call_gives_the_same_bits(hip, bf16):
    """Over one work buffer, sized for a larger call, that the call before left
    full; captured and replayed with other queries and lengths between."""
    print(f"case: shared, same bits bf16={bf16}", flush=True)
    rng = np.random.default_rng(10)
    d, lens, of = family(hip, rng, 32, 2, 64, [(1024, [1100 + 3 * i for i in range(24)]), (320, [350] * 4)])
    n = len(lens)
    share = found(d)[0]
    qs = [values(rng, n, 8, 64) for _ in range(2)]
    put = lambda x: ref.bf16_bits(x) if bf16 else x.astype(np.float32)  # noqa: E731
    qp, op, rows = d.put(put(qs[0])), d.put(put(qs[0])), d.ints(starts([1] * n))
    big = cb.BackendKv8Attn(heads=8, scale=0.125, causal=1, n_rows=200, max_rows=9)
    work = d.put(np.full(hip.backend_kv8_attn_shared_work(d.h, C.byref(big)) + 64, np.nan, np.float32))
    a = cb.BackendKv8Attn(out=op, q=qp, ld_out=512, ld_q=512, bf16=int(bf16), heads=8, scale=0.125, causal=1, rows=rows,
                          n_rows=n, max_rows=1, work=work)
    assert is_apart(d, a)

    def result():
        return d.get(op, qs[0].shape, np.uint16 if bf16 else np.uint32)

    def eager(i):
        d.write(qp, put(qs[i]))
        hip.backend_kv8_attn_shared(d.h, 0, C.byref(a), share)
        return result()

    want = [eager(0), eager(1)]
    for i, w in enumerate(want):
        got = ref.bf16_value(w) if bf16 else w.view(np.float32)
        check_rows(got, *d.model.attend(0, qs[i], 8, 0.125, True, 0, 0, starts([1] * n), n), bf16, i)
    hip.backend_graph_begin_capture(2)
    hip.backend_kv8_attn_shared(d.h, 0, C.byref(a), share)
    hip.backend_graph_end_capture(2, 9, 9, 9)
    for i in (0, 1, 1, 0):
        d.write(qp, put(qs[i]))
        d.write(op, put(np.zeros(qs[0].shape)))
        assert hip.backend_graph_replay(2, 9, 9, 9) == 1
        replayed = np.array_equal(result(), want[i])
        assert replayed, i
        again = np.array_equal(eager(1 - i), want[1 - i])
        assert again, i


def long_texts(hip, rng, P, kv, D, lens, common, extra):
    """A cache of sequences whose tables name 211 pages again and again in an order of
    their own, after `common` tokens that all have; sequence 0 misses a page far behind."""
    pages, width = 211, -(-max(lens) // P) + 1
    d = ref.Dev(hip, 1, pages, P, kv, D, len(lens), width, extra)
    m = d.model
    m.k[:], m.v[:] = (ref.to_codes(64 * rng.standard_normal(m.k.shape).astype(np.float32)) for _ in range(2))
    m.ks[:], m.vs[:] = (2.0 ** rng.integers(-9, -5, m.ks.shape) for _ in range(2))
    m.table[:] = rng.integers(0, pages - 1, m.table.shape)
    m.table[:, :common // P] = m.table[0, :common // P]
    m.table[:, common // P] = rng.permutation(pages - 1)[:len(lens)]      # another one each
    m.table[0, (lens[0] - 100) // P] = -1
    m.len[:] = lens
    m.refs[:] = 1
    m.v[0, pages - 1, 1, 3, 5] = 0x7F
    d.push()
    return d


def attend_last(m, q, scale):
    """Cache.attend of a row a sequence, its last token, a page and a kv head at a time: for long texts."""
    _, pages, P, kv, D, seqs, _ = m.dims
    K, V = (ref.E4M3[x[0]] * s[0][..., None, None].astype(np.float64) for x, s in ((m.k, m.ks), (m.v, m.vs)))
    n, heads, _ = q.shape
    out, vmax, smax = np.zeros((n, heads, D)), np.zeros((n, heads, 1)), np.zeros((n, heads, 1))
    for s in range(seqs):
        page = m.table[s, :-(-int(m.len[s]) // P)]
        see = np.repeat((page >= 0) & (page < pages), P)[:int(m.len[s])]
        pg = np.where((page >= 0) & (page < pages), page, 0)
        for h in range(kv):
            k, v = (x[pg, h].reshape(-1, D)[:len(see)][see] for x in (K, V))
            at = slice(h * heads // kv, (h + 1) * heads // kv)
            qh = q[s, at].astype(np.float64)
            sc = qh @ k.T * scale
            smax[s, at, 0] = (np.abs(qh) @ np.abs(k).T).max(1) * scale
            w = np.exp(sc - sc.max(1, keepdims=True))
            out[s, at] = (w / w.sum(1, keepdims=True)) @ v
            vmax[s, at] = np.nanmax(np.abs(v))
    return out, vmax, smax


@pytest.mark.parametrize("P,kv,group,D,lens,common,least", [
    (64, 8, 1, 64, [15000 + 37 * i for i in range(20)], 0, 130),
    (128, 16, 2, 64, [9000 - 11 * i for i in range(24)], 384, 190),
    (16, 64, 1, 64, [36000, 35000, 36100, 35517], 0, 500),
    (32, 8, 4, 128, [15001 + 64 * i for i in range(20)], 96, 130),
    (64, 8, 8, 64, [70000 + 31 * i for i in range(8)], 69952, 130),
    (128, 8, 16, 64, [140001 + 50 * i for i in range(4)], 139904, 260)])
def test_chunks_of_many_pages(hip, P, kv, group, D, lens, common, least):
    """So many own or common tokens that a workgroup walks more than 128 steps of
    32, one that ends inside the last ones, with a page that is not there and a
    NaN behind the first of them."""
    print(f"case: shared, long chunks P={P} kv={kv} group={group} D={D} {lens[0]} x {len(lens)} {common}", flush=True)
    rng = np.random.default_rng(lens[0])
    n, heads = len(lens), kv * group
    d = long_texts(hip, rng, P, kv, D, lens, common, 1 << 24)
    m = d.model
    tiles = -(-n * group // 16) * (common // 32) if n * group <= 64 and common > 5000 else 0
    own = sum(-(-(x - common) // 32) for x in lens) if common < 5000 else 0
    assert max(tiles, own) / -(-512 // kv) > least        # steps of a chunk
    far = (min(lens) if not tiles else common) - 3 * P
    m.table[:2 if own else None, far // P] = m.dims[1] - 1
    d.push()
    q = values(rng, n, heads, D)
    p = found(d)[0]
    rows = starts([1] * n)
    want = attend_last(m, q, D ** -0.5)
    assert np.isnan(want[0]).any()
    for bf16 in (False, True):
        got = attend(d, 0, q, heads, p, rows, True, bf16)
        check_rows(got, *want, bf16, bf16)


@pytest.mark.parametrize("P,kv,group,D,lens,common", [
    (128, 8, 16, 64, [70001 + 50 * i for i in range(8)], 69888), (64, 8, 10, 128, [45000 + 7 * i for i in range(7)], 44992)])
def test_long_common_text_of_many_rows(hip, P, kv, group, D, lens, common):
    """The many-row kernel over common tokens whose chunks are longer than what it
    keeps places of at a time (32 iterations of 64), a page missing and a NaN near their end."""
    print(f"case: shared, long common text P={P} kv={kv} group={group} D={D} {lens[0]} x {len(lens)}", flush=True)
    rng = np.random.default_rng(lens[0])
    n, heads = len(lens), kv * group
    d = long_texts(hip, rng, P, kv, D, lens, common, 1 << 24)
    m = d.model
    assert n * group > 64 and (common // 32) / -(-128 // kv) > 64
    m.table[:, common // P - 3] = m.dims[1] - 1
    m.table[:, common // P - 9] = -1
    d.push()
    q, rows = values(rng, n, heads, D), starts([1] * n)
    p = found(d)[0]
    want = attend_last(m, q, D ** -0.5)
    assert np.isnan(want[0]).any()
    for bf16 in (False, True):
        check_rows(attend(d, 0, q, heads, p, rows, True, bf16), *want, bf16, bf16)
