"""The paged 8-bit key/value cache on the device against its 64-bit model
(kv8_ref.py) — needs an MI355X.

Appends and page calls must give the model's codes, scales and tables
exactly; attention must be within kv8_ref.tolerance of the 64-bit result.
"""
import ctypes as C

import numpy as np
import pytest

import ctbind as cb
import kv8_ref as ref

pytestmark = pytest.mark.gpu


def values(rng, *shape):
    """Normal values whose size differs from row to row, representable in bf16."""
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1] + (1,)))
    return ref.bf16_value(ref.bf16_bits(x.astype(np.float32)))


def check_rows(got, want, vmax, smax, bf16, what):
    """Rows of no sequence untouched (55), the others within the tolerance, NaN where the model has NaN."""
    none = np.isnan(want).all(axis=(1, 2)) & (vmax == 0).all(axis=(1, 2))
    assert np.all(got[none] == 55.0), what
    w, g = want[~none], got[~none].astype(np.float64)
    assert np.array_equal(np.isnan(w), np.isnan(g)), what
    t = ref.tolerance(w, vmax[~none], smax[~none], bf16, w.shape[2])
    with np.errstate(invalid="ignore"):
        d = np.abs(g - w)
    bad = ~(d <= t) & ~np.isnan(w)
    assert not bad.any(), (what, float(np.nanmax(d / np.maximum(t, 1e-300))), np.argwhere(bad)[:4])


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("P,D,kv,bf16", [(16, 64, 1, False), (32, 64, 3, True), (64, 128, 2, False),
                                         (128, 128, 1, True), (16, 128, 8, True), (128, 64, 2, False)])
def test_append(hip, P, D, kv, bf16):
    """Prompts over several pages, then tokens one by one and a few at a time,
    in the second of two layers; the other layer and what lies behind a
    sequence's last token stay as they were."""
    print(f"case: append P={P} D={D} kv={kv} bf16={bf16}", flush=True)
    rng = np.random.default_rng(P + D + kv)
    d = ref.Dev(hip, 2, 40, P, kv, D, 5, 6)
    d.model.k[:] = rng.integers(0, 256, d.model.k.shape)
    d.model.v[:] = rng.integers(0, 256, d.model.v.shape)
    d.model.ks[:] = 2.0 ** rng.integers(-8, 3, d.model.ks.shape)
    d.push()
    for add in ([P, 1, 0, 2 * P + 3, P - 1], [1, 1, 1, 1, 1], [0, P, 0, 1, 2], [1, 0, 3, P + 1, 1], [1, 1, 1, 1, 1]):
        d.reserve(add)
        n = sum(add)
        k, v = values(rng, n, kv, D), values(rng, n, kv, D)
        d.append(1, k, v, bf16)
        d.check(add)


def test_append_growing_scale_and_special_values(hip):
    """Later tokens larger than a page's scale holds (its codes are rounded
    again), smaller ones, zeros, values at 448 scales, subnormals, the largest
    floats, infinities (held at 448 scales) and NaN."""
    print("case: append special values", flush=True)
    D, kv = 64, 2
    d = ref.Dev(hip, 1, 8, 16, kv, D, 3, 3)
    rng = np.random.default_rng(4)
    sizes = [1.0, 2.0 ** -120, 3.0, 2.0 ** 9, 448.0, 449.0, 1e-44, 0.0, 3e38, 1.0, 2.0 ** 20]
    for i, size in enumerate(sizes):
        d.reserve([1, 2 if i < 5 else 0, 0])
        n = 3 if i < 5 else 1
        k = (np.clip(rng.standard_normal((n, kv, D)), -1, 1) * size).astype(np.float32)
        v = (np.sign(k) * size).astype(np.float32)
        if i in (2, 6):
            k[0, 0, :6] = [np.inf, -np.inf, np.nan, -0.0, size, -size]
            v[0, 1, 5] = np.nan
        d.append(0, k, v)
        d.check((i, size))


def test_append_rounds_every_tie_to_even(hip):
    """All midpoints between neighbouring codes, and their neighbours in fp32."""
    print("case: append ties", flush=True)
    d = ref.Dev(hip, 1, 8, 32, 1, 128, 1, 4)
    mid = ref._MID.astype(np.float32)
    x = np.concatenate([mid, np.nextafter(mid, np.float32(1e9)), np.nextafter(mid, np.float32(0)), ref._POS])
    x = np.concatenate([x, -x]).astype(np.float32)
    n = -(-x.size // 127)
    k = np.zeros((n, 1, 128), np.float32)
    k[:, 0, 0] = 448.0                       # the scale is 1 on every page
    k[:, 0, 1:].reshape(-1)[:] = 0
    k[:, 0, 1:] = np.pad(x, (0, n * 127 - x.size)).reshape(n, 127)
    d.reserve([n])
    d.append(0, k, k * np.float32(2.0 ** -30))
    d.check()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pad,off", [(0, 1), (1, 0), (8, 0), (512, 8), (3, 5)])
def test_append_strided_rows(hip, bf16, pad, off):
    """Rows apart, as a fused projection leaves them, and off 16 bytes."""
    print(f"case: append pad={pad} off={off} bf16={bf16}", flush=True)
    rng = np.random.default_rng(9)
    d = ref.Dev(hip, 1, 8, 32, 2, 64, 2, 3)
    d.reserve([37, 5])
    d.append(0, values(rng, 42, 2, 64), values(rng, 42, 2, 64), bf16, pad=pad, off=off)
    d.check()


def test_append_skips_what_it_must_not_write(hip):
    """Pages outside the pool or shared, rows outside [0, n_rows), rows before
    the first token, lengths past the table row."""
    print("case: append bad pages and rows", flush=True)
    rng = np.random.default_rng(10)
    d = ref.Dev(hip, 1, 12, 16, 1, 64, 8, 2)
    m = d.model
    m.table[:] = [[0, 1], [2, 12], [-1, 3], [4, -7], [5, 6], [7, 8], [9, 10], [11, 2 ** 31 - 1]]
    m.refs[:12] = 1
    m.refs[6] = 2
    m.len[:] = [20, 32, 32, 20, 24, 3, 50, 20]
    d.push()
    rows = [0, 20, 52, 84, 104, 128, 136, 146, 150]      # sequence 5 has 8 rows for 3 tokens, 6 passes its table row
    n = 148                                              # the last sequence's rows pass the end
    d.append(0, values(rng, n, 1, 64), values(rng, n, 1, 64), rows=rows)
    d.check()
    d.append(0, values(rng, n, 1, 64), values(rng, n, 1, 64), rows=[-3, 20, 10, 10, 200, 3, 2 ** 31 - 1, -2 ** 31, 5])
    d.check()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def filled(hip, rng, P, kv, D, lens, layers=1, spare=3, extra=1 << 22):
    """A cache whose sequences hold lens tokens on shuffled pages; every other
    byte of the pools, behind the last tokens too, is a NaN code or large."""
    held = [-(-n // P) for n in lens]
    width, pages = max(max(held), 1) + 1, max(sum(held), 1) + spare
    d = ref.Dev(hip, layers, pages, P, kv, D, len(lens), width, extra)
    m = d.model
    m.k[:] = rng.choice(np.array([0x7F, 0xFF, 0x7E, 0xFE], np.uint8), m.k.shape)
    m.v[:] = rng.choice(np.array([0x7F, 0xFF, 0x7E, 0xFE], np.uint8), m.v.shape)
    m.ks[:] = 2.0 ** 5
    m.vs[:] = 2.0 ** 5
    order = list(rng.permutation(pages)[:sum(held)])
    for s, n in enumerate(lens):
        m.len[s] = n
        for j in range(held[s]):
            p = int(order.pop())
            m.table[s, j] = p
            m.refs[p] = 1
            t = min(P, n - j * P)
            e = rng.integers(-9, -5, (2, layers, kv))
            m.k[:, p, :, :t] = ref.to_codes(rng.standard_normal((layers, kv, t, D)) / 2.0 ** e[0][..., None, None])
            m.v[:, p, :, :t] = ref.to_codes(rng.standard_normal((layers, kv, t, D)) / 2.0 ** e[1][..., None, None])
            m.ks[:, p], m.vs[:, p] = 2.0 ** e[0], 2.0 ** e[1]
    d.push()
    return d


def starts(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def run_attn(hip, rng, P, kv, group, D, lens, n, what, layer=0, layers=1, bf16=False, behind=0, **kw):
    d = filled(hip, rng, P, kv, D, lens, layers, extra=1 << 24)
    rows = starts(n)
    total = int(rows[-1]) + behind
    q = values(rng, total, kv * group, D)
    got = d.attn(layer, q, kv * group, bf16=bf16, rows=rows, **kw)
    args = {k: kw[k] for k in ("causal", "window", "sinks") if k in kw}
    want = d.model.attend(layer, q, kv * group, kw.get("scale") or D ** -0.5, args.get("causal", True),
                          args.get("window", 0), args.get("sinks", 0), rows, total, kw.get("max_len"))
    check_rows(got, *want, bf16, what)
    return d, q, got


SHAPES = [  # P, kv, group, D
    (16, 1, 1, 64), (64, 2, 1, 128), (32, 1, 4, 128), (128, 3, 3, 64), (16, 2, 8, 128), (64, 1, 16, 64), (32, 2, 5, 64)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", SHAPES)
def test_decode(hip, P, kv, group, D, bf16):
    """One token of each sequence: lengths 1 to several chunks, around every
    tile and page edge; a sequence without a row; rows behind the last one."""
    print(f"case: decode P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 40, 63, 64, 65, 127, 129, 257, 511, 513, 1030]
    n = [1] * len(lens)
    n[8] = 0
    run_attn(hip, np.random.default_rng(P + kv + group), P, kv, group, D, lens, n, "decode", layer=1, layers=2,
             bf16=bf16, behind=2)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", SHAPES)
def test_several_rows(hip, P, kv, group, D, bf16):
    """A few new tokens on held ones, whole prompts, and none, together."""
    print(f"case: rows P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    lens = [3, 70, 33, 300, 5, 64]
    n = [3, 7, 33, 40, 0, 64]
    run_attn(hip, np.random.default_rng(P + kv + group), P, kv, group, D, lens, n, "rows", bf16=bf16, behind=3)


WIDE = [  # P, kv, group, D: launches of so many rows that a workgroup takes 64 or 128
    (16, 4, 8, 64), (64, 8, 4, 128), (128, 3, 16, 128), (32, 8, 5, 64)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("P,kv,group,D", WIDE)
def test_many_rows(hip, P, kv, group, D, bf16):
    """Prompts, pieces over held tokens and single tokens in one launch, enough
    of them for the tiles of many rows."""
    print(f"case: many rows P={P} kv={kv} group={group} D={D} bf16={bf16}", flush=True)
    total = 11000 // (kv * group) + 20
    n = [total // 2, total // 3, 1, 0, 2, 17]
    lens = [n[0], n[1] + 150, 90, 33, 2, 300]
    run_attn(hip, np.random.default_rng(P + kv + group), P, kv, group, D, lens, n, "many rows", layer=1, layers=2, bf16=bf16,
             behind=2, pad=0 if D == 64 else 3, off=0 if D == 64 else 5)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=50, sinks=3), dict(window=130, sinks=70), dict(causal=False),
                                dict(causal=False, max_len=75), dict(window=2 ** 31 - 1, sinks=1)])
def test_many_rows_masks(hip, kw, bf16):
    print(f"case: many rows {kw} bf16={bf16}", flush=True)
    rng = np.random.default_rng(41)
    run_attn(hip, rng, 16, 4, 8, 64, [160, 350, 1, 0], [160, 190, 1, 3], "masks", bf16=bf16, **kw)
    run_attn(hip, rng, 64, 8, 4, 128, [200, 310], [200, 160], "masks", bf16=bf16, **kw)


@pytest.mark.parametrize("bf16", [False, True])
def test_many_rows_over_a_long_text(hip, bf16):
    """Few tiles over many tokens: the keys are split and joined."""
    print(f"case: many rows, split bf16={bf16}", flush=True)
    run_attn(hip, np.random.default_rng(42), 32, 2, 16, 64, [2600, 700], [330, 30], "split", bf16=bf16)
    run_attn(hip, np.random.default_rng(43), 128, 1, 32, 128, [2111], [340], "split", bf16=bf16, window=1500, sinks=5)


@pytest.mark.parametrize("bf16", [False, True])
def test_many_rows_bad_pages_and_values(hip, bf16):
    """Missing pages, NaN in K, V and q, rows that see nothing, in the tiles of many rows."""
    print(f"case: many rows, bad pages bf16={bf16}", flush=True)
    rng = np.random.default_rng(44)
    d = filled(hip, rng, 32, 4, 64, [230, 200, 90], extra=1 << 24)
    m = d.model
    m.table[0, [0, 4]] = [-1, 2 ** 31 - 1]
    m.table[2] = -1
    m.v[0, m.table[0, 5], 2, 20, 7] = 0x7F          # token 180 of sequence 0
    m.v[0, m.table[1, 0], 1, 3, 9] = 0xFF           # token 3 of sequence 1
    m.k[0, m.table[1, 3], 3, 16, 0] = 0x7F          # token 112
    d.push()
    n = [200, 160, 40]
    q = values(rng, 400, 32, 64)
    q[220, 3, 5], q[221, 30, 0] = np.inf, np.nan
    for kw in (dict(), dict(window=45, sinks=2), dict(window=45, sinks=6)):
        got = d.attn(0, q, 32, rows=starts(n), bf16=bf16, **kw)
        want = m.attend(0, q, 32, 0.125, True, kw.get("window", 0), kw.get("sinks", 0), starts(n), 400)
        check_rows(got, *want, bf16, kw)
        assert np.all(got[360:] == 0.0)
        if not kw:
            assert np.isnan(got[150:200, 16:24, 7]).all() and np.isfinite(got[:149, :, 7]).all()


def test_many_rows_scales_far_apart(hip):
    print("case: many rows, scales", flush=True)
    rng = np.random.default_rng(45)
    d = filled(hip, rng, 16, 4, 64, [200, 150], extra=1 << 23)
    d.model.vs[:] = 2.0 ** rng.integers(-20, 5, d.model.vs.shape)
    d.model.ks[:] = 2.0 ** rng.integers(-10, -5, d.model.ks.shape)
    d.push()
    q = values(rng, 350, 32, 64)
    rows = starts([200, 150])
    got = d.attn(0, q, 32, rows=rows)
    check_rows(got, *d.model.attend(0, q, 32, 0.125, True, 0, 0, rows, 350), False, "scales")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_many_rows_queries_of_every_size(hip, D, bf16):
    """Rows that are zero, subnormal, tiny or not finite beside ordinary ones of
    the same tile: only those with an infinity or NaN are NaN, and no others."""
    print(f"case: many rows, queries D={D} bf16={bf16}", flush=True)
    rng = np.random.default_rng(52)
    d = filled(hip, rng, 32, 4, D, [200, 150], extra=1 << 24)
    q = values(rng, 350, 32, D)
    q[3, 5] = 0
    q[4, 6] = ref.bf16_value(ref.bf16_bits(q[4, 6] * np.float32(1e-39)))
    q[5] = ref.bf16_value(ref.bf16_bits(q[5] * np.float32(1e-30)))
    q[6, :, 1:] = 0
    q[20, 7, 1], q[21, 8, D - 1], q[349, 31, 0] = np.inf, -np.inf, np.nan
    rows = starts([200, 150])
    got = d.attn(0, q, 32, rows=rows, bf16=bf16)
    check_rows(got, *d.model.attend(0, q, 32, D ** -0.5, True, 0, 0, rows, 350), bf16, D)
    assert np.isnan(got).any(axis=2).sum() == 3


@pytest.mark.parametrize("bf16", [False, True])
def test_sixteen_query_heads_of_128(hip, bf16):
    """A tile full of one token's heads, by four and by eight wavefronts (64 KB of joined sums)."""
    print(f"case: group 16 of 128 bf16={bf16}", flush=True)
    rng = np.random.default_rng(46)
    run_attn(hip, rng, 64, 1, 16, 128, [700, 1, 130], [1, 1, 1], "eight wavefronts", max_len=700, bf16=bf16)
    run_attn(hip, rng, 64, 2, 16, 128, [40] * 140 + [700], [1] * 141, "four wavefronts", max_len=700, bf16=bf16)
    run_attn(hip, rng, 64, 1, 32, 128, [700, 33], [1, 1], "two tiles", bf16=bf16)


@pytest.mark.parametrize("n", [[1, 1, 1], [150, 180, 20]])
def test_the_same_call_gives_the_same_bits(hip, n):
    """Twice in a row, over one work buffer that the call before left full, and
    with a larger one's work for a smaller call."""
    print(f"case: same bits n={n}", flush=True)
    rng = np.random.default_rng(47)
    d = filled(hip, rng, 32, 4, 64, [900, 600, 1500], extra=1 << 24)
    q = values(rng, sum(n), 32, 64)
    rows, fl = d.ints(starts(n)), q.reshape(len(q), -1)
    qp, outs = d.put(fl), []
    big = cb.BackendKv8Attn(heads=32, scale=0.125, causal=1, n_rows=400, max_rows=400, max_len=1500)
    work = d.put(np.full(hip.backend_kv8_attn_work(d.h, C.byref(big)) + 64, np.nan, np.float32))
    for i in range(3):
        op = d.put(np.zeros_like(fl))
        a = cb.BackendKv8Attn(out=op, q=qp, ld_out=2048, ld_q=2048, heads=32, scale=0.125, causal=1, rows=rows, n_rows=len(q),
                              max_rows=max(n), max_len=1500, work=work)
        hip.backend_kv8_attn(d.h, 0, C.byref(a))
        outs.append(d.get(op, fl.shape, np.float32))
        assert np.array_equal(outs[0].view(np.uint32), outs[i].view(np.uint32)), i
    want = d.model.attend(0, q, 32, 0.125, True, 0, 0, starts(n), len(q))
    check_rows(outs[0].reshape(q.shape), *want, False, "larger work")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 4), (33, 64), (100, 33), (64, 500), (2000, 4),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
def test_window(hip, window, sinks, bf16):
    """Windows and first tokens around the tile and page edges, single rows and prompts."""
    print(f"case: window={window} sinks={sinks} bf16={bf16}", flush=True)
    rng = np.random.default_rng(window % 1000 + sinks % 1000)
    run_attn(hip, rng, 16, 2, 3, 64, [1, 40, 129, 300, 700], [1, 1, 1, 1, 1], "one row", window=window, sinks=sinks, bf16=bf16)
    run_attn(hip, rng, 32, 1, 2, 128, [1, 90, 200, 333], [1, 90, 30, 130], "prompt", window=window, sinks=sinks, bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_not_causal(hip, bf16):
    """Every row sees all tokens: encoder frames; a sequence of none gives zeros."""
    print(f"case: not causal bf16={bf16}", flush=True)
    rng = np.random.default_rng(3)
    _, _, got = run_attn(hip, rng, 32, 2, 1, 128, [376, 0, 1, 33], [1, 1, 1, 1], "one", causal=False, bf16=bf16)
    assert np.all(got[1] == 0.0)
    _, _, got = run_attn(hip, rng, 64, 1, 4, 64, [100, 0, 1, 700], [9, 3, 2, 40], "more", causal=False, bf16=bf16)
    assert np.all(got[9:12] == 0.0)


def test_max_len_hides_what_is_past_it(hip):
    print("case: max_len", flush=True)
    rng = np.random.default_rng(5)
    run_attn(hip, rng, 32, 1, 2, 64, [100, 40, 700], [1, 1, 1], "cut", causal=False, max_len=64)
    run_attn(hip, rng, 32, 1, 2, 64, [100, 40, 700], [1, 1, 1], "cut at an odd length", causal=False, max_len=83)


@pytest.mark.parametrize("pad,off", [(1, 1), (8, 0), (64, 8), (0, 3)])
@pytest.mark.parametrize("bf16", [False, True])
def test_strided_rows(hip, pad, off, bf16):
    print(f"case: strides pad={pad} off={off} bf16={bf16}", flush=True)
    run_attn(hip, np.random.default_rng(6), 32, 2, 2, 64, [40, 100], [1, 1], "one", pad=pad, off=off, bf16=bf16)
    run_attn(hip, np.random.default_rng(6), 32, 2, 2, 64, [40, 100], [40, 30], "more", pad=pad, off=off, bf16=bf16)


@pytest.mark.parametrize("n", [[1, 1, 1, 1], [30, 20, 64, 90]])
def test_pages_that_are_not_there(hip, n):
    """Table entries -1 or outside the pool hide their tokens; a row that sees
    none of its tokens gets zeros."""
    print(f"case: missing pages n={n}", flush=True)
    rng = np.random.default_rng(7)
    d = filled(hip, rng, 16, 1, 64, [30, 50, 64, 200])
    m = d.model
    m.table[0] = -1
    m.table[1, 2] = m.dims[1]
    m.table[2, :] = [2 ** 31 - 1, m.table[2, 1], -5, -2 ** 31] + [-1] * (m.dims[6] - 4)
    m.table[3, [0, 5, 12]] = -1
    d.push()
    rows = starts(n)
    q = values(rng, int(rows[-1]), 2, 64)
    got = d.attn(0, q, 2, rows=rows)
    check_rows(got, *m.attend(0, q, 2, 0.125, True, 0, 0, rows, len(q)), False, "missing")
    assert np.all(got[:n[0]] == 0.0)


def test_bad_rows_and_lengths(hip):
    """Rows outside [0, n_rows), lengths below the rows or past the table: what
    is not followed is left, the other sequences are right."""
    print("case: bad rows", flush=True)
    rng = np.random.default_rng(8)
    for max_rows in (1, 40):
        d = filled(hip, rng, 16, 1, 64, [30, 50, 20, 16, 48], extra=1 << 23)
        m = d.model
        m.len[:] = [30, 2 ** 31 - 1, -4, 0, 48]
        d.push()
        rows = np.array([0, 1, 2, 3, 4, 5], np.int32)
        q = values(rng, 5, 1, 64)
        got = d.attn(0, q, 1, rows=rows, max_rows=max_rows, causal=False)
        check_rows(got, *m.attend(0, q, 1, 0.125, False, 0, 0, rows, 5), False, "lengths")
        rows = np.array([-1, 3, 2, 6, 4, 5], np.int32)
        m.len[:] = [30, 50, 20, 16, 48]
        d.push()
        got = d.attn(0, q, 1, rows=rows, max_rows=max_rows)
        check_rows(got, *m.attend(0, q, 1, 0.125, True, 0, 0, rows, 5), False, "rows")


@pytest.mark.parametrize("kv,group,lens,n,max_rows", [
    (1, 1, 40, [1, 4, 1, 3, 1], 1), (1, 1, 3000, [1, 4, 1, 3, 1], 1), (1, 4, 3000, [2, 4, 1, 3, 2], 2),
    (8, 8, 1200, [6, 7, 6, 6, 8, 6, 6, 5] * 3, 6)])
def test_more_rows_than_max_rows(hip, kv, group, lens, n, max_rows):
    """Sequences with more rows than max_rows that would still fit a tile: their
    rows are left as they are and the others are right, with the keys whole (40
    tokens) and in chunks, in tiles of 16 rows and of many."""
    print(f"case: rows past max_rows, kv {kv} group {group}, {lens} tokens", flush=True)
    rng = np.random.default_rng(51)
    d = filled(hip, rng, 64, kv, 64, [lens + 5 * i for i in range(len(n))], extra=1 << 24)
    rows = starts(n)
    q = values(rng, int(rows[-1]), kv * group, 64)
    got = d.attn(0, q, kv * group, rows=rows, max_rows=max_rows)
    want, vmax, smax = d.model.attend(0, q, kv * group, 0.125, True, 0, 0, rows, len(q))
    over = np.repeat(np.asarray(n) > max_rows, n)
    want[over], vmax[over] = np.nan, 0
    check_rows(got, want, vmax, smax, False, max_rows)


@pytest.mark.parametrize("bf16", [False, True])
def test_values_that_are_not_finite(hip, bf16):
    """NaN in a token reaches the rows that see it and no other, in V only its
    dim; a query row with an infinity or NaN is NaN alone."""
    print(f"case: NaN bf16={bf16}", flush=True)
    rng = np.random.default_rng(12)
    d = filled(hip, rng, 32, 1, 64, [100, 90, 80, 70])
    m = d.model
    m.v[0, m.table[0, 2], 0, 20, 7] = 0x7F          # token 84: rows 84.. see it
    m.v[0, m.table[0, 0], 0, 3, 9] = 0xFF           # token 3: with the window, the sinks do not reach it
    m.k[0, m.table[1, 2], 0, 16, 0] = 0x7F          # token 80
    d.push()
    n = [30, 20, 5, 1]
    rows = starts(n)
    q = values(rng, int(rows[-1]), 3, 64)
    q[52, 1, 5] = np.inf
    q[53, 0, 63] = np.nan
    q[54, 2, 0] = -np.inf
    for window, sinks in ((0, 0), (40, 2), (40, 5)):
        got = d.attn(0, q, 3, rows=rows, bf16=bf16, window=window, sinks=sinks)
        want = m.attend(0, q, 3, 0.125, True, window, sinks, rows, len(q))
        check_rows(got, *want, bf16, (window, sinks))
        assert np.isnan(got[14:30, :, 7]).all() and np.isfinite(got[:14, :, 7]).all()
    m.v[0, m.table[3, 1], 0, 5, 2] = 0x7F
    d.push()
    got = d.attn(0, q[:4], 3, rows=[0, 1, 2, 3, 4], bf16=bf16)
    check_rows(got, *m.attend(0, q[:4], 3, 0.125, True, 0, 0, [0, 1, 2, 3, 4], 4), bf16, "one row")


def test_scales_far_apart(hip):
    """Pages whose scales differ by up to 2^24, large and small scores, query
    rows of every size."""
    print("case: scales", flush=True)
    rng = np.random.default_rng(13)
    for size in (1e-30, 1e-3, 1.0, 1e4):
        d = filled(hip, rng, 16, 1, 64, [200, 64])
        m = d.model
        m.vs[:] = 2.0 ** rng.integers(-20, 5, m.vs.shape)
        d.push()
        q = (values(rng, 33, 2, 64) * np.float32(size)).astype(np.float32)
        for rows in (np.array([0, 1, 2], np.int32), np.array([0, 20, 33], np.int32)):
            got = d.attn(0, q, 2, rows=rows, scale=0.125 / size)
            check_rows(got, *m.attend(0, q, 2, 0.125 / size, True, 0, 0, rows, 33), False, size)


def test_a_sequence_alone_and_in_a_batch_gives_the_same_bits(hip):
    """Single-token rows: the same sequences, in other company and on other pages."""
    print("case: batch invariance", flush=True)
    rng = np.random.default_rng(14)
    lens = [700, 33, 1030, 5]
    d = filled(hip, rng, 32, 2, 128, lens, spare=8)
    q = values(rng, 4, 4, 128)
    both = d.attn(0, q, 4, rows=[0, 1, 2, 3, 4])
    for s in range(4):
        rows = [0] * (s + 1) + [1] * (4 - s)
        alone = d.attn(0, q[s:s + 1], 4, rows=rows)
        assert np.array_equal(alone[0].view(np.uint32), both[s].view(np.uint32)), s
    d.hip.backend_kv8_compact(d.h)
    d.model.compact()
    d.check("compacted")
    moved = d.attn(0, q, 4, rows=[0, 1, 2, 3, 4])
    assert np.array_equal(moved.view(np.uint32), both.view(np.uint32))


def test_pool_past_32_bit_offsets(hip):
    """A layer's pool of more than 4 GiB: appended, attended, forked and
    compacted at its far end."""
    print("case: large pool", flush=True)
    rng = np.random.default_rng(15)
    P, kv, D = 128, 8, 128
    pages = 33000                                     # 4.33 GB of K
    c = cb.BackendKv8(layers=1, pages=pages, page_tokens=P, kv_heads=kv, head_dim=D, seqs=2, table_w=3)
    h = C.byref(c)
    n = hip.backend_kv8_floats(h)
    base = hip.backend_arena_alloc(n + (1 << 22))
    hip.backend_kv8_bind(h, base)
    d = ref.Dev.__new__(ref.Dev)
    d.hip, d.c, d.h, d.at, d.end = hip, c, h, base + (n + 63) // 64 * 256, base + (n + (1 << 22)) * 4
    # the far pages of a small model stand for the last ones of the pool
    d.model = m = ref.Cache(1, 8, P, kv, D, 2, 3)
    shift = pages - 8
    refs = np.ones(pages, np.int32)
    refs[[1, pages - 5, pages - 1]] = 0               # one near page and two far ones are free
    table = np.array([[pages - 8, pages - 3, -1], [pages - 2, -1, -1]], np.int32)
    for ptr, x in ((c.refs, refs), (c.table, table), (c.len, np.array([140, 9], np.int32))):
        d.write(ptr, x)
    m.table[:] = np.where(table >= 0, table - shift, -1)
    m.refs[:] = 1
    m.len[:] = [140, 9]
    k, v = values(rng, 149, kv, D), values(rng, 149, kv, D)
    d.append(0, k, v, rows=[0, 140, 149])
    q = values(rng, 2, 8, D)
    got = d.attn(0, q, 8, rows=[0, 1, 2])
    want = m.attend(0, q, 8, D ** -0.5, True, 0, 0, [0, 1, 2], 2)
    check_rows(got, *want, False, "far pages")
    # sequence 1 becomes a copy of sequence 0: its partly filled page goes to page 1
    hip.backend_kv8_fork(h, d.ints([1]), d.ints([0]), 1)
    t = d.get(c.table, (2, 3), np.int32)
    assert t.tolist() == [[pages - 8, pages - 3, -1], [pages - 8, 1, -1]]
    again = d.attn(0, q[[0, 0]], 8, rows=[0, 1, 2])
    assert np.array_equal(again[1].view(np.uint32), got[0].view(np.uint32))
    # three pages are free now (pages - 5, pages - 2, pages - 1): page pages - 3 moves to pages - 5
    hip.backend_kv8_compact(h)
    r = d.get(c.refs, (pages,), np.int32)
    assert r[:pages - 3].all() and not r[pages - 3:].any()
    assert d.get(c.table, (2, 3), np.int32).tolist() == [[pages - 8, pages - 5, -1], [pages - 8, 1, -1]]
    third = d.attn(0, q[[0, 0]], 8, rows=[0, 1, 2])
    assert np.array_equal(third.view(np.uint32), again.view(np.uint32))
    assert hip.backend_kv8_status(h) == 0


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def test_reserve(hip):
    """Pages in order, all or nothing, and what a refused step does."""
    print("case: reserve", flush=True)
    d = ref.Dev(hip, 1, 11, 16, 1, 64, 4, 5)
    for add in ([1, 16, 0, 17], [15, 1, 0, 0], [1, 0, 16, 0], [0, 0, 0, 0], [0, 0, 64, 64], [200, 0, 0, 0], [0, -1, 0, 0],
                [2 ** 31 - 1, 0, 0, 0], [-2 ** 31, -1, 5, 5], [0, 14, 16, 0], [1, 1, 1, 1]):
        d.reserve(add)
        d.check(add)
    d.model.rows[:] = d.get(d.c.rows, (5,), np.int32)
    x = np.ones((4, 1, 64), np.float32)
    d.reserve([70, 70, 0, 0])                        # no room in the rows: the step does nothing
    before = d.state()
    d.append(0, x, x)
    assert np.all(d.attn(0, values(np.random.default_rng(0), 4, 1, 64), 1, max_rows=4) == 55.0)
    after = d.state()
    assert all(np.array_equal(before[k], after[k]) for k in before)


@pytest.mark.parametrize("seed", range(6))
def test_page_calls_together(hip, seed):
    """Random reserve, append, fork, free, trim and compact calls against the
    model, with pools that run out, swaps, chains, repeated and bad numbers."""
    rng = np.random.default_rng(seed)
    P = [16, 32, 64, 128, 16, 32][seed]
    pages, seqs, width, kv, layers = int(rng.integers(20, 70)), int(rng.integers(2, 9)), 9, 2, 2
    print(f"case: pages seed={seed} P={P} pages={pages} seqs={seqs}", flush=True)
    d = ref.Dev(hip, layers, pages, P, kv, 64, seqs, width, extra=1 << 23)
    for step in range(40):
        do = rng.choice(["add", "add", "add", "fork", "fork", "free", "trim", "compact"])
        if do == "add":
            add = [int(rng.choice([0, 1, 1, P // 3, P + 1, 3 * P])) for _ in range(seqs)]
            d.reserve(add)
            n = int(d.model.rows[-1])
            if n:
                for lay in range(layers):
                    d.append(lay, values(rng, n, kv, 64), values(rng, n, kv, 64))
        elif do == "fork":
            n = int(rng.integers(1, seqs + 1))
            dst = [int(x) for x in rng.permutation(seqs)[:n]]
            src = [int(x) for x in rng.integers(0, seqs, n)]
            if rng.random() < 0.1:
                src[0] = int(rng.choice([-1, seqs, 2 ** 31 - 1]))
            if n > 1 and rng.random() < 0.1:
                dst[1] = dst[0]
            d.hip.backend_kv8_fork(d.h, d.ints(dst), d.ints(src), n)
            d.model.fork(dst, src)
        elif do == "free":
            which = [int(x) for x in rng.integers(0, seqs, int(rng.integers(1, 3)))]
            if rng.random() < 0.2:
                which[0] = int(rng.choice([-1, seqs]))
            d.hip.backend_kv8_free(d.h, d.ints(which), len(which[:seqs]))
            d.model.free(which[:seqs])
        elif do == "trim":
            window, sinks = int(rng.integers(1, 4 * P)), int(rng.integers(0, P + 2))
            d.hip.backend_kv8_trim(d.h, window, sinks)
            d.model.trim(window, sinks)
        else:
            d.hip.backend_kv8_compact(d.h)
            d.model.compact()
        assert all(d.model.refs[p] == np.sum(d.model.table == p) for p in range(pages))
        d.check((step, do))


def test_many_pages_and_long_rows(hip):
    """Tables wider than a workgroup and pools larger than one: more pages than
    the planning workgroup has threads."""
    print("case: many pages", flush=True)
    rng = np.random.default_rng(20)
    d = ref.Dev(hip, 1, 5000, 16, 1, 64, 6, 1200, extra=1 << 24)
    m = d.model
    d.reserve([16 * 900, 16 * 300 + 5, 0, 7, 16 * 1100, 0])
    d.check_book("reserve")
    dst, src = [2, 0, 3], [0, 1, 4]
    d.hip.backend_kv8_fork(d.h, d.ints(dst), d.ints(src), 3)
    m.fork(dst, src)
    d.check_book("fork")
    d.hip.backend_kv8_trim(d.h, 1000, 100)
    m.trim(1000, 100)
    d.check_book("trim")
    m.k[:] = rng.integers(0, 127, m.k.shape)
    m.vs[:] = rng.random(m.vs.shape)
    d.push()
    d.hip.backend_kv8_compact(d.h)
    m.compact()
    d.check("compact")
    d.hip.backend_kv8_free(d.h, d.ints([0, 2, 4]), 3)
    m.free([0, 2, 4])
    d.check_book("free")


def test_plan_and_empty_calls(hip):
    """Calls with nothing to do: no rows, no pairs, an empty cache."""
    print("case: empty calls", flush=True)
    d = ref.Dev(hip, 1, 4, 16, 1, 64, 2, 2)
    x = np.zeros((0, 1, 64), np.float32)
    d.hip.backend_kv8_fork(d.h, None, None, 0)
    d.hip.backend_kv8_free(d.h, None, 0)
    d.hip.backend_kv8_trim(d.h, 1, 0)
    d.hip.backend_kv8_compact(d.h)
    d.reserve([0, 0])
    d.hip.backend_kv8_append(d.h, 0, None, None, 64, 0, d.c.rows, 0)
    d.hip.backend_kv8_free(d.h, d.ints([1, 1]), 2)
    dst = [0, 1]
    d.hip.backend_kv8_fork(d.h, d.ints(dst), d.ints([1, 0]), 2)
    d.check()
    assert x.size == 0


# ---------------------------------------------------------------------------
# together, as a program uses them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bf16", [False, True])
def test_beam_search_run(hip, bf16):
    """A clip's prompt, then beams that fork at every step: each layer's new
    rows appended and attended, the window's old pages given back, the pool
    compacted on the way; every step's rows within the tolerance and the state
    the model's."""
    print(f"case: beam run bf16={bf16}", flush=True)
    rng = np.random.default_rng(30)
    layers, kv, group, D, P, beams = 2, 2, 2, 64, 16, 4
    d = ref.Dev(hip, layers, 48, P, kv, D, beams, 8, extra=1 << 24)
    window, sinks = 40, 3

    def layer_step(n):
        for lay in range(layers):
            d.append(lay, values(rng, n, kv, D), values(rng, n, kv, D), bf16)
            q = values(rng, n, kv * group, D)
            got = d.attn(lay, q, kv * group, bf16=bf16, window=window, sinks=sinks)
            check_rows(got, *d.model.attend(lay, q, kv * group, D ** -0.5, True, window, sinks, d.model.rows, n), bf16, lay)

    d.reserve([23, 0, 0, 0])
    layer_step(23)
    dst, src = [1, 2, 3], [0, 0, 0]
    d.hip.backend_kv8_fork(d.h, d.ints(dst), d.ints(src), 3)
    d.model.fork(dst, src)
    for step in range(30):
        d.reserve([1] * beams)
        layer_step(beams)
        parents = [int(x) for x in rng.integers(0, beams, beams)]
        d.hip.backend_kv8_fork(d.h, d.ints(range(beams)), d.ints(parents), beams)
        d.model.fork(list(range(beams)), parents)
        if step % 7 == 6:
            d.hip.backend_kv8_trim(d.h, window, sinks)
            d.model.trim(window, sinks)
            d.hip.backend_kv8_compact(d.h)
            d.model.compact()
        d.check(step)


def test_many_kv_heads(hip):
    """256 kv heads: pages of 256 KB a layer, their scales copied with them."""
    print("case: 256 kv heads", flush=True)
    rng = np.random.default_rng(48)
    d = ref.Dev(hip, 2, 8, 16, 256, 64, 3, 3, extra=1 << 23)
    d.reserve([20, 3, 0])
    for lay in (0, 1):
        d.append(lay, values(rng, 23, 256, 64), values(rng, 23, 256, 64))
    d.hip.backend_kv8_fork(d.h, d.ints([2, 1]), d.ints([0, 0]), 2)
    d.model.fork([2, 1], [0, 0])
    d.hip.backend_kv8_free(d.h, d.ints([0]), 1)
    d.model.free([0])
    d.hip.backend_kv8_compact(d.h)
    d.model.compact()
    d.check()
    q = values(rng, 2, 256, 64)
    got = d.attn(1, q, 256, rows=[0, 0, 1, 2])
    check_rows(got, *d.model.attend(1, q, 256, 0.125, True, 0, 0, [0, 0, 1, 2], 2), False, "attention")


def test_two_threads_with_a_cache_each(hip):
    """Two threads, each with its own stream, arena and cache, at once: the
    results each gets alone."""
    print("case: two threads", flush=True)
    import threading

    def program(seed):
        rng = np.random.default_rng(seed)
        d = ref.Dev(hip, 1, 60, 16, 2, 64, 4, 12, extra=1 << 23)
        got = []
        for step in range(12):
            add = [int(x) for x in rng.integers(0, 9, 4)]
            d.reserve(add)
            n = sum(add)
            if n:
                d.append(0, values(rng, n, 2, 64), values(rng, n, 2, 64))
                got.append(d.attn(0, values(rng, n, 4, 64), 4))
            d.hip.backend_kv8_fork(d.h, d.ints([3]), d.ints([int(rng.integers(3))]), 1)
        return got, d.state()

    alone = [program(50), program(51)]
    both = [None, None]

    def run(i):
        hip.backend_init(0)
        both[i] = program(50 + i)
        hip.backend_thread_cleanup()

    ts = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for x in ts:
        x.start()
    for x in ts:
        x.join(60)
    for (a, sa), (b, sb) in zip(alone, both):
        assert len(a) == len(b) and all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(a, b))
        assert all(np.array_equal(sa[k], sb[k]) for k in sa)


def test_captured_step(hip):
    """A step (reserve, append, attention in two layers) captured once and
    replayed as the texts grow, with eager work and waits in between: the bits
    of the same steps run eagerly."""
    print("case: captured step", flush=True)
    layers, kv, D, P, seqs = 2, 2, 64, 16, 3

    def program(graph):
        d = ref.Dev(hip, layers, 40, P, kv, D, seqs, 10, extra=1 << 22)
        r = np.random.default_rng(32)
        d.reserve([20, 1, 40])
        for lay in range(layers):
            d.append(lay, values(r, 61, kv, D), values(r, 61, kv, D))
        add, x = d.ints([1] * seqs), d.put(np.zeros((3, seqs, kv * D), np.float32))
        out = d.put(np.zeros((layers, seqs, kv * D), np.float32))
        step = seqs * kv * D * 4
        calls = []
        for lay in range(layers):
            a = cb.BackendKv8Attn(out=out + lay * step, q=x, ld_out=kv * D, ld_q=kv * D, heads=kv, scale=0.125, causal=1,
                                  rows=d.c.rows, n_rows=seqs, max_rows=1)
            a.work = d.take(hip.backend_kv8_attn_work(d.h, C.byref(a)) * 4 + 16)
            calls.append(a)

        def region():
            hip.backend_kv8_reserve(d.h, add)
            for lay in range(layers):
                hip.backend_kv8_append(d.h, lay, x + step, x + 2 * step, kv * D, 0, d.c.rows, seqs)
                hip.backend_kv8_attn(d.h, lay, C.byref(calls[lay]))

        got = []
        for i in range(25):
            d.write(x, values(r, 3, seqs, kv * D))
            if not graph:
                region()
            elif not hip.backend_graph_replay(9, 1, 1, seqs):
                hip.backend_graph_begin_capture(9)
                region()
                hip.backend_graph_end_capture(9, 1, 1, seqs)
            got.append(d.get(out, (layers, seqs, kv * D), np.float32))
            if i % 5 == 2:
                hip.backend_add_inplace(d.put(np.ones(64, np.float32)), d.put(np.ones(64, np.float32)), 64)
        return np.stack(got), d.state()

    (a, sa), (b, sb) = program(False), program(True)
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    assert all(np.array_equal(sa[k], sb[k]) for k in sa)
    assert np.isfinite(a).all()


@pytest.mark.parametrize("sized", [False, True])
def test_work_sized_with_the_other_row_type(hip, sized):
    """Work sized with fp32 rows used by bf16 ones, and the other way round:
    right, and nothing behind it written (most rows of the call belong to no
    sequence)."""
    print(f"case: work sized with bf16={sized}", flush=True)
    rng = np.random.default_rng(53)
    d = filled(hip, rng, 16, 1, 64, [2490], spare=1, extra=1 << 24)
    n, heads, rows = 2110, 5, starts([268])
    q = values(rng, n, heads, 64)
    call = dict(ld_out=320, ld_q=320, heads=heads, scale=0.125, causal=1, rows=d.ints(rows), n_rows=n, max_rows=268)
    for bf16 in (not sized, sized):
        floats = hip.backend_kv8_attn_work(d.h, C.byref(cb.BackendKv8Attn(bf16=int(sized), **call)))
        guard = 1 << 19
        fl, work = q.reshape(-1), d.put(np.full(floats + guard, 7.0, np.float32))
        old = np.full(fl.shape, 55.0, np.float32)
        qp, op = d.put(ref.bf16_bits(fl) if bf16 else fl), d.put(ref.bf16_bits(old) if bf16 else old)
        a = cb.BackendKv8Attn(out=op, q=qp, bf16=int(bf16), work=work, **call)
        hip.backend_kv8_attn(d.h, 0, C.byref(a))
        got = d.get(op, q.shape, np.uint16 if bf16 else np.float32)
        got = ref.bf16_value(got) if bf16 else got
        assert np.all(d.get(work + floats * 4, (guard,), np.float32) == 7.0), bf16
        check_rows(got, *d.model.attend(0, q, heads, 0.125, True, 0, 0, rows, n), bf16, bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_the_largest_scale(hip, bf16):
    """Scores of ordinary size, and zeros, from tiny queries and the largest scale allowed."""
    print(f"case: largest scale bf16={bf16}", flush=True)
    rng = np.random.default_rng(54)
    scale = float(np.float32(2.0e38))
    for n, heads in (([1, 1], 4), ([30, 60], 4), ([190, 170], 32)):
        d = filled(hip, rng, 32, 4, 64, [200, 190], extra=1 << 24)
        q = values(rng, sum(n), heads, 64) * np.float32(0.125 / scale * 2.0 ** 14) * np.float32(2.0 ** -14)
        q = ref.bf16_value(ref.bf16_bits(q))
        q[:, 1] = 0
        got = d.attn(0, q, heads, bf16=bf16, rows=starts(n), scale=scale)
        check_rows(got, *d.model.attend(0, q, heads, scale, True, 0, 0, starts(n), len(q)), bf16, n)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group,n,kw", [(16, [1, 1, 1, 1], {}), (4, [4, 1, 2, 3], {}), (8, [1, 2, 0, 2], dict(window=300, sinks=5)),
                                        (5, [3, 3, 3, 3], dict(max_len=700))])
def test_one_tile_a_sequence_gives_the_same_bits(hip, group, n, kw, bf16):
    """Up to 16 (row, query head) pairs a kv head: the same sequences in other
    company, and behind rows of none."""
    print(f"case: batch invariance group={group} n={n} {kw} bf16={bf16}", flush=True)
    rng = np.random.default_rng(55)
    d = filled(hip, rng, 32, 2, 64, [700, 33, 1030, 5], extra=1 << 25)
    rows, most = starts(n), 16 // group
    q = values(rng, int(rows[-1]), 2 * group, 64)
    both = d.attn(0, q, 2 * group, rows=rows, max_rows=most, bf16=bf16, **kw)
    check_rows(both, *d.model.attend(0, q, 2 * group, 0.125, True, kw.get("window", 0), kw.get("sinks", 0), rows, len(q), kw.get("max_len")), bf16, n)
    for s in range(4):
        one = np.where(np.arange(5) > s, n[s], 0)
        for behind in (0, 40):
            x = np.concatenate([q[rows[s]:rows[s + 1]], np.zeros((behind, 2 * group, 64), np.float32)])
            if len(x):
                alone = d.attn(0, x, 2 * group, rows=one, max_rows=most, bf16=bf16, **kw)[:n[s]]
                assert np.array_equal(alone.view(np.uint32), both[rows[s]:rows[s + 1]].view(np.uint32)), (s, behind)


def test_reserve_and_fork_in_a_pool_of_many_pages(hip):
    """More than 65536 pages, the free ones late in each planning thread's run:
    taken lowest first, to the last one, and refused when there is one too few."""
    print("case: pool of 150000 pages", flush=True)
    pages, P = 150000, 16
    c = cb.BackendKv8(layers=1, pages=pages, page_tokens=P, kv_heads=1, head_dim=64, seqs=4, table_w=300)
    h = C.byref(c)
    n = hip.backend_kv8_floats(h)
    base = hip.backend_arena_alloc(n + (1 << 20))
    hip.backend_kv8_bind(h, base)
    d = ref.Dev.__new__(ref.Dev)
    d.hip, d.c, d.h, d.at, d.end = hip, c, h, base + (n + 63) // 64 * 256, base + (n + (1 << 20)) * 4
    rng = np.random.default_rng(56)
    per = -(-pages // 1024)
    free = np.sort(rng.choice([p for p in range(pages) if p % per >= 60], 500, replace=False))
    refs = np.ones(pages, np.int32)
    refs[free] = 0
    d.write(c.refs, refs)

    def table():
        return d.get(c.table, (4, 300), np.int32)

    hip.backend_kv8_reserve(h, d.ints([P * 200 + 3, 0, P * 150, 1]))             # 201 + 150 + 1 pages
    got = table()
    assert np.array_equal(got[0, :201], free[:201]) and np.array_equal(got[2, :150], free[201:351]) and got[3, 0] == free[351]
    hip.backend_kv8_fork(h, d.ints([1]), d.ints([0]), 1)                         # copies one page
    got = table()
    assert np.array_equal(got[1, :200], free[:200]) and got[1, 200] == free[352]
    hip.backend_kv8_reserve(h, d.ints([0, 0, P * 148, 0]))                       # one more than there are
    assert hip.backend_kv8_status(h) == 1 and np.array_equal(table(), got)
    hip.backend_kv8_reserve(h, d.ints([0, 0, P * 147, 0]))
    assert hip.backend_kv8_status(h) == 0 and np.array_equal(table()[2, 150:297], free[353:])
    refs[free] = 1
    refs[free[:200]] = 2
    assert np.array_equal(d.get(c.refs, (pages,), np.int32), refs)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,heads", [([1, 1, 1], 4), ([60, 30, 20], 4), ([190, 170, 20], 32)])
def test_window_past_max_len(hip, n, heads, bf16):
    """Rows behind max_len with a window: some see its end, some the first tokens alone, some nothing."""
    print(f"case: window past max_len n={n} bf16={bf16}", flush=True)
    rng = np.random.default_rng(57)
    for window, sinks, most in ((40, 3, 150), (10, 0, 333), (100, 40, 33)):
        run_attn(hip, rng, 16, 4, heads // 4, 64, [340, 200, 150], n, (window, sinks, most), window=window, sinks=sinks,
                 max_len=most, bf16=bf16)
