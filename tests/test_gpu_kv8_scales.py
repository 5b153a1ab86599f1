"""Attention over the 8-bit cache where the pages' value scales lie far apart,
pages of zeros among them, against the 64-bit model (kv8_ref.py) — needs an
MI355X."""
import numpy as np
import pytest

import kv8_ref as ref
from test_gpu_kv8 import check_rows, starts, values

pytestmark = pytest.mark.gpu

ORDERS = {"after": lambda j, n: j >= (n + 1) // 2, "before": lambda j, n: j < n // 2, "among": lambda j, n: j % 2 == 1}


def appended(hip, rng, P, kv, D, lens, small, order, scale=1.0, extra=1 << 26):
    """Sequences of lens tokens appended at once, with values of size `scale`;
    those on the pages that `order` names are `small` times as large."""
    held = [-(-n // P) for n in lens]
    d = ref.Dev(hip, 1, sum(held) + 2, P, kv, D, len(lens), max(held) + 1, extra)
    k, v = values(rng, sum(lens), kv, D) * np.float32(0.25), values(rng, sum(lens), kv, D) * np.float32(scale)
    for s, r0 in enumerate(starts(lens)[:-1]):
        for j in range(held[s]):
            if ORDERS[order](j, held[s]):
                v[r0 + j * P:r0 + min((j + 1) * P, lens[s])] *= np.float32(small)
    d.reserve(lens)
    d.append(0, k, v)
    d.check(order)
    return d


def attends(d, rng, n, heads, bf16, what, **kw):
    rows = starts(n)
    q = values(rng, int(rows[-1]), heads, d.model.dims[4])
    got = d.attn(0, q, heads, bf16=bf16, rows=rows, **kw)
    want = d.model.attend(0, q, heads, q.shape[2] ** -0.5, kw.get("causal", True), kw.get("window", 0), kw.get("sinks", 0),
                          rows, len(q))
    check_rows(got, *want, bf16, what)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -24, 2.0 ** -30, 2.0 ** -60])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_pages_of_small_values_keep_their_weight(hip, order, small, bf16):
    """Values that vanish beside the others' still take their share of the
    softmax: single rows (the keys whole and in chunks) and a few rows."""
    print(f"case: small pages {order} {small} bf16={bf16}", flush=True)
    rng = np.random.default_rng(60)
    for P in (16, 32, 64):
        d = appended(hip, rng, P, 2, 64, [6 * P + 5, 40, 2 * P, 700], small, order)
        attends(d, rng, [1] * 4, 4, bf16, ("single", P))
        attends(d, rng, [1] * 4, 4, bf16, ("single, whole", P), max_len=700)
        attends(d, rng, [9, 12, 1, 30], 4, bf16, ("few", P), causal=False)
    d = appended(hip, rng, 128, 1, 128, [900, 400], small, order)
    attends(d, rng, [1] * 2, 16, bf16, "heads of 128")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -30])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_many_rows_pages_of_small_values_keep_their_weight(hip, order, small, bf16):
    """The same in the tiles of many rows, whose rows all see every token."""
    print(f"case: small pages, many rows {order} {small} bf16={bf16}", flush=True)
    rng = np.random.default_rng(61)
    for P in (16, 64):
        d = appended(hip, rng, P, 4, 64, [190, 300], small, order)
        attends(d, rng, [170, 190], 32, bf16, ("many", P), causal=False)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_prompts_over_pages_of_zeros(hip, order, bf16):
    """Causal prompts over pages that are all zero: rows that see nothing else give zeros."""
    print(f"case: prompts over zeros {order} bf16={bf16}", flush=True)
    rng = np.random.default_rng(62)
    for P in (16, 32):
        d = appended(hip, rng, P, 4, 64, [190, 170], 0.0, order)
        attends(d, rng, [190, 170], 32, bf16, ("many", P))
        attends(d, rng, [60, 0], 4, bf16, ("few", P))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small", [2.0 ** -20, 2.0 ** -40, 2.0 ** -85])
def test_rows_that_see_small_values_alone(hip, small, bf16):
    """Rows whose tokens are all small, beside rows of the same tile, and masked
    tokens of the same step, with large ones: as accurate, relative to what
    they see, as without those."""
    print(f"case: rows of small values {small} bf16={bf16}", flush=True)
    rng = np.random.default_rng(63)
    for P in (16, 32, 64):
        d = appended(hip, rng, P, 4, 64, [190, 170], small, "before")
        attends(d, rng, [190, 170], 32, bf16, ("many", P))
        attends(d, rng, [190, 170], 4, bf16, ("few", P))
        d = appended(hip, rng, P, 4, 64, [190, 170, 6 * P + 3, 7 * P + 3], small, "among")
        for kw in (dict(window=1), dict(window=7), dict(window=7, sinks=3), dict(window=P // 2, sinks=P + 2)):
            attends(d, rng, [190, 170, 0, 0], 32, bf16, ("many", P, kw), **kw)
            attends(d, rng, [190, 170, 1, 3], 4, bf16, ("few", P, kw), **kw)
            attends(d, rng, [1, 1, 1, 1], 4, bf16, ("single", P, kw), **kw)
    d = appended(hip, rng, 16, 1, 128, [330, 90], small, "before")
    attends(d, rng, [330, 90], 64, bf16, "heads of 128")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small,scale", [(0.0, 2.0 ** 20), (2.0 ** -110, 2.0 ** 60), (0.0, 2.0 ** 100)])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_the_whole_range_of_scales(hip, order, small, scale, bf16):
    """Value scales up to 2^200 apart: weights that have no room beside their
    page's scale still count."""
    print(f"case: whole range {order} {small} {scale} bf16={bf16}", flush=True)
    rng = np.random.default_rng(64)
    for P in (16, 64):
        d = appended(hip, rng, P, 4, 64, [190, 700], small, order, scale=scale)
        for causal in (True, False):
            attends(d, rng, [170, 190], 32, bf16, ("many", P, causal), causal=causal)
            attends(d, rng, [30, 60], 4, bf16, ("few", P, causal), causal=causal)
        attends(d, rng, [1, 1], 4, bf16, ("single", P))


@pytest.mark.parametrize("bf16", [False, True])
def test_scales_of_every_size_together(hip, bf16):
    """Each page its own scale, up to 2^25 apart: prompts and single rows."""
    print(f"case: mixed scales bf16={bf16}", flush=True)
    rng = np.random.default_rng(65)
    for P in (16, 32):
        d = appended(hip, rng, P, 4, 64, [200, 150], 1.0, "among")
        d.model.vs[:] *= 2.0 ** rng.integers(-20, 6, d.model.vs.shape)
        d.push()
        attends(d, rng, [200, 150], 32, bf16, ("many", P))
        attends(d, rng, [33, 20], 4, bf16, ("few", P))
        attends(d, rng, [1, 1], 4, bf16, ("single", P))


@pytest.mark.parametrize("bf16", [False, True])
def test_values_near_the_largest_float(hip, bf16):
    """Values up to 1e38: sums of several of them stay in range, whatever their
    weights are relative to the largest score found so far."""
    print(f"case: largest values bf16={bf16}", flush=True)
    rng = np.random.default_rng(66)
    P, kv, D, lens = 32, 4, 64, [190, 700]
    d = ref.Dev(hip, 1, 40, P, kv, D, 2, 24, 1 << 24)
    # keys of growing size along one direction, which the queries have too: scores rise by 5 bits over the text
    k = values(rng, sum(lens), kv, D) * np.float32(0.05)
    k[:, :, 0] = np.concatenate([np.linspace(0, 3.5, n) for n in lens])[:, None]
    k = ref.bf16_value(ref.bf16_bits(k))
    v = ref.bf16_value(ref.bf16_bits((rng.uniform(-1, 1, (sum(lens), kv, D)) * 1e38).astype(np.float32)))
    d.reserve(lens)
    d.append(0, k, v)
    d.check()
    for n, heads, kw in (([170, 190], 32, {}), ([170, 190], 32, dict(causal=False)), ([30, 60], 4, {}), ([1, 1], 4, {}),
                         ([1, 1], 4, dict(max_len=700))):
        rows = starts(n)
        q = values(rng, int(rows[-1]), heads, D) * np.float32(0.05)
        q[:, :, 0] = 8.0
        q = ref.bf16_value(ref.bf16_bits(q))
        got = d.attn(0, q, heads, bf16=bf16, rows=rows, **kw)
        want = d.model.attend(0, q, heads, D ** -0.5, kw.get("causal", True), 0, 0, rows, len(q))
        assert np.isfinite(got).all(), (n, kw)
        check_rows(got, *want, bf16, (n, kw))
