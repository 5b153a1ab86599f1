"""Attention over the 8-bit cache where the pages' value scales lie far apart,
pages of zeros among them, against the 64-bit model (kv8_ref.py) — needs an
MI355X."""
import numpy as np
import pytest

import kv8_ref as ref
from test_gpu_kv8 import check_rows, starts, values

pytestmark = pytest.mark.gpu

ORDERS = {"after": lambda j, n: j >= (n + 1) // 2, "before": lambda j, n: j < n // 2, "among": lambda j, n: j % 2 == 1}


def appended(hip, rng, P, kv, D, lens, small, order, extra=1 << 24):
    """Sequences of lens tokens appended at once; the values of the pages that
    `order` names are `small` times as large as the others'."""
    held = [-(-n // P) for n in lens]
    d = ref.Dev(hip, 1, sum(held) + 2, P, kv, D, len(lens), max(held) + 1, extra)
    k, v = values(rng, sum(lens), kv, D) * np.float32(0.25), values(rng, sum(lens), kv, D)
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
