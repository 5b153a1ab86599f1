"""Refusals of the paged 8-bit cache's calls, and its 64-bit model (no GPU
needed: the checks run before any device work)."""
import ctypes as C
import subprocess
import sys

import numpy as np
import pytest

import ctbind as cb
import kv8_ref as ref

GOOD = dict(layers=2, pages=8, page_tokens=16, kv_heads=2, head_dim=64, seqs=3, table_w=4)
PTRS = dict(k=4096, v=8192, kscale=4096, vscale=4096, table=4096, len=4096, refs=4096, rows=4096, plan=4096)
CALL = dict(out=4096, q=4096, ld_out=128, ld_q=128, heads=2, scale=0.125, causal=1, rows=4096, n_rows=4, max_rows=2,
            work=4096)


def program(call, cache=None, attn=None):
    c = {**GOOD, **PTRS, **(cache or {})}
    a = {**CALL, **(attn or {})}
    return (f"import sys; sys.path.insert(0, {cb.PKG_DIR!r}); import ctypes as C, ctbind as cb; L = cb.hip(); "
            f"c = cb.BackendKv8(**{c!r}); h = C.byref(c); nan = float('nan'); a = cb.BackendKv8Attn(**{a!r}); p = C.byref(a); {call}; print('returned')")


APPEND = "L.backend_kv8_append(h, 0, 4096, 4096, 128, 0, 4096, 4)"
ATTN = "L.backend_kv8_attn(h, 0, p)"
CASES = {
    "no_cache": ("L.backend_kv8_compact(None)", {}, {}, "no cache"),
    "layers": (APPEND, dict(layers=0), {}, "layers outside"),
    "pages": (APPEND, dict(pages=0), {}, "pages outside"),
    "pages_many": ("L.backend_kv8_floats(h)", dict(pages=(1 << 24) + 1), {}, "pages outside"),
    "page_tokens": ("L.backend_kv8_plan_ints(h)", dict(page_tokens=48), {}, "page_tokens is not"),
    "head_dim": (ATTN, dict(head_dim=160), {}, "head_dim is not"),
    "kv_heads": (ATTN, dict(kv_heads=257), {}, "kv_heads outside"),
    "seqs": (APPEND, dict(seqs=257), {}, "seqs outside"),
    "table_w": (APPEND, dict(table_w=0), {}, "table_w outside"),
    "table_w_long": (APPEND, dict(table_w=(1 << 20) + 1), {}, "table_w outside"),
    "null_pool": (APPEND, dict(v=0), {}, "a pointer of the cache is NULL"),
    "null_plan": ("L.backend_kv8_trim(h, 1, 0)", dict(plan=0), {}, "a pointer of the cache is NULL"),
    "pool_alignment": (APPEND, dict(k=4104), {}, "not 16-byte aligned"),
    "bind_null": ("L.backend_kv8_bind(h, None)", {}, {}, "memory is NULL"),
    "bind_alignment": ("L.backend_kv8_bind(h, 4100)", {}, {}, "not 16-byte aligned"),
    "reserve_null": ("L.backend_kv8_reserve(h, None)", {}, {}, "add or the cache's rows"),
    "reserve_rows": ("L.backend_kv8_reserve(h, 4096)", dict(rows=0), {}, "add or the cache's rows"),
    "append_layer": ("L.backend_kv8_append(h, 2, 4096, 4096, 128, 0, 4096, 4)", {}, {}, "layer outside"),
    "append_layer_negative": ("L.backend_kv8_append(h, -1, 4096, 4096, 128, 0, 4096, 4)", {}, {}, "layer outside"),
    "append_rows_null": ("L.backend_kv8_append(h, 0, 4096, 4096, 128, 0, None, 4)", {}, {}, "rows are NULL"),
    "append_rows_negative": ("L.backend_kv8_append(h, 0, 4096, 4096, 128, 0, 4096, -1)", {}, {}, "n_rows outside"),
    "append_rows_many": ("L.backend_kv8_append(h, 0, 4096, 4096, 128, 0, 4096, (1 << 24) + 1)", {}, {}, "n_rows outside"),
    "append_rows_heads": ("L.backend_kv8_append(h, 0, 4096, 4096, 8192, 0, 4096, 1 << 20)", dict(kv_heads=128), {}, "n_rows * kv_heads above"),
    "append_null": ("L.backend_kv8_append(h, 0, 4096, None, 128, 0, 4096, 4)", {}, {}, "k or v is NULL"),
    "append_alignment": ("L.backend_kv8_append(h, 0, 4098, 4096, 128, 0, 4096, 4)", {}, {}, "not aligned"),
    "append_alignment_bf16": ("L.backend_kv8_append(h, 0, 4097, 4096, 128, 1, 4096, 4)", {}, {}, "not aligned"),
    "append_ld": ("L.backend_kv8_append(h, 0, 4096, 4096, 127, 0, 4096, 4)", {}, {}, "ld below"),
    "attn_null_call": ("L.backend_kv8_attn(h, 0, None)", {}, {}, "no arguments"),
    "attn_heads": (ATTN, {}, dict(heads=3), "heads is not a multiple"),
    "attn_heads_none": (ATTN, {}, dict(heads=0), "heads is not a multiple"),
    "attn_rows_many": ("L.backend_kv8_attn_work(h, p)", {}, dict(n_rows=1 << 24, heads=16), "n_rows * heads above"),
    "attn_rows_negative": (ATTN, {}, dict(n_rows=-1), "n_rows outside"),
    "attn_max_rows": (ATTN, {}, dict(max_rows=0), "max_rows < 1"),
    "attn_max_len": (ATTN, {}, dict(max_len=-1), "max_len < 0"),
    "attn_window": (ATTN, {}, dict(window=-1), "window or sinks < 0"),
    "attn_sinks": (ATTN, {}, dict(sinks=-1), "window or sinks < 0"),
    "attn_window_causal": (ATTN, {}, dict(window=4, causal=0), "a window needs causal rows"),
    "attn_scale_zero": (ATTN, {}, dict(scale=0.0), "scale is not positive"),
    "attn_scale_nan": (ATTN, {}, dict(scale=float("nan")), "scale is not positive"),
    "attn_rows_null": (ATTN, {}, dict(rows=0), "rows are NULL"),
    "attn_q": (ATTN, {}, dict(q=0), "q or out is NULL"),
    "attn_out_alignment": (ATTN, {}, dict(out=4098), "not aligned"),
    "attn_ld": (ATTN, {}, dict(ld_q=127), "ld_q or ld_out below"),
    "attn_layer": ("L.backend_kv8_attn(h, 5, p)", {}, {}, "layer outside"),
    "attn_work": (ATTN, dict(table_w=4096), dict(work=0), "work is NULL"),
    "attn_work_alignment": (ATTN, dict(table_w=4096), dict(work=4100), "work is NULL or not 16-byte"),
    "fork_n": ("L.backend_kv8_fork(h, 4096, 4096, 4)", {}, {}, "n outside"),
    "fork_null": ("L.backend_kv8_fork(h, 4096, None, 2)", {}, {}, "dst or src is NULL"),
    "free_n": ("L.backend_kv8_free(h, 4096, -1)", {}, {}, "n outside"),
    "free_null": ("L.backend_kv8_free(h, None, 1)", {}, {}, "seqs is NULL"),
    "trim_window": ("L.backend_kv8_trim(h, 0, 0)", {}, {}, "window < 1"),
    "trim_sinks": ("L.backend_kv8_trim(h, 4, -1)", {}, {}, "window < 1 or sinks < 0"),
    "before_init": (APPEND, {}, {}, "has not called backend_init"),
    "before_init_attn": (ATTN, {}, {}, "has not called backend_init"),
    "stream_before_init": ("L.backend_stream()", {}, {}, "has not called backend_init"),
}


# a scale whose product with log2(e), by which the kernels multiply it, overflows: a score of 0 would be NaN
CASES["attn_scale_large"] = (ATTN, {}, dict(scale=2.4e38), "scale is not positive and at most")


@pytest.mark.parametrize("case", sorted(CASES))
def test_refused_before_device_work(case):
    call, cache, attn, msg = CASES[case]
    r = subprocess.run([sys.executable, "-c", program(call, cache, attn)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1, (r.returncode, r.stdout, r.stderr)
    assert msg in r.stderr, r.stderr
    assert "returned" not in r.stdout


def test_sizes():
    """The arena's share covers the arrays; more rows, tokens or heads never take less work."""
    L = cb.hip()
    c = cb.BackendKv8(**GOOD)
    h = C.byref(c)
    pool = 2 * 8 * 2 * 16 * 64
    least = 2 * pool // 4 + 2 * (2 * 8 * 2) + 3 * 4 + 3 + 8 + 4 + L.backend_kv8_plan_ints(h)
    assert least <= L.backend_kv8_floats(h) <= least + 4 * 9
    big = cb.BackendKv8(**{**GOOD, "pages": 1 << 24, "page_tokens": 128, "head_dim": 128, "kv_heads": 8})
    assert L.backend_kv8_floats(C.byref(big)) > 2 * (1 << 24) * 2 * 8 * 128 * 128 // 4       # past 32 bits
    c.table_w = 4096
    work = []
    for n, heads in ((1, 2), (3, 2), (3, 8), (40, 8), (400, 8)):
        a = cb.BackendKv8Attn(**{**CALL, "n_rows": n, "max_rows": n, "heads": heads, "ld_q": 512, "ld_out": 512})
        work.append(L.backend_kv8_attn_work(h, C.byref(a)))
    assert work[0] > 0
    # one chunk needs none, whatever the pointers
    short = cb.BackendKv8Attn(**{**CALL, "max_len": 40})
    assert L.backend_kv8_attn_work(h, C.byref(short)) == 0


def test_work_is_enough_for_smaller_calls():
    """Whatever a call with no more rows and tokens splits into, its partial
    results fit the work of the larger one (the bound and the need are host
    functions of the sizes)."""
    L = cb.hip()
    L.ctk_kv8_attn_need.argtypes, L.ctk_kv8_attn_need.restype = [C.c_void_p, C.c_void_p], C.c_size_t
    rng = np.random.default_rng(3)

    def log(a, b):
        return int(round(float(np.exp(rng.uniform(np.log(a), np.log(b))))))

    split = 0
    for _ in range(4000):
        kv, group = int(rng.choice([1, 2, 3, 8, 16, 256])), int(rng.choice([1, 2, 3, 5, 8, 16, 32]))
        c = cb.BackendKv8(layers=1, pages=8, page_tokens=int(rng.choice([16, 32, 64, 128])), kv_heads=kv,
                          head_dim=int(rng.choice([64, 128])), seqs=log(1, 256), table_w=log(1, 100000))
        window = int(rng.choice([0, 0, 1])) * log(1, 100000)
        fixed = dict(bf16=int(rng.integers(2)), heads=kv * group, scale=1.0, causal=1, window=window,
                     sinks=log(1, 1000) if window else 0)
        n = log(1, min(1 << 16, (1 << 27) // (kv * group)))
        rows, most = log(1, n), int(rng.integers(2)) * log(1, 1 << 20)
        work = L.backend_kv8_attn_work(C.byref(c), C.byref(cb.BackendKv8Attn(n_rows=n, max_rows=rows, max_len=most, **fixed)))
        for k in range(4):
            a = cb.BackendKv8Attn(n_rows=n if k == 0 else log(1, n), max_rows=rows if k == 0 else log(1, rows),
                                  max_len=most if k == 0 else log(1, most) if most else int(k > 1) * log(1, 1 << 18), **fixed)
            need = L.ctk_kv8_attn_need(C.byref(c), C.byref(a))
            split += need > 0
            assert need <= work, (kv, group, n, rows, most, a.n_rows, a.max_rows, a.max_len)
    assert split > 1000


def test_work_is_enough_for_either_row_type():
    """Work sized with fp32 rows is enough for bf16 ones and the other way
    round: the type is not among what has to stay the same."""
    L = cb.hip()
    L.ctk_kv8_attn_need.argtypes, L.ctk_kv8_attn_need.restype = [C.c_void_p, C.c_void_p], C.c_size_t
    rng = np.random.default_rng(5)

    def log(a, b):
        return int(round(float(np.exp(rng.uniform(np.log(a), np.log(b))))))

    def check(c, a, **smaller):
        p = C.byref(c)
        for sized in (0, 1):
            work = L.backend_kv8_attn_work(p, C.byref(cb.BackendKv8Attn(bf16=sized, **a)))
            for used in (0, 1):
                need = L.ctk_kv8_attn_need(p, C.byref(cb.BackendKv8Attn(bf16=used, **{**a, **smaller})))
                assert need <= work, (sized, used, need, work, a, smaller)

    for kv, group, seqs, width, P, n, rows, D in ((1, 8, 46, 88, 32, 3358, 3358, 128), (27, 25, 9, 52, 64, 11, 5, 64)):
        c = cb.BackendKv8(layers=1, pages=8, page_tokens=P, kv_heads=kv, head_dim=D, seqs=seqs, table_w=width)
        check(c, dict(heads=kv * group, scale=1.0, causal=1, n_rows=n, max_rows=rows))
    for _ in range(6000):
        kv, group = int(rng.choice([1, 1, 2, 3, 8, 27, 256])), int(rng.choice([1, 2, 3, 5, 8, 16, 25, 32]))
        c = cb.BackendKv8(layers=1, pages=8, page_tokens=int(rng.choice([16, 32, 64, 128])), kv_heads=kv,
                          head_dim=int(rng.choice([64, 128])), seqs=log(1, 256), table_w=log(1, 2000))
        n = log(1, min(1 << 14, (1 << 27) // (kv * group)))
        rows, window = log(1, n), int(rng.integers(2)) * log(1, 20000)
        a = dict(heads=kv * group, scale=1.0, causal=1, window=window, sinks=log(1, 300) if window else 0, n_rows=n, max_rows=rows)
        check(c, a)
        check(c, a, n_rows=log(1, n), max_rows=log(1, rows), max_len=log(1, 1 << 16))


def test_more_rows_tokens_or_heads_never_take_less_work():
    """And they do take more, where texts are split."""
    L = cb.hip()
    rng = np.random.default_rng(6)

    def log(a, b):
        return int(round(float(np.exp(rng.uniform(np.log(a), np.log(b))))))

    more = {"n_rows": 0, "max_rows": 0, "max_len": 0, "heads": 0}
    for _ in range(3000):
        kv, group = int(rng.choice([1, 2, 8, 256])), int(rng.choice([1, 2, 5, 8, 16]))
        c = cb.BackendKv8(layers=1, pages=8, page_tokens=64, kv_heads=kv, head_dim=128, seqs=log(1, 256), table_w=4000)
        n, window = log(1, min(20000, (1 << 25) // (kv * (group + 8)))), int(rng.integers(2)) * log(1, 20000)
        a = dict(heads=kv * group, scale=1.0, causal=1, bf16=int(rng.integers(2)), window=window,
                 sinks=log(1, 300) if window else 0, n_rows=n, max_rows=log(1, n), max_len=log(1, 200000))
        least = L.backend_kv8_attn_work(C.byref(c), C.byref(cb.BackendKv8Attn(**a)))
        for name in more:
            b = {**a, name: a[name] * 2 if name != "heads" else a[name] + kv * log(1, 8)}
            work = L.backend_kv8_attn_work(C.byref(c), C.byref(cb.BackendKv8Attn(**b)))
            assert work >= least, (name, a)
            more[name] += work > least
    assert min(more.values()) > 100, more


def test_model_rounding():
    """The model's rounding against the definition: every code is its own
    nearest, midpoints go to the even code, values past the largest are held."""
    fine = np.array([c for c in range(256) if c & 0x7F != 0x7F], np.uint8)
    assert np.array_equal(ref.to_codes(ref.E4M3[fine]), fine)
    mid = ref.to_codes(ref._MID)
    assert np.all(mid % 2 == 0)
    below, above = np.nextafter(ref._MID, 0), np.nextafter(ref._MID, 1e9)
    assert np.array_equal(ref.to_codes(below), np.arange(126)) and np.array_equal(ref.to_codes(above), np.arange(1, 127))
    assert ref.to_codes([449, np.inf, -np.inf, np.nan, -0.0]).tolist() == [0x7E, 0x7E, 0xFE, 0x7F, 0x80]
    assert ref.need_exp([448.0]) == 0 and ref.need_exp([448.1, np.inf]) == 1 and ref.need_exp([0.0]) == -100
