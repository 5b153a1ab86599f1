"""Refusals of the 4-bit linear maps, the attention with a shared prefix and the
logits call, and their models against the definitions (no GPU needed: the
checks run before any device work)."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import ctbind as cb
import logits_ref
import w4_ref

W4 = dict(in_d=256, out_d=64, group=64, scale_f16=0, codes=4096, scales=8192)
LINEAR = dict(y=4096, x=8192, ld_y=64, ld_x=256, rows=3)
LOGITS = dict(logits=4096, out=8192, ld=9000, ld_out=9000, rows=3, vocab=9000, id=4096, score=4096, work=4096)
HIST = dict(hist=4096, ld_hist=10, hist_len=4096)
KV8 = dict(layers=2, pages=8, page_tokens=16, kv_heads=2, head_dim=64, seqs=3, table_w=4, k=4096, v=8192, kscale=4096,
           vscale=4096, table=4096, len=4096, refs=4096, rows=4096, plan=4096)
ATTN = dict(out=4096, q=4096, ld_out=128, ld_q=128, heads=2, scale=0.125, causal=1, rows=4096, n_rows=4, max_rows=2, work=4096)


def program(call, **change):
    parts = {n: {**d, **{k: v for k, v in change.items() if k in dict(c._fields_)}}
             for n, d, c in (("w", W4, cb.BackendW4), ("a", LINEAR, cb.BackendW4Linear), ("l", LOGITS, cb.BackendLogits),
                             ("c", KV8, cb.BackendKv8), ("t", ATTN, cb.BackendKv8Attn))}
    return (f"import sys; sys.path.insert(0, {cb.PKG_DIR!r}); import ctypes as C, ctbind as cb; L = cb.hip(); r = C.byref; "
            f"w = cb.BackendW4(**{parts['w']!r}); a = cb.BackendW4Linear(**{parts['a']!r}); "
            f"l = cb.BackendLogits(**{parts['l']!r}); c = cb.BackendKv8(**{parts['c']!r}); "
            f"t = cb.BackendKv8Attn(**{parts['t']!r}); {call}; print('returned')")


LIN, LOG, SHARED = "L.backend_linear_w4(r(w), r(a))", "L.backend_logits(r(l))", "L.backend_kv8_attn_shared(r(c), 0, r(t), 4096)"
CASES = {
    "no_weight": ("L.backend_w4_floats(None)", {}, "no weight"),
    "in_d": (LIN, dict(in_d=0), "in_d or out_d outside"),
    "out_d": (LIN, dict(out_d=(1 << 20) + 1), "in_d or out_d outside"),
    "product": ("L.backend_w4_floats(r(w))", dict(in_d=1 << 16, out_d=(1 << 15) + 1), "their product above"),
    "group": (LIN, dict(group=96), "group is not"),
    "scale_f16": (LIN, dict(scale_f16=2), "scale_f16 is not"),
    "codes_null": (LIN, dict(codes=0), "codes or scales are NULL"),
    "scales_alignment": (LIN, dict(scales=8200), "codes or scales are NULL or not 16-byte"),
    "w4_bind": ("L.backend_w4_bind(r(w), 4100)", {}, "memory is NULL or not 16-byte"),
    "load_null": ("L.backend_w4_load(r(w), None, 4096, None)", {}, "w4_load"),
    "load_alignment": ("L.backend_w4_load(r(w), 4096, 4097, None)", {}, "w4_load"),
    "quantize_null": ("L.backend_w4_quantize(r(w), None)", {}, "w4_quantize"),
    "unpack_alignment": ("L.backend_w4_unpack(r(w), 4098)", {}, "w4_unpack"),
    "linear_null": ("L.backend_linear_w4(r(w), None)", {}, "no arguments"),
    "linear_rows": (LIN, dict(rows=-1), "rows outside"),
    "linear_rows_many": (LIN, dict(rows=(1 << 24) + 1), "rows outside"),
    "linear_act": (LIN, dict(act=4), "unknown act"),
    "linear_x": (LIN, dict(x=0), "x or y is NULL"),
    "linear_y_alignment": (LIN, dict(y=4098), "x or y is NULL or not aligned"),
    "linear_bf16_alignment": (LIN, dict(y=4097, bf16=1), "x or y is NULL or not aligned"),
    "linear_ld_x": (LIN, dict(ld_x=255), "ld_x below"),
    "linear_ld_y": (LIN, dict(ld_y=63), "ld_y below"),
    "linear_bias": (LIN, dict(bias=4097), "bias is not aligned"),
    "linear_before_init": (LIN, {}, "has not called backend_init"),
    "linear_in_place": (LIN, dict(y=4096, x=4096), "y is x"),
    "load_before_init": ("L.backend_w4_load(r(w), 4096, 4096, None)", {}, "has not called backend_init"),
    "logits_null": ("L.backend_logits(None)", {}, "no arguments"),
    "logits_rows": (LOG, dict(rows=65536), "rows outside"),
    "logits_vocab": ("L.backend_logits_work(r(l))", dict(vocab=0), "vocab outside"),
    "logits_pointer": (LOG, dict(logits=0), "logits are NULL"),
    "logits_out_alignment": (LOG, dict(out=8194), "a pointer is not aligned"),
    "logits_nothing": (LOG, dict(out=0, id=0, score=0), "nothing to write"),
    "logits_ld": (LOG, dict(ld=8999), "ld or ld_out below"),
    "logits_ld_out": (LOG, dict(ld_out=8999), "ld or ld_out below"),
    "logits_in_place": (LOG, dict(out=4096, ld_out=9001), "in place with another"),
    "logits_hist_len": (LOG, dict(hist=4096, ld_hist=3), "a history without hist_len"),
    "logits_ld_hist": (LOG, dict(hist=4096, hist_len=4096, ld_hist=-1), "ld_hist outside"),
    "logits_penalty": (LOG, dict(repeat=4096), "penalties without a history"),
    "logits_ngram_alignment": (LOG, dict(HIST, ngram=4098), "its penalties is not aligned"),
    "logits_biases": (LOG, dict(bias_start=4096, biases=-1), "biases < 0"),
    "logits_bias_list": (LOG, dict(bias_start=4096, biases=3, bias_id=4096), "without bias_id or bias"),
    "logits_masks": (LOG, dict(mask=4096, ld_mask=282), "masks < 1 or"),
    "logits_ld_mask": (LOG, dict(mask=4096, masks=1, ld_mask=281), "masks < 1 or"),
    "logits_work": (LOG, dict(work=0), "work is NULL"),
    "logits_before_init": (LOG, dict(HIST, repeat=4096), "has not called backend_init"),
    "share_null": ("L.backend_kv8_share(r(c), None)", {}, "share is NULL"),
    "share_alignment": ("L.backend_kv8_share(r(c), 4098)", {}, "share is NULL or not aligned"),
    "share_cache": ("L.backend_kv8_share(r(c), 4096)", dict(refs=0), "a pointer of the cache is NULL"),
    "shared_window": (SHARED, dict(window=5), "no window"),
    "shared_work_window": ("L.backend_kv8_attn_shared_work(r(c), r(t))", dict(window=5), "no window"),
    "shared_share": ("L.backend_kv8_attn_shared(r(c), 0, r(t), None)", {}, "share is NULL"),
    "shared_layer": ("L.backend_kv8_attn_shared(r(c), 2, r(t), 4096)", {}, "layer outside"),
    "shared_null": ("L.backend_kv8_attn_shared(r(c), 0, None, 4096)", {}, "no arguments"),
    "shared_heads": (SHARED, dict(heads=3), "heads is not a multiple"),
    "shared_ld": (SHARED, dict(ld_q=127), "ld_q or ld_out below"),
    "shared_work": (SHARED, dict(table_w=4096, work=0), "work is NULL"),
    "shared_before_init": (SHARED, {}, "has not called backend_init"),
}


@pytest.mark.parametrize("case", sorted(CASES))
def test_refused_before_device_work(case):
    call, change, msg = CASES[case]
    r = subprocess.run([sys.executable, "-c", program(call, **change)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1, (r.returncode, r.stdout, r.stderr)
    assert msg in r.stderr, r.stderr
    assert "returned" not in r.stdout


def test_nothing_to_do_needs_no_device():
    """No rows: the calls return before they look for a device."""
    call = ("a.rows = l.rows = t.n_rows = 0; a.x = l.logits = t.q = None; L.backend_linear_w4(r(w), r(a)); "
            "L.backend_logits(r(l)); L.backend_kv8_attn_shared(r(c), 0, r(t), 4096)")
    r = subprocess.run([sys.executable, "-c", program(call)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "returned" in r.stdout, r.stderr


def test_w4_sizes():
    """Codes of whole tiles of 16 x 128, a word for each output and group."""
    L = cb.hip()
    for in_d, out_d, group, words in ((128, 16, 128, 256 + 16), (129, 17, 32, 4 * (256 + 64)), (1, 1, 64, 256 + 32),
                                      (1 << 11, 1 << 20, 128, (1 << 28) + (1 << 24))):
        assert L.backend_w4_floats(C.byref(cb.BackendW4(in_d=in_d, out_d=out_d, group=group))) == words
    w = cb.BackendW4(in_d=129, out_d=17, group=32)
    L.backend_w4_bind(C.byref(w), 1 << 20)
    assert (w.codes, w.scales) == (1 << 20, (1 << 20) + 4 * 1024)


def test_logits_work():
    """None where a row is one workgroup's; no less for more rows or a larger vocabulary."""
    L = cb.hip()
    work = [[L.backend_logits_work(C.byref(cb.BackendLogits(rows=r, vocab=v))) for v in (10, 5000, 1 << 24)] for r in (0, 1, 700)]
    assert work[0] == [0, 0, 0] and work[2][2] > 0
    for a in work:
        assert a == sorted(a)
    for a, b in zip(work, work[1:]):
        assert all(x <= y for x, y in zip(a, b))


def test_shared_work_covers_smaller_calls():
    """Work sized once is enough for every smaller call, of either type, and
    never less for a larger one; what a call needs is within what it is told."""
    L = cb.hip()
    for f in (L.ctk_kv8_attn_shared_need, L.backend_kv8_attn_shared_work):
        f.argtypes, f.restype = [C.c_void_p, C.c_void_p], C.c_size_t
    rng = np.random.default_rng(0)
    apart = 0
    for _ in range(300):
        kv, group = int(rng.choice([1, 2, 8, 16])), int(rng.choice([1, 2, 4, 8]))
        c = cb.BackendKv8(layers=1, pages=50, page_tokens=int(rng.choice([16, 64, 128])), kv_heads=kv, head_dim=int(rng.choice([64, 128])),
                          seqs=int(rng.choice([1, 2, 7, 64, 256])), table_w=int(np.exp(rng.uniform(0, 9))))

        def call(n_rows, max_rows, max_len, bf16, causal):
            return cb.BackendKv8Attn(out=4096, q=4096, ld_out=kv * group * 128, ld_q=kv * group * 128, heads=kv * group, scale=1.0,
                                     rows=4096, n_rows=n_rows, max_rows=max_rows, max_len=max_len, bf16=bf16, causal=causal)
        n, m, ml = (int(np.exp(rng.uniform(0, x))) for x in (8, 6, 11))
        whole = L.backend_kv8_attn_shared_work(C.byref(c), C.byref(call(n, m, ml, 0, 1)))
        assert whole == L.backend_kv8_attn_shared_work(C.byref(c), C.byref(call(n, m, ml, 1, 0)))
        for _ in range(10):
            a = call(int(rng.integers(1, n + 1)), int(rng.integers(1, m + 1)), int(rng.integers(1, ml + 1)), int(rng.integers(2)),
                     int(rng.integers(2)))
            need, work = (f(C.byref(c), C.byref(a)) for f in (L.ctk_kv8_attn_shared_need, L.backend_kv8_attn_shared_work))
            assert need <= work <= whole
            apart += need > 0
    assert apart > 300


def test_struct_mirrors(tmp_path):
    """The ctypes structs have the C structs' sizes and last fields' places."""
    names = {"BackendW4": "scales", "BackendW4Linear": "scale", "BackendLogits": "work", "BackendKv8": "plan", "BackendKv8Attn": "work"}
    src = tmp_path / "sizes.c"
    src.write_text('#include "backend.h"\n#include <stdio.h>\nint main(void) {\n' + "".join(
        f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, {f}));\n' for n, f in names.items()) + "return 0; }\n")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split("\n")
    for line, (n, f) in zip(out, names.items()):
        assert line == f"{C.sizeof(getattr(cb, n))} {getattr(getattr(cb, n), f).offset}", n


def test_w4_model():
    """The model's quantiser: an integer grid comes back as it is; errors of at
    most half a step, a step where the zero point or an end was held; packing."""
    rng = np.random.default_rng(1)
    z = rng.integers(0, 16, (8, 4))
    codes = rng.integers(0, 16, (8, 4, 32))
    codes[:, :, 0], codes[:, :, 1] = 0, 15
    W = (codes - z[..., None]).reshape(8, 128) * 0.5
    c, bits, zero = w4_ref.quantize(W.astype(np.float32), 32, False)
    assert np.array_equal(w4_ref.values(c, bits, zero, 32, False), W)
    assert np.array_equal(w4_ref.pack(c)[:, 3], c[:, 6] | c[:, 7] << 4)
    W = w4_ref.bf16_value(w4_ref.bf16_bits(rng.standard_normal((20, 200)).astype(np.float32)))
    for f16 in (False, True):
        c, bits, zero = w4_ref.quantize(W, 64, f16)
        V = w4_ref.values(c, bits, zero, 64, f16)
        s = w4_ref.wide(bits.view(np.float16).astype(np.float64) if f16 else w4_ref.bf16_value(bits).astype(np.float64), 64, 200)
        # scale rounded: 15 steps of it may miss the range by 15 * 2^-9 of a step at each end
        assert np.all(np.abs(V - W) <= s * (1 + 15 * 2.0 ** -8))
        assert np.mean(np.abs(V - W) <= 0.5 * s * (1 + 1e-6)) > 0.9


def test_logits_model():
    """The restatement on a row small enough to do by hand."""
    x = np.array([[1.0, -2.0, 3.0, 0.5, 4.0, -1.0]], np.float32)
    kw = dict(hist=np.array([[2, 1, 4, 2, 1]]), hist_len=[5], prompt_len=[2], repeat=[2.0], frequency=[0.25], presence=[0.5])
    y, i, s = logits_ref.process(x, **kw)
    assert y[0].tolist() == [1.0, -4.75, 0.75, 0.5, 1.25, -1.0] and i[0] == 4 and s[0] == 1.25
    y, i, _ = logits_ref.process(x, ngram=[3], bias_start=[0, 3], bias_id=[0, 3, 0], bias=[9.0, 1.0, 1.0], **kw)
    assert y[0].tolist() == [2.0, -4.75, 0.75, 1.5, -np.inf, -1.0] and i[0] == 0      # 2 1 was followed by 4
    y, i, s = logits_ref.process(x, mask=np.array([[0b000010]], np.uint32), mask_of=[0])
    assert i[0] == 1 and s[0] == -2.0 and np.isneginf(y[0, [0, 2, 3, 4, 5]]).all()
    assert logits_ref.process(x, mask=np.zeros((1, 1), np.uint32))[1][0] == -1


def test_shared_join_fits_a_grid():
    """Rows that no sequence has count too: a call whose join would be a wavefront for
    each of 2^26 rows and heads or more (2^32 threads) goes through every sequence's own table."""
    L = cb.hip()
    for f in (L.ctk_kv8_attn_shared_need, L.ctk_kv8_attn_need):
        f.argtypes, f.restype = [C.c_void_p, C.c_void_p], C.c_size_t
    c = cb.BackendKv8(layers=1, pages=50, page_tokens=64, kv_heads=2, head_dim=64, seqs=64, table_w=4096)
    for heads in (2, 8, 32):
        for rows in (64, 1 << 10, 1 << 19, 1 << 20, 1 << 21, 1 << 22, 1 << 24):
            if rows * heads > 1 << 27:
                continue
            a = cb.BackendKv8Attn(out=4096, q=4096, ld_out=heads * 64, ld_q=heads * 64, heads=heads, scale=1.0, rows=4096,
                                  n_rows=rows, max_rows=1, causal=1)
            shared, own = (f(C.byref(c), C.byref(a)) for f in (L.ctk_kv8_attn_shared_need, L.ctk_kv8_attn_need))
            apart = shared != own
            threads = 2 * -(-rows * (heads // 2) // 4) * 256
            assert not apart or threads < 1 << 32, (heads, rows)
            assert apart or rows * heads > 1 << 20, (heads, rows)
            assert shared <= L.backend_kv8_attn_shared_work(C.byref(c), C.byref(a))


@pytest.mark.parametrize("change", [dict(y=8196), dict(y=8192 + 1024 - 4), dict(y=8192 - 3 * 256 + 4), dict(y=8192 + 2 * 1024 + 1020),
                                    dict(y=8192 + 2 * 600, bf16=1, ld_y=300, ld_x=300), dict(y=8194, bf16=1, rows=1)])
def test_overlapping_rows_are_refused(change):
    """Outputs among the inputs, from their first to their last value."""
    r = subprocess.run([sys.executable, "-c", program(LIN, **change)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1 and "y and x overlap" in r.stderr, r.stderr


@pytest.mark.parametrize("change", [dict(y=8192 + 1024, ld_x=320, ld_y=320), dict(x=8192 + 256, y=8192, ld_x=320, ld_y=320),
                                    dict(y=8192 + 3 * 1024), dict(y=8192 - 3 * 256), dict(y=8192 + 512, bf16=1, ld_x=288 + 32, ld_y=320)])
def test_columns_of_one_array_are_not(change):
    """Inputs and outputs side by side in one array, or right behind each other."""
    r = subprocess.run([sys.executable, "-c", program(LIN, **change)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1 and "has not called backend_init" in r.stderr, r.stderr


def test_rows_that_meet():
    """The check of two sets of rows against every pair of bytes."""
    L = cb.hip()
    L.ct_rows_meet.argtypes, L.ct_rows_meet.restype = [C.c_void_p, C.c_size_t, C.c_size_t] * 2 + [C.c_long], C.c_int
    rng = np.random.default_rng(5)
    seen = [0, 0]
    for _ in range(4000):
        wa, wb, rows = (int(v) for v in rng.integers(1, 9, 3))
        lda, ldb = wa + int(rng.integers(0, 12)), wb + int(rng.integers(0, 12))
        if rng.random() < 0.5:
            lda = ldb = max(lda, ldb)
        a, b = 1000, 1000 + int(rng.integers(-100, 100))
        at = [{p + i * ld + k for i in range(rows) for k in range(w)} for p, ld, w in ((a, lda, wa), (b, ldb, wb))]
        want = bool(at[0] & at[1])
        assert bool(L.ct_rows_meet(a, lda, wa, b, ldb, wb, rows)) == want, (a, lda, wa, b, ldb, wb, rows)
        seen[want] += 1
    assert min(seen) > 500
