"""Linear maps with 4-bit weights on the device against their 64-bit model
(w4_ref.py) — needs an MI355X."""
import ctypes as C

import numpy as np
import pytest

import ctbind as cb
import w4_ref as ref

pytestmark = pytest.mark.gpu


def weight(hip, rng, in_d, out_d, group, f16=False, zeros=True, floats=1 << 23):
    mem = ref.Mem(hip, floats)
    g = -(-in_d // group)
    codes = rng.integers(0, 16, (out_d, in_d)).astype(np.uint8)
    s = (np.exp(0.5 * rng.standard_normal((out_d, g))) / np.sqrt(in_d) / 4).astype(np.float32)
    bits = s.astype(np.float16).view(np.uint16) if f16 else ref.bf16_bits(s)
    z = rng.integers(0, 16, (out_d, g)).astype(np.uint8) if zeros else None
    w = ref.Weight(hip, mem, in_d, out_d, group, f16)
    w.load(codes, bits, z)
    return w, ref.values(codes, bits, z, group, f16)


def inputs(rng, rows, in_d, bf16):
    x = (rng.standard_normal((rows, in_d)) * np.exp(rng.standard_normal((1, in_d)))).astype(np.float32)
    return ref.bf16_value(ref.bf16_bits(x)) if bf16 else x


def check(got, W, x, bf16, what, **kw):
    v, size = ref.expected(W, x, **kw)
    t = ref.tolerance(W, x, v, size, bf16)
    bad = ~(np.abs(got - v) <= t)
    assert not bad.any(), (what, float((np.abs(got - v) / t).max()), np.argwhere(bad)[:4])


SHAPES = [  # in_d, out_d, group
    (1024, 1024, 128), (128, 16, 128), (1, 1, 32), (7, 33, 64), (33, 16, 32), (127, 17, 32), (129, 15, 64),
    (300, 130, 128), (1280, 100, 64), (2047, 65, 32), (4096, 48, 128), (1030, 257, 128)]


@pytest.mark.parametrize("in_d,out_d,group", SHAPES)
@pytest.mark.parametrize("f16,zeros", [(False, True), (True, False), (True, True)])
def test_load_and_unpack(hip, in_d, out_d, group, f16, zeros):
    """Every code, scale and zero point comes back as the value it stands for, exactly."""
    print(f"case: load {in_d} {out_d} {group} f16={f16} zeros={zeros}", flush=True)
    w, W = weight(hip, np.random.default_rng(in_d), in_d, out_d, group, f16, zeros)
    assert np.array_equal(w.unpack().astype(np.float64), W)


@pytest.mark.parametrize("in_d,out_d,group", SHAPES)
@pytest.mark.parametrize("f16", [False, True])
def test_quantize(hip, in_d, out_d, group, f16):
    """The documented rule, bit for bit; values at the scale types' ends, groups
    of zeros, of one sign and of one outlier."""
    print(f"case: quantize {in_d} {out_d} {group} f16={f16}", flush=True)
    rng = np.random.default_rng(out_d)
    W = (rng.standard_normal((out_d, in_d)) * np.exp(2 * rng.standard_normal((out_d, 1)))).astype(np.float32)
    W[0] = 0
    if out_d > 8:
        W[1], W[2], W[3], W[4] = np.abs(W[1]), -np.abs(W[2]), W[3] * 1e-30, W[4] * 1e30
        W[5] = 0
        W[5, in_d // 2] = 3.0
        W[6] = 3.3e38 * np.sign(W[6])
        W[7] *= 1e-6
    W = ref.bf16_value(ref.bf16_bits(W))
    mem = ref.Mem(hip, 1 << 23)
    w = ref.Weight(hip, mem, in_d, out_d, group, f16)
    hip.backend_w4_quantize(w.h, mem.put(ref.bf16_bits(W)))
    assert np.array_equal(w.unpack().astype(np.float64), ref.values(*ref.quantize(W, group, f16), group, f16))


ROWS = [1, 2, 5, 16, 17, 40, 64, 65, 130, 300]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("in_d,out_d,group", SHAPES)
def test_linear(hip, in_d, out_d, group, bf16):
    """Row counts around every tile, with a bias and each activation in turn."""
    print(f"case: linear {in_d} {out_d} {group} bf16={bf16}", flush=True)
    rng = np.random.default_rng(in_d + out_d)
    w, W = weight(hip, rng, in_d, out_d, group, f16=group == 64)
    first = w.mem.at
    for i, rows in enumerate(ROWS):
        w.mem.at = first
        x, act = inputs(rng, rows, in_d, bf16), i % 4
        kw = dict(act=act, bias=ref.bf16_value(ref.bf16_bits(rng.standard_normal(out_d).astype(np.float32))) if i % 3 else None)
        if act == cb.W4_ADD:
            kw |= dict(scale=0.37, y=inputs(rng, rows, out_d, bf16))
        got = w.linear(x, bf16=bf16, behind=2, **kw)
        check(got, W, x, bf16, (rows, act), **kw)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pad,off", [((0, 0), 1), ((1, 3), 0), ((8, 16), 8), ((3, 1), 5)])
def test_strided_rows(hip, pad, off, bf16):
    """Rows apart and off 16 bytes, inputs that end inside a piece of eight."""
    print(f"case: strided {pad} {off} bf16={bf16}", flush=True)
    rng = np.random.default_rng(3)
    for in_d, out_d, rows in ((260, 70, 3), (515, 40, 33), (1024, 64, 150)):
        w, W = weight(hip, rng, in_d, out_d, 64)
        x = inputs(rng, rows, in_d, bf16)
        check(w.linear(x, bf16=bf16, pad=pad, off=off, behind=1), W, x, bf16, (in_d, rows))


@pytest.mark.parametrize("bf16", [False, True])
def test_a_rows_bits_are_its_own(hip, bf16):
    """A row gives the same bits alone, among others, in any place, at every row
    count and over inputs of any length."""
    print(f"case: own bits bf16={bf16}", flush=True)
    rng = np.random.default_rng(8)
    for in_d, out_d, group in ((1024, 528, 128), (2200, 96, 32), (100, 4096, 64)):
        w, _ = weight(hip, rng, in_d, out_d, group, floats=1 << 24)
        x = inputs(rng, 700, in_d, bf16)
        first = w.mem.at
        whole = w.linear(x, bf16=bf16)
        for a, b in ((0, 1), (5, 6), (3, 7), (0, 16), (10, 43), (1, 65), (100, 228), (7, 400)):
            w.mem.at = first
            assert np.array_equal(w.linear(x[a:b], bf16=bf16).view(np.uint32), whole[a:b].view(np.uint32)), (in_d, a, b)


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_special_inputs(hip, rows):
    """Zero rows, tiny and huge ones, blocks of very different sizes beside each
    other; a row with an infinity or NaN touches no other row."""
    print(f"case: special inputs rows={rows}", flush=True)
    rng = np.random.default_rng(9)
    for bf16 in (False, True):
        w, W = weight(hip, rng, 640, 80, 64)
        x = inputs(rng, rows, 640, bf16)
        q = lambda v: ref.bf16_value(ref.bf16_bits(v.astype(np.float32)))  # noqa: E731
        x[0, 128:256] = q(x[0, 128:256] * 1e12)
        x[0, 256:384] = q(x[0, 256:384] * 1e-12)
        if rows > 8:
            x[1] = 0
            x[2] = q(x[2] * 1e-30)
            x[3] = q(x[3] * 1e-37)
            x[4] = q(x[4] * 1e34)
            x[5, 10:] = 0
            x[6, 3], x[7, 639], x[8, 200] = np.inf, np.nan, -np.inf
        got = w.linear(x, bf16=bf16)
        fine = np.isfinite(x).all(1)
        check(got[fine], W, x[fine], bf16, (rows, bf16))
        assert not np.isfinite(got[~fine]).any()
        if rows > 8:
            assert np.all(got[1] == 0)
            relu = w.linear(x, bf16=bf16, act=cb.W4_RELU)
            assert np.isnan(relu[7]).all()


def test_large_offsets(hip):
    """A weight of 2^31 values, the most there may be: its last codes lie past 2^30 bytes."""
    print("case: large", flush=True)
    rng = np.random.default_rng(12)
    in_d, out_d = 1 << 11, 1 << 20
    mem = ref.Mem(hip, 600_000_000)
    w = ref.Weight(hip, mem, in_d, out_d, 128, False)
    part = 1 << 13                            # the rows of W repeat
    codes = rng.integers(0, 16, (part, in_d)).astype(np.uint8)
    bits = ref.bf16_bits(np.exp(rng.standard_normal((part, in_d // 128))).astype(np.float32))
    z = rng.integers(0, 16, (part, in_d // 128)).astype(np.uint8)
    cp, sp, zp = (mem.put(np.tile(v, (out_d // part, 1))) for v in (ref.pack(codes), bits, z))
    hip.backend_w4_load(w.h, cp, sp, zp)
    x = inputs(rng, 2, in_d, False)
    got = w.linear(x)
    v, size = ref.expected(ref.values(codes, bits, z, 128, False), x)
    t = ref.tolerance(ref.values(codes, bits, z, 128, False), x, v, size, False)
    for k in (0, 1, out_d // part - 1):
        assert np.all(np.abs(got[:, k * part:(k + 1) * part] - v) <= t)
    assert np.array_equal(got.reshape(2, -1, part), np.repeat(got[:, None, :part], out_d // part, 1))


MANY = [  # in_d, out_d, group, rows: tiles of 64 rows, by 128 outputs or, the last three of them, by 256
    (1024, 528, 128, 2300), (129, 20, 64, 11300), (128, 130, 32, 5700), (300, 1030, 64, 1300), (2200, 1030, 32, 1345),
    (129, 4100, 32, 1000), (1030, 2600, 64, 1290), (640, 25700, 128, 100)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("in_d,out_d,group,rows", MANY)
def test_many_rows(hip, in_d, out_d, group, rows, bf16):
    """Enough rows and outputs for the kernel of 64 rows; the last rows, outputs
    and inputs end inside its tiles.  The same bits as of few rows."""
    print(f"case: many rows {in_d} {out_d} {group} {rows} bf16={bf16}", flush=True)
    rng = np.random.default_rng(rows)
    w, W = weight(hip, rng, in_d, out_d, group, f16=group == 32, floats=1 << 25)
    x = inputs(rng, rows, in_d, bf16)
    first = w.mem.at
    whole = w.linear(x, bf16=bf16, pad=(1, 3), off=1, behind=2)
    some = np.unique(np.concatenate([np.arange(70), rng.integers(0, rows, 100), np.arange(rows - 70, rows)]) % rows)
    check(whole[some], W, x[some], bf16, rows)
    for a, b in ((0, 5), (61, 77), (rows - 30, rows)):
        w.mem.at = first
        assert np.array_equal(w.linear(x[a:b], bf16=bf16).view(np.uint32), whole[a:b].view(np.uint32)), (a, b)
    for act in (cb.W4_SILU, cb.W4_ADD):
        w.mem.at = first
        kw = dict(act=act, bias=ref.bf16_value(ref.bf16_bits(rng.standard_normal(out_d).astype(np.float32))), scale=-1.5)
        if act == cb.W4_ADD:
            kw["y"] = inputs(rng, rows, out_d, bf16)
        got = w.linear(x, bf16=bf16, **kw)
        if act == cb.W4_ADD:
            kw["y"] = kw["y"][some]
        check(got[some], W, x[some], bf16, (rows, act), **kw)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("in_d,out_d,group,rows", [
    (260, 17000, 32, 1), (260, 17000, 64, 3), (520, 17000, 128, 7), (260, 17000, 64, 13), (2048, 16500, 64, 13), (2300, 16450, 128, 6),
    (7, 17000, 128, 2), (130, 4200, 64, 200), (130, 4200, 32, 190), (1100, 4200, 128, 65), (96, 4100, 32, 260)])
def test_many_outputs(hip, in_d, out_d, group, rows, bf16):
    """Inputs kept in LDS while a workgroup goes from outputs to outputs, one tile and two at a time."""
    print(f"case: many outputs {in_d} {out_d} {group} {rows} bf16={bf16}", flush=True)
    rng = np.random.default_rng(in_d + rows)
    w, W = weight(hip, rng, in_d, out_d, group, f16=group == 64, floats=1 << 25)
    x, first = inputs(rng, rows, in_d, bf16), w.mem.at
    whole = w.linear(x, bf16=bf16, pad=(1, 3), off=3, behind=2)
    check(whole, W, x, bf16, rows)
    w.mem.at = first
    last = w.linear(x[-1:], bf16=bf16)
    assert np.array_equal(last.view(np.uint32), whole[-1:].view(np.uint32))
    kw = dict(act=cb.W4_ADD, bias=ref.bf16_value(ref.bf16_bits(rng.standard_normal(out_d).astype(np.float32))), scale=0.3,
              y=inputs(rng, rows, out_d, bf16))
    check(w.linear(x, bf16=bf16, **kw), W, x, bf16, (rows, "add"), **kw)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_long_inputs(hip, group, bf16):
    """Inputs that do not fit LDS, one, two and four tiles of outputs together, the last ones fewer."""
    print(f"case: long inputs {group} bf16={bf16}", flush=True)
    rng = np.random.default_rng(group)
    in_d, out_d = 4300, 1030
    w, W = weight(hip, rng, in_d, out_d, group, f16=group == 64, floats=1 << 25)
    x = inputs(rng, 700, in_d, bf16)
    first, one = w.mem.at, None
    for i, rows in enumerate((700, 300, 70, 33, 17, 4)):
        w.mem.at = first
        kw = dict(act=i % 4, bias=ref.bf16_value(ref.bf16_bits(rng.standard_normal(out_d).astype(np.float32))))
        if kw["act"] == cb.W4_ADD:
            kw |= dict(scale=0.7, y=inputs(rng, rows, out_d, bf16))
        got = w.linear(x[:rows], bf16=bf16, pad=(3, 1), off=i, behind=1, **kw)
        check(got, W, x[:rows], bf16, (rows, kw["act"]), **kw)
        plain = w.linear(x[:rows], bf16=bf16)
        one = plain if one is None else one
        assert np.array_equal(plain.view(np.uint32), one[:rows].view(np.uint32)), rows


@pytest.mark.parametrize("ld", [(1 << 24) - 1, (1 << 24) + 4])
def test_rows_far_apart(hip, ld):
    """Inputs whose offsets pass 32 bits, and nearly do."""
    print(f"case: far apart {ld}", flush=True)
    rng = np.random.default_rng(14)
    for in_d, out_d in ((200, 22600), (200, 100)):
        w, W = weight(hip, rng, in_d, out_d, 64, floats=66 * ld + (1 << 25))
        x, at = inputs(rng, 66, in_d, False), w.mem.take(4 * 66 * ld)
        for i, row in enumerate(x):
            w.mem.write(at + 4 * i * ld, row)
        y = w.mem.take(4 * 66 * out_d)
        a = cb.BackendW4Linear(y=y, x=at, ld_y=out_d, ld_x=ld, rows=66)
        hip.backend_linear_w4(w.h, C.byref(a))
        check(w.mem.get(y, (66, out_d), np.float32), W, x, False, ld)


@pytest.mark.parametrize("rows", [1 << 24, 70000])
def test_the_most_rows(hip, rows):
    """Inputs shorter than a tile and so many rows that they take more than 65535 workgroups."""
    print(f"case: most rows {rows}", flush=True)
    rng = np.random.default_rng(15)
    w, W = weight(hip, rng, 3, 2, 32, floats=1 << 27)
    x = inputs(rng, rows, 3, False)
    got = w.linear(x)
    check(got, W, x, False, rows)


def test_nothing_to_do_and_captured(hip):
    """No rows: y stays.  Captured once and replayed, with eager calls between:
    the same bits, from the inputs of the moment."""
    print("case: captured", flush=True)
    rng = np.random.default_rng(13)
    w, W = weight(hip, rng, 1024, 300, 128)
    mem = w.mem
    y = mem.put(np.full((40, 300), 55.0, np.float32))
    xs = [inputs(rng, 40, 1024, False) for _ in range(3)]
    xp = mem.put(xs[0])
    a = cb.BackendW4Linear(y=y, x=xp, ld_y=300, ld_x=1024, rows=0)
    hip.backend_linear_w4(w.h, C.byref(a))
    assert np.all(mem.get(y, (40, 300), np.float32) == 55.0)
    a.rows = 40
    want = []
    for x in xs:
        mem.write(xp, x)
        hip.backend_linear_w4(w.h, C.byref(a))
        want.append(mem.get(y, (40, 300), np.float32))
        check(want[-1], W, x, False, "eager")
    tag = 1
    assert hip.backend_graph_replay(tag, 7, 7, 7) == 0
    hip.backend_graph_begin_capture(tag)
    hip.backend_linear_w4(w.h, C.byref(a))
    hip.backend_graph_end_capture(tag, 7, 7, 7)
    for i in (1, 0, 2, 2, 1):
        mem.write(xp, xs[i])
        mem.write(y, np.zeros((40, 300), np.float32))
        assert hip.backend_graph_replay(tag, 7, 7, 7) == 1
        assert np.array_equal(mem.get(y, (40, 300), np.float32).view(np.uint32), want[i].view(np.uint32))
        hip.backend_linear_w4(w.h, C.byref(a))
        assert np.array_equal(mem.get(y, (40, 300), np.float32).view(np.uint32), want[i].view(np.uint32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("in_d,out_d,group,rows", [
    (1024, 48, 128, 1), (640, 80, 32, 20), (4300, 1030, 64, 33), (260, 17000, 64, 3), (300, 1030, 64, 1300), (640, 4100, 128, 700)])
def test_scales_and_inputs_of_any_size(hip, in_d, out_d, group, rows, bf16):
    """Scales up to the type's largest value over inputs so small that the result
    is finite, the smallest ones over large inputs, and both beside scales of 1."""
    print(f"case: scales of any size {in_d} {out_d} {group} {rows} bf16={bf16}", flush=True)
    rng = np.random.default_rng(rows)
    mem = ref.Mem(hip, 1 << 25)
    w = ref.Weight(hip, mem, in_d, out_d, group, False)
    g, first = -(-in_d // group), mem.at
    for top, low in ((127.99, -60), (127.99, -100), (-133, 100), (-110, 80), (0, 106), (0, -80)):
        mem.at = first
        codes, z = rng.integers(0, 16, (out_d, in_d)).astype(np.uint8), rng.integers(0, 16, (out_d, g)).astype(np.uint8)
        bits = ref.bf16_bits((2.0 ** (top - 3 * rng.random((out_d, g)) * (top > 0))).astype(np.float32))
        if top in (127.99, -110):
            some = rng.random((out_d, g)) < 0.5
            bits[some] = ref.bf16_bits(np.ones(some.sum(), np.float32))
        w.load(codes, bits, z)
        W = ref.values(codes, bits, z, group, False)
        x = (inputs(rng, rows, in_d, bf16).astype(np.float64) * 2.0 ** low).astype(np.float32)
        some = np.unique(np.concatenate([np.arange(min(rows, 40)), np.arange(max(rows - 40, 0), rows)]))
        got = w.linear(x, bf16=bf16)
        assert np.isfinite(got).all(), (top, low)
        check(got[some], W, x[some], bf16, (top, low))


def test_quantized_weights_of_any_size(hip):
    """Weights up to the largest finite one through quantising and a product."""
    print("case: quantized, any size", flush=True)
    rng = np.random.default_rng(16)
    for size, low in ((3.3e38, 1e-12), (1e34, 1e-20), (1e-34, 1e20)):
        W = np.clip(rng.standard_normal((48, 512)) * size, -3.38e38, 3.38e38).astype(np.float32)
        mem = ref.Mem(hip, 1 << 22)
        w = ref.Weight(hip, mem, 512, 48, 64, False)
        hip.backend_w4_quantize(w.h, mem.put(ref.bf16_bits(W)))
        x = (inputs(rng, 5, 512, False) * np.float32(low)).astype(np.float32)
        check(w.linear(x), w.unpack().astype(np.float64), x, False, size)


@pytest.mark.parametrize("rows", [9, 200])
def test_what_relu_leaves_of_infinite_inputs(hip, rows):
    """A row with an infinity: a finite output is the zero of a product of
    -infinity, of bf16 rows; everything else is not finite."""
    print(f"case: relu of infinities rows={rows}", flush=True)
    rng = np.random.default_rng(17)
    for bf16 in (False, True):
        w, W = weight(hip, rng, 640, 80, 64)
        x = inputs(rng, rows, 640, bf16)
        x[6, 3], x[7, 639], x[8, 200] = np.inf, np.nan, -np.inf
        plain, relu, silu = (w.linear(x, bf16=bf16, act=a)[6:9] for a in (cb.W4_STORE, cb.W4_RELU, cb.W4_SILU))
        assert not np.isfinite(plain).any() and np.isnan(plain[1]).all()
        assert np.array_equal(relu == 0, plain == -np.inf) and not np.isfinite(relu[relu != 0]).any()
        assert (bf16 or np.isnan(relu).all()) and not np.isfinite(silu).any()
