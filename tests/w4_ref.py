"""Linear maps with 4-bit weights restated in numpy, in 64 bits, and memory of
the backend's arena for the tests around them."""
import ctypes as C

import numpy as np

import ctbind as cb


class Mem:
    """Pieces of the backend's arena."""

    def __init__(self, hip, floats):
        self.hip = hip
        self.at = hip.backend_arena_alloc(floats)
        self.end = self.at + 4 * floats

    def take(self, nbytes):
        p = self.at
        self.at += (nbytes + 255) // 256 * 256
        assert self.at <= self.end, "test memory exhausted"
        return p

    def write(self, p, a):
        flat = np.ascontiguousarray(a).view(np.uint8).reshape(-1)
        flat = np.concatenate([flat, np.zeros(-len(flat) % 4, np.uint8)]).view(np.float32)
        if flat.size:
            self.hip.backend_htod(p, flat.ctypes.data, flat.size)

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.take(a.nbytes + 16)
        self.write(p, a)
        return p

    def get(self, p, shape, dtype):
        a = np.empty(shape, dtype)
        if a.nbytes:
            self.hip.backend_dtoh(a.ctypes.data, p, a.nbytes)
        return a


def bf16_bits(x):
    """fp32 to bf16 bits, to nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_value(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def pack(codes):
    """Codes [out][in] two a byte, the first in the low bits."""
    c = np.pad(codes, ((0, 0), (0, codes.shape[1] % 2))).astype(np.uint8)
    return c[:, 0::2] | c[:, 1::2] << 4


def wide(x, group, n):
    return np.repeat(x, group, 1)[:, :n]


def values(codes, scale_bits, zeros, group, f16):
    """W in 64 bits."""
    n = codes.shape[1]
    s = scale_bits.view(np.float16).astype(np.float64) if f16 else bf16_value(scale_bits).astype(np.float64)
    z = 8.0 if zeros is None else wide((zeros & 15).astype(np.float64), group, n)
    return (codes.astype(np.float64) - z) * wide(s, group, n)


def quantize(W, group, f16):
    """(codes, scale bits, zeros) by the documented rule, in fp32."""
    out_d, in_d = W.shape
    g = -(-in_d // group)
    p = np.pad(W.astype(np.float32), ((0, 0), (0, g * group - in_d))).reshape(out_d, g, group)
    lo, hi = np.minimum(p.min(2), 0), np.maximum(p.max(2), 0)
    with np.errstate(all="ignore"):
        want = ((hi - lo) / np.float32(15)).astype(np.float32)
        if f16:
            bits = np.minimum(want, np.float32(65504)).astype(np.float16).view(np.uint16)
            s = bits.view(np.float16).astype(np.float32)
        else:
            bits = bf16_bits(np.minimum(want, np.float32(3.3895313892515355e38)))
            s = bf16_value(bits)
        z = np.where(s > 0, np.clip(np.rint(-lo / s), 0, 15), 0).astype(np.float32)
        c = np.where(s[..., None] > 0, np.clip(np.rint(p / s[..., None]) + z[..., None], 0, 15), 0)
    return c.reshape(out_d, -1)[:, :in_d].astype(np.uint8), bits, z.astype(np.uint8)


class Weight:
    """A laid-out weight on the device."""

    def __init__(self, hip, mem, in_d, out_d, group, f16):
        self.hip, self.mem = hip, mem
        self.w = cb.BackendW4(in_d=in_d, out_d=out_d, group=group, scale_f16=int(f16))
        self.h = C.byref(self.w)
        n = hip.backend_w4_floats(self.h)
        self.at = mem.take(4 * n)
        hip.backend_w4_bind(self.h, self.at)

    def load(self, codes, scale_bits, zeros):
        m = self.mem
        self.hip.backend_w4_load(self.h, m.put(pack(codes)), m.put(scale_bits), 0 if zeros is None else m.put(zeros))

    def unpack(self):
        p = self.mem.take(4 * self.w.in_d * self.w.out_d)
        self.hip.backend_w4_unpack(self.h, p)
        return self.mem.get(p, (self.w.out_d, self.w.in_d), np.float32)

    def linear(self, x, bias=None, act=0, scale=0.0, bf16=False, y=None, pad=(0, 0), off=0, behind=0):
        """Device result as fp32 [rows][out_d]; what lies between, before and behind the rows has to stay 55."""
        rows, (px, py) = x.shape[0], pad
        ldx, ldy, m, size = self.w.in_d + px, self.w.out_d + py, self.mem, 2 if bf16 else 4
        fx = np.full(off + rows * ldx + 8, 77.0, np.float32)
        fx[off:off + rows * ldx].reshape(rows, ldx)[:, :self.w.in_d] = x
        fy = np.full(off + (rows + behind) * ldy + 8, 55.0, np.float32)
        if y is not None:
            fy[off:off + rows * ldy].reshape(rows, ldy)[:, :self.w.out_d] = y
        xp, yp = m.put(bf16_bits(fx) if bf16 else fx), m.put(bf16_bits(fy) if bf16 else fy)
        a = cb.BackendW4Linear(y=yp + off * size, x=xp + off * size, ld_y=ldy, ld_x=ldx, bf16=int(bf16), rows=rows,
                               bias=0 if bias is None else m.put(bf16_bits(bias)), act=act, scale=scale)
        self.hip.backend_linear_w4(self.h, C.byref(a))
        got = m.get(yp, fy.shape, np.uint16 if bf16 else np.float32)
        got = bf16_value(got) if bf16 else got
        body = got[off:off + rows * ldy].reshape(rows, ldy)
        assert np.all(got[:off] == 55.0) and np.all(got[off + rows * ldy:] == 55.0) and np.all(body[:, self.w.out_d:] == 55.0)
        return body[:, :self.w.out_d].copy()


def expected(W, x, bias=None, act=0, scale=0.0, y=None):
    """(result, what its tolerance is relative to: the sum of the products' sizes), in 64 bits."""
    v = x.astype(np.float64) @ W.T
    size = np.abs(x).astype(np.float64) @ np.abs(W).T
    if bias is not None:
        v, size = v + bias, size + np.abs(bias)
    if act == cb.W4_SILU:
        with np.errstate(over="ignore"):
            v = v / (1 + np.exp(-v))
    elif act == cb.W4_RELU:
        v = np.maximum(v, 0)
    elif act == cb.W4_ADD:
        v, size = y + scale * v, np.abs(y) + abs(scale) * size
    return v, size


def tolerance(W, x, v, size, bf16):
    """With eps = 2^-24: an input is split to 2^-22 of itself or, of a block of
    128, 2^-38 of its largest, whichever is more (fp32; bf16: exact, or 2^-39).
    A product's sum is rounded once a product in a group (in_d eps at most over
    all, relative to the terms' sizes; the matrix unit adds at least as well as
    one after another), then twice a group, 8 times for the segments, and for the
    bias, the activation (silu: x times the derivative is at most 1.1 in its
    argument, and 4 eps of itself) and the sum: in_d + 32 in all.  bf16: 2^-8 of
    the result on top."""
    eps, in_d = 2.0 ** -24, W.shape[1]
    blocks = [np.abs(x[:, k:k + 128]).max(1, keepdims=True).astype(np.float64) @ np.abs(W[:, k:k + 128]).sum(1, keepdims=True).T
              for k in range(0, in_d, 128)]
    t = 1.1 * ((in_d + 32) * eps + (0 if bf16 else 2.0 ** -22)) * size + 2.0 ** (-39 if bf16 else -38) * sum(blocks)
    return t + 4 * eps * np.abs(v) + (2.0 ** -8 * np.abs(v) if bf16 else 0) + 2.0 ** -120
