"""The paged 8-bit key/value cache restated in numpy, in 64 bits: rounding to
e4m3 with power-of-two scales, the page book-keeping, and attention.

Cache is the model of a cache's whole state; Dev holds the same state in
device memory behind the backend_kv8_* calls.
"""
import ctypes as C

import numpy as np

import ctbind as cb

# the 256 e4m3 values: sign, 4 bits of exponent (bias 7), 3 of fraction; 0x7f is NaN
_c = np.arange(256)
_e, _f = (_c >> 3) & 15, _c & 7
E4M3 = np.where(_e > 0, (8 + _f) * 2.0 ** (_e - 10), _f * 2.0 ** -9) * np.where(_c >= 128, -1.0, 1.0)
E4M3[[0x7F, 0xFF]] = np.nan
_POS = E4M3[:0x7F]                       # ascending
_MID = (_POS[1:] + _POS[:-1]) / 2


def to_codes(x):
    """Nearest code of each value (64 bits), ties to the even code, clamped at +-448; NaN is 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    i = np.searchsorted(_MID, np.nan_to_num(a), side="left")     # a <= mid: the lower one
    tie = (i < len(_MID)) & (np.nan_to_num(a) == _MID[np.minimum(i, len(_MID) - 1)])
    i = np.where(tie & (i % 2 == 1), i + 1, i)
    code = np.where(np.isnan(x), 0x7F, i | np.where(np.signbit(x), 128, 0))
    return code.astype(np.uint8)


def same_codes(a, b):
    """Equal codes, any NaN code equal to any other."""
    na, nb = (a & 0x7F) == 0x7F, (b & 0x7F) == 0x7F
    return np.array_equal(na, nb) and np.array_equal(a[~na], b[~nb])


def need_exp(x):
    """The smallest e >= -100 with every finite |x| <= 448 * 2^e."""
    a = np.abs(np.asarray(x, np.float64))
    a = a[np.isfinite(a)].max(initial=0.0)
    e = -100
    while 448.0 * 2.0 ** e < a:
        e += 1
    return e


class Cache:
    def __init__(self, layers, pages, P, kv, D, seqs, width):
        self.dims = (layers, pages, P, kv, D, seqs, width)
        self.k = np.zeros((layers, pages, kv, P, D), np.uint8)
        self.v = np.zeros_like(self.k)
        self.ks = np.zeros((layers, pages, kv), np.float32)
        self.vs = np.zeros_like(self.ks)
        self.table = np.full((seqs, width), -1, np.int32)
        self.len = np.zeros(seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.rows = np.zeros(seqs + 1, np.int32)
        self.status = 0

    @property
    def P(self):
        return self.dims[2]

    def free_pages(self):
        return [int(p) for p in np.flatnonzero(self.refs == 0)]

    def reserve(self, add):
        P, width = self.P, self.dims[6]
        add = [int(a) for a in add]
        bad = (4 if any(a < 0 for a in add) else 0) | (2 if any(int(n) + max(a, 0) > P * width for n, a in zip(self.len, add)) else 0)
        need = [-(-(int(n) + max(a, 0)) // P) - -(-int(n) // P) for n, a in zip(self.len, add)]
        free = self.free_pages()
        if not bad and sum(need) > len(free):
            bad = 1
        if bad:
            self.rows[:] = 0
            self.status |= bad
            return
        for s, (n, a) in enumerate(zip(need, add)):
            at = -(-int(self.len[s]) // P)
            for j in range(n):
                p = free.pop(0)
                self.table[s, at + j] = p
                self.refs[p] = 1
            self.len[s] += a
        self.rows[:] = np.concatenate([[0], np.cumsum(add)])

    def append(self, layer, k, v, rows, n_rows):
        """k, v: [n_rows][kv][D] as the kernel reads them."""
        _, pages, P, kv, D, seqs, width = self.dims
        for s in range(seqs):
            r0, r1, n = int(rows[s]), int(rows[s + 1]), int(self.len[s])
            if r0 < 0 or r1 <= r0 or r1 > n_rows:
                continue
            pos = n - (r1 - r0)
            todo = [(pos + i, r0 + i) for i in range(r1 - r0) if 0 <= pos + i < width * P]
            for j in sorted({p // P for p, _ in todo}):
                page = int(self.table[s, j])
                if not 0 <= page < pages or self.refs[page] > 1:
                    continue
                mine = [(p % P, r) for p, r in todo if p // P == j]
                a = mine[0][0]
                for x, pool, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                    for h in range(kv):
                        e = need_exp(x[[r for _, r in mine], h])
                        now = 2.0 ** e
                        if a:
                            was = float(scale[layer, page, h])
                            now = max(was, now)
                            if was < now:
                                pool[layer, page, h, :a] = to_codes(E4M3[pool[layer, page, h, :a]] * (was / now))
                        scale[layer, page, h] = now
                        for t, r in mine:
                            pool[layer, page, h, t] = to_codes(x[r, h].astype(np.float64) / now)

    def _give(self, p):
        if 0 <= p < self.dims[1]:
            self.refs[p] -= 1

    def fork(self, dst, src):
        pages, P, seqs = self.dims[1], self.P, self.dims[5]
        if (any(not 0 <= x < seqs for x in list(dst) + list(src)) or len(set(dst)) < len(dst)):
            self.status |= 4
            return
        free = self.free_pages()
        was, lens = self.table.copy(), self.len.copy()
        moves = [(d, s) for d, s in zip(dst, src) if d != s]
        need = [lens[s] % P != 0 and 0 <= was[s, lens[s] // P] < pages for _, s in moves]
        if sum(need) > len(free):
            self.status |= 1
            return
        for (d, s), n in zip(moves, need):
            used = -(-int(lens[s]) // P)
            row = np.full_like(was[s], -1)
            row[:used] = was[s, :used]
            for j in range(used):
                if n and j == lens[s] // P:
                    p, old = free.pop(0), row[j]
                    for x in (self.k, self.v, self.ks, self.vs):
                        x[:, p] = x[:, old]
                    row[j] = p
                    self.refs[p] = 1
                elif 0 <= row[j] < pages:
                    self.refs[row[j]] += 1
            self.table[d] = row
            self.len[d] = lens[s]
        for d, _ in moves:
            for p in was[d]:
                self._give(p)

    def free(self, seqs):
        if any(not 0 <= s < self.dims[5] for s in seqs):
            self.status |= 4
            return
        for s in set(seqs):
            for p in self.table[s]:
                self._give(p)
            self.table[s] = -1
            self.len[s] = 0

    def trim(self, window, sinks):
        P = self.P
        for s in range(self.dims[5]):
            for j in range(self.dims[6]):
                # the row at position len sees token t if t > len - window or t < sinks
                if j * P >= sinks and (j + 1) * P - 1 <= self.len[s] - window and self.table[s, j] >= 0:
                    self._give(self.table[s, j])
                    self.table[s, j] = -1

    def compact(self):
        live = [int(p) for p in np.flatnonzero(self.refs)]
        m = len(live)
        holes = [p for p in range(m) if self.refs[p] == 0]
        to = dict(zip([p for p in live if p >= m], holes))
        for a, b in to.items():
            for x in (self.k, self.v, self.ks, self.vs):
                x[:, b] = x[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = np.array([[to.get(int(p), p) for p in r] for r in self.table], np.int32)

    def attend(self, layer, q, heads, scale, causal, window, sinks, rows, n_rows, cap=None):
        """(o, vmax, smax): rows [n_rows][heads][D] in 64 bits (NaN-filled where no
        sequence has the row), the largest |v| a row weighs and the largest
        scale * sum |q_d k_d| among its scores."""
        _, pages, P, kv, D, seqs, width = self.dims
        cap = width * P if not cap else min(cap, width * P)
        out = np.full((n_rows, heads, D), np.nan)
        vmax, smax = np.zeros((n_rows, heads, 1)), np.zeros((n_rows, heads, 1))
        for s in range(seqs):
            r0, r1, n = int(rows[s]), int(rows[s + 1]), max(int(self.len[s]), 0)
            if r0 < 0 or r1 <= r0 or r1 > n_rows:
                continue
            j = np.arange(min(n, cap))
            page = self.table[s, j // P] if len(j) else np.zeros(0, np.int32)
            there = (page >= 0) & (page < pages)
            pg, tk = np.where(there, page, 0), j % P
            K = E4M3[self.k[layer, pg, :, tk]] * self.ks[layer, pg][..., None].astype(np.float64)
            V = E4M3[self.v[layer, pg, :, tk]] * self.vs[layer, pg][..., None].astype(np.float64)
            for r in range(r0, r1):
                p = n - (r1 - r0) + (r - r0)
                see = there.copy()
                if causal:
                    see &= j <= p
                if window:
                    see &= (j > p - window) | (j < sinks)
                if not see.any():
                    out[r] = 0.0
                    continue
                for h in range(heads):
                    g = h // (heads // kv)
                    with np.errstate(all="ignore"):
                        sc = K[see, g] @ q[r, h].astype(np.float64) * scale
                        smax[r, h] = (np.abs(K[see, g]) @ np.abs(q[r, h].astype(np.float64))).max() * scale
                        w = np.exp(sc - sc.max())
                        out[r, h] = (w / w.sum()) @ V[see, g]
                        vmax[r, h] = np.nanmax(np.abs(V[see, g]))
        return out, vmax, smax


def bf16_bits(x):
    """fp32 to bf16 bits, to nearest even (finite values, infinities, NaN)."""
    u = np.asarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_value(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Dev:
    """A cache in device memory, bound in the backend's arena, with what the calls around it need."""

    def __init__(self, hip, layers, pages, P, kv, D, seqs, width, extra=1 << 22):
        self.hip = hip
        self.c = cb.BackendKv8(layers=layers, pages=pages, page_tokens=P, kv_heads=kv, head_dim=D, seqs=seqs,
                               table_w=width)
        self.h = C.byref(self.c)
        n = hip.backend_kv8_floats(self.h)
        self.base = hip.backend_arena_alloc(n + extra)
        self.at, self.end = self.base + (n + 63) // 64 * 256, self.base + (n + extra) * 4
        hip.backend_kv8_bind(self.h, self.base)
        self.model = Cache(layers, pages, P, kv, D, seqs, width)
        for name, x in (("k", self.model.k), ("v", self.model.v), ("kscale", self.model.ks), ("vscale", self.model.vs)):
            self.write(getattr(self.c, name), x)

    def take(self, nbytes):
        p = self.at
        self.at += (nbytes + 255) // 256 * 256
        assert self.at <= self.end, "test memory exhausted"
        return p

    def write(self, ptr, a):
        a = np.ascontiguousarray(a)
        flat = a.view(np.uint8).reshape(-1)
        if len(flat) % 4:
            flat = np.concatenate([flat, np.zeros(-len(flat) % 4, np.uint8)])
        flat = flat.view(np.float32)
        self.hip.backend_htod(ptr, flat.ctypes.data, flat.size)

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.take(a.nbytes + 16)
        self.write(p, a)
        return p

    def get(self, ptr, shape, dtype):
        a = np.empty(shape, dtype)
        if a.nbytes:
            self.hip.backend_dtoh(a.ctypes.data, ptr, a.nbytes)
        return a

    def ints(self, v):
        return self.put(np.asarray(v, np.int32))

    def push(self):
        """Writes the model's state to the device."""
        m = self.model
        for name, x in (("k", m.k), ("v", m.v), ("kscale", m.ks), ("vscale", m.vs), ("table", m.table),
                        ("len", m.len), ("refs", m.refs), ("rows", m.rows)):
            self.write(getattr(self.c, name), x)

    def state(self):
        m = self.model
        return {"k": self.get(self.c.k, m.k.shape, np.uint8), "v": self.get(self.c.v, m.v.shape, np.uint8),
                "ks": self.get(self.c.kscale, m.ks.shape, np.float32), "vs": self.get(self.c.vscale, m.vs.shape, np.float32),
                **self.book()}

    def book(self):
        m = self.model
        return {"table": self.get(self.c.table, m.table.shape, np.int32), "len": self.get(self.c.len, m.len.shape, np.int32),
                "refs": self.get(self.c.refs, m.refs.shape, np.int32),
                "rows": self.get(self.c.rows, m.rows.shape, np.int32)}

    def check_book(self, what=""):
        got, m = self.book(), self.model
        for n in ("table", "len", "refs", "rows"):
            assert np.array_equal(got[n], getattr(m, n)), (what, n, got[n], getattr(m, n))
        flags = self.hip.backend_kv8_status(self.h)
        assert flags == m.status, (what, flags, m.status)
        m.status = 0

    def check(self, what=""):
        self.check_book(what)
        got, m = self.state(), self.model
        for n in ("k", "v"):
            assert same_codes(got[n], getattr(m, n)), (what, n)
        for n in ("ks", "vs"):
            assert np.array_equal(got[n], getattr(m, n)), (what, n)

    # the calls, on the device and in the model
    def reserve(self, add):
        self.hip.backend_kv8_reserve(self.h, self.ints(add))
        self.model.reserve(add)

    def append(self, layer, k, v, bf16=False, rows=None, pad=0, off=0):
        """k, v fp32 [n][kv][D] (representable in bf16 if bf16); pad: values between rows; off: values before the first."""
        n, kv, D = k.shape
        ld = kv * D + pad
        ptr = []
        for x in (k, v):
            flat = np.full(off + n * ld + 8, 77.0, np.float32)
            flat[off:off + n * ld].reshape(n, ld)[:, :kv * D] = x.reshape(n, -1)
            ptr.append(self.put(bf16_bits(flat) if bf16 else flat) + off * (2 if bf16 else 4))
        r = self.model.rows if rows is None else np.asarray(rows, np.int32)
        self.hip.backend_kv8_append(self.h, layer, ptr[0], ptr[1], ld, int(bf16), self.c.rows if rows is None else self.ints(r), n)
        self.model.append(layer, k, v, r, n)

    def attn(self, layer, q, heads, scale=None, causal=True, window=0, sinks=0, bf16=False, rows=None, max_rows=None,
             max_len=0, pad=0, off=0, fill=None):
        """Device result [n][heads][D] as fp32; rows of no sequence hold `fill` (default 55)."""
        n, D = q.shape[0], q.shape[2]
        ld, size = heads * D + pad, 2 if bf16 else 4
        flat = np.full(off + n * ld + 8, 77.0, np.float32)
        flat[off:off + n * ld].reshape(n, ld)[:, :heads * D] = q.reshape(n, -1)
        ofl = np.full(flat.shape, 55.0, np.float32)
        qp, op = self.put(bf16_bits(flat) if bf16 else flat), self.put(bf16_bits(ofl) if bf16 else ofl)
        r = self.model.rows if rows is None else np.asarray(rows, np.int32)
        a = cb.BackendKv8Attn(out=op + off * size, q=qp + off * size, ld_out=ld, ld_q=ld, bf16=int(bf16), heads=heads,
                              scale=scale or D ** -0.5, causal=int(causal), window=window, sinks=sinks,
                              rows=self.c.rows if rows is None else self.ints(r), n_rows=n,
                              max_rows=max_rows or max(1, int(np.diff(r).max())), max_len=max_len)
        w = self.hip.backend_kv8_attn_work(self.h, C.byref(a))
        a.work = self.take(w * 4 + 16)
        self.hip.backend_kv8_attn(self.h, layer, C.byref(a))
        got = self.get(op, flat.shape, np.uint16 if bf16 else np.float32)
        got = bf16_value(got) if bf16 else got
        body = got[off:off + n * ld].reshape(n, ld)
        assert np.all(got[:off] == 55.0) and np.all(got[off + n * ld:] == 55.0) and np.all(body[:, heads * D:] == 55.0)
        return body[:, :heads * D].reshape(n, heads, D).copy()


def tolerance(o, vmax, smax, bf16, D):
    """How far a row may be off.  With eps = 2^-24 (fp32's half step): a score
    is a sum of D products whose terms add up to at most smax, rounded D + 8
    times (the products' sum, the split of q, the scaling): d = (D + 8) eps
    smax, in the exponent; 8 eps more for exp2 and the running maximum's
    rescaling.  Each weight and their sum are off by that much, so o by twice
    it times vmax, and by 2^-20 vmax for the sums over tokens in units of a
    32-key step, the join and the division.  bf16: each weight is also rounded
    to f16 (2^-11), and o to bf16 (2^-8)."""
    eps = 2.0 ** -24
    d = (D + 8) * eps * smax + 8 * eps
    t = (2 * d + 2.0 ** -20) * vmax
    return t + (2.0 ** -11 * vmax + 2.0 ** -8 * np.abs(o) if bf16 else 0.0)
