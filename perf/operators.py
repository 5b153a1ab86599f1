"""The operators around a paged key/value cache held in 8 bits, as timed cases.

The cache keeps K and V as e4m3 codes in pages of P tokens, pools
[layer][page][kv head][token][head dim], with one power-of-two scale for each
page and kv head; a table gives each sequence's pages, and refs counts the
table entries that hold a page (0: free).  The cases:

  append   new K/V rows of a step or a prompt rounded into their pages
  attend   softmax attention of new query rows over the pages: single tokens,
           several rows, whole prompts; grouped heads; a sliding window with
           first tokens that stay visible
  fork     sequences that take over other sequences' pages (beams)
  compact  the pages in use moved to the front of the pool

own = False computes each in its plain form; own = True makes the calls a
program makes of the library.
"""
import ctypes as C
import math
import os
import random
import sys

import torch

own = False

E4M3_MAX = 448.0
MIN_EXP = -100          # smallest exponent of a scale
CHUNK = 1 << 27         # values made at once when a pool is filled


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # The batched decode loop of one layer: a token of each of 64 requests at
        # its own position, the model's 8 heads of 128.
        {"name": "append_step_64", "kind": "append", "seqs": 64, "old": 1000, "new": 1, "kv": 8, "dim": 128,
         "page": 64, "bf16": False},
        # Cross-attention keys and values of a batch of 24 clips up to 30 s,
        # written once when the clips have been encoded.
        {"name": "append_clips_24", "kind": "append", "seqs": 24, "old": 0, "new": 376, "kv": 8, "dim": 128,
         "page": 32, "bf16": False},
        # Long prompts entering the cache in one go.
        {"name": "append_prompts_8", "kind": "append", "seqs": 8, "old": 0, "new": 12000, "kv": 8, "dim": 128,
         "page": 128, "bf16": True},
        # One token of one clip over its 376 encoder frames: the smallest call,
        # where latency counts.
        {"name": "attend_clip", "kind": "attend", "seqs": 1, "len": 376, "rows": 1, "heads": 8, "kv": 8, "dim": 128,
         "page": 64, "causal": False, "window": 0, "sinks": 0, "bf16": False},
        # One token of each of 64 requests over its own text so far.
        {"name": "attend_step_64", "kind": "attend", "seqs": 64, "len": 1000, "rows": 1, "heads": 8, "kv": 8,
         "dim": 128, "page": 64, "causal": True, "window": 0, "sinks": 0, "bf16": False},
        # One token of each of 32 long documents, four query heads to a key head:
        # the largest decode step.
        {"name": "attend_long_32", "kind": "attend", "seqs": 32, "len": 30000, "rows": 1, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "causal": True, "window": 0, "sinks": 0, "bf16": True},
        # Streams that never end: the last 1000 tokens and the first 4, small
        # pages, heads of 64.
        {"name": "attend_window_48", "kind": "attend", "seqs": 48, "len": 9000, "rows": 1, "heads": 16, "kv": 4,
         "dim": 64, "page": 16, "causal": True, "window": 1000, "sinks": 4, "bf16": True},
        # Whole prompts of mixed lengths.
        {"name": "attend_prompts_6", "kind": "attend", "seqs": 6, "len": 2500, "rows": 2500, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "causal": True, "window": 0, "sinks": 0, "bf16": True},
        # The next piece of three prompts that enter in pieces, over what they
        # hold already, in fp32.
        {"name": "attend_pieces_3", "kind": "attend", "seqs": 3, "len": 7001, "rows": 201, "heads": 8, "kv": 8,
         "dim": 128, "page": 32, "causal": True, "window": 0, "sinks": 0, "bf16": False},
        # A beam search step of one clip: five hypotheses continue from their
        # parents, small pages.
        {"name": "fork_beams_5", "kind": "fork", "seqs": 5, "beam": 5, "len": 200, "layers": 8, "kv": 8, "dim": 128,
         "page": 16},
        # The same for 32 clips with 4 hypotheses each.
        {"name": "fork_beams_128", "kind": "fork", "seqs": 128, "beam": 4, "len": 1000, "layers": 8, "kv": 8,
         "dim": 128, "page": 64},
        # A pool two thirds empty, with its pages spread all over, drawn together
        # before its upper part is given back.
        {"name": "compact_900", "kind": "compact", "seqs": 40, "len": 1000, "pages": 2400, "layers": 8, "kv": 8,
         "dim": 128, "page": 32},
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "fork", "compact"])
    kv, dim, page = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if kind == "append":
        new = rng.choice([1, 1, _log(rng, 2, 12000)])
        seqs = _log(rng, 1, max(2, min(64, 60000 // new)))
        return {"kind": kind, "seqs": seqs, "old": rng.choice([0, _log(rng, 1, 4000)]), "new": new, "kv": kv,
                "dim": dim, "page": page, "bf16": rng.random() < 0.5}
    if kind == "attend":
        shape = rng.choice(["one", "one", "few", "prompt"])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        if shape == "prompt":
            n = _log(rng, 20, 2500)
            length, seqs = n + rng.choice([0, _log(rng, 1, 2000)]), _log(rng, 1, 6)
        else:
            n = 1 if shape == "one" else rng.randint(2, 12)
            length = max(n, _log(rng, 1, 30000))
            seqs = _log(rng, 1, max(2, min(64, 900000 // length)))
        window = rng.choice([0, 0, _log(rng, 1, 2000)])
        causal = window > 0 or rng.random() < 0.8
        return {"kind": kind, "seqs": seqs, "len": length, "rows": n, "heads": kv * group, "kv": kv, "dim": dim,
                "page": page, "causal": causal, "window": window, "sinks": rng.randint(0, 70) if window else 0,
                "bf16": rng.random() < 0.5}
    if kind == "fork":
        beam = rng.randint(2, 8)
        return {"kind": kind, "seqs": beam * _log(rng, 1, 128 // beam), "beam": beam, "len": _log(rng, 2, 1000),
                "layers": rng.choice([1, 2, 5, 8]), "kv": kv, "dim": dim, "page": page}
    seqs, length = _log(rng, 2, 40), _log(rng, 4, 1000)
    return {"kind": kind, "seqs": seqs, "len": length, "pages": round(seqs * (length // page + 1) * rng.uniform(1.2, 2.4)),
            "layers": rng.choice([1, 2, 5, 8]), "kv": kv, "dim": dim, "page": page}


def _spread(n, lo, hi, phase=0.0):
    """n whole numbers over [lo, hi], mixed, the last one hi."""
    got = [lo + int((hi - lo + 1) * math.modf(0.6180339887 * (i + 1) + phase)[0]) for i in range(n)]
    got[-1] = hi
    return got


def _sizes(c):
    """Tokens held (the new ones among them) and new rows of each sequence."""
    if c["kind"] == "append":
        new = _spread(c["seqs"], max(1, c["new"] // 3), c["new"])
        old = _spread(c["seqs"], c["old"] // 4, c["old"], 0.37)
        return [a + b for a, b in zip(old, new)], new
    if c["kind"] == "attend":
        new = _spread(c["seqs"], max(1, c["rows"] // 3), c["rows"])
        if c["len"] == c["rows"]:
            return new, new
        return [max(n, x) for n, x in zip(new, _spread(c["seqs"], max(1, c["len"] // 3), c["len"], 0.37))], new
    return _spread(c["seqs"], max(1, c["len"] // 3), c["len"]), [0] * c["seqs"]


def _parents(c):
    """Each hypothesis's parent, in its own group of `beam`; some continue themselves."""
    rng = random.Random(c["seqs"] * 1000 + c["beam"])
    return [i // c["beam"] * c["beam"] + rng.randrange(c["beam"]) for i in range(c["seqs"])]


# ---------------------------------------------------------------------------
# e4m3 with a power-of-two scale, plain
# ---------------------------------------------------------------------------
def _need(amax):
    """The smallest power of two s >= 2^MIN_EXP with amax <= 448 s."""
    m, e = torch.frexp(amax)                       # amax = m 2^e, m in [1/2, 1); 448 = (7/8) 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _codes(x, scale):
    return (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _finite_abs(x):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))


# ---------------------------------------------------------------------------
# What a program holds before the call
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _pool(g, layers, pages, kv, page, dim):
    """Codes and scales of pages as earlier appends left them: normal values
    whose size differs from channel to channel and from page to page."""
    codes = torch.empty(layers, pages, kv, page, dim, dtype=torch.uint8, device="cuda")
    scale = torch.empty(layers, pages, kv, device="cuda")
    step = max(1, CHUNK // (kv * page * dim))
    chan = torch.exp(0.5 * torch.randn(kv, 1, dim, generator=g, device="cuda"))
    for lay in range(layers):
        for p in range(0, pages, step):
            n = min(step, pages - p)
            x = torch.randn(n, kv, page, dim, generator=g, device="cuda") * chan
            x *= torch.exp(0.3 * torch.randn(n, kv, 1, 1, generator=g, device="cuda"))
            s = _need(x.abs().amax((2, 3)))
            codes[lay, p:p + n] = _codes(x, s[:, :, None, None]).view(torch.uint8)
            scale[lay, p:p + n] = s
    return codes, scale


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    c = case
    lens, new = _sizes(c)
    page, kv, dim = c["page"], c["kv"], c["dim"]
    held = [-(-n // page) for n in lens]
    used = sum(held)
    # attention and append run in the second layer of two, so that a layer's place in the pool counts
    layers = c.get("layers") or (2 if used * kv * page * dim <= 1 << 28 else 1)
    spare = 8 + used // 8 + (c["seqs"] if c["kind"] == "fork" else 0)
    pages = max(c.get("pages") or 0, used + spare)
    width = max(held) + 2
    k, ks = _pool(g, layers, pages, kv, page, dim)
    v, vs = _pool(g, layers, pages, kv, page, dim)
    order = torch.randperm(pages, generator=g, device="cuda")[:used].to(torch.int32)
    table = torch.full((c["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = _i32([[i, j] for i, n in enumerate(held) for j in range(n)]).long()
    table[at[:, 0], at[:, 1]] = order
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order.long()] = 1
    st = {"case": dict(c), "layers": layers, "layer": layers - 1, "k": k, "v": v, "ks": ks, "vs": vs, "table": table,
          "refs": refs, "len": _i32(lens), "lens": lens, "new": new, "max_len": max(lens), "max_rows": max(new)}
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    st["rows"], st["n_rows"] = _i32(start), start[-1]
    kind = torch.bfloat16 if c.get("bf16") else torch.float32
    n = start[-1]
    if c["kind"] == "append":
        size = torch.exp(0.5 * torch.randn(n, kv, 1, generator=g, device="cuda"))
        st["xk"] = (torch.randn(n, kv, dim, generator=g, device="cuda") * size).to(kind)
        st["xv"] = (torch.randn(n, kv, dim, generator=g, device="cuda") * size).to(kind)
    elif c["kind"] == "attend":
        st["q"] = torch.randn(n, c["heads"], dim, generator=g, device="cuda").to(kind)
        st["out"] = torch.empty_like(st["q"])
    elif c["kind"] == "fork":
        st["dst"], st["src"] = _i32(list(range(c["seqs"]))), _i32(_parents(c))
    else:
        st["table0"], st["refs0"] = table.clone(), refs.clone()
    return st


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _row_places(st):
    """Sequence and position of each new row."""
    start = st["rows"].long()
    row = torch.arange(st["n_rows"], device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    pos = st["len"].long()[seq] - (start[seq + 1] - start[seq]) + (row - start[seq])
    return row, seq, pos


def _plain_append(st):
    page = st["case"]["page"]
    lay = st["layer"]
    _, seq, pos = _row_places(st)
    place, tok = st["table"][seq, pos // page].long(), pos % page
    first = torch.full((st["refs"].numel(),), page, dtype=torch.int64, device="cuda")
    first.scatter_reduce_(0, place, tok, "amin")            # first new token of each page
    touched = torch.nonzero(first < page).flatten()
    begun = first[touched] > 0                              # pages that held tokens before
    held = torch.arange(page, device="cuda")[None, :] < first[touched][:, None]
    for x, pool, scale in ((st["xk"], st["k"][lay], st["ks"][lay]), (st["xv"], st["v"][lay], st["vs"][lay])):
        x = x.float()
        amax = torch.zeros_like(scale)
        top = _finite_abs(x).amax(2)
        amax.scatter_reduce_(0, place[:, None].expand_as(top), top, "amax")
        old = scale[touched]
        now = _need(amax[touched])
        now = torch.where(begun[:, None], torch.maximum(old, now), now)
        was = pool[touched].view(torch.float8_e4m3fn).float() * (old / now)[:, :, None, None]
        was = torch.where(held[:, None, :, None], was.to(torch.float8_e4m3fn).view(torch.uint8), pool[touched])
        pool[touched] = was
        scale[touched] = now
        pool[place, :, tok] = _codes(x, scale[place][:, :, None]).view(torch.uint8)
    return _pools(st)


def _pools(st):
    return {"k": st["k"].view(torch.float8_e4m3fn), "v": st["v"].view(torch.float8_e4m3fn), "ks": st["ks"],
            "vs": st["vs"]}


def _book(st):
    return {"table": st["table"], "len": st["len"], "refs": st["refs"], **_pools(st)}


def _plain_attend(st):
    c = st["case"]
    page, lay, kv, dim = c["page"], st["layer"], c["kv"], c["dim"]
    group, n, top = c["heads"] // kv, st["max_rows"], st["max_len"]
    length = st["len"].long()
    key = torch.arange(top, device="cuda")
    place = st["table"][:, key // page].long().clamp(min=0)             # [seqs, top]

    def whole(pool, scale):                                            # [seqs, kv, top, dim] fp32
        x = pool[lay][place, :, key % page].view(torch.float8_e4m3fn).float() * scale[lay][place][..., None]
        return x.permute(0, 2, 1, 3).contiguous()

    row, seq, pos = _row_places(st)
    at = row - st["rows"].long()[seq]
    q = torch.zeros(c["seqs"], n, c["heads"], dim, device="cuda")
    q[seq, at] = st["q"].float()
    place_of = torch.full((c["seqs"], n), -1, dtype=torch.int64, device="cuda")
    place_of[seq, at] = pos
    q = q.view(c["seqs"], n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(c["seqs"], kv, group * n, dim)
    s = torch.matmul(q, whole(st["k"], st["ks"]).transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim))
    p, j = place_of[:, :, None], key[None, None, :]
    seen = (j < length[:, None, None]) & (p >= 0)
    if c["causal"]:
        seen = seen & (j <= p)
    if c["window"]:
        seen = seen & ((j > p - c["window"]) | (j < c["sinks"]))
    s = s.view(c["seqs"], kv, group, n, top).masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(torch.isfinite(m), m, torch.zeros_like(m))).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(c["seqs"], kv, group * n, top), whole(st["v"], st["vs"])).view(c["seqs"], kv, group, n, dim)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(c["seqs"], n, c["heads"], dim)[seq, at].to(st["q"].dtype)


def _plain_fork(st):
    page = st["case"]["page"]
    moves = st["dst"] != st["src"]
    dst, src = st["dst"][moves].long(), st["src"][moves].long()
    table, length, refs = st["table"], st["len"], st["refs"]
    rows, n = table[src], length[src]
    part = torch.nonzero(n % page).flatten()                # whose last page is partly filled
    col = n[part].long() // page
    fresh = torch.nonzero(refs == 0).flatten()[:part.numel()]
    last = rows[part, col].long()
    for x in (st["k"], st["v"], st["ks"], st["vs"]):
        x[:, fresh] = x[:, last]
    rows[part, col] = fresh.to(torch.int32)
    old = table[dst].flatten()
    for ids, by in ((rows.flatten(), 1), (old, -1)):
        ids = ids[ids >= 0].long()
        refs.scatter_add_(0, ids, torch.full_like(ids, by, dtype=torch.int32))
    table[dst] = rows
    length[dst] = n
    return _book(st)


def _plain_compact(st):
    st["table"].copy_(st["table0"])                         # the spread pages of this pass
    st["refs"].copy_(st["refs0"])
    table, refs = st["table"], st["refs"]
    live = refs > 0
    n = live.sum()
    page = torch.arange(refs.numel(), device="cuda")
    move, hole = torch.nonzero(live & (page >= n)).flatten(), torch.nonzero(~live & (page < n)).flatten()
    for x in (st["k"], st["v"], st["ks"], st["vs"]):
        x[:, hole] = x[:, move]
    to = page.clone()
    to[move] = hole
    refs[hole] = refs[move]
    refs[move] = 0
    table.copy_(torch.where(table >= 0, to[table.long().clamp(min=0)].to(torch.int32), table))
    return _book(st)


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
_lib = None


def _library():
    global _lib
    if _lib is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "cohere-transcribe_amd"))
        import ctbind as cb
        lib = cb.hip()
        lib.backend_init(0)
        _lib = cb, lib, torch.cuda.ExternalStream(lib.backend_stream())
    return _lib


def _handle(st):
    """The cache's descriptor, and an attention call's with its workspace, as a program keeps them."""
    if "handle" not in st:
        cb, lib, _ = _library()
        c = st["case"]
        h = cb.BackendKv8(layers=st["layers"], pages=st["refs"].numel(), page_tokens=c["page"], kv_heads=c["kv"],
                          head_dim=c["dim"], seqs=c["seqs"], table_w=st["table"].shape[1], k=st["k"].data_ptr(),
                          v=st["v"].data_ptr(), kscale=st["ks"].data_ptr(), vscale=st["vs"].data_ptr(),
                          table=st["table"].data_ptr(), len=st["len"].data_ptr(), refs=st["refs"].data_ptr())
        st["plan"] = torch.zeros(lib.backend_kv8_plan_ints(C.byref(h)), dtype=torch.int32, device="cuda")
        h.plan = st["plan"].data_ptr()
        st["handle"] = C.byref(h)
        if c["kind"] == "attend":
            a = cb.BackendKv8Attn(out=st["out"].data_ptr(), q=st["q"].data_ptr(), ld_out=c["heads"] * c["dim"],
                                  ld_q=c["heads"] * c["dim"], bf16=c["bf16"], heads=c["heads"],
                                  scale=1.0 / math.sqrt(c["dim"]), causal=c["causal"], window=c["window"],
                                  sinks=c["sinks"], rows=st["rows"].data_ptr(), n_rows=st["n_rows"],
                                  max_rows=st["max_rows"], max_len=st["max_len"])
            st["work"] = torch.empty(lib.backend_kv8_attn_work(st["handle"], C.byref(a)), device="cuda")
            a.work = st["work"].data_ptr()
            st["call"] = C.byref(a)
    return st["handle"]


def _own_run(st):
    _, lib, stream = _library()
    c, h = st["case"], _handle(st)
    if c["kind"] == "append":
        lib.backend_kv8_append(h, st["layer"], st["xk"].data_ptr(), st["xv"].data_ptr(), c["kv"] * c["dim"], c["bf16"],
                               st["rows"].data_ptr(), st["n_rows"])
        return _pools(st)
    if c["kind"] == "attend":
        lib.backend_kv8_attn(h, st["layer"], st["call"])
        return st["out"]
    if c["kind"] == "fork":
        lib.backend_kv8_fork(h, st["dst"].data_ptr(), st["src"].data_ptr(), c["seqs"])
        return _book(st)
    with torch.cuda.stream(stream):
        st["table"].copy_(st["table0"])
        st["refs"].copy_(st["refs0"])
    lib.backend_kv8_compact(h)
    return _book(st)


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "attend": _plain_attend, "fork": _plain_fork,
            "compact": _plain_compact}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _visible(c, n, length):
    """Keys some row of a sequence sees, and the (row, key) pairs it computes."""
    if not c["causal"]:
        return length, n * length
    w, pairs, first = c["window"], 0, length - n
    if not w:
        return length, n * first + n * (n + 1) // 2
    for p in range(first, length):
        lo = max(0, p + 1 - w)
        pairs += p + 1 - lo + min(c["sinks"], lo)
    lo = max(0, first + 1 - w)
    return length - lo + min(c["sinks"], lo), pairs


def work(case):
    c = case
    lens, new = _sizes(c)
    row, wide = c["kv"] * c["dim"], 2 if c.get("bf16") else 4
    page_bytes = c.get("layers", 1) * c["kv"] * 2 * (c["page"] * c["dim"] + 4)
    if c["kind"] == "append":
        return {"bytes": sum(new) * row * 2 * (wide + 1), "flops": sum(new) * row * 2}
    if c["kind"] == "attend":
        seen = [_visible(c, n, x) for n, x in zip(new, lens)]
        return {"bytes": sum(s for s, _ in seen) * row * 2 + 2 * sum(new) * c["heads"] * c["dim"] * wide,
                "flops": 4 * c["dim"] * c["heads"] * sum(p for _, p in seen)}
    if c["kind"] == "fork":
        moved = [(i, p) for i, p in enumerate(_parents(c)) if i != p]
        copies = sum(1 for _, p in moved if lens[p] % c["page"])
        return {"bytes": 2 * copies * page_bytes + 8 * sum(-(-lens[p] // c["page"]) for _, p in moved) + 8, "flops": 0}
    held = sum(-(-n // c["page"]) for n in lens)
    pages = max(c["pages"], held + 8 + held // 8)
    # the pages lie anywhere: a share (pages - held) / pages of them is past the front
    return {"bytes": 2 * round(held * (pages - held) / pages) * page_bytes + 8 * held + 8 * pages, "flops": 0}


# ---------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------
def _round_e4m3(x):
    """Nearest e4m3 value, ties to even, of values within +-448."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _value(code):
    """e4m3 codes as 64-bit values: sign, 4 bits of exponent with bias 7, 3 of fraction."""
    c = code.to(torch.int64)
    e, f = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(e > 0, (8 + f) * torch.pow(2.0, (e - 10).double()), f * 2.0 ** -9)
    return torch.where(c >= 128, -mag, mag)


def _exact_append(st):
    c, lay, page = st["case"], st["layer"], st["case"]["page"]
    table, row = st["table"].tolist(), 0
    got = {"k": st["k"].view(torch.float8_e4m3fn).clone(), "v": st["v"].view(torch.float8_e4m3fn).clone(),
           "ks": st["ks"].clone(), "vs": st["vs"].clone()}
    for i, (length, n) in enumerate(zip(st["lens"], st["new"])):
        pos = length - n
        while pos < length:
            a, p = pos % page, table[i][pos // page]
            b = min(page, a + length - pos)
            for x, pool, scale in ((st["xk"], "k", "ks"), (st["xv"], "v", "vs")):
                x = x[row:row + b - a].double().permute(1, 0, 2)                      # [kv, tokens, dim]
                e = torch.ceil(torch.log2(x.abs().amax((1, 2)).clamp(min=1e-300) / E4M3_MAX)).clamp(min=MIN_EXP)
                s = torch.ldexp(torch.ones_like(e), e.int())       # pow(2, e) is off by an ulp on some devices
                if a:
                    was = got[scale][lay, p].double()
                    s = torch.maximum(s, was)
                    held = _value(got[pool][lay, p, :, :a].view(torch.uint8)) * (was / s)[:, None, None]
                    got[pool][lay, p, :, :a] = _round_e4m3(held).to(torch.float8_e4m3fn)
                got[scale][lay, p] = s.float()
                got[pool][lay, p, :, a:b] = _round_e4m3(x / s[:, None, None]).to(torch.float8_e4m3fn)
            row, pos = row + b - a, pos + b - a
    return got


def _exact_attend(st):
    c, lay, page = st["case"], st["layer"], st["case"]["page"]
    group, row = c["heads"] // c["kv"], 0
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for i, (length, n) in enumerate(zip(st["lens"], st["new"])):
        pages = st["table"][i, :-(-length // page)].long()
        kv = []
        for pool, scale in (("k", "ks"), ("v", "vs")):
            x = _value(st[pool][lay, pages]) * st[scale][lay, pages].double()[:, :, None, None]
            kv.append(x.permute(1, 0, 2, 3).reshape(c["kv"], -1, c["dim"])[:, :length])
        j = torch.arange(length, device="cuda")
        for r in range(0, n, 512):                                      # some rows at a time
            m = min(512, n - r)
            p = length - n + r + torch.arange(m, device="cuda")[:, None]
            seen = torch.ones(m, length, dtype=torch.bool, device="cuda")
            if c["causal"]:
                seen &= j <= p
            if c["window"]:
                seen &= (p - j < c["window"]) | (j < c["sinks"])
            for h in range(c["heads"]):
                q = st["q"][row + r:row + r + m, h].double()
                s = (q @ kv[0][h // group].T / math.sqrt(c["dim"])).masked_fill(~seen, -math.inf)
                out[row + r:row + r + m, h] = torch.softmax(s, 1) @ kv[1][h // group]
        row += n
    return out


def _exact_fork(st):
    c, page = st["case"], st["case"]["page"]
    got = {n: x.clone() for n, x in _book(st).items()}
    table, refs = st["table"].tolist(), st["refs"].tolist()
    free = [i for i, n in enumerate(refs) if n == 0]
    was = [list(t) for t in table]
    for d, s in enumerate(_parents(c)):
        if d == s:
            continue
        table[d] = list(was[s])
        if st["lens"][s] % page:
            col, p = st["lens"][s] // page, free.pop(0)
            for n in ("k", "v", "ks", "vs"):
                got[n][:, p] = st[n][:, was[s][col]].view(got[n].dtype)
            table[d][col] = p
        got["len"][d] = st["lens"][s]
    got["table"] = _i32(table)
    got["refs"] = torch.bincount(got["table"][got["table"] >= 0].long(), minlength=len(refs)).to(torch.int32)
    return got


def _exact_compact(st):
    got = {n: x.clone() for n, x in _book(st).items()}
    refs = st["refs"].tolist()
    live = [i for i, n in enumerate(refs) if n]
    front = set(live)
    holes = [i for i in range(len(live)) if i not in front]
    to = dict(zip([i for i in live if i >= len(live)], holes))
    for a, b in to.items():
        for n in ("k", "v", "ks", "vs"):
            got[n][:, b] = got[n][:, a]
        refs[b], refs[a] = refs[a], 0
    got["table"] = _i32([[to.get(p, p) for p in t] for t in st["table"].tolist()])
    got["refs"] = _i32(refs)
    return got


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "fork": _exact_fork,
            "compact": _exact_compact}[case["kind"]](prepare(case, seed))
