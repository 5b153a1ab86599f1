"""A decode step's linear maps, attention and logits, as timed cases.

  linear   linear maps whose weights are held in 4 bits with a scale and a zero
           point for each group of inputs: single tokens, batches, prompts
  shared   attention over the paged 8-bit cache of sequences whose first tokens
           are the same pages (a clip's hypotheses, samples of one prompt,
           requests with one instruction): those are read once for all
  logits   penalties for tokens that were said, biases, n-gram bans and grammar
           masks on a step's logits, and the token they leave on top

own = False computes each in its plain form; own = True makes the calls a
program makes of the library.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

E4M3_MAX = 448.0
MIN_EXP = -100          # smallest exponent of a page's scale
CHUNK = 1 << 27         # values made at once when a pool is filled


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One token through a decoder projection: the smallest call, where latency counts.
        {"name": "linear_token", "kind": "linear", "rows": 1, "in": 1024, "out": 1024, "group": 128, "zeros": False,
         "act": "store", "bf16": False},
        # The decoder's FFN up-projection for 64 requests.
        {"name": "linear_ffn_64", "kind": "linear", "rows": 64, "in": 1024, "out": 4096, "group": 64, "zeros": True,
         "act": "silu", "bf16": False},
        # The LM head for a clip's hypotheses.
        {"name": "linear_head_5", "kind": "linear", "rows": 5, "in": 1024, "out": 16384, "group": 32, "zeros": True,
         "act": "store", "bf16": False},
        # One token through a large map.
        {"name": "linear_wide", "kind": "linear", "rows": 1, "in": 8192, "out": 24576, "group": 128, "zeros": True,
         "act": "store", "bf16": True},
        # Two clips of 30 s through the encoder's FFN up-projection.
        {"name": "linear_clips", "kind": "linear", "rows": 752, "in": 1280, "out": 5120, "group": 128, "zeros": True,
         "act": "silu", "bf16": False},
        # A beam of 5 over its clip's 376 encoder frames.
        {"name": "shared_beam", "kind": "shared", "groups": 1, "each": 5, "prefix": 376, "own": 0, "rows": 1,
         "heads": 8, "kv": 8, "dim": 128, "page": 64, "bf16": False},
        # The same for 24 clips up to 30 s, small pages.
        {"name": "shared_clips_24", "kind": "shared", "groups": 24, "each": 5, "prefix": 376, "own": 0, "rows": 1,
         "heads": 8, "kv": 8, "dim": 128, "page": 16, "bf16": False},
        # A step of 64 requests that begin with one instruction of 8000 tokens, four
        # query heads to a key head.
        {"name": "shared_step_64", "kind": "shared", "groups": 1, "each": 64, "prefix": 8000, "own": 1000, "rows": 1,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "bf16": True},
        # The prompts of four requests behind each of two such instructions.
        {"name": "shared_prompts_8", "kind": "shared", "groups": 2, "each": 4, "prefix": 6000, "own": 401, "rows": 401,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "bf16": True},
        # A beam of 5 over the model's vocabulary; the next beam step wants the logits.
        {"name": "logits_beam", "kind": "logits", "rows": 5, "vocab": 16384, "history": 200, "ngram": 3, "biases": 20,
         "masks": 0, "out": True},
        # The greedy step of 64 requests, half of them under a grammar.
        {"name": "logits_step_64", "kind": "logits", "rows": 64, "vocab": 16384, "history": 1000, "ngram": 4,
         "biases": 60, "masks": 8, "out": False},
        # A large vocabulary of odd size, long texts.
        {"name": "logits_wide_200", "kind": "logits", "rows": 200, "vocab": 100003, "history": 4000, "ngram": 0,
         "biases": 300, "masks": 200, "out": True},
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "shared", "shared", "logits"])
    if kind == "linear":
        ins = _log(rng, 64, 8192)
        outs = _log(rng, 32, min(24576, 200000000 // ins))
        rows = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 752)])
        return {"kind": kind, "rows": max(1, min(rows, 4900000000 // (ins * outs))), "in": ins, "out": outs,
                "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.7,
                "act": rng.choice(["store", "silu", "relu", "add"]), "bf16": rng.random() < 0.5}
    if kind == "shared":
        kv, group, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4]), rng.choice([64, 128])
        each, groups = _log(rng, 1, 64), rng.choice([1, 1, 2, 4, 16])
        each = min(each, 128 // groups)
        own = rng.choice([0, _log(rng, 1, 1000)])
        rows = 1 if not own else min(own, rng.choice([1, 1, rng.randint(2, 8), max(1, 1600 // (each * groups))]))
        return {"kind": kind, "groups": groups, "each": each, "prefix": _log(rng, 300, 8000), "own": own,
                "rows": rows, "heads": kv * group, "kv": kv, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "bf16": rng.random() < 0.5}
    vocab = _log(rng, 50, 200000)
    return {"kind": kind, "rows": _log(rng, 1, min(256, 20000000 // vocab)), "vocab": vocab,
            "history": _log(rng, 1, 4000), "ngram": rng.choice([0, 1, 2, 3, 5]), "biases": rng.choice([0, _log(rng, 1, 300)]),
            "masks": rng.choice([0, 1, _log(rng, 2, 64)]), "out": rng.random() < 0.6}


def _spread(n, lo, hi, phase=0.0):
    """n whole numbers over [lo, hi], mixed, the last one hi."""
    got = [lo + int((hi - lo + 1) * math.modf(0.6180339887 * (i + 1) + phase)[0]) for i in range(n)]
    got[-1] = hi
    return got


def _sizes(c):
    """Of a `shared` case: each group's common tokens, and each sequence's
    group, tokens held and new rows.  Groups take turns, so that a group's
    sequences do not lie side by side; a clip's hypotheses do."""
    n = c["groups"] * c["each"]
    if not c["own"]:
        pre = _spread(c["groups"], max(1, c["prefix"] // 3), c["prefix"])
        of = [i // c["each"] for i in range(n)]
        return pre, of, [pre[g] for g in of], [1] * n
    pre = [p // c["page"] * c["page"] for p in _spread(c["groups"], max(1, c["prefix"] // 2), c["prefix"])]
    of = [i % c["groups"] for i in range(n)]
    new = _spread(n, max(1, c["rows"] // 2), c["rows"])
    mine = new if c["own"] == c["rows"] else [max(a, b) for a, b in zip(new, _spread(n, max(1, c["own"] // 3), c["own"], 0.37))]
    return pre, of, [pre[g] + m for g, m in zip(of, mine)], new


# ---------------------------------------------------------------------------
# What a program holds before the call
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _prepare_linear(c, g):
    ins, outs, rows = c["in"], c["out"], c["rows"]
    kind = torch.bfloat16 if c["bf16"] else torch.float32
    groups = -(-ins // c["group"])
    # as a checkpoint has them: two codes a byte, the first in the low bits; bf16 scales
    zero = _randint(g, 6, 10, outs, groups).to(torch.uint8) if c["zeros"] else None
    mid = 8 if zero is None else zero.float().repeat_interleave(c["group"], 1)[:, :ins]
    code = (torch.randn(outs, ins, generator=g, device="cuda") * 2.8 + mid).round_().clamp_(0, 15).to(torch.uint8)
    if ins % 2:
        code = torch.nn.functional.pad(code, (0, 1))
    size = torch.exp(0.3 * torch.randn(outs, groups, generator=g, device="cuda")) / (2.8 * math.sqrt(ins))
    chan = torch.exp(0.5 * torch.randn(ins, generator=g, device="cuda"))
    x = ((torch.randn(rows, ins, generator=g, device="cuda") + 0.1) * chan).to(kind)
    return {"codes": code[:, 0::2] | code[:, 1::2] << 4, "scales": size.to(torch.bfloat16), "zeros": zero, "x": x,
            "bias": (0.1 * torch.randn(outs, generator=g, device="cuda")).to(torch.bfloat16),
            # what an "add" adds to
            "acc": torch.randn(rows, outs, generator=g, device="cuda").to(kind),
            "y": torch.zeros(rows, outs, dtype=kind, device="cuda")}


def _pool(g, pages, kv, page, dim):
    """Codes and scales of pages as earlier appends left them: normal values
    whose size differs from channel to channel and from page to page."""
    codes = torch.empty(1, pages, kv, page, dim, dtype=torch.uint8, device="cuda")
    scale = torch.empty(1, pages, kv, device="cuda")
    step = max(1, CHUNK // (kv * page * dim))
    chan = torch.exp(0.5 * torch.randn(kv, 1, dim, generator=g, device="cuda"))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, kv, page, dim, generator=g, device="cuda") * chan
        x *= torch.exp(0.3 * torch.randn(n, kv, 1, 1, generator=g, device="cuda"))
        m, e = torch.frexp(x.abs().amax((2, 3)))        # 448 = (7/8) 2^9
        e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=MIN_EXP)
        s = torch.ldexp(torch.ones_like(m), e)
        codes[0, p:p + n] = (x / s[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        scale[0, p:p + n] = s
    return codes, scale


def _prepare_shared(c, g):
    pre, of, lens, new = _sizes(c)
    page, n = c["page"], len(of)
    held = [-(-x // page) for x in lens]
    common = [-(-p // page) for p in pre]
    used = sum(common) + sum(h - common[k] for h, k in zip(held, of))
    pages, width = used + 8, max(held) + 2
    k, ks = _pool(g, pages, c["kv"], page, c["dim"])
    v, vs = _pool(g, pages, c["kv"], page, c["dim"])
    order = torch.randperm(pages, generator=g, device="cuda")[:used].to(torch.int32)
    first = [sum(common[:i]) for i in range(len(common))]       # the common pages come first in `order`
    at, rows, index = sum(common), [], []
    for i, q in enumerate(of):
        mine = held[i] - common[q]
        rows += [i * width + j for j in range(held[i])]
        index += list(range(first[q], first[q] + common[q])) + list(range(at, at + mine))
        at += mine
    table = torch.full((n * width,), -1, dtype=torch.int32, device="cuda")
    table[torch.tensor(rows, device="cuda")] = order[torch.tensor(index, device="cuda")]
    table = table.view(n, width)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs.scatter_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
    lead = [of.index(q) for q in of]
    start = [0]
    for m in new:
        start.append(start[-1] + m)
    kind = torch.bfloat16 if c["bf16"] else torch.float32
    q = torch.randn(start[-1], c["heads"], c["dim"], generator=g, device="cuda").to(kind)
    return {"k": k, "v": v, "ks": ks, "vs": vs, "table": table, "refs": refs, "len": _i32(lens), "lens": lens,
            "new": new, "rows": _i32(start), "n_rows": start[-1], "max_rows": max(new), "max_len": max(lens),
            "pre": pre, "of": of, "share": _i32([lead, [pre[x] for x in of]]), "q": q, "out": torch.empty_like(q),
            "by_group": torch.tensor(sorted(range(n), key=lambda i: of[i]), device="cuda")}


def _prepare_logits(c, g):
    n, vocab, top = c["rows"], c["vocab"], c["history"]
    lens = _spread(n, top // 3, top)
    # text repeats itself: few tokens often, many seldom
    u = torch.rand(n, top, generator=g, device="cuda")
    hist = (torch.exp(u * math.log(vocab)) - 1).to(torch.int32).clamp_(0, vocab - 1)
    if top > 60:                                               # the last words were said before
        hist[:, 5:20] = hist[:, 45:60]
        for_end = (torch.tensor(lens, device="cuda")[:, None] - 5 + torch.arange(5, device="cuda")).clamp(min=0).long()
        hist.scatter_(1, for_end, hist[:, 5:10].clone())
    st = {"logits": 3 * torch.randn(n, vocab, generator=g, device="cuda"), "hist": hist, "hist_len": _i32(lens),
          "prompt_len": _i32([x // 4 for x in lens]),
          "repeat": 1 + 0.5 * torch.rand(n, generator=g, device="cuda"),
          "frequency": 0.3 * torch.rand(n, generator=g, device="cuda"),
          "presence": 0.5 * torch.rand(n, generator=g, device="cuda"),
          "ngram": torch.full((n,), c["ngram"], dtype=torch.int32, device="cuda"),
          "id": torch.empty(n, dtype=torch.int32, device="cuda"), "score": torch.empty(n, device="cuda"),
          "out": torch.empty(n, vocab, device="cuda") if c["out"] else None, "bias": None, "mask": None}
    if n > 1:                                                  # the first row has no penalties
        st["repeat"][0], st["frequency"][0], st["presence"][0], st["ngram"][0] = 1.0, 0.0, 0.0, 0
    if c["biases"]:
        many = _spread(n, 0, c["biases"])
        start = [0]
        for m in many:
            start.append(start[-1] + m)
        st["bias_start"] = _i32(start)
        st["bias_id"] = _randint(g, 0, vocab, start[-1])        # some twice
        st["bias"] = 4 * torch.randn(start[-1], generator=g, device="cuda")
    if c["masks"]:
        words = -(-vocab // 32)
        allowed = torch.rand(c["masks"], words * 32, generator=g, device="cuda") < 0.3
        if c["masks"] > 1:
            allowed[1] = False                                  # a dead end
        bit = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        w = (allowed.view(c["masks"], words, 32) * bit).sum(2)
        st["mask"] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
        st["mask_of"] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, -1, _randint(g, 0, c["masks"], n))
    return st


def prepare(case, seed):
    g = _gen(seed)
    st = {"linear": _prepare_linear, "shared": _prepare_shared, "logits": _prepare_logits}[case["kind"]](case, g)
    st["case"] = dict(case)
    return st


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_linear(st):
    c = st["case"]
    code = torch.stack([st["codes"] & 15, st["codes"] >> 4], 2).view(c["out"], -1)[:, :c["in"]].float()
    wide = lambda t: t.float().repeat_interleave(c["group"], 1)[:, :c["in"]]  # noqa: E731
    w = (code - (8 if st["zeros"] is None else wide(st["zeros"]))) * wide(st["scales"])
    y = st["x"].float() @ w.t() + st["bias"].float()
    if c["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif c["act"] == "relu":
        y = y.clamp(min=0)
    elif c["act"] == "add":
        y = st["acc"].float() + 0.5 * y
    return y.to(st["x"].dtype)


def _row_places(st):
    """Sequence, position and place in its sequence of each new row."""
    start = st["rows"].long()
    row = torch.arange(st["n_rows"], device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    at = row - start[seq]
    return seq, st["len"].long()[seq] - (start[seq + 1] - start[seq]) + at, at


def _plain_shared(st):
    c = st["case"]
    page, kv, dim = c["page"], c["kv"], c["dim"]
    group, n, each, groups = c["heads"] // kv, st["max_rows"], c["each"], c["groups"]
    seqs = each * groups
    seq, pos, at = _row_places(st)
    lead, pre = st["share"][0].long(), st["share"][1].long()
    length = st["len"].long()

    def whole(pool, scale, seqs_of, key):                       # [.., kv, keys, dim] fp32 of keys [.., keys]
        place = torch.gather(st["table"][seqs_of], 1, (key // page).clamp(max=st["table"].shape[1] - 1)).long().clamp(min=0)
        x = pool[0][place, :, key % page].view(torch.float8_e4m3fn).float() * scale[0][place][..., None]
        return x.permute(0, 2, 1, 3).contiguous()

    q = torch.zeros(seqs, n, kv, group, dim, device="cuda")
    q[seq, at] = st["q"].float().view(-1, kv, group, dim)
    where = torch.full((seqs, n), -1, dtype=torch.int64, device="cuda")
    where[seq, at] = pos
    # the groups' rows against the common keys
    firsts = torch.unique(lead)
    order = st["by_group"]                                      # sequences, group by group
    top = max(st["pre"])
    key = torch.arange(top, device="cuda").expand(groups, top)
    qg = q[order].view(groups, each, n, kv, group, dim).permute(0, 3, 4, 1, 2, 5).reshape(groups, kv, group * each * n, dim)
    s1 = torch.matmul(qg, whole(st["k"], st["ks"], firsts, key).transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim))
    s1.masked_fill_((key >= pre[firsts][:, None])[:, None, None], -math.inf)
    m = s1.amax(-1)                                             # [groups, kv, group * each * n]
    own_keys = max(x - st["pre"][g] for x, g in zip(st["lens"], st["of"]))
    back = torch.argsort(order)

    def by_seq(x):                                              # of [groups, kv, group * each * n, ..]: [seqs, kv, group * n, ..]
        tail = x.shape[3:]
        x = x.view(groups, kv, group, each, n, *tail).transpose(2, 3).transpose(1, 2)
        return x.reshape(seqs, kv, group * n, *tail)[back]

    m1 = by_seq(m)
    if own_keys:
        key2 = pre[:, None] + torch.arange(own_keys, device="cuda")
        seen = (key2[:, None, :] <= where[:, :, None]) & (key2 < length[:, None])[:, None, :]
        qs = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * n, dim)
        ids = torch.arange(seqs, device="cuda")
        s2 = torch.matmul(qs, whole(st["k"], st["ks"], ids, key2).transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim))
        s2 = s2.view(seqs, kv, group, n, own_keys).masked_fill_(~seen[:, None, None], -math.inf).view(seqs, kv, group * n, own_keys)
        m1 = torch.maximum(m1, s2.amax(-1))
        s2 = s2.sub_(m1[..., None]).exp_()
        num2, den2 = torch.matmul(s2, whole(st["v"], st["vs"], ids, key2)), s2.sum(-1)
        mg = m1[order].view(groups, each, kv, group, n).permute(0, 2, 3, 1, 4).reshape(groups, kv, group * each * n)
    else:
        num2, den2, mg = 0.0, 0.0, m
    s1 = s1.sub_(mg[..., None]).exp_()
    num = by_seq(torch.matmul(s1, whole(st["v"], st["vs"], firsts, key))) + num2
    den = by_seq(s1.sum(-1)) + den2
    o = (num / den[..., None]).view(seqs, kv, group, n, dim)
    return o.permute(0, 3, 1, 2, 4).reshape(seqs, n, c["heads"], dim)[seq, at].to(st["q"].dtype)


def _plain_logits(st):
    c = st["case"]
    n, vocab, k = c["rows"], c["vocab"], c["ngram"]
    x, hist = st["logits"], st["hist"].long()
    length, prompt = st["hist_len"].long()[:, None], st["prompt_len"].long()[:, None]
    at = torch.arange(hist.shape[1], device="cuda")[None]
    held = at < length
    count = torch.zeros(n, vocab, device="cuda").scatter_add_(1, hist, (held & (at >= prompt)).float())
    seen = torch.zeros(n, vocab, device="cuda").scatter_add_(1, hist, held.float()) > 0
    r = st["repeat"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(count > 0, x - st["frequency"][:, None] * count - st["presence"][:, None], x)
    if st["bias"] is not None:
        entry = torch.arange(st["bias"].numel(), device="cuda")
        row = torch.searchsorted(st["bias_start"].long(), entry, right=True) - 1
        last = torch.full((n * vocab,), -1, dtype=torch.int64, device="cuda")
        last.scatter_reduce_(0, row * vocab + st["bias_id"].long(), entry, "amax")
        last = last.view(n, vocab)
        x = torch.where(last >= 0, x + st["bias"][last.clamp(min=0)], x)
    if k:
        # position i + k - 1 is banned where the k - 1 tokens before it are the last ones
        same = held & (at >= k - 1) & (st["ngram"] > 0)[:, None]
        back = torch.arange(1, k, device="cuda")[:, None, None]
        end = torch.gather(hist, 1, (length - torch.arange(1, k, device="cuda")[None]).clamp(min=0)) if k > 1 else None
        if k > 1:
            before = hist[torch.arange(n, device="cuda")[None, :, None], (at[None] - back).clamp(min=0)]
            same = same & (before == end.t()[:, :, None]).all(0) & (length >= k)
        ban = torch.zeros(n, vocab, device="cuda").scatter_add_(1, hist, same.float()) > 0
        x = x.masked_fill(ban, -math.inf)
    if st["mask"] is not None:
        v = torch.arange(vocab, device="cuda")
        ok = (st["mask"].long()[:, v // 32] >> (v % 32)) & 1
        ok = (ok[st["mask_of"].long().clamp(min=0)] > 0) | (st["mask_of"] < 0)[:, None]
        x = torch.where(ok, x, -math.inf)
    top = x.amax(1)
    v = torch.arange(vocab, device="cuda")
    first = torch.where(x == top[:, None], v, vocab).amin(1)
    got = {"id": torch.where(top > -math.inf, first, -1).to(torch.int32), "score": top}
    return {**got, "out": x} if c["out"] else got


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
        _lib = cb, lib
    return _lib


def _at(t):
    return 0 if t is None else t.data_ptr()


def _handle(st):
    """What a program keeps: the laid-out weight or the cache's descriptor, and
    the call with its workspace."""
    if "handle" in st:
        return st["handle"]
    cb, lib = _library()
    c = st["case"]
    if c["kind"] == "linear":
        w = cb.BackendW4(in_d=c["in"], out_d=c["out"], group=c["group"], scale_f16=0)
        st["mem"] = torch.empty(lib.backend_w4_floats(C.byref(w)), device="cuda")
        lib.backend_w4_bind(C.byref(w), st["mem"].data_ptr())
        lib.backend_w4_load(C.byref(w), _at(st["codes"]), _at(st["scales"]), _at(st["zeros"]))
        a = cb.BackendW4Linear(y=_at(st["y"]), x=_at(st["x"]), ld_y=c["out"], ld_x=c["in"], bf16=c["bf16"],
                               rows=c["rows"], bias=_at(st["bias"]), scale=0.5,
                               act={"store": cb.W4_STORE, "silu": cb.W4_SILU, "relu": cb.W4_RELU, "add": cb.W4_ADD}[c["act"]])
        st["handle"] = C.byref(w), C.byref(a)
    elif c["kind"] == "shared":
        h = cb.BackendKv8(layers=1, pages=st["refs"].numel(), page_tokens=c["page"], kv_heads=c["kv"],
                          head_dim=c["dim"], seqs=len(st["lens"]), table_w=st["table"].shape[1], k=_at(st["k"]),
                          v=_at(st["v"]), kscale=_at(st["ks"]), vscale=_at(st["vs"]), table=_at(st["table"]),
                          len=_at(st["len"]), refs=_at(st["refs"]))
        st["plan"] = torch.zeros(lib.backend_kv8_plan_ints(C.byref(h)), dtype=torch.int32, device="cuda")
        h.plan = _at(st["plan"])
        a = cb.BackendKv8Attn(out=_at(st["out"]), q=_at(st["q"]), ld_out=c["heads"] * c["dim"],
                              ld_q=c["heads"] * c["dim"], bf16=c["bf16"], heads=c["heads"],
                              scale=1.0 / math.sqrt(c["dim"]), causal=c["own"] > 0, window=0, sinks=0,
                              rows=_at(st["rows"]), n_rows=st["n_rows"], max_rows=st["max_rows"], max_len=st["max_len"])
        st["work"] = torch.empty(lib.backend_kv8_attn_shared_work(C.byref(h), C.byref(a)), device="cuda")
        a.work = _at(st["work"])
        st["handle"] = C.byref(h), C.byref(a)
    else:
        a = cb.BackendLogits(logits=_at(st["logits"]), out=_at(st["out"]), ld=c["vocab"], ld_out=c["vocab"],
                             rows=c["rows"], vocab=c["vocab"], id=_at(st["id"]), score=_at(st["score"]),
                             hist=_at(st["hist"]), ld_hist=st["hist"].shape[1], hist_len=_at(st["hist_len"]),
                             prompt_len=_at(st["prompt_len"]), repeat=_at(st["repeat"]),
                             frequency=_at(st["frequency"]), presence=_at(st["presence"]), ngram=_at(st["ngram"]))
        if st["bias"] is not None:
            a.bias_start, a.bias_id, a.bias = _at(st["bias_start"]), _at(st["bias_id"]), _at(st["bias"])
            a.biases = st["bias"].numel()
        if st["mask"] is not None:
            a.mask, a.ld_mask, a.masks, a.mask_of = _at(st["mask"]), st["mask"].shape[1], c["masks"], _at(st["mask_of"])
        st["work"] = torch.zeros(lib.backend_logits_work(C.byref(a)), device="cuda")
        torch.cuda.current_stream().synchronize()              # zeroed before the library's stream uses it
        a.work = _at(st["work"])
        st["handle"] = (C.byref(a),)
    return st["handle"]


def _own_run(st):
    cb, lib = _library()
    h = _handle(st)
    kind = st["case"]["kind"]
    if kind == "linear":
        if st["case"]["act"] == "add":                          # every pass adds to the same values
            with torch.cuda.stream(torch.cuda.ExternalStream(lib.backend_stream())):
                st["y"].copy_(st["acc"])
        lib.backend_linear_w4(*h)
        return st["y"]
    if kind == "shared":
        lib.backend_kv8_attn_shared(h[0], 0, h[1], st["share"].data_ptr())
        return st["out"]
    lib.backend_logits(*h)
    got = {"id": st["id"], "score": st["score"]}
    return {**got, "out": st["out"]} if st["case"]["out"] else got


def run(state):
    if own:
        return _own_run(state)
    return {"linear": _plain_linear, "shared": _plain_shared, "logits": _plain_logits}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    wide = 2 if c.get("bf16") else 4
    if c["kind"] == "linear":
        groups = -(-c["in"] // c["group"])
        weight = c["out"] * ((c["in"] + 1) // 2 + groups * (3 if c["zeros"] else 2) + 2)
        io = c["rows"] * (c["in"] + c["out"] * (2 if c["act"] == "add" else 1)) * wide
        return {"bytes": weight + io, "flops": 2 * c["rows"] * c["in"] * c["out"]}
    if c["kind"] == "shared":
        pre, of, lens, new = _sizes(c)
        keys = sum(pre) + sum(x - pre[g] for x, g in zip(lens, of))
        pairs = sum(n * (x - n) + n * (n + 1) // 2 if c["own"] else n * x for n, x in zip(new, lens))
        return {"bytes": keys * c["kv"] * 2 * c["dim"] + 2 * sum(new) * c["heads"] * c["dim"] * wide,
                "flops": 4 * c["dim"] * c["heads"] * pairs}
    n, vocab = c["rows"], c["vocab"]
    values = n * vocab * (8 if c["out"] else 4)
    lists = 4 * sum(_spread(n, c["history"] // 3, c["history"])) + (8 * sum(_spread(n, 0, c["biases"])) if c["biases"] else 0)
    masks = min(c["masks"], n) * -(-vocab // 32) * 4
    return {"bytes": values + lists + masks + 36 * n, "flops": 5 * n * vocab}


# ---------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_linear(st):
    c = st["case"]
    outs, step = [], max(1, (1 << 27) // c["in"])
    x = st["x"].double()
    for o in range(0, c["out"], step):                          # some outputs at a time
        byte = st["codes"][o:o + step].to(torch.int64)
        y = st["bias"][o:o + step].double().expand(c["rows"], -1).clone()
        for g in range(st["scales"].shape[1]):
            a, b = g * c["group"], min(c["in"], (g + 1) * c["group"])
            i = torch.arange(a, b, device="cuda")
            code = (byte[:, i // 2] >> (4 * (i % 2))) & 15
            z = 8.0 if st["zeros"] is None else st["zeros"][o:o + step, g:g + 1].double()
            y += (x[:, a:b] @ (code.double() - z).t().contiguous()) * st["scales"][o:o + step, g].double()
        outs.append(y)
    y = torch.cat(outs, 1)
    if c["act"] == "silu":
        return y * torch.sigmoid(y)
    if c["act"] == "relu":
        return torch.relu(y)
    return st["acc"].double() + y / 2 if c["act"] == "add" else y


def _value(code):
    """e4m3 codes as 64-bit values: sign, 4 bits of exponent with bias 7, 3 of fraction."""
    c = code.to(torch.int64)
    e, f = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(e > 0, (8 + f) * torch.pow(2.0, (e - 10).double()), f * 2.0 ** -9)
    return torch.where(c >= 128, -mag, mag)


def _exact_shared(st):
    c, page = st["case"], st["case"]["page"]
    group, row = c["heads"] // c["kv"], 0
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for i, (length, n) in enumerate(zip(st["lens"], st["new"])):   # each sequence by itself, over all its pages
        pages = st["table"][i, :-(-length // page)].long()
        kv = []
        for pool, scale in (("k", "ks"), ("v", "vs")):
            x = _value(st[pool][0, pages]) * st[scale][0, pages].double()[:, :, None, None]
            kv.append(x.permute(1, 0, 2, 3).reshape(c["kv"], -1, c["dim"])[:, :length])
        j = torch.arange(length, device="cuda")
        p = length - n + torch.arange(n, device="cuda")[:, None]
        for h in range(c["heads"]):
            s = st["q"][row:row + n, h].double() @ kv[0][h // group].T / math.sqrt(c["dim"])
            if c["own"]:
                s = s.masked_fill(j > p, -math.inf)
            out[row:row + n, h] = torch.softmax(s, 1) @ kv[1][h // group]
        row += n
    return out


def _exact_logits(st):
    c = st["case"]
    x = st["logits"].double().clone()
    words = st["mask"].long().cpu() if st["mask"] is not None else None
    hist, lens, prompts = st["hist"].long().cpu(), st["hist_len"].tolist(), st["prompt_len"].tolist()
    bias_start = st["bias_start"].tolist() if st["bias"] is not None else None
    for i in range(c["rows"]):
        said = hist[i, :lens[i]]
        seen = torch.unique(said).cuda()
        r, f, p = (st[name][i].double() for name in ("repeat", "frequency", "presence"))
        v = x[i, seen]
        x[i, seen] = torch.where(v > 0, v / r, v * r)
        ids, many = torch.unique(said[prompts[i]:], return_counts=True)
        x[i, ids.cuda()] -= f * many.cuda() + p
        if bias_start:
            a, b = bias_start[i], bias_start[i + 1]
            for t, y in dict(zip(st["bias_id"][a:b].tolist(), st["bias"][a:b].tolist())).items():
                x[i, t] += y
        k = int(st["ngram"][i])
        if k and lens[i] >= k:
            end = said[lens[i] - k + 1:]
            runs = said.unfold(0, k, 1)
            x[i, runs[(runs[:, :-1] == end).all(1), -1].cuda()] = -math.inf
        if words is not None and int(st["mask_of"][i]) >= 0:
            w = words[int(st["mask_of"][i])]
            bits = ((w[:, None] >> torch.arange(32)) & 1).flatten()[:c["vocab"]]
            x[i, (bits == 0).cuda()] = -math.inf
    score, at = x.max(1)
    got = {"id": torch.where(score > -math.inf, at, -1).to(torch.int32), "score": score}
    return {**got, "out": x} if c["out"] else got


def exact(case, seed):
    return {"linear": _exact_linear, "shared": _exact_shared, "logits": _exact_logits}[case["kind"]](prepare(case, seed))
