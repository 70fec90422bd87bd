"""The operators of a 4-bit paged K/V cache whose rows are weighed and evicted, as a serving loop calls them.

* "append": `Context.pagedAttnPrologue4`: the rows of a step, a prompt or a mixed batch get their norms and rotation; q goes
            on to the attention, k and v into the pages as 4-bit floats (e2m1) with a power-of-two scale per 32 dims;
* "attend": `Context.pagedAttn4`: attention over such pages, one row per sequence (a decode step) or many;
* "weigh":  the same call where it also adds up, for each cached row, the attention weight that it got;
* "evict":  `Context.kvEvict4`: of every sequence that has outgrown its budget, the first rows, the latest and the
            heaviest others are kept and moved together.

Where `own` is false, `run` computes the same with elementary torch operations.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
F64 = torch.float64
LEAST = -20  # the least exponent of a scale


def listed():
    return [
        # a decode step's append: one row for each of a full server's sequences, whose caches have lost rows; q/k/v as
        # the split-K partial sums of their projections
        {"name": "append4-step-64", "kind": "append", "sequences": 64, "longest": 4096, "rows": 1, "parts": 3,
         "heads": 8, "kv": 1, "dim": 256, "page": 16, "gone": 3000},
        # a whole prompt's append in a global layer
        {"name": "append4-prompt-1900", "kind": "append", "sequences": 1, "longest": 1900, "rows": 1900, "parts": 1,
         "heads": 8, "kv": 1, "dim": 512, "page": 16, "gone": 0},
        # one chat's token in a window layer: the smallest call
        {"name": "attend4-1", "kind": "attend", "sequences": 1, "longest": 777, "rows": 1, "window": 512, "heads": 8,
         "kv": 1, "dim": 256, "page": 16},
        # a full server's step over ragged contexts
        {"name": "attend4-64", "kind": "attend", "sequences": 64, "longest": 8192, "rows": 1, "window": 0, "heads": 8,
         "kv": 1, "dim": 256, "page": 16},
        # a step over long documents in a global layer
        {"name": "attend4-32-long", "kind": "attend", "sequences": 32, "longest": 32000, "rows": 1, "window": 0,
         "heads": 8, "kv": 1, "dim": 512, "page": 16},
        # a few drafted tokens of each sequence to verify, two K/V heads
        {"name": "attend4-verify-13", "kind": "attend", "sequences": 13, "longest": 3001, "rows": 4, "window": 1024,
         "heads": 8, "kv": 2, "dim": 128, "page": 32},
        # chunks of several prompts over earlier turns, in a window layer
        {"name": "attend4-mixed-6", "kind": "attend", "sequences": 6, "longest": 4100, "rows": 601, "window": 512,
         "heads": 8, "kv": 1, "dim": 256, "page": 16},
        # a full server's step in a global layer whose rows are weighed
        {"name": "weigh-64", "kind": "weigh", "sequences": 64, "longest": 4352, "rows": 1, "window": 0, "heads": 8,
         "kv": 1, "dim": 512, "page": 16},
        # a whole prompt whose rows are weighed, to be cut down to a budget afterwards
        {"name": "weigh-prompt-1500", "kind": "weigh", "sequences": 1, "longest": 1500, "rows": 1500, "window": 0,
         "heads": 8, "kv": 1, "dim": 512, "page": 16},
        # one chat that has outgrown its budget
        {"name": "evict-1", "kind": "evict", "sequences": 1, "longest": 2304, "keep": 2048, "first": 4, "recent": 512,
         "kv": 1, "dim": 512, "page": 16},
        # a full server, most of whose sequences have
        {"name": "evict-64", "kind": "evict", "sequences": 64, "longest": 1280, "keep": 1024, "first": 4,
         "recent": 256, "kv": 1, "dim": 256, "page": 16},
        # long prompts cut down at once, two K/V heads that each keep their own rows
        {"name": "evict-8-long", "kind": "evict", "sequences": 8, "longest": 32000, "keep": 4000, "first": 16,
         "recent": 1000, "kv": 2, "dim": 128, "page": 32},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "weigh", "evict"))
    heads, kv = rng.choice(((8, 1), (8, 1), (8, 2), (4, 1), (16, 4), (4, 4)))
    c = {"kind": kind, "kv": kv, "dim": rng.choice((64, 128, 256, 256, 512)), "page": rng.choice((16, 16, 32, 64))}
    if kind == "evict":
        keep = _log_int(rng, 40, 4000)
        first, recent = rng.choice((0, 1, 4, 16)), rng.choice((0, keep // 8, keep // 4, keep // 2))
        c.update(sequences=_log_int(rng, 1, 64), keep=keep, first=first, recent=min(recent, keep - first),
                 longest=keep + rng.choice((1, 64, 256, keep, 7 * keep)))
        c["sequences"] = max(1, min(c["sequences"], 16000000 // (keep * kv * c["dim"]), 250000 // c["longest"]))
        return c
    c["heads"] = heads
    form = rng.choice(("step", "step", "verify", "prompt", "mixed"))
    if form == "step":
        c.update(sequences=_log_int(rng, 1, 64), longest=_log_int(rng, 100, 9000), rows=1)
    elif form == "verify":
        c.update(sequences=_log_int(rng, 1, 32), longest=_log_int(rng, 100, 5000), rows=rng.randint(2, 8))
    elif form == "prompt":
        c.update(sequences=1, rows=_log_int(rng, 9, 1500))
        c["longest"] = c["rows"] + rng.choice((0, 0, _log_int(rng, 1, 1500)))
    else:
        c.update(sequences=rng.randint(2, 8), longest=_log_int(rng, 300, 2900), rows=_log_int(rng, 9, 290))
    if kind == "append":
        c.update(parts=rng.choice((1, 1, 2, 3, 6)), gone=rng.choice((0, 0, 1, 1000)))
    else:
        c["window"] = rng.choice((0, 0, 512, 1024, 333))
    return c


# ---- inputs, from the seed alone ------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(c):
    """Each sequence's length at the call and its new rows, in an order of their own: spread over their logarithms, or
    (evict) from the longest to a little below the budget."""
    n = c["sequences"]
    if n == 1:
        return np.array([c["longest"]]), np.array([c.get("rows", 1)])
    rs = np.random.RandomState(n + 64 * c["longest"] % 65521)
    f = np.arange(n) / (n - 1)
    least = c["keep"] / c["longest"] * 0.8 if c["kind"] == "evict" else 1 / 16
    lens = np.maximum(1, np.round(c["longest"] * least ** f)).astype(np.int64)
    rows = np.maximum(1, np.round(c.get("rows", 1) ** f)).astype(np.int64)
    lens, rows = lens[rs.permutation(n)], rows[rs.permutation(n)]
    return np.maximum(lens, rows), rows


def _encode(x):
    """Codes of x [..., dim], two a byte, and the exponents of its blocks: the least from LEAST on with |x| <= 7 * 2^e."""
    b = x.unflatten(-1, (-1, 32))
    largest = b.abs().amax(-1)
    m, e = torch.frexp(largest)
    e = torch.where(largest > 0, e - 3 + (m > 0.875).int(), e.new_tensor(LEAST)).clamp_min(LEAST)
    y = b.abs() * torch.exp2(-e.to(x.dtype))[..., None]
    c = torch.where(y < 2, torch.round(2 * y), torch.where(y < 4, torch.round(y) + 2, torch.round(y / 2) + 4))
    c = (c.clamp_max(7).to(torch.uint8) | (torch.signbit(b).to(torch.uint8) << 3)).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), e


def _by_tile(e, page):
    """V's scales: sixteen rows of a block next to each other."""
    return e.unflatten(1, (page // 16, 16)).permute(0, 1, 3, 4, 2).contiguous()


def _by_row(scale):
    return scale.permute(0, 1, 4, 2, 3).flatten(1, 2)


def _paged(c, seed):
    """The page lists and lengths of a batch, and a 4-bit pool: rows near N(0, 1) as the norms leave them, some dims and
    rows smaller and larger."""
    g = _gen(seed)
    lens, rows = _lengths(c)
    ps, kv, dim = c["page"], c["kv"], c["dim"]
    per = -(-lens // ps)
    total = int(per.sum()) + 3
    order = torch.randperm(total, device=DEV, generator=g)[:total - 3].int()
    width = int(per.max())
    valid = torch.from_numpy(np.arange(width)[None, :] < per[:, None]).to(DEV)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    table[valid] = order
    s = {"case": c, "table": table, "lens": torch.from_numpy(lens.astype(np.int32)).to(DEV),
         "starts": torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).to(DEV)}
    for name in "kv":
        x = torch.randn(total, ps, kv, dim, device=DEV, generator=g)
        x.mul_(torch.exp2(torch.randint(-1, 2, (dim,), device=DEV, generator=g).float() / 2))
        s[name + "_pool"], e = _encode(x)
        e = (e + 127).to(torch.uint8)
        s[name + "_scale"] = e.contiguous() if name == "k" else _by_tile(e, ps)
    # what a few earlier steps have added up: some heavy rows, some that got nothing
    s["mass"] = torch.randn(total, ps, kv, device=DEV, generator=g).mul_(2).exp_().mul_(2.0 ** -9)
    s["mass"].mul_(torch.rand(total, ps, kv, device=DEV, generator=g) > 0.1)
    return s, lens, rows, g


def _pages_of(s, first, last):
    """The ids of each sequence's pages first .. last of its list, one after the other."""
    n = last - first + 1
    which = np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n) + np.repeat(first, n)
    return s["table"][torch.from_numpy(np.repeat(np.arange(len(n)), n)).to(DEV), torch.from_numpy(which).to(DEV)].contiguous()


def prepare(case, seed):
    c = case
    s, lens, rows, g = _paged(c, seed)
    kv, dim, ps = c["kv"], c["dim"], c["page"]
    if c["kind"] == "evict":
        s["before"] = s["lens"].clone()
        s["kept"] = torch.zeros(len(lens), kv, c["keep"], dtype=torch.int32, device=DEV)
        s["touched"] = _pages_of(s, 0 * lens, (np.minimum(lens, c["keep"]) - 1) // ps)
    else:
        r, h = int(rows.sum()), c["heads"]
        if c["kind"] == "append":
            for name, n in (("q", h), ("k", kv), ("v", kv)):
                s[name] = torch.randn(c["parts"], r, n, dim, device=DEV, generator=g)
            for name in ("q_w", "k_w"):
                s[name] = (1 + 0.1 * torch.randn(dim, device=DEV, generator=g)).half()
            s["positions"] = s["lens"] + c["gone"]
            t = torch.arange(int(lens.max()) + c["gone"], device=DEV, dtype=F64)
            angle = t[:, None] * 10000.0 ** (-2 * torch.arange(dim // 2, device=DEV, dtype=F64) / dim)[None, :]
            s["rope"] = torch.stack([angle.cos(), angle.sin()], 2).float().contiguous()
            s["touched"] = _pages_of(s, (lens - rows) // ps, (lens - 1) // ps)
        else:
            s["q"] = torch.randn(r, h, dim, device=DEV, generator=g) * (2 / math.sqrt(dim))
        s["out"] = torch.zeros(r, h, dim, device=DEV)
    if "touched" in s:
        s["values"] = torch.zeros(2, s["touched"].numel(), ps, kv, dim, dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------

_kept = {}


def _context():
    """One context and one workspace, kept as a serving program keeps them. Its calls go to a stream of the context's
    own, which torch's work neither waits for nor is waited for by: `prepare` ends with a wait for the device, and who
    reads a pass's outputs waits first."""
    if "ctx" not in _kept:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "gemma4-webgpu_amd"))
        from g4hip import Context
        _kept["ctx"], _kept["ws"] = Context(0), None
    return _kept["ctx"]


def _workspace(ctx, nbytes):
    if _kept["ws"] is None or _kept["ws"].nbytes < nbytes:
        _kept["ws"] = ctx.alloc(nbytes)
    return _kept["ws"]


def _run_own(s):
    ctx, c = _context(), s["case"]
    p = torch.Tensor.data_ptr
    n, width = s["table"].shape
    cache = (p(s["k_pool"]), p(s["v_pool"]), p(s["k_scale"]), p(s["v_scale"]))
    par = ctx.kv4_params(n, c.get("heads", c["kv"]), c["kv"], c["dim"], c["page"], width, c["longest"],
                         s["k_pool"].shape[0], num_rows=s["out"].shape[0] if "out" in s else n, max_rows=c.get("rows", 1),
                         window=c.get("window", 0), eps=EPS)
    starts = p(s["starts"]) if c.get("rows", 1) > 1 else None

    def values():
        k, v = s["values"]
        ctx.kv4Values(*cache, p(s["touched"]), s["touched"].numel(), c["page"], c["kv"], c["dim"], s["k_pool"].shape[0],
                      p(k), p(v))
        return [k, v]

    if c["kind"] == "evict":
        ctx.copy(p(s["lens"]), p(s["before"]), 4 * n)
        ctx.kvEvict4(*cache, p(s["mass"]), p(s["table"]), p(s["lens"]), par, c["keep"], c["first"], c["recent"],
                     p(s["kept"]), _workspace(ctx, ctx.evict4_workspace_bytes(par, c["keep"])))
        return [s["kept"], s["lens"], s["mass"]] + values()
    if c["kind"] == "append":
        ctx.pagedAttnPrologue4(p(s["q"]), p(s["k"]), p(s["v"]), c["parts"], p(s["q_w"]), p(s["k_w"]), None, p(s["out"]),
                               *cache, p(s["table"]), p(s["lens"]), par, row_starts=starts,
                               positions=p(s["positions"]) if c["gone"] else None, mass=p(s["mass"]),
                               rope_cs=p(s["rope"]), rope_rows=s["rope"].shape[0])
        return [s["out"], s["mass"]] + values()
    weigh = c["kind"] == "weigh"
    ctx.pagedAttn4(p(s["q"]), *cache, p(s["table"]), p(s["lens"]), p(s["out"]), par,
                   _workspace(ctx, ctx.attn4_workspace_bytes(par, mass=weigh)), row_starts=starts,
                   mass=p(s["mass"]) if weigh else None)
    return [s["out"], s["mass"]] if weigh else s["out"]


# ---- the plain forms ------------------------------------------------------------------------------------------------

_PAIRS = {}


def _decode(codes, e):
    """Values of codes [..., dim / 2] with the scales' exponents [..., dim / 32]."""
    if "of" not in _PAIRS:
        v = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=DEV)
        v = torch.cat([v, -v])
        b = torch.arange(256, device=DEV)
        _PAIRS["of"] = torch.stack([v[b & 15], v[b >> 4]], 1)
    x = _PAIRS["of"][codes.int()].flatten(-2)
    return (x.unflatten(-1, (-1, 32)) * torch.exp2(e.float())[..., None]).flatten(-2)


def _values_of(s, pages):
    """K and V values of the pages of an index tensor, in float32."""
    k = _decode(s["k_pool"][pages], s["k_scale"][pages].int() - 127)
    return k, _decode(s["v_pool"][pages], _by_row(s["v_scale"][pages.flatten()].int() - 127).unflatten(0, pages.shape))


def _rows(s):
    """Each row's sequence and place in it, each sequence's first new place."""
    starts, lens = s["starts"].long(), s["lens"].long()
    r = torch.arange(s["out"].shape[0], device=DEV)
    seq = torch.bucketize(r, starts[1:], right=True)
    base = lens - (starts[1:] - starts[:-1])
    return seq, base[seq] + r - starts[seq], base


def _normed(x, w=None):
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
    return y if w is None else y * w.to(x.dtype)


def _rotated(x, cs):
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    c, s = cs[:, None, :, 0].to(x.dtype), cs[:, None, :, 1].to(x.dtype)
    return torch.cat([lo * c - hi * s, lo * s + hi * c], -1)


def _run_append(s):
    seq, at, _ = _rows(s)
    ps, cs = s["case"]["page"], s["rope"][at + s["case"]["gone"]]
    q = _rotated(_normed(s["q"].sum(0), s["q_w"]), cs)
    # (codes in 64 bits: a value next to the border of two)
    k = _rotated(_normed(s["k"].double().sum(0), s["k_w"]), cs)
    v = _normed(s["v"].double().sum(0))
    page, slot = s["table"].long()[seq, at // ps], at % ps
    s["k_pool"][page, slot], e = _encode(k)
    s["k_scale"][page, slot] = (e + 127).to(torch.uint8)
    s["v_pool"][page, slot], e = _encode(v)
    s["v_scale"][page, slot // 16, :, :, slot % 16] = (e + 127).to(torch.uint8)
    s["mass"][page, slot] = 0
    k, v = _values_of(s, s["touched"].long())
    return [q, s["mass"], k.half(), v.half()]


def _run_attend(s):
    c = s["case"]
    n, most, kv, dim, ps = c["sequences"], c["rows"], c["kv"], c["dim"], c["page"]
    g = c["heads"] // kv
    table = s["table"].long()
    k, v = (x.view(n, -1, kv, dim).transpose(1, 2).contiguous() for x in _values_of(s, table.clamp_min(0)))
    seq, pos, base = _rows(s)
    i = torch.arange(most, device=DEV)
    at = (s["starts"][:-1, None].long() + i).clamp_max(pos.numel() - 1)
    q = s["q"][at].view(n, most, kv, g, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, most * g, dim)
    x = (q @ k.transpose(2, 3)).view(n, kv, most, g, -1)
    t, p = torch.arange(x.shape[-1], device=DEV), (base[:, None] + i)[:, None, :, None, None]
    dead = t > p
    if c["window"]:
        dead = dead | (t <= p - c["window"])
    x = x.masked_fill(dead, -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    z = w.sum(-1, keepdim=True).clamp_min(1e-38)
    o = (w.view(n, kv, most * g, -1) @ v).view(n, kv, most, g, dim) / z
    o = o.permute(0, 2, 1, 3, 4).reshape(n, most, kv * g, dim)[seq, pos - base[seq]]
    if c["kind"] == "attend":
        return o
    mine = (i < (s["starts"][1:] - s["starts"][:-1])[:, None])[:, None, :, None, None]
    more = torch.where(mine, w / z, 0.0).double().sum((2, 3)).float()  # [sequence][K/V head][place]
    more = more.transpose(1, 2).unflatten(1, (-1, ps))
    s["mass"][table[table >= 0]] += more[table >= 0]
    return [o, s["mass"]]


def _run_evict(s):
    c = s["case"]
    n, kv, keep, ps = c["sequences"], c["kv"], c["keep"], c["page"]
    s["lens"].copy_(s["before"])
    lens, table = s["lens"].long()[:, None, None], s["table"].long()
    mass = s["mass"][table.clamp_min(0)].view(n, -1, kv).transpose(1, 2)
    t = torch.arange(mass.shape[2], device=DEV)
    # the order of the rows, equal masses by their place: one whole number of both; kept rows before it, none behind
    key = torch.where(mass > 0, mass, 0.0).view(torch.int32).long() * 2 ** 31 - t
    key = torch.where((t < c["first"]) | (t >= lens - c["recent"]), 2 ** 62, key)
    key = torch.where(t < lens, key, -2 ** 62)
    best = torch.topk(key, min(keep, mass.shape[2]), dim=2).indices
    chosen = torch.zeros_like(key, dtype=torch.bool).scatter_(2, best, True) & (t < lens)
    src = torch.sort(torch.where(chosen, t, 2 ** 40), dim=2).values[:, :, :keep]
    full = src.new_full((n, kv, keep), 2 ** 40)
    full[:, :, :src.shape[2]] = src
    s["kept"].copy_(torch.where(full < 2 ** 40, full, -1))
    over = (lens > keep)[:, 0, 0]
    i = torch.arange(keep, device=DEV)
    head = torch.arange(kv, device=DEV)[None, :, None]
    src = full[over]
    from_, to = table[over].gather(1, (src // ps).flatten(1)).view(src.shape), table[over][:, None, i // ps]
    a, b = src % ps, (i % ps)[None, None, :]
    for name in ("k_pool", "v_pool", "k_scale", "mass"):
        s[name][to, b, head] = s[name][from_, a, head]
    s["v_scale"][to, b // 16, head, :, b % 16] = s["v_scale"][from_, a // 16, head, :, a % 16]
    s["lens"].clamp_(max=keep)
    k, v = _values_of(s, s["touched"].long())
    return [s["kept"], s["lens"], s["mass"], k.half(), v.half()]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return {"append": _run_append, "attend": _run_attend, "weigh": _run_attend, "evict": _run_evict}[kind](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    c = case
    lens, rows = _lengths(c)
    kv, dim, ps = c["kv"], c["dim"], c["page"]
    row = kv * (dim + dim // 16)  # bytes of K and V of a cached row
    if c["kind"] == "evict":  # masses; rows that move, read and written; the values that come back, and their codes
        over = lens[lens > c["keep"]]
        pages = int((-(-np.minimum(lens, c["keep"]) // ps)).sum())
        moved = len(over) * (c["keep"] - c["first"])
        return {"bytes": 4.0 * kv * int(over.sum()) + 2.0 * moved * (row + 4 * kv) + pages * ps * (row + 4.0 * kv * dim)
                + 4.0 * len(lens) * kv * c["keep"], "flops": 0.0}
    r, h = int(rows.sum()), c["heads"]
    if c["kind"] == "append":  # the parts, q, the codes; the values that come back of the pages, and their codes
        pages = int(((lens - 1) // ps + 1 - (lens - rows) // ps).sum())
        return {"bytes": 4.0 * c["parts"] * r * (h + 2 * kv) * dim + 4.0 * r * h * dim + r * (row + 4.0 * kv)
                + pages * ps * (row + 4.0 * kv * dim) + 4.0 * r * dim, "flops": 8.0 * r * (h + 2 * kv) * dim}
    seen = read = 0
    for n, m in zip(lens.tolist(), rows.tolist()):
        ends = np.arange(n - m + 1, n + 1)
        spans = np.minimum(ends, c["window"]) if c["window"] else ends
        seen += int(spans.sum())
        read += n - int(max(0, n - m + 1 - c["window"])) if c["window"] else n
    weigh = c["kind"] == "weigh"
    return {"bytes": 1.0 * read * (row + (8 * kv if weigh else 0)) + 8.0 * r * h * dim, "flops": 4.0 * seen * h * dim}


# ---- the same in float64 --------------------------------------------------------------------------------------------

_LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
_BORDERS = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5])


def _host(s):
    """The pools as values in float64: [page][row][head][dim]."""
    out = []
    for name in "kv":
        codes, scale = s[name + "_pool"].cpu().numpy(), s[name + "_scale"].cpu().numpy().astype(np.float64)
        if name == "v":
            pages, tiles, kv, blocks, _ = scale.shape
            scale = np.moveaxis(scale, 4, 2).reshape(pages, 16 * tiles, kv, blocks)
        x = np.empty(codes.shape[:-1] + (2 * codes.shape[-1],))
        x[..., ::2], x[..., 1::2] = _LEVELS[codes & 15], _LEVELS[codes >> 4]
        out.append(x * np.repeat(2.0 ** (scale - 127), 32, -1))
    return out


def _exact_append(s):
    c = s["case"]
    ps, half = c["page"], c["dim"] // 2
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist()
    q, k, v = (s[n].to(F64).sum(0) for n in "qkv")
    q, k, v = (x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS).sqrt() for x in (q, k, v))
    q, k = q * s["q_w"].to(F64), k * s["k_w"].to(F64)
    where = torch.cat([torch.arange(n - (b - a), n) for n, a, b in zip(lens, starts, starts[1:])]).to(DEV) + c["gone"]
    turn = torch.view_as_complex(s["rope"].to(F64))[where][:, None]
    q, k = (torch.view_as_real(torch.complex(x[..., :half], x[..., half:]) * turn) for x in (q, k))
    q, k = (torch.cat([x[..., 0], x[..., 1]], -1) for x in (q, k))
    mass, pools = s["mass"].to(F64).cpu().numpy(), _host(s)
    for x, pool in ((k.cpu().numpy(), pools[0]), (v.cpu().numpy(), pools[1])):
        b = x.reshape(x.shape[:-1] + (-1, 32))
        e = np.maximum(np.ceil(np.log2(np.maximum(np.abs(b).max(-1), 1e-30) / 7)), LEAST)
        y = b / 2.0 ** e[..., None]
        a = np.abs(y)
        near = np.searchsorted(_BORDERS, a) + np.isin(a, (.75, 1.75, 3.5))
        x = (np.where(y < 0, -1, 1) * _LEVELS[near] * 2.0 ** e[..., None]).reshape(x.shape)
        for i, n in enumerate(lens):
            for r in range(starts[i], starts[i + 1]):
                t = n - starts[i + 1] + r
                pool[table[i][t // ps], t % ps] = x[r]
                mass[table[i][t // ps], t % ps] = 0
    at = s["touched"].cpu().numpy()
    return [q, torch.from_numpy(mass)] + [torch.from_numpy(x[at]) for x in pools]


def _exact_attend(s):
    c, out = s["case"], torch.empty_like(s["q"], dtype=F64)
    starts, lens, mass = s["starts"].tolist(), s["lens"].tolist(), s["mass"].to(F64)
    g, ps = c["heads"] // c["kv"], c["page"]
    level = torch.from_numpy(_LEVELS).to(DEV)
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        first = max(0, n - (b - a) + 1 - c["window"]) if c["window"] else 0
        pages = s["table"][i][first // ps:-(-n // ps)].long()
        t = torch.arange(n, device=DEV)[first // ps * ps:]
        p = torch.arange(n - (b - a), n, device=DEV)
        see = t[None, :] <= p[:, None]
        if c["window"]:
            see &= t[None, :] > p[:, None] - c["window"]
        for h in range(c["kv"]):
            x = []
            for name in "kv":
                codes, e = s[name + "_pool"][pages][:, :, h].long(), s[name + "_scale"][pages]
                e = e[:, :, h] if name == "k" else e[:, :, h].transpose(2, 3).flatten(1, 2)
                y = torch.stack([level[codes & 15], level[codes >> 4]], -1).flatten(-2)
                x.append((y * torch.exp2(e.to(F64) - 127).repeat_interleave(32, -1)).view(-1, c["dim"])[:len(t)])
            got = torch.zeros(len(t), dtype=F64, device=DEV)
            for j in range(h * g, (h + 1) * g):
                y = s["q"][a:b, j].to(F64) @ x[0].T
                y = torch.softmax(torch.where(see, y, torch.full_like(y, -math.inf)), 1)
                out[a:b, j] = y @ x[1]
                got += y.sum(0)
            mass[pages[(t // ps) - first // ps], t % ps, h] += got
    return [out, mass] if c["kind"] == "weigh" else out


def _exact_evict(s):
    c, pools = s["case"], _host(s)
    ps, keep = c["page"], c["keep"]
    table, mass = s["table"].cpu().numpy(), s["mass"].to(F64).cpu().numpy()
    lens = s["before"].cpu().numpy().copy()
    kept = np.full((len(lens), c["kv"], keep), -1, np.int32)
    for i, n in enumerate(lens):
        t = np.arange(n)
        pages, slots = table[i][t // ps], t % ps
        for h in range(c["kv"]):
            if n <= keep:
                kept[i, h, :n] = t
                continue
            middle = t[c["first"]:n - c["recent"]]
            heavy = middle[np.argsort(-mass[pages, slots, h][middle], kind="stable")[:keep - c["first"] - c["recent"]]]
            src = np.concatenate([t[:c["first"]], np.sort(heavy), t[n - c["recent"]:]])
            kept[i, h] = src
            for x in (*pools, mass):
                x[pages[:keep], slots[:keep], h] = x[pages[src], slots[src], h]
        lens[i] = min(n, keep)
    at = s["touched"].cpu().numpy()
    return [torch.from_numpy(x) for x in (kept, lens, mass, *(x[at] for x in pools))]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    return {"append": _exact_append, "attend": _exact_attend, "weigh": _exact_attend, "evict": _exact_evict}[kind](s)
