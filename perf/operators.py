"""The operators of an 8-bit paged K/V cache, and log probabilities of tokens, as a serving loop calls them.

* "append":   `Context.pagedAttnPrologue8`: the rows of a step, a prompt or a mixed batch get their norms and rotation; q
              goes on to the attention, k and v into the pages as 8-bit codes with a power-of-two scale per page and head;
* "attend":   `Context.pagedAttn8`: attention over such pages, one row per sequence (a decode step) or many (a prompt, a
              mixed batch, drafted tokens to verify);
* "logprobs": `Context.logprobsBatch`: log probability of a given token per row of logits, entropy, top alternatives.

Where `own` is false, `run` computes the same with elementary torch operations.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
VOCAB = 262144
EPS = 1e-6
F64 = torch.float64


def listed():
    return [
        # a decode step's append: one row for each of a full server's sequences, q/k/v as the split-K partial sums of
        # their projections
        {"name": "append-step-64", "kind": "append", "sequences": 64, "longest": 8192, "rows": 1, "parts": 3,
         "heads": 8, "kv": 1, "dim": 256, "page": 16},
        # a whole prompt's append in a global layer
        {"name": "append-prompt-1900", "kind": "append", "sequences": 1, "longest": 1900, "rows": 1900, "parts": 1,
         "heads": 8, "kv": 1, "dim": 512, "page": 16},
        # chunks of several prompts at once, begun in the middle of pages
        {"name": "append-mixed-7", "kind": "append", "sequences": 7, "longest": 2100, "rows": 301, "parts": 2,
         "heads": 8, "kv": 2, "dim": 128, "page": 32},
        # one chat's token in a window layer: the smallest call
        {"name": "attend-1", "kind": "attend", "sequences": 1, "longest": 777, "rows": 1, "window": 512, "heads": 8,
         "kv": 1, "dim": 256, "page": 16},
        # a full server's step over ragged contexts
        {"name": "attend-64", "kind": "attend", "sequences": 64, "longest": 8192, "rows": 1, "window": 0, "heads": 8,
         "kv": 1, "dim": 256, "page": 16},
        # a step over long documents in a global layer
        {"name": "attend-32-long", "kind": "attend", "sequences": 32, "longest": 32000, "rows": 1, "window": 0,
         "heads": 8, "kv": 1, "dim": 512, "page": 16},
        # a few drafted tokens of each sequence to verify, two K/V heads
        {"name": "attend-verify-13", "kind": "attend", "sequences": 13, "longest": 3001, "rows": 4, "window": 1024,
         "heads": 8, "kv": 2, "dim": 128, "page": 32},
        # a whole prompt in a global layer
        {"name": "attend-prompt-1900", "kind": "attend", "sequences": 1, "longest": 1900, "rows": 1900, "window": 0,
         "heads": 8, "kv": 1, "dim": 512, "page": 16},
        # chunks of several prompts over earlier turns, in a window layer
        {"name": "attend-mixed-6", "kind": "attend", "sequences": 6, "longest": 4100, "rows": 601, "window": 512,
         "heads": 8, "kv": 1, "dim": 256, "page": 16},
        # the sampled token of one chat with a few alternatives
        {"name": "logprobs-1", "kind": "logprobs", "rows": 1, "vocab": VOCAB, "top": 5},
        # a full server's step, the most alternatives an interface gives
        {"name": "logprobs-64", "kind": "logprobs", "rows": 64, "vocab": VOCAB, "top": 20},
        # a text's tokens scored, another vocabulary
        {"name": "logprobs-score-500", "kind": "logprobs", "rows": 500, "vocab": 100003, "top": 1},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "logprobs"))
    if kind == "logprobs":
        vocab = rng.choice((VOCAB, VOCAB, _log_int(rng, 1000, VOCAB)))
        return {"kind": kind, "rows": _log_int(rng, 1, min(4000, 60000000 // vocab)), "vocab": vocab,
                "top": rng.choice((0, 1, 5, 20, 32))}
    heads, kv = rng.choice(((8, 1), (8, 1), (8, 2), (4, 1), (16, 4), (4, 4)))
    c = {"kind": kind, "heads": heads, "kv": kv, "dim": rng.choice((64, 128, 256, 256, 512)),
         "page": rng.choice((16, 16, 32, 64))}
    form = rng.choice(("step", "step", "verify", "prompt", "mixed"))
    if form == "step":
        c.update(sequences=_log_int(rng, 1, 64), longest=_log_int(rng, 100, 9000), rows=1)
    elif form == "verify":
        c.update(sequences=_log_int(rng, 1, 32), longest=_log_int(rng, 100, 5000), rows=rng.randint(2, 8))
    elif form == "prompt":
        c.update(sequences=1, rows=_log_int(rng, 9, 1500))
        c["longest"] = c["rows"] + rng.choice((0, 0, _log_int(rng, 1, 1500)))
    else:
        c.update(sequences=rng.randint(2, 8), longest=_log_int(rng, 300, 3000), rows=_log_int(rng, 9, 290))
    if kind == "append":
        c["parts"] = rng.choice((1, 1, 2, 3, 6))
    else:
        c["window"] = rng.choice((0, 0, 512, 1024, 333))
    return c


# ---- inputs, from the seed alone ------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(c):
    """Each sequence's length after the call and its new rows: spread over their logarithms, in an order of their own."""
    n = c["sequences"]
    if n == 1:
        return np.array([c["longest"]]), np.array([c["rows"]])
    rs = np.random.RandomState(n + 64 * c["longest"] % 65521)
    f = np.arange(n) / (n - 1)
    lens = np.round(c["longest"] * 16.0 ** -f).astype(np.int64)
    rows = np.maximum(1, np.round(c["rows"] ** f)).astype(np.int64)
    lens, rows = lens[rs.permutation(n)], rows[rs.permutation(n)]
    return np.maximum(lens, rows), rows


def _paged(c, seed):
    """The page lists, lengths and row starts of a batch, and an 8-bit pool with its scales."""
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
    pools = []
    for _ in range(2):  # values near N(0, 1) as the norms leave them; pages of smaller and larger values among them
        e = torch.randint(4, 7, (total, kv), device=DEV, generator=g)
        codes = torch.randn(total, ps, kv, dim, device=DEV, generator=g).mul_(torch.exp2(e.float())[:, None, :, None])
        pools += [codes.round_().clamp_(-127, 127).to(torch.int8), torch.exp2(-e.float())]
    s = {"k_pool": pools[0], "k_scale": pools[1], "v_pool": pools[2], "v_scale": pools[3], "table": table,
         "lens": torch.from_numpy(lens.astype(np.int32)).to(DEV),
         "starts": torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).to(DEV)}
    return s, lens, rows, g


def prepare(case, seed):
    c = case
    if c["kind"] == "logprobs":
        g = _gen(seed)
        n, v = c["rows"], c["vocab"]
        # softcapped logits of a trained head: a broad bulk, a few likely tokens
        x = torch.randn(n, v, device=DEV, generator=g).mul_(2.5).sub_(4.0)
        peak = torch.randint(0, v, (n, 8), device=DEV, generator=g)
        x.scatter_add_(1, peak, torch.rand(n, 8, device=DEV, generator=g) * 16 + 4)
        x = x.div_(30).tanh_().mul_(30)
        token = torch.where(torch.rand(n, device=DEV, generator=g) < 0.7, peak[:, 0],
                            torch.randint(0, v, (n,), device=DEV, generator=g)).int()
        s = {"case": c, "logits": x, "tokens": token, "logprob": torch.zeros(n, device=DEV),
             "entropy": torch.zeros(n, device=DEV), "ids": torch.zeros(n, c["top"], dtype=torch.int32, device=DEV),
             "top": torch.zeros(n, c["top"], device=DEV)}
    else:
        s, lens, rows, g = _paged(c, seed)
        r, h, kv, dim = int(rows.sum()), c["heads"], c["kv"], c["dim"]
        s["case"] = c
        if c["kind"] == "attend":
            s["q"] = torch.randn(r, h, dim, device=DEV, generator=g) * (2 / math.sqrt(dim))
            s["out"] = torch.zeros(r, h, dim, device=DEV)
        else:
            for name, n in (("q", h), ("k", kv), ("v", kv)):
                s[name] = torch.randn(c["parts"], r, n, dim, device=DEV, generator=g)
            for name in ("q_w", "k_w"):
                s[name] = (1 + 0.1 * torch.randn(dim, device=DEV, generator=g)).half()
            t, i = torch.arange(int(lens.max()), device=DEV, dtype=F64), torch.arange(dim // 2, device=DEV, dtype=F64)
            angle = t[:, None] * 10000.0 ** (-2 * i / dim)[None, :]
            s["rope"] = torch.stack([angle.cos(), angle.sin()], 2).float().contiguous()
            first = (lens - rows) // c["page"]
            n = (lens - 1) // c["page"] + 1 - first
            which = np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n) + np.repeat(first, n)
            s["touched"] = s["table"][torch.from_numpy(np.repeat(np.arange(len(lens)), n)).to(DEV),
                                      torch.from_numpy(which).to(DEV)].contiguous()
            s["q_out"] = torch.zeros(r, h, dim, device=DEV)
            s["values"] = torch.zeros(2, len(which), c["page"], kv, dim, dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------

_kept = {}


def _context():
    """One context and one workspace, kept as a serving program keeps them. Its calls go to a stream of the context's
    own, which torch's work neither waits for nor is waited for by: `prepare` ends with a wait for the device, and who
    reads a pass's outputs waits first. A program without such waits has torch and the context on one stream
    (Context.set_stream with a torch.cuda.Stream's handle; the default stream's, 0, stands for the context's own)."""
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


def _params(ctx, s, window=0):
    c = s["case"]
    n, width = s["table"].shape
    return ctx.kv8_params(n, c["heads"], c["kv"], c["dim"], c["page"], width, c["longest"],
                          s["k_pool"].shape[0], num_rows=s["q"].shape[-3], max_rows=c["rows"], window=window, eps=EPS)


def _run_own(s):
    ctx, c = _context(), s["case"]
    p = torch.Tensor.data_ptr
    if c["kind"] == "logprobs":
        ws = _workspace(ctx, ctx.logprobs_workspace_bytes(c["vocab"], c["rows"], c["top"]))
        ctx.logprobsBatch(p(s["logits"]), p(s["tokens"]), c["vocab"], c["rows"], p(s["logprob"]), p(s["entropy"]),
                          c["top"], p(s["ids"]), p(s["top"]), ws)
        return [s["logprob"], s["entropy"], s["ids"], s["top"]]
    cache = (p(s["k_pool"]), p(s["v_pool"]), p(s["k_scale"]), p(s["v_scale"]))
    starts = p(s["starts"]) if c["rows"] > 1 else None
    if c["kind"] == "attend":
        par = _params(ctx, s, c["window"])
        ctx.pagedAttn8(p(s["q"]), *cache, p(s["table"]), p(s["lens"]), p(s["out"]), par,
                       _workspace(ctx, ctx.attn8_workspace_bytes(par)), row_starts=starts)
        return s["out"]
    ctx.pagedAttnPrologue8(p(s["q"]), p(s["k"]), p(s["v"]), c["parts"], p(s["q_w"]), p(s["k_w"]), None, p(s["q_out"]),
                           *cache, p(s["table"]), p(s["lens"]), _params(ctx, s), row_starts=starts,
                           rope_cs=p(s["rope"]), rope_rows=s["rope"].shape[0])
    k, v = s["values"]
    ctx.kv8Values(*cache, p(s["touched"]), s["touched"].numel(), c["page"], c["kv"], c["dim"], s["k_pool"].shape[0],
                  p(k), p(v))
    return [s["q_out"], k, v]


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _rows(s):
    """Each row's sequence and position, each sequence's first new position."""
    starts, lens = s["starts"].long(), s["lens"].long()
    r = torch.arange(s["q"].shape[-3], device=DEV)
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


def _scale_of(largest):
    """The least power of two times 127 that is not below `largest`, from the exponent of it: 2^e."""
    m, x = torch.frexp(largest)
    e = x - 7 + (m > 127 / 128).int()
    return torch.exp2(torch.where(largest > 0, e, e.new_tensor(-64)).clamp_min(-64).float())


def _store(s, pool, scale, x, page, slot):
    """Codes of the new rows (decided in 64 bits: a value next to a border) and of the rows before them in their pages."""
    pages, ps = pool.shape[:2]
    kv = pool.shape[2]
    largest = torch.zeros(pages, kv, dtype=F64, device=DEV).scatter_reduce_(
        0, page[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
    first = torch.full((pages,), ps, device=DEV).scatter_reduce_(0, page, slot, "amin")
    t = s["touched"].long()
    new = _scale_of(largest[t])
    begun = (first[t] == 0)[:, None]
    new = torch.where(begun, new, torch.maximum(new, scale[t]))
    again = torch.round(pool[t].float() * (scale[t] / new)[:, None, :, None]).to(torch.int8)
    earlier = torch.arange(ps, device=DEV)[None, :] < first[t][:, None]
    pool[t] = torch.where(earlier[:, :, None, None], again, pool[t])
    scale[t] = new
    pool[page, slot] = torch.round(x / scale[page][..., None].double()).to(torch.int8)
    return (pool[t].float() * new[:, None, :, None]).half()


def _run_append(s):
    seq, pos, _ = _rows(s)
    ps, cs = s["case"]["page"], s["rope"][pos]
    q = _rotated(_normed(s["q"].sum(0), s["q_w"]), cs)
    k = _rotated(_normed(s["k"].double().sum(0), s["k_w"]), cs)
    v = _normed(s["v"].double().sum(0))
    page, slot = s["table"].long()[seq, pos // ps], pos % ps
    return [q, _store(s, s["k_pool"], s["k_scale"], k, page, slot), _store(s, s["v_pool"], s["v_scale"], v, page, slot)]


def _run_attend(s):
    c = s["case"]
    n, most, kv, dim = c["sequences"], c["rows"], c["kv"], c["dim"]
    g = c["heads"] // kv
    table = s["table"].long().clamp_min(0)

    def dense(pool, scale):  # [sequence][K/V head][position][dim]
        x = pool[table].float() * scale[table][:, :, None, :, None]
        return x.view(n, -1, kv, dim).permute(0, 2, 1, 3).contiguous()

    seq, pos, base = _rows(s)
    i = torch.arange(most, device=DEV)
    at = (s["starts"][:-1, None].long() + i).clamp_max(pos.numel() - 1)
    q = s["q"][at].view(n, most, kv, g, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, most * g, dim)
    x = (q @ dense(s["k_pool"], s["k_scale"]).transpose(2, 3)).view(n, kv, most, g, -1)
    t, p = torch.arange(x.shape[-1], device=DEV), (base[:, None] + i)[:, None, :, None, None]
    dead = t > p
    if c["window"]:
        dead = dead | (t <= p - c["window"])
    x = x.masked_fill(dead, -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    o = (w.view(n, kv, most * g, -1) @ dense(s["v_pool"], s["v_scale"])).view(n, kv, most, g, dim)
    o = o / w.sum(-1, keepdim=True).clamp_min(1e-38)
    return o.permute(0, 2, 1, 3, 4).reshape(n, most, kv * g, dim)[seq, pos - base[seq]]


def _run_logprobs(s):
    x, n = s["logits"], s["case"]["top"]
    y = x - x.amax(1, keepdim=True)
    e = torch.exp(y)
    z = e.sum(1)
    logprob = y.gather(1, s["tokens"].long()[:, None])[:, 0] - torch.log(z)
    entropy = torch.log(z) - (e * y).sum(1) / z
    # the order of the values, equal ones by their index: one whole number of both
    bits = x.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff)) * 2 ** 31 - torch.arange(x.shape[1], device=DEV)
    best = torch.topk(order, n, dim=1, sorted=True).values
    ids = (-best) & (2 ** 31 - 1)
    return [logprob, entropy, ids.int(), y.gather(1, ids) - torch.log(z)[:, None]]


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "attend": _run_attend, "logprobs": _run_logprobs}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4.0 * n + c["rows"] * (12 + 8 * c["top"]), "flops": 6.0 * n}
    lens, rows = _lengths(c)
    r, h, kv, dim = int(rows.sum()), c["heads"], c["kv"], c["dim"]
    if c["kind"] == "append":  # the parts, q, the codes; the values that come back of the pages, and their codes
        pages = int(((lens - 1) // c["page"] + 1 - (lens - rows) // c["page"]).sum())
        back = 6.0 * pages * c["page"] * kv * dim
        return {"bytes": 4.0 * c["parts"] * r * (h + 2 * kv) * dim + 4.0 * r * h * dim + 2.0 * r * kv * dim + back
                + 4.0 * r * dim, "flops": 8.0 * r * (h + 2 * kv) * dim}
    seen = read = 0
    for n, m in zip(lens.tolist(), rows.tolist()):
        ends = np.arange(n - m + 1, n + 1)
        spans = np.minimum(ends, c["window"]) if c["window"] else ends
        seen += int(spans.sum())
        read += n - int(max(0, n - m + 1 - c["window"])) if c["window"] else n
    return {"bytes": 2.0 * read * kv * dim + 8.0 * r * h * dim, "flops": 4.0 * seen * h * dim}


# ---- the same in float64 --------------------------------------------------------------------------------------------

def _exact_append(s):
    c, out = s["case"], []
    ps, half = c["page"], c["dim"] // 2
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist()
    q, k, v = (s[n].to(F64).sum(0) for n in "qkv")
    q, k, v = (x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS).sqrt() for x in (q, k, v))
    q, k = q * s["q_w"].to(F64), k * s["k_w"].to(F64)
    where = torch.cat([torch.arange(n - (b - a), n) for n, a, b in zip(lens, starts, starts[1:])]).to(DEV)
    turn = torch.view_as_complex(s["rope"].to(F64))[where][:, None]
    q, k = (torch.view_as_real(torch.complex(x[..., :half], x[..., half:]) * turn) for x in (q, k))
    q, k = (torch.cat([x[..., 0], x[..., 1]], -1) for x in (q, k))
    out.append(q)
    for x, pool, scale in ((k, s["k_pool"], s["k_scale"]), (v, s["v_pool"], s["v_scale"])):
        pages, back = pool.to(F64).cpu().numpy(), []
        scale, x = scale.to(F64).cpu().numpy(), x.cpu().numpy()
        for i, n in enumerate(lens):
            p0 = n - (starts[i + 1] - starts[i])
            for j in range(p0 // ps, (n - 1) // ps + 1):
                a, b = max(p0, j * ps), min(n, (j + 1) * ps)
                new = x[starts[i] + a - p0:starts[i] + b - p0]
                pg, lo, hi = table[i][j], a - j * ps, b - j * ps
                e = np.ceil(np.log2(np.maximum(np.abs(new).max((0, 2)) / 127, 2.0 ** -64)))
                e = np.maximum(e, np.log2(scale[pg])) if lo else e
                page = pages[pg]
                page[:lo] = np.rint(page[:lo] * (scale[pg] / 2.0 ** e)[:, None])
                page[lo:hi] = np.rint(new / (2.0 ** e)[:, None])
                back.append(page * (2.0 ** e)[:, None])
        out.append(torch.from_numpy(np.stack(back)))
    return out


def _exact_attend(s):
    c, out = s["case"], torch.empty_like(s["q"], dtype=F64)
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    g = c["heads"] // c["kv"]
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        first = max(0, n - (b - a) + 1 - c["window"]) if c["window"] else 0
        pages = s["table"][i][first // c["page"]:-(-n // c["page"])].long()
        t = torch.arange(n, device=DEV)[first // c["page"] * c["page"]:]
        p = torch.arange(n - (b - a), n, device=DEV)
        see = t[None, :] <= p[:, None]
        if c["window"]:
            see &= t[None, :] > p[:, None] - c["window"]
        for h in range(c["kv"]):
            k, v = ((pool[pages, :, h].to(F64) * scale[pages, h].to(F64)[:, None, None]).view(-1, c["dim"])[:len(t)]
                    for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])))
            for j in range(h * g, (h + 1) * g):
                x = s["q"][a:b, j].to(F64) @ k.T
                out[a:b, j] = torch.softmax(torch.where(see, x, torch.full_like(x, -math.inf)), 1) @ v
    return out


def _exact_logprobs(s):
    out = []
    for x, t in zip(s["logits"], s["tokens"].tolist()):
        lp = x.to(F64) - torch.logsumexp(x.to(F64), 0)
        val, idx = torch.sort(x, descending=True, stable=True)
        out.append((lp[t], -(lp.exp() * lp).sum(), idx[:s["case"]["top"]].int(), lp[idx[:s["case"]["top"]]]))
    return [torch.stack(o) for o in zip(*out)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](s)
