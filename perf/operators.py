"""The operators of a decoder layer around its experts, one call at a time: layer norm, rotary positions, the write of new keys and
values into a paged cache, and attention of new tokens over that cache.

* ``layer_norm``: the norm before a layer's projections. Generating programs call it on a few rows, training ones on many and
  with the gradients of its input, weight and bias.
* ``rotary``: positions turned into the queries and keys of a batch of tokens, both pair layouts, whole heads or their first part,
  with the gradients when training.
* ``append``: a step's new keys and values, turned to their positions on the way into the pages, and the turned queries.
* ``attention``: a step's queries over all pages of their sequences: single tokens, chunks behind a long cache, whole prompts.

Head layouts are those of the models that the framework's configurations name (32 query and 4 key heads of 128 with a window of
4096; 64 and 8 of 64 with sinks and a window of 128; 16 and 2 of 256 with a quarter of the head turned; 10 and 10 of 128), widths
their hidden sizes, prompts the benchmark's lengths.
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# query heads, key heads, head size, turned part of the head, interleaved pairs
HEADS = {
    "north": (32, 4, 128, 128, True),
    "gpt_oss": (64, 8, 64, 64, False),
    "qwen3_next": (16, 2, 256, 64, False),
    "deepseek": (10, 10, 128, 128, False),
}


# ---- cases ------------------------------------------------------------------------------------------------------------


def _norm(name, rows, cols, dtype, train, bias):
    return {"name": name, "op": "layer_norm", "rows": rows, "cols": cols, "dtype": dtype, "train": train, "bias": bias}


def _rotary(name, heads, tokens, start, dtype, train, scale=1.0):
    return {"name": name, "op": "rotary", "heads": heads, "tokens": tokens, "start": start, "dtype": dtype, "train": train,
            "scale": scale}


def _append(name, heads, seqs, new, context, page, dtype, fused, mix):
    return {"name": name, "op": "append", "heads": heads, "seqs": seqs, "new": new, "context": context, "page": page,
            "dtype": dtype, "fused": fused, "mix": mix}


def _attention(name, heads, seqs, new, context, page, dtype, window, sinks, mix):
    return {"name": name, "op": "attention", "heads": heads, "seqs": seqs, "new": new, "context": context, "page": page,
            "dtype": dtype, "window": window, "sinks": sinks, "mix": mix}


def listed():
    return [
        # the norm of one generated token of one user
        _norm("norm_1", 1, 2048, "bf16", False, False),
        # training: a batch of eight sequences of 2048 tokens, gradients of input and weight
        _norm("norm_train_16384", 16384, 2880, "bf16", True, False),
        # training in full precision with a bias, odd sizes throughout
        _norm("norm_train_odd", 5003, 1111, "fp32", True, True),
        # the queries and keys of eight generating users' tokens, deep in their contexts
        _rotary("rotary_8", "north", 8, 100003, "bf16", False),
        # training: two sequences' worth of tokens, half layout, positions scaled for a long context
        _rotary("rotary_train_8192", "gpt_oss", 8192, 0, "bf16", True, 1.3465735902799727),
        # 64 generating users: one new token each, slices of one fused projection
        _append("append_64", "north", 64, 1, 4096, 16, "bf16", True, 1),
        # prompts of three users written in one step
        _append("append_prompts", "north", 3, 2167, 0, 64, "bf16", False, 2),
        # one user generating behind the benchmark's prompt
        _attention("attend_1", "north", 1, 1, 2167, 16, "bf16", 4096, False, 3),
        # a serving batch of generating users, contexts of very different lengths
        _attention("attend_64", "north", 64, 1, 8192, 16, "bf16", 0, False, 4),
        # generating with sinks, an odd number of users and contexts that end inside pages
        _attention("attend_sinks_17", "gpt_oss", 17, 1, 3001, 32, "fp16", 0, True, 5),
        # three prompts of different lengths, no context yet
        _attention("attend_prompts", "north", 3, 2167, 0, 64, "bf16", 4096, False, 6),
        # one chunk of a long prompt: 509 new tokens behind 32 thousand
        _attention("attend_chunk_509", "north", 1, 509, 32003, 16, "bf16", 0, False, 7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "rotary", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads = rng.choice(list(HEADS))
    if op == "layer_norm":
        cols = rng.choice([2048, 1280, 2880, _log(rng, 64, 8192)])
        c = _norm("", _log(rng, 1, 16384 * 2880 // max(cols, 2880)), cols, dtype, rng.random() < 0.5, rng.random() < 0.5)
    elif op == "rotary":
        c = _rotary("", heads, _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 1 << 20)]), dtype, rng.random() < 0.5,
                    rng.choice([1.0, round(rng.uniform(1.0, 1.5), 4)]))
        if dtype == "fp32":
            c["tokens"] = 1 + c["tokens"] // 2
    else:
        dtype = rng.choice(["bf16", "fp16"])
        while True:
            new = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 17, 2167)])
            seqs = _log(rng, 1, 64 if new == 1 else 16 if new <= 16 else 4)
            context = rng.choice([0, _log(rng, 16, 32768), _log(rng, 16, 4096)]) if new > 1 else _log(rng, 16, 16384)
            page, mix = rng.choice([16, 32, 64, 128]), rng.randint(10, 10**6)
            if op == "append":
                c = _append("", heads, seqs, new, min(context, 4096), page, dtype, rng.random() < 0.5, mix)
            else:
                c = _attention("", heads, seqs, new, context, page, dtype, rng.choice([0, 0, 128, 4096]), rng.random() < 0.3, mix)
            # the work, and what the plain form holds at once, at most the largest listed case's
            hq, hk, d = HEADS[heads][:3]
            long = context + new
            if seqs * long * hk * d <= 64 * 8193 * 4 * 128 and seqs * new * hq * long <= 509 * 32 * 32512:
                break
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, whole length) of each sequence: the first has the case's own sizes, the others spread below them."""
    r = random.Random(case["mix"])
    new, length = [], []
    for b in range(case["seqs"]):
        n = case["new"] if b == 0 or case["new"] == 1 else max(1, int(case["new"] * r.uniform(0.1, 1.0)))
        ctx = case["context"] if b == 0 else int(case["context"] * math.exp(r.uniform(math.log(0.02), 0.0)))
        new.append(n)
        length.append(ctx + n)
    return new, length


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _inverse_frequencies(rotary):
    return 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(t)

    s = dict(case)
    if case["op"] == "layer_norm":
        s["x"] = (randn(case["rows"], case["cols"]) * 1.5 + 0.25).requires_grad_(case["train"])
        s["weight"] = (1 + 0.1 * randn(case["cols"])).requires_grad_(case["train"])
        s["bias"] = (0.1 * randn(case["cols"])).requires_grad_(case["train"]) if case["bias"] else None
        s["dy"] = randn(case["rows"], case["cols"]) if case["train"] else None
        return s
    hq, hk, d, rotary, s["interleaved"] = HEADS[case["heads"]]
    s["inv_freq"] = _inverse_frequencies(rotary).float().to(DEV)
    if case["op"] == "rotary":
        n = case["tokens"]
        s["q"], s["k"] = randn(n, hq, d).requires_grad_(case["train"]), randn(n, hk, d).requires_grad_(case["train"])
        s["positions"] = torch.arange(case["start"], case["start"] + n, device=DEV)
        s["dq"], s["dk"] = (randn(n, hq, d), randn(n, hk, d)) if case["train"] else (None, None)
        return s
    new, length = _lengths(case)
    page, total = case["page"], sum(new)
    blocks = max(-(-n // page) for n in length)
    pages = sum(-(-n // page) for n in length) + 7
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(new), blocks, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(length):
        need = -(-n // page)
        table[b, :need] = order[at:at + need]
        at += need
    s["table"] = table
    s["lengths"] = torch.tensor(length, dtype=torch.int32, device=DEV)
    s["offsets"] = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    s["max_new"], s["max_length"] = max(new), max(length)
    s["k_pages"], s["v_pages"] = randn(pages, page, hk, d), randn(pages, page, hk, d)
    if case["op"] == "append":
        if case["fused"]:
            s["q"], s["k"], s["v"] = randn(total, hq + 2 * hk, d).split([hq, hk, hk], dim=1)
        else:
            s["q"], s["k"], s["v"] = randn(total, hq, d), randn(total, hk, d), randn(total, hk, d)
        return s
    s["q"] = 1.5 * randn(total, hq, d)
    s["sink"] = torch.randn(hq, generator=g, device=DEV) if case["sinks"] else None
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------


def _turn(x, cos, sin, interleaved):
    """x [tokens, heads, d] in 32 bits with its first part turned by the angles of cos, sin [tokens, part / 2]."""
    n = 2 * cos.shape[1]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    c, s = cos[:, None], sin[:, None]
    y = x.clone()
    if interleaved:
        y[..., 0:n:2], y[..., 1:n:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :n // 2], y[..., n // 2:n] = a * c - b * s, b * c + a * s
    return y


def _angles(positions, inv_freq, scale):
    turn = positions.double()[:, None] * inv_freq.double()
    return (turn.cos() * scale).float(), (turn.sin() * scale).float()


def _norm_plain(s):
    t = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    xc = x - x.mean(1, keepdim=True)
    r = (xc.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    h = xc * r
    y = h * w if s["bias"] is None else h * w + s["bias"].float()
    if not s["train"]:
        return y.to(t)
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    out = [y.to(t), dx.to(t), (dy * h).sum(0).to(t)]
    return out if s["bias"] is None else out + [dy.sum(0).to(t)]


def _rotary_plain(s):
    t = s["q"].dtype
    cos, sin = _angles(s["positions"], s["inv_freq"], s["scale"])
    out = [_turn(x.float(), cos, sin, s["interleaved"]).to(t) for x in (s["q"], s["k"])]
    if s["train"]:
        out += [_turn(x.float(), cos, -sin, s["interleaved"]).to(t) for x in (s["dq"], s["dk"])]
    return out


def _places(s):
    """Sequence and position of every new token."""
    n = (s["offsets"][1:] - s["offsets"][:-1]).long()
    token = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(s["offsets"][1:].long(), token, right=True)
    return seq, token - s["offsets"][seq] + s["lengths"][seq] - n[seq]


def _append_plain(s):
    t = s["q"].dtype
    seq, at = _places(s)
    cos, sin = _angles(at, s["inv_freq"], 1.0)
    page = s["table"][seq, at // s["page"]].long()
    s["k_pages"][page, at % s["page"]] = _turn(s["k"].float(), cos, sin, s["interleaved"]).to(t)
    s["v_pages"][page, at % s["page"]] = s["v"]
    return [_turn(s["q"].float(), cos, sin, s["interleaved"]).to(t), s["k_pages"], s["v_pages"]]


def _attention_plain(s):
    q = s["q"]
    total, hq, d = q.shape
    hk, bsz = s["k_pages"].shape[2], s["table"].shape[0]
    new, long = s["max_new"], s["table"].shape[1] * s["page"]
    seq, at = _places(s)
    row = torch.arange(total, device=DEV) - s["offsets"][seq]
    # every sequence's queries padded to the longest chunk, its keys to the whole table: [B, key head, group x new, .]
    qp = torch.zeros(bsz, new, hq, d, device=DEV)
    qp[seq, row] = q.float() * d ** -0.5
    qp = qp.view(bsz, new, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(bsz, hk, -1, d)
    k = s["k_pages"][s["table"].long()].view(bsz, long, hk, d).permute(0, 2, 3, 1).float()
    score = torch.matmul(qp, k).view(bsz, hk, hq // hk, new, long)
    del k
    pos = torch.full((bsz, new), -1, device=DEV)
    pos[seq, row] = at
    key = torch.arange(long, device=DEV)
    seen = key <= pos[..., None]
    if s["window"]:
        seen &= key > pos[..., None] - s["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True).clamp_min(-1e30)
    if s["sink"] is not None:
        sink = s["sink"].view(hk, hq // hk, 1, 1)
        most = torch.maximum(most, sink)
    score.sub_(most).exp_()
    total_p = score.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total_p = total_p + (sink - most).exp()
    v = s["v_pages"][s["table"].long()].view(bsz, long, hk, d).permute(0, 2, 1, 3).float()
    o = torch.matmul(score.view(bsz, hk, -1, long), v).view(bsz, hk, hq // hk, new, d) / total_p
    return o.permute(0, 3, 1, 2, 4).reshape(bsz, new, hq, d)[seq, row].to(q.dtype)


_PLAIN = {"layer_norm": _norm_plain, "rotary": _rotary_plain, "append": _append_plain, "attention": _attention_plain}


def _own_run(s):
    from cernels_amd import ops

    if s["op"] == "layer_norm":
        y = ops.layer_norm(s["x"], s["weight"], s["bias"], 1e-5)
        if not s["train"]:
            return y
        leaves = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
    if s["op"] == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["interleaved"], scale=s["scale"])
        if not s["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    if s["op"] == "append":
        q = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["offsets"], q=s["q"],
                             inv_freq=s["inv_freq"], interleaved=s["interleaved"])
        return [q, s["k_pages"], s["v_pages"]]
    return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["offsets"], window=s["window"],
                               sinks=s["sink"], max_new=s["max_new"])


def run(state):
    if own:
        return _own_run(state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "layer_norm":
        n = case["rows"] * case["cols"]
        return {"bytes": size * n * (4 if case["train"] else 2), "flops": n * (20 if case["train"] else 8)}
    hq, hk, d, rotary, _ = HEADS[case["heads"]]
    if case["op"] == "rotary":
        n, passes = case["tokens"], 2 if case["train"] else 1
        return {"bytes": size * n * (hq + hk) * d * 2 * passes + 8 * n, "flops": 3 * n * (hq + hk) * rotary * passes}
    new, length = _lengths(case)
    if case["op"] == "append":
        n = sum(new)
        return {"bytes": size * n * (hq + 2 * hk) * d * 2, "flops": 3 * n * (hq + hk) * rotary}
    keys = pairs = 0
    for n, total in zip(new, length):
        w = case["window"] or total
        keys += min(total, n - 1 + w)
        # query i sees the keys up to its own, at most w of them
        short = min(n, max(0, w - (total - n)))
        pairs += sum(range(total - n + 1, total - n + short + 1)) + (n - short) * w
    return {"bytes": size * (2 * keys * hk * d + 2 * sum(new) * hq * d), "flops": 4 * d * hq * pairs}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------


def _exact_norm(s):
    x, w = s["x"].detach().double().requires_grad_(), s["weight"].detach().double().requires_grad_()
    b = None if s["bias"] is None else s["bias"].detach().double().requires_grad_()
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    y = (x - mean) / torch.sqrt(var + 1e-5) * w + (0 if b is None else b)
    if not s["train"]:
        return y.detach()
    return [y.detach(), *torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], s["dy"].double())]


def _exact_turn(x, positions, inv_freq, scale, interleaved, back=False):
    x, n = x.detach().double().clone(), 2 * inv_freq.numel()
    part = x[..., :n].unflatten(-1, (n // 2, 2)) if interleaved else x[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2)
    angle = positions.double()[:, None] * inv_freq.double() * (-1 if back else 1)
    z = torch.view_as_complex(part.contiguous()) * torch.polar(torch.full_like(angle, scale), angle)[:, None]
    pairs = torch.view_as_real(z)
    x[..., :n] = (pairs if interleaved else pairs.transpose(-1, -2)).flatten(-2)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        return _exact_norm(s)
    if case["op"] == "rotary":
        args = (s["positions"], s["inv_freq"], s["scale"], s["interleaved"])
        out = [_exact_turn(s["q"], *args), _exact_turn(s["k"], *args)]
        return out + [_exact_turn(s["dq"], *args, back=True), _exact_turn(s["dk"], *args, back=True)] if s["train"] else out
    new, length = _lengths(case)
    hq, hk, d, _, _ = HEADS[case["heads"]]
    if case["op"] == "append":
        kp, vp, at, q = s["k_pages"].double(), s["v_pages"].double(), 0, []
        for b, (n, total) in enumerate(zip(new, length)):
            pos = torch.arange(total - n, total, device=DEV)
            rows = slice(at, at + n)
            page, slot = s["table"][b].long()[pos // case["page"]], pos % case["page"]
            kp[page, slot] = _exact_turn(s["k"][rows], pos, s["inv_freq"], 1.0, s["interleaved"])
            vp[page, slot] = s["v"][rows].double()
            q.append(_exact_turn(s["q"][rows], pos, s["inv_freq"], 1.0, s["interleaved"]))
            at += n
        return [torch.cat(q), kp, vp]
    out, at = [], 0
    for b, (n, total) in enumerate(zip(new, length)):
        pages = s["table"][b, :-(-total // case["page"])].long()
        k = s["k_pages"][pages].double().flatten(0, 1)[:total]
        v = s["v_pages"][pages].double().flatten(0, 1)[:total]
        pos = torch.arange(total - n, total, device=DEV)[:, None]
        key = torch.arange(total, device=DEV)
        hidden = key > pos
        if case["window"]:
            hidden = hidden | (key <= pos - case["window"])
        heads = []
        for h in range(hq):
            logit = s["q"][at:at + n, h].double() @ k[:, h // (hq // hk)].T.contiguous() / math.sqrt(d)
            logit = logit.masked_fill(hidden, -math.inf)
            if s["sink"] is not None:
                logit = torch.cat([logit, s["sink"][h].double().expand(n, 1)], 1)
            heads.append(torch.softmax(logit, -1)[:, :total] @ v[:, h // (hq // hk)])
        out.append(torch.stack(heads, 1))
        at += n
    return torch.cat(out)
