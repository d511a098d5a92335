"""The paged cache's writes (ops.paged_append) and attention over it (ops.paged_attention) against fp64.

Bounds of attention, per output element, with A = sum_j p_j |v_j| (p the exact probabilities):
  rounding of the result u |o|; rounding of each probability to the values' type u A; scores in fp32, off by at most
  d = (dim + 4) 2^-24 scale max_j sum |q k_j|, which changes each exponential by a factor within 1 +- d, in numerator and sum; the
  hardware exponential and the fp32 sums, (keys + 64) 2^-24 A.
"""

from __future__ import annotations

import math

import pytest
import torch

from cernels_amd import ops
from test_gpu_rotary import assert_turned

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def make_step(seqs, hq, hk, dim, page, dtype, device, seed=0, blocks=None, behind=0, layout="slots", fill=None):
    """seqs: (new tokens, whole length) of each sequence. Slots that no token fills hold `fill` (NaN by default)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-total // page) for _, total in seqs]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(seqs), blocks or max(max(need), 1)), -1, dtype=torch.int32)
    bad = math.nan if fill is None else fill
    shape = (pages, page, hk, dim) if layout == "slots" else (pages, hk, page, dim)
    k, v = torch.full(shape, bad, dtype=dtype), torch.full(shape, bad, dtype=dtype)
    if layout != "slots":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    keys, values, at = [], [], 0
    for b, (_, total) in enumerate(seqs):
        ids = order[at:at + need[b]]
        table[b, :need[b]] = ids
        at += need[b]
        keys.append(torch.randn(total, hk, dim, generator=g).to(dtype))
        values.append(torch.randn(total, hk, dim, generator=g).to(dtype))
        p = torch.arange(total)
        k[ids.long()[p // page], p % page] = keys[b]
        v[ids.long()[p // page], p % page] = values[b]
    tokens = sum(n for n, _ in seqs)
    q = (1.5 * torch.randn(tokens + behind, hq, dim, generator=g)).to(dtype)
    offsets = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).to(torch.int32)
    lengths = torch.tensor([t for _, t in seqs], dtype=torch.int32)
    move = lambda t: t.to(device)  # noqa: E731
    return dict(q=move(q), k_pages=move(k), v_pages=move(v), block_table=move(table), lengths=move(lengths), q_offsets=move(offsets),
                keys=keys, values=values, seqs=seqs)


def call(s, **kw):
    return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], kw.pop("q_offsets", s["q_offsets"]), **kw)


def exact_attention(s, window=0, sinks=None, scale=None, hidden=None):
    """(o, tolerance) of every sequence's rows. hidden(b, keys): keys of sequence b that have no page."""
    q, out, tol, at = s["q"].cpu(), [], [], 0
    hq, dim = q.shape[1:]
    scale = dim ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    for b, (n, total) in enumerate(s["seqs"]):
        k, v = s["keys"][b].double(), s["values"][b].double()
        rep = hq // k.shape[1]
        k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
        qb = q[at:at + n].double()
        score = torch.einsum("nhd,lhd->hnl", qb, k) * scale
        pos, key = torch.arange(total - n, total)[:, None], torch.arange(total)[None]
        dark = key > pos
        if window:
            dark = dark | (key <= pos - window)
        if hidden is not None:
            dark = dark | hidden(b, torch.arange(total))[None]
        score = score.masked_fill(dark, -math.inf)
        size = torch.einsum("nhd,lhd->hnl", qb.abs(), k.abs()).masked_fill(dark, 0)
        d = (dim + 4) * U32 * scale * (size.amax(-1, keepdim=True) if total else size.sum(-1, keepdim=True))
        m = score.amax(-1, keepdim=True) if total else torch.full((hq, n, 1), -math.inf, dtype=torch.float64)
        if sinks is not None:
            m = torch.maximum(m, sinks.double().cpu()[:, None, None])
        m = m.masked_fill(m == -math.inf, 0)
        e = (score - m).exp()
        total_e = e.sum(-1, keepdim=True)
        if sinks is not None:
            total_e = total_e + (sinks.double().cpu()[:, None, None] - m).exp()
        p = e / total_e.masked_fill(total_e == 0, 1)
        o = torch.einsum("hnl,lhd->nhd", p, v)
        a = torch.einsum("hnl,lhd->nhd", p, v.abs())
        out.append(o)
        tol.append(u * o.abs() + (u + 3 * d.permute(1, 0, 2) + (total + 64) * U32) * a + 1e-30)
        at += n
    return torch.cat(out), torch.cat(tol)


def check(s, got, **kw):
    want, tol = exact_attention(s, **kw)
    got = got[:want.shape[0]].double().cpu()
    assert torch.isfinite(got).all(), "not finite"
    worst = ((got - want).abs() / tol).max().item() if want.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} of the bound"


HEADS = [(32, 4, 128), (64, 8, 64), (16, 2, 256), (10, 10, 128), (3, 1, 64), (40, 2, 128)]
SEQS = {
    "one token": [(1, 1)],
    "single": [(1, 700), (1, 1), (1, 33), (1, 64), (1, 129)],
    "short chunks": [(4, 100), (1, 17), (3, 3), (2, 300)],
    "prompts": [(70, 70), (200, 200), (1, 1)],
    "chunks": [(130, 900), (65, 66), (33, 2000)],
    "mixed, some empty": [(0, 50), (150, 400), (0, 0), (1, 999), (5, 5), (0, 16)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seqs", list(SEQS))
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_attention(device, heads, seqs, dtype):
    s = make_step(SEQS[seqs], *heads, 16 if heads[0] % 3 else 48, dtype, device, seed=len(seqs))
    print(f"[attend {heads} {seqs} {dtype}]", flush=True)
    check(s, call(s))
    check(s, call(s, max_new=max(n for n, _ in s["seqs"])))


@pytest.mark.parametrize("window", [1, 16, 100, 4096])
@pytest.mark.parametrize("seqs", ["single", "chunks", "mixed, some empty"])
def test_window_and_sinks(device, window, seqs):
    s = make_step(SEQS[seqs], 16, 2, 64, 32, torch.bfloat16, device, seed=window)
    sinks = torch.randn(16, device=device) * 3
    print(f"[window {window} {seqs}]", flush=True)
    check(s, call(s, window=window), window=window)
    check(s, call(s, window=window, sinks=sinks, scale=0.3), window=window, sinks=sinks, scale=0.3)


def test_long_cache_splits_and_joins(device):
    """Long keys for few rows: many splits, some of them empty, in both kernels."""
    for seqs, heads in (([(1, 9001), (1, 40), (1, 3000)], (8, 1, 128)), ([(40, 9000)], (4, 1, 64)), ([(20, 5000), (1, 2)], (16, 2, 256))):
        s = make_step(seqs, *heads, 64, torch.bfloat16, device, seed=7, blocks=160)
        print(f"[long {seqs} {heads}]", flush=True)
        check(s, call(s))
        check(s, call(s, window=2500), window=2500)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new", [1, 60])
def test_one_key_over_a_long_flat_rest(device, new, dtype):
    """One key has e^11 times the weight of each of the 9000 others, which together still weigh 0.15 of it: probabilities of 2^-16, below
    fp16's normal numbers. Bound: as everywhere, and 2^-25 for each such probability (half of fp16's smallest step) against the sum of
    the weights, times max |v|."""
    s = make_step([(new, 9000)], 2, 1, 64, 64, dtype, device, seed=new)
    q = torch.zeros_like(s["q"])
    q[..., 0] = 8.0
    s["q"] = q
    k = torch.zeros(9000, 1, 64, dtype=dtype)
    k[4000, 0, 0] = 11.0
    s["keys"][0] = k
    j = torch.arange(9000, device=device)
    s["k_pages"][s["block_table"][0, j // 64].long(), j % 64] = k.to(device)
    for scale in (0.125, 0.17):
        got = call(s, scale=scale).double().cpu()
        want, tol = exact_attention(s, scale=scale)
        tol = tol + 9000 * 2.0 ** -25 * float(s["values"][0].abs().max())
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


def test_small_values(device):
    """Values below fp16's smallest normal number keep their own precision: steps of 2^-24."""
    for new in (1, 40):
        s = make_step([(new, 200)], 4, 1, 64, 16, torch.float16, device, seed=new)
        small = (s["values"][0].double() * 2.0 ** -17).half()
        s["values"][0] = small
        j = torch.arange(200, device=device)
        s["v_pages"][s["block_table"][0, j // 16].long(), j % 16] = small.to(device)
        got = call(s).double().cpu()
        want, tol = exact_attention(s)
        assert ((got - want).abs() <= tol + 2.0 ** -25).all()


def test_wrong_max_new_changes_nothing(device):
    s = make_step([(90, 300), (1, 50), (300, 310)], 8, 2, 128, 16, torch.bfloat16, device)
    for most in (1, 2, 10, 100, 10_000):
        check(s, call(s, max_new=most))


def test_uniform_steps_without_offsets(device):
    for n in (1, 3, 80):
        s = make_step([(n, 200), (n, n), (n, 97 + n)], 8, 2, 64, 16, torch.float16, device, seed=n)
        check(s, call(s, q_offsets=None))


@pytest.mark.parametrize("n,count", [(1, 70), (1, 300), (5, 64), (20, 9)])
def test_many_uniform_sequences_without_offsets(device, n, count):
    """The workspace is the one of the kernels that a uniform step takes, whether the caller names its length or not."""
    g = torch.Generator().manual_seed(count)
    s = make_step([(n, n + int(torch.randint(0, 700, (1,), generator=g))) for _ in range(count)], 8, 2, 64, 16, torch.bfloat16, device, blocks=300)
    want = call(s, q_offsets=None)
    check(s, want)
    for most in (None, 1, n, 10 * n):
        assert torch.equal(call(s, q_offsets=None, max_new=most), want)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_in_other_orders(device, new):
    """Pages as [pages, heads, slots, dim], queries as a slice of a fused projection, a table that is a slice of a wider one."""
    s = make_step([(new, 300), (new, 77)], 8, 2, 128, 32, torch.bfloat16, device, layout="heads")
    assert not s["k_pages"].is_contiguous()
    fused = torch.randn(2 * new, 12, 128, device=device, dtype=torch.bfloat16)
    fused[:, 2:10] = s["q"]
    s["q"] = fused[:, 2:10]
    wide = torch.full((2, 50), -1, dtype=torch.int32, device=device)
    wide[:, 3:3 + s["block_table"].shape[1]] = s["block_table"]
    s["block_table"] = wide[:, 3:3 + s["block_table"].shape[1]]
    check(s, call(s))


def test_strides_of_single_heads_and_pages_do_not_matter(device):
    s = make_step([(1, 16)], 4, 1, 64, 16, torch.bfloat16, device)
    page = int(s["block_table"][0, 0])
    want = call(s)
    k, v = (s[n][page:page + 1].contiguous().as_strided((1, 16, 1, 64), (3, 64, 5, 1)) for n in ("k_pages", "v_pages"))
    got = ops.paged_attention(s["q"], k, v, torch.zeros_like(s["block_table"]), s["lengths"], s["q_offsets"])
    assert torch.equal(got, want)


def test_refusals(device):
    """What breaks the contract is refused before a launch, on the GPU's own tensors."""
    s = make_step([(2, 40), (1, 5)], 8, 2, 64, 16, torch.bfloat16, device, fill=0.0)
    bad = [dict(q=s["q"].float()), dict(q=s["q"][..., :32]), dict(q=s["q"][:, :7]), dict(q=s["q"].cpu()), dict(lengths=s["lengths"].long()),
           dict(lengths=s["lengths"][:1]), dict(q_offsets=s["q_offsets"][:2]), dict(block_table=s["block_table"].long()),
           dict(block_table=s["block_table"][:1].expand(2, -1)), dict(block_table=s["block_table"].cpu()),
           dict(k_pages=s["k_pages"][:, :8]), dict(k_pages=s["k_pages"].half()), dict(v_pages=s["v_pages"][:1]),
           dict(k_pages=s["k_pages"].transpose(2, 3)), dict(q_offsets=None)]
    for change in bad:
        with pytest.raises(RuntimeError):
            call({**s, **change}, q_offsets=change.get("q_offsets", s["q_offsets"]))
        t = {**s, **change}
        if t["q"] is not s["q"]:
            continue
        with pytest.raises(RuntimeError):
            ops.paged_append(s["q"][:, :2], s["q"][:, :2], t["k_pages"], t["v_pages"], t["block_table"], t["lengths"], t["q_offsets"])
    for kw in (dict(window=-1), dict(window=2 ** 32 + 5), dict(scale=0.0), dict(scale=math.nan), dict(sinks=torch.zeros(4, device=device)),
               dict(sinks=torch.zeros(8, device=device, dtype=torch.bfloat16)), dict(out=s["q"][:, :4]), dict(max_new=-1)):
        with pytest.raises(RuntimeError):
            call(s, **kw)
    off = torch.empty(s["k_pages"].numel() + 4, dtype=torch.bfloat16, device=device)[4:].view_as(s["k_pages"])
    with pytest.raises(RuntimeError, match="aligned"):
        call({**s, "k_pages": off})
    inv = torch.ones(33, device=device)
    for f in (inv, inv[:32].half(), inv[:32].cpu(), inv[:20][::2]):
        with pytest.raises(RuntimeError):
            ops.paged_append(s["q"][:, :2], s["q"][:, :2], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], s["q_offsets"], inv_freq=f)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="backward"):
        call({**s, "q": s["q"].clone().requires_grad_()})
    x = torch.zeros(4, 8, device=device)
    for args in ((x.t(), torch.ones(4, device=device)), (x, torch.ones(7, device=device)), (x, torch.ones(8)), (x.double(), torch.ones(8, device=device)),
                 (x, torch.ones(8, device=device).half()), (x, torch.ones(8, device=device), torch.ones(8, device=device).half())):
        with pytest.raises(RuntimeError):
            ops.layer_norm(*args)
    q, pos, f = torch.zeros(4, 2, 8, device=device), torch.arange(4, device=device), torch.ones(4, device=device)
    for args in ((q, None, pos[:3], f), (q, None, pos.float(), f), (q, q[:3], pos, f), (q, q.half(), pos, f), (q, None, pos, torch.ones(5, device=device)),
                 (q.transpose(1, 2), None, pos, f), (q[0], None, pos, f), (q, None, pos.cpu(), f)):
        with pytest.raises(RuntimeError):
            ops.rotary(*args)


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("fill", [math.nan, math.inf])
def test_stale_slots_and_missing_pages(device, new, fill):
    """Slots past a sequence's end and pages outside the table hold NaN or infinities; entries of the table that name no page hide
    their keys (all of them in the last sequence, whose rows are 0)."""
    s = make_step([(new, 333), (new, 200), (new, new)], 8, 2, 128, 16, torch.bfloat16, device, fill=fill)
    pages = s["k_pages"].shape[0]
    s["block_table"][1, 3] = pages          # one past the pool
    s["block_table"][1, 5] = -5
    s["block_table"][2, :] = 2 ** 31 - 1
    out = call(s)
    hidden = lambda b, j: ((j // 16 == 3) | (j // 16 == 5)) if b == 1 else torch.full_like(j, b == 2, dtype=torch.bool)  # noqa: E731
    check(s, out, hidden=hidden)
    assert not out[2 * new:3 * new].any()


def test_keys_behind_a_window_may_be_anything(device):
    """Single tokens with a window: pages wholly behind it may have been given away, and hold anything."""
    s = make_step([(1, 500), (1, 250)], 8, 2, 64, 16, torch.bfloat16, device)
    for b, (_, total) in enumerate(s["seqs"]):
        for blk in range((total - 100) // 16):
            page = int(s["block_table"][b, blk])
            s["k_pages"][page] = math.nan
            s["v_pages"][page] = math.inf
    check(s, call(s, window=100), window=100)


def test_infinite_scores_and_values(device):
    """A NaN key reaches the rows that see it and no others."""
    s = make_step([(3, 40), (1, 40)], 4, 1, 64, 16, torch.bfloat16, device)
    page, slot = int(s["block_table"][0, 37 // 16]), 37 % 16
    clean = call(s)
    s["k_pages"][page, slot] = math.nan
    out = call(s)
    assert torch.isnan(out[:3]).all() and torch.equal(out[3], clean[3])


@pytest.mark.parametrize("new,heads", [(3, (8, 2, 64)), (2, (4, 1, 256)), (100, (8, 2, 128)), (70, (4, 4, 64)), (40, (4, 1, 256))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [0, 20])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(device, window, dtype, new, heads):
    """Infinities and NaN in the values of some of the step's own keys: rows before such a key, or past its window, are what they are
    without it; rows that see it get the infinity or NaN, in the columns that hold one."""
    total = new + 37
    s = make_step([(new, total)], *heads, 16, dtype, device, seed=new)
    clean, tol = exact_attention(s, window=window)
    put = {total - 1: (5, math.inf), total - 2: (5, -math.inf), total - new: (7, math.nan), total - new // 2: (9, -math.inf), 3: (2, math.inf)}
    for key, (d, x) in put.items():
        s["v_pages"][int(s["block_table"][0, key // 16]), key % 16, :, d] = x
    got = call(s, window=window).double().cpu()
    want = clean.clone()
    for i in range(new):
        pos = total - new + i
        sees = [key <= pos and (not window or key > pos - window) for key in put]
        add = {}
        for (key, (d, x)), see in zip(put.items(), sees):
            if see:
                add[d] = add.get(d, 0.0) + x
        for d, x in add.items():
            want[i, :, d] = x
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[odd].nan_to_num(1.0), want[odd].nan_to_num(1.0))
    assert ((got[~odd] - want[~odd]).abs() <= tol[~odd]).all()


def test_rows_behind_the_last_sequence_stay(device):
    for seqs in ([(1, 30), (1, 500)], [(70, 300), (2, 40)], [(1, 5000), (1, 3)]):
        s = make_step(seqs, 8, 2, 64, 16, torch.bfloat16, device, behind=5)
        out = torch.full(s["q"].shape, 7.0, dtype=torch.bfloat16, device=device)
        assert call(s, out=out) is out
        check(s, out)
        assert (out[-5:] == 7).all()


def test_many_sequences(device):
    """More sequences than a wave has lanes, all kinds of lengths."""
    g = torch.Generator().manual_seed(1)
    n = torch.randint(0, 4, (150,), generator=g).tolist()
    n[70], n[149] = 90, 41
    seqs = [(a, a + int(torch.randint(0, 200, (1,), generator=g))) for a in n]
    s = make_step(seqs, 4, 2, 64, 16, torch.bfloat16, device)
    check(s, call(s))


def test_offsets_past_32_bits(device):
    """A pool of more than 2^31 elements: pages at its far end."""
    pages, page, hk, dim = 70000, 64, 4, 128
    assert pages * page * hk * dim > 2 ** 31
    for new in (1, 40):
        s = make_step([(new, 300)], 8, hk, dim, page, torch.bfloat16, device, seed=new)
        small = s["block_table"].clone()
        k, v = (torch.empty(pages, page, hk, dim, dtype=torch.bfloat16, device=device) for _ in range(2))
        k[pages - 8:], v[pages - 8:] = s["k_pages"][:8], s["v_pages"][:8]
        s.update(k_pages=k, v_pages=v, block_table=(small + pages - 8).to(torch.int32))
        assert int(small.max()) < 8
        check(s, call(s))
        del k, v
        s.clear()


def test_two_streams_at_once(device):
    """Calls on two streams, each with its own scratch, give what calls one after the other give."""
    steps = [make_step([(1, 4000)] * 3, 8, 2, 128, 16, torch.bfloat16, device, seed=i) for i in range(2)]
    want = [call(s) for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(s))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_captured_decoding_step_replays(device):
    """One captured step (append, attention) replayed while lengths grow in place, against eager calls on a copy."""
    s = make_step([(1, 60), (1, 31), (1, 129)], 8, 2, 64, 16, torch.bfloat16, device, blocks=20, fill=0.0)
    s["block_table"][:] = torch.arange(60, dtype=torch.int32, device=device).view(3, 20)
    kp, vp = (torch.randn(60, 16, 2, 64, device=device).bfloat16() for _ in range(2))
    ke, ve = kp.clone(), vp.clone()
    inv = ops.rotary_frequencies(64, device=device)[0]
    q, k, v = (torch.randn(3, h, 64, device=device).bfloat16() for h in (8, 2, 2))

    def step(kp, vp):
        qt = ops.paged_append(k, v, kp, vp, s["block_table"], s["lengths"], q=q, inv_freq=inv, interleaved=True)
        return ops.paged_attention(qt, kp, vp, s["block_table"], s["lengths"], window=100)

    step(kp, vp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(kp, vp)
    for i in range(4):
        for t in (q, k, v):
            t.normal_()
        s["lengths"].add_(1)
        ke.copy_(kp), ve.copy_(vp)
        want = step(ke, ve)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want) and torch.equal(kp, ke) and torch.equal(vp, ve), i


# ---- append -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,dim,rotary,interleaved", [(32, 4, 128, 128, True), (64, 8, 64, 64, False), (16, 2, 256, 64, False),
                                                          (2, 1, 24, 10, True), (2, 1, 24, 10, False), (4, 2, 64, 0, False)])
@pytest.mark.parametrize("seqs", ["single", "mixed, some empty"])
def test_append(device, seqs, hq, hk, dim, rotary, interleaved, dtype):
    s = make_step(SEQS[seqs], hq, hk, dim, 16, dtype, device, fill=0.0, behind=2)
    tokens = s["q"].shape[0]
    fused = torch.randn(tokens, hq + 2 * hk, dim, device=device).to(dtype)
    q, k, v = fused.split([hq, hk, hk], dim=1)
    inv = ops.rotary_frequencies(rotary, device=device)[0] if rotary else None
    kp, vp = torch.full_like(s["k_pages"], 3.0), torch.full_like(s["v_pages"], 3.0)
    print(f"[append {seqs} {hq}/{hk}x{dim} part {rotary} {dtype}]", flush=True)
    qt = ops.paged_append(k, v, kp, vp, s["block_table"], s["lengths"], s["q_offsets"], q=q, inv_freq=inv, interleaved=interleaved,
                          scale=1.5 if rotary else 1.0)
    assert ops.paged_append(k, v, kp, vp, s["block_table"], s["lengths"], s["q_offsets"], inv_freq=inv, interleaved=interleaved,
                            scale=1.5 if rotary else 1.0) is None
    at, seen = 0, torch.zeros(kp.shape[:2], dtype=torch.bool)
    freq = inv if rotary else torch.empty(0)
    for b, (n, total) in enumerate(s["seqs"]):
        rows, pos = slice(at, at + n), torch.arange(total - n, total)
        page, slot = s["block_table"][b].cpu().long()[pos // 16], pos % 16
        assert not seen[page, slot].any()
        seen[page, slot] = True
        scale = 1.5 if rotary else 1.0
        assert_turned(qt[rows], q[rows], pos, freq, interleaved, scale, what="q")
        assert_turned(kp[page.to(device), slot.to(device)], k[rows], pos, freq, interleaved, scale, what="k")
        assert torch.equal(vp[page.to(device), slot.to(device)], v[rows])
        at += n
    rest = ~seen.to(device)
    assert (kp[rest] == 3).all() and (vp[rest] == 3).all()  # nothing else was written


def test_append_drops_what_has_no_page(device):
    """Missing pages, positions past the table and negative ones: nothing is written, the rest is."""
    kp, vp = (torch.zeros(4, 16, 1, 64, device=device, dtype=torch.bfloat16) for _ in range(2))
    table = torch.tensor([[0, 4], [1, 2], [-1, 3]], dtype=torch.int32, device=device)
    lengths = torch.tensor([20, 40, 1], dtype=torch.int32, device=device)   # 16..19 on page 4 (none); 32.. past the table; no page
    offsets = torch.tensor([0, 8, 18, 21], dtype=torch.int32, device=device)  # the last: positions -2, -1, 0
    k = torch.ones(21, 1, 64, device=device, dtype=torch.bfloat16)
    q = torch.ones(21, 2, 64, device=device, dtype=torch.bfloat16)
    out = ops.paged_append(k, k, kp, vp, table, lengths, offsets, q=q)
    wrote = kp[:, :, 0, 0].cpu()
    want = torch.zeros(4, 16)
    want[0, 12:16] = 1   # positions 12..15 of the first
    want[2, 14:16] = 1   # positions 30, 31 of the second
    assert torch.equal(wrote.float(), want) and torch.equal(vp, kp) and torch.equal(out, q)
    s = dict(q=q, k_pages=kp, v_pages=vp, block_table=table, lengths=lengths, q_offsets=offsets)
    rows = call(s)
    assert torch.isfinite(rows).all() and not rows[18:21].any()


def test_step_on_another_stream_and_order(device):
    """A prompt in two chunks and then single tokens give the rows that the whole prompt gives at once."""
    hq, hk, dim, total = 8, 2, 128, 120
    x = torch.randn(total, hq + 2 * hk, dim, device=device).bfloat16()
    q, k, v = x.split([hq, hk, hk], dim=1)
    inv = ops.rotary_frequencies(dim, device=device)[0]
    table = torch.randperm(12, device=device).to(torch.int32)[None, :9]

    def run(cuts):
        kp, vp = (torch.full((12, 16, hk, dim), math.nan, device=device, dtype=torch.bfloat16) for _ in range(2))
        rows, at = [], 0
        for n in cuts:
            cut = slice(at, at + n)
            at += n
            lengths = torch.tensor([at], dtype=torch.int32, device=device)
            qt = ops.paged_append(k[cut], v[cut], kp, vp, table, lengths, q=q[cut], inv_freq=inv)
            rows.append(ops.paged_attention(qt, kp, vp, table, lengths))
        return torch.cat(rows).double(), kp, vp

    whole, kp, vp = run([total])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        parts, kp2, vp2 = run([70, 40] + [1] * 10)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(kp.nan_to_num(), kp2.nan_to_num()) and torch.equal(vp.nan_to_num(), vp2.nan_to_num())
    # both are within u |o| + (u + small) A of the exact row, A <= max |v|
    assert (whole - parts).abs().max() <= 2 * (2.0 ** -8 * whole.abs().max() + 2.0 ** -7 * float(v.abs().max()))
