"""Layer norm and its gradients (ops.layer_norm) against fp64.

Bounds: every fp32 sum of n terms is off by at most its longest chain of additions times 2^-24 of the sum of magnitudes; the result
is rounded once (torch.finfo(t).eps / 2 of the value).
"""

from __future__ import annotations

import pytest
import torch

from cernels_amd import ops

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def _case(rows, cols, dtype, wdtype, bias, seed=0, mean=0.25):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * 1.5 + mean).to(dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(wdtype)
    b = (0.3 * torch.randn(cols, generator=g)).to(wdtype) if bias else None
    dy = torch.randn(rows, cols, generator=g).to(dtype)
    return x, w, b, dy


def _exact(x, w, b, dy, eps):
    x, w, dy = x.double(), w.double(), dy.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    y = h * w + (0 if b is None else b.double())
    g = dy * w
    gm, ghm = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - gm - h * ghm)
    # magnitudes that the bounds take: the error of h, in units of U32 times the longest chain
    he = x.abs().mean(-1, keepdim=True) * rstd + h.abs()
    dxe = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + h.abs() * (g * h).abs().mean(-1, keepdim=True)
                  + he * ghm.abs() + h.abs() * (g.abs() * he).mean(-1, keepdim=True))
    return dict(y=y, dx=dx, dw=(dy * h).sum(0), db=dy.sum(0), he=he, dxe=dxe, dwe=(dy.abs() * he).sum(0),
                dwa=(dy * h).abs().sum(0), dba=dy.abs().sum(0), h=h)


def _check(name, got, want, tol):
    off = (got.double().cpu() - want).abs()
    worst = (off / tol.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"{name}: {worst:.3f} of the bound"


def _run(device, rows, cols, dtype, wdtype, bias, train, eps=1e-5, seed=0):
    x, w, b, dy = _case(rows, cols, dtype, wdtype, bias, seed)
    e = _exact(x, w, b, dy, eps)
    xd, wd = x.to(device).requires_grad_(train), w.to(device).requires_grad_(train)
    bd = None if b is None else b.to(device).requires_grad_(train)
    print(f"[norm {rows}x{cols} {dtype} {wdtype} bias={bias}]", flush=True)
    y = ops.layer_norm(xd, wd, bd, eps)
    u, uw = torch.finfo(dtype).eps / 2, torch.finfo(wdtype).eps / 2
    chain = cols / 64 + 24  # a lane's vectors, the wave's tree, the waves of a row, the arithmetic around
    _check("y", y, e["y"], u * e["y"].abs() + chain * U32 * (w.double().abs() * e["he"] + e["y"].abs()) + 1e-30)
    if not train:
        assert not y.requires_grad
        return
    grads = torch.autograd.grad(y, [t for t in (xd, wd, bd) if t is not None], dy.to(device))
    _check("dx", grads[0], e["dx"], u * e["dx"].abs() + 2 * chain * U32 * e["dxe"] + 1e-30)
    down = rows / 64 + 64  # rows that a lane adds, the rows of a workgroup, the partial rows
    _check("dw", grads[1], e["dw"], uw * e["dw"].abs() + U32 * (down * e["dwa"] + chain * e["dwe"]) + 1e-30)
    if b is not None:
        _check("db", grads[2], e["db"], uw * e["db"].abs() + U32 * down * e["dba"] + 1e-30)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2048), (2, 7), (3, 64), (5, 511), (9, 513), (33, 1280), (257, 1111), (1030, 2880),
                                       (4100, 192), (17, 8191), (3, 12288), (2, 24577)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_and_gradients(device, rows, cols, dtype):
    _run(device, rows, cols, dtype, dtype, bias=cols % 2 == 1, train=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [1000, 2048, 30001])
def test_norm_with_fp32_weights(device, dtype, cols):
    _run(device, 37, cols, dtype, torch.float32, bias=True, train=True)
    _run(device, 37, cols, dtype, torch.float32, bias=False, train=False)


def test_large_mean_keeps_its_variance(device):
    """A row of mean 4096 and deviation 1 in fp32: a variance taken as E[x^2] - E[x]^2 would lose it."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 1500, generator=g) + 4096
    w = torch.ones(1500)
    y = ops.layer_norm(x.to(device), w.to(device), None, 1e-5)
    e = _exact(x, w, None, x, 1e-5)
    # the mean is off by at most chain * U32 * 4096, which shifts h by that
    assert (y.cpu().double() - e["y"]).abs().max() <= (1500 / 64 + 24) * U32 * 4100 * 1.1


def test_rows_of_one_value_and_no_rows(device):
    x = torch.full((4, 300), 2.5, device=device, dtype=torch.bfloat16)
    w, b = torch.ones(300, device=device), torch.full((300,), 0.5, device=device)
    assert torch.equal(ops.layer_norm(x, w, b), torch.full_like(x, 0.5))  # variance 0: the bias
    leaves = [torch.empty(0, 300, device=device, dtype=torch.bfloat16, requires_grad=True), w.clone().requires_grad_(),
              b.clone().requires_grad_()]
    y = ops.layer_norm(*leaves)
    assert y.shape == (0, 300)
    dx, dw, db = torch.autograd.grad(y.sum(), leaves)
    assert dx.shape == (0, 300) and not dw.any() and not db.any()


def test_infinities_stay_in_their_row(device):
    x = torch.randn(3, 700, device=device)
    x[1, 5], x[2, 699] = float("inf"), float("nan")
    y = ops.layer_norm(x, torch.ones(700, device=device))
    assert torch.isfinite(y[0]).all() and torch.isnan(y[2]).all() and torch.isnan(y[1, 5])


def test_gradients_against_differences(device):
    """The gradients as derivatives of the forward pass: central differences of fp32 calls along random directions."""
    x, w, b, dy = _case(6, 320, torch.float32, torch.float32, True, 5)
    leaves = [t.to(device).requires_grad_() for t in (x, w, b)]
    dyd = dy.to(device)
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dyd)
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, device=device)
        step = 2.0 ** -6
        ends = []
        for s in (step, -step):
            args = [t.detach() + s * v if j == i else t.detach() for j, t in enumerate(leaves)]
            ends.append((ops.layer_norm(*args).double() * dyd.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * step)
        want = (grads[i].double() * v.double()).sum()
        # fp32 rounding of 1920 outputs of size 1 over 2 * step, and the third derivative's step^2 / 6 part
        scale = float((grads[i].double() * v.double()).abs().sum()) + 1
        assert abs(float(slope - want)) <= 2e-3 * scale, (i, float(slope), float(want))


def test_some_gradients_only_and_shapes(device):
    x, w, b, dy = _case(24, 96, torch.bfloat16, torch.bfloat16, True, 7)
    x3 = x.to(device).view(2, 3, 4, 96)
    wd, bd = w.to(device), b.to(device)
    ref = _exact(x, w, b, torch.ones_like(dy), 1e-5)
    for which in range(3):
        leaves = [t.detach().requires_grad_(i == which) for i, t in enumerate((x3, wd, bd))]
        y = ops.layer_norm(*leaves)
        assert y.shape == x3.shape
        (g,) = torch.autograd.grad(y.sum(), [leaves[which]])  # an expanded gradient: stride 0
        want = (ref["dx"].view(2, 3, 4, 96), ref["dw"], ref["db"])[which]
        slack = (ref["dxe"].view(2, 3, 4, 96), ref["dwa"], ref["dba"])[which]
        _check(f"leaf {which}", g, want, 2.0 ** -8 * want.abs() + 128 * U32 * slack + 1e-6)


def test_backward_is_the_same_bits_every_run(device):
    x, w, b, dy = (t.to(device) for t in _case(3000, 777, torch.bfloat16, torch.bfloat16, True, 9))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    for _ in range(3):
        again = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_captured_training_step_replays(device):
    x, w, b, dy = (t.to(device) for t in _case(640, 1024, torch.bfloat16, torch.bfloat16, True, 11))
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = ops.layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x) + i)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want)), i


def test_more_than_2_31_elements(device):
    rows, cols = 1_050_000, 2053
    assert rows * cols > 2 ** 31
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=device)
    g = torch.Generator(device=device).manual_seed(5)
    tail = torch.randn(7, cols, generator=g, device=device).bfloat16()
    x[:-7], x[-7:] = 1.0, tail
    w = torch.randn(cols, generator=g, device=device).bfloat16()
    y = ops.layer_norm(x, w)
    assert torch.equal(y[-7:], ops.layer_norm(tail, w)) and not y[:3].any()
    del y
    x.requires_grad_()
    dy = torch.ones(1, cols, dtype=torch.bfloat16, device=device).expand(rows, cols).contiguous()
    (dx,) = torch.autograd.grad(ops.layer_norm(x, w), x, dy)
    leaf = tail.clone().requires_grad_()
    (want,) = torch.autograd.grad(ops.layer_norm(leaf, w), leaf, dy[-7:])
    assert torch.equal(dx[-7:], want)


def test_gradients_have_no_gradients(device):
    x, w, b, dy = (t.to(device) for t in _case(7, 96, torch.float32, torch.float32, True))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    plain = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    graphed = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy.clone().requires_grad_(), create_graph=True)
    for a, c in zip(plain, graphed):
        assert torch.equal(a, c)
        with pytest.raises(RuntimeError, match="differentia"):
            c.sum().backward(retain_graph=True)
