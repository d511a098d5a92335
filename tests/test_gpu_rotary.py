"""Rotary positions (ops.rotary) and their gradients against complex multiplication in fp64.

Bounds: the angle is formed in fp64 and its sine and cosine are fp32 (a few units of 2^-24 of 1), the turned pair is two products and
a sum in fp32, rounded once: |error| <= u |y| + 8 * 2^-24 * scale * (|a| + |b|), and below a type's smallest normal number, where its
values are multiples of smallest_normal * eps, half of that (fp16: 2^-14 * 2^-10 / 2 = 2^-25) in the place of u |y|.
"""

from __future__ import annotations

import pytest
import torch

from cernels_amd import ops

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def exact_turn(x, positions, inv_freq, interleaved, scale=1.0, back=False):
    """(turned x, magnitude |a| + |b| of each element's pair) in fp64."""
    x, n = x.double().cpu(), 2 * inv_freq.numel()
    angle = positions.double().cpu()[:, None] * inv_freq.double().cpu() * (-1 if back else 1)
    z = torch.polar(torch.full_like(angle, scale), angle)[:, None]
    y, size = x.clone(), x.abs()
    if n:
        a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
        t = torch.complex(a, b) * z
        parts = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
        for part, v in zip(parts, (t.real, t.imag)):
            y[..., part] = v
            size[..., part] = scale * (a.abs() + b.abs())
    return y, size


def assert_turned(got, x, positions, inv_freq, interleaved, scale=1.0, back=False, what=""):
    want, size = exact_turn(x, positions, inv_freq, interleaved, scale, back)
    t = torch.finfo(got.dtype)
    tol = t.eps / 2 * want.abs().clamp_min(t.smallest_normal) + 8 * U32 * size
    worst = ((got.double().cpu() - want).abs() / tol).max().item() if want.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary", [(1, 32, 4, 128, 128), (8, 64, 8, 64, 64), (5, 16, 2, 256, 64), (33, 10, 10, 128, 128),
                                                     (3, 3, 1, 96, 32), (7, 2, 1, 20, 6), (4, 1, 1, 6, 2), (2, 5, 5, 128, 0),
                                                     (300, 4, 2, 80, 80), (2, 1, 1, 37, 14)])
def test_turns_and_gradients(device, tokens, hq, hk, dim, rotary, dtype, interleaved):
    g = torch.Generator().manual_seed(tokens + dim)
    q, k = (torch.randn(tokens, h, dim, generator=g).to(dtype).to(device).requires_grad_() for h in (hq, hk))
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g).to(device)
    inv, _ = ops.rotary_frequencies(rotary, device=device)
    scale = 1.25
    print(f"[rotary {tokens} {hq}/{hk}x{dim} part {rotary} {dtype} interleaved={interleaved}]", flush=True)
    q2, k2 = ops.rotary(q, k, pos, inv, interleaved=interleaved, scale=scale)
    assert q2.shape == q.shape and q2.is_contiguous()
    assert_turned(q2, q.detach(), pos, inv, interleaved, scale, what="q")
    assert_turned(k2, k.detach(), pos, inv, interleaved, scale, what="k")
    dq, dk = torch.randn_like(q2), torch.randn_like(k2)
    gq, gk = torch.autograd.grad((q2, k2), (q, k), (dq, dk))
    assert_turned(gq, dq, pos, inv, interleaved, scale, back=True, what="dq")
    assert_turned(gk, dk, pos, inv, interleaved, scale, back=True, what="dk")


@pytest.mark.parametrize("ptype", [torch.int32, torch.int64])
@pytest.mark.parametrize("ftype", [torch.float32, torch.float64])
def test_position_and_frequency_types(device, ptype, ftype):
    x = torch.randn(6, 2, 64, device=device)
    pos = torch.tensor([0, 1, -7, 65535, 1 << 24, (1 << 31) - 1], dtype=ptype, device=device)
    inv = ops.rotary_frequencies(64, base=500000.0, device=device)[0].to(ftype)
    y, none = ops.rotary(x, None, pos, inv)
    assert none is None
    # at 2^31 the product of position and frequency is rounded at 2^-22 of a turn in fp64
    want, size = exact_turn(x, pos, inv, False)
    far = 2 * 3.1416 * (pos.double().abs().cpu() * 2.0 ** -53)[:, None, None]
    assert ((y.double().cpu() - want).abs() <= (U32 * 10 + far) * size).all()


def test_strided_views_and_other_gradients(device):
    """q and k as slices of one fused projection; a gradient for k alone, and one that is a transposed view."""
    fused = torch.randn(9, 12, 64, device=device, dtype=torch.bfloat16)
    pos, inv = torch.arange(100, 109, device=device), ops.rotary_frequencies(64, device=device)[0]
    q, k = fused[:, 1:9], fused[:, 10:]
    q2, k2 = ops.rotary(q, k, pos, inv)
    assert_turned(q2, q, pos, inv, False)
    assert_turned(k2, k, pos, inv, False)
    heads_first = torch.randn(3, 9, 64, device=device).transpose(0, 1)  # [tokens, heads, dim] over [heads, tokens, dim]
    assert_turned(ops.rotary(heads_first, None, pos, inv)[0], heads_first, pos, inv, False)
    odd = torch.randn(9 * 3 * 64 + 1, device=device, dtype=torch.bfloat16)[1:].view(9, 3, 64)  # 2-byte alignment only
    assert_turned(ops.rotary(odd, None, pos, inv, interleaved=True)[0], odd, pos, inv, True)
    qg, kg = q.detach().clone(), k.detach().clone().requires_grad_()
    a, b = ops.rotary(qg, kg, pos, inv)
    dk = torch.randn(64, 9, 2, device=device, dtype=torch.bfloat16).permute(1, 2, 0)
    (gk,) = torch.autograd.grad(b, kg, dk)
    assert_turned(gk, dk, pos, inv, False, back=True)
    shared = kg.expand(9, 2, 64)
    a, b = ops.rotary(shared, shared, pos, inv)  # one leaf twice: its gradients add
    (gs,) = torch.autograd.grad((a, b), kg, (dk, dk))
    want, size = exact_turn(dk, pos, inv, False, back=True)
    assert ((gs.double().cpu() - 2 * want).abs() <= 2.0 ** -7 * 2 * want.abs() + 16 * U32 * size).all()


def test_gradient_against_differences(device):
    x = torch.randn(5, 2, 32, device=device, requires_grad=True)
    pos, inv = torch.arange(5, device=device) * 1000, ops.rotary_frequencies(32, device=device)[0]
    w = torch.randn(5, 2, 32, device=device)
    (g,) = torch.autograd.grad(ops.rotary(x, None, pos, inv, interleaved=True, scale=0.8)[0], x, w)
    v = torch.randn_like(x)
    f = lambda t: float((ops.rotary(t, None, pos, inv, interleaved=True, scale=0.8)[0].double() * w.double()).sum())  # noqa: E731
    slope = (f(x.detach() + v) - f(x.detach() - v)) / 2  # the map is linear: any step gives the derivative
    # 320 outputs, each off by 8 U32 of its pair's size (<= 20 here) and weighted by |w| <= 5
    assert abs(slope - float((g.double() * v.double()).sum())) <= 320 * 8 * U32 * 20 * 5


def test_no_tokens(device):
    inv = ops.rotary_frequencies(64, device=device)[0]
    q, k = ops.rotary(torch.empty(0, 4, 64, device=device), torch.empty(0, 1, 64, device=device),
                      torch.empty(0, dtype=torch.int64, device=device), inv)
    assert q.shape == (0, 4, 64) and k.shape == (0, 1, 64)


def test_captured_call_replays(device):
    q = torch.randn(17, 4, 128, device=device, dtype=torch.bfloat16)
    pos, inv = torch.arange(17, device=device), ops.rotary_frequencies(128, device=device)[0]
    ops.rotary(q, None, pos, inv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = ops.rotary(q, None, pos, inv)[0]
    for i in range(3):
        q.normal_()
        pos.add_(1000)
        want = ops.rotary(q, None, pos, inv)[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want), i


def test_more_than_2_31_elements(device):
    tokens = 263_000
    q = torch.empty(tokens, 64, 128, dtype=torch.bfloat16, device=device)
    assert q.numel() > 2 ** 31
    q[-5:].normal_()
    pos, inv = torch.arange(tokens, device=device), ops.rotary_frequencies(128, device=device)[0]
    y, _ = ops.rotary(q, None, pos, inv, interleaved=True)
    assert_turned(y[-5:], q[-5:], pos[-5:], inv, True)


def test_gradients_have_no_gradients(device):
    q = torch.randn(5, 3, 64, device=device, requires_grad=True)
    pos, inv = torch.arange(5, device=device), ops.rotary_frequencies(64, device=device)[0]
    dy = torch.randn_like(q)
    plain, = torch.autograd.grad(ops.rotary(q, None, pos, inv)[0], q, dy)
    graphed, = torch.autograd.grad(ops.rotary(q, None, pos, inv)[0], q, dy.clone().requires_grad_(), create_graph=True)
    assert torch.equal(plain, graphed)
    with pytest.raises(RuntimeError, match="differentia"):
        graphed.sum().backward()
