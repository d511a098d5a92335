"""Refusals of the decoder-layer entries, on the CPU: a call that breaks the contract raises RuntimeError before any pointer reaches
the library, and the C entries return their status before any launch."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from cernels_amd import _native, ops


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.layer_norm(x, w)
    q = torch.zeros(2, 1, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary(q, None, torch.arange(2), torch.ones(4))
    k = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    pages = torch.zeros(3, 16, 1, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_append(k, k, pages, pages, table, lengths)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(k, pages, pages, table, lengths)
    with pytest.raises(RuntimeError, match="tensor"):
        ops.paged_attention(None, pages, pages, table, lengths)
    with pytest.raises(RuntimeError, match="tensors"):
        ops.layer_norm(x, None)


def test_serving_entries_refuse_to_carry_a_gradient():
    k = torch.zeros(2, 1, 64, dtype=torch.bfloat16, requires_grad=True)
    pages = torch.zeros(3, 16, 1, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="backward"):
        ops.paged_append(k, k, pages, pages, table, lengths)
    with pytest.raises(RuntimeError, match="backward"):
        ops.paged_attention(k, pages, pages, table, lengths)


# ---- rotary_frequencies -----------------------------------------------------------------------------------------------------


def test_frequencies():
    inv, scale = ops.rotary_frequencies(8, 10000.0)
    assert scale == 1.0 and inv.dtype == torch.float64
    assert torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    lin, _ = ops.rotary_frequencies(8, scaling={"rope_type": "linear", "factor": 4.0})
    assert torch.equal(lin * 4, inv)
    assert ops.rotary_frequencies(0)[0].numel() == 0
    for bad in (lambda: ops.rotary_frequencies(7), lambda: ops.rotary_frequencies(8, scaling={"rope_type": "none", "factor": 2})):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 8.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 32.0, "beta_fast": 32.0, "beta_slow": 1.0, "original_max_position_embeddings": 4096,
     "truncate": False},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768, "attention_factor": 1.5},
], ids=lambda s: f"{s['rope_type']}{s['factor']:.0f}")
def test_scaled_frequencies_match_the_checkpoints_library(scaling):
    """The same frequencies and scale as transformers forms from a checkpoint's rope settings (in fp32)."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    base = 150000.0
    settings = dict(scaling, rope_theta=base)
    cfg = LlamaConfig(hidden_size=64 * 4, num_attention_heads=4, head_dim=64, rope_parameters=settings,
                      max_position_embeddings=int(scaling.get("original_max_position_embeddings", 4096) * scaling["factor"]))
    want, want_scale = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    inv, scale = ops.rotary_frequencies(64, base, scaling)
    # fp32 powers of the base: the exponent of ln(150000) = 12 is off by 2^-24 of itself
    assert (inv - want.double()).abs().div(want.double()).max() <= 64 * 2.0 ** -24
    assert abs(scale - want_scale) <= 1e-9


# ---- C entries --------------------------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def L():
    return _native.lib()


def _p(n=0x10000):
    return ctypes.c_void_p(n)


def test_norm_entry_statuses(L):
    f = lambda x=_p(), w=_p(), rows=4, cols=64, dt=0, wdt=0, y=_p(): L.cernels_layer_norm(x, w, None, rows, cols, dt, wdt, 1e-5, y, None, None)  # noqa: E731
    assert f(rows=0) == 0
    assert f(rows=-1) == 1 and f(cols=0) == 1 and f(dt=3) == 1 and f(dt=0, wdt=1) == 1 and f(dt=2, wdt=0) == 1 and f(x=None) == 1
    assert f(rows=1 << 31) == 2 and f(cols=(1 << 24) + 1) == 2
    assert f(x=_p(0x10001)) == 3 and f(dt=2, wdt=2, y=_p(0x10002)) == 3
    b = lambda rows=4, dy=_p(), dw=_p(), ws=_p(), n=1 << 30, dx=_p(): L.cernels_layer_norm_backward(  # noqa: E731
        dy, _p(), _p(), _p(), rows, 64, 0, 0, dx, dw, None, ws, ctypes.c_size_t(n), None)
    assert b(dy=None) == 1 and b(ws=None) == 1 and b(n=16) == 4 and b(dx=_p(0x10001)) == 3
    assert b(rows=0, dw=None) == 0 and b(dx=None, dw=None) == 0
    size = L.cernels_layer_norm_backward_workspace_bytes
    assert size(0, 64, 0) == 2 * 64 * 4 and size(100, 0, 0) == 0 and size(10**6, 2880, 0) <= 512 * 2 * 2880 * 4


def test_rotary_entry_statuses(L):
    def f(q=_p(), k=_p(), pos=_p(), ptype=0, inv=_p(), ftype=2, tokens=4, dim=64, pairs=32, dt=0, qo=_p(), ko=_p(), heads=4):
        return L.cernels_rotary(q, heads * dim, dim, heads, k, dim, dim, 1, pos, ptype, inv, ftype, tokens, dim, pairs, 0, 1.0, 0, dt,
                                qo, ko, None)

    assert f(tokens=0) == 0 and f(q=None, k=None) == 0
    assert f(pairs=33) == 1 and f(ptype=2) == 1 and f(ftype=1) == 1 and f(dt=3) == 1 and f(pos=None) == 1 and f(inv=None) == 1
    assert f(qo=None) == 1 and f(ko=None) == 1 and f(tokens=-1) == 1
    assert f(dim=4096, pairs=1025) == 2 and f(heads=1 << 24, dim=64) == 2
    assert f(q=_p(0x10001)) == 3 and f(pos=_p(0x10004), ptype=1) == 3 and f(inv=_p(0x10004), ftype=3) == 3


def _strides(page=16 * 64, slot=64, head=64):
    return (ctypes.c_int64 * 6)(page, slot, head, page, slot, head)


def _step(table=_p(), stride=4, blocks=4, lengths=_p(), offsets=_p(), seqs=2, tokens=4):
    return table, stride, blocks, lengths, offsets, seqs, tokens


def test_append_entry_statuses(L):
    def f(k=_p(), kp=_p(), dt=0, dim=64, kv=1, pairs=0, inv=None, ftype=0, pages=8, page=16, q=None, qo=None, **step):
        return L.cernels_paged_append(q, 64, 64, 1, qo, k, 64, 64, _p(), 64, 64, kv, dim, dt, inv, ftype, pairs, 0, 1.0, kp, _p(),
                                      _strides(), pages, page, *_step(**step), None)

    assert f(tokens=0) == 0 and f(seqs=0) == 0
    assert f(k=None) == 1 and f(dt=2) == 1 and f(kv=0) == 1 and f(q=_p()) == 1 and f(pairs=4, ftype=2) == 1 and f(pairs=4, inv=_p()) == 1
    assert f(table=None) == 1 and f(lengths=None) == 1 and f(stride=3) == 1 and f(offsets=None, tokens=5) == 1 and f(page=0) == 1
    assert f(page=24) == 2 and f(pages=0) == 2 and f(seqs=65536) == 2 and f(blocks=1 << 27, stride=1 << 27) == 2
    assert f(k=_p(0x10001)) == 3 and f(lengths=_p(0x10002)) == 3 and f(kp=_p(0x10001)) == 3


def test_attention_entry_statuses(L):
    def f(q=_p(), heads=4, kv=2, dim=64, dt=0, kp=_p(), strides=None, pages=8, page=16, max_new=0, scale=0.1, window=0, out=_p(),
          ws=_p(), n=1 << 40, **step):
        table, stride, blocks, lengths, offsets, seqs, tokens = _step(**step)
        return L.cernels_paged_attention(q, heads * dim, dim, heads, kv, dim, dt, kp, _p(), strides or _strides(), pages, page, table,
                                         stride, blocks, lengths, offsets, seqs, tokens, max_new, scale, window, None, out, ws,
                                         ctypes.c_size_t(n), None)

    assert f(tokens=0) == 0 and f(seqs=0) == 0
    assert f(heads=3) == 1 and f(kv=0) == 1 and f(window=-1) == 1 and f(max_new=-1) == 1 and f(dt=2) == 1 and f(q=None) == 1
    for bad in (0.0, -1.0, math.inf, math.nan):
        assert f(scale=bad) == 1
    assert f(offsets=None, tokens=5) == 1 and f(stride=2) == 1 and f(ws=None) == 1
    assert f(dim=96) == 2 and f(page=8) == 2 and f(pages=0) == 2 and f(seqs=65536) == 2
    assert f(kp=_p(0x10008)) == 3 and f(strides=_strides(head=60)) == 3 and f(strides=_strides(slot=-64)) == 3 and f(out=_p(0x10008)) == 3
    assert f(n=8) == 4
    size = L.cernels_paged_attention_workspace_bytes
    assert size(4, 2, 4, 3, 64, 16, 4, 0) == 0 and size(4, 2, 4, 2, 80, 16, 4, 0) == 0 and size(0, 2, 4, 2, 64, 16, 4, 0) > 0
    need = size(1, 1, 32, 4, 128, 16, 500, 1)
    assert need > 16 and f(tokens=1, seqs=1, heads=32, kv=4, dim=128, blocks=500, stride=500, n=need - 1, max_new=1) == 4


def test_attention_workspace_stays_small(L):
    """Whatever a step holds, partial results are a few megabytes: splits are for steps of few rows."""
    for tokens, seqs, blocks in ((1, 1, 8192), (64, 64, 8192), (4096, 1, 8192), (4096, 64, 512), (100000, 100, 8192), (1 << 20, 3, 100)):
        for heads, kv, dim in ((32, 4, 128), (64, 8, 64), (16, 2, 256)):
            for most in (0, 1, 4096):
                n = L.cernels_paged_attention_workspace_bytes(tokens, seqs, heads, kv, dim, 16, blocks, most)
                assert 16 <= n <= 256 << 20, (tokens, seqs, heads, most, n)
