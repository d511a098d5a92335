"""The paged decoder (cernels_amd.modeling.paged): pages and their tables on the CPU; on the GPU the library's norm, rotary, cache and
attention run together on the real transformers architectures, against the stock model."""

from __future__ import annotations

import pytest
import torch

from cernels_amd.modeling import models as M
from cernels_amd.modeling import paged, swaps

_NMC = dict(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=64,
            prefix_dense_intermediate_size=256, num_experts=8, vocab_size=1000, sliding_window=24)
_DS = dict(hidden_size=128, intermediate_size=256, moe_intermediate_size=64, num_attention_heads=2,
           num_key_value_heads=2, n_routed_experts=8, num_experts_per_tok=2, vocab_size=1000)


def test_pool_grows_returns_and_refuses():
    pool = paged.PagePool(2, 6, 1, 64, torch.float32, torch.device("cpu"), page_size=16)
    pool.open(3)
    pool.grow([17, 0, 16])
    assert [len(h) for h in pool.held] == [2, 0, 1] and pool.counts == [17, 0, 16]
    assert pool.table.shape == (3, 2) and int(pool.table[2, 1]) == -1 and (pool.table[1] == -1).all()
    held = [p for h in pool.held for p in h]
    assert len(set(held)) == 3 and not set(held) & set(pool.free)
    before = (pool.counts, pool.table)
    with pytest.raises(RuntimeError, match="exhausted"):
        pool.grow([0, 65, 0])
    assert (pool.counts, pool.table) == before and len(pool.free) == 3
    pool.grow([0, 0, 1])
    assert pool.table.shape == (3, 2) and pool.counts == [17, 0, 17]
    pool.open(1)
    assert len(pool.free) == 6 and pool.counts == [0]


def test_other_models_are_refused():
    with pytest.raises(RuntimeError, match="PagedDecoder runs"):
        paged.PagedDecoder(type("M", (), {"model": torch.nn.Linear(1, 1)})(), 4)


def _model(name, dtype=torch.bfloat16):
    spec, tiny = (M.NORTH_MINI_CODE, _NMC) if name == "north_mini_code" else (M.DEEPSEEK_OCR_2, _DS)
    model = M.build(spec, device="cuda", layers=5, **tiny).to(dtype)
    model.set_experts_implementation("eager")
    return model


def _prompts(lengths):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(100, 999, (n,), generator=g).cuda() for n in lengths]


def _stock_logits(model, ids):
    return model(input_ids=ids[None], attention_mask=torch.ones_like(ids)[None]).logits[0].float()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["north_mini_code", "deepseek_ocr_2"])
def test_ragged_steps_match_the_stock_model(device, name):
    """Three prompts of different lengths in one step, then chunks and single tokens, one sequence pausing: every step's logits
    against the stock forward of that sequence alone. fp16 weights keep 5 layers of rounding small: the bound is 2% of the logits'
    largest, some 40 half steps of fp16 (2^-11) through 5 layers."""
    model = _model(name, torch.float16)
    prompts = _prompts([70, 9, 41])
    print(f"[paged {name}]", flush=True)
    with torch.no_grad():
        want = [_stock_logits(model, p) for p in prompts]
    decoder = paged.PagedDecoder(model, pages=20, page_size=16)
    for cuts in ([[70, 9, 41]], [[33, 5, 40], [30, 0, 1], [1, 1, 0], [1, 1, 0], [5, 2, 0]]):
        decoder.pool.open(3)
        at = [0, 0, 0]
        for cut in cuts:
            got = decoder.step([p[a:a + n] for p, a, n in zip(prompts, at, cut)])
            at = [a + n for a, n in zip(at, cut)]
            for b, n in enumerate(cut):
                if n == 0:
                    assert not got[b].any()
                    continue
                ref = want[b][at[b] - 1]
                assert float((got[b].float() - ref).abs().max()) <= 0.02 * float(ref.abs().max()), (cuts, b)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["north_mini_code", "deepseek_ocr_2"])
def test_swapped_experts_in_the_paged_decoder(device, name):
    """bf16 with the library's experts: prompt logits close to stock's (the whole-model runner's bar), greedy tokens come out, whole
    prompts and chunks alike."""
    model = _model(name)
    prompts = _prompts([50, 13])
    with torch.no_grad():
        want = [_stock_logits(model, p)[-1] for p in prompts]
    swaps.SWAPS[name][0](model, "custom")
    try:
        decoder = paged.PagedDecoder(model, pages=16, page_size=16)
        got = decoder.step(prompts).float()
        for g, w in zip(got, want):
            assert float((g - w).abs().max()) <= 0.05 * float(w.abs().max()) + 1e-3
        tokens = decoder.generate(prompts, 6)
        assert tokens.shape == (2, 6)
        again = decoder.generate(prompts, 6)
        assert torch.equal(tokens, again)
        assert decoder.generate(prompts, 2, chunk=16).shape == (2, 2)
    finally:
        swaps.SWAPS[name][0](model, "stock")


@pytest.mark.gpu
def test_measured_as_a_variant(device):
    from cernels_amd.modeling import main as runner

    model = _model("north_mini_code")
    inputs = M.prompt_ids(M.NORTH_MINI_CODE, 40, "cuda", vocab=1000)
    opts = runner.Options(gate_tokens=4, decode_tokens=4, decode_runs=1, prefill_seconds=0.02)
    ref = runner.trace(model, inputs, 4)
    got = paged.measure(model, inputs, opts, ref)
    stock = {"prefill_ms", "decode_tok_s", "generate_s", "gate_token_match", "gate_prefix", "last_logits_max_diff", "last_logits_std"}
    assert set(got) == stock and got["decode_tok_s"] > 0
