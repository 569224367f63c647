"""The decoder's prompts computed in chunks, then decode steps, over 16-bit and 8-bit caches:
every attention call against 64 bits, every written row against its definition."""

from __future__ import annotations

import pytest
import torch

from mxflashattn_amd.integrations.vllm import decode_step
from mxflashattn_amd.integrations.vllm.decode_step import (
    ROW_CACHE_DTYPES,
    DecoderModel,
    DecoderShape,
    RowCache,
)

from paged_reference import Paged, attend, check, half_step, quantise, rows_of

TINY = DecoderShape(layers=2, hidden=256, q_heads=8, kv_heads=2, head_dim=128, intermediate=512,
                    vocab=1000)
KINDS = pytest.mark.parametrize("kind", ["auto", "fp8", *ROW_CACHE_DTYPES])


def test_passes_cover_the_prompts_in_order():
    passes = decode_step.prompt_passes([5, 40, 200, 17, 64], 64)
    assert [sum(e - f for _, f, e in p) for p in passes] == [64, 64, 64, 64, 64, 6]
    at = [0] * 5
    for b, first, end in (part for p in passes for part in p):
        assert first == at[b] and end > first
        at[b] = end
    assert at == [5, 40, 200, 17, 64]


def test_prompts_that_do_not_fit_are_refused():
    model = DecoderModel(TINY, torch.device("cpu"))
    st = decode_step.build_state(model, 2, torch.tensor([5, 9]), new_tokens=2)
    with pytest.raises(ValueError, match="every prompt"):
        decode_step.fill_prompts(model, st, torch.zeros(13, dtype=torch.int64))
    with pytest.raises(ValueError, match="at least one token"):
        decode_step.fill_prompts(model, st, torch.zeros(14, dtype=torch.int64), chunk=0)


@pytest.mark.parametrize("kind", list(ROW_CACHE_DTYPES))
def test_synthetic_row_caches(kind):
    x = torch.randn(2, 3, 16, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    cache = RowCache.of(x, kind)
    codes, scales = quantise(x, ROW_CACHE_DTYPES[kind][0])
    assert cache.scales.shape == (2, 3, 2, 16)
    # (A division by a number may go through its reciprocal: one step of 2^-23 more.)
    torch.testing.assert_close(cache.scales.transpose(2, 3), scales, rtol=2.0 ** -22, atol=0)
    back = cache.codes.float() * cache.scales.transpose(2, 3)[..., None]
    step = 0.5 / 127 if kind == "int8_rows" else half_step(torch.float8_e4m3fn)
    assert bool(((back - x.float()).abs() <= 1.01 * step * x.float().abs().amax(-1, True)).all())


class Watched(DecoderModel):
    """Checks each attention call: its output over the cache as it then stands, and the rows
    that it wrote."""

    calls = 0

    def _check(self, q, k, v, kv_cache, meta, out):
        self.calls += 1
        torch.cuda.synchronize()
        rows = isinstance(kv_cache, RowCache)
        one = 1.0 if self.kv_cache_dtype == "fp8" else None
        kc, vc = (kv_cache.codes if rows else kv_cache).cpu().unbind(0)
        ks, vs = kv_cache.scales.cpu().unbind(0) if rows else (None, None)
        p = Paged(kc, vc, ks, vs, meta.block_table.cpu(), meta.seq_lens.cpu())
        cu = meta.query_start_loc.tolist()
        for b, (a, e) in enumerate(zip(cu, cu[1:])):
            want, bound = attend(q[a:e].cpu(), *rows_of(p, b), self.scale,
                                 weight_step=half_step(q.dtype), out_step=half_step(q.dtype))
            check(out.view(q.shape)[a:e], want, bound, f"sequence {b}, tokens {a} to {e}")
        slots, ps = meta.slot_mapping.cpu(), kc.shape[1]
        for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
            held = codes[slots // ps, slots % ps]
            if rows:
                want, scale = quantise(x.cpu(), held.dtype)
                assert torch.equal(scales[slots // ps, :, slots % ps], scale)
            else:
                want = x.cpu() if one is None else x.cpu().float().clamp(-448, 448).to(held.dtype)
            assert torch.equal(held.float(), want.float())

    def attention(self, layer, q, k, v, kv_cache, meta, out):
        super().attention(layer, q, k, v, kv_cache, meta, out)
        self._check(q, k, v, kv_cache, meta, out)

    def prompt_attention(self, layer, q, k, v, kv_cache, meta, out):
        super().prompt_attention(layer, q, k, v, kv_cache, meta, out)
        self._check(q, k, v, kv_cache, meta, out)


@pytest.mark.gpu
@KINDS
def test_prompts_then_steps(device, kind):
    model = Watched(TINY, device, seed=5, kv_cache_dtype=kind)
    prompt = torch.tensor([5, 40, 200, 17, 64])
    st = decode_step.build_state(model, 5, prompt, new_tokens=4)
    g = torch.Generator().manual_seed(9)
    tokens = torch.randint(0, TINY.vocab, (326,), generator=g).to(device)
    logits = decode_step.fill_prompts(model, st, tokens, chunk=64)
    assert model.calls == 2 * 6 and bool(logits.isfinite().all())
    for _ in range(2):
        st.tokens.copy_(logits.argmax(-1))
        logits = model.step(st.tokens, st.positions, st.kv_caches, st.meta)
        decode_step.advance(st)
    assert model.calls == 2 * 8 and bool(logits.isfinite().all())


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("eager", [False, True], ids=["graph", "eager"])
def test_run_with_computed_prompts(device, kind, eager):
    res = decode_step.run(batch=4, new_tokens=5, shape=TINY, median=64, lo=16, hi=256,
                          device=device, kv_cache_dtype=kind, eager=eager, prefill=100)
    assert res["logits_finite"] and res["prefill_tok_s"] > 0
    assert res["prefill_tokens"] == sum(decode_step.lognormal_prompt_lengths(
        4, 64, 1.0, 16, 256, 20261007).tolist())
