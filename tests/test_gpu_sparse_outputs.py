"""Sparse decode where something is left to select, in the output types, attention variants and grids that the dense wrapper has."""
import math

import pytest
import torch

from oracle import mla_fp4_oracle as O
from oracle import sparse_oracle as S
from test_gpu_sparse import E4M3, _sparse_case, _wrapper

pytestmark = pytest.mark.gpu


def _variant(which, heads, q):
    """(variant of the wrapper, arguments of the oracle): sinks from below to above the scores, a cap that the scores reach."""
    from flashinfer_mla_fp4_b200 import AttentionWithSink, SoftCappingAttention

    sink = (torch.rand(heads, generator=torch.Generator().manual_seed(heads)) * 12.0 - 4.0).to(q.device)
    cap = max(1.0, 0.5 * O.decode_e4m3(q.cpu()).float()[..., :512].norm(dim=-1).mean().item())
    return {"plain": (None, {}), "sink": (AttentionWithSink(sink), dict(sink=sink.cpu())), "cap": (SoftCappingAttention(cap), dict(logits_soft_cap=cap)),
            "cap and sink": (SoftCappingAttention(cap, sink=sink), dict(logits_soft_cap=cap, sink=sink.cpu()))}[which]


@pytest.mark.parametrize("which", ["plain", "sink", "cap", "cap and sink"])
@pytest.mark.parametrize("out_dtype,output_scale", [(torch.bfloat16, 1.0), (torch.float32, 0.37), (E4M3, 8.0)])
@pytest.mark.parametrize("lens,heads,page,q_len,budget,causal,max_ctas", [
    ([9000, 1, 0, 700, 512], 64, 64, 1, 8, False, None),
    ([3000, 5, 1999], 40, 16, 3, 20, True, 7),
    ([4000, 2500], 128, 32, 2, 12, False, 40),
    ([6000], 16, 8, 1, 40, False, 1),
])
def test_sparse_decode_in_every_type_variant_and_grid(lens, heads, page, q_len, budget, causal, max_ctas, out_dtype, output_scale, which):
    cache, bt, sl, q = _sparse_case(lens, heads, page, q_len, seed=heads)
    scale = 512 ** -0.5
    variant, kw = _variant(which, heads, q)
    w = _wrapper(num_heads=heads, page_size=page, budget_pages=budget, causal=causal, out_dtype=out_dtype, variant=variant, max_ctas=max_ctas)
    out, lse = w.run(q, cache.kv_cache, bt, sl, max(lens), scale, output_scale, kv_cache_sf=cache.kv_cache_sf, summary=cache.summary,
                     summary_sf=cache.summary_sf, return_lse=True)
    torch.cuda.synchronize()
    w.check_device_status()
    sel, sel_lens = S.select(q.cpu(), cache.summary.cpu(), cache.summary_sf.cpu(), bt.cpu(), sl.cpu(), page, budget, 1, 2, causal)
    ref, ref_lse = O.mla_decode(q.cpu().reshape(-1, 1, heads, 576), cache.kv_cache, cache.kv_cache_sf, sel, sel_lens, scale, output_scale, **kw)
    ref, ref_lse = ref.view(len(lens), q_len, heads, 512), ref_lse.view(len(lens), q_len, heads)
    got = out.float().cpu()
    assert out.dtype == out_dtype
    if out_dtype == E4M3:
        # half a step of a 3-bit mantissa, the bar for the other types (of a head's RMS), half a subnormal step
        tol = ref.abs() * 2.0 ** -4 + 2e-2 * ref.pow(2).mean(dim=-1, keepdim=True).sqrt() + 2.0 ** -10
        assert bool(torch.isfinite(got).all()) and bool(((got - ref).abs() <= tol).all()), float(((got - ref).abs() - tol).max())
    else:
        O.assert_parity(got, ref, f"sparse decode, {which}")
    there = torch.isfinite(ref_lse)
    torch.testing.assert_close(lse.cpu()[there], ref_lse[there], atol=2e-3, rtol=1e-4)
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any()
            assert which != "plain" or bool((lse[b] == -math.inf).all())
