"""Sparse decode on the GPU: page summaries and selections equal to the oracle's to the last bit (both are whole numbers, or one rounding of a
product that 64 bits hold), attention over the selected pages within the dense decode's tolerance, and the call in all the ways it is used."""
import math

import pytest
import torch

from oracle import mla_fp4_oracle as O
from oracle import sparse_oracle as S

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def _pages(n, page, seed):
    """Cache pages on the host whose tokens have something in common."""
    from flashinfer_mla_fp4_b200.kvcache import quantize_tokens

    g = torch.Generator().manual_seed(seed)
    lat = (torch.randn(n, 1, 512, generator=g) + torch.randn(n, page, 512, generator=g)) * (0.2 + 3 * torch.rand(n, page, 1, generator=g))
    return quantize_tokens(lat, torch.randn(n, 1, 64, generator=g) + torch.randn(n, page, 64, generator=g))


def _oracle_summaries(kv, sf):
    got = [S.summarize(kv[i], sf[i]) for i in range(kv.shape[0])]
    return torch.stack([c for c, _ in got]), torch.tensor([s for _, s in got], dtype=torch.float32)


def _same(a, b):
    return torch.equal(a.nan_to_num(nan=-1.0), b.nan_to_num(nan=-1.0)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128])
def test_summaries_of_ordinary_and_outlying_pages(page):
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import summarize_pages

    kv, sf = _pages(24, page, page)
    sf[1] = 0.0
    sf[2, 3] = float("inf")
    sf[3, 0] = float("nan")
    kv[4, page - 1, 300] = 0x7F  # NaN among the RoPE values
    kv[5, 0, 256] = 0xFF
    sf[6, ::2] *= -1
    sf[7] *= 1e-38  # products with these are subnormal
    sf[8] = 1e-45
    kv[8, :, 256:] = 0
    sf[9] = 3e38
    kv[9, :, :256] = 0x77  # a mean above FP32
    sf[10, 1:] = sf[10, 0] * 1e-6  # one token outweighs the others
    kv[11] = 0
    kv[12, :, 256:] = 0x7E  # 448 everywhere
    kv[13, :, :256], sf[13] = 0xFF, 1.0
    sf[14] = 2.0 ** -149
    ids = torch.tensor([*range(15), -1, 24, 2**31 - 1, 17, 17, 23], dtype=torch.int32)
    summary, ssf = torch.full((24, 576), 9, dtype=torch.int8, device=dev), torch.full((24,), 9.0, device=dev)
    summarize_pages(kv.to(dev), sf.to(dev), summary, ssf, ids.to(dev))
    want, want_sf = _oracle_summaries(kv, sf)
    for i in (15, 16, 18, 19, 20, 21, 22):  # not named
        want[i], want_sf[i] = 9, 9.0
    for i in range(24):
        assert torch.equal(summary[i].cpu(), want[i]), i
    assert _same(ssf.cpu(), want_sf)


@pytest.mark.parametrize("page,new", [(8, 1), (8, 20), (64, 1), (64, 200), (128, 3)])
def test_summaries_of_the_pages_that_a_step_has_filled(page, new):
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import summarize_new_pages

    lens = [0, 1, page, page + 1, 2 * page, 5 * page, 5 * page - 1, 6 * page, 100 * page, -3]  # (one is longer than its row, one negative)
    width, pool = 6, len(lens) * 6 + 5
    kv, sf = _pages(pool, page, 5)
    g = torch.Generator().manual_seed(1)
    bt = torch.randperm(pool, generator=g)[: len(lens) * width].view(len(lens), width).int()
    bt[7, 5] = pool + 7  # outside the pool
    wide = torch.zeros(len(lens), 9, dtype=torch.int32)
    wide[:, :width] = bt
    summary, ssf = torch.full((pool, 576), 9, dtype=torch.int8, device=dev), torch.full((pool,), 9.0, device=dev)
    summarize_new_pages(kv.to(dev), sf.to(dev), summary, ssf, wide.to(dev)[:, :width], torch.tensor(lens, dtype=torch.int32, device=dev), new)
    codes, scales = _oracle_summaries(kv, sf)
    want, want_sf = torch.full((pool, 576), 9, dtype=torch.int8), torch.full((pool,), 9.0)
    for b, n in enumerate(lens):
        n = min(n, width * page)
        for k in range(width):
            if n - new < (k + 1) * page <= n and bt[b, k] < pool:
                want[bt[b, k]], want_sf[bt[b, k]] = codes[bt[b, k]], scales[bt[b, k]]
    assert torch.equal(summary.cpu(), want) and torch.equal(ssf.cpu(), want_sf)


@pytest.mark.parametrize("page", [32, 64, 128])
def test_summaries_of_many_pages(page):
    """Enough pages for the kernel that has the sums made by the tensor cores: the bytes that the other one writes, page for page, and the oracle's
    for some; outlying pages among them, pages that are not named, an odd number of them, a last tile that is not full."""
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import summarize_pages

    few = 24
    kv, sf = _pages(few, page, page + 1)
    sf[1], sf[2, 3], sf[3, 0] = 0.0, float("inf"), float("nan")
    kv[4, page - 1, 300], kv[5, 0, 256] = 0x7F, 0xFF
    sf[6, ::2] *= -1
    sf[7] *= 1e-38
    sf[8], kv[8, :, 256:] = 1e-45, 0
    sf[9], kv[9, :, :256] = 3e38, 0x77
    sf[10, 1:] = sf[10, 0] * 1e-6
    kv[11] = 0
    kv[12, :, 256:] = 0x7E
    kv[13, :, :256], sf[13] = 0xFF, 1.0
    want, want_sf = _oracle_summaries(kv, sf)
    pool = 140000 // page + 3
    g = torch.Generator(device=dev).manual_seed(page)
    which = torch.randint(0, few, (pool,), generator=g, device=dev)
    kv_all, sf_all = kv.to(dev)[which], sf.to(dev)[which]
    ids = torch.randperm(pool, generator=g, device=dev).int()[: pool - 5]
    ids = torch.cat((ids, torch.tensor([-1, pool, 2**31 - 1], dtype=torch.int32, device=dev), ids[:1]))
    ids = ids[torch.randperm(ids.numel(), generator=g, device=dev)].contiguous()
    assert ids.numel() * page >= 131072
    summary, ssf = torch.full((pool, 576), 9, dtype=torch.int8, device=dev), torch.full((pool,), 9.0, device=dev)
    status = torch.zeros(8, dtype=torch.int32, device=dev)
    summarize_pages(kv_all, sf_all, summary, ssf, ids, status)
    named = torch.zeros(pool, dtype=torch.bool, device=dev)
    named[ids[(ids >= 0) & (ids < pool)].long()] = True
    exp, exp_sf = want.to(dev)[which], want_sf.to(dev)[which]
    exp[~named], exp_sf[~named] = 9, 9.0
    torch.cuda.synchronize()
    assert int(status[0]) == 0
    assert torch.equal(summary, exp) and _same(ssf, exp_sf)
    # a cache that starts on 16 bytes but not on 32 goes to the other kernel
    raw = torch.empty(kv_all.numel() + 64, dtype=torch.uint8, device=dev)
    start = (16 - raw.data_ptr()) % 32
    odd = raw[start:start + kv_all.numel()].view_as(kv_all).copy_(kv_all)
    again, again_sf = torch.full_like(summary, 9), torch.full_like(ssf, 9.0)
    summarize_pages(odd, sf_all, again, again_sf, ids)
    assert torch.equal(again, exp) and _same(again_sf, exp_sf)
    # ... and so do scales that start on 4
    raw = torch.empty(sf_all.numel() + 1, device=dev)
    odd = raw[1:].view_as(sf_all).copy_(sf_all)
    assert odd.data_ptr() % 16 == 4
    again.fill_(9), again_sf.fill_(9.0)
    summarize_pages(kv_all, odd, again, again_sf, ids)
    assert torch.equal(again, exp) and _same(again_sf, exp_sf)


def _selection_case(lens, heads, page, q_len, seed, odd=False):
    g = torch.Generator().manual_seed(seed)
    used = [max(0, -(-n // page)) for n in lens]
    width, pool = max(1, max(used)), sum(used) + 3
    perm = torch.randperm(pool, generator=g).int()
    bt, at = torch.zeros(len(lens), width, dtype=torch.int32), 0
    for b, n in enumerate(used):
        bt[b, :n] = perm[at:at + n]
        at += n
    summary = torch.randint(-127, 128, (pool, 576), generator=g, dtype=torch.int8)
    ssf = torch.rand(pool, generator=g) * 0.1
    q = (torch.randn(len(lens), q_len, heads, 576, generator=g) * torch.exp(torch.randn(1, 1, heads, 1, generator=g))).to(E4M3)
    if odd:
        ssf[::7] = float("nan")
        ssf[1::7] = 0.0
        summary[2::7], ssf[2::7] = summary[2], ssf[2]  # ties
        qb = q.view(torch.uint8)
        qb[0, 0, 0, 5] = 0x7F  # NaN counts as zero
        qb[0, 0, heads - 1] = 0
        qb[0, 0, heads // 2] = 0x01  # the smallest subnormal
        qb[-1, -1, 0] = 0xFE  # -448
        bt[0, 2] = pool + 5
        bt[0, 3] = -7
    return q, summary, ssf, bt, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.parametrize("lens,heads,page,q_len,budget,sink,local,causal,odd", [
    ([700], 16, 8, 1, 12, 1, 2, False, False),
    ([1, 0, 64, 65, 640, 641, 704, 6400], 64, 64, 1, 10, 1, 2, False, False),
    ([5000, 3, 9999, 0, 4097], 40, 16, 3, 33, 2, 3, True, False),
    ([5000, 3, 9999, 0, 4097], 40, 16, 3, 33, 2, 3, False, True),
    ([2000, 1000], 128, 8, 2, 7, 0, 1, True, True),
    ([4000], 1, 32, 1, 4, 0, 4, False, False),  # nothing left for scores
    ([4000], 3, 32, 1, 5, 4, 1, False, False),
    ([4000], 5, 32, 1, 5, 0, 1, False, True),
    ([30000, 257 * 128], 96, 128, 1, 40, 1, 2, False, True),
    ([9000, 100], 64, 64, 1, 1000, 1, 2, False, False),  # a budget beyond the tables
    ([66000, 40000], 17, 8, 1, 600, 3, 5, False, True),
    ([8000, 8001], 33, 8, 1, 990, 3, 5, False, False),  # nearly all
    ([140000, 131200], 8, 8, 1, 700, 1, 2, False, True),  # more candidates than a CTA's registers hold
    ([1030] * 1100, 4, 128, 1, 8, 1, 2, False, False),  # more rows than a launch, hardly a tile each
    ([300, 9000, 17, 1100, 0, 128 * 130], 112, 8, 2, 20, 1, 2, True, True),  # tiles of different rows in turn
    ([300, 90] * 200, 70, 8, 3, 8, 1, 2, True, True),  # a launch that ends inside a request
    ([131000, 2401, 2400, 2402, 0], 8, 8, 3, 300, 1, 2, True, True),  # positions together; some of a request within the budget, others not
    ([70000, 0, 69999, 8 * 40 + 1], 20, 16, 4, 16, 0, 1, True, True),
    ([70000, 0, 69999, 8 * 40 + 1], 64, 16, 2, 16, 1, 2, False, True),
    ([700, 1500, 90] * 134, 4, 8, 3, 8, 1, 2, True, True),
    ([300, 90] * 550, 3, 8, 2, 8, 1, 2, True, False),  # ... of more requests than a launch
    ([1030, 50, 900] * 30, 6, 8, 3, 8, 1, 2, True, True),  # a CTA a row, more of them than SMs
])
def test_selection_equals_the_oracle(lens, heads, page, q_len, budget, sink, local, causal, odd):
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import select_pages

    q, summary, ssf, bt, sl = _selection_case(lens, heads, page, q_len, seed=len(lens) + heads, odd=odd)
    want, want_lens = S.select(q, summary, ssf, bt, sl, page, budget, sink, local, causal)
    got, got_lens = select_pages(q.to(dev), summary.to(dev), ssf.to(dev), bt.to(dev), sl.to(dev), page, budget, sink_pages=sink,
                                 local_pages=local, causal=causal)
    assert torch.equal(got_lens.cpu(), want_lens)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("pages", [40, 3000, 17000])
@pytest.mark.parametrize("shape", ["negative", "negative and NaN", "two values", "one value", "one page stands out", "infinite"])
def test_selection_over_scores_of_any_spread(pages, shape):
    """Scores made to order: a summary with one code, a query with one value."""
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import select_pages

    g = torch.Generator().manual_seed(pages)
    summary, ssf = torch.zeros(pages, 576, dtype=torch.int8), torch.ones(pages)
    summary[:, 7] = 1
    q = torch.zeros(1, 1, 1, 576)
    q[..., 7] = 2.0
    if shape.startswith("negative"):
        ssf = -torch.rand(pages, generator=g) * 10.0 ** torch.randint(-30, 30, (pages,), generator=g)
        if shape != "negative":
            ssf[torch.randperm(pages, generator=g)[: pages // 9]] = math.nan
    elif shape == "two values":
        ssf[torch.randperm(pages, generator=g)[: pages // 2]] = 1.0 + 2.0 ** -23
    elif shape == "one page stands out":
        ssf[pages // 2] = 2.0
    elif shape == "infinite":
        ssf[3], ssf[5], summary[9, 7] = math.inf, -math.inf, 0
        ssf[9] = math.inf  # times zero: NaN
    bt = torch.randperm(pages, generator=g).int().view(1, -1)
    sl = torch.tensor([pages * 8 - 3], dtype=torch.int32)
    want, want_lens = S.select(q.to(E4M3), summary, ssf, bt, sl, 8, 20, 1, 2, False)
    room = torch.full((1 + pages // 20 + 1, 20), -9, dtype=torch.int32, device=dev)
    got, lens = select_pages(q.to(E4M3).to(dev), summary.to(dev), ssf.to(dev), bt.to(dev), sl.to(dev), 8, 20, selected=room[:1])
    assert torch.equal(got.cpu(), want) and torch.equal(lens.cpu(), want_lens)
    assert bool((room[1:] == -9).all())


def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right():
    """A poll budget of one: the first wait for a tile's loads gives up.  What is selected then are pages of the request all the same."""
    dev = _dev()
    import ctypes as C

    from flashinfer_mla_fp4_b200 import _cabi

    q, summary, ssf, bt, sl = _selection_case([9000, 700, 12000], 64, 8, 1, seed=3)
    want, want_lens = S.select(q, summary, ssf, bt, sl, 8, 30, 1, 2, False)
    qd, summary, ssf, btd, sld = (t.to(dev) for t in (q, summary, ssf, bt, sl))
    sel, lens = torch.empty(3, 30, dtype=torch.int32, device=dev), torch.empty(3, dtype=torch.int32, device=dev)
    ws, status = torch.zeros(_cabi.select_workspace_bytes(3, 1, bt.shape[1]), dtype=torch.int8, device=dev), torch.zeros(8, dtype=torch.int32, device=dev)
    a = _cabi.SelectArgs()
    a.q, a.q_stride_batch, a.q_stride_qpos, a.q_stride_head = qd.data_ptr(), qd.stride(0), qd.stride(1), qd.stride(2)
    a.summary, a.summary_sf, a.num_pages = summary.data_ptr(), ssf.data_ptr(), summary.shape[0]
    a.block_tables, a.block_table_stride, a.seq_lens = btd.data_ptr(), btd.stride(0), sld.data_ptr()
    a.selected, a.selected_lens, a.workspace, a.workspace_bytes = sel.data_ptr(), lens.data_ptr(), ws.data_ptr(), ws.numel()
    a.batch, a.q_len, a.num_heads, a.page_size, a.width = 3, 1, 64, 8, bt.shape[1]
    a.budget, a.sink_pages, a.local_pages, a.status, a.wait_polls = 30, 1, 2, status.data_ptr(), 1
    a.stream = torch.cuda.current_stream().cuda_stream
    _cabi.check(_cabi.lib.mla_fp4_select_pages(C.byref(a)))
    torch.cuda.synchronize()
    assert int(status[0]) in (0, _cabi.ERR_DEVICE_TIMEOUT)
    assert torch.equal(lens.cpu(), want_lens)
    for b in range(3):
        assert set(sel[b].tolist()) <= set(bt[b].tolist())
    status.zero_()
    a.wait_polls = 0
    _cabi.check(_cabi.lib.mla_fp4_select_pages(C.byref(a)))
    torch.cuda.synchronize()
    assert int(status[0]) == 0 and torch.equal(sel.cpu(), want)


def test_selection_from_strided_queries_and_tables_into_given_buffers():
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import select_pages

    q, summary, ssf, bt, sl = _selection_case([3000, 2000], 24, 16, 2, seed=9)
    sl = sl + 10**6  # beyond what the table can hold: cut to its width
    wide_q = torch.zeros(2, 2, 40, 640, dtype=torch.uint8, device=dev)
    wide_q[:, :, 8:32, 32:608] = q.view(torch.uint8).to(dev)
    wide_bt = torch.full((2, bt.shape[1] + 5), -1, dtype=torch.int32, device=dev)
    wide_bt[:, 2:-3] = bt.to(dev)
    sel, lens = torch.empty(4, 20, dtype=torch.int32, device=dev), torch.empty(4, dtype=torch.int32, device=dev)
    ws = torch.empty(4 * 4 * ((bt.shape[1] + 3) // 4 * 4), dtype=torch.int8, device=dev)
    got = select_pages(wide_q.view(E4M3)[:, :, 8:32, 32:608], summary.to(dev), ssf.to(dev), wide_bt[:, 2:-3], sl.to(dev), 16, 20,
                       selected=sel, selected_lens=lens, workspace=ws)
    assert got[0] is sel and got[1] is lens
    want, want_lens = S.select(q, summary, ssf, bt, sl, 16, 20, 1, 2, False)
    assert torch.equal(sel.cpu(), want) and torch.equal(lens.cpu(), want_lens)


def _sparse_case(lens, heads, page, q_len, seed):
    """A cache with its summaries on the GPU, filled through the public writers of the format."""
    from flashinfer_mla_fp4_b200 import FP4MLAPagedCache
    from flashinfer_mla_fp4_b200.sparse import summarize_new_pages

    dev = _dev()
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    width, pool = max(1, max(used)), sum(used) + 3
    cache = FP4MLAPagedCache(pool, page, dev, summaries=True)
    kv, sf = _pages(pool, page, seed)
    cache.kv_cache.copy_(kv)
    cache.kv_cache_sf.copy_(sf)
    perm, at = torch.randperm(pool, generator=g).int(), 0
    bt = torch.zeros(len(lens), width, dtype=torch.int32)
    for b, n in enumerate(used):
        bt[b, :n] = perm[at:at + n]
        at += n
    bt, sl = bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    summarize_new_pages(cache.kv_cache, cache.kv_cache_sf, cache.summary, cache.summary_sf, bt, sl, max(max(lens), 1))
    q = torch.randn(len(lens), q_len, heads, 576, generator=g).to(E4M3).to(dev)
    return cache, bt, sl, q


def _expected(cache, bt, sl, q, page, budget, sink, local, causal, scale, **kw):
    B, q_len, H, _ = q.shape
    sel, lens = S.select(q.cpu(), cache.summary.cpu(), cache.summary_sf.cpu(), bt.cpu(), sl.cpu(), page, budget, sink, local, causal)
    out, lse = O.mla_decode(q.cpu().reshape(B * q_len, 1, H, 576), cache.kv_cache, cache.kv_cache_sf, sel, lens, scale, **kw)
    return out.view(B, q_len, H, 512), lse.view(B, q_len, H)


def _wrapper(**plan):
    from flashinfer_mla_fp4_b200 import BatchMLASparseDecodeFP4Wrapper

    w = BatchMLASparseDecodeFP4Wrapper(torch.empty(32 << 20, dtype=torch.int8, device=_dev()))
    w.plan(**plan)
    return w


@pytest.mark.parametrize("lens,heads,page,q_len,budget,causal,out_dtype", [
    ([3000], 16, 64, 1, 8, False, torch.bfloat16),
    ([9000, 1, 0, 700, 512], 64, 64, 1, 8, False, torch.float32),
    ([3000, 5, 1999], 40, 16, 3, 20, True, torch.bfloat16),
    ([4000, 2500], 128, 32, 2, 12, False, torch.float32),
    ([2000, 130], 128, 8, 1, 30, False, torch.bfloat16),
])
def test_sparse_decode_attends_to_the_selected_pages(lens, heads, page, q_len, budget, causal, out_dtype):
    cache, bt, sl, q = _sparse_case(lens, heads, page, q_len, seed=heads)
    scale = 512 ** -0.5
    w = _wrapper(num_heads=heads, page_size=page, budget_pages=budget, causal=causal, out_dtype=out_dtype)
    out, lse = w.run(q, cache.kv_cache, bt, sl, max(lens), scale, kv_cache_sf=cache.kv_cache_sf, summary=cache.summary,
                     summary_sf=cache.summary_sf, return_lse=True)
    torch.cuda.synchronize()
    w.check_device_status()
    ref, ref_lse = _expected(cache, bt, sl, q, page, budget, 1, 2, causal, scale)
    O.assert_parity(out.float().cpu(), ref, "sparse decode")
    there = torch.isfinite(ref_lse)
    torch.testing.assert_close(lse.cpu()[there], ref_lse[there], atol=2e-3, rtol=1e-4)
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].float().any() and bool((lse[b] == -math.inf).all())
    assert out.dtype == out_dtype


def test_a_budget_that_holds_everything_is_the_dense_decode():
    from flashinfer_mla_fp4_b200 import AttentionWithSink, BatchMLADecodeCuteDSLFP4Wrapper

    cache, bt, sl, q = _sparse_case([900, 1, 333], 32, 16, 1, seed=3)
    sink = torch.randn(32, generator=torch.Generator().manual_seed(4)).to(q.device)
    w = _wrapper(num_heads=32, page_size=16, budget_pages=bt.shape[1], variant=AttentionWithSink(sink))
    dense = BatchMLADecodeCuteDSLFP4Wrapper(torch.empty(32 << 20, dtype=torch.int8, device=q.device))
    dense.plan(num_heads=32, page_size=16, variant=AttentionWithSink(sink))
    out, lse = torch.empty(3, 1, 32, 512, dtype=torch.bfloat16, device=q.device), torch.empty(3, 1, 32, device=q.device)
    got = w.run(q, cache.kv_cache, bt, sl, 900, 0.05, 0.5, out=out, kv_cache_sf=cache.kv_cache_sf, summary=cache.summary,
                summary_sf=cache.summary_sf, return_lse=True, lse_out=lse)
    want = dense.run(q, cache.kv_cache, bt, sl, 900, 0.05, 0.5, kv_cache_sf=cache.kv_cache_sf, return_lse=True)
    assert got[0] is out and got[1] is lse
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_captured_step_follows_lengths_tables_and_queries():
    cache, bt, sl, q = _sparse_case([4000, 3000, 50], 64, 16, 1, seed=11)
    w = _wrapper(num_heads=64, page_size=16, budget_pages=24)
    out = torch.empty(3, 1, 64, 512, dtype=torch.bfloat16, device=q.device)

    def step():
        w.run(q, cache.kv_cache, bt, sl, 4000, 0.04, out=out, kv_cache_sf=cache.kv_cache_sf, summary=cache.summary, summary_sf=cache.summary_sf)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens, rows in (([4000, 3000, 50], [0, 1, 2]), ([1, 2999, 0], [1, 0, 2]), ([2999, 16 * 24 + 1, 16], [1, 0, 2])):
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        bt.copy_(bt[torch.tensor(rows, device=bt.device)].clone())
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(sum(lens))).to(E4M3))
        graph.replay()
        torch.cuda.synchronize()
        ref, _ = _expected(cache, bt, sl, q, 16, 24, 1, 2, False, 0.04)
        O.assert_parity(out.float().cpu(), ref, f"replay {lens}")
    w.check_device_status()


def test_two_streams_with_a_wrapper_each():
    cases = [_sparse_case([6000, 2000], 64, 32, 1, seed=s) for s in (1, 2)]
    ws = [_wrapper(num_heads=64, page_size=32, budget_pages=10) for _ in cases]
    streams, outs = [torch.cuda.Stream() for _ in cases], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (cache, bt, sl, q) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ws[i].run(q, cache.kv_cache, bt, sl, 6000, 0.04, kv_cache_sf=cache.kv_cache_sf, summary=cache.summary,
                                         summary_sf=cache.summary_sf))
    torch.cuda.synchronize()
    for i, (cache, bt, sl, q) in enumerate(cases):
        ref, _ = _expected(cache, bt, sl, q, 32, 10, 1, 2, False, 0.04)
        O.assert_parity(outs[i][0].float().cpu(), ref, f"stream {i}")
        assert all(torch.equal(o, outs[i][0]) for o in outs[i])


def test_sparse_run_refuses():
    cache, bt, sl, q = _sparse_case([900, 700], 16, 16, 2, seed=5)
    w = _wrapper(num_heads=16, page_size=16, budget_pages=8)
    ok = dict(q=q, kv_cache=cache.kv_cache, block_tables=bt, seq_lens=sl, max_seq_len=900, softmax_scale=0.05, kv_cache_sf=cache.kv_cache_sf,
              summary=cache.summary, summary_sf=cache.summary_sf)
    w.run(**ok)
    wide = torch.zeros(2, 3, 16, 576, dtype=torch.uint8, device=q.device).view(E4M3)
    for bad in (dict(q=q[:, :, :8]), dict(q=wide[:, :2]), dict(q=q.float()), dict(kv_cache_sf=None), dict(summary=None), dict(summary=cache.summary[:-1]),
                dict(summary_sf=cache.summary_sf.half()), dict(summary=cache.summary.cpu()), dict(seq_lens=sl.long()), dict(block_tables=bt.long()),
                dict(block_tables=bt[:1]), dict(max_seq_len=0), dict(max_seq_len=10**6), dict(kv_cache=cache.kv_cache[:, :8]),
                dict(out=torch.empty(2, 2, 16, 512, device=q.device)), dict(out=torch.empty(2, 1, 16, 512, dtype=torch.bfloat16, device=q.device))):
        with pytest.raises(ValueError):
            w.run(**{**ok, **bad})
    from flashinfer_mla_fp4_b200 import BatchMLASparseDecodeFP4Wrapper, FP4MLADecodeBackend, FP4MLAPagedCache, SparsePages

    small = BatchMLASparseDecodeFP4Wrapper(torch.empty(20 << 20, dtype=torch.int8, device=q.device))
    with pytest.raises(RuntimeError, match="plan"):
        small.run(**ok)
    small.plan(num_heads=16, page_size=16, budget_pages=8)
    need = BatchMLASparseDecodeFP4Wrapper.workspace_bytes(2, 2, 16, bt.shape[1], 8, torch.cuda.get_device_properties(0).multi_processor_count)
    short = BatchMLASparseDecodeFP4Wrapper(torch.empty(need - 1, dtype=torch.int8, device=q.device))
    short.plan(num_heads=16, page_size=16, budget_pages=8)
    with pytest.raises(ValueError, match=str(need)):
        short.run(**ok)
    exactly = BatchMLASparseDecodeFP4Wrapper(torch.empty(need, dtype=torch.int8, device=q.device))
    exactly.plan(num_heads=16, page_size=16, budget_pages=8)
    assert torch.equal(exactly.run(**ok), w.run(**ok))
    backend = FP4MLADecodeBackend(16, 16, 2, 900, 0.05, q.device, sparse=SparsePages(8))
    with pytest.raises(ValueError, match="summaries"):
        backend.forward(q[:, :1].contiguous(), torch.zeros(2, 512, device=q.device), torch.zeros(2, 64, device=q.device), FP4MLAPagedCache(4, 16, q.device))
    with pytest.raises(ValueError, match="context-parallel"):
        FP4MLADecodeBackend(16, 16, 2, 900, 0.05, q.device, sparse=SparsePages(8), cp_group=object())


@pytest.mark.parametrize("graph", [False, True])
def test_a_backend_with_sparse_pages_over_growing_requests(graph):
    """Prompts, then steps that fill pages, through allocation, a fork and compaction on the way, as a serving program would run them."""
    dev = _dev()
    from flashinfer_mla_fp4_b200 import FP4MLADecodeBackend, FP4MLAPagedCache, FP4MLAPagePool, SparsePages, decode_slot_mapping
    from flashinfer_mla_fp4_b200.kvcache import write_tokens
    from flashinfer_mla_fp4_b200.sparse import summarize_new_pages

    H, ps, budget, rows, scale = 32, 8, 9, 4, 576 ** -0.5
    cache = FP4MLAPagedCache(140, ps, dev, summaries=True)
    pool = FP4MLAPagePool([cache])
    backend = FP4MLADecodeBackend(H, ps, rows, 400, scale, dev, sparse=SparsePages(budget, 1, 2))
    step = backend.capture(cache) if graph else None
    bt, sl = torch.zeros(rows, 50, dtype=torch.int32, device=dev), torch.zeros(rows, dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(8)
    lens = torch.tensor([130, 200, 20, 0], dtype=torch.int32)
    pool.allocate(bt, sl, lens.to(dev))
    for b, n in enumerate(lens.tolist()):
        if n:
            slots = decode_slot_mapping(bt[b:b + 1], lens[b:b + 1].to(dev), ps, n)
            lat, rope = torch.randn(n, 512, generator=g).bfloat16().to(dev), torch.randn(n, 64, generator=g).bfloat16().to(dev)
            write_tokens(lat, rope, slots, cache.kv_cache, cache.kv_cache_sf)
    sl.copy_(lens)
    summarize_new_pages(cache.kv_cache, cache.kv_cache_sf, cache.summary, cache.summary_sf, bt, sl, 200)
    for i in range(24):
        if i == 5:
            pool.fork(bt, sl, torch.tensor([1], dtype=torch.int32, device=dev), torch.tensor([3], dtype=torch.int32, device=dev))
        if i == 12:
            pool.free(bt, sl, torch.tensor([0], dtype=torch.int32, device=dev))
        if i == 15:
            pool.compact(bt, sl)
        new = torch.where(sl > 0, sl + 1, sl)
        pool.allocate(bt, sl, new)
        sl.copy_(new)
        backend.prepare(bt, sl)
        q = torch.randn(rows, 1, H, 576, generator=g).to(E4M3).to(dev)
        lat, rope = torch.randn(rows, 512, generator=g).bfloat16().to(dev), torch.randn(rows, 64, generator=g).bfloat16().to(dev)
        if graph:
            step.q.copy_(q)
            step.latent.copy_(lat)
            step.rope.copy_(rope)
            out = step.replay()
        else:
            out = backend.forward(q, lat, rope, cache)
        if i in (0, 6, 11, 14, 16, 23):
            torch.cuda.synchronize()
            backend.wrapper.check_device_status()
            pool.check_status()
            for b, n in enumerate(sl.tolist()):  # every full page that a request has is summarised as it is
                for p in bt[b, : n // ps].tolist():
                    code, s = S.summarize(cache.kv_cache[p].cpu(), cache.kv_cache_sf[p].cpu())
                    assert torch.equal(cache.summary[p].cpu(), code) and float(cache.summary_sf[p]) == s, (i, b, p)
            ref, _ = _expected(cache, bt, sl, q, ps, budget, 1, 2, False, scale)
            O.assert_parity(out.float().cpu(), ref, f"step {i}")
    assert pool.num_free() == 140 - len({p for b, n in enumerate(sl.tolist()) for p in bt[b, : -(-n // ps)].tolist()})


def test_page_ids_are_validated_on_demand(monkeypatch):
    cache, bt, sl, q = _sparse_case([900, 700], 16, 16, 1, seed=6)
    w = _wrapper(num_heads=16, page_size=16, budget_pages=8)
    args = (q, cache.kv_cache, bt, sl, 900, 0.05)
    kw = dict(kv_cache_sf=cache.kv_cache_sf, summary=cache.summary, summary_sf=cache.summary_sf)
    want = w.run(*args, **kw)
    monkeypatch.setenv("MLA_FP4_VALIDATE", "1")
    assert torch.equal(w.run(*args, **kw), want)
    bt[1, 20] = cache.num_pages
    with pytest.raises(ValueError, match=r"block_tables\[1, 20\]"):
        w.run(*args, **kw)


def test_offsets_beyond_32_bits():
    """Pages at the far end of caches and summaries of more than 2^31 bytes."""
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import select_pages, summarize_pages

    pool, page, some = 3_900_000, 8, 300  # summaries of 2.2 GB
    far = 900_000  # pages of the cache: 2.3 GB
    kv, sf = _pages(some, page, 77)
    cache, scales = torch.zeros(far, page, 320, dtype=torch.uint8, device=dev), torch.zeros(far, page, 1, device=dev)
    cache[-some:], scales[-some:] = kv.to(dev), sf.to(dev)
    summary, ssf = torch.zeros(far, 576, dtype=torch.int8, device=dev), torch.zeros(far, device=dev)
    summarize_pages(cache, scales, summary, ssf, torch.arange(far - some, far, dtype=torch.int32, device=dev))
    codes, want_sf = _oracle_summaries(kv, sf)
    assert torch.equal(summary[-some:].cpu(), codes) and torch.equal(ssf[-some:].cpu(), want_sf)
    assert not bool(summary[:-some].any())
    big, big_sf = torch.zeros(pool, 576, dtype=torch.int8, device=dev), torch.zeros(pool, device=dev)
    big[-some:], big_sf[-some:] = summary[-some:], ssf[-some:]
    q = torch.randn(1, 1, 24, 576, generator=torch.Generator().manual_seed(1)).to(E4M3)
    order = torch.randperm(some, generator=torch.Generator().manual_seed(2)).int().view(1, -1)
    sl = torch.tensor([some * page], dtype=torch.int32)
    want, _ = S.select(q, codes, want_sf, order, sl, page, 30, 1, 2, False)
    got, _ = select_pages(q.to(dev), big, big_sf, (order + (pool - some)).int().to(dev), sl.to(dev), page, 30)
    assert torch.equal(got.cpu(), want + (pool - some))


def test_empty_batches_and_tables():
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import select_pages, summarize_new_pages

    cache, bt, sl, q = _sparse_case([900], 16, 16, 1, seed=6)
    sel, lens = select_pages(q[:0], cache.summary, cache.summary_sf, bt[:0], sl[:0], 16, 8)
    assert sel.shape == (0, 8) and lens.shape == (0,)
    sel, lens = select_pages(q, cache.summary, cache.summary_sf, bt[:, :0], sl, 16, 8)
    assert sel.tolist() == [[0] * 8] and lens.tolist() == [0]
    summarize_new_pages(cache.kv_cache, cache.kv_cache_sf, cache.summary, cache.summary_sf, bt[:, :0], sl, 5)
    summarize_new_pages(cache.kv_cache, cache.kv_cache_sf, cache.summary, cache.summary_sf, bt, sl, 0)
    torch.cuda.synchronize()


_FIRST = """
import sys, torch
sys.path.insert(0, {root!r})
sys.path.insert(0, {tests!r})
import test_gpu_sparse as T
from flashinfer_mla_fp4_b200 import FP4MLAPagedCache, FP4MLAPagePool
from flashinfer_mla_fp4_b200.sparse import select_pages, summarize_pages
dev = torch.device("cuda:0")
q, summary, ssf, bt, sl = (t.to(dev) for t in T._selection_case([3000, 2000], 24, 16, 1, seed=9))
kv, sf = T._pages(8200, 16, 3)
kv, sf = kv.to(dev), sf.to(dev)
kv64, sf64 = kv.view(-1, 64, 320), sf.view(-1, 64, 1)
out = [torch.zeros(n, 576, dtype=torch.int8, device=dev) for n in (8200, 2050, 2050)]
out_sf = [torch.zeros(n, device=dev) for n in (8200, 2050, 2050)]
ids, ids64 = torch.arange(8200, dtype=torch.int32, device=dev), torch.arange(2050, dtype=torch.int32, device=dev)
pool = FP4MLAPagePool([FP4MLAPagedCache(40, 16, dev)])
table, lens, ask = torch.zeros(2, 4, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), torch.tensor([40, 0], dtype=torch.int32, device=dev)
zero, one = torch.zeros(1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = select_pages(q, summary, ssf, bt, sl, 16, 20)
    summarize_pages(kv, sf, out[0], out_sf[0], ids)
    summarize_pages(kv64, sf64, out[1], out_sf[1], ids64)
    summarize_pages(kv64, sf64, out[2], out_sf[2], ids64[:64])
    pool.allocate(table, lens, ask)
    lens.copy_(ask)
    pool.fork(table, lens, zero, one)
    pool.free(table, lens, zero)
    pool.compact(table, lens)
graph.replay()
torch.cuda.synchronize()
again = select_pages(q, summary, ssf, bt, sl, 16, 20)
assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
assert torch.equal(out[1][:64], out[2][:64]) and bool(out[0].any())
assert lens.tolist() == [0, 40] and pool.refcounts.tolist()[:3] == [1, 1, 1] and pool.num_free() == 37
print("captured")
"""


def test_first_calls_of_a_process_under_capture():
    """No kernel has run before its first call is recorded."""
    _dev()
    import subprocess
    import sys
    from pathlib import Path

    here = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", _FIRST.format(root=str(here.parent), tests=str(here))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
