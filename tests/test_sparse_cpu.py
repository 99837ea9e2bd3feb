"""What sparse decode and the page pool refuse, and their oracle against small cases worked out by hand: no GPU is needed."""
import ctypes as C

import pytest
import torch

from oracle import sparse_oracle as S

E4M3 = torch.float8_e4m3fn


def test_sparse_pages_are_checked():
    from flashinfer_mla_fp4_b200 import SparsePages

    assert SparsePages(3, 1, 2).budget_pages == 3
    for bad in ((2, 1, 2), (4, -1, 2), (4, 0, 0)):
        with pytest.raises(ValueError, match="local_pages"):
            SparsePages(*bad)


def test_host_tensors_and_wrong_forms_are_refused():
    from flashinfer_mla_fp4_b200 import FP4MLAPagedCache
    from flashinfer_mla_fp4_b200.pages import FP4MLAPagePool, copy_pages
    from flashinfer_mla_fp4_b200.sparse import select_pages, summarize_new_pages, summarize_pages

    kv, sf = torch.zeros(4, 16, 320, dtype=torch.uint8), torch.zeros(4, 16, 1)
    summary, ssf, ids = torch.zeros(4, 576, dtype=torch.int8), torch.zeros(4), torch.zeros(2, dtype=torch.int32)
    bt, sl = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        summarize_pages(kv, sf, summary, ssf, ids)
    with pytest.raises(ValueError, match="CUDA"):
        summarize_new_pages(kv, sf, summary, ssf, bt, sl, 1)
    with pytest.raises(ValueError, match="page_size"):
        summarize_pages(torch.zeros(4, 24, 320, dtype=torch.uint8), sf, summary, ssf, ids)
    with pytest.raises(ValueError, match="E4M3"):
        select_pages(torch.zeros(1, 1, 8, 576), summary, ssf, bt, sl, 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        select_pages(torch.zeros(1, 1, 8, 576).to(E4M3), summary, ssf, bt, sl, 16, 4)
    cache = FP4MLAPagedCache(4, 16, "cpu", summaries=True)
    assert cache.bytes() == 4 * (16 * 324 + 580)
    with pytest.raises(ValueError, match="CUDA"):
        FP4MLAPagePool([cache])
    with pytest.raises(ValueError, match="at least one"):
        copy_pages([], ids, ids)
    with pytest.raises(ValueError, match="belong together"):
        FP4MLAPagedCache.from_tensors(kv, sf, summary)
    with pytest.raises(ValueError, match="kv_cache_sf"):
        FP4MLAPagedCache.from_tensors(kv, torch.zeros(4, 16))
    same = FP4MLAPagedCache.from_tensors(kv, sf, summary, ssf)
    assert same.kv_cache is kv and same.num_pages == 4 and same.page_size == 16
    assert FP4MLAPagedCache(4, 16, "cpu").summary is None


def test_abi_refuses_before_any_launch():
    from flashinfer_mla_fp4_b200 import _cabi

    lib, bad, P = _cabi.lib, _cabi.ERR_BAD_ARG, 4096  # an address that is looked at as a number only
    assert lib.mla_fp4_select_pages(None) == bad
    assert _cabi.select_workspace_bytes(3, 2, 98) == 3 * 2 * 100 * 4
    n = C.c_size_t(0)
    assert lib.mla_fp4_select_workspace_bytes(3, 0, 100, C.byref(n)) == bad

    def args_of(**kw):
        a = _cabi.SelectArgs()
        base = dict(q=P, q_stride_batch=576 * 8, q_stride_qpos=576 * 8, q_stride_head=576, summary=P, summary_sf=P, num_pages=9,
                    block_tables=P, block_table_stride=8, seq_lens=P, selected=P, selected_lens=P, workspace=P, workspace_bytes=32,
                    batch=1, q_len=1, num_heads=8, page_size=64, width=8, budget=4, sink_pages=1, local_pages=2)
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return lib.mla_fp4_select_pages(C.byref(a))

    for kw, code in ((dict(num_heads=129), _cabi.ERR_UNSUPPORTED), (dict(page_size=24), _cabi.ERR_UNSUPPORTED), (dict(num_heads=0), bad),
                     (dict(sink_pages=-1), bad), (dict(local_pages=0), bad), (dict(sink_pages=3), bad), (dict(q=None), bad),
                     (dict(selected=None), bad), (dict(num_pages=0), bad), (dict(q=P + 8), bad), (dict(q_stride_head=580), bad),
                     (dict(summary=P + 4), bad), (dict(workspace_bytes=31), _cabi.ERR_WORKSPACE_TOO_SMALL),
                     (dict(workspace=None), _cabi.ERR_WORKSPACE_TOO_SMALL), (dict(batch=0), _cabi.OK)):
        assert args_of(**kw) == code, (kw, _cabi.last_error())
    assert lib.mla_fp4_summarize_pages(P, P, 4, 24, P, 1, P, P, None, None) == _cabi.ERR_UNSUPPORTED
    assert lib.mla_fp4_summarize_pages(P, P, 0, 16, P, 1, P, P, None, None) == bad
    assert lib.mla_fp4_summarize_pages(P + 4, P, 4, 16, P, 1, P, P, None, None) == bad
    assert lib.mla_fp4_summarize_pages(P, P, 4, 16, None, 1, P, P, None, None) == bad
    assert lib.mla_fp4_summarize_pages(P, P, 4, 16, None, 0, P, P, None, None) == _cabi.OK
    assert lib.mla_fp4_summarize_new_pages(P, P, 4, 16, P, 4, 4, P, 1, -1, P, P, None, None) == bad
    assert lib.mla_fp4_summarize_new_pages(P, P, 4, 16, None, 4, 4, P, 1, 1, P, P, None, None) == bad
    assert lib.mla_fp4_summarize_new_pages(P, P, 4, 16, P, 4, 4, P, 0, 1, P, P, None, None) == _cabi.OK
    layer = (_cabi.PageLayer * 1)()
    layer[0].kv_cache, layer[0].kv_cache_sf = P, P
    assert lib.mla_fp4_copy_pages(layer, 0, 4, 16, P, P, 1, None) == bad
    assert lib.mla_fp4_copy_pages(layer, 1, 4, 16, P, P, -1, None) == bad
    assert lib.mla_fp4_copy_pages(layer, 1, 4, 16, None, P, 1, None) == bad
    assert lib.mla_fp4_copy_pages(layer, 1, 4, 16, None, None, 0, None) == _cabi.OK
    layer[0].summary = P
    assert lib.mla_fp4_copy_pages(layer, 1, 4, 16, P, P, 1, None) == bad  # a summary without its scale
    layer[0].summary = None
    a = _cabi.PoolArgs()
    a.layers, a.num_layers, a.page_size, a.num_pages = layer, 1, 16, 4
    a.refcounts, a.block_tables, a.block_table_stride, a.width, a.rows, a.seq_lens = P, P, 4, 4, 2, P
    a.workspace, a.workspace_bytes = P, _cabi.pool_workspace_bytes(4, 2, 0)
    assert lib.mla_fp4_pool_allocate(C.byref(a), None) == bad
    assert lib.mla_fp4_pool_compact(C.byref(a), None) == bad
    assert lib.mla_fp4_pool_fork(C.byref(a), P, P, 1) == _cabi.ERR_WORKSPACE_TOO_SMALL
    assert lib.mla_fp4_pool_fork(C.byref(a), None, None, 0) == _cabi.OK
    assert lib.mla_fp4_pool_free(C.byref(a), None, 0) == _cabi.OK
    a.refcounts = None
    assert lib.mla_fp4_pool_free(C.byref(a), P, 1) == bad
    assert lib.mla_fp4_pool_free(None, P, 1) == bad


def test_oracle_summary_by_hand():
    kv, sf = torch.zeros(8, 320, dtype=torch.uint8), torch.ones(8, 1)
    kv[:, 0] = 0x7  # element 0: 6.0, element 1: 0
    kv[0, 1] = 0xA0  # element 3 of token 0: -1.0
    kv[3, 256] = 0x38  # RoPE 0 of token 3: 1.0
    code, scale = S.summarize(kv, sf)
    assert scale == pytest.approx(6 / 127, rel=1e-6)
    assert code[0] == 127 and code[1] == 0 and code[3] == round(-0.125 / (6 / 127)) and code[512] == round(0.125 / (6 / 127))
    sf[2] = float("inf")
    assert S.summarize(kv, sf)[1] != S.summarize(kv, sf)[1]


def test_oracle_query_codes_keep_the_large_values():
    q = torch.zeros(2, 576)
    q[0, :4] = torch.tensor([448.0, -256.0, 4.0, 3.5])  # binade of 256: unit 4
    q[1, 0] = 2.0 ** -9
    codes, units = S.query_codes(q.to(E4M3))
    assert codes[0, :4].tolist() == [112, -64, 1, 1] and units[0] == 4
    assert codes[1, 0] == 8 and units[1] == 2.0 ** -12


def test_oracle_pool_by_hand():
    p = S.Pool([1, 1, 0, 0, 1, 0], [[0, 4, 1], [0, 0, 0], [0, 0, 0]], [10, 0, 0], 4)
    p.fork([0, 0], [1, 2])
    assert p.bt == [[0, 4, 1], [0, 4, 2], [0, 4, 3]] and p.ref == [3, 1, 1, 1, 3, 0] and p.moves == [(1, 2), (1, 3)]
    p.free([0])
    assert p.ref == [2, 0, 1, 1, 2, 0] and p.sl == [0, 10, 10]
    assert p.compact() == [0, -1, 2, 3, 1, -1] and p.bt[1] == [0, 1, 2] and p.ref == [2, 2, 1, 1, 0, 0]
