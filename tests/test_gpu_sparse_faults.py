"""Inputs at which sparse decode's kernels could go wrong although ordinary ones came out right: ties throughout, extreme scales, waits that run out."""
import ctypes as C

import pytest
import torch

from oracle import mla_fp4_oracle as O
from test_gpu_sparse import E4M3, _dev, _oracle_summaries, _pages, _same, _selection_case, _sparse_case, _wrapper

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages,rows", [(140, 400), (140, 1), (900, 300), (1900, 64), (4000, 150), (4000, 1), (12000, 40), (17000, 20)])
@pytest.mark.parametrize("of", ["zero queries", "NaN scores", "pages outside the pool"])
def test_rows_of_pages_that_all_tie(pages, rows, of):
    """More than 128 candidates with one key: the first ones, in every row and every time, and nothing behind a row's places.  A warp that leaves the
    search for the range late must not meet the counts of the scan behind it, so rows start together and on a cold instruction cache too."""
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import select_pages

    budget, sink, local = 40, 1, 2
    g = torch.Generator().manual_seed(pages)
    summary, ssf = torch.randint(-127, 128, (pages, 576), generator=g, dtype=torch.int8).to(dev), torch.ones(pages, device=dev)
    q = torch.randn(rows, 1, 4, 576, generator=g)
    bt = torch.randperm(pages, generator=g).int().repeat(rows, 1)
    if of == "zero queries":
        q.zero_()
    elif of == "NaN scores":
        ssf.fill_(float("nan"))
    else:
        bt += pages
    sl = torch.full((rows,), pages * 8 - 3, dtype=torch.int32)
    want = torch.cat((bt[:, :budget - local], bt[:, -local:]), 1).to(dev)  # (the sink and the first of the rest are the first pages)
    qd, btd, sld = q.to(E4M3).to(dev), bt.to(dev), sl.to(dev)
    cold = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    for i in range(12):
        room = torch.full((rows + 60, budget), -9, dtype=torch.int32, device=dev)
        if i % 3 == 0:
            cold.fill_(i)
        got, lens = select_pages(qd, summary, ssf, btd, sld, 8, budget, sink_pages=sink, local_pages=local, selected=room[:rows])
        assert torch.equal(got, want) and bool((room[rows:] == -9).all())
        assert bool((lens == budget * 8 - 3).all())


class _Slow:
    """A selection of 124 rows of 2048 pages, 128 heads, from inputs that are not in L2: with a poll budget of one a wait runs out for certain."""

    def __init__(self):
        from flashinfer_mla_fp4_b200 import _cabi
        from flashinfer_mla_fp4_b200.sparse import select_pages

        dev, rows, pages, budget = _dev(), 124, 2048, 64
        self.inputs = q, summary, ssf, bt, sl = [t.to(dev) for t in _selection_case([pages * 64] * rows, 128, 64, 1, seed=4)]
        self.bt, self.want = bt, select_pages(q, summary, ssf, bt, sl, 64, budget)
        self.sel, self.lens = (torch.empty_like(t) for t in self.want)
        self.ws = torch.zeros(_cabi.select_workspace_bytes(rows, 1, pages), dtype=torch.int8, device=dev)
        self.status, self.cold = torch.zeros(8, dtype=torch.int32, device=dev), torch.empty(300 << 20, dtype=torch.uint8, device=dev)
        a = self.args = _cabi.SelectArgs()
        a.q, a.q_stride_batch, a.q_stride_qpos, a.q_stride_head = q.data_ptr(), q.stride(0), q.stride(1), q.stride(2)
        a.summary, a.summary_sf, a.num_pages = summary.data_ptr(), ssf.data_ptr(), summary.shape[0]
        a.block_tables, a.block_table_stride, a.seq_lens = bt.data_ptr(), bt.stride(0), sl.data_ptr()
        a.selected, a.selected_lens, a.workspace, a.workspace_bytes = self.sel.data_ptr(), self.lens.data_ptr(), self.ws.data_ptr(), self.ws.numel()
        a.batch, a.q_len, a.num_heads, a.page_size, a.width = rows, 1, 128, 64, pages
        a.budget, a.sink_pages, a.local_pages, a.status = budget, 1, 2, self.status.data_ptr()
        a.stream = torch.cuda.current_stream().cuda_stream

    def run(self, polls, status=(0,) * 8):
        """The status words after a call with that poll budget."""
        from flashinfer_mla_fp4_b200 import _cabi

        self.status.copy_(torch.tensor(status, dtype=torch.int32))
        self.cold.fill_(polls)
        self.args.wait_polls = polls
        _cabi.check(_cabi.lib.mla_fp4_select_pages(C.byref(self.args)))
        torch.cuda.synchronize()
        return self.status.tolist()


def test_a_wait_that_runs_out_for_certain():
    """The status says so, the kernel ends, what is selected are pages of the request, and the next call is right."""
    slow = _Slow()
    from flashinfer_mla_fp4_b200 import _cabi

    for _ in range(3):
        code, _, cta, thread, parity = slow.run(1)[:5]
        assert code == _cabi.ERR_DEVICE_TIMEOUT and 0 <= cta < 148 and thread % 32 == 0 and parity in (0, 1)  # one warp's record
        assert torch.equal(slow.lens, slow.want[1])
        assert bool((slow.sel.unsqueeze(2) == slow.bt.unsqueeze(1)).any(2).all())
        assert slow.run(0)[0] == 0 and torch.equal(slow.sel, slow.want[0]) and torch.equal(slow.lens, slow.want[1])


def test_the_first_record_of_a_wait_that_ran_out_stays():
    """A status that nobody has looked at yet keeps what it says, as with the decode kernel, whose status words sparse decode shares."""
    slow, before = _Slow(), [5, 1, 2, 3, 4, 9, 9, 9]
    assert slow.run(1, before) == before


_BOUND = ("mla_fp4_summarize_pages", "mla_fp4_summarize_new_pages", "mla_fp4_select_workspace_bytes", "mla_fp4_select_pages",
          "mla_fp4_pool_workspace_bytes", "mla_fp4_pool_allocate", "mla_fp4_pool_fork", "mla_fp4_pool_free", "mla_fp4_pool_compact")


@pytest.fixture
def one_poll(monkeypatch):
    """Selections with a poll budget of one, whichever way the library is called."""
    from flashinfer_mla_fp4_b200 import _cabi

    _dev()
    real = _cabi.lib.mla_fp4_select_pages

    def with_one_poll(args):
        a = args.contents if hasattr(args, "contents") else args._obj
        a.wait_polls = 1
        return real(C.byref(a))

    stand_in = C.CFUNCTYPE(C.c_int, C.POINTER(_cabi.SelectArgs))(with_one_poll)
    addresses = {n: C.cast(getattr(_cabi.lib, n), C.c_void_p).value for n in _BOUND}
    monkeypatch.setattr(_cabi.lib, "mla_fp4_select_pages", with_one_poll)
    _cabi.native.bind_sparse(*{**addresses, "mla_fp4_select_pages": C.cast(stand_in, C.c_void_p).value}.values())
    yield
    _cabi.native.bind_sparse(*addresses.values())


class _Decline:
    """A native call path that leaves every call to the Python one."""

    def __getattr__(self, name):
        return lambda *args: False if name == "summarize" else None


@pytest.mark.parametrize("native", [True, False])
def test_select_pages_reports_a_wait_that_ran_out(native, monkeypatch, request):
    slow = _Slow()  # (before the poll budget is cut)
    request.getfixturevalue("one_poll")
    from flashinfer_mla_fp4_b200 import _cabi, sparse

    if not native:
        monkeypatch.setattr(sparse, "_native", _Decline())
    slow.cold.fill_(1)
    got, lens = sparse.select_pages(*slow.inputs, 64, 64, status=slow.status)
    torch.cuda.synchronize()
    assert int(slow.status[0]) == _cabi.ERR_DEVICE_TIMEOUT and torch.equal(lens, slow.want[1])
    for wrong in (slow.status[:7], slow.status.long(), slow.status.cpu(), torch.zeros(16, dtype=torch.int32, device=slow.bt.device)[::2]):
        with pytest.raises(ValueError, match="status"):
            sparse.select_pages(*slow.inputs, 64, 64, status=wrong)


@pytest.mark.parametrize("validate", ["0", "1"])
def test_a_sparse_step_reports_a_wait_of_its_selection(validate, monkeypatch, request):
    """Also when the page ids are checked on the host first, which the native call leaves to the Python one."""
    slow = _Slow()
    request.getfixturevalue("one_poll")
    from flashinfer_mla_fp4_b200 import BatchMLASparseDecodeFP4Wrapper

    monkeypatch.setenv("MLA_FP4_VALIDATE", validate)
    q, summary, ssf, bt, sl = slow.inputs
    dev, pages = q.device, summary.shape[0]
    kv, sf = torch.zeros(pages, 64, 320, dtype=torch.uint8, device=dev), torch.ones(pages, 64, 1, device=dev)
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    w = BatchMLASparseDecodeFP4Wrapper(torch.empty(BatchMLASparseDecodeFP4Wrapper.workspace_bytes(124, 1, 128, 2048, 64, sms), dtype=torch.int8, device=dev))
    w.plan(num_heads=128, page_size=64, budget_pages=64)
    slow.cold.fill_(1)
    w.run(q, kv, bt, sl, 2048 * 64, 0.04, kv_cache_sf=sf, summary=summary, summary_sf=ssf)
    with pytest.raises(RuntimeError):
        w.check_device_status()


def test_a_causal_that_is_neither_true_nor_false_is_refused():
    _dev()
    from flashinfer_mla_fp4_b200.sparse import select_pages

    args = [t.cuda() for t in _selection_case([700], 8, 16, 1, seed=2)]
    with pytest.raises((ValueError, RuntimeError), match="ambiguous"):
        select_pages(*args, 16, 8, causal=torch.tensor([True, False]))


def test_more_requests_than_a_plan_holds_whose_lengths_come_and_go():
    """Lengths that the kernel ahead of the decode writes in every step, from tokens to none and back: a plan must not be made from both."""
    cache, _, _, _ = _sparse_case([64], 8, 8, 1, seed=2)
    dev, rows = cache.kv_cache.device, 20600
    bt = (torch.arange(rows, device=dev) % 8).int().view(rows, 1).repeat(1, 2).contiguous()
    q = torch.randn(1, 1, 8, 576, generator=torch.Generator().manual_seed(3)).to(E4M3).to(dev).expand(rows, 1, 8, 576)
    w = _wrapper(num_heads=8, page_size=8, budget_pages=3)
    some = torch.zeros(rows, dtype=torch.int32, device=dev)
    some[20500:] = 5
    every, none, sl = torch.full_like(some, 5), torch.zeros_like(some), torch.zeros_like(some)
    want = None
    for i in range(60):
        lens = (every, none, some, none)[i % 4]
        sl.copy_(lens)
        out = w.run(q, cache.kv_cache, bt, sl, 16, 0.05, kv_cache_sf=cache.kv_cache_sf, summary=cache.summary, summary_sf=cache.summary_sf)
        want = out.clone() if want is None else want
        assert torch.equal(out, torch.where((lens > 0).view(rows, 1, 1, 1), want, torch.zeros_like(want)))
    w.check_device_status()
    ref, _ = O.mla_decode(q[:8].cpu(), cache.kv_cache, cache.kv_cache_sf, bt[:8].cpu(), every[:8].cpu(), 0.05)
    O.assert_parity(want[:8].float().cpu(), ref, "the first requests")
    assert torch.equal(want, want[:8].repeat(rows // 8, 1, 1, 1))


def _one_sided_pages(page):
    """Pages one part of whose summary is nothing beside the other: the factor that takes a sum to a code is beyond FP32 where the sums are all zero."""
    kv, sf = _pages(12, page, page + 7)
    kv[:6, :, :256] = 0
    kv[:6, :, 256:] = 0x30  # RoPE 0.5 throughout, latent zero under huge scales
    for i, scale in enumerate((1e30, 1e37, 3e38, -3e38)):
        sf[i] = scale
    kv[4, 0, 3], sf[4] = 0x21, 1e37  # ... one latent value that is not
    sf[5] = 0.0
    kv[6:, :, 256:] = 0  # RoPE zero, scales whose means are subnormal
    for i, scale in enumerate((1e-41, 3e-42, 1e-39, -1e-41)):
        sf[6 + i] = scale
    kv[6:10, 0, :256] = 0x77  # (a mean that does not round to zero)
    kv[10, :, 256], kv[10, :, 257], sf[10] = 0x01, 0x81, 1e-41  # RoPE values of 2^-9: beside them the latent is nothing
    return kv, sf


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128])
def test_summaries_of_pages_with_one_empty_part(page):
    dev = _dev()
    from flashinfer_mla_fp4_b200.sparse import summarize_pages

    kv, sf = _one_sided_pages(page)
    want, want_sf = _oracle_summaries(kv, sf)
    assert not want[:4, :512].any() and not want[6:10, 512:].any() and bool((want_sf[6:10] > 0).all())
    for copies in (1, 140000 // (12 * page) + 1):  # a few pages, and enough for the tensor cores
        kvd, sfd, n = kv.repeat(copies, 1, 1).to(dev), sf.repeat(copies, 1, 1).to(dev), 12 * copies
        summary, ssf = torch.full((n, 576), 9, dtype=torch.int8, device=dev), torch.full((n,), 9.0, device=dev)
        summarize_pages(kvd, sfd, summary, ssf, torch.arange(n, dtype=torch.int32, device=dev))
        for i in range(12):
            assert torch.equal(summary.view(copies, 12, 576)[:, i].cpu(), want[i].expand(copies, -1)), (copies, i)
        assert _same(ssf.cpu(), want_sf.repeat(copies))
