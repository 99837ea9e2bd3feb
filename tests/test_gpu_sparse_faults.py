"""Inputs at which sparse decode's kernels could go wrong although ordinary ones came out right: ties throughout, extreme scales, waits that run out."""
import pytest
import torch

from test_gpu_sparse import E4M3, _dev

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
