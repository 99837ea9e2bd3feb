"""The page pool where it runs short."""
import random

import pytest
import torch

from oracle import sparse_oracle as S
from test_gpu_pages import _bytes, _caches, _check, _dev, _i32

pytestmark = pytest.mark.gpu


def test_a_row_that_does_not_fit_takes_nothing_from_those_behind_it():
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    pool = FP4MLAPagePool(_caches(1, 6, 8, False))
    pool.refcounts[2] = 1
    bt, sl = torch.full((5, 9), -5, dtype=torch.int32, device=_dev()), _i32([0] * 5)
    pool.allocate(bt, sl, _i32([64, 8, 16, 32, 16]))  # 8 pages, 1, 2, 4, 2, of which 5 are free
    assert [row[:2] for row in bt.tolist()] == [[-5, -5], [0, -5], [1, 3], [-5, -5], [4, 5]]
    assert pool.refcounts.tolist() == [1] * 6
    with pytest.raises(RuntimeError, match="entry [03]"):
        pool.check_status()


@pytest.mark.parametrize("seed,pages,rows,width", [(1, 40, 31, 12), (2, 40, 33, 12), (3, 500, 70, 30), (4, 9000, 1500, 30), (5, 20, 1025, 3), (6, 8192, 2, 9000), (7, 300, 2500, 300),
                                                   (8, 17000, 4000, 9), (10, 8192, 6, 9000)])
def test_allocation_from_a_pool_that_is_short(seed, pages, rows, width):
    """Rows of a few pages among rows of more than there are left (seed 6: none is refused), twice in a row; the second time some have pages already."""
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    rng = random.Random(seed)
    caches = _caches(1, pages, 8, False)
    pool = FP4MLAPagePool(caches)
    pool.refcounts.copy_(_i32([int(rng.random() < 0.2) for _ in range(pages)]))
    bt, sl = torch.zeros(rows, width, dtype=torch.int32, device=_dev()), torch.zeros(rows, dtype=torch.int32, device=_dev())
    want = S.Pool(pool.refcounts.tolist(), bt.tolist(), sl.tolist(), 8)
    for _ in range(2):
        before = _bytes(caches)
        new = [n + rng.choice((0, 3, 8 * rng.randint(1, 4), 8 * rng.randint(1, width + 1))) for n in want.sl]
        pool.allocate(bt, sl, _i32(new))
        held = want.allocate(new)
        _check(pool, caches, before, want, bt, sl)
        sl.copy_(_i32(held))
        want.sl = held


@pytest.mark.parametrize("rows,width", [(3000, 4), (2100, 2**20)])
def test_rows_that_ask_for_far_too_much(rows, width):
    """More than their table rows hold, or more in all than 32 bits do: the few rows among them that fit are served."""
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    pool = FP4MLAPagePool(_caches(1, 50, 8, False))
    bt, sl = torch.full((rows, width), -5, dtype=torch.int32, device=_dev()), torch.zeros(rows, dtype=torch.int32, device=_dev())
    new = torch.full_like(sl, 8 * width if width > 4 else 2**31 - 1)
    some = [1, 33, rows - 1]
    new[some] = 16
    pool.allocate(bt, sl, new)
    assert bt[some, :2].tolist() == [[0, 1], [2, 3], [4, 5]] and pool.num_free() == 44 and int((bt != -5).sum()) == 6
    with pytest.raises((RuntimeError, ValueError), match="page pool"):
        pool.check_status()
