"""Sparse decode and the page pool where they could go wrong: what needs no GPU."""
import numpy as np
import pytest
import torch

from oracle import sparse_oracle as S

E4M3 = torch.float8_e4m3fn


def test_ties_of_the_oracle():
    """Where all pages tie the first ones are taken, whatever it is that they share."""
    summary, ssf, bt = torch.ones(300, 576, dtype=torch.int8), torch.ones(300), torch.arange(299, -1, -1).int().view(1, -1)
    for q, scale in ((torch.zeros(1, 1, 2, 576), ssf), (torch.randn(1, 1, 2, 576), ssf * float("nan"))):
        got, lens = S.select(q.to(E4M3), summary, scale, bt, torch.tensor([2397]), 8, 40, 1, 2, False)
        assert got.tolist() == [bt[0, :38].tolist() + bt[0, -2:].tolist()] and lens.tolist() == [317]


def test_oracle_allocation_from_a_pool_that_is_short():
    p = S.Pool([0, 0, 1, 0, 0, 0], [[-1] * 9 for _ in range(5)], [0] * 5, 8)
    assert p.allocate([64, 8, 16, 32, 16]) == [0, 8, 16, 0, 16] and p.trouble
    assert [r[:2] for r in p.bt] == [[-1, -1], [0, -1], [1, 3], [-1, -1], [4, 5]] and p.ref == [1] * 6


@pytest.mark.parametrize("causal", [np.array([1, 2]), torch.tensor([1, 2])])
def test_a_causal_that_is_neither_true_nor_false_is_no_internal_error(causal):
    """The native call must not return with Python's error of that value still set."""
    from flashinfer_mla_fp4_b200.sparse import select_pages

    q, summary, ssf = torch.zeros(1, 1, 8, 576).to(E4M3), torch.zeros(4, 576, dtype=torch.int8), torch.zeros(4)
    bt, sl = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):  # (what is wrong with these tensors otherwise)
        select_pages(q, summary, ssf, bt, sl, 16, 4, causal=causal)


def test_counts_beyond_32_bits_are_refused():
    """They would be cut to their low bits on their way to the kernels: a budget of 2^32 + 8 would be one of 8."""
    from flashinfer_mla_fp4_b200 import SparsePages
    from flashinfer_mla_fp4_b200.sparse import check_tables

    assert SparsePages(2**31 - 1).budget_pages == 2**31 - 1
    for budget in (2**31, 2**32 + 8):
        with pytest.raises(ValueError, match="2\\^31"):
            SparsePages(budget)
    for shape in ((1, 2**31), (2**31, 1)):
        with pytest.raises(ValueError, match="2\\^31"):
            check_tables(torch.empty(shape, dtype=torch.int32, device="meta"), None, torch.device("cuda:0"))
