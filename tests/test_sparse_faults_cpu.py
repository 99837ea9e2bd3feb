"""Sparse decode and the page pool where they could go wrong: what needs no GPU."""
import torch

from oracle import sparse_oracle as S

E4M3 = torch.float8_e4m3fn


def test_ties_of_the_oracle():
    """Where all pages tie the first ones are taken, whatever it is that they share."""
    summary, ssf, bt = torch.ones(300, 576, dtype=torch.int8), torch.ones(300), torch.arange(299, -1, -1).int().view(1, -1)
    for q, scale in ((torch.zeros(1, 1, 2, 576), ssf), (torch.randn(1, 1, 2, 576), ssf * float("nan"))):
        got, lens = S.select(q.to(E4M3), summary, scale, bt, torch.tensor([2397]), 8, 40, 1, 2, False)
        assert got.tolist() == [bt[0, :38].tolist() + bt[0, -2:].tolist()] and lens.tolist() == [317]
