"""The page pool on the GPU against its oracle: tables, counts, lengths and every byte of every layer."""
import random

import pytest
import torch

from oracle import sparse_oracle as S

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def _caches(layers, pages, page, summaries, seed=0):
    from flashinfer_mla_fp4_b200 import FP4MLAPagedCache

    g = torch.Generator(device=_dev()).manual_seed(seed)
    out = []
    for _ in range(layers):
        c = FP4MLAPagedCache(pages, page, _dev(), summaries=summaries)
        c.kv_cache.random_(0, 256, generator=g)
        c.kv_cache_sf.uniform_(generator=g)
        if summaries:
            c.summary.random_(-127, 128, generator=g)
            c.summary_sf.uniform_(generator=g)
        out.append(c)
    return out


def _bytes(caches):
    return [[t.clone() for t in (c.kv_cache, c.kv_cache_sf, c.summary, c.summary_sf) if t is not None] for c in caches]


def _moved(before, moves):
    """The caches after all the copies at once."""
    out = [[t.clone() for t in layer] for layer in before]
    if moves:
        src, dst = (torch.tensor(x, device=_dev()) for x in zip(*moves))
        for a, b in zip(before, out):
            for s, d in zip(a, b):
                d[dst] = s[src]
    return out


def _check(pool, caches, before, want, bt, sl):
    torch.cuda.synchronize()
    assert pool.refcounts.tolist() == want.ref
    assert bt.tolist() == want.bt
    assert sl.tolist() == want.sl
    for got, exp in zip(_bytes(caches), _moved(before, want.moves)):
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, exp))
    if want.trouble:
        with pytest.raises((ValueError, RuntimeError), match="page pool"):
            pool.check_status()
    pool.check_status()
    want.moves, want.trouble = [], False


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=_dev())


@pytest.mark.parametrize("page,summaries", [(8, True), (16, False), (32, True), (64, False), (128, True)])
def test_copy_pages(page, summaries):
    from flashinfer_mla_fp4_b200.pages import copy_pages

    caches = _caches(3, 20, page, summaries)
    before = _bytes(caches)
    copy_pages(caches, _i32([0, 1, 1, -1, 5, 20, 9, 2]), _i32([10, 11, 12, 13, -1, 14, 25, 2]))  # a source twice, padding, outside, onto itself
    torch.cuda.synchronize()
    for got, exp in zip(_bytes(caches), _moved(before, [(0, 10), (1, 11), (1, 12)])):
        assert all(torch.equal(a, b) for a, b in zip(got, exp))
    copy_pages(caches, _i32([]), _i32([]))


def test_copy_pages_refuses(monkeypatch):
    from flashinfer_mla_fp4_b200.pages import FP4MLAPagePool, copy_pages

    caches = _caches(2, 8, 16, False)
    for src, dst in (([0, 1], [2]), ([0], torch.tensor([1]))):
        with pytest.raises(ValueError):
            copy_pages(caches, _i32(src), dst if isinstance(dst, torch.Tensor) else _i32(dst))
    with pytest.raises(ValueError, match="share"):
        copy_pages(caches + _caches(1, 9, 16, False), _i32([0]), _i32([1]))
    with pytest.raises(ValueError, match="twice"):
        FP4MLAPagePool([caches[0], caches[0]])
    monkeypatch.setenv("MLA_FP4_VALIDATE", "1")
    for src, dst in (([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(ValueError, match="named twice"):
            copy_pages(caches, _i32(src), _i32(dst))


def test_more_layers_than_a_launch_takes():
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool
    from flashinfer_mla_fp4_b200.pages import copy_pages

    caches = _caches(131, 12, 8, True)
    before = _bytes(caches)
    copy_pages(caches, _i32([0, 1]), _i32([10, 11]))
    exp = _moved(before, [(0, 10), (1, 11)])
    assert all(torch.equal(a, b) for g, e in zip(_bytes(caches), exp) for a, b in zip(g, e))
    pool = FP4MLAPagePool(caches)
    bt, sl = _i32([[3, 5, 0], [0, 0, 0]]), _i32([13, 0])
    pool.refcounts.copy_(_i32([0, 0, 0, 1, 0, 1, 0, 0, 0, 0, 0, 0]))
    before, want = _bytes(caches), S.Pool(pool.refcounts.tolist(), bt.tolist(), sl.tolist(), 8)
    pool.fork(bt, sl, _i32([0]), _i32([1]))
    want.fork([0], [1])
    _check(pool, caches, before, want, bt, sl)
    before = _bytes(caches)
    assert pool.compact(bt, sl).tolist() == want.compact()
    _check(pool, caches, before, want, bt, sl)


@pytest.mark.parametrize("seed,page,layers,pages,rows,width", [(1, 8, 1, 30, 5, 8), (6, 8, 1, 20001, 50, 900), (7, 8, 1, 8192, 20, 700), (2, 16, 2, 5000, 40, 200), (3, 64, 1, 300, 1100, 3),
                                                              (4, 128, 3, 64, 9, 12), (5, 32, 1, 9000, 2100, 6)])
def test_random_histories(seed, page, layers, pages, rows, width):
    """Allocations, forks, frees and compactions in any order, with lists that repeat rows, name none, and ask for too much."""
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    rng = random.Random(seed)
    caches = _caches(layers, pages, page, seed % 2 == 1, seed)
    pool = FP4MLAPagePool(caches)
    table = torch.zeros(rows, width + 3, dtype=torch.int32, device=_dev())
    bt, sl = table[:, 1:width + 1], torch.zeros(rows, dtype=torch.int32, device=_dev())
    want = S.Pool([0] * pages, bt.tolist(), sl.tolist(), page)
    for _ in range(14):
        before = _bytes(caches)
        kind = rng.choice(("allocate", "allocate", "fork", "fork", "free", "compact"))
        remap = None
        if kind == "allocate":
            new = [max(0, n + rng.choice((0, 1, page, -3, rng.randint(0, (width + 1) * page)))) if rng.random() < 0.5 else n for n in want.sl]
            pool.allocate(bt, sl, _i32(new))
            held = want.allocate(new)
            _check(pool, caches, before, want, bt, sl)
            sl.copy_(_i32(held))  # the program takes over the lengths of the rows that got their pages
            want.sl = held
            continue
        if kind == "fork":
            n = rng.randint(1, min(rows, 1500))
            parents = [rng.randint(-1, rows) for _ in range(n)]
            children = [rng.randint(-1, rows) for _ in range(n)]
            pool.fork(bt, sl, _i32(parents), _i32(children))
            want.fork(parents, children)
        elif kind == "free":
            some = [rng.randint(-1, rows) for _ in range(rng.randint(1, max(1, rows // 3)))]
            pool.free(bt, sl, _i32(some))
            want.free(some)
        else:
            remap = pool.compact(bt, sl).tolist()
            assert remap == want.compact()
        _check(pool, caches, before, want, bt, sl)


@pytest.mark.parametrize("pages", [1, 8, 9, 8191, 8192, 8193])
@pytest.mark.parametrize("use", ["all", "none", "the first", "the last", "all but the first"])
def test_compaction_at_the_ends(pages, use):
    """Pools of about what a planning CTA looks at in a round, with a list of new numbers that starts anywhere."""
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    caches = _caches(1, pages, 8, False)
    pool = FP4MLAPagePool(caches)
    used = {"all": range(pages), "none": (), "the first": (0,), "the last": (pages - 1,), "all but the first": range(1, pages)}[use]
    pool.refcounts[list(used)] = 3
    bt, sl = torch.zeros(1, 2, dtype=torch.int32, device=_dev()), _i32([0])
    want, before = S.Pool(pool.refcounts.tolist(), bt.tolist(), sl.tolist(), 8), _bytes(caches)
    remap = torch.full((pages + 2,), -9, dtype=torch.int32, device=_dev())
    assert pool.compact(bt, sl, remap[1:-1]).tolist() == want.compact()
    assert int(remap[0]) == -9 and int(remap[-1]) == -9
    _check(pool, caches, before, want, bt, sl)


def test_a_pool_that_runs_out():
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    caches = _caches(1, 6, 8, False)
    pool = FP4MLAPagePool(caches)
    bt, sl = torch.full((4, 4), -5, dtype=torch.int32, device=_dev()), _i32([0, 0, 0, 0])
    pool.allocate(bt, sl, _i32([17, 40, 16, 2]))  # 3 pages, more than its row holds, 2, 1
    assert bt.tolist() == [[0, 1, 2, -5], [-5] * 4, [3, 4, -5, -5], [5, -5, -5, -5]]
    with pytest.raises(ValueError, match="entry 1"):
        pool.check_status()
    sl.copy_(_i32([17, 0, 16, 2]))
    pool.fork(bt, sl, _i32([2, 0]), _i32([1, 1]))  # shares two full pages; the second names the child again
    assert sl.tolist() == [17, 16, 16, 2] and bt[1].tolist() == [3, 4, -5, -5] and pool.refcounts.tolist() == [1, 1, 1, 2, 2, 1]
    with pytest.raises(ValueError, match="entry 1"):
        pool.check_status()
    pool.free(bt, sl, _i32([1, 1, -1]))
    assert pool.refcounts.tolist() == [1] * 6 and sl.tolist() == [17, 0, 16, 2]
    pool.fork(bt, sl, _i32([0]), _i32([1]))  # no page for the tail: nothing is done
    assert pool.refcounts.tolist() == [1] * 6 and sl.tolist() == [17, 0, 16, 2]
    with pytest.raises(RuntimeError, match="no page"):
        pool.check_status()
    assert pool.num_free() == 0
    pool.allocate(bt, sl, _i32([17, 2**31 - 1, 17, 2]))
    assert sl.tolist() == [17, 0, 16, 2] and pool.refcounts.tolist() == [1] * 6
    with pytest.raises((RuntimeError, ValueError)):
        pool.check_status()


def test_captured_forks_and_compactions_replay():
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    caches = _caches(2, 40, 16, True)
    pool = FP4MLAPagePool(caches)
    bt, sl = torch.zeros(6, 8, dtype=torch.int32, device=_dev()), _i32([0] * 6)
    parents, children, gone = _i32([0, 0, -1]), _i32([3, 4, 5]), _i32([0, 3])
    remap = torch.empty(40, dtype=torch.int32, device=_dev())

    def work():
        pool.fork(bt, sl, parents, children)
        pool.free(bt, sl, gone)
        pool.compact(bt, sl, remap)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    pool.check_status()
    for n in (50, 33, 128):
        pool.refcounts.zero_()
        bt.zero_()
        sl.zero_()
        new = _i32([n, 20, 7, 0, 0, 0])
        pool.allocate(bt, sl, new)
        sl.copy_(new)
        before, want = _bytes(caches), S.Pool(pool.refcounts.tolist(), bt.tolist(), sl.tolist(), 16)
        graph.replay()
        want.fork([0, 0, -1], [3, 4, 5])
        want.free([0, 3])
        first, want.moves = want.moves, []
        middle = _moved(before, first)
        assert remap.tolist() == want.compact()
        _check(pool, caches, middle, want, bt, sl)


def test_pool_refuses():
    from flashinfer_mla_fp4_b200 import FP4MLAPagePool

    pool = FP4MLAPagePool(_caches(1, 8, 16, False))
    bt, sl = torch.zeros(2, 4, dtype=torch.int32, device=_dev()), _i32([0, 0])
    for call in (lambda: pool.allocate(bt, sl, _i32([1])), lambda: pool.allocate(bt, sl, _i32([1, 1]).long()), lambda: pool.allocate(bt.long(), sl, sl),
                 lambda: pool.allocate(bt, sl[:1], sl), lambda: pool.allocate(bt.t(), _i32([0] * 4), _i32([0] * 4)),
                 lambda: pool.fork(bt, sl, _i32([0]), _i32([0, 1])), lambda: pool.fork(bt, sl, [0], [1]), lambda: pool.free(bt, sl, torch.tensor([0])),
                 lambda: pool.free(bt.cpu(), sl, _i32([0])), lambda: pool.free(bt[:1].expand(2, 4), sl, _i32([0])),
                 lambda: pool.compact(bt, sl, torch.empty(7, dtype=torch.int32, device=_dev()))):
        with pytest.raises(ValueError):
            call()
    for wrong in (torch.zeros(9, dtype=torch.int32, device=_dev()), torch.zeros(7, dtype=torch.int32, device=_dev()), torch.zeros(8, device=_dev())):
        pool.refcounts = wrong
        with pytest.raises(ValueError, match="refcounts"):
            pool.allocate(bt, sl, _i32([1, 1]))
