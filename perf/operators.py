"""Sparse FP4 MLA decode over pages that a cheap score selects, and the care of the pages it reads: what is measured, and its plain forms.

Five operators, told apart by ``kind``:

* ``summary``  the 8-bit mean key of full pages of a paged cache, by page ids or of the pages that a step's new tokens have filled;
* ``select``   for each query the pages whose summaries score best, as a block table and lengths;
* ``sparse``   selection and attention over the selected pages: one attention call of one layer and decode step;
* ``fork``     rows of a block table forked (full pages shared, the partial last one copied in every layer) and freed again;
* ``compact``  the pages in use moved to the low end of the pool, in every layer, block tables and reference counts with them.

A page of n tokens with scales s_t, latent values e_td (E2M1) and RoPE values r_td (E4M3) has the mean key m: with S = max |s_t| and
w_t = round(32767 s_t / S), m_d = S / (32767 n) sum_t w_t e_td in the latent and 1/n sum_t r_td in the RoPE part; its scale is
max |m_d| / 127 rounded to 32 bits, its codes are round(m_d / scale).  A page with a scale that is not finite or a RoPE value that is NaN has the scale
NaN.  A query's head h is taken as integers, q 2^k rounded, where k brings its largest binade to [64, 128); a page scores
scale * max_h 2^-k_h <q_h, code>, rounded to 32 bits.  The first ``sink`` and the last ``local`` pages of a request are always taken, the
rest of the budget goes to the best scores (NaN first, then by value, ties to the lowest index).
"""
import math
import random

import torch

own = False

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_EDGES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


# ---------------------------------------------------------------------------------------------- cases
def _summary(name, pages, page, batch=0, new=0, lens=0):
    c = {"kind": "summary", "pages": pages, "page": page, "batch": batch, "new": new, "lens": lens}
    return dict(c, name=name) if name else c


def _sparse(kind, name, batch, heads, lo, hi, page, budget, sink=1, local=2, q_len=1, causal=False, lens=0):
    c = {"kind": kind, "batch": batch, "heads": heads, "lo": lo, "hi": hi, "page": page, "budget": budget, "sink": sink, "local": local,
         "q_len": q_len, "causal": causal, "lens": lens}
    return dict(c, name=name) if name else c


def _fork(name, parents, children, lo, hi, page, layers, summaries, lens=0):
    c = {"kind": "fork", "parents": parents, "children": children, "lo": lo, "hi": hi, "page": page, "layers": layers,
         "summaries": summaries, "lens": lens}
    return dict(c, name=name) if name else c


def _compact(name, pages, live, page, layers, summaries):
    c = {"kind": "compact", "pages": pages, "live": live, "page": page, "layers": layers, "summaries": summaries}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a chunk of 50 new tokens of each of 61 requests: the few pages that it fills, small pages; latency
        _summary("summary_step", 61 * 40, 16, batch=61, new=50, lens=61),
        # prompts of 512k tokens in all, just written
        _summary("summary_prompt", 8192, 64),
        # the smallest call: one chat on a tensor-parallel shard of 16 heads
        _sparse("select", "select_small", 1, 16, 9000, 9000, 64, 32),
        # many long documents, all 128 heads
        _sparse("select", "select_long", 64, 128, 131072, 131072, 64, 64),
        # the smallest attention call
        _sparse("sparse", "sparse_small", 1, 16, 9000, 9000, 64, 32),
        # long documents at a small batch: the headline configuration of the dense decode, 4096 tokens of each attended
        _sparse("sparse", "sparse_uniform", 8, 64, 32768, 32768, 64, 64),
        # odd everything: heads that fill no group, three query positions under a causal rule, ragged lengths of which some are within the budget
        _sparse("sparse", "sparse_ragged", 5, 40, 700, 60000, 16, 75, sink=2, local=3, q_len=3, causal=True, lens=5),
        # very long contexts of a data-parallel rank
        _sparse("sparse", "sparse_long", 32, 128, 131072, 131072, 64, 64),
        # four beams from one prompt, a draft model of two layers
        _fork("fork_small", 1, 4, 777, 777, 64, 2, False),
        # parallel samples of twelve prompts, all layers of a model at once
        _fork("fork_large", 12, 96, 3000, 30000, 128, 32, True, lens=12),
        # a small pool after a few requests have gone
        _compact("compact_small", 300, 170, 32, 2, True),
        # a pool of which a third is in use, in scattered pages
        _compact("compact_large", 6000, 2000, 64, 8, False),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("summary", "select", "sparse", "sparse", "sparse", "fork", "compact"))
    page = rng.choice((8, 16, 32, 64, 64, 128))
    if kind == "summary":
        if rng.random() < 0.5:
            batch, new = _log_uniform(rng, 1, 128), _log_uniform(rng, 1, 200)
            return _summary(None, batch * 300 + rng.randint(0, 9), page, batch, new, rng.randrange(1 << 30))
        return _summary(None, _log_uniform(rng, 1, 524288 // page), page)
    if kind == "fork":
        parents, layers = _log_uniform(rng, 1, 16), _log_uniform(rng, 1, 32)
        hi = _log_uniform(rng, page, 30000)
        return _fork(None, parents, _log_uniform(rng, 1, 96), max(1, int(hi * rng.uniform(0.1, 1.0))), hi, page, layers, rng.random() < 0.5,
                     rng.randrange(1 << 30))
    if kind == "compact":
        layers = _log_uniform(rng, 1, 16)
        pages = _log_uniform(rng, 20, 6000 * 8 * 64 // (layers * page * 2))
        return _compact(None, pages, max(1, int(pages * rng.uniform(0.02, 0.98))), page, layers, rng.random() < 0.5)
    heads = rng.choice((8, 16, 32, 64, 64, 128, 128, rng.randint(1, 128)))
    q_len = rng.choice((1, 1, 1, 2, 3))
    hi = _log_uniform(rng, 16, 131072)
    lo = hi if rng.random() < 0.4 else max(1, int(hi / math.exp(rng.uniform(0.0, 4.0))))
    sink, local = rng.randint(0, 3), rng.randint(1, 4)
    budget = max(sink + local, _log_uniform(rng, 2, max(2, 4096 // page)))
    batch = _log_uniform(rng, 1, max(1, min(64, 32 * 131072 // (hi * q_len * -(-64 // page)))))
    return _sparse(kind, None, batch, heads, lo, hi, page, budget, sink, local, q_len, rng.random() < 0.5, rng.randrange(1 << 30))


def _lengths(case, count):
    """The requests' lengths: part of the case, the same whatever the inputs."""
    rng = random.Random(case["lens"])
    return [_log_uniform(rng, case["lo"], case["hi"]) for _ in range(count)]


def _step_lengths(case):
    """Lengths after the step: every row of its table can hold them, and they count the new tokens."""
    rng, most = random.Random(case["lens"]), case["pages"] // case["batch"] * case["page"]
    return [rng.randint(min(case["new"], most), most) for _ in range(case["batch"])]


def _filled(case):
    """Pages that the step has filled."""
    return sum(n // case["page"] - max(0, n - case["new"]) // case["page"] for n in _step_lengths(case))


# ---------------------------------------------------------------------------------------------- inputs
def _rows(pages, page, gen, dev):
    """Cache rows and scales of that many pages: tokens of a page have a direction in common, and magnitudes of their own."""
    size = torch.rand(pages, page, 1, generator=gen, device=dev) * 3 + 0.25
    lat = torch.randn(pages, 1, 512, generator=gen, device=dev) * 0.7 + torch.randn(pages, page, 512, generator=gen, device=dev)
    lat *= size
    rope = torch.randn(pages, 1, 64, generator=gen, device=dev) + torch.randn(pages, page, 64, generator=gen, device=dev)
    sf = lat.abs().amax(-1, keepdim=True) / 6
    lat /= sf
    code = torch.bucketize(lat.abs(), torch.tensor(_EDGES, device=dev)).to(torch.uint8) | ((lat < 0).to(torch.uint8) << 3)
    return torch.cat((code[..., 0::2] | (code[..., 1::2] << 4), rope.to(torch.float8_e4m3fn).view(torch.uint8)), -1), sf


def _prepare_summary(case, gen, dev):
    pages, page = case["pages"], case["page"]
    s = {"page": page, "summary": torch.zeros(pages, 576, dtype=torch.int8, device=dev), "summary_sf": torch.zeros(pages, device=dev),
         "values": torch.empty(pages, 576, device=dev)}
    s["kv"], s["sf"] = _rows(pages, page, gen, dev)
    order = torch.randperm(pages, generator=gen, device=dev).int()
    if case["batch"]:
        width = pages // case["batch"]
        s["bt"] = order[: width * case["batch"]].view(case["batch"], width).contiguous()
        s["sl"], s["new"] = torch.tensor(_step_lengths(case), dtype=torch.int32, device=dev), case["new"]
    else:
        s["ids"] = order
    return s


def _prepare_sparse(case, gen, dev):
    page, heads, q_len = case["page"], case["heads"], case["q_len"]
    lens = _lengths(case, case["batch"])
    used = [-(-n // page) for n in lens]
    need, chunk = sum(used), 262144 // page
    pool = need + need // 8 + 1
    order = torch.randperm(pool, generator=gen, device=dev).int()
    bt = torch.zeros(case["batch"], max(used), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        bt[b, :n] = order[at:at + n]
        at += n
    kv = torch.empty(pool, page, 320, dtype=torch.uint8, device=dev)
    sf = torch.empty(pool, page, 1, device=dev)
    summary, summary_sf = torch.empty(pool, 576, dtype=torch.int8, device=dev), torch.empty(pool, device=dev)
    for lo in range(0, pool, chunk):
        n = min(chunk, pool - lo)
        kv[lo:lo + n], sf[lo:lo + n] = _rows(n, page, gen, dev)
        summary[lo:lo + n], summary_sf[lo:lo + n] = _summaries(kv[lo:lo + n], sf[lo:lo + n])
    q = torch.randn(case["batch"], q_len, heads, 576, generator=gen, device=dev) * torch.exp(0.5 * torch.randn(1, 1, heads, 1, generator=gen, device=dev))
    s = {"kv": kv, "sf": sf, "summary": summary, "summary_sf": summary_sf, "bt": bt, "sl": torch.tensor(lens, dtype=torch.int32, device=dev),
         "q": q.to(torch.float8_e4m3fn), "page": page, "budget": case["budget"], "sink": case["sink"], "local": case["local"],
         "causal": case["causal"], "longest": max(lens), "scale": 512 ** -0.5}
    if own and case["kind"] == "sparse":
        from flashinfer_mla_fp4_b200 import BatchMLASparseDecodeFP4Wrapper

        s["w"] = BatchMLASparseDecodeFP4Wrapper(torch.empty(64 << 20, dtype=torch.int8, device=dev))
        s["w"].plan(num_heads=heads, page_size=page, budget_pages=case["budget"], sink_pages=case["sink"], local_pages=case["local"],
                    causal=case["causal"])
    return s


def _layers(layers, pages, page, summaries, gen, dev):
    s = {"kv": torch.randint(0, 256, (layers, pages, page, 320), generator=gen, device=dev, dtype=torch.uint8),
         "sf": torch.rand(layers, pages, page, 1, generator=gen, device=dev)}
    if summaries:
        s["summary"] = torch.randint(-127, 128, (layers, pages, 576), generator=gen, device=dev, dtype=torch.int8)
        s["summary_sf"] = torch.rand(layers, pages, generator=gen, device=dev)
    if own:
        from flashinfer_mla_fp4_b200 import FP4MLAPagedCache, FP4MLAPagePool

        of = lambda key, i: s[key][i] if key in s else None  # noqa: E731
        s["pool"] = FP4MLAPagePool([FP4MLAPagedCache.from_tensors(of("kv", i), of("sf", i), of("summary", i), of("summary_sf", i))
                                    for i in range(layers)])
    return s


def _prepare_fork(case, gen, dev):
    page, parents, children = case["page"], case["parents"], case["children"]
    lens = _lengths(case, parents)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 2 * children + 16
    s = _layers(case["layers"], pages, page, case["summaries"], gen, dev)
    order = torch.randperm(pages, generator=gen, device=dev).int()
    bt = torch.zeros(parents + children, max(used), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        bt[b, :n] = order[at:at + n]
        at += n
    ref = torch.zeros(pages, dtype=torch.int32, device=dev)
    ref[order[:at].long()] = 1
    rows = torch.randperm(parents + children, generator=gen, device=dev).int()  # which rows of the table the requests have
    table, sl = torch.zeros_like(bt), torch.zeros(parents + children, dtype=torch.int32, device=dev)
    table[rows[:parents].long()] = bt[:parents]
    sl[rows[:parents].long()] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s |= {"bt": table, "sl": sl, "page": page, "children": rows[parents:].contiguous(), "ref": ref,
          "parents": rows[torch.randint(0, parents, (children,), generator=gen, device=dev)].contiguous()}
    if own:
        s["pool"].refcounts.copy_(ref)
    return s


def _prepare_compact(case, gen, dev):
    pages, live = case["pages"], case["live"]
    s = _layers(case["layers"], pages, case["page"], case["summaries"], gen, dev)
    order = torch.randperm(pages, generator=gen, device=dev)[:live]
    rows = min(16, live)
    width = -(-live // rows)
    bt = torch.cat((order, order[: rows * width - live])).int().view(rows, width)  # (the last row shares its end with the first)
    ref = torch.zeros(pages, dtype=torch.int32, device=dev).index_add_(0, bt.reshape(-1), torch.ones(rows * width, dtype=torch.int32, device=dev))
    full = torch.full((rows,), width * case["page"], dtype=torch.int32, device=dev)
    s |= {"bt0": bt, "ref0": ref, "bt": bt.clone(), "ref": ref.clone(), "sl": full, "page": case["page"]}
    return s


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    make = {"summary": _prepare_summary, "select": _prepare_sparse, "sparse": _prepare_sparse, "fork": _prepare_fork, "compact": _prepare_compact}
    return dict(make[case["kind"]](case, gen, dev), kind=case["kind"])


# ---------------------------------------------------------------------------------------------- the plain forms
def _values(kv):
    """Latent [..., 512] and RoPE [..., 64] of cache rows, in 32 bits."""
    table = torch.tensor(_E2M1, device=kv.device)
    low, high = kv[..., :256] & 15, kv[..., :256] >> 4
    return table[torch.stack((low, high), -1).flatten(-2).int()], kv[..., 256:].contiguous().view(torch.float8_e4m3fn).float()


def _summaries(kv, sf):
    """Codes int8 [n, 576] and scales [n] of full pages.  In 64 bits: a code next to the middle of two would go either way in 32."""
    lat, rope = _values(kv)
    s = sf.squeeze(-1).double()
    top = s.abs().amax(-1, keepdim=True)
    n = kv.shape[1]
    w = torch.round(32767 * s / torch.where(top > 0, top, 1.0))
    mean = torch.cat(((w.unsqueeze(1) @ lat.double()).squeeze(1) * (top / (32767 * n)), rope.double().sum(1) / n), -1)
    scale = (mean.abs().amax(-1) / 127).float()
    sound = torch.isfinite(top.squeeze(-1)) & torch.isfinite(scale)
    code = torch.round(mean / torch.where(sound & (scale > 0), scale, 1.0).double().unsqueeze(-1)).clamp(-127, 127)
    code = torch.where((sound & (scale > 0)).unsqueeze(-1), code, 0.0).to(torch.int8)
    return code, torch.where(sound, scale, math.nan)


def _selection(s):
    """Block table [rows, budget] and lengths [rows] of every query position."""
    q, bt, page, budget = s["q"], s["bt"], s["page"], s["budget"]
    batch, q_len, heads, _ = q.shape
    width, free = bt.shape[1], budget - s["sink"] - s["local"]
    back = torch.arange(q_len - 1, -1, -1, device=q.device, dtype=torch.int32) if s["causal"] else torch.zeros(q_len, device=q.device, dtype=torch.int32)
    lens = (s["sl"].unsqueeze(1) - back).clamp(min=0).reshape(-1)
    used = (lens + page - 1) // page
    table = bt.repeat_interleave(q_len, 0)
    raw = q.reshape(batch, q_len * heads, 576)
    bits = raw.view(torch.uint8).int() & 127
    e = torch.where(bits == 127, 0, bits >> 3).amax(-1, keepdim=True).clamp(min=1)
    unit = ((e + 114) << 23).view(torch.float32)  # 2^(e - 13)
    ints = torch.round(torch.nan_to_num(raw.float(), nan=0.0) / unit)
    dots = ints @ s["summary"][bt].float().transpose(1, 2)  # whole numbers below 2^24
    best = (dots * unit).view(batch, q_len, heads, width).amax(2).reshape(-1, width)
    score = best * s["summary_sf"][table]
    at = torch.arange(width, device=q.device).unsqueeze(0)
    rest = (at >= s["sink"]) & (at < (used - s["local"]).unsqueeze(1))
    order = torch.sort(torch.where(rest, score, -math.inf), dim=1, descending=True, stable=True).indices
    slot = torch.arange(budget, device=q.device).unsqueeze(0)
    picked = torch.gather(order, 1, (slot - s["sink"]).clamp(0, width - 1).expand(lens.numel(), -1))
    picked = torch.where(slot < s["sink"], slot, torch.where(slot < s["sink"] + free, picked, used.unsqueeze(1) - budget + slot))
    whole = (used <= budget).unsqueeze(1)
    picked = torch.where(whole, slot, picked.sort(1).values)
    chosen = torch.gather(table, 1, picked.clamp(0, width - 1).long())
    kept = torch.where(used <= budget, lens, lens - (used - budget) * page)
    return torch.where(slot < used.unsqueeze(1), chosen, 0), kept.int()


def _attention(s, table, lens):
    batch, q_len, heads, _ = s["q"].shape
    kv = s["kv"][table].flatten(1, 2)
    lat, rope = _values(kv)
    lat *= s["sf"][table].flatten(1, 2)
    q = s["q"].reshape(batch * q_len, heads, 576).float()
    x = (q[..., :512] @ lat.transpose(1, 2) + q[..., 512:] @ rope.transpose(1, 2)) * s["scale"]
    there = (torch.arange(kv.shape[1], device=q.device) < lens.unsqueeze(1)).unsqueeze(1)
    x = torch.where(there, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.where(there, torch.exp(x - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
    out = (p @ lat) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.view(batch, q_len, heads, 512).to(torch.bfloat16)


def _summary_plain(s):
    page = s["page"]
    if "ids" in s:
        ids = s["ids"].long()
    else:
        sl = s["sl"].unsqueeze(1)
        at = sl // page - 1 - torch.arange(-(-s["new"] // page), device=sl.device)
        fresh = (at >= 0) & ((at + 1) * page > sl - s["new"])
        ids = torch.gather(s["bt"], 1, at.clamp(min=0))[fresh].long()
    s["summary"][ids], s["summary_sf"][ids] = _summaries(s["kv"][ids], s["sf"][ids])


def _fork_plain(s):
    bt, sl, ref, page = s["bt"], s["sl"], s["ref"], s["page"]
    parents, children = s["parents"].long(), s["children"].long()
    lens, at = sl[parents], torch.arange(bt.shape[1], device=bt.device)
    row = bt[parents]
    shared = at < (lens // page).unsqueeze(1)
    tail = (lens % page > 0).nonzero().squeeze(1)
    fresh = (ref == 0).nonzero().squeeze(1)[: tail.numel()]
    last = (lens[tail] // page).long()
    old = row[tail, last].long()
    row[tail, last] = fresh.int()
    inside = at < ((lens + page - 1) // page).unsqueeze(1)
    bt[children] = torch.where(inside, row, bt[children])
    sl[children] = lens
    ref.index_add_(0, row[shared].long(), torch.ones_like(row[shared]))
    ref[fresh] = 1
    for_all = [s[k] for k in ("kv", "sf", "summary", "summary_sf") if k in s]
    [x.index_copy_(1, fresh, x[:, old]) for x in for_all]


def _free_plain(s):
    bt, sl, ref, rows = s["bt"], s["sl"], s["ref"], s["children"].long()
    inside = torch.arange(bt.shape[1], device=bt.device) < ((sl[rows] + s["page"] - 1) // s["page"]).unsqueeze(1)
    gone = bt[rows][inside]
    ref.index_add_(0, gone.long(), -torch.ones_like(gone))
    sl[rows] = 0


def _compact_plain(s):
    bt, ref = s["bt"], s["ref"]
    at, live = torch.arange(ref.numel(), device=ref.device), ref > 0
    count = live.sum()
    holes, high = (~live & (at < count)).nonzero().squeeze(1), (live & (at >= count)).nonzero().squeeze(1)
    [x.index_copy_(1, holes, x[:, high]) for x in [s[k] for k in ("kv", "sf", "summary", "summary_sf") if k in s]]
    remap = torch.where(live, at, -1).int()
    remap[high] = holes.int()
    ref[holes] = ref[high]
    ref[high] = 0
    bt.copy_(remap[bt.long()])
    return remap


def run(state):
    s, kind = state, state["kind"]
    if kind == "summary":
        if not own:
            _summary_plain(s)
        elif "ids" in s:
            from flashinfer_mla_fp4_b200.sparse import summarize_pages

            summarize_pages(s["kv"], s["sf"], s["summary"], s["summary_sf"], s["ids"])
        else:
            from flashinfer_mla_fp4_b200.sparse import summarize_new_pages

            summarize_new_pages(s["kv"], s["sf"], s["summary"], s["summary_sf"], s["bt"], s["sl"], s["new"])
        return torch.mul(s["summary"], s["summary_sf"].unsqueeze(1), out=s["values"])  # 8 bits and a scale, as the values they stand for
    if kind == "select":
        if not own:
            return _selection(s)
        from flashinfer_mla_fp4_b200.sparse import select_pages

        return select_pages(s["q"], s["summary"], s["summary_sf"], s["bt"], s["sl"], s["page"], s["budget"], sink_pages=s["sink"],
                            local_pages=s["local"], causal=s["causal"])
    if kind == "sparse":
        if not own:
            return _attention(s, *_selection(s))
        return s["w"].run(s["q"], s["kv"], s["bt"], s["sl"], s["longest"], s["scale"], kv_cache_sf=s["sf"], summary=s["summary"],
                          summary_sf=s["summary_sf"])
    buffers = {"kv": s["kv"], "sf": s["sf"].view(torch.int32), "bt": s["bt"], "sl": s["sl"]}  # copied scales: their bits
    if "summary" in s:
        buffers |= {"summary": s["summary"], "summary_sf": s["summary_sf"].view(torch.int32)}
    if kind == "fork":
        if not own:
            _fork_plain(s)
            _free_plain(s)
            return dict(buffers, ref=s["ref"])
        s["pool"].fork(s["bt"], s["sl"], s["parents"], s["children"])
        s["pool"].free(s["bt"], s["sl"], s["children"])
        return dict(buffers, ref=s["pool"].refcounts)
    s["bt"].copy_(s["bt0"])  # the pool as it was before the pass
    ref = s["pool"].refcounts if own else s["ref"]
    ref.copy_(s["ref0"])
    remap = s["pool"].compact(s["bt"], s["sl"]) if own else _compact_plain(s)
    return dict(buffers, ref=ref, remap=remap)


# ---------------------------------------------------------------------------------------------- floors
def _selected(case):
    """Per request: length, candidate pages (0 where the budget holds all), tokens attended by a query position."""
    page, budget = case["page"], case["budget"]
    for n in _lengths(case, case["batch"]):
        used = -(-n // page)
        yield n, (0 if used <= budget else used - case["sink"] - case["local"]), (n if used <= budget else n - (used - budget) * page)


def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "summary":
        pages = _filled(case) if case["batch"] else case["pages"]
        return {"bytes": max(1, pages) * (324 * page + 580 + 4) + 4 * case["batch"], "flops": 2 * 576 * page * pages}
    if kind in ("select", "sparse"):
        rows, heads, budget = case["batch"] * case["q_len"], case["heads"], case["budget"]
        some = list(_selected(case))
        pages = sum(c for _, c, _ in some)
        total = {"bytes": 584 * pages + rows * (heads * 576 + 4 * budget + 4) + 4 * case["batch"], "flops": 2 * 576 * heads * pages * case["q_len"]}
        if kind == "sparse":  # query positions of a request may have selected the same pages
            total["bytes"] += sum(328 * t for _, _, t in some) + rows * heads * 1024
            total["flops"] += sum(2176 * t for _, _, t in some) * heads * case["q_len"]
        return total
    each = case["layers"] * (324 * page + (580 if case["summaries"] else 0))
    if kind == "fork":
        used = max(1, max(-(-n // page) for n in _lengths(case, case["parents"])))
        return {"bytes": case["children"] * (2 * each + 8 * used), "flops": 0}
    moved = case["live"] * (case["pages"] - case["live"]) // case["pages"]  # of a random choice
    return {"bytes": max(1, moved) * 2 * each + 12 * case["pages"] + 8 * case["live"], "flops": 0}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _page_means(kv, sf):
    """[pages, 576] mean keys in 64 bits, summed token by token."""
    half = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=torch.int64, device=kv.device)
    pages, n = kv.shape[:2]
    top = sf.abs().amax(1).double()
    total = torch.zeros(pages, 512, dtype=torch.int64, device=kv.device)
    rope = torch.zeros(pages, 64, dtype=torch.float64, device=kv.device)
    for t in range(n):
        w = (sf[:, t].double() / top * 32767).round().long()
        b = kv[:, t, :256].long()
        total[:, 0::2] += w * half[b % 16]
        total[:, 1::2] += w * half[b // 16]
        rope += kv[:, t, 256:].contiguous().view(torch.float8_e4m3fn).double()
    return torch.cat((total.double() * top / (65534 * n), rope / n), 1)


def exact(case, seed):
    if case["kind"] not in ("summary", "sparse"):
        return None
    s = prepare(case, seed)
    dev, page = s["kv"].device, s["page"]
    if case["kind"] == "summary":
        out = torch.zeros(case["pages"], 576, dtype=torch.float64, device=dev)
        ids = s["ids"].tolist() if "ids" in s else [
            p for row, n in zip(s["bt"].tolist(), _step_lengths(case)) for i, p in enumerate(row) if n - case["new"] < (i + 1) * page <= n]
        for lo in range(0, len(ids), 2048):
            some = torch.tensor(ids[lo:lo + 2048], device=dev)
            mean = _page_means(s["kv"][some], s["sf"][some])
            scale = (mean.abs().amax(1, keepdim=True) / 127).float().double()
            out[some] = (mean / scale).round() * scale
        return out
    heads, q_len, budget, lens = case["heads"], case["q_len"], case["budget"], _lengths(case, case["batch"])
    out = torch.zeros(case["batch"], q_len, heads, 512, dtype=torch.float64, device=dev)
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=dev)
    for b, n in enumerate(lens):
        for i in range(q_len):
            length = max(0, n - (q_len - 1 - i if case["causal"] else 0))
            used = -(-length // page)
            if not used:
                continue
            ids = s["bt"][b, :used].long()
            q = s["q"][b, i].double()
            if used > budget:
                top = q.abs().amax(1, keepdim=True).clamp(min=2.0 ** -6)
                unit = torch.tensor([2.0 ** (k - 7) for k in range(-8, 12)], dtype=torch.float64, device=dev)[torch.frexp(top).exponent.long() + 8]
                score = ((q / unit).round() @ s["summary"][ids].double().T * unit).amax(0) * s["summary_sf"][ids].double()
                score = score.float().tolist()  # the score is a value of 32 bits
                middle = sorted(range(case["sink"], used - case["local"]), key=lambda p: (-score[p], p))[: budget - case["sink"] - case["local"]]
                keep = sorted(set(range(case["sink"])) | set(middle) | set(range(used - case["local"], used)))
                length -= (used - len(keep)) * page
                ids = ids[torch.tensor(keep, device=dev)]
            row = s["kv"][ids].flatten(0, 1)[:length]
            codes = torch.stack((row[:, :256] % 16, row[:, :256] // 16), -1).flatten(1).long()
            key = grid[codes] * s["sf"][ids].flatten(0, 1)[:length].double()
            rope = row[:, 256:].contiguous().view(torch.float8_e4m3fn).double()
            x = (q[:, :512] @ key.T + q[:, 512:] @ rope.T) * s["scale"]
            out[b, i] = torch.softmax(x, 1) @ key
    return out
