"""CPU restatement of sparse decode's selection and of the page pool, one value at a time: test infrastructure only."""
from __future__ import annotations

import math

import torch

_TWICE = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=torch.int64)


def summarize(kv, sf):
    """Codes int8 [576] and the scale of one full page: kv u8 [n, 320], sf f32 [n, 1].  Whole numbers, and Python floats (64 bits)."""
    n = kv.shape[0]
    s = [float(x) for x in sf.view(-1)]
    rope = kv[:, 256:].contiguous().view(torch.float8_e4m3fn).double()
    if not all(math.isfinite(x) for x in s) or bool(rope.isnan().any()):
        return torch.zeros(576, dtype=torch.int8), math.nan
    top = max(abs(x) for x in s)
    w = torch.tensor([round(32767 * x / top) if top > 0 else 0 for x in s], dtype=torch.int64)
    codes = torch.stack((kv[:, :256] & 15, kv[:, :256] >> 4), -1).flatten(1).long()
    total = (w.unsqueeze(1) * _TWICE[codes]).sum(0)
    mean = torch.cat((total.double() * (top / (65534.0 * n)), rope.sum(0) / n))
    scale = float((mean.abs().max() / 127).float())
    if not math.isfinite(scale):
        return torch.zeros(576, dtype=torch.int8), math.nan
    if scale == 0:
        return torch.zeros(576, dtype=torch.int8), 0.0
    return (mean / scale).round().clamp(-127, 127).to(torch.int8), scale


def query_codes(q):
    """Whole numbers [H, 576] and the units [H] that they count, of one query position q e4m3 [H, 576]."""
    x = q.double().nan_to_num(nan=0.0)
    codes, units = [], []
    for h in range(x.shape[0]):
        top = float(x[h].abs().max())
        unit = 2.0 ** ((math.frexp(top)[1] - 1 if top >= 2.0 ** -6 else -6) - 6)
        codes.append((x[h] / unit).round())
        units.append(unit)
    return torch.stack(codes), torch.tensor(units, dtype=torch.float64)


def scores(q, summary, summary_sf, ids):
    """FP32 scores of the pages `ids` for one query position; -inf-and-below (None) for a page outside the pool."""
    codes, units = query_codes(q)
    out = []
    for p in ids:
        if not 0 <= p < summary.shape[0]:
            out.append(None)
            continue
        best = float(((codes @ summary[p].double()) * units).max())
        out.append(float(torch.tensor(best * float(summary_sf[p]), dtype=torch.float64).float()))
    return out


def select(q, summary, summary_sf, block_tables, seq_lens, page_size, budget, sink, local, causal):
    """(table int32 [B * q_len, budget], lengths int32 [B * q_len]) with all tensors on the host."""
    B, q_len = q.shape[:2]
    tables, lens = [], []
    width = block_tables.shape[1]
    for b in range(B):
        for i in range(q_len):
            n = min(int(seq_lens[b]), width * page_size)
            n = max(0, n - (q_len - 1 - i if causal else 0))
            ids = [int(x) for x in block_tables[b, : -(-n // page_size)]]
            if len(ids) > budget:
                used = len(ids)
                middle = list(range(sink, used - local))

                def rank(pos, s=dict(zip(middle, scores(q[b, i], summary, summary_sf, [ids[m] for m in middle])))):
                    v = s[pos]
                    return (2, 0.0, pos) if v is None else (0, 0.0, pos) if math.isnan(v) else (1, -v, pos)

                best = sorted(middle, key=rank)[: budget - sink - local]
                keep = sorted(list(range(sink)) + best + list(range(used - local, used)))
                n -= (used - budget) * page_size
                ids = [ids[k] for k in keep]
            tables.append(ids + [0] * (budget - len(ids)))
            lens.append(n)
    return torch.tensor(tables, dtype=torch.int32).view(B * q_len, budget), torch.tensor(lens, dtype=torch.int32)


class Pool:
    """Reference counts, tables and lengths as Python lists; what moved as (from, to) pairs in order."""

    def __init__(self, refcounts, block_tables, seq_lens, page_size):
        self.ref, self.bt, self.sl, self.ps = list(refcounts), [list(r) for r in block_tables], list(seq_lens), page_size
        self.moves, self.trouble = [], False

    def pages(self, n):
        return max(0, -(-n // self.ps))

    def free_pages(self):
        return [p for p, r in enumerate(self.ref) if r <= 0]

    def allocate(self, new_lens):
        """Returns the lengths that the rows have pages for now: the new one, or the old one of a row that got none."""
        free, at, held = self.free_pages(), 0, list(self.sl)
        for r, n in enumerate(new_lens):
            have, want = self.pages(self.sl[r]), self.pages(n)
            if want > len(self.bt[r]):
                self.trouble = True
                continue
            if want <= have:
                held[r] = n if want == have else self.sl[r]
                continue
            got = free[at:at + want - have]
            if len(got) < want - have:  # (what there is stays for the rows behind it)
                self.trouble = True
                continue
            at += want - have
            for k, p in enumerate(got):
                self.bt[r][have + k] = p
                self.ref[p] = 1
            held[r] = n
        return held

    def fork(self, parents, children):
        free, at, seen, done = self.free_pages(), 0, set(), []
        for a, c in zip(parents, children):
            if a < 0 or c < 0:
                continue
            named = c in seen
            if 0 <= c < len(self.bt) and 0 <= a < len(self.bt):
                seen.add(c)
            if named or a >= len(self.bt) or c >= len(self.bt) or self.sl[c] > 0 or self.pages(self.sl[a]) > len(self.bt[a]):
                self.trouble = True
                continue
            n = max(0, self.sl[a])
            tail = None
            if n % self.ps:
                at += 1
                if at > len(free):
                    self.trouble = True
                    continue
                tail = free[at - 1]
            done.append((a, c, n, tail))
        for a, c, n, tail in done:
            for k in range(self.pages(n)):
                p = self.bt[a][k]
                if k < n // self.ps:
                    self.ref[p] += 1
                else:
                    self.moves.append((p, tail))
                    self.ref[tail] = 1
                    p = tail
                self.bt[c][k] = p
        for a, c, n, tail in done:
            self.sl[c] = n

    def free(self, rows):
        for r in rows:
            if r < 0:
                continue
            if r >= len(self.bt):
                self.trouble = True
                continue
            for p in self.bt[r][: self.pages(self.sl[r])]:
                if self.ref[p] > 0:
                    self.ref[p] -= 1
                else:
                    self.trouble = True
            self.sl[r] = 0

    def compact(self):
        n = sum(r > 0 for r in self.ref)
        remap = [p if r > 0 else -1 for p, r in enumerate(self.ref)]
        holes = [p for p in range(n) if self.ref[p] <= 0]
        high = [p for p in range(n, len(self.ref)) if self.ref[p] > 0]
        for p, h in zip(high, holes):
            remap[p], self.ref[h], self.ref[p] = h, self.ref[p], 0
            self.moves.append((p, h))
        for r, row in enumerate(self.bt):
            for k in range(min(self.pages(self.sl[r]), len(row))):
                if remap[row[k]] >= 0:
                    row[k] = remap[row[k]]
        return remap
