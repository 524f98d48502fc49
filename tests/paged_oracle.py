"""A paged cache for tests, and the plain 64-bit forms of the operators around it."""
from __future__ import annotations

import math

import torch

import attn_oracle


class Cache:
    """Sequences of ``lens`` tokens in pages of their own, in no order; unused slots and pages
    that belong to nobody hold NaN."""

    def __init__(self, lens, H_KV, D, dtype=torch.bfloat16, page=16, cols=None, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.lens_list, self.page, self.dtype, self.device = list(lens), page, dtype, device
        pages = [-(-n // page) for n in lens]
        self.cols = cols or max(max(pages, default=1), 1)
        self.blocks = sum(pages) + 2
        ids = torch.randperm(self.blocks, generator=g).tolist()
        table = torch.full((len(lens), self.cols), -1, dtype=torch.int32)
        k = torch.full((self.blocks, page, H_KV, D), math.nan, dtype=dtype)
        v = k.clone()
        self.k_rows, self.v_rows = [], []
        for s, n in enumerate(lens):
            kr, vr = (torch.randn(n, H_KV, D, generator=g).to(dtype) for _ in range(2))
            self.k_rows.append(kr)
            self.v_rows.append(vr)
            for j in range(pages[s]):
                b = ids.pop()
                if j < self.cols:
                    table[s, j] = b
                some = slice(j * page, min(n, (j + 1) * page))
                k[b, :some.stop - some.start] = kr[some]
                v[b, :some.stop - some.start] = vr[some]
        self.table, self.k, self.v = table.to(device), k.to(device), v.to(device)
        self.lens = torch.tensor(lens, dtype=torch.int32).to(device)

    def set(self, s, pos, k=None, v=None):
        """Overwrites the key or value of position ``pos`` of sequence s (all heads)."""
        b, slot = int(self.table[s, pos // self.page]), pos % self.page
        if k is not None:
            self.k[b, slot] = k
            self.k_rows[s][pos] = k
        if v is not None:
            self.v[b, slot] = v
            self.v_rows[s][pos] = v


def offsets(new, device="cuda"):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def attend(cache, q, new, scale, there=None):
    """attn_oracle.attend's results of every sequence's tokens q [T, H_Q, D], joined.  ``there``:
    per sequence the positions that it has (default: all)."""
    outs, at = [], 0
    for s, n in enumerate(new):
        m = cache.lens_list[s]
        limit = torch.arange(n) + (m - n) + 1
        k, v = cache.k_rows[s], cache.v_rows[s]
        if there is not None:
            keep = torch.tensor(there[s], dtype=torch.long)
            limit = (keep[None] < limit[:, None]).sum(1)
            k, v = k[keep], v[keep]
        outs.append(attn_oracle.attend(q[at:at + n], k, v, scale, limit)[:3])
        at += n
    return tuple(torch.cat(x) for x in zip(*outs))


def attend_pages(cache, q, new, pages, scale):
    """The same over the pages [T, H_KV, n] that every token sees."""
    H_KV, P = pages.shape[1], cache.page
    G = q.shape[1] // H_KV
    outs, at = [], 0
    for s, n in enumerate(new):
        m = cache.lens_list[s]
        for i in range(n):
            heads = []
            for h in range(H_KV):
                pos = [p for j in pages[at + i, h].tolist() if 0 <= j < cache.cols
                       for p in range(j * P, min((j + 1) * P, m - n + i + 1))]
                k, v = (x[s][pos, h:h + 1] for x in (cache.k_rows, cache.v_rows))
                heads.append(attn_oracle.attend(q[at + i:at + i + 1, h * G:(h + 1) * G], k, v, scale,
                                                torch.tensor([len(pos)]))[:3])
            outs.append(tuple(torch.cat(x, 1) for x in zip(*heads)))
        at += n
    return tuple(torch.cat(x) for x in zip(*outs))


def tables(old, new, table, free, n_tokens, page, cursor=0):
    """paged_tables, token by token: (table, lens, cu, seq, pos, slots, taken)."""
    table = [list(r) for r in table]
    cols = len(table[0])
    lens, cu, rows = [], [0], []
    for s, (o, n) in enumerate(zip(old, new)):
        o, n = max(o, 0), max(n, 0)
        n = min(n, 2 ** 31 - 1 - o, n_tokens - cu[-1])
        for j in range(-(-o // page), min(-(-(o + n) // page), cols)):
            table[s][j] = free[cursor] if cursor < len(free) else -1
            cursor += 1
        for p in range(o, o + n):
            b = table[s][p // page] if p // page < cols else -1
            rows.append((s, p, b * page + p % page if b >= 0 else -1))
        lens.append(o + n)
        cu.append(cu[-1] + n)
    rows += [(-1, -1, -1)] * (n_tokens - len(rows))
    seq, pos, slots = ([r[i] for r in rows] for i in range(3))
    return table, lens, cu, seq, pos, slots, cursor


def bounds(cache, s, j):
    """Least and largest key [H_KV, 2, D] of page j of sequence s."""
    k = cache.k_rows[s][j * cache.page:(j + 1) * cache.page].float()
    return torch.stack([k.amin(0), k.amax(0)], 1)


def select(q, boxes, last, take, first, recent, there):
    """Pages of one token and head: q [G, D], boxes [pages, 2, D], both exact in float64; ``last``
    its own page; ``there`` the pages that are there."""
    score = {}
    for j in range(min(last + 1, boxes.shape[0])):
        b = boxes[j].double()
        term = torch.maximum(q.double() * b[0], q.double() * b[1])
        score[j] = torch.where(q == 0, 0.0, term).sum().item()
    kept = {j for j in score if j < first or j > last - recent} & there
    rest = [j for j in score if j not in kept and j in there and first <= j <= last - recent]
    rest.sort(key=lambda j: (-math.inf if math.isnan(score[j]) else -score[j], not math.isnan(score[j]), j))
    kept |= set(rest[:max(0, take - len(kept))])
    kept = sorted(kept)[:take]
    return kept + [-1] * (take - len(kept))
