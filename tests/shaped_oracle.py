"""Shaped attention, key mass and eviction from their definitions, in 64 bits, and random caches to try them on."""
import math

import torch

F64 = torch.float64


class Cache:
    """Pools, block table and positions of sequences with the given numbers of cached tokens; row 0 and the scratch page are nobody's (NaN)."""

    def __init__(self, lens, Hkv, D, *, device="cuda", seed=0, order="scattered", shed=False, spare=0):
        g = torch.Generator(device=device).manual_seed(seed)
        total = sum(lens) + spare
        self.lens, self.Hkv, self.D = list(lens), Hkv, D
        self.k, self.v = (torch.randn(total + 1, Hkv * D, device=device, generator=g).bfloat16() for _ in range(2))
        self.k[0] = self.v[0] = float("nan")
        ids = torch.randperm(total, device=device, generator=g) if order == "scattered" else torch.arange(total, device=device)
        if order == "down":
            ids = ids.flip(0)
        self.table = torch.zeros(len(lens) + 1, max(max(lens), 1) + 5, dtype=torch.int32, device=device)
        self.key_pos, at = (torch.zeros_like(self.table) if shed else None), 0
        for i, n in enumerate(lens):
            self.table[i + 1, :n] = ids[at:at + n].int() + 1
            at += n
            if shed and n:
                steps = torch.randint(1, 4, (n,), device=device, generator=g)
                steps[-min(n, 3):] = 1
                self.key_pos[i + 1, :n] = (steps.cumsum(0) - 1).int()

    def positions(self, row):
        n = self.lens[row - 1]
        return torch.arange(n, device=self.table.device) if self.key_pos is None else self.key_pos[row, :n].long()


def attend(cache, runs, q, Hq, *, scale, softcap=0.0, slopes=None, bounds=None):
    """out [T, Hq, D], lse [T, Hq] and the mass per row [Hkv, tokens] of runs (row, held, at, n); held < 0: the first tokens are padding."""
    D, Hkv = cache.D, cache.Hkv
    T = q.shape[0]
    out = torch.zeros(T, Hq, D, dtype=F64, device=q.device)
    lse = torch.full((T, Hq), -math.inf, dtype=F64, device=q.device)
    mass = {}
    for row, held, at, n in runs:
        L, lead = held + n, max(0, -held)
        mass[row] = torch.zeros(Hkv, max(L, 0), dtype=F64, device=q.device)
        if L <= 0 or n <= lead:
            continue
        pages, pos = cache.table[row, :L].long(), cache.positions(row)[:L]
        k, v = (x[pages].view(L, Hkv, D).double().repeat_interleave(Hq // Hkv, 1) for x in (cache.k, cache.v))
        mine = pos[max(held, 0):]
        s = torch.einsum("qhd,khd->hqk", q[at + lead:at + n].view(-1, Hq, D).double(), k) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes.double().view(-1, 1, 1) * (mine[:, None] - pos).abs()
        first, last = (torch.zeros_like(mine), mine) if bounds is None else bounds[at + lead:at + n].long().unbind(1)
        hidden = (pos < first[:, None]) | (pos > last[:, None])
        s = s.masked_fill(hidden, -math.inf)
        empty = hidden.all(1)
        z = torch.logsumexp(s, -1)
        w = torch.exp(s - z[..., None]).masked_fill(empty[:, None], 0.0)
        out[at + lead:at + n] = torch.einsum("hqk,khd->qhd", w, v)
        lse[at + lead:at + n] = z.T
        mass[row] += w.view(Hkv, -1, w.shape[1], L).sum((1, 2))
    return out, lse, mass


def choose(score, keep, first, last):
    """Indices that stay, ascending: plain sorting of Python numbers."""
    n = len(score)
    if n <= keep:
        return list(range(n))
    inner = range(first, n - last)
    worth = lambda j: (-math.inf if math.isnan(score[j]) else -score[j], j)                # noqa: E731  NaN above all, ties to the lower index
    best = sorted(inner, key=worth)[:keep - first - last]
    return sorted(list(range(first)) + best + list(range(n - last, n)))


def head_sums(mass):
    """fp32 sums over the heads in their order, of mass [heads, n]."""
    s = mass[0].clone()
    for h in range(1, mass.shape[0]):
        s = s + mass[h]
    return s
