"""Plain 64-bit implementations of the serving operators, and the tolerances their results are held to."""
from __future__ import annotations

import math

import torch

from huggingfaceeacp_b200 import native

TYPES = {"f32": (native.F32, torch.float32), "bf16": (native.BF16, torch.bfloat16), "f16": (native.F16, torch.float16)}
PAGE = native.PAGE_ROWS


def attend(q, k, v, seen, scale):
    """(out, weight) in 64 bits of q [n, H, D] over k, v [m, KVH, D] where seen [n, m]: weight is sum_j p_j |v_j|, the
    scale of the rounding errors. Keys that a row does not see are not used, whatever they hold."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(n, heads, d, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for i in range(n):
        at = seen[i].nonzero()[:, 0]
        if not len(at):
            continue
        kk, vv = (x[at].double().repeat_interleave(group, 1) for x in (k, v))
        scores = torch.einsum("hd,jhd->hj", q[i].double(), kk) * scale
        weights = torch.softmax(scores, 1)
        out[i] = torch.einsum("hj,jhd->hd", weights, vv)
        size[i] = torch.einsum("hj,jhd->hd", weights, vv.abs())
    return out, size


def tolerance(out, size, q, k, scale, keys, dtype):
    """Elementwise bound. With u = 2^-24: a score is a sum of D products whose partial sums stay below |q||k|, so it is off by
    about (sqrt(D) + 8) u scale |q||k|, or 8 times that with operands of 22 bits (the fp32 path may split them in two
    halves), and a weight by twice that; each weight is rounded once, to the type's half step (2^-21 in fp32), and summed
    in chains of at most sqrt(keys) + 8 rounding steps; the result is rounded once to the type."""
    u = 2.0 ** -24
    half = torch.finfo(dtype).eps / 2
    big = float(q.double().norm(dim=-1).nan_to_num(0, 0, 0).max() * k.double().norm(dim=-1).nan_to_num(0, 0, 0).max())
    score = (math.sqrt(q.shape[-1]) + 8) * 8 * u * scale * big
    weight = 2.0 ** -21 if dtype == torch.float32 else half
    return size * (2 * score + weight + (math.sqrt(max(keys, 1)) + 8) * u) + half * out.abs() + torch.finfo(dtype).smallest_normal


def close(got, out, size, q, k, scale, keys):
    tol = tolerance(out, size, q, k, scale, keys, got.dtype)
    off = (got.double() - out).abs()
    bad = ~((off <= tol) | (torch.isnan(out) & torch.isnan(got)))
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} values are off, the worst by "
                                 f"{float((off / tol).nan_to_num(math.inf)[bad].max()):.3g} tolerances, first at "
                                 f"{bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(out[bad][0])}")


def packed(q, k, v, lengths, scale, begin=0):
    out, size = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for n in lengths:
        rows = slice(begin, begin + n)
        if n:
            seen = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
            out[rows], size[rows] = attend(q[rows], k[rows], v[rows], seen, scale)
        begin += n
    return out, size


def path(parents, n):
    """The nodes on the path from node n up; a parent that is not before its child ends it."""
    nodes = []
    while n >= 0:
        nodes.append(n)
        n = parents[n] if parents[n] < n else -1
    return nodes


def tree(q, k, v, nodes, parents, keys, values, table, lengths, scale):
    """keys, values [pages, PAGE, KVH, D]; table and lengths are lists; parents one list a sequence."""
    out, size = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    begin = 0
    for s, n in enumerate(nodes):
        rows = slice(begin, begin + n)
        length = max(lengths[s], 0)
        ids = [table[s][j // PAGE] for j in range(length)]
        there = torch.tensor([0 <= p < keys.shape[0] for p in ids], dtype=torch.bool, device=q.device)
        at = torch.tensor([(p if 0 <= p < keys.shape[0] else 0) * PAGE + j % PAGE for j, p in enumerate(ids)],
                          dtype=torch.long, device=q.device)
        cached = [x.reshape(-1, *x.shape[2:])[at] for x in (keys, values)]
        seen = torch.zeros(n, length + n, dtype=torch.bool, device=q.device)
        seen[:, :length] = there
        for i in range(n):
            seen[i, [length + j for j in path(parents[s], i)]] = True
        if n:
            out[rows], size[rows] = attend(q[rows], torch.cat([cached[0], k[rows]]), torch.cat([cached[1], v[rows]]), seen,
                                           scale)
        begin += n
    return out, size


class Book:
    """The cache's book and pools in plain Python, step by step as the header says."""

    def __init__(self, keys, values, table, lengths, refs):
        self.keys, self.values = keys.clone(), values.clone()
        self.table, self.lengths, self.refs = ([list(r) for r in table], list(lengths), list(refs))
        self.pages, self.stride = len(refs), len(table[0])

    def held(self, length):
        return min(self.stride, -(-max(length, 0) // PAGE))

    def update(self, release=(), forks=(), grow=None):
        for s in release:
            if not 0 <= s < len(self.lengths):
                continue
            for j in range(self.held(self.lengths[s])):
                if 0 <= self.table[s][j] < self.pages:
                    self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lengths[s] = 0
        before, named = list(self.lengths), set()
        for source, target in forks:
            ok = 0 <= source < len(before) and 0 <= target < len(before) and before[target] <= 0 and target not in named
            named.add(target)
            if not ok or before[source] <= 0:
                continue
            for j in range(self.held(before[source])):
                self.table[target][j] = self.table[source][j]
                if 0 <= self.table[source][j] < self.pages:
                    self.refs[self.table[source][j]] += 1
            self.lengths[target] = before[source]
        free = [p for p in range(self.pages) if self.refs[p] <= 0]
        plan, refs, past = [], list(self.refs), 0
        for s, more in enumerate(grow or []):
            if more < 1:
                continue
            n = self.lengths[s]
            if n + more > self.stride * PAGE:
                past += 1
                continue
            copy = False
            if n % PAGE:
                p = self.table[s][n // PAGE]
                copy = 0 <= p < self.pages and refs[p] > 1
                if copy:
                    refs[p] -= 1
            plan.append((s, more, copy, self.held(n + more) - self.held(n)))
        wanted = sum(copy + new for _, _, copy, new in plan)
        if wanted > len(free) or past:
            return [len(free), max(0, wanted - len(free)), past]
        for s, more, copy, new in plan:
            n = self.lengths[s]
            if copy:
                old, fresh = self.table[s][n // PAGE], free.pop(0)
                for pool in (self.keys, self.values):
                    pool[:, fresh, : n % PAGE] = pool[:, old, : n % PAGE]
                self.refs[old] -= 1
                self.refs[fresh], self.table[s][n // PAGE] = 1, fresh
            for j in range(new):
                fresh = free.pop(0)
                self.refs[fresh], self.table[s][self.held(n) + j] = 1, fresh
            self.lengths[s] = n + more
        return [len(free), 0, 0]

    def compact(self):
        live = [p for p in range(self.pages) if self.refs[p] > 0]
        count = len(live)
        holes = [p for p in range(count) if self.refs[p] <= 0]
        for old in [p for p in live if p >= count]:
            new = holes.pop(0)
            for pool in (self.keys, self.values):
                pool[:, new] = pool[:, old]
            self.refs[new], self.refs[old] = self.refs[old], 0
            for s, row in enumerate(self.table):
                for j in range(self.held(self.lengths[s])):
                    if row[j] == old:
                        row[j] = new
        return count

    def write(self, layer, k, v, offsets, index=None):
        for s in range(len(self.lengths)):
            for r in range(offsets[s], offsets[s + 1]):
                position = self.lengths[s] - offsets[s + 1] + r
                source = r if index is None else index[r]
                if not (0 <= position < self.stride * PAGE and 0 <= source < len(k)):
                    continue
                p = self.table[s][position // PAGE]
                if 0 <= p < self.pages:
                    self.keys[layer, p, position % PAGE] = k[source]
                    self.values[layer, p, position % PAGE] = v[source]
