"""Plain 64-bit forms on the CPU of rotary positions, attention over an encoder's states and a pool's pages, and the bounds
their results are held to.

Attention, as in paged_ref: a weight is rounded once to the input's type, a logit that is off by delta makes every weight off by
at most 2 delta of itself, and sums are fp32:
  |out - ref| <= u |ref| + (u + 2 delta + (n + 16) 2^-24) sum_j p_j |v_j|        (+ the smallest number)
Rotary: the angle, brought to [-pi, pi], is rounded to fp32 (2^-23), its cosine and sine are off by two units of the last place
at most (2^-23), each product and the sum by 2^-24 of its size:
  |y - ref| <= u |ref| + (|x1| + |x2|) 2^-21                                     (+ the smallest number)
"""
from __future__ import annotations

import math

import torch

from paged_ref import TINY, U


def cross_attention_ref(q, k, v, cu_q, cu_k, states, scale, sink=None):
    """(out, bound, lse, its bound); rows in no sequence: 0 and -inf."""
    N, H, D = q.shape
    g = H // k.size(1)
    out = torch.zeros(N, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((N, H), -math.inf, dtype=torch.float64)
    lb = torch.zeros(N, H, dtype=torch.float64)
    E = len(cu_k) - 1
    for b in range(len(cu_q) - 1):
        e = b if states is None else states[b]
        rows = slice(cu_q[b], cu_q[b + 1])
        keys = slice(cu_k[e], cu_k[e + 1]) if 0 <= e < E else slice(0, 0)
        n = keys.stop - keys.start
        for h in range(H):
            sk = -math.inf if sink is None else float(sink[h])
            if n == 0:
                # the sink in units of log2 and back: two products and the rounding of both constants, 4 2^-24 of it
                lse[rows, h], lb[rows, h] = sk, 2.0 ** -22 * abs(sk) if sk > -math.inf else 0.0
                continue
            kk, vv, qq = k[keys, h // g].double(), v[keys, h // g].double(), q[rows, h].double()
            logit = qq @ kk.T * scale
            m = logit.amax(1, keepdim=True).clamp(min=sk)
            w = torch.exp(logit - m)
            z = w.sum(1, keepdim=True) + (torch.exp(sk - m) if sk > -math.inf else 0.0)
            p = w / z
            out[rows, h] = p @ vv
            delta = (abs(scale) * (qq.abs() @ kk.abs().T) * (D + 8) * 2.0 ** -24 + logit.abs() * 2.0 ** -21).amax(1, keepdim=True)
            rel = U[q.dtype] + 2 * delta + (n + 16) * 2.0 ** -24
            bound[rows, h] = U[q.dtype] * out[rows, h].abs() + rel * (p @ vv.abs()) + TINY[q.dtype]
            lse[rows, h] = (m + torch.log(z))[:, 0]
            lb[rows, h] = (2 * delta + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * (1 + m.abs()))[:, 0]
    return out, bound, lse, lb


def rotate_ref(x, positions, freq, axis, first, halves, inverse=False):
    """(y, bound) for x [N, H, D], positions [axes, N]."""
    R = len(axis)
    y, bound = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    tiny = TINY.get(x.dtype, 2.0 ** -149)
    for i in range(R):
        a, b = (first + i, first + R + i) if halves else (first + 2 * i, first + 2 * i + 1)
        t = positions[axis[i]].double() * float(freq[i]) * (-1 if inverse else 1)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        x1, x2 = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
        for d in (a, b):
            bound[..., d] = U[x.dtype] * y[..., d].abs() + (x1.abs() + x2.abs()) * 2.0 ** -21 + tiny
    return y, bound


class PoolRef:
    """Tables and counts as lists; what happens to bytes as a list of (from, to) pages, in order."""

    def __init__(self, refs, size):
        self.refs, self.size, self.lacking, self.copies = list(refs), size, 0, []

    def has(self, p):
        return 0 <= p < len(self.refs)

    def pages(self, n, width):
        return min(max(0, -(-n // self.size)), width)

    def reserve(self, table, filled, wanted, first=None):
        first = filled if first is None else first
        entries = [(b, i) for b in range(len(table)) if wanted[b] > max(first[b], 0) for i in range(max(first[b], 0) // self.size, self.pages(wanted[b], len(table[b])))]
        holders = {}
        for b, i in entries:
            if self.has(table[b][i]) and self.refs[table[b][i]] > 1:
                holders.setdefault(table[b][i], []).append((b, i))
        keeps = {w[-1] for p, w in holders.items() if len(w) == self.refs[p]}
        unused = [p for p in range(len(self.refs)) if self.refs[p] <= 0]
        for b, i in entries:
            p = table[b][i]
            if self.has(p) and ((b, i) in keeps or p not in holders):
                continue
            to = unused.pop(0) if unused else -1
            self.lacking += to < 0
            if self.has(p):
                self.refs[p] -= 1
            table[b][i] = to
            if to >= 0:
                self.refs[to] = 1
                if self.has(p) and i * self.size < filled[b]:
                    self.copies.append((p, to))

    def release(self, table, keep):
        for b, row in enumerate(table):
            for i in range(self.pages(keep[b], len(row)), len(row)):
                if self.has(row[i]):
                    self.refs[row[i]] -= 1
                row[i] = -1

    def fork(self, table, filled, source, target):
        old = [list(r) for r in table]
        ok = [j for j in range(len(source)) if 0 <= source[j] < len(table) and 0 <= target[j] < len(table)]
        for j in ok:
            if j != max(i for i in ok if target[i] == target[j]) or source[j] == target[j]:
                continue
            row = table[target[j]]
            n = self.pages(filled[source[j]], len(row))
            for i in range(len(row)):
                now = old[source[j]][i] if i < n else -1
                if self.has(row[i]):
                    self.refs[row[i]] -= 1
                if self.has(now):
                    self.refs[now] += 1
                row[i] = now

    def compact(self, *tables):
        n = sum(r > 0 for r in self.refs)
        holes = [p for p in range(n) if self.refs[p] <= 0]
        movers = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        to = {p: -1 for p in range(n, len(self.refs))}
        for p, q in zip(movers, holes):
            self.copies.append((p, q))
            self.refs[q], self.refs[p] = self.refs[p], 0
            to[p] = q
        for t in tables:
            for row in t:
                row[:] = [to.get(p, p) if self.has(p) else p for p in row]
