"""Plain 64-bit forms of the paged-cache and prompt operators on the CPU, and the bounds their results are held to.

Bounds.  u(t): a rounding to type t is off by at most eps / 2 of the value.  The kernels may round each softmax weight
once to 16 bits (u(f16) in the paged attention, u of the input type in the prompt attention) before the products with V,
which sum in fp32; a logit that is off by delta makes every weight off by at most 2 delta of itself (numerator and sum),
to first order.  So
  |out - ref| <= u(out) |ref| + (u(weight) + 2 delta + (n + 16) 2^-24) * sum_j p_j |V_j|        (+ the smallest number)
where for the paged attention the sum is in the rotated domain, brought back by the worst case of the rotation:
c sum_e sum_j p_j s_j |codes_je|.
"""
from __future__ import annotations

import math

import numpy as np
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def signs(d):
    g = torch.Generator().manual_seed(42 * 10007 + d)
    return torch.where(torch.rand(d, generator=g) > 0.5, 1.0, -1.0).double()


def hadamard(d):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.size(0) < d:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)])
    return h


def values(codes, bits):
    if bits == 8:
        return codes.double()
    c = codes.to(torch.int64)
    return torch.stack([((c & 15) ^ 8) - 8, ((c >> 4) ^ 8) - 8], -1).flatten(-2).double()


class HostCache:
    """CPU copies of a pool, with its slots read one sequence and head at a time."""

    def __init__(self, cache, table):
        self.bits, self.dim, self.page = cache.bits, cache.dim, cache.page_size
        self.k = (cache.k_codes.cpu(), cache.k_scale.cpu())
        self.v = (cache.v_codes.cpu(), cache.v_scale.cpu())
        self.table, self.pages = table.cpu().long(), cache.pages

    def rows(self, b, head, n):
        """(slots in use, rotated K, rotated V) of the first n slots; bad pages are left out."""
        slot = torch.arange(max(0, min(n, self.table.size(1) * self.page)))
        page = self.table[b][slot // self.page]
        slot = slot[(page >= 0) & (page < self.pages)]
        page, row = self.table[b][slot // self.page], slot % self.page
        return slot, *(values(c[page, head, row], self.bits) * s[page, head, row].double()[:, None] for c, s in (self.k, self.v))


def paged_attention_ref(host, q, lengths, scale, sink=None, capacity=None):
    """(out, bound, weights added, their bound) for q [B, T, H, D]; weights [B, heads, capacity]."""
    B, T, H, D = q.shape
    heads = host.k[1].size(1)
    g, c = H // heads, D ** -0.5
    had, sg = hadamard(D), signs(D)
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    cap = capacity if capacity is not None else 0
    w = torch.zeros(B, heads, cap, dtype=torch.float64)
    wb = torch.zeros_like(w)
    for b in range(B):
        for kh in range(heads):
            n = int(lengths[b]) if capacity is None else min(int(lengths[b]), capacity)
            n = min(n, host.table.size(1) * host.page)
            slot, k, v = host.rows(b, kh, n)
            for h in range(kh * g, kh * g + g):
                for t in range(T):
                    vis = slot < n - T + 1 + t
                    kk, vv, sl = k[vis], v[vis], slot[vis]
                    qd = q[b, t, h].double()
                    rq = (qd * sg) @ had * c
                    logit = kk @ rq * scale
                    if sl.numel() == 0:
                        continue
                    sk = -math.inf if sink is None else float(sink[h])
                    m = max(float(logit.max()), sk)
                    e = torch.exp(logit - m)
                    p = e / (e.sum() + (math.exp(sk - m) if sk > -math.inf else 0.0))
                    out[b, t, h] = ((p @ vv) @ had * c) * sg
                    # the query is rotated in fp32 (7 stages and a product) and split into two 11-bit parts of its largest
                    dq = rq.abs().max() * 2.0 ** -21 + 2.0 ** -21 * c * qd.abs().sum()
                    delta = abs(scale) * (kk.abs().sum(1) * dq + (kk.abs() @ rq.abs()) * (D + 8) * 2.0 ** -24) + logit.abs() * 2.0 ** -21
                    rel = U[torch.float16] + 2 * delta.max() + (sl.numel() + 16) * 2.0 ** -24
                    bound[b, t, h] = U[q.dtype] * out[b, t, h].abs() + rel * c * (p @ vv.abs()).sum() + TINY[q.dtype]
                    if cap:
                        w[b, kh, sl] += p
                        wb[b, kh, sl] += p * (delta + delta.max() + (sl.numel() + 16) * 2.0 ** -24)
    return out, bound, w, wb + 2.0 ** -23 * T * g * w


def prompt_attention_ref(q, k, v, cu_q, cu_k, scale, sink=None):
    """(out, bound, lse, its bound); rows in no sequence: 0 and -inf."""
    N, H, D = q.shape
    g = H // k.size(1)
    out = torch.zeros(N, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((N, H), -math.inf, dtype=torch.float64)
    lb = torch.zeros(N, H, dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        lq, lk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        for h in range(H):
            kk, vv = k[cu_k[b]:cu_k[b + 1], h // g].double(), v[cu_k[b]:cu_k[b + 1], h // g].double()
            for i in range(lq):
                n = max(0, i + 1 + lk - lq)
                sk = -math.inf if sink is None else float(sink[h])
                r = cu_q[b] + i
                if n == 0:
                    # the sink in units of log2 and back: two products and the rounding of both constants, 4 2^-24 of it
                    lse[r, h], lb[r, h] = sk, 2.0 ** -22 * abs(sk) if sk > -math.inf else 0.0
                    continue
                qd = q[r, h].double()
                logit = kk[:n] @ qd * scale
                m = max(float(logit.max()), sk)
                e = torch.exp(logit - m)
                z = e.sum() + (math.exp(sk - m) if sk > -math.inf else 0.0)
                p = e / z
                out[r, h] = p @ vv[:n]
                delta = float((abs(scale) * (kk[:n].abs() @ qd.abs()) * (D + 8) * 2.0 ** -24 + logit.abs() * 2.0 ** -21).max())
                rel = U[q.dtype] + 2 * delta + (n + 16) * 2.0 ** -24
                bound[r, h] = U[q.dtype] * out[r, h].abs() + rel * (p @ vv[:n].abs()) + TINY[q.dtype]
                lse[r, h] = m + torch.log(z)
                lb[r, h] = 2 * delta + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * (1 + abs(m))
    return out, bound, lse, lb


def evict_ref(weights, tokens, n, seen, keep, first, recent):
    """[(source, destination)] of one row, by a full sort."""
    if n <= keep:
        return []
    held = lambda i: tokens[i] < first or tokens[i] >= seen - recent  # noqa: E731
    rank = sorted(range(n), key=lambda i: (0, 0.0, i) if held(i) else (1, 0.0, i) if math.isnan(weights[i]) else (2, -weights[i], i))
    stay = set(rank[:keep])
    holes = [i for i in range(keep) if i not in stay]
    return list(zip(sorted(i for i in stay if i >= keep), holes))


def within(got, want, bound, what):
    d = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    over = d > bound
    assert not over.any(), f"{what}: {int(over.sum())} of {over.numel()} beyond the bound, worst {float((d / bound.clamp(min=1e-300)).max()):.3g} times it, at {np.unravel_index(int((d - bound).argmax()), tuple(d.shape))}"
