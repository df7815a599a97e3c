"""Operators over a key / value cache in 64 bits on the CPU, from their
definitions (test infrastructure, as ops.py). Beside each result come the
quantities its rounding error is bounded by."""

import torch

from .ops import EPS


def _sigma(s):
    # 0.5 (s / (|s| + 1) + 1), written without cancellation for s < 0
    r = 1.0 / (s.abs() + 1.0)
    return torch.where(s < 0, 0.5 * r, 1.0 - 0.5 * r)


U32 = 2.0 ** -24


def _weights(q, k, slope, scale, dist, fused):
    """f of one query q [D] against keys k [n, D] at distances dist [n], and a
    bound on its relative error in 32 bits: with ds the error of the score (a
    D-term product, a scale and a bias), d ln f / ds = 2 / ((|s| + 1)^2 sigma) <= 4;
    plus a reciprocal (1 ulp) and five roundings, each at most 4-fold in f. fused:
    sigma taken as 1 + s r, whose absolute errors of 2 ulp weigh (1 + |s|)-fold."""
    d = q.shape[0]
    s = (k @ q) * scale - slope * dist
    size = (k.abs() @ q.abs()) * abs(scale)
    ds = U32 * ((d + 4) * size + 4 * (slope * dist).abs())
    f = _sigma(s) ** 4
    rel = 4 * ds + 40 * U32 * ((1 + s.abs()) if fused else 1.0)
    return f, rel


def attention_rows(q, k, v, slope, scale, dist, eps=EPS, fused=False):
    """One query over the rows it sees: (o, L, p, A, E): p the attention
    weights, A = sum p |v|, E the largest relative error of an f."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    f, rel = _weights(q, k, float(slope), scale, dist.double().cpu(), fused)
    L = f.sum()
    p = f / (L + eps)
    e = float(rel.max()) if len(rel) else 0.0
    return p @ v, L, p, p @ v.abs(), e + U32 * (len(f) / 4 + 64)


def tree_lines(parents):
    """For every token the tokens from the root to it, or None if it is absent."""
    lines = []
    for i, up in enumerate(parents):
        if up == -1:
            lines.append([i])
        elif 0 <= up < i and lines[up] is not None:
            lines.append(lines[up] + [i])
        else:
            lines.append(None)
    return lines


def key_weights(q, k, slope, scale, L, mask, last, eps=EPS):
    """One (b, h): w [T] and a bound on its absolute error."""
    T = q.shape[0]
    q, k, L = q.double().cpu(), k.double().cpu(), L.double().cpu()
    w, tol = torch.zeros(T, dtype=torch.float64), torch.zeros(T, dtype=torch.float64)
    for i in range(max(0, T - (last or T)), T):
        if mask is not None and not bool(mask[i]):
            continue
        f, rel = _weights(q[i], k[:i + 1], float(slope), scale, (i - torch.arange(i + 1)).double(), True)
        p = f / (L[i] + eps)
        if mask is not None:
            p = torch.where(mask[:i + 1].cpu().bool(), p, torch.zeros_like(p))
            rel = torch.where(mask[:i + 1].cpu().bool(), rel, torch.zeros_like(rel))
        w[:i + 1] += p
        tol[:i + 1] += p * (rel + 4 * U32)
    return w, tol + U32 * (T / 16 + 64) * w


def evict_rows(weights, positions, n, keep, recent):
    """The rows that stay, ascending (lists of one (b, h))."""
    def rank(j):
        if positions[j] > positions[n - 1] - recent:
            return (0, 0.0, j)
        w = weights[j]
        return (1, float("-inf"), j) if w != w else (2, -w, j)
    return sorted(sorted(range(n), key=rank)[:keep])
