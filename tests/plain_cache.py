"""Plain 64-bit statements of attention over a paged cache, of the weight it gives each position, and of eviction; and the bounds
that the kernels' results are held to.

Bounds.  Scores are sums of D products in 32 bits (tensor cores may cut an addition short by a whole step, 2^-23 of the sum):
off by at most (D + 8) 2^-22 S, S the largest sum of |q_d k_d|; a softmax weight then by twice that relative to itself, and by a few
steps for its power.  A result is a sum of up to L such weights times values, in 32 bits: L 2^-23 of A = sum p |v| more.  In
bfloat16 each weight is rounded for the second product, half a step, 2^-8 of itself, and the result once more, 2^-8."""
import torch

PAGE = 64


def rows(cache, table, n):
    """The first n positions of one sequence, [n, heads, size] in 64 bits."""
    ids = table[:-(-n // PAGE)].long()
    return cache[ids].double().transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:n]


def attention(q, k, v, first):
    """q [T, H, D] at positions first..first + T - 1; k, v [n, G, D], all 64 bits.  (out [T, H, D], weights [T, H, n], A [T, H, D], S)"""
    T, H, D = q.shape
    n, G, _ = k.shape
    k, v = k.repeat_interleave(H // G, 1), v.repeat_interleave(H // G, 1)
    s = torch.einsum("thd,jhd->thj", q, k)
    S = float(torch.einsum("thd,jhd->thj", q.abs(), k.abs()).max())
    late = torch.arange(n, device=q.device) > torch.arange(first, first + T, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(late[:, None], -float("inf")), -1)
    return torch.einsum("thj,jhd->thd", p, v), p, torch.einsum("thj,jhd->thd", p, v.abs()), S


def weight_error(D, S):
    """Of a softmax weight, relative to itself."""
    return 2 * (D + 8) * 2 ** -22 * max(1.0, S) + 2 ** -20


def out_bound(dtype, want, A, D, L, S):
    e = weight_error(D, S) + L * 2 ** -23
    if dtype == torch.bfloat16:
        return 2 ** -8 * want.abs() + (2 ** -8 + e) * A * (1 + 2 ** -7)
    return 2 ** -24 * want.abs() + e * A


def sums_bound(before, given, terms, D, S):
    """Of a position's sum: ``terms`` weights added up in 32 bits, then added to what was there."""
    return (weight_error(D, S) + (terms + 4) * 2 ** -23) * given + 2 ** -23 * (before.abs() + given) + 1e-30


def evict(sums, n, keep, first, recent):
    """Positions of one head that stay, by sorting (weight falling, position rising); NaN below everything."""
    if n <= keep:
        return list(range(n))
    w = [(-float("inf") if x != x else float(x), 0 if x != x else 1) for x in sums[:n].tolist()]
    between = sorted(range(first, n - recent), key=lambda j: (-w[j][0], -w[j][1], j))
    return sorted(list(range(first)) + between[:keep - first - recent] + list(range(n - recent, n)))
