"""Attention that keeps the weight every cached position was given, against a plain 64-bit statement."""
import pytest
import torch

import plain_cache as plain

pytestmark = pytest.mark.gpu
PAGE = 64
BF, F = torch.bfloat16, torch.float32


def build(ctx, qlen, H, G, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    B = len(ctx)
    most = max(1, max(-(-(c + n) // PAGE) for c, n in zip(ctx, qlen)))
    ids = torch.randperm(B * most + 1, generator=g).to(torch.int32)
    table = ids[:-1].view(B, most).clone()
    k, v = (torch.full((B * most + 1, G, PAGE, D), float("nan")) for _ in range(2))
    for b in range(B):
        for j in range(ctx[b] + qlen[b]):
            for t in (k, v):
                t[int(table[b, j // PAGE]), :, j % PAGE] = torch.randn(G, D, generator=g)
    sums = torch.full((B * most + 1, G, PAGE), float("nan"))
    for b in range(B):
        for j in range(ctx[b]):                                    # (what is not cached yet has no sum yet)
            sums[int(table[b, j // PAGE]), :, j % PAGE] = torch.rand(G, generator=g)
    q = torch.randn(sum(qlen), H * D, generator=g) * (2 * D ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return (q.to(dtype).cuda(), k.to(dtype).cuda(), v.to(dtype).cuda(), sums.cuda(), i32([sum(qlen[:b]) for b in range(B)]), i32(qlen), i32(ctx), table.cuda())


def check(out, sums, before, q, k, v, start, qlen, ctx, table, H, G, D, last=0):
    touched = torch.zeros(sums.shape, dtype=torch.bool, device="cuda")
    for b in range(len(ctx)):
        T, c, at = int(qlen[b]), int(ctx[b]), int(start[b])
        if T == 0:
            continue
        n = c + T
        want, p, A, S = plain.attention(q[at:at + T].double().view(T, H, D), plain.rows(k, table[b], n), plain.rows(v, table[b], n), c)
        off = (out[at:at + T].double().view(T, H, D) - want).abs()
        assert (off <= plain.out_bound(q.dtype, want, A, D, n, S)).all(), (b, float(off.max()))
        counted = p[-last:] if last else p
        given = counted.sum(0).view(G, H // G, n).sum(1)                                   # [G, n]
        page, slot = table[b].long()[torch.arange(n, device="cuda") // PAGE], torch.arange(n, device="cuda") % PAGE
        had = torch.where(torch.arange(n, device="cuda")[:, None] < c, before[page, :, slot].double(), 0.0).T
        off = (sums[page, :, slot].double().T - had - given).abs()
        assert (off <= plain.sums_bound(had, given, counted.shape[0] * H // G, D, S)).all(), (b, float(off.max()))
        touched[page, :, slot] = True
    same = (sums == before) | (torch.isnan(sums) & torch.isnan(before))
    assert (same | touched).all()                                  # nothing else moved


def call(s, H, G, D, max_qlen, max_len, last=0):
    from gopherllm_b200 import ops
    q, k, v, sums, start, qlen, ctx, table = s
    out = torch.full_like(q, float("nan"))
    now = sums.clone()
    ops.attention_weighed(q, out, k, v, now, start, qlen, ctx, table, H, G, D, max_qlen, max_len, last)
    return out, now


HEADS = [(BF, 4, 4, 16), (BF, 4, 2, 64), (BF, 5, 5, 80), (BF, 8, 2, 128), (BF, 16, 1, 64), (BF, 40, 1, 32), (BF, 4, 2, 256),
         (F, 4, 4, 64), (F, 4, 1, 50), (F, 20, 2, 36), (F, 2, 2, 256), (F, 3, 1, 1)]


@pytest.mark.parametrize("dtype,H,G,D", HEADS)
@pytest.mark.parametrize("ctx", [[0], [63, 0, 64, 500, 1, 130], [2000, 127]])
def test_one_token(dtype, H, G, D, ctx):
    s = build(ctx, [1] * len(ctx), H, G, D, dtype, 1)
    out, now = call(s, H, G, D, 1, max(ctx) + 1)
    check(out, now, s[3], *s[:3], *s[4:], H, G, D)


@pytest.mark.parametrize("dtype,H,G,D", HEADS)
@pytest.mark.parametrize("ctx,qlen,last", [([0], [2], 0), ([0, 100, 63], [70, 1, 65], 0), ([10, 200], [130, 33], 0), ([0, 64, 5], [150, 20, 3], 16), ([0, 90], [129, 64], 1000)])
def test_runs(dtype, H, G, D, ctx, qlen, last):
    s = build(ctx, qlen, H, G, D, dtype, 2)
    out, now = call(s, H, G, D, max(qlen), max(c + n for c, n in zip(ctx, qlen)), last)
    check(out, now, s[3], *s[:3], *s[4:], H, G, D, last)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("qlen", [[1, 0, 1], [0, 40, 3]])
def test_a_sequence_without_tokens_leaves_everything_as_it_is(dtype, qlen):
    s = build([70, 20, 5], qlen, 4, 2, 64, dtype, 3)
    out, now = call(s, 4, 2, 64, max(qlen), 80)
    check(out, now, s[3], *s[:3], *s[4:], 4, 2, 64)


@pytest.mark.parametrize("dtype", [BF, F])
def test_token_after_token_is_the_run(dtype):
    """A prompt, then tokens one at a time, sum up to what the whole run sums up to; and the sum over the positions is the number of queries."""
    from gopherllm_b200 import ops
    H, G, D, n, T = 8, 2, 64, 90, 12
    q, k, v, sums, start, qlen, ctx, table = build([0], [n + T], H, G, D, dtype, 4)
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    whole, steps = sums.clone(), sums.clone()
    out = torch.empty_like(q)
    ops.attention_weighed(q, out, k, v, whole, start, qlen, ctx, table, H, G, D, n + T, n + T)
    part = torch.empty_like(q[:n])
    ops.attention_weighed(q[:n].contiguous(), part, k, v, steps, start, i32(n), ctx, table, H, G, D, n, n)
    for t in range(n, n + T):
        one = torch.empty_like(q[:1])
        ops.attention_weighed(q[t:t + 1].contiguous(), one, k, v, steps, i32(0), i32(1), i32(t), table, H, G, D, 1, n + T)
    a, b = (x[table[0].long()].transpose(0, 1).reshape(G, -1)[:, :n + T].double() for x in (whole, steps))
    given = (n + T) * H // G
    e = 2 * (plain.weight_error(D, 40.0) + given * 2 ** -23)
    assert ((a - b).abs() <= e * a + T * 2 ** -24 * a).all()
    assert ((a.sum(-1) - given).abs() <= e * given).all()


@pytest.mark.parametrize("dtype", [BF, F])
def test_captured_and_replayed(dtype):
    from gopherllm_b200 import ops
    H, G, D = 4, 2, 64
    q, k, v, sums, start, qlen, ctx, table = s = build([300, 64], [1, 1], H, G, D, dtype, 5)
    want, now = call(s, H, G, D, 1, 320)
    live, out, at = sums.clone(), torch.empty_like(q), torch.zeros_like(ctx)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.attention_weighed(q, out, k, v, live, start, qlen, at, table, H, G, D, 1, 320)
    at.copy_(ctx)
    graph.replay()
    assert torch.equal(out, want)
    assert torch.equal(torch.nan_to_num(live), torch.nan_to_num(now))


def test_refusals():
    from gopherllm_b200 import ops
    q, k, v, sums, start, qlen, ctx, table = build([5, 9], [1, 1], 4, 2, 64, BF, 1)
    out = torch.empty_like(q)
    good = [q, out, k, v, sums, start, qlen, ctx, table, 4, 2, 64, 1, 10, 0]
    ops.attention_weighed(*good)
    for i, x in ((0, q.float()), (1, out[:1]), (2, k.float()), (3, v[:1]), (4, sums.double()), (4, sums[:, :1].contiguous()), (5, start.long()), (6, qlen[:1]),
                 (7, ctx.cpu()), (8, table.t()), (9, 3), (10, 3), (11, 32), (12, -1), (13, 0), (13, 65), (14, -1), (4, sums.cpu())):
        with pytest.raises(ops.KernelError):
            ops.attention_weighed(*good[:i], x, *good[i + 1:])


@pytest.mark.parametrize("dtype,H,G,D", [(BF, 4, 2, 64), (BF, 2, 2, 128), (BF, 40, 1, 32), (BF, 4, 2, 256), (F, 4, 4, 64), (F, 4, 1, 50), (F, 20, 2, 36)])
@pytest.mark.parametrize("ctx,qlen,last", [([200, 150, 128, 190, 700], [1] * 5, 0), ([128, 131, 300, 192, 129], [1, 140, 0, 40, 3], 0), ([128, 131, 300, 192, 129], [1, 140, 70, 40, 3], 2),
                                           ([5000, 5100], [1, 1], 0)])
def test_sequences_on_common_pages(dtype, H, G, D, ctx, qlen, last):
    """Every other sequence lies on the same first two pages: a position there is given what all of them give it, the same in every run."""
    from gopherllm_b200 import ops
    s = build(ctx, qlen, H, G, D, dtype, 7)
    q, k, v, sums, start, qlens, ctxs, table = s
    for b in range(2, len(ctx)):
        table[b, :2] = table[b % 2, :2]
    if len(ctx) == 2:
        table[1, :2] = table[0, :2]
    outs = []
    for _ in range(3):
        out, now = torch.full_like(q, float("nan")), sums.clone()
        ops.attention_weighed(q, out, k, v, now, start, qlens, ctxs, table, H, G, D, max(qlen), max(c + n for c, n in zip(ctx, qlen)), last, shared=True)
        outs.append((out, now))
    assert all(torch.equal(x, outs[0][0]) and torch.equal(y.nan_to_num(-1.0), outs[0][1].nan_to_num(-1.0)) for x, y in outs)
    out, now = outs[0]
    given, terms, most = torch.zeros_like(sums, dtype=torch.float64), torch.zeros_like(sums, dtype=torch.float64), 0.0
    had, touched = sums.double().clone(), torch.zeros_like(sums, dtype=torch.bool)
    for b in range(len(ctx)):
        if not qlen[b]:
            continue
        at, T, n = sum(qlen[:b]), qlen[b], ctx[b] + qlen[b]
        want, p, A, S = plain.attention(q[at:at + T].double().view(T, H, D), plain.rows(k, table[b], n), plain.rows(v, table[b], n), ctx[b])
        assert ((out[at:at + T].double().view(T, H, D) - want).abs() <= plain.out_bound(dtype, want, A, D, n, S)).all()
        j = torch.arange(n, device="cuda")
        page, slot = table[b].long()[j // PAGE], j % PAGE
        p = p[-last:] if last else p
        given[page, :, slot] += p.sum(0).view(G, H // G, n).sum(1).T
        terms[page, :, slot] += p.shape[0] * H // G
        new = j >= ctx[b]
        had[page[new], :, slot[new]] = 0.0
        touched[page, :, slot] = True
        most = max(most, S)
    off = (now.double() - had - given).abs()
    assert (off <= plain.sums_bound(had, given, terms + len(ctx), D, most))[touched].all(), float(off[touched].max())
    same = (now == sums) | (torch.isnan(now) & torch.isnan(sums))
    assert (same | touched).all()
