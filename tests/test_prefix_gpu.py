"""Attention of one token a sequence behind shared pages, against a plain 64-bit statement."""
import pytest
import torch

import plain_cache as plain

pytestmark = pytest.mark.gpu
PAGE = 64
BF, F = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def shared_however_little(monkeypatch):
    from gopherllm_b200 import ops
    monkeypatch.setattr(ops, "PREFIX_SPARED_BYTES", 0)


def build(groups, ctx, H, G, D, dtype, seed, spare=3):
    """Pages in a random order, NaN wherever no position was written; (q, keys, values, seq_ctx, table)."""
    g = torch.Generator().manual_seed(seed)
    B = len(ctx)
    shared = [0] * B
    for members, n in groups:
        for b in members:
            shared[b] = n
    own = [max(0, c // PAGE + 1 - s // PAGE) for c, s in zip(ctx, shared)]
    total = sum(own) + sum(n // PAGE for _, n in groups) + spare
    ids = torch.randperm(total, generator=g).to(torch.int32)
    bad = ids[-1]                                                  # nothing lies there
    table = torch.full((B, max(s // PAGE + o for s, o in zip(shared, own)) + 1), int(bad), dtype=torch.int32)
    k, v = (torch.full((total, G, PAGE, D), float("nan")) for _ in range(2))
    at = 0
    for members, n in groups:
        table[members, :n // PAGE] = ids[at:at + n // PAGE]
        for t in (k, v):
            t[ids[at:at + n // PAGE].long()] = torch.randn(n // PAGE, G, PAGE, D, generator=g)
        at += n // PAGE
    for b in range(B):
        table[b, shared[b] // PAGE:shared[b] // PAGE + own[b]] = ids[at:at + own[b]]
        at += own[b]
        for j in range(shared[b], ctx[b] + 1):
            for t in (k, v):
                t[int(table[b, j // PAGE]), :, j % PAGE] = torch.randn(G, D, generator=g)
    q = torch.randn(B, H * D, generator=g) * (2 * D ** -0.5)
    return q.to(dtype).cuda(), k.to(dtype).cuda(), v.to(dtype).cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), table.cuda()


def check(out, q, k, v, ctx, table, H, G, D):
    for b, c in enumerate(ctx.tolist()):
        want, _, A, S = plain.attention(q[b].double().view(1, H, D), plain.rows(k, table[b], c + 1), plain.rows(v, table[b], c + 1), c)
        off = (out[b].double().view(1, H, D) - want).abs()
        assert (off <= plain.out_bound(q.dtype, want, A, D, c + 1, S)).all(), (b, float(off.max()))


HEADS = [(BF, 4, 4, 16), (BF, 4, 2, 64), (BF, 5, 5, 80), (BF, 8, 2, 128), (BF, 16, 1, 64), (BF, 40, 1, 32), (BF, 4, 2, 256), (BF, 6, 2, 48),
         (F, 4, 4, 64), (F, 4, 1, 50), (F, 20, 2, 36), (F, 2, 2, 256), (F, 3, 1, 1)]


@pytest.mark.parametrize("dtype,H,G,D", HEADS)
def test_groups_of_unequal_sequences(dtype, H, G, D):
    """Two groups out of order, one of a single member, a sequence of none; lengths that end at a page's first, last and middle place."""
    from gopherllm_b200 import ops
    groups = [([6, 0, 3], 192), ([2, 5], 64), ([4], 320)]
    ctx = [192, 30, 64 + 63, 192 + 130, 320 + 1, 64 + 64, 192 + 63, 0]
    q, k, v, c, table = build(groups, ctx, H, G, D, dtype, 3)
    out = torch.full_like(q, float("nan"))
    plan = ops.prefix_plan(groups, len(ctx), H, G, D, dtype, 131, "cuda")
    ops.attention_prefix(q, out, k, v, c, table, plan, H, G, D)
    check(out, q, k, v, c, table, H, G, D)


@pytest.mark.parametrize("dtype,H,G,D,members,shared", [(BF, 4, 4, 64, 70, 640), (BF, 8, 2, 128, 45, 1344), (BF, 4, 2, 32, 150, 128), (F, 4, 4, 64, 21, 256), (BF, 16, 2, 256, 9, 192)])
def test_many_members(dtype, H, G, D, members, shared):
    """More rows than one block takes, a number of them that does not divide, pages that do not divide among the blocks."""
    from gopherllm_b200 import ops
    groups = [(list(range(members))[::-1], shared)]
    ctx = [shared + (7 * b) % 90 for b in range(members)]
    q, k, v, c, table = build(groups, ctx, H, G, D, dtype, 4)
    out = torch.full_like(q, float("nan"))
    ops.attention_prefix(q, out, k, v, c, table, ops.prefix_plan(groups, members, H, G, D, dtype, 90, "cuda"), H, G, D)
    check(out, q, k, v, c, table, H, G, D)


def test_nothing_shared_and_nothing_of_its_own():
    """A plan without groups is attention as ever; a sequence whose newest position ends its shared pages has nothing of its own."""
    from gopherllm_b200 import ops
    for groups, ctx in (([], [5, 64, 200]), ([([0, 1, 2], 128)], [127, 127, 140])):
        q, k, v, c, table = build(groups, ctx, 4, 2, 64, BF, 5)
        out = torch.full_like(q, float("nan"))
        ops.attention_prefix(q, out, k, v, c, table, ops.prefix_plan(groups, 3, 4, 2, 64, BF, 201, "cuda"), 4, 2, 64)
        check(out, q, k, v, c, table, 4, 2, 64)


@pytest.mark.parametrize("dtype", [BF, F])
def test_a_plan_serves_longer_sequences_and_a_captured_call_later_steps(dtype):
    """The plan was made for one page of their own; captured, the call reads the lengths that stand there when it is replayed."""
    from gopherllm_b200 import ops
    H, G, D, groups = 4, 2, 64, [([0, 2], 128), ([1, 3], 64)]
    late = [128 + 300, 64 + 7, 128 + 64, 64 + 200]
    q, k, v, c, table = build(groups, late, H, G, D, dtype, 6)
    plan = ops.prefix_plan(groups, 4, H, G, D, dtype, 1, "cuda")
    out = torch.full_like(q, float("nan"))
    early = torch.tensor([128, 64, 128 + 63, 64 + 64], dtype=torch.int32, device="cuda")
    now = early.clone()
    ops.attention_prefix(q, out, k, v, now, table, plan, H, G, D)
    check(out, q, k, v, early, table, H, G, D)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.attention_prefix(q, out, k, v, now, table, plan, H, G, D)
    now.copy_(c)
    graph.replay()
    check(out, q, k, v, c, table, H, G, D)
    now.copy_(early)
    graph.replay()
    assert torch.equal(out, first)                                 # the same call, the same numbers


def test_two_streams_at_once():
    """Calls on two streams have scratch of their own."""
    from gopherllm_b200 import ops
    H, G, D, groups = 8, 8, 64, [(list(range(20)), 512)]
    sets = [build(groups, [512 + b for b in range(20)], H, G, D, BF, s) for s in (7, 8)]
    plan = ops.prefix_plan(groups, 20, H, G, D, BF, 20, "cuda")
    alone = []
    for q, k, v, c, t in sets:
        o = torch.empty_like(q)
        ops.attention_prefix(q, o, k, v, c, t, plan, H, G, D)
        alone.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.empty_like(sets[0][0]) for _ in range(2)]
    for _ in range(20):
        for s, (q, k, v, c, t), o in zip(streams, sets, outs):
            with torch.cuda.stream(s):
                ops.attention_prefix(q, o, k, v, c, t, plan, H, G, D)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))


def test_a_nan_key_shows_in_the_rows_that_see_it_and_in_no_other():
    from gopherllm_b200 import ops
    H, G, D, groups = 4, 2, 64, [([0, 1], 128), ([2, 3], 128)]
    for dtype in (BF, F):
        q, k, v, c, table = build(groups, [128, 150, 128, 150], H, G, D, dtype, 9)
        k[int(table[2, 1]), 0, 5, 3] = float("nan")                # shared by sequences 2 and 3, key head 0
        out = torch.empty_like(q)
        ops.attention_prefix(q, out, k, v, c, table, ops.prefix_plan(groups, 4, H, G, D, dtype, 23, "cuda"), H, G, D)
        nan = torch.isnan(out.view(4, H, D)).all(-1).cpu()
        assert torch.isnan(out).sum() == nan.sum() * D
        assert nan.tolist() == [[False] * 4, [False] * 4, [True, True, False, False], [True, True, False, False]]


def test_a_call_on_a_device_tensor_of_another_type_is_refused():
    from gopherllm_b200 import ops
    q, k, v, c, table = build([([0, 1], 64)], [64, 65], 4, 2, 64, BF, 1)
    plan = ops.prefix_plan([([0, 1], 64)], 2, 4, 2, 64, BF, 2, "cuda")
    out = torch.empty_like(q)
    for args in ((q.float(), out, k, v, c, table), (q, out.float(), k, v, c, table), (q, out, k.float(), v, c, table), (q, out, k, v, c.long(), table),
                 (q, out, k, v, c, table[:1].contiguous()), (q, out, k, v, c, table.t()), (q.half(), out.half(), k.half(), v.half(), c, table)):
        with pytest.raises(ops.KernelError):
            ops.attention_prefix(*args, plan, 4, 2, 64)
    with pytest.raises(ops.KernelError):
        ops.attention_prefix(q, out, k, v, c, table, ops.prefix_plan([], 2, 4, 4, 64, BF, 2, "cuda"), 4, 2, 64)


@pytest.mark.parametrize("dtype", [BF, F])
def test_pages_not_worth_a_kernel_are_read_by_each(dtype, monkeypatch):
    from gopherllm_b200 import ops
    monkeypatch.setattr(ops, "PREFIX_SPARED_BYTES", 1 << 40)
    H, G, D, groups = 4, 2, 64, [([0, 2], 640), ([1], 64)]
    q, k, v, c, table = build(groups, [640 + 70, 64 + 7, 640], H, G, D, dtype, 12)
    plan = ops.prefix_plan(groups, 3, H, G, D, dtype, 71, "cuda")
    assert plan.layout.n_items == 0 and plan.layout.launches == 1
    out = torch.full_like(q, float("nan"))
    ops.attention_prefix(q, out, k, v, c, table, plan, H, G, D)
    check(out, q, k, v, c, table, H, G, D)


@pytest.mark.parametrize("dtype,H,G,D,members", [(BF, 4, 4, 64, 40), (BF, 8, 1, 128, 40), (BF, 4, 2, 64, 3), (F, 4, 2, 64, 6)])
@pytest.mark.parametrize("rise", [30.0, -30.0])
def test_scores_that_rise_or_fall_from_page_to_page(dtype, H, G, D, members, rise):
    """Each page's scores lie e^+-30 and more above the page's before: every page of a span has its own maximum to deal with, and all but the
    largest few weights vanish."""
    from gopherllm_b200 import ops
    groups = [(list(range(members)), 64 * 7)]
    q, k, v, c, table = build(groups, [64 * 7 + b % 70 for b in range(members)], H, G, D, dtype, 13)
    with torch.no_grad():
        q.view(members, H, D)[..., 0] = 1.0
        for p in range(table.shape[1]):
            k[table[0, p].long(), :, :, 0] += rise * p
    out = torch.full_like(q, float("nan"))
    ops.attention_prefix(q, out, k, v, c, table, ops.prefix_plan(groups, members, H, G, D, dtype, 70, "cuda"), H, G, D)
    check(out, q, k, v, c, table, H, G, D)
