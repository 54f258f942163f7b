"""Eviction by accumulated weight against sorting, to the bit: what stays, where it goes, and what is left as it was."""
import pytest
import torch

import plain_cache as plain

pytestmark = pytest.mark.gpu
PAGE = 64
BF, F = torch.bfloat16, torch.float32


def build(lengths, G, D, dtype, layers, fresh, seed, DV=None):
    g = torch.Generator().manual_seed(seed)
    B = len(lengths)
    most = max(1, max(-(-n // PAGE) for n in lengths))
    ids = torch.randperm(B * (most + fresh) + 1, generator=g).to(torch.int32)
    n = ids.numel()
    k = torch.randn(layers, n, G, PAGE, D, generator=g).to(dtype)
    v = torch.randn(layers, n, G, PAGE, DV or D, generator=g).to(dtype)
    sums = torch.rand(layers, n, G, PAGE, generator=g) ** 4
    return (k.cuda(), v.cuda(), sums.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), ids[:B * most].view(B, most).cuda(),
            ids[B * most:B * (most + fresh)].view(B, fresh).cuda() if fresh else None)


def expected(k, v, sums, length, pages, to, keep, recent, first):
    """Everything as it should stand afterwards, position by position."""
    k, v, sums = (t.cpu() for t in (k, v, sums))
    after = [t.clone() for t in (k, v, sums)]
    pages = pages.cpu().long()
    goes = pages if to is None else to.cpu().long()
    layers, _, G = k.shape[:3]
    kept = torch.full((layers, len(length), G, keep), -1, dtype=torch.int32)
    for b, n in enumerate(length.tolist()):
        at = torch.arange(n)
        page, slot = pages[b][at // PAGE], at % PAGE
        for layer in range(layers):
            for h in range(G):
                stay = torch.tensor(plain.evict(sums[layer, page, h, slot], n, keep, first, recent), dtype=torch.long)
                m = len(stay)
                kept[layer, b, h, :m] = stay.int()
                if m:
                    i = torch.arange(m)
                    for t, a in zip((k, v, sums), after):
                        a[layer, goes[b][i // PAGE], h, i % PAGE] = t[layer, page[stay], h, slot[stay]]
    return (kept, *after)


def same(a, b):
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.cpu().contiguous().view(kind), b.cpu().contiguous().view(kind))


def check(s, keep, recent, first, in_place):
    from gopherllm_b200 import ops
    k, v, sums, length, pages, to = s
    want = expected(k, v, sums, length, pages, None if in_place else to, keep, recent, first)
    got = [t.clone() for t in (k, v, sums)]
    kept = ops.cache_evict(*got, length, pages, keep, recent=recent, first=first, to_pages=None if in_place else to)
    assert torch.equal(kept.cpu(), want[0])
    assert all(same(a, b) for a, b in zip(got, want[1:]))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype,G,D,layers", [(BF, 2, 16, 3), (BF, 4, 80, 1), (F, 3, 64, 1), (F, 1, 50, 2), (BF, 2, 7, 1), (BF, 1, 256, 1), (F, 2, 36, 1)])
@pytest.mark.parametrize("lengths,keep,recent,first", [([300, 64, 0, 65, 129, 1], 64, 16, 4), ([200, 130], 100, 0, 0), ([500, 333], 130, 130, 0), ([90], 89, 40, 49), ([70, 400], 1, 0, 0)])
def test_what_stays_and_where(dtype, G, D, layers, lengths, keep, recent, first, in_place):
    check(build(lengths, G, D, dtype, layers, -(-keep // PAGE), 1), keep, recent, first, in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_values_of_another_size(in_place):
    check(build([200, 90], 2, 64, BF, 2, 2, 2, DV=24), 80, 8, 1, in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("fill", ["equal", "few", "zeros", "odd"])
def test_ties_and_numbers_that_are_none(fill, in_place):
    """Equal sums go by position; both zeros are equal; infinities stand at the ends and a NaN below everything."""
    s = build([400, 129, 64], 2, 16, BF, 2, 2, 3)
    sums = s[2]
    if fill == "equal":
        sums.fill_(0.25)
    elif fill == "few":
        sums.copy_((sums * 3).floor())
    elif fill == "zeros":
        sums.copy_(torch.where(sums > 0.3, 0.0, -0.0))
    else:
        g = torch.Generator(device="cuda").manual_seed(1)
        r = torch.randint(0, 7, sums.shape, generator=g, device="cuda")
        values = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 1e-42, -1.5], device="cuda")
        sums.copy_(values[r])
    check(s, 100, 10, 3, in_place)


@pytest.mark.parametrize("lengths,keep", [([5000, 4097], 700), ([4096], 4000), ([50000], 1000), ([33000, 200], 32000)])
def test_long_sequences(lengths, keep):
    """Blocks of either size, and more positions than a block's shared memory holds."""
    s = build(lengths, 1, 16, BF, 1, -(-keep // PAGE), 4)
    for in_place in (True, False):
        check(s, keep, keep // 4, 4, in_place)


@pytest.mark.parametrize("lengths,keep", [([4500], 4544), ([5000, 0, 4999, 70], 6000), ([52000, 300, 51300], 51300)])
@pytest.mark.parametrize("G", [1, 2])
def test_short_sequences_of_long_tables_are_copied_whole(lengths, keep, G):
    """Tables beyond 4,096 positions and a list of what stays that shared memory does not hold: several blocks copy a head's rows, and each
    must know all of them.  Ten times, as what another block has not written yet shows only now and then."""
    s = build(lengths, G, 16, BF, 1, -(-min(keep, max(lengths)) // PAGE), 7)
    k, v, sums, length, pages, to = s
    assert pages.shape[1] * PAGE > 4096 and (keep >= pages.shape[1] * PAGE or 4 * keep > 200 * 1024)
    from gopherllm_b200 import ops
    want = expected(k, v, sums, length, pages, to, keep, 5, 3)
    for _ in range(10):
        got = [t.clone() for t in (k, v, sums)]
        kept = ops.cache_evict(*got, length, pages, keep, recent=5, first=3, to_pages=to)
        assert torch.equal(kept.cpu(), want[0])
        assert all(same(a, b) for a, b in zip(got, want[1:]))


def test_rows_beside_one_another_do_not_matter_and_captured_it_runs_again():
    from gopherllm_b200 import ops
    k, v, sums, length, pages, to = build([300, 250, 400], 2, 32, BF, 2, 2, 5)
    want = [t.clone() for t in (k, v, sums)]
    kept = ops.cache_evict(*want, length, pages, 128, recent=20, to_pages=to)
    for b in range(3):
        one = [t.clone() for t in (k, v, sums)]
        got = ops.cache_evict(*one, length[b:b + 1].clone(), pages[b:b + 1].contiguous(), 128, recent=20, to_pages=to[b:b + 1].contiguous())
        assert torch.equal(got[:, 0], kept[:, b])
        assert all(torch.equal(x[:, to[b].long()], y[:, to[b].long()]) for x, y in zip(one, want))
    live = [t.clone() for t in (k, v, sums)]
    n = torch.zeros_like(length)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.cache_evict(*live, n, pages, 128, recent=20, to_pages=to)
    n.copy_(length)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(live, want))


def test_a_layer_alone_and_refusals():
    from gopherllm_b200 import ops
    k, v, sums, length, pages, to = build([100, 90], 2, 16, BF, 1, 1, 6)
    whole = [t.clone() for t in (k, v, sums)]
    kept = ops.cache_evict(*whole, length, pages, 64)
    flat = [t.clone() for t in (k, v, sums)]
    got = ops.cache_evict(*[t[0] for t in flat], length, pages, 64)
    assert torch.equal(got, kept[0]) and all(torch.equal(a, b) for a, b in zip(flat, whole))
    for args, kw in (((k, v, sums, length, pages, 0), {}), ((k, v, sums, length, pages, 10), dict(recent=6, first=5)), ((k, v, sums, length, pages, 10), dict(recent=-1)),
                     ((k, v, sums.double(), length, pages, 10), {}), ((k, v.float(), sums, length, pages, 10), {}), ((k.half(), v.half(), sums, length, pages, 10), {}),
                     ((k, v[:, :1], sums, length, pages, 10), {}), ((k, v, sums, length.long(), pages, 10), {}), ((k, v, sums, length, pages[:1], 10), {}),
                     ((k, v, sums, length, pages, 65), dict(to_pages=to)), ((k, v, sums, length, pages, 10), dict(to_pages=pages)), ((k, v, sums, length, pages, 10), dict(to_pages=to.long())),
                     ((k.cpu(), v, sums, length, pages, 10), {})):
        with pytest.raises(ops.KernelError):
            ops.cache_evict(*args, **kw)
