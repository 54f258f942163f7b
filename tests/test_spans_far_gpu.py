"""Caches of more than 2^31 numbers, and rows of queries behind the last sequence's: the calls on pages at the end of a large cache give
what the same calls give on a small one, bit for bit, and rows that are nobody's stay as they were."""
import pytest
import torch

import test_evict_gpu as evict
import test_prefix_gpu as prefix
import test_weighed_gpu as weighed

pytestmark = pytest.mark.gpu
PAGE = 64
BF, F = torch.bfloat16, torch.float32
H, G, D = 8, 4, 128
PAGES = (1 << 31) // (G * PAGE * D) + 3000                         # a little over 2^31 numbers


@pytest.fixture(autouse=True)
def shared_however_little(monkeypatch):
    from gopherllm_b200 import ops
    monkeypatch.setattr(ops, "PREFIX_SPARED_BYTES", 0)


def far(t, axis=0):
    """The same pages at the end of a cache of PAGES pages."""
    shape = list(t.shape)
    n, shape[axis] = shape[axis], PAGES
    big = torch.empty(shape, dtype=t.dtype, device="cuda")
    big.narrow(axis, PAGES - n, n).copy_(t)
    return big, PAGES - n


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("members", [3, 40])
def test_shared_pages_at_the_end_of_a_large_cache(dtype, members):
    from gopherllm_b200 import ops
    ctx = [128 + 37 * i % 200 for i in range(members)]
    q, k, v, c, table = prefix.build([(list(range(members)), 128)], ctx, H, G, D, dtype, 3)
    plan = ops.prefix_plan([(list(range(members)), 128)], members, H, G, D, dtype, 256, "cuda")
    near, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_prefix(q, near, k, v, c, table, plan, H, G, D)
    (bk, at), (bv, _) = far(k), far(v)
    ops.attention_prefix(q, out, bk, bv, c, table + at, plan, H, G, D)
    assert torch.equal(out, near)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("ctx,qlen", [([300, 64], [1, 1]), ([100, 0], [70, 150])])
def test_weights_at_the_end_of_a_large_cache(dtype, ctx, qlen):
    from gopherllm_b200 import ops
    s = weighed.build(ctx, qlen, H, G, D, dtype, 4)
    most = max(c + n for c, n in zip(ctx, qlen))
    near, sums = weighed.call(s, H, G, D, max(qlen), most)
    q, k, v, w, start, qlens, ctxs, table = s
    (bk, at), (bv, _), (bw, _) = far(k), far(v), far(w)
    out = torch.full_like(q, float("nan"))
    ops.attention_weighed(q, out, bk, bv, bw, start, qlens, ctxs, table + at, H, G, D, max(qlen), most)
    assert torch.equal(out, near) and torch.equal(bw[at:].nan_to_num(-1.0), sums.nan_to_num(-1.0))


@pytest.mark.parametrize("in_place", [True, False])
def test_a_cut_at_the_end_of_a_large_cache(in_place):
    from gopherllm_b200 import ops
    k, v, w, length, pages, to = evict.build([300, 130], G, D, BF, 1, 0 if in_place else 2, 5)
    (bk, at), (bv, _), (bw, _) = far(k, 1), far(v, 1), far(w, 1)
    kept = ops.cache_evict(k, v, w, length, pages, 100, 20, 2, to)
    far_kept = ops.cache_evict(bk, bv, bw, length, pages + at, 100, 20, 2, None if in_place else to + at)
    assert torch.equal(kept, far_kept)
    for big, small in ((bk, k), (bv, v), (bw, w)):
        assert torch.equal(big[:, at:], small)


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 256), (F, 64)])
@pytest.mark.parametrize("ctx,qlen", [([0, 90, 5], [0, 1, 1]), ([10, 0, 64], [0, 70, 3])])
def test_rows_behind_the_last_sequence_stay_as_they_were(dtype, hd, ctx, qlen):
    from gopherllm_b200 import ops
    s = weighed.build(ctx, qlen, H, G, hd, dtype, 6)
    q, k, v, w, start, qlens, ctxs, table = s
    alone, sums = weighed.call(s, H, G, hd, max(qlen), max(c + n for c, n in zip(ctx, qlen)))
    wide = torch.cat([q, torch.full((9, H * hd), float("nan"), dtype=dtype, device="cuda")])
    out, now = torch.full_like(wide, 7.0), w.clone()
    ops.attention_weighed(wide, out, k, v, now, start, qlens, ctxs, table, H, G, hd, max(qlen), max(c + n for c, n in zip(ctx, qlen)))
    assert torch.equal(out[:len(q)], alone) and bool((out[len(q):] == 7.0).all())
    assert torch.equal(now.nan_to_num(-1.0), sums.nan_to_num(-1.0))
