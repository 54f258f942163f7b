"""What the host decides for attention over shared pages, and what it refuses (no device needed)."""
import random

import pytest
import torch

from gopherllm_b200 import ops

BF, F = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def shared_however_little(monkeypatch):
    from gopherllm_b200 import ops
    monkeypatch.setattr(ops, "PREFIX_SPARED_BYTES", 0)


def covered(lay, groups):
    """Every (member, head of the group, page) of a group's shared pages, as often as an item covers it; and the slots it goes to."""
    order = lay.ints[:lay.items_at].tolist()
    items = lay.ints[lay.items_at:lay.shared_at].reshape(-1, 6).tolist()
    shared = lay.ints[lay.shared_at:].reshape(-1, 2).tolist()
    g = lay.num_heads // lay.num_kv_heads
    seen = {}
    for at, first, rows, p0, p1, slot in items:
        assert 1 <= rows <= lay.rows and p0 < p1
        for r in range(first, first + rows):
            b = order[at + r // g]
            assert slot < shared[b][1] and p1 <= shared[b][0]
            for p in range(p0, p1):
                assert (b, r % g, p) not in seen
                seen[b, r % g, p] = slot
    return seen, shared


@pytest.mark.parametrize("seed", range(40))
def test_items_cover_every_shared_page_of_every_row_once(seed):
    rng = random.Random(seed)
    kv, g = rng.choice((1, 2, 8)), rng.choice((1, 3, 4, 16, 40))
    dtype = rng.choice((BF, F))
    batch = rng.randint(1, 60)
    who = list(range(batch))
    rng.shuffle(who)
    groups, at = [], 0
    while at < batch and rng.random() < 0.8:
        n = rng.randint(1, batch - at)
        groups.append((who[at:at + n], 64 * rng.randint(1, 200)))
        at += n
    lay = ops.PrefixLayout(groups, batch, kv * g, kv, rng.choice((64, 256)), dtype, rng.randint(1, 900), 148)
    seen, shared = covered(lay, groups)
    want = {(b, h, p) for members, n in groups for b in members for h in range(g) for p in range(n // 64)}
    assert set(seen) == want
    for b in range(batch):
        # a sequence's slots are used without a gap, from 0 on; where a second kernel joins them its own spans come behind
        assert {s for (c, _, _), s in seen.items() if c == b} == set(range(shared[b][1])) and shared[b][1] + (0 if lay.joined else lay.splits) <= lay.slots
    assert lay.n_items == len(lay.ints[lay.items_at:lay.shared_at]) // 6
    assert ops.span_rows(dtype, lay.head_dim) * lay.chunks >= g


def test_plans_that_are_refused():
    ok = dict(batch=4, num_heads=4, num_kv_heads=2, head_dim=64, dtype=BF, own=5, sms=148)
    ops.PrefixLayout([([0, 1], 64)], **ok)
    for groups, change in (([([0, 0], 64)], {}), ([([0, 4], 64)], {}), ([([-1], 64)], {}), ([([0], 64), ([0, 1], 64)], {}), ([([], 64)], {}), ([([0], 0)], {}),
                           ([([0], 100)], {}), ([], dict(num_heads=5)), ([], dict(head_dim=40)), ([], dict(head_dim=272)), ([], dict(dtype=torch.float16)),
                           ([], dict(dtype=F, head_dim=257)), ([], dict(own=0)), ([], dict(batch=0)), ([], dict(num_kv_heads=0))):
        with pytest.raises(ops.KernelError):
            ops.PrefixLayout(groups, **{**ok, **change})


def test_tensors_off_the_device_are_refused():
    t = torch.zeros(2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError):
        ops.attention_weighed(t, t, t.view(1, 1, 2, 64), t, t, i, i, i, i.view(2, 1), 1, 1, 64, 1, 1)
    with pytest.raises(ops.KernelError):
        ops.attention_prefix(t, t, t, t, i, i.view(2, 1), None, 1, 1, 64)
    with pytest.raises(ops.KernelError):
        ops.cache_evict(torch.zeros(1, 1, 64, 8), torch.zeros(1, 1, 64, 8), torch.zeros(1, 1, 64), i, i.view(2, 1), 4)


def test_no_launch_behind_a_refusal(monkeypatch):
    """The checks of shapes, types and sizes, with the device's own taken out: none of these calls reaches a launcher."""
    monkeypatch.setattr(ops, "_one_device", lambda *a: None)
    monkeypatch.setattr(ops, "_launch_device", lambda t: t.get_device())

    def need(t, name, dtype=None, shape=None):
        if not t.is_contiguous() or (dtype is not None and t.dtype != dtype) or (shape is not None and tuple(t.shape) != tuple(shape)):
            raise ops.KernelError(name)
    monkeypatch.setattr(ops, "_need", need)
    monkeypatch.setattr(ops, "sm_count", lambda d: 148)
    launched = []
    monkeypatch.setattr(ops, "_launch", lambda *a: launched.append(a) or 0)
    monkeypatch.setattr(ops, "_stream", lambda: None)

    class Lib:
        def __getattr__(self, name):
            return name
    monkeypatch.setattr(ops, "_lib", lambda *a: Lib())
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    q, k, w = torch.zeros(2, 256, dtype=BF), torch.zeros(6, 2, 64, 64, dtype=BF), torch.zeros(6, 2, 64)
    good = [q, q.clone(), k, k.clone(), w, i32(2), i32(2), i32(2), i32(2, 3), 4, 2, 64, 1, 100, 0]
    ops.attention_weighed(*good)
    assert len(launched) == 1
    for i, x in ((0, q.float()), (1, q[:1]), (2, k.float()), (3, k[:1]), (4, w.double()), (5, i32(3)), (6, i32(1)), (7, i32(2, 1)), (8, i32(1, 3)), (9, 3), (10, 0),
                 (11, 60), (12, -1), (13, 0), (13, 193), (14, -1)):
        with pytest.raises(ops.KernelError):
            ops.attention_weighed(*good[:i], x, *good[i + 1:])
    plan = ops.PrefixPlan(ops.PrefixLayout([([0, 1], 128)], 2, 4, 2, 64, BF, 5, 148), i32(9))
    good = [q, q.clone(), k, k.clone(), i32(2), i32(2, 3), plan, 4, 2, 64]
    ops.attention_prefix(*good)
    other = ops.PrefixPlan(ops.PrefixLayout([], 3, 4, 2, 64, BF, 5, 148), i32(9))
    for i, x in ((0, q.float()), (1, q[:1]), (3, k[:1]), (4, i32(3)), (5, i32(2, 1)), (6, other), (7, 8), (8, 4), (9, 32)):
        with pytest.raises(ops.KernelError):
            ops.attention_prefix(*good[:i], x, *good[i + 1:])
    assert len(launched) == 2


def test_a_cache_of_no_pages_is_refused(monkeypatch):
    """Whatever a table says, nothing lies there: no launcher is reached."""
    monkeypatch.setattr(ops, "_launch_device", lambda t: t.get_device())
    monkeypatch.setattr(ops, "sm_count", lambda d: 148)
    monkeypatch.setattr(ops, "_lib", lambda *a: pytest.fail("a launcher was asked for"))
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for dtype in (BF, F):
        q, k = torch.zeros(2, 256, dtype=dtype), torch.zeros(0, 2, 64, 64, dtype=dtype)
        for run in (1, 3):
            with pytest.raises(ops.KernelError, match="no pages"):
                ops.attention_weighed(q, q.clone(), k, k.clone(), torch.zeros(0, 2, 64), i32(2), i32(2), i32(2), i32(2, 3), 4, 2, 64, run, 100)
        ops.attention_weighed(q, q.clone(), k, k.clone(), torch.zeros(0, 2, 64), i32(2), i32(2), i32(2), i32(2, 3), 4, 2, 64, 0, 0)      # (no tokens: nothing to do)
        plan = ops.PrefixPlan(ops.PrefixLayout([([0, 1], 128)], 2, 4, 2, 64, dtype, 5, 148), i32(9))
        with pytest.raises(ops.KernelError, match="no pages"):
            ops.attention_prefix(q, q.clone(), k, k.clone(), i32(2), i32(2, 3), plan, 4, 2, 64)


ALIGN = -3                                                         # GL_ERR_ALIGN (csrc/common.cuh)


@pytest.mark.parametrize("name,off", [("out", 2), ("out", 4), ("q", 2), ("q", 8), ("k_cache", 2), ("v_cache", 4)])
def test_tensors_at_odd_places_are_refused_by_the_launchers(name, off):
    """A contiguous view into a larger buffer may begin anywhere; the kernels read and write in wider pieces.  The launchers look at addresses
    before they do anything else, so no device is needed (and none is reached: every call here is refused)."""
    lib = ops._lib("attention_spans.cu", ("GL_HEAD_DIM=64",))
    at = dict(q=1 << 20, out=2 << 20, k_cache=3 << 20, v_cache=4 << 20)
    at[name] += off
    sizes = dict(B=2, nH=4, nKV=2, max_pages=3, n_pages=6, splits=1, chunks=1, reach=100)
    one = ops._SpanArgs(**at, **sizes, seq_row=5 << 20, seq_qlen=5 << 20, seq_ctx=5 << 20, pages=5 << 20, weights=6 << 20)
    assert lib.gl_attention_weighed(ops.byref(one), None) == ALIGN
    two = ops._SpanArgs(**at, **sizes, seq_ctx=5 << 20, pages=5 << 20, seq_shared=5 << 20)
    assert lib.gl_attention_prefix(ops.byref(two), ops.c_int(8), ops.c_int(1), None) == ALIGN


@pytest.mark.parametrize("name,off", [("out", 2), ("q", 2), ("q", 8), ("k_cache", 2), ("v_cache", 4)])
def test_the_attention_behind_weighed_runs_of_wide_heads_refuses_odd_places(name, off):
    """Runs of several tokens with heads above 128 reach this launcher before any of attention over spans."""
    lib = ops._lib("attention_prefill.cu", ("GL_HEAD_DIM=256",))
    at = dict(q=1 << 20, out=2 << 20, k_cache=3 << 20, v_cache=4 << 20)
    at[name] += off
    a = ops._AttnArgs(**at, seq_qstart=5 << 20, seq_qlen=5 << 20, seq_ctx=5 << 20, pages=5 << 20, B=1, nH=4, nKV=2, hd=256, max_pages=3, max_qlen=5, score_scale=1.0)
    assert lib.gl_attention_prefill(ops.byref(a), None) == ALIGN
