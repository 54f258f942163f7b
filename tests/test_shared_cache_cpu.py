"""Sequences that share pages, sequences that are cut down: the cache's books, and what the generation loop decides (no device needed)."""
import random

import pytest
import torch

from gopherllm_b200.cache.pool import CacheFull
from gopherllm_b200.cache.sequence_cache import PAGE, SequenceCache
from gopherllm_b200.engine.generate import GenerationOptions, begin_alike, pages_for, plan_batches
from gopherllm_b200.parts.base import KVRequest, StateRequest


def make(pages=20, reqs=(KVRequest(2, 16), KVRequest(2, 16)), slots=6, allocate=False, positions=640, weigh=False, last=None):
    return SequenceCache(list(reqs), pages * PAGE, positions, torch.float32, "cpu", max_slots=slots, allocate=allocate, weigh=weigh, last_position=last)


def grow(c, slot, n):
    c.reserve([(slot, n)])
    c.commit(slot, n)


def test_fork_shares_whole_pages_and_copies_the_one_begun():
    c = make(allocate=True, weigh=True)
    a = c.open()
    grow(c, a, 150)
    g = c.groups[0]
    for t in (g.keys, g.values, g.weights):
        t.copy_(torch.arange(t.numel(), dtype=torch.float32).view(t.shape))
    b = c.fork(a)
    pa, pb = c._pages[a][0], c._pages[b][0]
    assert pa[:2] == pb[:2] and pa[2] != pb[2] and c.length(b) == 150
    for t in (g.keys, g.values, g.weights):
        assert torch.equal(t[:, pa[2]], t[:, pb[2]])
    c.check()
    assert c.tokens_held() == 4 * PAGE and g.pool.held_count == 4 and c.shares_pages(a) and c.shares_pages(b)
    grow(c, b, 300)
    assert c._pages[a][0] == pa and len(c._pages[b][0]) == 5
    d = c.fork(b, 64)
    assert c._pages[d][0] == pa[:1] and c.groups[0].more == {pa[0]: 2, pa[1]: 1}
    c.close(a)
    c.check()
    assert c.groups[0].more == {pa[0]: 1}
    c.close(b)
    c.check()
    assert c.groups[0].pool.held_count == 1 and not c.shares_pages(d)
    c.close(d)
    c.check()
    assert c.groups[0].pool.held_count == 0


def test_shared_prefixes():
    c = make(pages=60, slots=12)
    a = c.open()
    grow(c, a, 400)
    b, d = c.fork(a), c.fork(a, 200)
    other = c.open()
    grow(c, other, 70)
    e = c.fork(other, 64)
    lone = c.open()
    grow(c, lone, 10)
    grow(c, b, 500)
    assert c.shared_prefixes([a, b]) == [([0, 1], 384)]
    assert c.shared_prefixes([d, lone, b, a]) == [([0, 2, 3], 192)]
    assert c.shared_prefixes([e, a, other, b]) == [([0, 2], 64), ([1, 3], 384)]
    assert c.shared_prefixes([a, lone]) == [] and c.shared_prefixes([lone]) == []
    f = c.fork(b)                                     # shares more with b than with a
    assert c.shared_prefixes([b, f]) == [([0, 1], 448)] and c.shared_prefixes([f, a, b]) == [([0, 1, 2], 384)]


def test_forks_that_are_refused():
    c = make(pages=5)
    a = c.open()
    grow(c, a, 200)
    for n in (-1, 201):
        with pytest.raises(ValueError):
            c.fork(a, n)
    with pytest.raises(ValueError):
        c.fork(5)
    with pytest.raises(CacheFull):
        b = c.fork(a)                                 # takes the last page ...
        c.fork(a)                                     # ... and there is none for another's begun page
    c.check()
    c.close(b)
    s = make(reqs=(KVRequest(2, 16), StateRequest((3,))), allocate=True)
    a = s.open()
    grow(s, a, 100)
    s._states[0][a] = 7.0
    with pytest.raises(ValueError, match="no longer held"):
        s.fork(a, 64)                                 # the state has moved on
    assert s._states[0][s.fork(a)].tolist() == [7.0] * 3
    w = make(reqs=(KVRequest(2, 16, window=100),))
    a = w.open()
    grow(w, a, 400)
    with pytest.raises(ValueError, match="no longer held"):
        w.fork(a, 64)
    b = w.fork(a)                                     # pages given back before the window stay given back
    w.check()
    grow(w, a, 600)
    w.check()
    assert w.shared_prefixes([a, b]) == []            # (a window's pages are not read as a prefix)
    w.close(a)
    w.check()
    w.close(b)
    w.check()
    assert w.groups[0].pool.held_count == 0


def test_shrink():
    c = make(weigh=True, last=2000)
    a = c.open()
    grow(c, a, 300)
    c.shrink(a, 100)
    c.check()
    assert c.length(a) == 100 and c.position(a) == 300 and len(c._pages[a][0]) == 2
    grow(c, a, 130)
    assert c.position(a) == 330
    b = c.fork(a)
    assert c.position(b) == 330
    with pytest.raises(ValueError, match="no longer held"):
        c.fork(a, 64)
    with pytest.raises(ValueError, match="of its own"):
        c.shrink(b, 64)
    onto = c.fresh_pages([(b, 70)])
    c.shrink(b, 70, onto[b])
    c.check()
    assert c.length(b) == 70 and c.position(b) == 330 and not c.shares_pages(a)
    for n in (0, 71):
        with pytest.raises(ValueError):
            c.shrink(b, n)
    with pytest.raises(CacheFull):
        c.fresh_pages([(a, 64 * 30)])
    c.close(a)
    c.close(b)
    c.check()
    d = c.open()
    assert c.position(d) == 0
    with pytest.raises(CacheFull, match="the cache holds"):
        c.reserve([(d, 641)])
    small = make(weigh=True, last=700)
    a = small.open()
    grow(small, a, 600)
    small.shrink(a, 64)
    small.reserve([(a, 164)])
    with pytest.raises(CacheFull, match="position"):
        small.reserve([(a, 165)])


@pytest.mark.parametrize("seed", range(20))
def test_books_under_random_use(seed):
    rng = random.Random(seed)
    c = make(pages=40, slots=8, reqs=(KVRequest(1, 8), KVRequest(1, 16)), positions=600, weigh=True, last=5000)
    for _ in range(200):
        live = c.live_slots()
        try:
            what = rng.random()
            if not live or what < 0.2:
                c.open()
            elif what < 0.4:
                s = rng.choice(live)
                c.fork(s, None if c._forgotten[s] else rng.choice((None, rng.randint(0, c.length(s)))))
            elif what < 0.7:
                s = rng.choice(live)
                grow(c, s, c.length(s) + rng.randint(1, 150))
            elif what < 0.85:
                s = rng.choice(live)
                if c.length(s) > 1:
                    keep = rng.randint(1, c.length(s))
                    c.shrink(s, keep, c.fresh_pages([(s, keep)])[s] if c.shares_pages(s) else None)
            else:
                c.close(rng.choice(live))
        except CacheFull:
            pass
        c.check()
        live = c.live_slots()
        for members, n in c.shared_prefixes(live):
            heads = {tuple(c._pages[live[i]][0][:n // PAGE]) for i in members}
            assert n >= PAGE and len(heads) == 1 and all(c.length(live[i]) >= n for i in members)
    for s in c.live_slots():
        c.close(s)
    c.check()
    assert all(g.pool.held_count == 0 and not g.more for g in c.groups)


def test_begin_alike():
    a = list(range(1000))
    assert begin_alike([a[:300], a[:100] + [5] * 300, a[:130]]) == [([0, 1, 2], 64)]
    assert begin_alike([a[:300], a[:300]]) == [([0, 1], 256)]
    assert begin_alike([a[:257], a[:257]]) == [([0, 1], 256)] and begin_alike([a[:256], a[:257]]) == [([0, 1], 192)]
    assert begin_alike([a[:64], a[:64]]) == [] and begin_alike([a[:65], a[:66]]) == [([0, 1], 64)]
    assert begin_alike([a[:90], [7] * 90, a[:80], [7] * 200, [8] * 70]) == [([0, 2], 64), ([1, 3], 64)]


def test_pages_and_options_of_a_sequence_that_is_cut():
    assert pages_for(1000, 5000, 2048) == 32 and pages_for(1000, 5000, 20480, keep=512) == 16 and pages_for(100, 5000, 20480, keep=512) == 9
    assert pages_for(100, 20, 20480, keep=512) == 2 and pages_for(1000, 5000, 20480, keep=512, shares=True) == 25
    assert plan_batches([100, 100], 5000, 20480, page_budget=18, slot_budget=8, keep=512) == [[0, 1]]
    GenerationOptions(cache_keep=10, cache_recent=6, cache_first=4).validate()
    for kw in (dict(cache_keep=-1), dict(cache_keep=10, cache_recent=11), dict(cache_recent=1), dict(cache_keep=4, cache_first=-1), dict(cache_keep=4.0)):
        with pytest.raises(ValueError):
            GenerationOptions(**kw).validate()


class _Net:
    class spec:
        vocab = 100
        max_positions = 640


def cutting_engine(monkeypatch, fail_at=0, pages=40, slots=6):
    """An engine on the CPU whose cuts are written down and of which the ``fail_at``-th fails; its cache has two groups of entries."""
    import contextlib
    from gopherllm_b200 import ops
    from gopherllm_b200.engine.step import Engine
    c = make(pages=pages, slots=slots, reqs=(KVRequest(1, 8), KVRequest(1, 16), KVRequest(1, 8)), allocate=True, weigh=True, last=5000)
    assert len(c.groups) == 2
    calls = []

    def cut(keys, values, weights, length, table, keep, recent, first, to=None):
        calls.append((keys.shape[-1], length.tolist(), to is None))
        if len(calls) == fail_at:
            raise ops.KernelError("no")
    monkeypatch.setattr(ops, "cache_evict", cut)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return Engine(_Net(), c, torch.float32, "cpu"), c, calls


@pytest.mark.parametrize("fail_at", [0, 1, 2, 3, 4])
def test_a_cut_that_fails_midway(monkeypatch, fail_at):
    """Cuts onto fresh pages come first, as they can be taken back.  One that fails leaves every sequence as it was; where a sequence's own pages
    have been cut in one group of layers and not in the next, it can only be closed."""
    eng, c, calls = cutting_engine(monkeypatch, fail_at)
    a, short = c.open(), c.open()
    grow(c, a, 300)
    grow(c, short, 50)
    b = c.fork(a, 200)
    alone = c.open()
    grow(c, alone, 130)
    free = [g.pool.free_count for g in c.groups]
    held = {s: [list(p) for p in c._pages[s]] for s in (a, b, alone)}
    if fail_at:
        with pytest.raises(Exception, match="no"):
            eng.evict([a, alone, short, b], 64)
    else:
        eng.evict([a, alone, short, b], 64)
    assert [x[1:] for x in calls] == [([300, 200], False), ([300, 200], False), ([130], True), ([130], True)][:fail_at or 4]
    if fail_at:
        assert [g.pool.free_count for g in c.groups] == free and c.length(a) == 300 and c.length(b) == 200
        assert all([list(p) for p in c._pages[s]] == held[s] for s in held)
        if fail_at == 4:
            for use in (lambda: c.length(alone), lambda: c.position(alone), lambda: c.fork(alone), lambda: c.reserve([(alone, 140)]),
                        lambda: eng.plan([(alone, [1])], None), lambda: eng.evict([alone], 64)):
                with pytest.raises(ValueError, match="closed"):
                    use()
        else:
            assert c.length(alone) == 130
    else:
        assert [c.length(s) for s in (a, b, alone, short)] == [64, 64, 64, 50]
    c.check()
    for s in (a, b, alone, short):
        c.close(s)
    c.check()
    assert all(g.pool.held_count == 0 for g in c.groups)
    s = c.open()
    while s != alone:                                              # the slot serves another sequence
        s = c.open()
    assert c.length(s) == 0


def test_more_layers_and_sequences_than_a_launch_takes_are_cut_in_parts(monkeypatch):
    from gopherllm_b200 import ops
    eng, c, calls = cutting_engine(monkeypatch)
    slots = [c.open() for _ in range(3)]
    for i, s in enumerate(slots):
        grow(c, s, 130 + i)
    slots.append(c.fork(slots[0]))
    monkeypatch.setattr(ops, "EVICT_MOST", 3)                      # (one group has two layers, the other one)
    eng.evict(slots, 64)
    # the group of two layers decides: one sequence a launch
    assert [x[1:] for x in calls] == [([130], False)] * 4 + [([131], True)] * 2 + [([132], True)] * 2
    assert [c.length(s) for s in slots] == [64] * 4
    c.check()
    monkeypatch.setattr(ops, "EVICT_MOST", 65535)
    calls.clear()
    for s in slots:
        grow(c, s, 70)
    eng.evict(slots, 64)
    assert [x[1:] for x in calls] == [([70] * 4, True)] * 2


def host_generate(monkeypatch, engine, prompts, options, vocab=100):
    """generate() on an engine without a device: every sequence ends with the stop token 9 when ``engine.ends`` says, and says 5 until then."""
    from gopherllm_b200.engine import generate as gen

    class Sampler:
        def __init__(self, *a, **k):
            pass

        def sample(self, logits, rows=None):
            return logits.argmax(-1).to(torch.int32)
    monkeypatch.setattr(gen, "DeviceSampler", Sampler)
    return gen.generate(engine, prompts, options)


class _HostEngine:
    """The cache's side of an engine; ``most``: the most sequences of a step."""
    device, prepare_decode = "cpu", None

    def __init__(self, cache, evict, ends):
        self.model, self.cache, self.evict, self.ends, self.most = _Net(), cache, evict, ends, 0
        self.open, self.close, self.fork = cache.open, cache.close, cache.fork

    def step(self, runs, want=None):
        self.most = max(self.most, len(runs))
        self.cache.reserve([(s, self.cache.length(s) + len(t)) for s, t in runs])
        out = torch.zeros(len(runs), 100)
        for i, (s, t) in enumerate(runs):
            self.cache.commit(s, self.cache.length(s) + len(t))
            out[i, 9 if self.ends(self.cache.position(s)) else 5] = 1.0
        return out


def test_requests_behind_one_text_share_its_pages_when_they_are_counted(monkeypatch):
    """Four requests behind a text of 640 tokens: ten common pages and one more each, where four sequences of their own take 44."""
    text = list(range(640))
    prompts = [[t % 100 for t in text] + [k] * 5 for k in range(4)]
    for pages, most in ((14, 4), (13, 3), (11, 1)):
        eng, c, _ = cutting_engine(monkeypatch, pages=pages)
        host = _HostEngine(c, eng.evict, lambda n: False)
        host.model = type("N", (), dict(spec=type("S", (), dict(vocab=100, max_positions=2000, stop_tokens=()))))
        c.max_positions = 2000
        out = host_generate(monkeypatch, host, prompts, GenerationOptions(max_tokens=20, seed=1, share_prefix=True))
        assert [len(r.tokens) for r in out] == [20] * 4 and host.most == most
        c.check()
        assert all(g.pool.held_count == 0 for g in c.groups)
    assert plan_batches([645] * 4, 20, 2000, 14, 8, alike=prompts) == [[0, 1, 2, 3]]
    assert plan_batches([645] * 4, 20, 2000, 14, 8) == [[0], [1], [2], [3]]
    # a request that shares nothing, or is never cut, needs no second place
    assert plan_batches([100], 5000, 20480, 9, 8, keep=512, alike=[[1] * 100]) == [[0]]
    assert plan_batches([100, 100], 20, 20480, 3, 8, keep=512, alike=[[1] * 100, [1] * 100]) == [[0, 1]]


@pytest.mark.parametrize("seed", range(30))
def test_a_batch_fits_whenever_its_sequences_end_or_are_cut(monkeypatch, seed):
    """Families of prompts with random ends, cut or not, in a cache of just the pages that the batches were planned for."""
    rng = random.Random(seed)
    texts = [[rng.randrange(10, 100) for _ in range(400)] for _ in range(3)]
    prompts = [rng.choice(texts)[:rng.randint(1, 399)] + [rng.randrange(10, 100) for _ in range(rng.randint(1, 80))] for _ in range(8)]
    keep = rng.choice((0, 70, 130, 200))
    pages = rng.randint(10, 40)
    eng, c, _ = cutting_engine(monkeypatch, pages=pages, slots=5)
    host = _HostEngine(c, eng.evict, lambda n: rng.random() < 0.01)
    options = GenerationOptions(max_tokens=rng.randint(1, 150), seed=1, stop_tokens=(9,), share_prefix=True, cache_keep=keep, cache_recent=keep // 3)
    out = host_generate(monkeypatch, host, prompts, options)
    assert all(r.finish_reason in ("stop", "length") for r in out)
    c.check()
    assert all(g.pool.held_count == 0 for g in c.groups)
