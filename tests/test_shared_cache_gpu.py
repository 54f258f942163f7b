"""Models whose sequences share pages or are cut down, through the public calls, against plain implementations that do neither or both by hand."""
import numpy as np
import pytest
import torch

import plain_phi
import tiny

pytestmark = pytest.mark.gpu


@pytest.fixture
def load(monkeypatch):
    import gopherllm_b200 as gl
    from gopherllm_b200 import ops
    from gopherllm_b200.engine import step
    for where, name in ((ops, "PREFIX_SPARED_BYTES"), (step, "SHARED_BYTES"), (step, "SHARED_BYTES_A_SEQUENCE")):
        monkeypatch.setattr(where, name, 0)                        # (tiny models would never be worth it)
    models = []

    def make(name, dtype, **kw):
        models.append(gl.load(tiny.folder(name), dtype=dtype, **{"max_tokens": 64 * 40, **kw}))
        return models[-1]
    yield make
    for m in models:
        m.close()


def plain_logits(name, tokens):
    cfg, W = plain_phi.read_folder(tiny.folder(name))
    return plain_phi.phi_logits(tokens, W, cfg)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_forked_sequences_step_as_if_each_were_alone(load, name, dtype):
    """One sequence of 70 tokens, forked whole, at a page's end, and earlier; then one token at a time, then a run, then one again.
    Steps of one token read the shared pages once (the fifth and later ones from a captured graph)."""
    from gopherllm_b200 import ops
    m = load(name, dtype)
    cfg = tiny.TINY[name][0]
    rng = np.random.default_rng(3)
    base = tiny.prompt(rng, 70, cfg["vocab_size"])
    s = m.open_sequence()
    m.step([(s, base)], [[]])
    slots = [s, m.fork_sequence(s), m.fork_sequence(s, 64), m.fork_sequence(s, 3)]
    text = [list(base), list(base), base[:64], base[:3]]
    seen = []
    called = ops.attention_prefix
    ops.attention_prefix = lambda *a: (seen.append(a[6].layout.n_items), called(*a))[1]
    try:
        for i, n in enumerate([1, 1, 1, 1, 5, 1, 1, 1]):
            new = [tiny.prompt(rng, n, cfg["vocab_size"]) for _ in slots]
            got = m.step(list(zip(slots, new)), [[n - 1]] * 4).cpu().numpy()
            for t, x in zip(text, new):
                t += x
            if i in (0, 3, 4, 7):
                want = np.stack([plain_logits(name, t)[-1].numpy() for t in text])
                err, bound = tiny.close(got, want, dtype)
                assert err <= bound, (i, err, bound)
    finally:
        ops.attention_prefix = called
    assert seen and all(n > 0 for n in seen)                       # (the shared pages were read through the plan)
    for x in slots:
        m.close_sequence(x)
    m.engine.cache.check()
    assert all(g.pool.held_count == 0 for g in m.engine.cache.groups)


@pytest.mark.parametrize("name", ["A", "C"])
def test_generate_with_shared_prompts_says_the_same(load, name):
    """In 32 bits greedy tokens do not depend on what is shared; two families of prompts and one prompt apart."""
    m = load(name, "float32")
    cfg = tiny.TINY[name][0]
    rng = np.random.default_rng(5)
    V = cfg["vocab_size"]
    one, two = tiny.prompt(rng, 80, V), tiny.prompt(rng, 66, V)
    prompts = [one + tiny.prompt(rng, k, V) for k in (1, 9, 4)] + [two + tiny.prompt(rng, k, V) for k in (2, 5)] + [tiny.prompt(rng, 20, V)]
    options = dict(max_tokens=8, temperature=0.0, top_k=0, top_p=1.0, repeat_penalty=1.0, stop_tokens=())
    apart = m.generate(prompts, **options)
    shared = m.generate(prompts, share_prefix=True, **options)
    assert [r.tokens for r in apart] == [r.tokens for r in shared]
    m.engine.cache.check()


def test_decode_loop_on_shared_pages(load):
    from gopherllm_b200.sampling.sampler import DeviceSampler, SamplerConfig
    m = load("A", "float32")
    rng = np.random.default_rng(6)
    V = tiny.TINY_A["vocab_size"]
    base = tiny.prompt(rng, 70, V)
    cfg = SamplerConfig(temperature=0.0, top_k=0, top_p=1.0, repeat_penalty=1.0)

    def run(shared):
        slots = [m.open_sequence()]
        m.step([(slots[0], base)], [[]])
        if shared:
            slots += [m.fork_sequence(slots[0], 64 + 3 * k) for k in range(2)]
        else:
            slots += [m.open_sequence() for _ in range(2)]
            m.step([(x, base[:64 + 3 * k]) for k, x in enumerate(slots[1:])], [[], []])
        sampler = DeviceSampler(cfg, [1, 2, 3], [base] * 3, V, m.engine.device)
        out = m.engine.decode_loop(slots, [5, 6, 7], 20, sampler).cpu().tolist()
        for x in slots:
            m.close_sequence(x)
        return out
    assert run(True) == run(False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("shared", [False, True])
def test_decode_loop_weighs_every_token_once(load, dtype, shared):
    """A loop's first call of a shape, which warms up before it is captured, and a second: every query head gives a layer's positions one for
    each token fed, whether sequences share pages or not; and the same sums as one token at a time."""
    from gopherllm_b200.sampling.sampler import DeviceSampler, SamplerConfig
    m = load("B", dtype, weigh=True)
    rng = np.random.default_rng(21)
    V = tiny.TINY_B["vocab_size"]
    base = tiny.prompt(rng, 128, V)
    g, cache = m.engine.cache.groups[0], m.engine.cache
    heads = m.engine.model.blocks[0].mixer.spec.num_heads
    cfg = SamplerConfig(temperature=0.0, top_k=0, top_p=1.0, repeat_penalty=1.0)

    def begin():
        slots = [m.open_sequence()]
        m.step([(slots[0], base)], [[]])
        for _ in range(2):
            if shared:
                slots.append(m.fork_sequence(slots[0]))
            else:
                slots.append(m.open_sequence())
                m.step([(slots[-1], base)], [[]])
        return slots

    def sums(slots):
        """Weights on the pages held, each page once, places without a position left out: [pages, layers, heads, PAGE]."""
        out, seen = [], set()
        for s in slots:
            for i, p in enumerate(cache._pages[s][0]):
                n = min(64, cache.length(s) - 64 * i)
                if p not in seen and n > 0:
                    seen.add(p)
                    page = g.weights[:, p].double().clone()
                    page[:, :, n:] = 0.0
                    out.append(page)
        return torch.stack(out)

    prompts = 128 if shared else 3 * 128
    slots = begin()
    sampler = DeviceSampler(cfg, [1, 2, 3], [base] * 3, V, m.engine.device)
    fed, tokens = 0, [5, 6, 7]
    text = [[], [], []]
    for steps in (4, 3):
        chosen = m.engine.decode_loop(slots, tokens, steps, sampler).cpu().tolist()
        for t, x, column in zip(text, tokens, zip(*chosen)):
            t += [x, *column[:-1]]
        tokens = chosen[-1]
        fed += steps
        got = sums(slots)
        want = (prompts + 3 * fed) * heads
        # a weight is off by a few 2^-20 of itself at most, a position's sum of fewer than 500 of them by as many roundings of 2^-24
        assert ((got.sum((0, 2, 3)) - want).abs() <= want * 2 ** -14).all(), (steps, got.sum((0, 2, 3)), want)
    for s in slots:
        m.close_sequence(s)
    slots = begin()
    for i in range(fed):
        m.step([(s, [t[i]]) for s, t in zip(slots, text)], [[]] * 3)
    err, bound = tiny.close(got.cpu().numpy(), sums(slots).cpu().numpy(), dtype)
    assert err <= bound, (err, bound)
    cache.check()


def test_heads_with_a_gate_and_values_that_are_keys(load):
    """The mixer that has both, without a window, on shared pages and in a cache that is weighed: as without either."""
    import gopherllm_b200 as gl
    import dibedra_models
    cfg = dict(dibedra_models.BETA)
    for dtype in ("float32", "bfloat16"):
        rng = np.random.default_rng(4)
        m = gl.load_random(cfg, seed=1, dtype=dtype, max_tokens=64 * 30)
        V = m.spec.vocab
        base, tails = tiny.prompt(rng, 70, V), [tiny.prompt(rng, 4, V) for _ in range(3)]

        def run(shared):
            s = m.open_sequence()
            m.step([(s, base)], [[]])
            slots = [s]
            for _ in tails[1:]:
                if shared:
                    slots.append(m.fork_sequence(s))
                else:
                    slots.append(m.open_sequence())
                    m.step([(slots[-1], base)], [[]])
            out = [m.step([(x, [t[i]]) for x, t in zip(slots, tails)]).cpu().numpy() for i in range(4)]
            for x in slots:
                m.close_sequence(x)
            return np.stack(out)
        err, bound = tiny.close(run(True), run(False), dtype)
        assert err <= bound, (dtype, err, bound)
        m.engine.cache.check()
        m.close()


def test_gated_heads_are_weighed(load):
    """Weighing changes no logits, with a gate on the result and values that are keys either; and all layers without a window can be cut."""
    import gopherllm_b200 as gl
    import dibedra_models
    cfg = dict(dibedra_models.BETA)
    cfg["layers"] = [dict(cfg["layers"][0], weights_of=None, mixer=dibedra_models._B1, mlp=None) for _ in range(2)]
    cfg["layers"] = [{k: v for k, v in x.items() if v is not None or k == "mlp"} for x in cfg["layers"]]
    rng = np.random.default_rng(6)
    text = tiny.prompt(rng, 100, 257)
    out = {}
    for weigh in (False, True):
        m = gl.load_random(cfg, seed=1, dtype="float32", max_tokens=64 * 10, weigh=weigh)
        s = m.open_sequence()
        got = [m.step([(s, text[:90])])] + [m.step([(s, [t])]) for t in text[90:]]
        out[weigh] = torch.cat(got).cpu().numpy()
        if weigh:
            m.evict([s], 64, recent=64)
            assert m.engine.cache.length(s) == 64 and np.isfinite(m.step([(s, [5])]).cpu().numpy()).all()
        m.close()
    err, bound = tiny.close(out[True], out[False], "float32")
    assert err <= bound, (err, bound)


@pytest.mark.parametrize("module,name", [("vopedra_models", "ALPHA"), ("gozolix_models", "ALPHA"), ("lilupel_models", "ALPHA"), ("nakurax_models", "ALPHA"), ("darusun_models", "ALPHA")])
def test_designs_with_state_and_windows_can_be_forked_whole(load, module, name):
    """State rows are copied, begun pages too, pages behind a window shared or given back: a forked sequence goes on as the one it was forked from."""
    import importlib
    import gopherllm_b200 as gl
    m = gl.load_random(dict(getattr(importlib.import_module(module), name)), seed=2, dtype="float32", max_tokens=64 * 30)
    rng = np.random.default_rng(5)
    V = m.spec.vocab
    s = m.open_sequence()
    m.step([(s, tiny.prompt(rng, 75, V))], [[]])
    for n in (1, 1, 3, 1):
        f = m.fork_sequence(s)
        new = tiny.prompt(rng, n, V)
        a = m.step([(s, new), (f, new)]).cpu().numpy()
        assert np.isfinite(a).all() and np.abs(a[0] - a[1]).max() <= 1e-5 * max(1.0, np.abs(a).max())
        m.close_sequence(f)
        m.engine.cache.check()
    m.close_sequence(s)
    m.engine.cache.check()
    m.close()


class Forgetful:
    """The plain model one token at a time, each key/value head with the positions it still holds and the weight they were given."""

    def __init__(self, name):
        self.cfg, self.W = plain_phi.read_folder(tiny.folder(name))
        self.heads = [[([], [], [], []) for _ in range(plain_phi.sizes(self.cfg)[1])] for _ in range(self.cfg["num_hidden_layers"])]
        self.n = 0

    def feed(self, token):
        cfg, W = self.cfg, self.W
        nh, nkv, hd, _ = plain_phi.sizes(cfg)
        layer = iter(self.heads)

        def attention(q, k, v, window=0):
            out = torch.zeros_like(q)
            for g, (ks, vs, given, at) in enumerate(next(layer)):
                ks.append(k[0, g]), vs.append(v[0, g]), given.append(0.0), at.append(self.n)
                for h in range(g * nh // nkv, (g + 1) * nh // nkv):
                    p = torch.softmax(torch.stack(ks) @ q[0, h], 0)
                    out[0, h] = p @ torch.stack(vs)
                    for j, x in enumerate(p.tolist()):
                        given[j] += x
            return out
        keep, plain_phi.attention = plain_phi.attention, attention
        try:
            x = plain_phi.embedding([token], W["model.embed_tokens.weight"])
            for i in range(cfg["num_hidden_layers"]):
                x = plain_phi.phi_block(x, [self.n], W, i, cfg)
        finally:
            plain_phi.attention = keep
        self.n += 1
        x = plain_phi.layer_norm(x, W["model.final_layernorm.weight"], W["model.final_layernorm.bias"], cfg.get("layer_norm_eps", 1e-5))
        logits = x @ (W["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings", False) else W["lm_head.weight"]).T
        return (logits + W["lm_head.bias"] if "lm_head.bias" in W else logits)[0].numpy()

    def cut(self, keep, recent, first):
        for layer in self.heads:
            for g, (ks, vs, given, at) in enumerate(layer):
                n = len(at)
                if n <= keep:
                    continue
                best = sorted(range(first, n - recent), key=lambda j: (-given[j], j))[:keep - first - recent]
                stay = sorted([*range(first), *best, *range(n - recent, n)])
                layer[g] = tuple([x[j] for j in stay] for x in (ks, vs, given, at))


@pytest.mark.parametrize("name,dtype,keep,recent,first", [("B", "float32", 70, 20, 2), ("C", "float32", 40, 0, 0), ("A", "float32", 50, 50, 0),
                                                          ("A", "bfloat16", 70, 66, 4), ("C", "bfloat16", 40, 40, 0)])
def test_a_model_that_forgets(load, name, dtype, keep, recent, first):
    """A prompt, tokens, a cut, a run, tokens, a cut, tokens: logits as the plain model's that forgets by hand.  (In bfloat16 the
    cuts go by position alone: which of two nearly equal weights is larger depends on rounding.)"""
    m = load(name, dtype, weigh=True)
    V = tiny.TINY[name][0]["vocab_size"]
    rng = np.random.default_rng(7)
    plain, s, other = Forgetful(name), m.open_sequence(), m.open_sequence()
    m.step([(other, tiny.prompt(rng, 30, V))], [[]])

    def both(tokens):
        want = [plain.feed(t) for t in tokens][-1]
        got = m.step([(other, tiny.prompt(rng, 1, V)), (s, tokens)], [[], [len(tokens) - 1]]).cpu().numpy()
        err, bound = tiny.close(got[0], want, dtype)
        assert err <= bound, (plain.n, err, bound)

    def cut():
        m.evict([s, other], keep, recent=recent, first=first)
        plain.cut(keep, recent, first)
        m.engine.cache.check()
        assert m.engine.cache.length(s) == keep and m.engine.cache.position(s) == plain.n
    both(tiny.prompt(rng, 80, V))
    for _ in range(4):
        both(tiny.prompt(rng, 1, V))
    cut()
    for _ in range(3):
        both(tiny.prompt(rng, 1, V))
    both(tiny.prompt(rng, 20, V))
    cut()
    for _ in range(4):
        both(tiny.prompt(rng, 1, V))
    if dtype == "float32":                                         # what the cache says of its positions is what the plain model says
        g = m.engine.cache.groups[0]
        ids = torch.tensor(m.engine.cache._pages[s][0])
        n = m.engine.cache.length(s)
        for layer, heads in enumerate(plain.heads):
            got = g.weights[layer].cpu()[ids].transpose(0, 1).reshape(len(heads), -1)[:, :n].double().numpy()
            want = np.array([given for _, _, given, _ in heads])
            assert np.abs(got - want).max() <= 1e-4 * max(1.0, want.max())


def test_a_forked_sequence_is_cut_onto_pages_of_its_own(load):
    """... and the one it was forked from goes on as if nothing had happened."""
    m = load("B", "float32", weigh=True)
    V = tiny.TINY_B["vocab_size"]
    rng = np.random.default_rng(8)
    base = tiny.prompt(rng, 150, V)
    s = m.open_sequence()
    m.step([(s, base)], [[]])
    f = m.fork_sequence(s)
    m.evict([f], 40, recent=10, first=1)
    m.engine.cache.check()
    forgot = Forgetful("B")
    for t in base:
        forgot.feed(t)
    forgot.cut(40, 10, 1)
    text = list(base)
    for _ in range(3):
        new = tiny.prompt(rng, 1, V)
        text += new
        got = m.step([(s, new), (f, new)]).cpu().numpy()
        for x, want in zip(got, (plain_logits("B", text)[-1].numpy(), forgot.feed(new[0]))):
            err, bound = tiny.close(x, want, "float32")
            assert err <= bound, (err, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_positions_of_forked_sequences_are_given_what_all_give(load, dtype):
    """Two forks of one sequence, token by token (captured) and with a run, twice: the same weights to the last bit, and on
    the common pages what each step gave from both: every step gives a layer's positions one for each token and query head."""
    m = load("B", dtype, weigh=True)
    V = tiny.TINY_B["vocab_size"]
    rng = np.random.default_rng(12)
    base, runs = tiny.prompt(rng, 128, V), [tiny.prompt(rng, 12, V) for _ in range(3)]

    def run():
        s = m.open_sequence()
        m.step([(s, base)], [[]])
        slots = [s, m.fork_sequence(s), m.fork_sequence(s)]
        for i in range(8):
            m.step(list(zip(slots, [[r[i]] for r in runs])))
        m.step([(x, r[8:]) for x, r in zip(slots, runs)])
        g = m.engine.cache.groups[0]
        lists = [m.engine.cache._pages[x][0] for x in slots]
        assert all(p[:2] == lists[0][:2] and p[2] != lists[0][2] for p in lists[1:])
        got = torch.cat([g.weights[:, lists[0][:2]], *(g.weights[:, p[2:3]] for p in lists)], 1)      # [layers, 5 pages, heads, PAGE]
        got[:, 2:, :, 12:] = 0.0                                   # (nothing is there)
        for x in slots:
            m.close_sequence(x)
        return got

    run()                                                          # (the first steps of the first time are not captured: they divide sequences otherwise)
    one, two = run(), run()
    assert torch.equal(one, two)
    spec = m.engine.model.blocks[0].mixer.spec
    total = one.double().sum((1, 2, 3))
    want = (128 + 3 * 12) * spec.num_heads                         # every query and head gives one altogether
    # each weight is off by a few 2^-20 of itself at most, a sum of fewer than 200 of them by that and 200 roundings of 2^-24
    assert ((total - want).abs() <= want * (2 ** -14)).all(), total


def test_generate_in_a_bounded_cache(load):
    """Six pages serve prompts of 100 tokens and 120 more each, two at a time, where 220 positions would take four pages a sequence;
    the tokens are those of stepping and cutting by hand."""
    m = load("B", "float32", weigh=True, max_tokens=64 * 6)
    V = tiny.TINY_B["vocab_size"]
    rng = np.random.default_rng(9)
    prompts = [tiny.prompt(rng, n, V) for n in (100, 90)]
    options = dict(max_tokens=120, temperature=0.0, top_k=0, top_p=1.0, repeat_penalty=1.0, stop_tokens=())
    out = m.generate(prompts, cache_keep=64, cache_recent=20, cache_first=2, **options)
    assert [len(r.tokens) for r in out] == [120, 120]
    m.engine.cache.check()
    slots = [m.open_sequence() for _ in prompts]
    logits = m.step(list(zip(slots, prompts)))
    tokens = [[], []]
    for i in range(120):
        new = logits.argmax(-1).tolist()
        for t, x in zip(tokens, new):
            t.append(x)
        m.evict([s for s in slots if m.engine.cache.length(s) >= 128], 64, recent=20, first=2)
        if i < 119:
            logits = m.step([(s, [x]) for s, x in zip(slots, new)])
    assert [r.tokens for r in out] == tokens
    for s in slots:
        m.close_sequence(s)
    again = m.generate([prompts[0] + [3], prompts[0] + [4]], cache_keep=64, cache_recent=20, share_prefix=True, **options)
    assert [len(r.tokens) for r in again] == [120, 120]
    m.engine.cache.check()


def test_a_stop_token_leaves_no_weights_on_shared_pages(load):
    """Three sequences on two common pages, of which one ends with a stop token before the first cut: the token that ends it is never fed,
    so the others are cut by the weights, and say the tokens, of stepping and cutting by hand."""
    from gopherllm_b200.sampling.sampler import DeviceSampler, SamplerConfig
    m = load("B", "float32", weigh=True)
    V = tiny.TINY_B["vocab_size"]
    rng = np.random.default_rng(30)
    base = tiny.prompt(rng, 128, V)
    prompts = [base + tiny.prompt(rng, n, V) for n in (3, 2, 5)]
    cut = dict(cache_keep=100, cache_recent=20, cache_first=2)
    sampling = dict(temperature=0.0, top_k=0, top_p=1.0, repeat_penalty=1.5)
    cache, g = m.engine.cache, m.engine.cache.groups[0]
    evict, masses = m.engine.evict, []

    def watched(slots, *a):
        pages = sorted({p for s in cache.live_slots() for p in cache._pages[s][0][:2]})          # whole pages of all that goes on
        masses.append(g.weights[:, pages].double().sum((1, 2, 3)).cpu())
        evict(slots, *a)
    m.engine.evict = watched
    free = [r.tokens for r in m.generate(prompts, share_prefix=True, max_tokens=60, stop_tokens=(), **cut, **sampling)]
    ends = next((r, t) for r in range(3) for i, t in enumerate(free[r][:25]) if i >= 3 and t not in free[r][:i]
                and not any(t in o for k, o in enumerate(free) if k != r))
    masses.clear()
    got = m.generate(prompts, share_prefix=True, max_tokens=60, stop_tokens=(ends[1],), **cut, **sampling)
    assert got[ends[0]].finish_reason == "stop" and [r.finish_reason for r in got].count("length") == 2
    said, masses = masses[0], []
    # by hand, as stepped; the stop token ends its sequence before anything else is done
    slots = [m.open_sequence()]
    m.step([(slots[0], base)], [[]])
    slots += [m.fork_sequence(slots[0]) for _ in prompts[1:]]
    logits = m.step([(s, p[128:]) for s, p in zip(slots, prompts)])
    sampler = DeviceSampler(SamplerConfig(**sampling), [1, 2, 3], prompts, V, m.engine.device)
    live, tokens = [0, 1, 2], [[], [], []]
    while live:
        chosen = sampler.sample(logits, torch.tensor(live, dtype=torch.int32, device=m.engine.device)).tolist()
        for r, t in zip(list(live), chosen):
            if t == ends[1] or len(tokens[r]) == 59:
                if t != ends[1]:
                    tokens[r].append(t)
                m.close_sequence(slots[r])
                live.remove(r)
            else:
                tokens[r].append(t)
        due = [slots[r] for r in live if cache.length(slots[r]) >= 164]
        if due:
            watched(due, 100, 20, 2)
        if live:
            logits = m.step([(slots[r], [tokens[r][-1]]) for r in live])
    # (weights are off by a few 2^-20 of themselves and a sum's roundings; one token too many is 4 heads' worth among some 900)
    assert ((said - masses[0]).abs() <= masses[0] * 2 ** -14).all(), (said, masses[0])
    assert [r.tokens for r in got] == tokens
    cache.check()


def test_refusals(load):
    import gopherllm_b200 as gl
    m = load("A", "bfloat16")
    s = m.open_sequence()
    m.step([(s, [1, 2, 3])], [[]])
    with pytest.raises(ValueError, match="weigh"):
        m.evict([s], 2)
    with pytest.raises(ValueError, match="weigh"):
        m.generate([1, 2, 3], max_tokens=2, cache_keep=64)
    with pytest.raises(ValueError):
        m.fork_sequence(s, 4)
    w = load("A", "bfloat16", weigh=True)
    s = w.open_sequence()
    w.step([(s, [1, 2, 3])], [[]])
    for slots, keep, kw in (([s, s], 2, {}), ([s], 0, {}), ([s], 2, dict(recent=3)), ([s + 1], 2, {})):
        with pytest.raises(ValueError):
            w.evict(slots, keep, **kw)
    w.evict([s], 3)                                                # nothing to do
    assert w.engine.cache.length(s) == 3
    import vopedra_models
    with pytest.raises(ValueError, match="weigh=True"):
        gl.load_random(dict(vopedra_models.ALPHA), weigh=True, max_tokens=256)


def test_a_cut_that_fails_holds_no_pages(load, monkeypatch):
    from gopherllm_b200 import ops
    m = load("B", "float32", weigh=True)
    s = m.open_sequence()
    m.step([(s, list(range(1, 131)))], [[]])
    f = m.fork_sequence(s)
    cache = m.engine.cache
    free, length = cache.groups[0].pool.free_count, cache.length(f)

    def refuse(*_):
        raise ops.KernelError("no")
    monkeypatch.setattr(ops, "cache_evict", refuse)
    with pytest.raises(ops.KernelError):
        m.evict([f], 40)
    cache.check()
    assert cache.groups[0].pool.free_count == free and cache.length(f) == length
    m.close_sequence(s)
    m.close_sequence(f)
