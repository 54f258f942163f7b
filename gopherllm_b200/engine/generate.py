"""The generation loop above the step function.

Requests (prompts of token ids) are cut into batches that fit the cache; the
prompts of a batch run in one step, then every live sequence gets one token per
step.  A sequence that ends leaves the batch at once and its slot and pages go
back to the cache; the next batch reuses them.  Per sequence the order of
events is the reference's (runtime.go:1130-1165, emitToken :1059-1095): sample
from the current logits; a stop token ends the sequence with "stop" and is
neither emitted nor fed; otherwise the token is emitted, and the sequence ends
with "length" once max_tokens are out or the cache cannot take another
position; otherwise the token is fed.
"""
from __future__ import annotations

import time
from dataclasses import dataclass, field
from typing import Callable, List, Optional, Sequence, Tuple

from ..cache.sequence_cache import PAGE
from ..sampling.sampler import DeviceSampler, SamplerConfig, request_seed


@dataclass
class GenerationOptions:
    """The reference's GenerationOptions (runtime.go:90-125) for token-level use:
    max_tokens (default 256), sampler, seed (0: taken from the clock,
    runtime.go:906-910), stop_tokens (default: the model's end-of-sequence id,
    runtime.go:1914), should_stop (polled between steps, as the reference polls
    its context, runtime.go:1131), on_token(request index, token): called for every
    emitted token as it is known; returning False cancels the generation with what
    was generated so far (the reference's streaming callback, runtime.go:793-815,
    1024, which gets text; this library is token-level).

    share_prefix: prompts of a batch that begin alike are run once as far as they do (whole pages), and
    their sequences share those pages.  cache_keep n > 0: a sequence that has come to hold a page more than n
    positions is cut down to n, the cache_first first, the cache_recent last and those between that
    attention has given the most weight (an engine whose cache keeps weights)."""
    max_tokens: int = 256
    sampler: SamplerConfig = field(default_factory=SamplerConfig)
    seed: int = 0
    stop_tokens: Tuple[int, ...] = ()
    should_stop: Optional[Callable[[], bool]] = None
    on_token: Optional[Callable[[int, int], Optional[bool]]] = None
    share_prefix: bool = False
    cache_keep: int = 0
    cache_recent: int = 0
    cache_first: int = 0

    @classmethod
    def from_kwargs(cls, spec=None, **kw) -> "GenerationOptions":
        s = SamplerConfig()
        for k in ("temperature", "top_p", "top_k", "min_p", "repeat_penalty"):
            if k in kw:
                setattr(s, k, kw.pop(k))
        if "sampler" in kw:
            s = kw.pop("sampler")
        stops = kw.pop("stop_tokens", None)
        if stops is None:
            stops = tuple(spec.stop_tokens) if spec is not None else ()
        o = cls(max_tokens=kw.pop("max_tokens", 256), sampler=s, seed=kw.pop("seed", 0),
                stop_tokens=tuple(int(t) for t in stops), should_stop=kw.pop("should_stop", None),
                on_token=kw.pop("on_token", None), share_prefix=bool(kw.pop("share_prefix", False)), cache_keep=kw.pop("cache_keep", 0),
                cache_recent=kw.pop("cache_recent", 0), cache_first=kw.pop("cache_first", 0))
        if kw:
            raise TypeError(f"unknown generation options: {', '.join(sorted(kw))}")
        return o

    def validate(self) -> None:
        if not isinstance(self.max_tokens, int) or self.max_tokens <= 0:
            raise ValueError("max_tokens must be greater than 0")
        if not isinstance(self.cache_keep, int) or self.cache_keep < 0 or self.cache_recent < 0 or self.cache_first < 0 \
                or self.cache_recent + self.cache_first > self.cache_keep:
            raise ValueError(f"the first {self.cache_first} and the last {self.cache_recent} positions do not go into {self.cache_keep}")
        self.sampler.validate()


@dataclass
class GenerationStats:
    """runtime.go:198-205; times in seconds."""
    prompt_tokens: int = 0
    generated_tokens: int = 0
    ttft: float = 0.0
    prefill_time: float = 0.0
    decode_time: float = 0.0
    total_time: float = 0.0
    token_times: List[float] = field(default_factory=list)   # seconds from the request's start to each token


@dataclass
class GenerationResult:
    tokens: List[int]
    finish_reason: str          # "stop", "length" or "canceled"
    stats: GenerationStats


class GenerationCanceled(RuntimeError):
    """should_stop() returned true; ``results`` holds what was generated so far."""

    def __init__(self, results):
        super().__init__("generation canceled")
        self.results = results


# ---------------------------------------------------------------------------
# decisions (no device involved)
# ---------------------------------------------------------------------------
def pages_for(prompt_len: int, max_tokens: int, max_positions: int, keep: int = 0, shares: bool = False) -> int:
    """Pages a request can come to hold: its prompt plus every token it may feed; with ``keep`` its prompt, and later no
    more than a page beyond that many positions.  What is kept of a sequence that ``shares`` pages moves to others."""
    most = min(prompt_len + max_tokens, max_positions)
    moves = shares and 0 < keep and keep + PAGE <= most            # (a shorter one is never cut)
    if keep > 0:
        most = min(most, max(prompt_len, keep + PAGE)) + (keep if moves else 0)
    return -(-most // PAGE) + (1 if moves else 0)


class _Alike:
    """Prompts that begin with the same page of tokens: their numbers and the tokens that all of them have in common, short of any
    one's last token (which is run by each, for its logits)."""

    def __init__(self, members: List[int], first: Sequence[int], common: int):
        self.members, self.first, self.common = members, first, common

    @staticmethod
    def key(prompt: Sequence[int]):
        """The same for prompts of a group; None for a prompt that is in none."""
        return tuple(prompt[:PAGE]) if len(prompt) > PAGE else None

    @classmethod
    def joined(cls, group: Optional["_Alike"], i: int, prompt: Sequence[int]) -> "_Alike":
        """The group with one more prompt (None: a group of it alone)."""
        if group is None:
            return cls([i], prompt, len(prompt) - 1)
        first, common = group.first, min(group.common, len(prompt) - 1)
        if first[:common] != prompt[:common]:
            common = next((n for n in range(common) if first[n] != prompt[n]), common)
        return cls(group.members + [i], first, common)

    @property
    def pages(self) -> int:
        return self.common // PAGE


def begin_alike(prompts: Sequence[Sequence[int]]) -> List[Tuple[List[int], int]]:
    """(members, tokens) for prompts that share their first page of tokens or more: how many whole pages of tokens all members
    have in common, short of any member's last token (which is run by each, for its logits)."""
    groups: dict = {}
    for i, p in enumerate(prompts):
        key = _Alike.key(p)
        if key is not None:
            groups[key] = _Alike.joined(groups.get(key), i, p)
    return [(g.members, g.pages * PAGE) for g in groups.values() if len(g.members) > 1]


def plan_batches(prompt_lens: Sequence[int], max_tokens: int, max_positions: int,
                 page_budget: int, slot_budget: int, keep: int = 0, alike: Optional[Sequence[List[int]]] = None) -> List[List[int]]:
    """Cut requests, in order, into batches whose worst-case page need fits the cache.  ``alike``: the prompts, where those of a batch that
    begin alike hold their common pages once."""
    batches: List[List[int]] = []
    cur: List[int] = []
    used = 0
    groups: dict = {}                                              # of the current batch: (prompts, pages of each beside the others, pages of all)
    for i, n in enumerate(prompt_lens):
        if n < 1:
            raise ValueError(f"request {i}: the prompt is empty")
        if n >= max_positions:
            # the reference rejects len(tokens) >= MaxSeqLen before any forward (runtime.go:866-868)
            raise ValueError(f"request {i}: prompt of {n} tokens does not fit {max_positions} positions")
        need = alone = pages_for(n, max_tokens, max_positions, keep)
        if alone > page_budget:
            raise ValueError(f"request {i} needs {alone * PAGE} cached positions, the cache holds {page_budget * PAGE}")
        key = None if alike is None else _Alike.key(alike[i])
        if key is not None:
            group, each, held = groups.get(key, (None, 0, 0))
            grown = _Alike.joined(group, i, alike[i])
            each += pages_for(n, max_tokens, max_positions, keep, True)
            need = alone if group is None else each - (len(grown.members) - 1) * grown.pages - held
        if cur and (used + need > page_budget or len(cur) >= slot_budget):
            batches.append(cur)
            cur, used, groups = [], 0, {}
            need = alone
            if key is not None:
                held = 0
                grown, each = _Alike.joined(None, i, alike[i]), pages_for(n, max_tokens, max_positions, keep, True)
        cur.append(i)
        used += need
        if key is not None:
            groups[key] = (grown, each, held + need)
    if cur:
        batches.append(cur)
    return batches


class SequenceState:
    """One request's progress; ``accept`` is the per-token decision."""

    def __init__(self, prompt: Sequence[int], max_tokens: int, stop_tokens, max_positions: int):
        self.prompt = list(prompt)
        self.max_tokens, self.max_positions = max_tokens, max_positions
        self.stop_tokens = frozenset(int(t) for t in stop_tokens)
        self.generated: List[int] = []
        self.fed = len(self.prompt)          # positions in the cache
        self.finish_reason: Optional[str] = None

    def may_continue(self) -> bool:
        """Whether a next token that is no stop token would be fed for another step."""
        return len(self.generated) + 1 < self.max_tokens and self.fed < self.max_positions

    def accept(self, token: int) -> bool:
        """Take the sampled token; True if it must be fed for another step."""
        if self.finish_reason is not None:
            raise RuntimeError("sequence already finished")
        if token in self.stop_tokens:
            self.finish_reason = "stop"
            return False
        self.generated.append(int(token))
        if len(self.generated) >= self.max_tokens or self.fed >= self.max_positions:
            self.finish_reason = "length"
            return False
        self.fed += 1
        return True


# ---------------------------------------------------------------------------
def generate(engine, prompts: Sequence[Sequence[int]], options: GenerationOptions) -> List[GenerationResult]:
    options.validate()
    import torch
    spec = engine.model.spec
    cache = engine.cache
    seed = options.seed if options.seed != 0 else time.time_ns()
    batches = plan_batches([len(p) for p in prompts], options.max_tokens, spec.max_positions,
                           cache.n_pages, cache.max_slots, options.cache_keep, [list(p) for p in prompts] if options.share_prefix else None)
    if options.cache_keep and not getattr(cache, "weigh", False):
        raise ValueError("cache_keep needs a cache that keeps the weight of its positions (load the model with weigh=True)")
    results: List[Optional[GenerationResult]] = [None] * len(prompts)
    prepare = getattr(engine, "prepare_decode", None)
    # kernels that gave up a bounded wait leave a status word: read where the host waits anyway, so that
    # an invalid result is an error here, as errors of the reference's forward pass end its loop
    # (runtime.go:1131-1165), and not a wrong token
    check = getattr(engine, "check_device", lambda: None)
    fetch = getattr(engine, "fetch", None) if prepare is not None else None
    for batch in batches:
        t_start = time.perf_counter()
        states = [SequenceState(prompts[i], options.max_tokens, options.stop_tokens, spec.max_positions)
                  for i in batch]
        sampler = DeviceSampler(options.sampler, [request_seed(seed, i) for i in batch],
                                [prompts[i] for i in batch], spec.vocab, engine.device)
        slots: List[Optional[int]] = [None] * len(batch)
        stats = [GenerationStats(prompt_tokens=len(prompts[i])) for i in batch]
        live = list(range(len(batch)))
        canceled = False
        try:
            skip = [0] * len(batch)                 # tokens of a prompt that lie on shared pages already
            if options.share_prefix:
                for members, n in begin_alike([s.prompt for s in states]):
                    # the first member runs the common tokens, the others go on from there
                    slots[members[0]] = engine.open()
                    engine.step([(slots[members[0]], states[members[0]].prompt[:n])], [[]])
                    for r in members:
                        skip[r] = n
                        if slots[r] is None:
                            slots[r] = engine.fork(slots[members[0]])
            for r in live:
                if slots[r] is None:
                    slots[r] = engine.open()
            logits = engine.step([(slots[r], states[r].prompt[skip[r]:]) for r in live])
            rows_dev = None
            first = True
            t_prefill_end = None
            while live:
                if rows_dev is None:
                    rows_dev = torch.tensor(live, dtype=torch.int32).to(engine.device)
                chosen = sampler.sample(logits, rows_dev)
                # While the device finishes the step and samples: the next step's descriptor, if every
                # sequence can go on.  An engine that can read its tokens on the device is given the
                # sampler's output and starts that step at once, before the host has seen the tokens, so
                # the device does not wait for the host between steps; should a sequence then end with
                # a stop token, the step has merely fed one token too many to a sequence that is closed,
                # and the rows of the others stand (a row does not depend on its neighbours).  Where sequences are
                # cut by the weight of their positions and share pages, that token would leave its weights on
                # pages that others are cut by: with a stop token about, such a step waits for the tokens.
                ahead, ahead_logits, sampled = None, None, None
                # (a sequence that has grown a page beyond what it may keep is cut before its next step)
                due = options.cache_keep and [slots[r] for r in live if cache.length(slots[r]) >= options.cache_keep + PAGE]
                if due:
                    engine.evict(due, options.cache_keep, options.cache_recent, options.cache_first)
                if prepare is not None and all(states[r].may_continue() for r in live):
                    ahead = prepare([slots[r] for r in live])
                    waits = options.cache_keep and options.stop_tokens and any(cache.shares_pages(slots[r]) for r in live)
                    if fetch is not None and not waits:
                        sampled = torch.cuda.Event()
                        sampled.record()
                        ahead_logits = engine.finish_decode(ahead, chosen)
                        ahead = None
                tokens = fetch(chosen, sampled) if sampled is not None else chosen.tolist()   # waits for the sampling
                now = time.perf_counter()
                if first:
                    check()                      # the prompts' step is over: the host has its tokens
                    t_prefill_end = now
                    for r in live:
                        stats[r].prefill_time = now - t_start
                        stats[r].ttft = now - t_start
                    first = False
                nxt, runs, kept = [], [], []
                for i, (r, tok) in enumerate(zip(live, tokens)):
                    stats[r].token_times.append(now - t_start)
                    emitted = len(states[r].generated)
                    goes_on = states[r].accept(tok)
                    if options.on_token is not None and len(states[r].generated) > emitted:
                        if options.on_token(batch[r], tok) is False:
                            canceled = True
                    if goes_on:
                        nxt.append(r)
                        runs.append((slots[r], [tok]))
                        kept.append(i)
                    else:
                        engine.close(slots[r])
                        slots[r] = None
                        stats[r].total_time = now - t_start
                        stats[r].decode_time = now - t_prefill_end
                if len(nxt) != len(live):
                    rows_dev = None
                live = nxt
                if canceled or (options.should_stop is not None and options.should_stop()):
                    canceled = True
                    break
                if runs:
                    if ahead_logits is not None:
                        logits = ahead_logits if len(kept) == len(tokens) else \
                            ahead_logits.index_select(0, torch.tensor(kept, dtype=torch.int64).to(engine.device))
                    elif ahead is not None and len(runs) == len(tokens):
                        logits = engine.finish_decode(ahead, tokens)
                    else:
                        logits = engine.step(runs)
            check()                              # the batch is over and the host has waited for its last tokens
        finally:
            for s in slots:
                if s is not None:
                    engine.close(s)
        now = time.perf_counter()
        for r, i in enumerate(batch):
            st = states[r]
            if st.finish_reason is None:
                st.finish_reason = "canceled"
                stats[r].total_time = now - t_start
                stats[r].decode_time = now - (t_prefill_end or now)
            stats[r].generated_tokens = len(st.generated)
            results[i] = GenerationResult(st.generated, st.finish_reason, stats[r])
        if canceled:
            done = [r if r is not None else GenerationResult([], "canceled", GenerationStats()) for r in results]
            raise GenerationCanceled(done)
    return results
