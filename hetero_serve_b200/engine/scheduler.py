"""The continuous-batching scheduler above the step function.

In the manner of the reference's per-device worker (heteroserve/worker/worker.py):

* requests are admitted in arrival order; admission reserves pages for the whole
  prompt after a prefix match (worker.py:378-416, heteroserve/kv/blocks.py:168-201);
* prompts are cut into portions of at most ``max_prefill_tokens`` (worker.py:599-657);
* every running request decodes one token per step, at most ``max_batch`` of them
  (worker.py:586-589, 659-703);
* a request finishes after ``max_new_tokens``, at an end-of-sequence token if
  ``stop_at_eos`` (worker.py:714-715), or when it reaches the context limit; its full
  pages are published for reuse and everything it holds is given back (worker.py:721-764);
* when pages run out while decoding, the NEWEST running request is preempted by
  recomputation: its pages are given back, its tokens kept, and it is prefilled again
  later (worker.py:738-757).

Two policies compose a step.  ``prefill_first`` is the reference's: while any prompt is
unfinished, a step is one portion of the oldest such prompt; otherwise a step decodes
(worker.py:580-591).  ``mixed`` puts the decoded tokens of all running requests and, in
what is left of the token budget, portions of waiting prompts into the same step.

What happens when pages run out — decided here:

1. at admission: the request waits (and blocks those behind it, keeping arrival order)
   until pages for its whole prompt are obtainable; a prompt that could never fit the
   pool is refused when it is submitted;
2. while decoding: preempt the newest running request and try again; a request that
   preempts itself sits the step out.  A request that has outgrown the whole pool on its
   own (nothing else is live and it still cannot be admitted) ends with the tokens it
   has, ``finish_reason == "out_of_pages"``.  A preempted request goes to the FRONT of the
   waiting queue, keeps its sampled tokens, and is prefilled again over prompt + outputs
   (all but the last token, which decoding feeds).  Because the random draw of a token
   depends only on (seed, position), a preempted request continues exactly as it would
   have.

Pipelining (``pipeline=True``).  ``step_fn`` may return, instead of a list of tokens, an object
whose ``tokens_host()`` yields them later.  The scheduler then launches step i+1 BEFORE it reads
step i's tokens: a request whose latest token is still on its way decodes with
``FROM_DEVICE`` (the step reads the token from device memory), so the host's work and the
transfer hide behind the device's.  What needs the token itself waits for it: a request that
reaches ``max_new_tokens`` or the context limit with the token in flight sits the next step
out (its end is known by counting); an end-of-sequence token is seen one step late, and the
request's part in the step launched meanwhile is discarded (its pages were still its own when
that step was launched, and whoever gets them next is ordered behind it on the stream);
preemption first waits for the tokens in flight, since a preempted request is prefilled again
over all of its tokens; a request whose grammar has to see the token before it can say what may
follow sits out the steps in which its token is in flight.

Several answers to one prompt (``Request.samples``).  The prompt is prefilled once, all but its
last token; then the request is forked (``fork_fn``): its full pages are shared, its last page and
state copied, and every sample decodes on its own, the last prompt token first, with a seed of its
own (``seed + i``).  A sample for which no page or slot can be had queues as a request of its own
at the front, and finds the prompt's pages by prefix reuse.  Sample i is named ``{req_id}#{i}``; of two
requests of one name the later waits until the earlier has ended.
"""

from __future__ import annotations

import itertools
import time
from collections import Counter, deque
from dataclasses import dataclass, field, replace
from typing import Callable, Hashable, Mapping, Sequence

from ..cache import CacheManager, OutOfPages
from ..kernels.ops import MAX_ALTERNATIVES
from ..sampling import LogitRules, is_whole, mask_words
from .step import FROM_DEVICE, StepEntry


class SeqState:                     # heteroserve/worker/protocol.py:38-42
    WAITING = "waiting"             # queued; nothing resident
    PREFILL = "prefill"             # admitted; prompt partly resident
    RUNNING = "running"             # generating
    DONE = "done"


class RequestRefused(ValueError):
    """A request that can never run: empty, too long, or larger than the whole pool."""


_ids = itertools.count()


@dataclass
class Request:
    """What a caller submits (heteroserve/sched/router.py:36-44, worker.py:53-61)."""

    prompt_ids: Sequence[int]
    max_new_tokens: int = 32
    temperature: float = 0.0
    top_k: int = 0
    seed: int = 0
    stop_at_eos: bool = True
    req_id: Hashable = field(default_factory=lambda: f"req-{next(_ids)}")
    # what may be said (see ``sampling.rules``)
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Mapping[int, float] | None = None
    grammar: object | None = None       # ``allowed(output_ids)``, asked with each answer's own tokens
    logprobs: int | None = None         # scores of every token, with this many alternatives
    samples: int = 1                    # answers to the prompt; answer i draws with seed + i

    def rules(self) -> LogitRules:
        return LogitRules(float(self.repetition_penalty), float(self.presence_penalty),
                          float(self.frequency_penalty), dict(self.logit_bias or {}))


@dataclass
class SequenceState:
    """A request inside the scheduler (heteroserve/worker/worker.py:53-87)."""

    request: Request
    output_ids: list[int] = field(default_factory=list)
    n_kv: int = 0                       # positions resident in the cache
    state: str = SeqState.WAITING
    admitted: bool = False
    cached_prefix_tokens: int = 0
    prefill_tokens_computed: int = 0
    preemptions: int = 0
    finish_reason: str = ""
    error: str = ""                     # what its grammar failed with (finish_reason "grammar_error")
    pending: int = 0                    # tokens sampled for it that the host has not read yet
    rules: LogitRules | None = None     # None: none that change anything
    recorded: bool = False              # its tokens are on the device, for penalties
    scores: list = field(default_factory=list)      # TokenLogprobs of its tokens, if asked for
    # the other answers to its prompt, while they wait for it to be prefilled, and once forked
    to_fork: list["SequenceState"] = field(default_factory=list)
    siblings: list["SequenceState"] = field(default_factory=list)
    t_submit: float = 0.0
    t_admit: float = 0.0
    t_first_token: float = 0.0
    t_done: float = 0.0

    @property
    def req_id(self):
        return self.request.req_id

    @property
    def ctx(self) -> list[int]:
        return list(self.request.prompt_ids) + self.output_ids

    @property
    def prefill_target(self) -> int:
        """How far prefill must reach before decoding takes over (worker.py:79-83): the last
        token is decoding's where it has been generated, or is fed by every sample."""
        n = len(self.request.prompt_ids) + len(self.output_ids)
        return n - 1 if self.output_ids or self.request.samples > 1 else n


@dataclass
class Planned:
    """One entry of a planned step."""

    seq: SequenceState
    start: int
    tokens: list[int]
    samples: bool           # the last of these tokens yields a new token


@dataclass
class SchedulerStats:
    steps: int = 0
    prefill_steps: int = 0
    decode_steps: int = 0
    mixed_steps: int = 0
    tokens_generated: int = 0
    tokens_prefilled: int = 0
    tokens_saved_by_cache: int = 0
    preemptions: int = 0
    finished: int = 0


class Scheduler:
    """Decides what each step runs.  ``step_fn(entries)`` runs a batch through the step
    function with device sampling and returns one token per entry that wanted one, in entry
    order — as a list, or as an object whose ``tokens_host()`` returns that list when asked
    (see "Pipelining" above); the scheduler owns everything around it."""

    def __init__(self, manager: CacheManager, step_fn: Callable[[list[StepEntry]], object],
                 *, max_batch: int, max_prefill_tokens: int, max_ctx: int,
                 eos_token_id: int | None, policy: str = "prefill_first",
                 vocab_size: int | None = None, clock: Callable[[], float] = time.perf_counter,
                 pipeline: bool = False,
                 fork_fn: Callable[[Hashable, Hashable], object] | None = None):
        if policy not in ("prefill_first", "mixed"):
            raise ValueError(f"unknown policy {policy!r}")
        self.manager = manager
        self.step_fn = step_fn
        self.max_batch = max_batch
        self.max_prefill_tokens = max_prefill_tokens
        self.max_ctx = max_ctx
        self.eos_token_id = eos_token_id
        self.policy = policy
        self.vocab_size = vocab_size
        self.clock = clock
        self.waiting: deque[SequenceState] = deque()
        self.active: list[SequenceState] = []          # admitted, in admission order
        self.finished: list[SequenceState] = []
        self.stats = SchedulerStats()
        self.pipeline = bool(pipeline)
        self.fork_fn = fork_fn or manager.fork
        self._in_phase = True
        self._inflight: tuple[list[Planned], object] | None = None   # launched, tokens unread
        self._late_done: list[SequenceState] = []     # finished while a plan was being made
        self._names: Counter = Counter()              # of the requests that have not ended

    # -- submission -----------------------------------------------------------
    def add(self, request: Request) -> SequenceState:
        n = len(request.prompt_ids)
        if n == 0:
            raise RequestRefused("the prompt is empty")
        if n >= self.max_ctx:
            raise RequestRefused(f"the prompt has {n} tokens; with one generated token it "
                                 f"would exceed the context limit of {self.max_ctx}")
        if request.max_new_tokens <= 0:
            raise RequestRefused("max_new_tokens must be positive")
        if self.vocab_size is not None:
            bad = [t for t in request.prompt_ids if not 0 <= t < self.vocab_size]
            if bad:
                raise RequestRefused(f"token id {bad[0]} is outside [0, {self.vocab_size})")
        for gi, pool in enumerate(self.manager.pools):
            if self.manager.pages_for(n + 1, gi) > pool.num_pages:
                raise RequestRefused(
                    f"the prompt needs {self.manager.pages_for(n + 1, gi)} pages, the pool has "
                    f"{pool.num_pages}")
        try:
            rules = request.rules()
            rules.check(self.vocab_size)
        except (TypeError, ValueError, OverflowError) as exc:
            raise RequestRefused(str(exc)) from None
        if request.grammar is not None and not callable(getattr(request.grammar, "allowed", None)):
            raise RequestRefused("a grammar needs a method allowed(output_ids)")
        if request.grammar is not None and self.vocab_size is None:
            raise RequestRefused("a grammar needs a vocabulary size")
        most = MAX_ALTERNATIVES if self.vocab_size is None else min(MAX_ALTERNATIVES, self.vocab_size)
        if request.logprobs is not None and not (is_whole(request.logprobs)
                                                 and 0 <= request.logprobs <= most):
            raise RequestRefused(f"logprobs={request.logprobs}: between 0 and {most} alternatives")
        if not (is_whole(request.samples) and request.samples >= 1):
            raise RequestRefused(f"samples={request.samples}: at least one answer")
        now = self.clock()
        state = lambda r: SequenceState(request=r, t_submit=now,              # noqa: E731
                                        rules=None if rules.neutral else rules)
        seq = state(request)
        for i in range(1, request.samples):
            seq.siblings.append(state(replace(request, seed=request.seed + i, samples=1,
                                              req_id=f"{request.req_id}#{i}")))
        answers = [seq, *seq.siblings]
        if len(answers) > 1 and any(s.req_id in self._names for s in answers):
            raise RequestRefused(f"request {request.req_id!r} is known already")
        self._names.update(s.req_id for s in answers)
        seq.to_fork = list(seq.siblings)
        self.waiting.append(seq)
        return seq

    def has_work(self) -> bool:
        return bool(self.waiting or self.active or self._inflight is not None)

    def pages_promised(self) -> list[int]:
        """Per group the pages that the longest request without a token of its own (or, preempted,
        without pages) needs: smaller pools would never admit what :meth:`add` took."""
        promised = [0] * len(self.manager.pools)
        for seq in [*self.waiting, *self.active]:
            for s in (seq, *seq.to_fork):
                if s.admitted and (s.output_ids or s.pending):
                    continue                        # (ends with what it has, should it come to that)
                n = len(s.ctx) + (not s.output_ids)
                for gi in range(len(promised)):
                    promised[gi] = max(promised[gi], self.manager.pages_for(n, gi))
        return promised

    # -- admission --------------------------------------------------------------
    def _admit(self) -> None:
        """Admit from the front of the queue while a state slot and the pages of the whole
        prompt (after the prefix match) can be had.  The head blocks those behind it."""
        mgr = self.manager
        while self.waiting:
            seq = self.waiting[0]
            if mgr.free_slots() == 0 or seq.req_id in mgr:     # (another of its name: after that)
                return
            ctx = seq.ctx
            target = seq.prefill_target
            opened = mgr.open(seq.req_id, ctx[:target] if target else None)
            try:
                mgr.reserve(seq.req_id, max(target, 1))
            except OutOfPages:
                mgr.close(seq.req_id)
                # correct the counters the failed attempt touched
                mgr.hit_tokens -= opened.cached_tokens
                mgr.miss_tokens -= (target - opened.cached_tokens) if target else 0
                return
            self.waiting.popleft()
            seq.admitted = True
            seq.n_kv = min(opened.cached_tokens, target)
            if not seq.preemptions:
                seq.cached_prefix_tokens = seq.n_kv
                seq.t_admit = self.clock()
            self.stats.tokens_saved_by_cache += seq.n_kv
            seq.state = SeqState.PREFILL if seq.n_kv < target else SeqState.RUNNING
            seq.recorded = False
            self.active.append(seq)
            if seq.state == SeqState.RUNNING:
                self._fork_samples(seq)

    def _fork_samples(self, seq: SequenceState) -> None:
        """The prompt is resident: start the other answers to it."""
        at = self.active.index(seq) + 1
        todo, seq.to_fork = deque(seq.to_fork), []
        try:
            while todo and todo[0].req_id not in self.manager:
                other = todo[0]
                try:
                    self.fork_fn(seq.req_id, other.req_id)
                except OutOfPages:
                    break
                todo.popleft()
                other.admitted, other.state, other.n_kv = True, SeqState.RUNNING, seq.n_kv
                other.cached_prefix_tokens = seq.n_kv
                other.t_admit = self.clock()
                self.stats.tokens_saved_by_cache += seq.n_kv
                self.active.insert(at, other)
                at += 1
        finally:
            self.waiting.extendleft(reversed(todo))     # they queue, whatever kept them

    # -- planning ----------------------------------------------------------------
    def plan(self) -> list[Planned]:
        """Choose the entries of the next step (reserving pages; may preempt)."""
        self._admit()
        prefilling = [s for s in self.active if s.state == SeqState.PREFILL]
        planned: list[Planned] = []
        budget = self.max_prefill_tokens
        if self.policy == "prefill_first":
            if prefilling:
                return [self._portion(prefilling[0], budget)]
            return self._decodes()
        planned = self._decodes()
        budget -= len(planned)
        for seq in prefilling:
            if budget <= 0:
                break
            if seq.state != SeqState.PREFILL:      # preempted meanwhile
                continue
            p = self._portion(seq, budget)
            planned.append(p)
            budget -= len(p.tokens)
        return planned

    def _portion(self, seq: SequenceState, budget: int) -> Planned:
        if seq.prefill_tokens_computed == 0 and self.manager.prefix_cache:
            # nothing of it has run yet: pages published since its admission (by requests
            # admitted together with it) may cover more of its prompt by now
            before = seq.n_kv
            got = min(self.manager.rematch(seq.req_id, seq.ctx[:seq.prefill_target]),
                      seq.prefill_target)
            if got > before:
                seq.n_kv = got
                if not seq.preemptions:
                    seq.cached_prefix_tokens = got
                self.stats.tokens_saved_by_cache += got - before
        start = seq.n_kv
        end = min(start + budget, seq.prefill_target)
        toks = seq.ctx[start:end]
        # pages for the whole prompt were reserved at admission
        samples = end >= len(seq.ctx)
        return Planned(seq, start, toks, samples)

    def _decodes(self) -> list[Planned]:
        mgr = self.manager
        planned: list[Planned] = []
        running = [s for s in self.active if s.state == SeqState.RUNNING][: self.max_batch]
        # requests with grammars decode in the same steps (every second one, pipelined) instead of
        # taking turns by halves; they sit out one step in a row for that, no more
        self._in_phase = not self._in_phase or not any(
            s.pending and s.request.grammar is not None for s in running)
        for seq in running:
            if seq.pending and self._ends_by_count(seq, seq.pending):
                continue                            # its token in flight is its last
            if seq.request.grammar is not None and (seq.pending or not self._in_phase):
                continue                            # its token in flight decides, or another's
            while seq.state == SeqState.RUNNING:    # else: preempted, or ended while we waited
                try:
                    mgr.reserve(seq.req_id, seq.n_kv + 1)
                    tok = FROM_DEVICE if seq.pending else seq.ctx[seq.n_kv]
                    planned.append(Planned(seq, seq.n_kv, [tok], True))
                    break
                except OutOfPages:
                    victim = self._preempt_newest()
                    if victim is seq or victim is None:
                        break
                    planned = [p for p in planned if p.seq is not victim]
        return planned

    def _ends_by_count(self, seq: SequenceState, extra: int) -> bool:
        """Would ``extra`` more tokens end the request whatever they are?"""
        n = len(seq.output_ids) + extra
        return (n >= seq.request.max_new_tokens
                or len(seq.request.prompt_ids) + n >= self.max_ctx)

    def _preempt_newest(self) -> SequenceState | None:
        """Recompute-preemption of the newest running request (worker.py:738-757)."""
        if self._inflight is not None:
            # a preempted request is prefilled again over all its tokens: have them first
            self._late_done.extend(self._resolve())
        running = [s for s in self.active if s.state == SeqState.RUNNING]
        if not running:
            return None
        victim = running[-1]
        self.manager.publish(victim.req_id, victim.ctx[: victim.n_kv])
        self.manager.close(victim.req_id)
        self.active.remove(victim)
        victim.n_kv = 0
        victim.admitted = False
        victim.state = SeqState.WAITING
        victim.preemptions += 1
        victim.recorded = False
        self.stats.preemptions += 1
        self.waiting.appendleft(victim)
        return victim

    def _masks(self, planned: list[Planned]) -> dict:
        """What the planned requests' grammars allow next, packed, by request.  A request whose
        grammar allows nothing any more (that its biases do not rule out) ends here, and so does
        one whose grammar raises or answers with anything but tokens of the vocabulary."""
        masks = {}
        for p in planned:
            grammar = p.seq.request.grammar
            if grammar is None or not p.samples:
                continue
            try:
                words = mask_words(grammar.allowed(tuple(p.seq.output_ids)), self.vocab_size)
            except Exception as exc:                # the caller's own code: its request alone ends
                words = None
                p.seq.error = f"{type(exc).__name__}: {exc}"
            if words is not None and p.seq.rules is not None:
                words = p.seq.rules.leave(words, self.vocab_size)
            if p.seq.error or (words is not None and not words.any()):
                p.seq.finish_reason = "grammar_error" if p.seq.error else "grammar"
                self._finish(p.seq, self.clock())
                self._late_done.append(p.seq)
            elif words is not None:
                masks[p.seq.req_id] = words
        return masks

    # -- running a step -------------------------------------------------------------
    def step(self) -> list[SequenceState]:
        """Plan and launch one step; returns the requests whose end became known in it.  With
        ``pipeline`` the tokens of the step launched here are read in the NEXT call."""
        planned = self.plan()
        # requests that ended while the plan waited for tokens in flight have left it
        planned = [p for p in planned
                   if p.seq.state in (SeqState.PREFILL, SeqState.RUNNING)]
        masks = self._masks(planned)
        planned = [p for p in planned if p.seq.state != SeqState.DONE]
        done, self._late_done = self._late_done, []
        if not planned:
            if self._inflight is not None:
                done.extend(self._resolve())
                return done
            if self.waiting and not self.active and not done:
                head = self.waiting[0]
                if head.output_ids:
                    # it outgrew the whole pool while generating: end it with what it has
                    self.waiting.popleft()
                    head.state, head.finish_reason = SeqState.DONE, "out_of_pages"
                    self._ended(head)
                    head.t_done = self.clock()
                    self.finished.append(head)
                    self.stats.finished += 1
                    return done + [head]
                raise RequestRefused(
                    f"request {head.req_id!r} cannot be admitted although nothing else is "
                    f"running: the pool is too small for it, or its name is open elsewhere")
            return done
        entries = []
        for p in planned:
            r, seq = p.seq.request, p.seq
            entry = StepEntry(
                seq.req_id, p.tokens, want=[len(p.tokens) - 1] if p.samples else (),
                temperature=r.temperature, top_k=r.top_k, seed=r.seed)
            if p.samples:
                entry.logprobs, entry.rules = r.logprobs, seq.rules
                entry.allowed = masks.get(seq.req_id)
                if seq.rules is not None and seq.rules.penalises and not seq.recorded:
                    entry.history = (r.prompt_ids, list(seq.output_ids))
            entries.append(entry)
        result = self.step_fn(entries)
        for p, entry in zip(planned, entries):
            p.seq.recorded |= entry.history is not None
        resident: list[SequenceState] = []
        n_dec = sum(1 for p in planned if len(p.tokens) == 1 and p.seq.state == SeqState.RUNNING)
        for p in planned:
            seq = p.seq
            was_prefill = seq.state == SeqState.PREFILL
            seq.n_kv = p.start + len(p.tokens)
            if was_prefill:
                seq.prefill_tokens_computed += len(p.tokens)
                self.stats.tokens_prefilled += len(p.tokens)
                if seq.n_kv >= seq.prefill_target:
                    # publish the finished prompt so that others can share it (worker.py:635-645)
                    self.manager.publish(seq.req_id, seq.ctx[: seq.n_kv])
                    seq.state = SeqState.RUNNING
                    if seq.to_fork:
                        resident.append(seq)
            if p.samples:
                seq.pending += 1
        self.stats.steps += 1
        if n_dec == len(planned):
            self.stats.decode_steps += 1
        elif n_dec == 0:
            self.stats.prefill_steps += 1
        else:
            self.stats.mixed_steps += 1
        earlier, self._inflight = self._inflight, (planned, result)
        failed = None
        for seq in resident:
            try:
                self._fork_samples(seq)
            except Exception as exc:                # (raised once nothing can be lost by it)
                failed = failed or exc
        if earlier is not None:
            done.extend(self._read(earlier))
        if not self.pipeline:
            done.extend(self._resolve())
        if failed is not None:
            self._late_done.extend(done)            # (the next call tells of them)
            raise failed
        return done

    def _resolve(self) -> list[SequenceState]:
        """Read the tokens of the step in flight, if any."""
        inflight, self._inflight = self._inflight, None
        return self._read(inflight) if inflight is not None else []

    def _read(self, inflight) -> list[SequenceState]:
        planned, result = inflight
        tokens = result.tokens_host() if hasattr(result, "tokens_host") else result
        it = iter(tokens)
        scores = itertools.repeat(None)
        if any(p.samples and p.seq.request.logprobs is not None for p in planned) \
                and hasattr(result, "logprobs_host"):
            scores = iter(result.logprobs_host())
        done: list[SequenceState] = []
        now = self.clock()
        for p in planned:
            if not p.samples:
                continue
            tok, score = int(next(it)), next(scores)
            seq = p.seq
            if seq.state == SeqState.DONE:
                continue            # ended (or aborted) while this step was in flight
            seq.pending -= 1
            seq.output_ids.append(tok)
            if score is not None:
                seq.scores.append(score)
            self.stats.tokens_generated += 1
            if not seq.t_first_token:
                seq.t_first_token = now
            if self._finished(seq, tok):
                self._finish(seq, now)
                done.append(seq)
        return done

    def _finished(self, seq: SequenceState, tok: int) -> bool:
        r = seq.request
        if len(seq.output_ids) >= r.max_new_tokens:
            seq.finish_reason = "max_new_tokens"
        elif r.stop_at_eos and self.eos_token_id is not None and tok == self.eos_token_id:
            seq.finish_reason = "eos"
        elif len(r.prompt_ids) + len(seq.output_ids) >= self.max_ctx:
            seq.finish_reason = "max_ctx"
        return bool(seq.finish_reason)

    def _finish(self, seq: SequenceState, now: float) -> None:
        seq.state = SeqState.DONE
        seq.t_done = now
        self._ended(seq)
        # what was generated becomes reusable too (worker.py:720-721)
        self.manager.publish(seq.req_id, seq.ctx[: seq.n_kv])
        self.manager.close(seq.req_id)
        self.active.remove(seq)
        self.finished.append(seq)
        self.stats.finished += 1

    def _ended(self, seq: SequenceState) -> None:
        """Its name may be taken again."""
        self._names[seq.req_id] -= 1
        if self._names[seq.req_id] <= 0:
            del self._names[seq.req_id]

    def abort(self, req_id) -> bool:
        """Drop a request wherever it is; what it holds is given back.  Answers that wait to be
        forked off it are dropped with it."""
        for seq in [*self.active, *self.waiting]:
            for other in seq.to_fork:
                if req_id in (seq.req_id, other.req_id):
                    other.state, other.finish_reason = SeqState.DONE, "aborted"
                    self._ended(other)
            forked = [o for o in seq.to_fork if o.state != SeqState.DONE]
            if seq.req_id != req_id and len(forked) < len(seq.to_fork):
                seq.to_fork = forked
                return True
            seq.to_fork = forked
        for seq in list(self.active):
            if seq.req_id == req_id:
                self.manager.close(req_id)
                self.active.remove(seq)
                seq.state, seq.finish_reason = SeqState.DONE, "aborted"
                self._ended(seq)
                return True
        for seq in list(self.waiting):
            if seq.req_id == req_id:
                self.waiting.remove(seq)
                seq.state, seq.finish_reason = SeqState.DONE, "aborted"
                self._ended(seq)
                return True
        return False

    def state_message(self) -> dict:
        """Counters in the manner of the worker's state message (worker.py:786-812)."""
        s = self.stats
        return {
            "kv": self.manager.snapshot(),
            "queued": len(self.waiting) + sum(1 for q in self.active if q.state == SeqState.PREFILL),
            "running": sum(1 for q in self.active if q.state == SeqState.RUNNING),
            "steps": s.steps, "prefill_steps": s.prefill_steps, "decode_steps": s.decode_steps,
            "mixed_steps": s.mixed_steps, "tokens_generated": s.tokens_generated,
            "tokens_prefilled": s.tokens_prefilled,
            "tokens_saved_by_cache": s.tokens_saved_by_cache, "preemptions": s.preemptions,
            "finished": s.finished,
        }
