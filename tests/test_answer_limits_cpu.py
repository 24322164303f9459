"""What may not disturb other requests, without a GPU: bad text to score, numbers out of range, grammars
that fail, queues, names, refused copies.  The engine over the plain twins of the kernels."""

import math
from collections import deque

import numpy as np
import pytest

from plain_answers import PlainAnswerOps
from test_answers_cpu import engine
from test_scheduler import expected_outputs, make, prompt, run
from hetero_serve_b200 import EngineConfig, LLMEngine, LogitRules, Request, StepEntry
from hetero_serve_b200.cache import OutOfPages
from hetero_serve_b200.engine.scheduler import RequestRefused
from hetero_serve_b200.kernels import KernelError
from hetero_serve_b200.engine.step import StepError
from hetero_serve_b200.sampling import mask_words


class ReportingOps(PlainAnswerOps):
    """Reports tokens outside the vocabulary in the runner's status word, as the kernel does."""

    def token_logprobs(self, logprob, rank, logits, tokens, top_ids=None, top_logprobs=None):
        super().token_logprobs(logprob, rank, logits, tokens, top_ids, top_logprobs)
        outside = (tokens != -1) & ((tokens < 0) | (tokens >= logits.shape[1]))
        if bool(outside.any()):
            self.status |= 1


def reporting(tiny, **kw):
    eng = engine(tiny, **kw)
    eng.runner.ops.__class__ = ReportingOps
    eng.runner.ops.status = eng.runner.status
    return eng


# -- scores of given text --------------------------------------------------------------------------


@pytest.mark.parametrize("pipeline", [False, True])
def test_a_bad_text_to_score_is_refused_beside_a_live_request(tiny_models, pipeline):
    """The first token, the first of a portion (24 here), one within and the last, which no step feeds."""
    tiny = tiny_models["tiny_a"]
    want = engine(tiny).generate([tiny.tokens(9, 4)], 14, stop_at_eos=False)[0]
    eng = reporting(tiny, pipeline=pipeline)
    live = eng.submit_nowait(Request(tiny.tokens(9, 4), 14, stop_at_eos=False))
    eng.step(), eng.step()
    text = tiny.tokens(60, 3)
    for at in (0, 24, 48, 30, 59):
        for bad in (-1, -2, 512, 99999, 2 ** 31, 2 ** 40):
            with pytest.raises(StepError):
                eng.score(text[:at] + [bad] + text[at + 1:])
        assert int(eng.runner.status) == 0
        eng.step()
    for one in ([-1], [512]):
        with pytest.raises(StepError):
            eng.score(one)
    eng.run_until_done()
    assert live.output_ids == want and live.state == "done"
    eng.runner.manager.check()
    assert eng.runner.manager.live() == []


def test_a_text_longer_than_the_model_is_refused_before_anything_runs(tiny_models):
    tiny = tiny_models["tiny_a"]                                  # 128 positions
    eng = engine(tiny)
    before = eng.runner.steps_run
    assert len(eng.score(tiny.tokens(129, 1))) == 128             # the last token is not fed
    ran = eng.runner.steps_run
    assert ran > before
    with pytest.raises(StepError):
        eng.score(tiny.tokens(130, 1))
    assert eng.runner.steps_run == ran and eng.runner.manager.live() == []


# -- numbers that 32 bits do not hold -----------------------------------------------------------------


@pytest.mark.parametrize("bad", [
    dict(repetition_penalty=1e-50), dict(repetition_penalty=1e-30), dict(repetition_penalty=1e30),
    dict(repetition_penalty=1e300), dict(presence_penalty=1e300), dict(presence_penalty=-1e39),
    dict(presence_penalty=1e30), dict(frequency_penalty=1e300), dict(frequency_penalty=-1e30),
    dict(logit_bias={3: 1e39}), dict(logit_bias={3: 1e300}), dict(logit_bias={3: 1e30}),
    dict(logit_bias={3: 3.4e38})])
def test_numbers_that_leave_no_finite_logit_are_refused(bad, recwarn):
    sch, _fake, _mgr = make()
    with pytest.raises(RequestRefused):
        sch.add(Request(prompt(5), **bad))
    assert not sch.has_work() and not recwarn.list


def test_numbers_at_the_edges_keep_logits_finite(recwarn):
    """The largest numbers that are taken, over the largest logits and counts there are: finite in 32
    bits, and still finite divided by a temperature of 1e-6."""
    most = 1e20
    low, high = LogitRules(1 / most, -most, -most, {3: most}), LogitRules(most, most, most, {3: -most})
    for rules in (low, high):
        for x in (1e8, -1e8, 0.0):
            y = x / rules.repetition if x > 0 else x * rules.repetition
            y += rules.bias_values[0] - rules.frequency * 1e7 - rules.presence
            assert math.isfinite(np.float32(y)) and math.isfinite(np.float32(y / 1e-6))
    lowest = float(np.finfo(np.float32).min)
    rules = LogitRules(bias={0: lowest, 1: -1e300, 2: -math.inf, 5: -1e10, 9: 1e-50, 10: 0.1})
    # finite: not ruled out, and far below every logit
    assert rules.bias_values.tolist() == [np.float32(-1e20), np.float32(-1e20), -math.inf,
                                          np.float32(-1e10), 0.0, np.float32(0.1)]
    assert rules.ruled_out == [2] and not recwarn.list


@pytest.mark.parametrize("temperature", [0.0, 0.5, 1.0])
def test_finite_biases_as_low_as_they_go_leave_the_rest(tiny_models, temperature):
    """Two tokens that a grammar allows, both biased to the type's lowest value: one of them is drawn."""
    tiny = tiny_models["tiny_b"]
    lowest = float(np.finfo(np.float32).min)

    class Two:
        def allowed(self, output):
            return [4, 9]
    seq = engine(tiny).submit(Request(tiny.tokens(9, 1), 6, temperature, grammar=Two(),
                                      logit_bias={4: lowest, 9: lowest}))
    assert len(seq.output_ids) == 6 and set(seq.output_ids) <= {4, 9}


# -- rules that leave no token -------------------------------------------------------------------------


def test_biases_that_rule_everything_out_are_refused(tiny_models):
    sch, _fake, _mgr = make()                                     # 97 tokens
    everything = {t: -math.inf for t in range(97)}
    with pytest.raises(RequestRefused, match="no token"):
        sch.add(Request(prompt(5), logit_bias=everything))
    sch.add(Request(prompt(5), logit_bias={**everything, 96: -1e30}))
    tiny = tiny_models["tiny_a"]                                  # 512 tokens, 16 words
    rn = engine(tiny).runner
    none = LogitRules(bias={t: -math.inf for t in range(512)})
    even = LogitRules(bias={t: -math.inf for t in range(0, 512, 2)})
    odd_mask = np.full(16, np.uint32(0xAAAAAAAA)).view(np.int32)
    for temperature in (0.0, 0.9):
        for kw in (dict(rules=none), dict(rules=none, allowed=odd_mask), dict(rules=even, allowed=~odd_mask)):
            with pytest.raises(StepError, match="no token"):
                rn.step([StepEntry("a", [1, 2], want=[1], temperature=temperature, **kw)], sample=True)
        assert rn.manager.live() == []
        res = rn.step([StepEntry("a", [1, 2], want=[1], temperature=temperature, rules=even,
                                 allowed=odd_mask)], sample=True)
        assert res.tokens_host()[0] % 2 == 1
        rn.close("a")


def test_masks_without_the_ruled_out_of_any_vocabulary():
    rules = LogitRules(bias={1: -math.inf, 33: -math.inf, 5: -2.0})
    for vocab in (40, 97, 40, 64):
        every = mask_words(range(vocab), vocab)
        assert np.array_equal(rules.leave(every, vocab),
                              mask_words([t for t in range(vocab) if t not in (1, 33)], vocab))
        assert np.array_equal(every, mask_words(range(vocab), vocab))          # the caller's own stays


# -- a cache of another size under a queue -----------------------------------------------------------


def finish(eng, limit=400):
    for _ in range(limit):
        if not eng.has_work():
            return
        eng.step()
        eng.runner.manager.check()
    raise AssertionError("requests are stuck")


def test_a_cache_is_not_made_too_small_for_a_queued_request(tiny_models):
    """Pages of 16: prompts of 60 and 5 tokens wait; what the longer one needs stays."""
    tiny = tiny_models["tiny_a"]
    prompts = [tiny.tokens(60, 1), tiny.tokens(5, 2)]
    want = engine(tiny).generate(prompts, 4, stop_at_eos=False)
    eng = engine(tiny)
    seqs = [eng.submit_nowait(Request(p, 4, stop_at_eos=False)) for p in prompts]
    for size in (3, 2, 1):
        with pytest.raises(OutOfPages):
            eng.resize_cache(size)
        assert eng.config.num_blocks == 24 == eng.runner.manager.pools[0].num_pages
    eng.resize_cache(4)
    finish(eng)
    assert [s.output_ids for s in seqs] == want
    eng.resize_cache(2)                                       # nobody waits any more
    assert eng.submit(Request(prompts[1], 4, stop_at_eos=False)).output_ids == want[1]
    with pytest.raises(RequestRefused):
        eng.submit(Request(prompts[0], 4))


def test_a_cache_is_not_made_too_small_for_answers_still_to_be_forked(tiny_models):
    """17 tokens, all but the last resident on one page: every answer needs a second one."""
    tiny = tiny_models["tiny_a"]
    p = tiny.tokens(17, 1)
    want = [r.output_ids for r in engine(tiny).submit_samples(Request(p, 4, 0.9, samples=3, stop_at_eos=False))]
    eng = engine(tiny, max_prefill_tokens=8)
    seq = eng.submit_nowait(Request(p, 4, 0.9, samples=3, stop_at_eos=False))
    eng.step()
    assert eng.runner.manager.pools[0].num_held() == 1
    with pytest.raises(OutOfPages):
        eng.resize_cache(1)
    eng.resize_cache(2)
    finish(eng)
    assert [s.output_ids for s in (seq, *seq.siblings)] == want


@pytest.mark.parametrize("pipeline", [False, True])
def test_preempted_requests_count_and_a_larger_cache_is_never_refused(tiny_models, pipeline):
    tiny = tiny_models["tiny_a"]
    prompts = [tiny.tokens(30, 70 + i) for i in range(3)]
    want = engine(tiny).generate(prompts, 30, stop_at_eos=False)
    eng = engine(tiny, num_blocks=6, prefix_cache=False, pipeline=pipeline)
    seqs = [eng.submit_nowait(Request(p, 30, stop_at_eos=False)) for p in prompts]
    while not eng.scheduler.stats.preemptions:
        eng.step()
    waits = max(len(s.ctx) for s in eng.scheduler.waiting)
    held = eng.runner.manager.pools[0].num_held()
    for size in range(1, 6):
        if size < max(held, -(-waits // 16)):
            with pytest.raises(OutOfPages):
                eng.resize_cache(size)
    eng.resize_cache(7)
    finish(eng)
    assert [s.output_ids for s in seqs] == want


def test_another_size_counts_every_group(putelix_cases):
    """Windows and companion rows beside full groups: every pool keeps what a queued prompt needs."""
    case = putelix_cases["case_a"]
    eng = LLMEngine(case.dir, EngineConfig(dtype="float32", num_blocks=40, max_batch=4, device="cpu",
                                           max_prefill_tokens=16, cuda_graphs=False), ops=PlainAnswerOps())
    seq = eng.submit_nowait(Request(case.tokens(50, 1), 2, stop_at_eos=False))
    with pytest.raises(OutOfPages):
        eng.resize_cache(3)
    eng.resize_cache(5)
    finish(eng)
    assert len(seq.output_ids) == 2


# -- grammars that fail -----------------------------------------------------------------------------------


class Failing:
    """Allows anything, and fails once ``n`` tokens have been generated."""

    def __init__(self, n, how):
        self.n, self.how = n, how

    def allowed(self, output):
        return self.how() if len(output) >= self.n else None


def _raise():
    raise KeyError("no such rule")


FAILURES = {"raises": _raise, "outside": lambda: [10 ** 7], "negative": lambda: [-1], "huge": lambda: [2 ** 70],
            "wide": lambda: np.ones(4000, dtype=bool), "short": lambda: np.zeros(1, dtype=np.int32),
            "number": lambda: 7, "text": lambda: "ab", "nothing in it": lambda: [None]}


@pytest.mark.parametrize("policy", ["prefill_first", "mixed"])
@pytest.mark.parametrize("pipeline", [False, True])
@pytest.mark.parametrize("how", FAILURES)
def test_a_grammar_that_fails_ends_its_own_request(tiny_models, how, pipeline, policy):
    tiny = tiny_models["tiny_b"]
    want = engine(tiny).generate([tiny.tokens(30, 2), tiny.tokens(9, 1)], 8, stop_at_eos=False)
    eng = engine(tiny, pipeline=pipeline, policy=policy)
    beside = eng.submit_nowait(Request(tiny.tokens(30, 2), 8, stop_at_eos=False))
    failing = [eng.submit_nowait(Request(tiny.tokens(9, 1), 8, grammar=Failing(n, FAILURES[how]), samples=1 + n,
                                         stop_at_eos=False)) for n in (0, 1, 3)]
    records = []
    for _ in range(200):
        if eng.has_work():
            records += eng.step()
            eng.runner.manager.check()
    assert not eng.has_work() and beside.output_ids == want[0]
    for n, seq in zip((0, 1, 3), failing):
        for s in (seq, *seq.siblings):
            assert s.finish_reason == "grammar_error" and s.output_ids == want[1][:n] and s.error
    if how == "raises":
        assert "no such rule" in failing[0].error
    by_name = {r.req_id: r for r in records}
    assert len(by_name) == 1 + 1 + 2 + 4
    record = by_name[failing[1].req_id]
    assert record.error == failing[1].error == record.as_dict()["error"]
    assert by_name[beside.req_id].error == "" and "error" not in by_name[beside.req_id].as_dict()
    assert eng.runner.manager.free_slots() == eng.config.live_requests


def test_answers_that_are_no_token_ids_are_refused():
    """A list or tensor of truth values is no list of the tokens 0 and 1, 1.5 is not token 1."""
    import torch
    flags = [t % 3 == 0 for t in range(40)]
    for bad in (flags, torch.tensor(flags), [1.5], [2.0], np.array([1.0, 3.0]), ["7"], [True], [np.True_]):
        with pytest.raises((TypeError, ValueError)):
            mask_words(bad, 40)
    want = mask_words([3, 39], 40)
    for good in ((3, 39), {3, 39}, range(3, 40, 36), iter([3, 39]), np.array([3, 39]), np.array([3, 39], np.uint8),
                 [np.int64(3), np.int32(39)], torch.tensor([3, 39]), {3: "a", 39: "b"}):
        assert np.array_equal(mask_words(good, 40), want)


@pytest.mark.parametrize("bad", [dict(logprobs=2.5), dict(logprobs=2.0), dict(logprobs="2"), dict(logprobs=True),
                                 dict(samples=2.5), dict(samples=2.0), dict(samples="2"), dict(samples=None)])
def test_numbers_of_answers_and_alternatives_are_whole(tiny_models, bad):
    """2.5 alternatives were taken, and the tokens of the step that brought them were lost."""
    sch, _fake, _mgr = make()
    with pytest.raises(RequestRefused):
        sch.add(Request(prompt(5), **bad))
    assert not sch.has_work()
    if "logprobs" in bad:
        eng = engine(tiny_models["tiny_a"])
        with pytest.raises(StepError):
            eng.runner.step([StepEntry("a", [1, 2], want=[1], **bad)], sample=True)
        with pytest.raises(ValueError):
            eng.score([1, 2, 3], alternatives=bad["logprobs"])
        assert eng.runner.manager.live() == []


def test_whole_numbers_of_any_kind_are_taken(tiny_models):
    tiny = tiny_models["tiny_a"]
    eng = engine(tiny)
    got = eng.submit_samples(Request(tiny.tokens(5, 1), 3, samples=np.int64(2), logprobs=np.int32(2), seed=np.int64(4)))
    assert [len(r.scores[0].top) for r in got] == [2, 2]
    assert len(eng.score([1, 2, 3], alternatives=np.int64(2))[0].top) == 2


# -- names ---------------------------------------------------------------------------------------------


def test_submitting_costs_the_same_however_many_wait():
    """Counted, not timed: nothing waiting is looked at when a request is added."""
    class Looked(deque):
        looks = 0

        def __iter__(self):
            Looked.looks += 1
            return super().__iter__()
    sch, _fake, _mgr = make()
    sch.waiting = Looked()
    for i in range(50):
        sch.add(Request(prompt(5), samples=1 + i % 3))
    assert len(sch.waiting) == 50 and Looked.looks == 0


def test_names_are_known_until_their_requests_end():
    sch, _fake, mgr = make(num_pages=8, page_size=4, prefix_cache=False)
    new = lambda name, **kw: Request(prompt(6), req_id=name, **{"max_new_tokens": 4, **kw})   # noqa: E731
    first = sch.add(new("r", samples=3))
    for name in ("r", "r#1"):
        with pytest.raises(RequestRefused, match="known"):
            sch.add(new(name, samples=2))
    assert sch.abort("r#2")
    other = sch.add(new("s"))
    with pytest.raises(RequestRefused):
        sch.add(new("s", samples=2))
    for _ in range(200):
        if sch.has_work():
            sch.step()
    assert first.finish_reason == other.finish_reason == first.siblings[0].finish_reason == "max_new_tokens"
    sch.add(new("r", samples=3)), sch.add(new("s", samples=2))
    sch.step()
    assert sch.abort("r") and sch.abort("s")
    for name in ("r#1", "r#2", "s#1"):
        sch.abort(name)
    assert not sch.has_work() and not sch._names
    # one that outgrows the pool (eight pages of four) ends, and its name with it
    grown = sch.add(new("g", max_new_tokens=100))
    for _ in range(200):
        if sch.has_work():
            sch.step()
    assert grown.finish_reason == "out_of_pages" and not sch._names


@pytest.mark.parametrize("policy", ["prefill_first", "mixed"])
@pytest.mark.parametrize("before", [True, False])
def test_a_name_that_an_answer_bears_waits_until_it_is_free(policy, before):
    """A plain request named as another's second answer, submitted before that is forked or after."""
    sch, _fake, mgr = make(budget=8, policy=policy)
    seq = sch.add(Request(prompt(20), max_new_tokens=6, seed=3, samples=3, req_id="r"))
    if not before:
        for _ in range(4):
            sch.step()
        assert "r#1" in mgr
    plain = sch.add(Request(prompt(7, 2), max_new_tokens=5, req_id="r#1"))
    last = sch.add(Request(prompt(9, 4), max_new_tokens=5))
    run(sch, mgr, limit=200)
    for i, s in enumerate([seq, *seq.siblings]):
        assert s.output_ids == expected_outputs(prompt(20), 6, seed=3 + i)
    assert plain.output_ids == expected_outputs(prompt(7, 2), 5)
    assert last.output_ids == expected_outputs(prompt(9, 4), 5)


def test_an_answer_waits_for_its_name():
    """The plain request runs when the prompt of the other is resident: the fork queues."""
    sch, _fake, mgr = make(budget=8)
    sch.add(Request(prompt(30), max_new_tokens=4, req_id="r", samples=3))
    plain = sch.add(Request(prompt(3), max_new_tokens=20, req_id="r#1"))
    sch.waiting.reverse()                                          # it is admitted first
    seq = sch.waiting[-1]
    run(sch, mgr, limit=200)
    assert plain.output_ids == expected_outputs(prompt(3), 20)
    for i, s in enumerate([seq, *seq.siblings]):
        assert s.output_ids == expected_outputs(prompt(30), 4, seed=i)


def test_two_plain_requests_of_one_name_run_in_turn():
    sch, _fake, mgr = make()
    both = [sch.add(Request(prompt(5 + i), max_new_tokens=4, req_id="same")) for i in range(2)]
    run(sch, mgr, limit=50)
    assert [s.output_ids for s in both] == [expected_outputs(prompt(5 + i), 4) for i in range(2)]


# -- copies that are refused ------------------------------------------------------------------------------


class RefusingOps(PlainAnswerOps):
    """Refuses the n-th page copy from now on, as the kernel refuses pages beyond its limits."""
    refuse = None

    def copy_pages(self, *args, **kw):
        if self.refuse is not None:
            self.refuse -= 1
            if self.refuse < 0:
                raise KernelError("copy_pages: unsupported")
        super().copy_pages(*args, **kw)


def refusing(case):
    eng = LLMEngine(case.dir, EngineConfig(dtype="float32", num_blocks=40, max_batch=4, device="cpu",
                                           max_prefill_tokens=64, cuda_graphs=False), ops=RefusingOps())
    vocab = eng.model.spec.vocab_size
    return eng, [(7 * i + 3) % vocab for i in range(37)]


@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_fork_whose_copies_are_refused_leaves_nothing_open(putelix_cases, at):
    """Several groups of pages and the tokens sampled last: copy 0, 1 or 2 of them is refused."""
    eng, p = refusing(putelix_cases["case_a"])
    rn = eng.runner
    rn.step([StepEntry("a", p, want=[36])], sample=True)
    free = [pool.num_free for pool in rn.manager.pools]
    rn.ops.refuse = at
    with pytest.raises(KernelError):
        rn.fork("a", "b")
    assert rn.manager.live() == ["a"] and [pool.num_free for pool in rn.manager.pools] == free
    rn.manager.check()
    rn.ops.refuse = None
    rn.fork("a", "b")
    res = rn.step([StepEntry(r, [5], want=[0]) for r in "ab"], sample=True)
    assert res.tokens_host()[0] == res.tokens_host()[1]


@pytest.mark.parametrize("at", [0, 1])
def test_a_resize_whose_copies_are_refused_changes_nothing(putelix_cases, at):
    case = putelix_cases["case_a"]
    eng, p = refusing(case)
    want = eng.generate([p], 12, stop_at_eos=False)[0]
    seq = eng.submit_nowait(Request(p, 12, stop_at_eos=False))
    for _ in range(3):
        eng.step()
    mgr = eng.runner.manager
    tables = [list(mgr.table(seq.req_id, gi)) for gi in range(len(mgr.groups))]
    sizes = [pool.num_pages for pool in mgr.pools]
    eng.runner.ops.refuse = at
    with pytest.raises(KernelError):
        eng.resize_cache(30)
    assert [pool.num_pages for pool in mgr.pools] == sizes == [t.shape[1] for t in eng.runner.storage.pools]
    assert [list(mgr.table(seq.req_id, gi)) for gi in range(len(mgr.groups))] == tables
    assert eng.config.num_blocks == 40
    mgr.check()
    eng.runner.ops.refuse = None
    eng.resize_cache(30)
    finish(eng)
    assert seq.output_ids == want


@pytest.mark.parametrize("pipeline", [False, True])
def test_refused_copies_of_a_fork_lose_no_token_and_no_answer(tiny_models, pipeline):
    """The second of three copies is refused, once, in a step that ends another request: that error
    comes up, and every answer and record comes all the same."""
    tiny = tiny_models["tiny_b"]
    p = tiny.tokens(37, 3)
    ask = lambda: Request(p, 6, 0.9, seed=5, samples=4, stop_at_eos=False, req_id="r")     # noqa: E731
    want = [r.output_ids for r in engine(tiny).submit_samples(ask())]
    eng = engine(tiny, pipeline=pipeline, policy="mixed", max_prefill_tokens=64)
    eng.runner.ops.__class__ = RefusingOps
    beside = eng.submit_nowait(Request(tiny.tokens(9, 4), 3, stop_at_eos=False, req_id="beside"))
    eng.step(), eng.step()
    seq = eng.submit_nowait(ask())
    eng.runner.ops.refuse = 3                                # (two copies a fork: the page and the token)
    records, errors = [], 0
    for _ in range(200):
        if eng.has_work():
            try:
                records += eng.step()
            except KernelError:
                errors += 1
                eng.runner.ops.refuse = None
            eng.runner.manager.check()
    assert errors == 1 and not eng.has_work()
    assert [s.output_ids for s in (seq, *seq.siblings)] == want and len(beside.output_ids) == 3
    assert sorted(r.req_id for r in records) == ["beside", "r", "r#1", "r#2", "r#3"]


def test_answers_are_forked_in_a_step_whose_reading_fails(tiny_models):
    """A kernel's report comes up in the step that makes a prompt resident: its answers run all the same."""
    tiny = tiny_models["tiny_b"]
    p = tiny.tokens(37, 3)
    ask = lambda: Request(p, 6, 0.9, seed=5, samples=3, stop_at_eos=False, req_id="r")     # noqa: E731
    want = [r.output_ids for r in engine(tiny).submit_samples(ask())]
    eng = engine(tiny, pipeline=True, policy="mixed", max_prefill_tokens=20)
    eng.submit_nowait(Request(tiny.tokens(9, 4), 50, stop_at_eos=False, req_id="beside"))
    eng.step(), eng.step()
    seq = eng.submit_nowait(ask())
    eng.runner.status |= 1
    eng.step()                                              # the first portion; the report rides along
    with pytest.raises(StepError):
        eng.step()                                          # the second; the report is read
    assert [s.state for s in seq.siblings] == ["running", "running"]
    eng.scheduler.abort("beside")
    with pytest.raises(StepError):
        eng.step()                                          # (it was in flight when the report was read)
    finish(eng)
    assert [s.output_ids for s in (seq, *seq.siblings)] == want
