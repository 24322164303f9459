"""Penalties, biases, grammars, several answers to one prompt, scores, and a cache of another size,
without a GPU: manager and scheduler alone, then the engine over the plain twins of the kernels,
against an oracle over the plain model's logits."""

import math
import random

import numpy as np
import pytest
import torch

import answers_cases as ac
from plain_answers import PlainAnswerOps
from test_scheduler import expected_outputs, make, prompt, run
from hetero_serve_b200 import EngineConfig, LLMEngine, LogitRules, OneOf, Request, StepEntry
from hetero_serve_b200.cache import CacheManager, GroupSpec, OutOfPages
from hetero_serve_b200.cache.manager import CacheError, PagePool
from hetero_serve_b200.engine.scheduler import RequestRefused
from hetero_serve_b200.engine.step import StepError
from hetero_serve_b200.sampling import mask_words

RULES = dict(repetition_penalty=1.4, presence_penalty=0.3, frequency_penalty=0.2,
             logit_bias={3: 0.4, 17: -math.inf, 40: -1.0})


# -- the manager --------------------------------------------------------------------------


def test_fork_shares_full_pages_and_copies_the_last():
    mgr = CacheManager([GroupSpec()], 8, 4, 4)
    mgr.open("a"); mgr.reserve("a", 13); mgr.commit("a", 10)
    copies = mgr.fork("a", "b")
    assert copies == [[(2, 4, 2)]]                       # two rows of the third page
    assert mgr.table("b") == [0, 1, 4] and mgr.table("a") == [0, 1, 2, 3]
    assert mgr.length("b") == 10 and mgr.slot("b") != mgr.slot("a")
    mgr.check()
    mgr.commit("a", 12)
    assert mgr.fork("a", "c") == [[]]                    # nothing is partly filled
    assert mgr.table("c") == [0, 1, 2]
    mgr.check()
    for r in "abc":
        mgr.close(r)
        mgr.check()
    assert mgr.pages_free() == 8 and mgr.free_slots() == 4


def test_fork_refuses_and_leaves_everything_as_it_was():
    mgr = CacheManager([GroupSpec(), GroupSpec(window=6)], 3, 4, 2)
    mgr.open("a"); mgr.reserve("a", 9); mgr.commit("a", 9)
    with pytest.raises(OutOfPages):
        mgr.fork("a", "b")
    with pytest.raises(CacheError):
        mgr.fork("nobody", "b")
    with pytest.raises(CacheError):
        mgr.fork("a", "a")
    assert mgr.live() == ["a"] and mgr.free_slots() == 1
    mgr.check()
    mgr.open("c")
    with pytest.raises(OutOfPages, match="slot"):
        mgr.fork("a", "d")
    mgr.check()


def test_fork_in_windowed_chunked_and_companion_groups():
    groups = [GroupSpec(), GroupSpec(window=6), GroupSpec(chunk=8), GroupSpec(stride=3),
              GroupSpec(window=6, keep_first=2)]
    for n in range(1, 40):
        mgr = CacheManager(groups, 24, 4, 3)
        mgr.open("a")
        for k in range(1, n + 1):
            mgr.reserve("a", k); mgr.commit("a", k)
        copies = mgr.fork("a", "b")
        mgr.check()
        for gi, g in enumerate(groups):
            rows = n // g.stride
            a, b = mgr.table("a", gi), mgr.table("b", gi)
            assert b[:rows // 4] == a[:rows // 4]
            for src, dst, filled in copies[gi]:
                assert (src, dst, filled) == (a[rows // 4], b[rows // 4], rows % 4)
            if g.window == 0 and g.chunk == 0:
                assert bool(copies[gi]) == bool(rows % 4)
        for k in range(n + 1, n + 12):                   # both go on alone
            for r in "ab":
                mgr.reserve(r, k); mgr.commit(r, k)
            mgr.check()
        mgr.close("a"); mgr.check()
        mgr.close("b"); mgr.check()
        assert all(p.num_free == 24 for p in mgr.pools)


def test_resize_moves_live_and_published_pages():
    mgr = CacheManager([GroupSpec()], 12, 4, 4)
    for r, n in (("a", 9), ("b", 8), ("c", 5)):
        mgr.open(r); mgr.reserve(r, n); mgr.commit(r, n)
        mgr.publish(r, [ord(r)] * n)
    before = {r: list(mgr.table(r)) for r in "abc"}
    mgr.close("b")                                       # two published pages nobody holds
    with pytest.raises(OutOfPages):
        mgr.resize([4])
    with pytest.raises(ValueError):
        mgr.resize([4, 4])
    mgr.check()
    [moved] = mgr.resize([6])                            # one of them has to go: the older
    mgr.check()
    assert [moved[p] for p in before["a"]] == mgr.table("a")
    assert [moved[p] for p in before["c"]] == mgr.table("c")
    assert sorted(moved.values()) == list(range(6)) and mgr.pools[0].evictions == 1
    [again] = mgr.resize([40])
    assert again == {p: p for p in range(6)} and mgr.pages_free() == 35
    mgr.open("d", [ord("a")] * 9)
    assert mgr.table("d") == mgr.table("a")[:2]          # a's prefix is still found
    mgr.check()
    for r in "acd":
        mgr.close(r)
    mgr.check()
    assert PagePool(4, True).resize(2) == {}


# -- the scheduler over a fake step ------------------------------------------------------------


@pytest.mark.parametrize("policy", ["prefill_first", "mixed"])
@pytest.mark.parametrize("n_prompt", [1, 2, 4, 5, 41])
@pytest.mark.parametrize("prefix_cache", [True, False])
def test_samples_are_what_single_requests_would_give(policy, n_prompt, prefix_cache):
    sch, fake, mgr = make(policy=policy, prefix_cache=prefix_cache)
    seq = sch.add(Request(prompt(n_prompt), max_new_tokens=6, seed=5, samples=4))
    other = sch.add(Request(prompt(9, 2), max_new_tokens=3))
    run(sch, mgr)
    for i, s in enumerate([seq, *seq.siblings]):
        assert s.output_ids == expected_outputs(prompt(n_prompt), 6, seed=5 + i), i
        assert s.finish_reason == "max_new_tokens"
    assert other.output_ids == expected_outputs(prompt(9, 2), 3)
    assert mgr.pages_free() == 64 and mgr.free_slots() == 8
    fed = sum(n for step in fake.log for r, _s, n, _w in step if r == seq.req_id)
    assert fed == n_prompt + 5                            # the prompt ran once
    for s in seq.siblings:
        assert sum(n for step in fake.log for r, _s, n, _w in step if r == s.req_id) == 6


@pytest.mark.parametrize("slots,pages", [(2, 64), (8, 13), (1, 64)])
def test_samples_without_a_slot_or_a_page_wait_their_turn(slots, pages):
    sch, fake, mgr = make(max_requests=slots, num_pages=pages)
    seq = sch.add(Request(prompt(42), max_new_tokens=5, seed=1, samples=5))
    later = sch.add(Request(prompt(3), max_new_tokens=2))
    run(sch, mgr)
    for i, s in enumerate([seq, *seq.siblings]):
        assert s.output_ids == expected_outputs(prompt(42), 5, seed=1 + i), i
    assert later.output_ids == expected_outputs(prompt(3), 2)
    assert mgr.pages_free() == pages


def test_samples_survive_preemption():
    sch, fake, mgr = make(num_pages=16, page_size=4, prefix_cache=False)
    seq = sch.add(Request(prompt(9), max_new_tokens=24, seed=2, samples=4))
    run(sch, mgr)
    assert sch.stats.preemptions > 0
    for i, s in enumerate([seq, *seq.siblings]):
        assert s.output_ids == expected_outputs(prompt(9), 24, seed=2 + i), i


def test_abort_takes_the_waiting_answers_along():
    sch, fake, mgr = make(budget=8)
    seq = sch.add(Request(prompt(30), max_new_tokens=5, samples=3))
    sch.step()
    assert sch.abort(seq.siblings[0].req_id) and seq.siblings[0].finish_reason == "aborted"
    assert sch.abort(seq.req_id)
    assert [s.finish_reason for s in seq.siblings] == ["aborted", "aborted"]
    assert not sch.has_work() and mgr.pages_free() == 64
    mgr.check()
    again = sch.add(Request(prompt(5), max_new_tokens=4, samples=3))
    for _ in range(2):
        sch.step()
    assert sch.abort(again.siblings[1].req_id)            # it decodes by now
    run(sch, mgr)
    assert [s.finish_reason for s in again.siblings] == ["max_new_tokens", "aborted"]


@pytest.mark.parametrize("bad", [
    dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.nan),
    dict(repetition_penalty=math.inf), dict(presence_penalty=math.inf),
    dict(frequency_penalty=math.nan), dict(logit_bias={97: 1.0}), dict(logit_bias={-1: 1.0}),
    dict(logit_bias={3: math.nan}), dict(logit_bias={3: math.inf}), dict(logit_bias={"3": 1.0}),
    dict(logit_bias={3: "x"}), dict(presence_penalty=None), dict(logprobs=-1), dict(logprobs=33),
    dict(samples=0), dict(grammar=object())])
def test_requests_that_are_refused(bad):
    sch, _fake, _mgr = make()
    with pytest.raises(RequestRefused):
        sch.add(Request(prompt(5), **bad))
    assert not sch.has_work()


def test_masks_of_every_form():
    assert mask_words(None, 40) is None
    ids = [0, 31, 32, 39]
    flags = np.zeros(40, dtype=bool)
    flags[ids] = True
    want = np.array([-2 ** 31 + 1, 129], dtype=np.int32)
    for form in (ids, set(ids), flags, want, want.astype(np.uint32) if False else want.view(np.uint32)):
        assert np.array_equal(mask_words(form, 40), want)
    assert np.array_equal(mask_words(np.array([-1, -1], dtype=np.int32), 40), [-1, 255])
    assert not mask_words([], 40).any()
    for bad in ([40], [-1], np.ones(39, bool), np.zeros(3, np.int32)):
        with pytest.raises(ValueError):
            mask_words(bad, 40)
    choice = OneOf([[5, 6], [5, 7, 8], [9]], end=2)
    assert sorted(choice.allowed(())) == [5, 9] and choice.allowed((5, 7)) == [8]
    assert choice.allowed((9,)) == [2] and choice.allowed((9, 2)) == []
    for bad in ([], [[1], []]):
        with pytest.raises(ValueError):
            OneOf(bad)


# -- the engine over the plain twins -------------------------------------------------------------


def engine(tiny, **kw):
    opts = dict(dtype="float32", num_blocks=24, max_batch=8, max_prefill_tokens=24, device="cpu",
                cuda_graphs=False)
    return LLMEngine(tiny.dir, EngineConfig(**{**opts, **kw}), ops=PlainAnswerOps())


@pytest.mark.parametrize("pipeline", [False, True])
def test_answers_follow_the_rules(tiny_models, pipeline):
    tiny = tiny_models["tiny_a"]
    vocab = tiny.config["vocab_size"]
    grammar = ac.Alternating(vocab)
    asked = [({}, 21), (RULES, 22), (dict(RULES, grammar=grammar), 5), (dict(grammar=grammar), 9),
             (dict(logit_bias={7: 3.0}), 13)]
    eng = engine(tiny, pipeline=pipeline, policy="mixed")
    seqs = [eng.submit_nowait(Request(tiny.tokens(n, 50 + n), 8, stop_at_eos=False, logprobs=3, **kw))
            for kw, n in asked]
    eng.run_until_done()
    for s, (kw, n) in zip(seqs, asked):
        plain = dict(kw, grammar=ac.Plain(kw["grammar"])) if "grammar" in kw else kw
        p = tiny.tokens(n, 50 + n)
        want, gaps = ac.greedy(tiny.logits, p, 8, **plain)
        assert min(gaps) > 1e-4                               # none is a close call
        assert s.output_ids == want, kw
        rows = tiny.logits(p + want)[n - 1:-1]
        lps = torch.log_softmax(rows, 1)
        for i, score in enumerate(s.scores):
            assert abs(score.logprob - float(lps[i, want[i]])) < 1e-4
            assert score.rank == int((rows[i] > rows[i, want[i]]).sum())
            best = torch.topk(lps[i], 3)
            assert [t for t, _ in score.top] == best.indices.tolist()
    assert {s.finish_reason for s in seqs} == {"max_new_tokens"}
    eng.runner.manager.check()


def test_the_rules_outlive_preemption(tiny_models):
    """Few pages: requests are preempted and come back into other slots; their records are made
    anew from prompt and answer."""
    tiny = tiny_models["tiny_a"]
    eng = engine(tiny, num_blocks=6, prefix_cache=False, max_batch=3)
    seqs = [eng.submit_nowait(Request(tiny.tokens(20, 70 + i), 24, stop_at_eos=False, **RULES))
            for i in range(3)]
    eng.run_until_done()
    assert eng.scheduler.stats.preemptions > 0
    for i, s in enumerate(seqs):
        want, gaps = ac.greedy(tiny.logits, tiny.tokens(20, 70 + i), 24, **RULES)
        assert min(gaps) > 1e-4 and s.output_ids == want


def test_grammars_decode_in_the_same_steps(tiny_models):
    """Pipelined, requests with grammars whose prompts ended in different steps share their steps
    all the same, and a plain request decodes in every one."""
    tiny = tiny_models["tiny_b"]
    eng = engine(tiny, pipeline=True, policy="mixed")
    sizes = []
    inner = eng.scheduler.step_fn

    def counted(entries):
        sizes.append([e.req_id for e in entries if e.want])
        return inner(entries)
    eng.scheduler.step_fn = counted
    grammar = ac.Alternating(tiny.config["vocab_size"])
    ruled = [eng.submit_nowait(Request(tiny.tokens(20, i), 12, stop_at_eos=False, grammar=grammar))
             for i in range(4)]
    plain = eng.submit_nowait(Request(tiny.tokens(5, 9), 40, stop_at_eos=False))
    eng.run_until_done()
    assert [len(s.output_ids) for s in ruled] == [12] * 4 and len(plain.output_ids) == 40
    names = {s.req_id for s in ruled}
    together = [len(names & set(step)) for step in sizes if len(step) > 0]
    later = together[12:24]                       # (prompts end in the first few steps)
    assert sorted(set(later)) == [0, 4], together
    at = [i for i, step in enumerate(sizes) if plain.req_id in step]
    assert at == list(range(at[0], at[0] + 40))


def test_a_grammar_that_ends_the_answer(tiny_models):
    tiny = tiny_models["tiny_b"]
    eng = engine(tiny)
    choices = [[4, 5, 6], [4, 9], [7]]
    open_end = eng.submit(Request(tiny.tokens(9, 1), 10, grammar=OneOf(choices)))
    assert open_end.output_ids in choices and open_end.finish_reason == "grammar"
    closed = eng.submit(Request(tiny.tokens(9, 1), 10, grammar=OneOf(choices, end=999)))
    assert closed.output_ids == [*open_end.output_ids, 999] and closed.finish_reason == "eos"

    banned = eng.submit(Request(tiny.tokens(9, 1), 10, grammar=OneOf([[4, 5], [6]]),
                                logit_bias={5: -math.inf, 6: -math.inf}))
    assert banned.output_ids == [4] and banned.finish_reason == "grammar"

    class Nothing:
        def allowed(self, output):
            return []
    beside = eng.submit_nowait(Request(tiny.tokens(30, 2), 4, stop_at_eos=False))
    none = eng.submit(Request(tiny.tokens(9, 1), 10, grammar=Nothing()))
    assert none.output_ids == [] and none.finish_reason == "grammar"
    eng.run_until_done()
    assert len(beside.output_ids) == 4
    eng.runner.manager.check()
    assert eng.runner.manager.free_slots() == eng.config.live_requests


@pytest.mark.parametrize("pipeline", [False, True])
def test_samples_equal_requests_of_their_own(tiny_models, pipeline):
    tiny = tiny_models["tiny_b"]
    for n in (1, 16, 17, 40):
        p = tiny.tokens(n, n)
        eng = engine(tiny, pipeline=pipeline)
        got = eng.submit_samples(Request(p, 7, 0.9, 0, 31, False, samples=4, logprobs=0, **RULES))
        single = engine(tiny, pipeline=pipeline)
        for i, record in enumerate(got):
            want = single.submit(Request(p, 7, 0.9, 0, 31 + i, False, logprobs=0, **RULES))
            assert record.output_ids == want.output_ids
            assert abs(record.cumulative_logprob - want.cumulative_logprob) < 1e-4
        assert len({tuple(r.output_ids) for r in got}) > 1
        eng.runner.manager.check()
    out = got[0].as_dict()
    assert len(out["logprobs"]) == 7 and out["top_logprobs"] == [[]] * 7


def test_given_text_is_scored(tiny_models):
    tiny = tiny_models["tiny_a"]
    eng = engine(tiny)
    text = tiny.tokens(60, 3)
    lps = torch.log_softmax(tiny.logits(text), 1)
    scores = eng.score(text, alternatives=2)
    assert len(scores) == 59
    for i, s in enumerate(scores):
        assert abs(s.logprob - float(lps[i, text[i + 1]])) < 1e-4
        assert s.rank == int((lps[i] > lps[i, text[i + 1]]).sum())
        assert [t for t, _ in s.top] == torch.topk(lps[i], 2).indices.tolist()
    assert eng.score(text[:1]) == [] and eng.score([]) == []
    with pytest.raises(StepError):
        eng.score([1, 512, 3])
    eng.runner.manager.check()
    assert eng.runner.manager.live() == []


def test_a_cache_of_another_size_keeps_its_requests(tiny_models):
    tiny = tiny_models["tiny_b"]
    prompts = [tiny.tokens(n, 90 + n) for n in (33, 20, 47)]
    want = engine(tiny).generate(prompts, 12, stop_at_eos=False)
    eng = engine(tiny)
    seqs = [eng.submit_nowait(Request(p, 12, stop_at_eos=False)) for p in prompts]
    sizes = iter((12, 40, 11, 24))
    while eng.has_work():
        if eng.scheduler.stats.steps % 4 == 3:
            size = next(sizes, 24)
            eng.resize_cache(size)
            assert eng.runner.storage.pools[0].shape[1] == eng.config.num_blocks == size
            eng.runner.manager.check()
        eng.step()
    assert [s.output_ids for s in seqs] == want
    live = eng.submit_nowait(Request(prompts[2], 12, stop_at_eos=False))
    eng.step(), eng.step()
    with pytest.raises(OutOfPages):
        eng.resize_cache(2)
    eng.run_until_done()
    assert live.output_ids == want[2]
    eng.resize_cache(3)                                       # published prefixes go, oldest first
    again = eng.submit(Request(prompts[1], 12, stop_at_eos=False))
    assert again.output_ids == want[1]


def test_steps_refuse_rules_they_cannot_follow(tiny_models):
    tiny = tiny_models["tiny_a"]
    rn = engine(tiny).runner
    rules = LogitRules(repetition=1.2)
    words = np.full(16, -1, dtype=np.int32)
    for entry in (StepEntry("a", [1, 2], want=[1], rules=rules),                      # no history
                  StepEntry("a", [1, 2], want=[0], rules=rules, history=([1], [])),
                  StepEntry("a", [1, 2], want=[0, 1], allowed=words),
                  StepEntry("a", [1, 2], want=[1], rules=LogitRules(bias={512: 1.0})),
                  StepEntry("a", [1, 2], want=[1], rules=rules, history=([512], [])),
                  StepEntry("a", [1, 2], want=[1], rules=rules, history=([1], [-1])),
                  StepEntry("a", [1, 2], want=[1], allowed=words[:15]),
                  StepEntry("a", [1, 2], want=[1], allowed=words.astype(np.int64)),
                  StepEntry("a", [1, 2], want=[1], allowed=[1, 2]),
                  StepEntry("a", [1, 2], want=[1], allowed=words * 0),
                  StepEntry("a", [1, 2], want=[1], logprobs=33),
                  StepEntry("a", [1, 2], want=[1], logprobs=-1)):
        with pytest.raises(StepError):
            rn.step([entry], sample=True)
    assert rn.manager.live() == []
    rn.step([StepEntry("a", [1, 2], want=[1], rules=rules, history=([1, 2], []))], sample=True)
    rn.step([StepEntry("a", [3], want=[0], rules=rules)], sample=True)      # the record goes on
    rn.close("a")
    with pytest.raises(StepError, match="history"):                          # another request
        rn.step([StepEntry("b", [1], want=[0], rules=rules)], sample=True)
    for bad in (dict(repetition=0.0), dict(bias={-1: 1.0}), dict(bias={2 ** 31: 1.0})):
        with pytest.raises(ValueError):
            LogitRules(**bad)
    with pytest.raises(ValueError, match="alternatives"):
        engine(tiny).score([1, 2], alternatives=33)
    with pytest.raises(ValueError, match="one answer"):
        engine(tiny).generate([[1, 2]], samples=2)


@pytest.mark.parametrize("family", ["pedorax", "putelix", "roritar", "mafuzen", "pivinex", "nukodra"])
@pytest.mark.parametrize("name", ["case_a", "case_b"])
def test_forks_in_every_architecture(request, family, name):
    """Windows, chunks, companion rows, shared latents, states, empty ones among them: a fork goes on
    as a request of its own that was fed the same tokens, bit for bit."""
    from hetero_serve_b200.engine import Runner
    from hetero_serve_b200.engine.loading import load_model
    case = request.getfixturevalue(f"{family}_cases")[name]
    vocab, n = case.config["vocab"], 23
    t = case.tokens(n + 2, 5)
    model, _ = load_model(case.dir, "float32", "cpu")
    rn = Runner(model, num_pages=48, page_size=16, max_requests=4, dtype=torch.float32, device="cpu",
                ops=PlainAnswerOps())
    rn.step([StepEntry("a", t[:n])])
    rn.fork("a", "b")
    rn.step([StepEntry("alone", t[:n])])
    for i in range(n, n + 2):
        other = [(t[i] + 1) % vocab]
        res = rn.step([StepEntry("a", [t[i]], want=[0]), StepEntry("b", other, want=[0]),
                       StepEntry("alone", other, want=[0])])
        assert torch.equal(res.logits[1], res.logits[2]) and not torch.equal(res.logits[0], res.logits[1])
    rn.manager.check()


def test_a_fork_goes_on_where_its_parent_stood(tiny_models):
    """Pages, the token on the device and the record: the child's next steps are the parent's."""
    from hetero_serve_b200.engine import FROM_DEVICE
    tiny = tiny_models["tiny_b"]
    rn = engine(tiny).runner
    rules = LogitRules(repetition=1.5, frequency=0.5)
    p = tiny.tokens(21, 4)
    rn.step([StepEntry("a", p, want=[20], rules=rules, history=(p, []))], sample=True)
    rn.fork("a", "b")
    for _ in range(4):
        res = rn.step([StepEntry(r, [FROM_DEVICE], want=[0], rules=rules) for r in "ab"], sample=True)
        a, b = res.tokens_host()
        assert a == b and torch.equal(res.logits[0], res.logits[1])
    rn.manager.check()


@pytest.mark.parametrize("seed", (0, 3, 4, 11))
def test_everything_at_once_depends_on_no_engine_setting(tiny_models, seed):
    """Penalties, biases, grammars, samples and scores of requests that come and go: batches, budgets,
    pipelining, prefix reuse, preemption and the cache's size change no answer."""
    tiny = tiny_models["tiny_a"]
    requests = ac.any_requests(random.Random(seed), tiny.config["vocab_size"])
    answers = [ac.run_through(engine(tiny, **options), requests, random.Random(seed + 100))
               for options in ac.ENGINES]
    first, scores = answers[0]
    for other, others in answers[1:]:
        # (a row's sum is taken in another order where it lies on other 16-byte borders)
        assert other == first and torch.allclose(others, scores, rtol=0, atol=1e-5)
