"""Penalties, biases, grammars, several answers to one prompt, scores and a cache of another size
through the engine on the GPU: captured and launched one by one, pipelined or not, in every
architecture's cache and state."""

import math
import random

import pytest
import torch

import answers_cases as ac
from hetero_serve_b200 import EngineConfig, LLMEngine, LogitRules, OneOf, Request, StepEntry
from hetero_serve_b200.cache import OutOfPages
from hetero_serve_b200.engine import FROM_DEVICE, Runner
from hetero_serve_b200.engine.loading import load_model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RULES = dict(repetition_penalty=1.4, presence_penalty=0.3, frequency_penalty=0.2,
             logit_bias={3: 0.4, 17: -math.inf, 40: -1.0})


def engine(folder, **kw):
    opts = dict(dtype="float32", num_blocks=32, max_batch=8, max_prefill_tokens=24, device=DEV)
    return LLMEngine(folder, EngineConfig(**{**opts, **kw}))


@pytest.mark.parametrize("graphs,pipeline", [(False, False), (True, False), (True, True)])
def test_answers_follow_the_rules(tiny_models, graphs, pipeline):
    tiny = tiny_models["tiny_a"]
    grammar = ac.Alternating(tiny.config["vocab_size"])
    asked = [({}, 21), (RULES, 22), (dict(RULES, grammar=grammar), 5), (dict(grammar=grammar), 9),
             (dict(logit_bias={7: 3.0}), 13)]
    eng = engine(tiny.dir, cuda_graphs=graphs, pipeline=pipeline, policy="mixed")
    for again in range(2):                        # the second time through captured steps
        seqs = [eng.submit_nowait(Request(tiny.tokens(n, 50 + n), 10, stop_at_eos=False,
                                          logprobs=3, **kw)) for kw, n in asked]
        eng.run_until_done()
        for s, (kw, n) in zip(seqs, asked):
            plain = dict(kw, grammar=ac.Plain(kw["grammar"])) if "grammar" in kw else kw
            p = tiny.tokens(n, 50 + n)
            want, gaps = ac.greedy(tiny.logits, p, 10, **plain)
            assert min(gaps) > 1e-4
            assert s.output_ids == want, kw
            rows = tiny.logits(p + want)[n - 1:-1]
            lps = torch.log_softmax(rows, 1)
            for i, score in enumerate(s.scores):
                assert abs(score.logprob - float(lps[i, want[i]])) < 1e-4
                assert [t for t, _ in score.top] == torch.topk(lps[i], 3).indices.tolist()
    eng.runner.check_status()
    eng.runner.manager.check()


def test_long_answers_with_penalties_over_hot_shapes(tiny_models):
    """Enough steps of one shape that its second metadata block and graph are used."""
    tiny = tiny_models["tiny_b"]
    eng = engine(tiny.dir, num_blocks=64)
    seqs = [eng.submit_nowait(Request(tiny.tokens(9, i), 120, stop_at_eos=False, **RULES))
            for i in range(2)]
    eng.run_until_done()
    for i, s in enumerate(seqs):
        p, out = tiny.tokens(9, i), s.output_ids
        rows = tiny.logits(p + out)
        assert len(out) == 120
        for k, t in enumerate(out):
            # each logit is within 2e-5 of the plain one (the tolerance of these models), which a
            # penalty multiplies by up to 1.4, and two of them are compared
            row = ac.ruled(rows[len(p) - 1 + k], p, out[:k], **RULES)
            assert float(row.max() - row[t]) <= 2 * 1.4 * 2e-5, k
    assert any(k[-1] == 1 and k[4].history for k in eng.runner._graphs)


@pytest.mark.parametrize("graphs", [False, True])
def test_rules_outlive_preemption_and_other_slots(tiny_models, graphs):
    tiny = tiny_models["tiny_a"]
    eng = engine(tiny.dir, num_blocks=6, prefix_cache=False, max_batch=3, cuda_graphs=graphs)
    seqs = [eng.submit_nowait(Request(tiny.tokens(20, 70 + i), 24, stop_at_eos=False, **RULES))
            for i in range(3)]
    eng.run_until_done()
    assert eng.scheduler.stats.preemptions > 0
    for i, s in enumerate(seqs):
        want, gaps = ac.greedy(tiny.logits, tiny.tokens(20, 70 + i), 24, **RULES)
        assert min(gaps) > 1e-4 and s.output_ids == want


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [False, True])
def test_samples_equal_requests_of_their_own(tiny_models, dtype, graphs):
    """In float32 token by token.  In bfloat16 other batches round otherwise, so only that every
    answer is complete and scored."""
    tiny = tiny_models["tiny_b"]
    for n in (1, 17, 64, 70):
        p = tiny.tokens(n, n)
        eng = engine(tiny.dir, dtype=dtype, cuda_graphs=graphs)
        got = eng.submit_samples(Request(p, 9, 0.9, 0, 31, False, samples=4, logprobs=0, **RULES))
        assert [len(r.output_ids) for r in got] == [9] * 4 == [len(r.scores) for r in got]
        eng.runner.manager.check()
        if dtype == "float32":
            single = engine(tiny.dir, dtype=dtype, cuda_graphs=graphs)
            for i, record in enumerate(got):
                want = single.submit(Request(p, 9, 0.9, 0, 31 + i, False, logprobs=0, **RULES))
                assert record.output_ids == want.output_ids
                assert abs(record.cumulative_logprob - want.cumulative_logprob) < 1e-3


@pytest.mark.parametrize("top_k", [0, 2, 40])
def test_a_choice_and_plain_requests_side_by_side(tiny_models, top_k):
    tiny = tiny_models["tiny_b"]
    eng = engine(tiny.dir, policy="mixed")
    choices = [[4, 5, 6], [4, 9], [7, 8, 9, 10]]
    beside = [eng.submit_nowait(Request(tiny.tokens(20 + i, i), 12, stop_at_eos=False))
              for i in range(3)]
    chosen = [eng.submit_nowait(Request(tiny.tokens(9 + i, 5 + i), 10, 0.8, top_k, seed=i,
                                        grammar=OneOf(choices, end=999))) for i in range(3)]
    eng.run_until_done()
    for s in chosen:
        assert s.finish_reason == "eos" and s.output_ids[:-1] in choices
    want = engine(tiny.dir).generate([tiny.tokens(20 + i, i) for i in range(3)], 12, stop_at_eos=False)
    assert [s.output_ids for s in beside] == want


@pytest.mark.parametrize("dtype,tol", [("float32", 1e-4), ("bfloat16", 0.2)])
def test_given_text_is_scored(tiny_models, dtype, tol):
    tiny = tiny_models["tiny_a"]
    eng = engine(tiny.dir, dtype=dtype)
    live = eng.submit_nowait(Request(tiny.tokens(11, 8), 8, stop_at_eos=False))
    eng.step(), eng.step()
    text = tiny.tokens(100, 3)
    lps = torch.log_softmax(tiny.logits(text, dtype), 1)
    scores = eng.score(text, alternatives=2)
    assert len(scores) == 99
    for i, s in enumerate(scores):
        assert abs(s.logprob - float(lps[i, text[i + 1]])) < tol
        assert s.top[0][1] >= s.top[1][1] and abs(s.top[0][1] - float(lps[i].max())) < tol
    eng.run_until_done()
    assert len(live.output_ids) == 8
    if dtype == "float32":
        assert live.output_ids == ac.greedy(tiny.logits, tiny.tokens(11, 8), 8)[0]


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_cache_of_another_size_keeps_its_requests(tiny_models, dtype, fused):
    tiny = tiny_models["tiny_b"]
    prompts = [tiny.tokens(n, 90 + n) for n in (33, 20, 47)]
    want = engine(tiny.dir, dtype=dtype, fused_decode=fused).generate(prompts, 16, stop_at_eos=False)
    eng = engine(tiny.dir, dtype=dtype, fused_decode=fused)
    seqs = [eng.submit_nowait(Request(p, 16, stop_at_eos=False)) for p in prompts]
    sizes = iter((15, 60, 14, 32))
    while eng.has_work():
        if eng.scheduler.stats.steps % 5 == 4:
            eng.resize_cache(next(sizes, 32))
            eng.runner.manager.check()
        eng.step()
    assert [s.output_ids for s in seqs] == want
    with pytest.raises(OutOfPages):
        eng.resize_cache(0)


def _models(request):
    for family in ("pedorax", "putelix", "roritar", "mafuzen", "pivinex", "nukodra"):
        cases = request.getfixturevalue(f"{family}_cases")
        yield family, cases["case_a"]
        yield family, cases["case_b"]
        if family in ("putelix", "nukodra"):
            yield family, cases["case_d"]


@pytest.mark.parametrize("graphs", [False, True])
def test_forks_in_every_architecture(request, graphs):
    """A fork behind n tokens goes on as a request of its own that was fed the same tokens, and its
    parent is not disturbed by it: windows, chunks, companion rows, shared latents and states."""
    for family, case in _models(request):
        vocab = case.config["vocab"]
        for n in (1, 16, 23, 61):
            t = case.tokens(n + 12, 7 * n)
            other = [(x + 1) % vocab for x in t]
            model, _ = load_model(case.dir, "float32", DEV)
            rn = Runner(model, num_pages=48, page_size=16, max_requests=4, dtype=torch.float32,
                        device=DEV, cuda_graphs=graphs)
            rn.step([StepEntry("a", t[:n])])
            rn.fork("a", "b")
            rn.manager.check()
            rn.step([StepEntry("alone_a", t[:n]), StepEntry("alone_b", t[:n])])
            for i in range(n, n + 12):
                res = rn.step([StepEntry("a", [t[i]], want=[0]), StepEntry("b", [other[i]], want=[0]),
                               StepEntry("alone_a", [t[i]], want=[0]),
                               StepEntry("alone_b", [other[i]], want=[0])])
                got, want = res.logits[:2].clone(), res.logits[2:]
                # (the same kernels over the same numbers in other pages and slots; prompts were
                # fed in batches of other sizes)
                assert float((got - want).abs().max()) <= 2e-4 * max(1.0, float(want.abs().max())), \
                    (family, n, i)
            rn.check_status()
            rn.manager.check()


def test_a_fork_takes_the_token_and_the_record_along(tiny_models):
    tiny = tiny_models["tiny_b"]
    model, _ = load_model(tiny.dir, "float32", DEV)
    rn = Runner(model, num_pages=32, page_size=16, max_requests=4, dtype=torch.float32, device=DEV,
                cuda_graphs=True)
    rules = LogitRules(repetition=1.5, frequency=0.5)
    p = tiny.tokens(21, 4)
    rn.step([StepEntry("a", p, want=[20], rules=rules, history=(p, []))], sample=True)
    rn.fork("a", "b")
    for _ in range(5):
        res = rn.step([StepEntry(r, [FROM_DEVICE], want=[0], rules=rules) for r in "ab"], sample=True)
        a, b = res.tokens_host()
        assert a == b and torch.equal(res.logits[0], res.logits[1])
    rn.manager.check()


def test_command_line_gives_scored_samples():
    import json
    import subprocess
    import sys
    out = subprocess.run([sys.executable, "-m", "hetero_serve_b200", "--model", "tiny",
                          "--random-prompts", "2:12", "--max-new-tokens", "4", "--samples", "3",
                          "--temperature", "0.8", "--repetition-penalty", "1.2", "--logit-bias",
                          "5:-inf", "--logprobs", "2", "--json", "--no-eos-stop"],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    lines = [json.loads(x) for x in out.stdout.splitlines()]
    assert len(lines) == 7
    for rec in lines[:6]:
        assert len(rec["output_ids"]) == 4 == len(rec["logprobs"]) and 5 not in rec["output_ids"]
        assert all(len(t) == 2 for t in rec["top_logprobs"])


@pytest.mark.parametrize("seed", range(24))
def test_everything_at_once_depends_on_no_engine_setting(tiny_models, seed):
    """Penalties, biases, grammars, samples and scores of requests that come and go: batches, budgets,
    pipelining, prefix reuse, preemption and the cache's size change no answer."""
    tiny = tiny_models["tiny_a"]
    requests = ac.any_requests(random.Random(seed), tiny.config["vocab_size"])
    answers = [ac.run_through(engine(tiny.dir, **options), requests, random.Random(seed + 100))
               for options in ac.ENGINES]
    first, scores = answers[0]
    for other, others in answers[1:]:
        # (a row's sum is taken in another order where it lies on other 16-byte borders)
        assert other == first and torch.allclose(others, scores, rtol=0, atol=1e-5)
