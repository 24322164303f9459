"""What may not disturb other requests, without a GPU: bad text to score, numbers out of range, grammars
that fail, queues, names, refused copies.  The engine over the plain twins of the kernels."""

import pytest

from plain_answers import PlainAnswerOps
from test_answers_cpu import engine
from hetero_serve_b200 import Request
from hetero_serve_b200.engine.step import StepError


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
