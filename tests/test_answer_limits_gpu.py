"""What may not disturb other requests, on the GPU: bad text to score beside live requests."""

import pytest
import torch

from test_answers_gpu import engine
from hetero_serve_b200 import Request
from hetero_serve_b200.engine.step import StepError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pipeline", [False, True])
def test_a_bad_text_to_score_is_refused_beside_a_live_request(tiny_models, pipeline):
    tiny = tiny_models["tiny_a"]
    want = engine(tiny.dir).generate([tiny.tokens(9, 4)], 14, stop_at_eos=False)[0]
    eng = engine(tiny.dir, pipeline=pipeline)
    live = eng.submit_nowait(Request(tiny.tokens(9, 4), 14, stop_at_eos=False))
    eng.step(), eng.step()
    text = tiny.tokens(60, 3)
    for at in (0, 24, 48, 30, 59):
        for bad in (-1, -2, 512, 99999):
            with pytest.raises(StepError):
                eng.score(text[:at] + [bad] + text[at + 1:], alternatives=2)
        assert len(eng.score(text)) == 59
        eng.step()
    eng.run_until_done()
    assert live.output_ids == want
    eng.runner.check_status()
    eng.runner.manager.check()


@pytest.mark.parametrize("temperature", [0.0, 0.5, 1.0])
def test_finite_biases_as_low_as_they_go_leave_the_rest(tiny_models, temperature):
    """Two tokens that a grammar allows, both biased to the type's lowest value: one of them is drawn."""
    tiny = tiny_models["tiny_b"]
    lowest = torch.finfo(torch.float32).min

    class Two:
        def allowed(self, output):
            return [4, 9]
    seq = engine(tiny.dir).submit(Request(tiny.tokens(9, 1), 12, temperature, grammar=Two(),
                                          logit_bias={4: lowest, 9: lowest}))
    assert len(seq.output_ids) == 12 and set(seq.output_ids) <= {4, 9}
