"""What may not disturb other requests, on the GPU: bad text to score beside live requests."""

import pytest

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
