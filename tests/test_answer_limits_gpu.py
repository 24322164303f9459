"""What may not disturb other requests, on the GPU: bad text to score beside live requests."""

import pytest
import torch

from test_answers_gpu import engine
from hetero_serve_b200 import Request
from hetero_serve_b200.engine.step import StepError
from hetero_serve_b200.kernels import CudaOps, TokenHistory

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


def test_a_prompt_said_to_be_longer_than_its_tokens():
    """All of a row's tokens are its prompt's then, up to the largest number; none are below zero."""
    ops = CudaOps()
    ops.status.zero_()
    h = TokenHistory.zeros(5, 100, "cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")          # noqa: E731
    most = 2 ** 31 - 1
    ops.history_begin(h, i32([0, 1, 2, 3, 4]), i32([7, 8, 9, 10, 11, 12]), i32([0, 1, 3, 4, 5, 6]),
                      i32([most, most, most - 2, -1, -most - 1]))
    assert [r.nonzero().flatten().tolist() for r in h.counts] == [[], [], [], [11], [12]]
    assert h.prompt[:, 0].tolist() == [1 << 7, (1 << 8) | (1 << 9), 1 << 10, 0, 0]
    assert int(ops.status.item()) == 0
