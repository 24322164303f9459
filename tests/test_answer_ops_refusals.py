"""What the operations around a step's answers refuse, without a GPU: the lists of page copies on
the host; the checks of tensors on an object whose library stands in for the CUDA one."""

import numpy as np
import pytest
import torch

from hetero_serve_b200.kernels import KernelError, TokenHistory
from hetero_serve_b200.kernels import ops as ops_module
from hetero_serve_b200.kernels.ops import CudaOps, history_words, page_lists


class NoLibrary:
    """Every entry point answers 0 and remembers that it was called."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


@pytest.fixture
def ops(monkeypatch):
    monkeypatch.setattr(ops_module, "_want",
                        lambda t, name, dtype=None, dim=None, cuda=True, _w=ops_module._want:
                        _w(t, name, dtype, dim, False))
    o = CudaOps.__new__(CudaOps)
    o.device, o._index, o.lib, o.launches = torch.device("cpu"), -1, NoLibrary(), 0
    o.status = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(CudaOps, "_stream", lambda self: 0)
    monkeypatch.setattr(CudaOps, "_drives", lambda self, what, *tensors: None)
    return o


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("to,of,rows,one,why", [
    ([0, 1], [2], None, True, "different lengths"),
    ([0, 1], [2, 3], [1], True, "different lengths"),
    ([0, 0], [2, 3], None, True, "written twice"),
    ([0, 0], [2, 3], None, False, "written twice"),
    ([0, 1], [1, 2], None, True, "also read"),
    ([5], [5], None, True, "also read"),
    ([10], [0], None, True, "outside"),
    ([-1], [0], None, True, "outside"),
    ([0], [8], None, False, "outside"),
    ([2 ** 32], [0], None, False, "outside"),
    ([0], [1], [17], True, "outside"),
    ([0], [1], [-1], True, "outside"),
    ([0.5], [1], None, True, "whole numbers"),
    ([[0]], [[1]], None, True, "whole numbers"),
])
def test_page_lists_that_are_refused(to, of, rows, one, why):
    with pytest.raises(KernelError, match=why):
        page_lists(to, of, rows, 10, 8 if not one else 10, 16, one)


def test_page_lists_that_are_taken():
    to, of, rows = page_lists([3, 0], [3, 3], [0, 16], 10, 8, 16, False)
    assert to.tolist() == [3, 0] and of.tolist() == [3, 3] and rows.tolist() == [0, 16]
    assert len(page_lists([], [], None, 10, 10, 16, True)[0]) == 0
    many = np.arange(400)
    for kind in (many, many.tolist(), many.astype(np.uint16), torch.arange(400)):
        to, of, rows = page_lists(kind, many + 400, many % 17, 800, 800, 16, True)
        assert to.tolist() == many.tolist() and of.tolist() == (many + 400).tolist()
        assert rows.tolist() == (many % 17).tolist()


@pytest.mark.parametrize("many,why", [
    (np.arange(400) % 399, "written twice"), (np.arange(400) - 1, "outside"),
    (np.arange(400) + 401, "outside"), (np.arange(400) + 2 ** 32, "outside"),
    (np.arange(400) + 0.0, "whole numbers"), (np.arange(400) + 1, "also read"),
])
def test_long_page_lists_that_are_refused(many, why):
    for kind in (many, many.tolist()):
        with pytest.raises(KernelError, match=why):
            page_lists(kind, np.arange(400) + 400, None, 800, 800, 16, True)


def test_page_copies_refuse_pools_that_do_not_match(ops):
    pool = torch.zeros(2, 8, 2, 1, 16, 4)
    for other in (torch.zeros(3, 8, 2, 1, 16, 4), torch.zeros(2, 8, 2, 1, 16, 8),
                  torch.zeros(2, 8, 2, 1, 16, 4, dtype=torch.bfloat16), torch.zeros(8, 2, 1, 16, 4),
                  torch.zeros(2, 8, 2, 1, 4, 16).transpose(-1, -2), torch.zeros(2, 8, 2, 1, 16, 4).half()):
        with pytest.raises(KernelError):
            ops.copy_pages(pool, other, [0], [1])
    both = torch.zeros(3, 8, 2, 1, 16, 4)
    with pytest.raises(KernelError, match="overlap"):
        ops.copy_pages(both[:2], both[1:], [0], [1])
    assert ops.lib.calls == []
    ops.copy_pages(pool, pool, [], [])
    assert ops.lib.calls == []
    ops.copy_pages(pool, pool, [0], [1])
    assert ops.lib.calls == ["hs_copy_pages"]


def test_rules_refuse_what_does_not_fit(ops):
    x, out = torch.zeros(3, 100), torch.zeros(3, 100)
    h, f = TokenHistory.zeros(4, 100, "cpu"), torch.ones(3)
    full = dict(history=h, slots=i32(3), repetition=f, presence=f, frequency=f)
    bad = [dict(full, slots=i32(2)), dict(full, slots=None), dict(full, repetition=f[:2]),
           dict(full, presence=f.double()), dict(full, frequency=None),
           dict(full, history=TokenHistory.zeros(4, 99, "cpu")),
           dict(full, history=h.counts), dict(slots=i32(3)),
           dict(bias_start=i32(3), bias_ids=i32(2), bias_values=torch.zeros(2)),
           dict(bias_start=i32(4), bias_ids=i32(2), bias_values=torch.zeros(1)),
           dict(bias_start=i32(4), bias_ids=i32(2)), dict(bias_ids=i32(2)),
           dict(mask=i32(2, 3), mask_row=i32(3)), dict(mask=i32(2, 4), mask_row=i32(2)),
           dict(mask=i32(2, 4)), dict(mask_row=i32(3)), dict(mask=i32(0, 4), mask_row=i32(3))]
    for kw in bad:
        with pytest.raises(KernelError):
            ops.logit_rules(out, x, **kw)
    for parts in ((h.prompt, h.output[:3], h.counts), (h.prompt, h.output, h.counts.float()),
                  (h.prompt[:, :3].contiguous(), h.output, h.counts), (h.prompt, None, h.counts)):
        with pytest.raises(KernelError):
            TokenHistory(*parts)
    for o, l in ((out[:2], x), (out.double(), x), (torch.zeros(100, 3).T, x), (out, x.bfloat16())):
        with pytest.raises(KernelError):
            ops.logit_rules(o, l)
    room = torch.zeros(400)
    with pytest.raises(KernelError, match="overlaps"):
        ops.logit_rules(room[:300].view(3, 100), room[100:].view(3, 100))
    assert ops.lib.calls == []
    ops.logit_rules(x, x, **full, bias_start=i32(4), bias_ids=i32(2), bias_values=torch.zeros(2),
                    mask=i32(2, history_words(100)), mask_row=i32(3))
    assert ops.lib.calls == ["hs_logit_rules"]


def test_histories_and_scores_refuse_what_does_not_fit(ops):
    h = TokenHistory.zeros(4, 100, "cpu")
    for kw in (dict(start=i32(2)), dict(n_prompt=i32(1)), dict(tokens=torch.zeros(5)),
               dict(slots=i32(2, 1))):
        args = dict(slots=i32(2), tokens=i32(5), start=i32(3), n_prompt=i32(2))
        with pytest.raises(KernelError):
            ops.history_begin(h, **{**args, **kw})
    with pytest.raises(KernelError):
        ops.history_add(h, i32(3), i32(2))
    ops.history_begin(h, i32(0), i32(0), i32(1), i32(0))
    ops.history_add(h, i32(0), i32(0))
    x, lp, rk = torch.zeros(3, 30), torch.zeros(3), i32(3)
    for args, kw in (((lp[:2], rk, x, i32(3)), {}), ((lp, rk, x, i32(2)), {}),
                     ((lp, lp, x, i32(3)), {}), ((lp, rk, x.double(), i32(3)), {}),
                     ((lp, rk, x, i32(3)), dict(top_ids=i32(3, 2))),
                     ((lp, rk, x, i32(3)), dict(top_ids=i32(3, 2), top_logprobs=torch.zeros(3, 3))),
                     ((lp, rk, x, i32(3)), dict(top_ids=i32(2, 2), top_logprobs=torch.zeros(2, 2))),
                     ((lp, rk, x, i32(3)), dict(top_ids=i32(3, 31), top_logprobs=torch.zeros(3, 31)))):
        with pytest.raises(KernelError):
            ops.token_logprobs(*args, **kw)
    wide = torch.zeros(3, 100)
    with pytest.raises(KernelError):
        ops.token_logprobs(lp, rk, wide, i32(3), i32(3, 33), torch.zeros(3, 33))
    assert ops.lib.calls == []
    ops.token_logprobs(lp, rk, wide, i32(3), i32(3, 32), torch.zeros(3, 32))
    assert ops.lib.calls == ["hs_token_logprobs"]
