"""Drawing from rows under rules: a token whose weight is zero (ruled out by a mask or a bias of -inf)
is never drawn, wherever the draw falls among the sums of the weights."""

import pytest
import torch

from hetero_serve_b200.kernels.ops import CudaOps

pytestmark = pytest.mark.gpu
DEV = "cuda"
# a vocabulary, the rows of a launch and the launches: a block a row in shared memory, a cluster a row, a
# block a row streamed from memory.  A thread sums a range of positions, the threads' sums are summed in
# another order, and so a draw in a few 2^-24 of the total falls between the end of one thread's sums and
# the beginning of the next one's (or behind the last): a million draws meet some.
WAYS = [(4096, 16384, 64), (24576, 64, 4096), (60000, 512, 96)]


def drawn(ops, x, launches, top_k):
    """Which tokens are ever drawn from one row of logits, for other positions of many seeds."""
    rows, vocab = x.shape
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    seeds, zero = torch.arange(rows, dtype=torch.int32, device=DEV), i32([0] * rows)
    temp, k = torch.full((rows,), 0.9, device=DEV), i32([top_k] * rows)
    out = torch.empty(rows, dtype=torch.int32, device=DEV)
    seen = torch.zeros(vocab, dtype=torch.bool, device=DEV)
    for i in range(launches):
        ops.sample(out, x, temp, k, seeds, zero, zero + i)
        seen[out.long()] = True
    return seen


@pytest.mark.parametrize("vocab,rows,launches", WAYS)
@pytest.mark.parametrize("kind", ["between", "behind", "few", "underflow", "top_k"])
def test_only_tokens_with_a_weight_are_drawn(vocab, rows, launches, kind):
    ops = CudaOps(DEV)
    g = torch.Generator(device=DEV).manual_seed(vocab)
    row = torch.randn(vocab, device=DEV, generator=g)
    keep = torch.zeros(vocab, dtype=torch.bool, device=DEV)
    if kind == "behind":                         # nothing behind the first three quarters
        keep[:3 * vocab // 4] = True
    elif kind == "few":                          # a grammar's two in a hundred
        keep = torch.rand(vocab, device=DEV, generator=g) < 0.02
    else:                                        # one in five
        keep[4::5] = True
    top_k = vocab - 5 if kind == "top_k" else 0  # (more than there are: the threshold is -inf)
    row = torch.where(keep, row, -1e4 if kind == "underflow" else -torch.inf)
    seen = drawn(ops, row.repeat(rows, 1), launches, top_k)
    assert not bool((seen & ~keep).any()), torch.nonzero(seen & ~keep).flatten().tolist()
    assert int(seen.sum()) > 0
