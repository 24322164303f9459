"""Rules on logits, the record of tokens they go by, log-probabilities and page copies: every kernel
against the plain float64 twin, at the sizes, masks and values where it can go wrong."""

import math

import pytest
import torch

import plain_answers
from plain_answers import PlainAnswerOps, pack

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN, INF = math.nan, math.inf


@pytest.fixture(scope="module")
def ops():
    from hetero_serve_b200.kernels import CudaOps
    return CudaOps()


@pytest.fixture(autouse=True)
def clean_status(ops):
    ops.status.zero_()
    yield
    torch.cuda.synchronize()


def status(ops):
    torch.cuda.synchronize()
    return int(ops.status.item())


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def history_of(slots, vocab, device="cpu"):
    from hetero_serve_b200.kernels import TokenHistory
    return TokenHistory.zeros(slots, vocab, device)


def moved(history, device):
    from hetero_serve_b200.kernels import TokenHistory
    return TokenHistory(*(t.to(device) for t in history.tensors()))


def texts(gen, lens, vocab):
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    tokens = (torch.rand(start[-1], generator=gen) ** 3 * vocab).long().clamp(0, vocab - 1)
    return tokens.to(torch.int32), start


def same_history(a, b):
    return all(torch.equal(x.cpu(), y.cpu()) for x, y in zip(a.tensors(), b.tensors()))


# -- the record of tokens -------------------------------------------------------------------


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 512, 4096, 4097, 50257])
def test_history_begin_and_add(ops, vocab):
    gen = torch.Generator().manual_seed(vocab)
    lens, n_prompt = [0, 1, 700, 33, 5000], [0, 1, 400, 33, 0]
    tokens, start = texts(gen, lens, vocab)
    slots = ints([4, -1, 0, 2, 5])
    want = history_of(7, vocab)
    for t in want.tensors():
        t.random_(0, 1 << 30, generator=gen)          # what earlier requests left
    got = moved(want, DEV)
    ops.history_begin(got, slots.to(DEV), tokens.to(DEV), ints(start).to(DEV), ints(n_prompt).to(DEV))
    PlainAnswerOps().history_begin(want, slots, tokens, start, n_prompt)
    assert same_history(got, want)
    add_slots, add = ints([0, 5, -1, 0, 4, 2]), ints([0, vocab - 1, 0, 0, vocab // 2, vocab // 3])
    for _ in range(2):
        ops.history_add(got, add_slots.to(DEV), add.to(DEV))
        PlainAnswerOps().history_add(want, add_slots, add)
    assert same_history(got, want)
    assert status(ops) == 0


def test_history_reports_what_lies_outside(ops):
    h = history_of(2, 100, DEV)
    d = lambda x: ints(x).to(DEV)                                       # noqa: E731
    ops.history_begin(h, d([0, 1]), d([3, 100, -1, 7]), d([0, 3, 4]), d([3, 0]))
    assert status(ops) == 1
    assert h.counts[1, 7].item() == 1 and h.counts.sum().item() == 1
    assert h.prompt.cpu().tolist() == [[8, 0, 0, 0], [0, 0, 0, 0]]
    ops.status.zero_()
    ops.history_add(h, d([2, 1, 0]), d([1, 100, 5]))
    assert status(ops) == 17
    assert h.counts.sum().item() == 2
    ops.status.zero_()
    ops.history_begin(h, d([2]), d([1]), d([0, 1]), d([1]))
    assert status(ops) == 16
    # offsets outside the tokens are cut to them
    ops.status.zero_()
    ops.history_begin(h, d([0, 1]), d([4, 5]), d([-5, 1, 90]), d([0, 0]))
    assert h.counts[0].nonzero().flatten().tolist() == [4]
    assert h.counts[1].nonzero().flatten().tolist() == [5]


def test_history_begin_of_one_slot_twice_keeps_the_last(ops):
    h = history_of(3, 9000, DEV)
    d = lambda x: ints(x).to(DEV)                                       # noqa: E731
    for _ in range(3):
        ops.history_begin(h, d([1, 1, 2, 1]), d([10, 11, 12, 8000]), d([0, 1, 2, 3, 4]), d([0, 1, 0, 0]))
        assert h.counts[1].nonzero().flatten().tolist() == [8000]
        assert int(h.prompt[1].abs().sum()) == 0


# -- rules ------------------------------------------------------------------------------------


def rules_case(gen, rows, vocab, *, history=True, bias=0, mask=None, slots=None):
    s = dict(logits=torch.randn(rows, vocab, generator=gen) * 4)
    if history:
        h = history_of(rows + 2, vocab)
        lens = torch.randint(0, 60, (rows,), generator=gen).tolist()
        tokens, start = texts(gen, lens, vocab)
        PlainAnswerOps().history_begin(h, ints(list(range(rows))), tokens, start,
                                       [n // 2 for n in lens])
        s.update(history=h, slots=torch.randperm(rows + 2, generator=gen)[:rows].to(torch.int32),
                 repetition=0.5 + torch.rand(rows, generator=gen),
                 presence=torch.randn(rows, generator=gen), frequency=torch.randn(rows, generator=gen))
        if rows > 1:
            s["slots"][1] = -1
    if bias:
        n = [int(x) for x in torch.randint(0, bias + 1, (rows,), generator=gen)]
        s["bias_start"] = ints([sum(n[:i]) for i in range(rows + 1)])
        s["bias_ids"] = torch.randint(0, vocab, (max(1, sum(n)),), generator=gen).to(torch.int32)
        s["bias_values"] = torch.randn(max(1, sum(n)), generator=gen) * 3
    if mask is not None:
        s["mask"] = pack(torch.rand(rows + 1, vocab, generator=gen) < mask)
        s["mask_row"] = torch.randint(-1, rows + 1, (rows,), generator=gen).to(torch.int32)
    return s


def on_device(s):
    out = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    if "history" in s:
        out["history"] = moved(s["history"], DEV)
    return out


def check_rules(ops, s, in_place=False):
    """The arithmetic is in 64 bits and rounded once: half a step of float32, and a few steps of
    float64 of the numbers that were added; what no rule touches keeps its bits."""
    d = on_device(s)
    want = torch.empty_like(s["logits"], dtype=torch.float64)
    args = {k: v for k, v in s.items() if k != "logits"}
    PlainAnswerOps().logit_rules(want, s["logits"], **args)
    args = {k: v for k, v in d.items() if k != "logits"}
    got = d["logits"] if in_place else torch.full_like(d["logits"], 7.0)
    ops.logit_rules(got, d["logits"], **args)
    got = got.cpu()
    rounded = want.float()                    # sums beyond the range of float32 are infinite
    finite, infinite = torch.isfinite(rounded), torch.isinf(rounded)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[infinite], rounded[infinite])
    err = (got.double() - want)[finite].abs()
    scale = want[finite].abs() * 2.0 ** -24 + 1e4 * 2.0 ** -52
    assert bool((err <= scale).all()), float((err - scale).max())
    same = want == s["logits"].double()
    assert torch.equal(got[same], s["logits"][same])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,vocab,kw", [
    (1, 1, dict(bias=3, mask=0.5)),
    (3, 31, dict(mask=0.5)),
    (2, 33, dict(bias=40)),
    (5, 1000, dict(bias=20, mask=0.1)),
    (4, 4097, dict(history=False, mask=0.02)),
    (3, 4099, dict(bias=300)),
    (2, 50257, dict(bias=100, mask=0.5)),
    (40, 517, dict(bias=9, mask=0.9)),
    (700, 65, dict(bias=2, mask=0.6)),
    (90, 13001, dict(bias=3)),
    (90, 13001, dict(mask=0.7)),
    (310, 9001, dict()),
    (310, 9001, dict(bias=5, mask=0.05)),
    (2, 4099, dict(bias=6000, mask=0.5)),        # more biases than a tile keeps at hand
    (130, 9001, dict(bias=3000)),
])
def test_rules_follow_the_plain_form(ops, rows, vocab, kw, in_place):
    gen = torch.Generator().manual_seed(rows * 131 + vocab)
    check_rules(ops, rules_case(gen, rows, vocab, **kw), in_place)
    assert status(ops) == 0


def test_rules_without_any_copy_the_logits(ops):
    x = torch.randn(3, 1001, device=DEV)
    out = torch.empty_like(x)
    ops.logit_rules(out, x)
    assert torch.equal(out, x)
    ops.logit_rules(x[:0], x[:0])


def test_rules_on_odd_bases(ops):
    """Logits and results that begin at any of the four places of a 16-byte piece."""
    gen = torch.Generator().manual_seed(4)
    s = on_device(rules_case(gen, 3, 1001, bias=5, mask=0.5))
    args = {k: v for k, v in s.items() if k != "logits"}
    want = torch.empty_like(s["logits"])
    ops.logit_rules(want, s["logits"], **args)
    for a in range(4):
        for b in range(4):
            x = torch.empty(3 * 1001 + 4, device=DEV)[a:a + 3003].view(3, 1001).copy_(s["logits"])
            room = torch.full((3 * 1001 + 8,), 5.0, device=DEV)
            out = room[b:b + 3003].view(3, 1001)
            ops.logit_rules(out, x, **args)
            assert torch.equal(out, want)
            assert bool((room[:b] == 5).all()) and bool((room[b + 3003:] == 5).all())


@pytest.mark.parametrize("in_place", [False, True])
def test_rules_on_numbers_that_are_none(ops, in_place):
    vocab = 70
    s = rules_case(torch.Generator().manual_seed(1), 4, vocab, bias=0, mask=0.5)
    s["logits"][:, ::7] = NAN
    s["logits"][:, 1::7] = -INF
    s["logits"][:, 2::7] = INF
    s["logits"][:, 3::7] = torch.finfo(torch.float32).min
    s["logits"][:, 4::7] = 0.0
    s["mask_row"] = ints([0, 1, -1, 2])
    s["mask"][1] = 0                                       # rules everything out
    s["bias_start"], s["bias_ids"] = ints([0, 4, 4, 8, 8]), ints([0, 1, 2, 3, 1, 2, 3, 5])
    s["bias_values"] = torch.tensor([-INF, INF, -INF, -1e38, 1.0, -INF, 3e38, -INF])
    check_rules(ops, s, in_place)
    got = s["logits"].to(DEV)
    d = on_device(s)
    ops.logit_rules(got, got, mask=d["mask"], mask_row=d["mask_row"])
    assert bool((got[1] == -INF).all())


def test_the_last_of_two_biases_of_one_token_counts(ops):
    s = dict(logits=torch.zeros(2, 5000), bias_start=ints([0, 300, 600]),
             bias_ids=ints([4321] * 600), bias_values=torch.arange(600.0))
    check_rules(ops, s)


def test_rules_report_what_lies_outside(ops):
    s = on_device(rules_case(torch.Generator().manual_seed(2), 3, 40, mask=0.5))
    base = s["logits"].clone()
    args = {k: v for k, v in s.items() if k != "logits"}
    args.update(slots=ints([900, -1, -7]).to(DEV), mask_row=ints([-1, -5, 99]).to(DEV))
    out = torch.empty_like(base)
    ops.logit_rules(out, base, **args)
    assert torch.equal(out, base) and status(ops) == 16
    ops.status.zero_()
    ops.logit_rules(out, base, bias_start=ints([-3, 2, 2, 99]).to(DEV),
                    bias_ids=ints([40, 3, -1, 5]).to(DEV),
                    bias_values=torch.ones(4, device=DEV))
    base[0, 3] += 1
    base[2, 5] += 1
    assert torch.equal(out, base) and status(ops) == 1


def test_counts_above_the_exact_integers_of_float32(ops):
    s = rules_case(torch.Generator().manual_seed(3), 1, 64)
    s["slots"][0] = 0
    s["history"].counts.fill_(2 ** 24 + 1)
    s["history"].output.fill_(-1)
    s["frequency"][0], s["presence"][0], s["repetition"][0] = 2.0 ** -20, 0.25, 1.25
    check_rules(ops, s)


@pytest.mark.parametrize("vocab", [40, 5003, 50257])
def test_sampling_stays_within_what_the_rules_leave(ops, vocab):
    """Every sampler over rows of which one, two or five tokens are left, with k below and above."""
    rows = 24
    gen = torch.Generator().manual_seed(vocab)
    left = [torch.randperm(vocab, generator=gen)[:(1, 2, 5)[r % 3]] for r in range(rows)]
    flags = torch.zeros(rows, vocab, dtype=torch.bool)
    for r, ids in enumerate(left):
        flags[r, ids] = True
    x = (torch.randn(rows, vocab, generator=gen) * 4).to(DEV)
    out = torch.empty_like(x)
    row = torch.arange(rows, dtype=torch.int32, device=DEV)
    ops.logit_rules(out, x, mask=pack(flags).to(DEV), mask_row=row)
    tokens, zero = torch.empty_like(row), torch.zeros_like(row)
    for k in (0, 1, 3, 30):
        for temperature in (0.0, 0.7, 3.0):
            for position in range(4):
                ops.sample(tokens, out, torch.full((rows,), temperature, device=DEV), zero + k, row, zero,
                           zero + position)
                assert all(t in ids.tolist() for t, ids in zip(tokens.tolist(), left)), (k, temperature)


# -- log-probabilities --------------------------------------------------------------------------


def check_logprobs(ops, logits, tokens, top):
    rows, vocab = logits.shape
    lp, rk = torch.empty(rows, dtype=torch.float64), torch.empty(rows, dtype=torch.int32)
    ids = torch.empty(rows, top, dtype=torch.int32) if top else None
    tl = torch.empty(rows, top, dtype=torch.float64) if top else None
    PlainAnswerOps().token_logprobs(lp, rk, logits, tokens, ids, tl)
    d = lambda t, dt: torch.full(t.shape, 77, dtype=dt, device=DEV) if t is not None else None  # noqa: E731
    g = [d(lp, torch.float32), d(rk, torch.int32), d(ids, torch.int32), d(tl, torch.float32)]
    ops.token_logprobs(g[0], g[1], logits.to(DEV), tokens.to(DEV), g[2], g[3])
    assert torch.equal(g[1].cpu(), rk)
    pairs = [(g[0], lp)]
    if top:
        assert torch.equal(g[2].cpu(), ids)
        pairs.append((g[3], tl))
    # A partial sum takes at most ceil(vocab / 256) additions of positive terms, the joining of
    # sums 16 more, each wrong by half a step of what it holds; a term exp(x - m) by two steps, and
    # by |x - m| half steps of its argument's rounding (of terms that weigh nothing where that is
    # large: e^-a a <= 1/e, so 2 together with the base change covers it).  The logarithm turns the
    # sum's relative error into an absolute one; its own and the two subtractions' errors are steps
    # of the numbers themselves.
    for got, want in pairs:
        got, finite = got.cpu().double(), torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)])
        steps = -(-vocab // 256) + 16 + 2 * 2 + 2 + math.log(vocab) + 4 * want[finite].abs()
        err = (got[finite] - want[finite]).abs()
        assert bool((err <= steps * 2.0 ** -24).all()), float(err.max())


@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 2), (2, 31, 31), (4, 33, 32), (5, 255, 0), (3, 257, 7), (2, 1000, 20),
    (3, 4099, 32), (2, 8193, 1), (1, 50257, 5), (3, 50257, 32), (2, 70001, 20), (300, 130, 20),
    (700, 67, 3), (150, 8200, 0), (150, 8200, 2),
    (600, 8200, 0), (20, 24600, 3), (70, 24600, 1)])
def test_logprobs_follow_the_plain_form(ops, rows, vocab, top):
    gen = torch.Generator().manual_seed(rows * 7 + vocab + top)
    logits = torch.randn(rows, vocab, generator=gen) * 3
    tokens = torch.randint(0, vocab, (rows,), generator=gen).to(torch.int32)
    if rows > 1:
        tokens[1] = int(logits[1].argmax())
    if rows > 2:
        tokens[2] = -1
    check_logprobs(ops, logits, tokens, top)
    assert status(ops) == 0


@pytest.mark.parametrize("vocab", [9, 700, 5003, 50257])
def test_equal_logits_stand_in_the_order_of_their_indices(ops, vocab):
    gen = torch.Generator().manual_seed(vocab)
    logits = torch.stack([torch.zeros(vocab), torch.full((vocab,), -INF),
                          torch.randint(0, 3, (vocab,), generator=gen).float(),
                          torch.where(torch.rand(vocab, generator=gen) < 0.5, 0.0, -0.0),
                          torch.arange(vocab).float() * 2.0 ** -10,
                          torch.arange(vocab).flip(0).float() * 2.0 ** -10])
    check_logprobs(ops, logits, ints([vocab - 1, vocab // 2, 0, vocab // 3, vocab - 2, 1]),
                   min(vocab, 20))


def test_all_large_logits_in_one_thread(ops):
    """The largest all lie where one thread reads, whatever the stride: dense runs and every
    256th, 512th, 1,024th and 2,048th place, more of them than there are alternatives."""
    vocab = 50257
    gen = torch.Generator().manual_seed(11)
    logits = torch.randn(6, vocab, generator=gen)
    logits[0, 1000:1200] += 50
    for r, stride in enumerate((256, 512, 1024, 2048), 1):
        logits[r, 3::stride] += 50
    logits[5, :40] += 50
    logits[5, -40:] += 50
    check_logprobs(ops, logits, ints([1100, 3, 3, 3, 3, vocab - 1]), 32)


@pytest.mark.parametrize("vocab", [40, 3001])
def test_logprobs_of_numbers_that_are_none(ops, vocab):
    gen = torch.Generator().manual_seed(vocab)
    base = torch.randn(vocab, generator=gen)
    rows = [base.clone() for _ in range(8)]
    rows[0][::2] = -INF                                    # masked tokens, one of them asked for
    rows[1][:] = -INF
    rows[1][17] = 2.5                                      # a single token is left
    rows[2][5] = NAN
    rows[3][6] = INF
    rows[4][:] = NAN
    rows[5][:] = -INF
    rows[5][3] = NAN
    rows[6][:] = torch.finfo(torch.float32).min
    rows[7][9] = torch.finfo(torch.float32).max
    logits = torch.stack(rows)
    check_logprobs(ops, logits, ints([0, 3, 5, 6, 7, 1, 8, 10]), 10)


def test_logprobs_report_tokens_outside(ops):
    logits = torch.randn(3, 50, device=DEV)
    lp, rk = torch.zeros(3, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    ops.token_logprobs(lp, rk, logits, ints([50, -1, 4]).to(DEV))
    assert status(ops) == 1
    assert rk.tolist()[:2] == [-1, -1] and torch.isnan(lp).tolist() == [True, True, False]


def test_logits_at_odd_bases(ops):
    for off in range(4):
        x = torch.randn(2 * 5003 + 4, generator=torch.Generator().manual_seed(off))
        view = x.to(DEV)[off:off + 10006].view(2, 5003)
        ids = torch.empty(2, 6, dtype=torch.int32, device=DEV)
        tl, lp = torch.empty(2, 6, device=DEV), torch.empty(2, device=DEV)
        rk = torch.empty(2, dtype=torch.int32, device=DEV)
        ops.token_logprobs(lp, rk, view, ints([1, 5002]).to(DEV), ids, tl)
        order = view.sort(dim=1, descending=True, stable=True)
        assert torch.equal(ids.long(), order.indices[:, :6])
        want = torch.log_softmax(view.double(), 1).gather(1, ids.long())
        assert float((tl - want).abs().max()) < 60 * 2.0 ** -24 * 4


# -- pages ----------------------------------------------------------------------------------------


def pools(gen, entries, planes, heads, page, dim, dtype, n_dst, n_src=None):
    shape = (planes, heads, page, dim)
    dst = torch.randn(entries, n_dst, *shape, generator=gen).to(dtype)
    if n_src is None:
        return dst, dst
    return dst, torch.randn(entries, n_src, *shape, generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("entries,planes,heads,page,dim,pairs", [
    (1, 1, 1, 16, 1, 1), (2, 2, 3, 4, 5, 3), (3, 1, 1, 16, 576, 9), (24, 2, 16, 16, 64, 7),
    (1, 2, 2, 32, 20, 40), (2, 2, 1, 16, 2, 1500)])
def test_copies_follow_the_plain_form(ops, dtype, entries, planes, heads, page, dim, pairs):
    gen = torch.Generator().manual_seed(pairs * 3 + dim)
    for one_pool in (True, False):
        for partial in (True, False):
            n = 2 * pairs + 3
            dst, src = pools(gen, entries, planes, heads, page, dim, dtype, n,
                             None if one_pool else pairs + 1)
            order = torch.randperm(n, generator=gen).tolist()
            to = order[:pairs]
            of = ([order[pairs + i % max(1, pairs // 2)] for i in range(pairs)] if one_pool
                  else [i % (pairs + 1) for i in range(pairs)])
            rows = torch.randint(0, page + 1, (pairs,), generator=gen).tolist() if partial else None
            got = dst.to(DEV)
            ops.copy_pages(got, got if one_pool else src.to(DEV), to, of, rows)
            PlainAnswerOps().copy_pages(dst, src, to, of, rows)
            assert torch.equal(got.cpu(), dst)


def test_copies_move_bits(ops):
    """NaNs, infinities and denormals arrive as they were, and an offset pool is served."""
    bits = torch.randint(-2 ** 15, 2 ** 15, (1 + 2 * 8 * 2 * 1 * 16 * 6,), dtype=torch.int16)
    flat = bits.to(DEV)
    pool = flat[1:].view(torch.bfloat16).view(2, 8, 2, 1, 16, 6)
    ops.copy_pages(pool, pool, [0, 7], [3, 3], [5, 16])
    want = bits[1:].view(2, 8, 2, 1, 16, 6).clone()
    want[:, 0, :, :, :5] = want[:, 3, :, :, :5]
    want[:, 7] = want[:, 3]
    assert torch.equal(flat[1:].cpu().view(2, 8, 2, 1, 16, 6), want)
    assert flat[0].item() == bits[0].item()


# -- large offsets, and what lies behind the rows ---------------------------------------------------


def _room(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes * 2 ** 30:
        pytest.skip("not enough free device memory")


def test_pages_behind_four_billion_numbers(ops):
    _room(12)
    pool = torch.empty(2, 34000, 2, 16, 32, 64, dtype=torch.bfloat16, device=DEV)     # 8.3 GiB
    assert pool.numel() > 2 ** 32
    pool[:, [5, 33999]] = torch.randn(2, 2, 2, 16, 32, 64, device=DEV).bfloat16()
    ops.copy_pages(pool, pool, [33998, 7, 33997], [5, 33999, 33999], [32, 32, 11])
    for e in range(2):
        assert torch.equal(pool[e, 33998], pool[e, 5]) and torch.equal(pool[e, 7], pool[e, 33999])
        assert torch.equal(pool[e, 33997, :, :, :11], pool[e, 33999, :, :, :11])
    del pool
    torch.cuda.empty_cache()


def test_rows_behind_two_billion_logits(ops):
    _room(24)
    rows, vocab = 17000, 131101
    x = torch.empty(rows, vocab, device=DEV)                                           # 8.3 GiB
    assert x.numel() > 2 ** 31
    x[-2:] = torch.randn(2, vocab, device=DEV)
    keep = x[-2:].clone()
    lp = torch.full((rows + 3,), 9.0, device=DEV)
    rk = torch.full((rows + 3,), 9, dtype=torch.int32, device=DEV)
    tokens = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    tokens[-1] = int(keep[1].argmax())
    ids = torch.full((rows + 1, 2), 9, dtype=torch.int32, device=DEV)
    lps = torch.full((rows + 1, 2), 9.0, device=DEV)
    ops.token_logprobs(lp, rk, x, tokens, ids, lps)
    want = torch.log_softmax(keep[1].double(), 0)
    assert rk[rows - 1].item() == 0 and abs(float(lp[rows - 1]) - float(want.max())) < 1e-4
    assert torch.equal(ids[rows - 2:rows].long(), keep.topk(2, dim=1).indices)
    assert bool((lp[rows:] == 9).all()) and bool((rk[rows:] == 9).all())               # left as they were
    assert bool((ids[rows:] == 9).all()) and bool((lps[rows:] == 9).all())
    history = history_of(17001, 1, DEV)            # (another vocabulary is refused)
    start = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
    start[rows] = 2
    bias = dict(bias_start=start, bias_ids=ints([0, vocab - 1]).to(DEV),
                bias_values=torch.tensor([1.0, -INF], device=DEV))
    from hetero_serve_b200.kernels import KernelError
    with pytest.raises(KernelError):
        ops.logit_rules(x, x, history, tokens, lp, lp, lp, **bias)
    ops.logit_rules(x, x, **bias)
    keep[1, 0] += 1
    keep[1, -1] = -INF
    assert torch.equal(x[-2:], keep)
    out = torch.empty_like(x)
    ops.logit_rules(out, x, **bias)
    keep[1, 0] += 1
    assert torch.equal(out[-2:], keep)
    del x, out
    torch.cuda.empty_cache()
    assert status(ops) == 0


def test_a_record_behind_two_billion_counts(ops):
    _room(12)
    slots, vocab = 16400, 131101
    h = history_of(slots, vocab, DEV)
    assert h.counts.numel() > 2 ** 31
    s = torch.tensor([slots - 1], dtype=torch.int32, device=DEV)
    d = lambda x: ints(x).to(DEV)                                       # noqa: E731
    ops.history_begin(h, s, d([vocab - 1, 3, 3]), d([0, 3]), d([1]))
    ops.history_add(h, s, d([vocab - 1]))
    assert h.counts[-1].nonzero().flatten().tolist() == [3, vocab - 1]
    assert int(h.counts.sum()) == 3 and int((h.prompt != 0).sum()) == 1
    x = torch.ones(1, vocab, device=DEV)
    one = torch.ones(1, device=DEV)
    ops.logit_rules(x, x, h, s, 2 * one, one, one)
    assert x[0, 3].item() == 0.5 - 3 and x[0, -1].item() == 0.5 - 2 and x[0, 4].item() == 1
    del h
    torch.cuda.empty_cache()


def test_tensors_elsewhere_are_refused(ops):
    from hetero_serve_b200.kernels import KernelError
    x = torch.zeros(2, 40, device=DEV)
    one, i = torch.ones(2, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    with pytest.raises(KernelError):
        ops.logit_rules(x.cpu(), x)
    with pytest.raises(KernelError):
        ops.logit_rules(x, x, history_of(2, 40), i, one, one, one)
    with pytest.raises(KernelError):
        ops.logit_rules(x, x, history_of(2, 40, DEV), i.cpu(), one, one, one)
    with pytest.raises(KernelError):
        ops.token_logprobs(one, i, x, i.cpu())
    with pytest.raises(KernelError):
        ops.token_logprobs(one, i[::2], x, i)
    pool = torch.zeros(1, 4, 1, 1, 16, 8, device=DEV)
    with pytest.raises(KernelError):
        ops.copy_pages(pool, pool.cpu(), [0], [1])
    with pytest.raises(KernelError):
        ops.copy_pages(pool.cpu(), pool, [0], [1])


# -- together, captured, on another stream --------------------------------------------------------


def end_of_step(ops, s, out, history, tokens, feedback, scores):
    """As the engine's step ends: rules, sampling, the sampled tokens counted, their scores."""
    rows = out.shape[0]
    ops.logit_rules(out, s["logits"], history, s["slots"], s["repetition"], s["presence"],
                    s["frequency"], bias_start=s["bias_start"], bias_ids=s["bias_ids"],
                    bias_values=s["bias_values"], mask=s["mask"], mask_row=s["mask_row"])
    zeros = torch.zeros(rows, dtype=torch.int32, device=DEV)
    ops.sample(tokens, out, torch.zeros(rows, device=DEV), zeros, zeros, zeros, zeros,
               feedback=feedback, feedback_slot=s["slots"])
    ops.history_add(history, s["slots"], tokens)
    ops.token_logprobs(scores[0], scores[1], s["logits"], tokens, scores[2], scores[3])


@pytest.mark.parametrize("how", ["eager", "stream", "graph"])
def test_the_end_of_a_step_repeats_itself_as_plain_code_does(ops, how):
    rows, vocab, steps = 5, 3001, 6
    gen = torch.Generator().manual_seed(8)
    s = rules_case(gen, rows, vocab, bias=30, mask=0.3)
    s["mask_row"] = ints([0, 1, -1, 2, 3])
    d = on_device(s)
    feedback = torch.zeros(rows + 2, dtype=torch.int32, device=DEV)
    tokens = torch.zeros(rows, dtype=torch.int32, device=DEV)
    out = torch.empty_like(d["logits"])
    scores = (torch.empty(rows, device=DEV), torch.empty(rows, dtype=torch.int32, device=DEV),
              torch.empty(rows, 4, dtype=torch.int32, device=DEV), torch.empty(rows, 4, device=DEV))
    run = lambda: end_of_step(ops, d, out, d["history"], tokens, feedback, scores)   # noqa: E731
    if how == "graph":
        run()
        for a, b in zip(d["history"].tensors(), s["history"].tensors()):
            a.copy_(b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        run = graph.replay
    side = torch.cuda.Stream()
    plain, want = PlainAnswerOps(), s["history"]
    for step in range(steps):
        x = torch.randn(rows, vocab, generator=gen) * 3
        s["logits"].copy_(x)
        if how == "stream":
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                d["logits"].copy_(x)
                run()
            torch.cuda.current_stream().wait_stream(side)
        else:
            d["logits"].copy_(x)
            run()
        ruled = torch.empty(rows, vocab, dtype=torch.float64)
        plain.logit_rules(ruled, **{k: v for k, v in s.items()})
        best = ruled.float().argmax(1).to(torch.int32)
        assert torch.equal(tokens.cpu(), best), step
        plain.history_add(want, s["slots"], best)
        assert same_history(d["history"], want)
        lp = torch.log_softmax(x.double(), 1).gather(1, best.long()[:, None])[:, 0]
        assert float((scores[0].cpu() - lp).abs().max()) < 100 * 2.0 ** -24
        assert torch.equal(scores[2].cpu().long(), x.topk(4, dim=1).indices)
    assert status(ops) == 0
