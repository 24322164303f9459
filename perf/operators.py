"""What the operators around the end of a decode step, and the cache's page copies, are measured by.

Each case is one pass through an operator, as the engine makes it (``CudaOps``):

``rules``     ``logit_rules``: penalties for tokens of the prompt and of the answer so far, biases,
              grammar masks, on the float32 logits of a step.
``history``   ``history_begin`` and ``history_add``: the record of what requests hold, made when they
              are admitted, and one sampled token each counted into it.
``logprobs``  ``token_logprobs``: log-probability and rank of given tokens, and the largest
              alternatives with theirs.
``pages``     ``copy_pages``: pages of a cache copied inside a pool (a fork: the rows that are
              filled) or from one pool into another (a cache that is made smaller or larger).

Vocabularies are that of the GPT-2 family and round ones; pools are those of GPT-2 small and medium.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
GPT2_VOCAB = 50257
MASKED = 0.98           # share of the vocabulary that a grammar rules out at a step
LARGEST_LOGITS = 256 * 131072       # rules: rows * vocabulary of the largest listed case
LARGEST_SCORED = 2048 * GPT2_VOCAB
LARGEST_COPY = 2500 * 12 * 2 * 12 * 16 * 64 * 2     # bytes moved, one way


def _rules(name, rows, vocab, prompt, generated, penalties=True, bias=0, grammar=False):
    return dict(kind="rules", name=name, rows=rows, vocab=vocab, prompt=prompt,
                generated=generated, penalties=penalties, bias=bias, grammar=grammar)


def _history(name, slots, vocab, prompt, generated):
    return dict(kind="history", name=name, slots=slots, vocab=vocab, prompt=prompt,
                generated=generated)


def _logprobs(name, rows, vocab, top):
    return dict(kind="logprobs", name=name, rows=rows, vocab=vocab, top=top)


def _pages(name, job, entries, planes, heads, dim, pages, pairs, page=16, dtype="bfloat16"):
    return dict(kind="pages", name=name, job=job, entries=entries, planes=planes, heads=heads,
                dim=dim, pages=pages, pairs=pairs, page=page, dtype=dtype)


def listed():
    return [
        # one user's request with a repetition penalty: a launch and a chain of loads
        _rules("rules_b1", 1, GPT2_VOCAB, 400, 100),
        # a decode batch whose requests all have penalties, some of them biased tokens
        _rules("rules_b64", 64, GPT2_VOCAB, 500, 200, bias=100),
        # answers that follow a grammar: nearly every token is ruled out
        _rules("rules_grammar_b32", 32, GPT2_VOCAB, 300, 60, penalties=False, grammar=True),
        # the largest batch over a large vocabulary, with everything at once
        _rules("rules_all_b256", 256, 131072, 1500, 500, bias=300, grammar=True),
        # a request is admitted
        _history("history_admit_1", 1, GPT2_VOCAB, 900, 0),
        # a full batch comes back after its pages ran out: long prompts, answers half way
        _history("history_admit_64", 64, GPT2_VOCAB, 3000, 900),
        # one user asks for five alternatives to each token
        _logprobs("logprobs_b1_top5", 1, GPT2_VOCAB, 5),
        # a decode batch with twenty alternatives
        _logprobs("logprobs_b64_top20", 64, GPT2_VOCAB, 20),
        # given text is scored: every place of a prompt, no alternatives
        _logprobs("logprobs_score_2048", 2048, GPT2_VOCAB, 0),
        # eight answers to one prompt: the partly filled page behind it, in every layer
        _pages("pages_fork_8", "fork", 24, 2, 16, 64, 256, 7),
        # sixteen such requests in 32 bits
        _pages("pages_fork_16x4_f32", "fork", 24, 2, 16, 64, 512, 48, dtype="float32"),
        # a cache made smaller while it holds requests: every live page moves
        _pages("pages_resize_2500", "resize", 12, 2, 12, 64, 4096, 2500),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rules"] * 3 + ["history"] * 2 + ["logprobs"] * 3 + ["pages"] * 2)
    if kind == "rules":
        vocab = rng.choice([GPT2_VOCAB, _spread(rng, 200, 131072)])
        case = _rules("", _spread(rng, 1, min(256, LARGEST_LOGITS // vocab)), vocab,
                      _spread(rng, 1, 1500), _spread(rng, 1, 500),
                      penalties=rng.random() < 0.8,
                      bias=rng.choice([0, _spread(rng, 1, 300)]), grammar=rng.random() < 0.4)
        case["bias"] = min(case["bias"], vocab // 2)
    elif kind == "history":
        case = _history("", _spread(rng, 1, 64), _spread(rng, 200, GPT2_VOCAB),
                        _spread(rng, 1, 3000), rng.choice([0, _spread(rng, 1, 900)]))
    elif kind == "logprobs":
        vocab = rng.choice([GPT2_VOCAB, _spread(rng, 200, 131072)])
        case = _logprobs("", _spread(rng, 1, min(2048, LARGEST_SCORED // vocab)), vocab,
                         rng.choice([0, 1, 5, 20, rng.randint(1, 32)]))
        if case["rows"] > 512:
            case["top"] = min(case["top"], 5)
    else:
        job = rng.choice(["fork", "resize"])
        case = _pages("", job, rng.randint(1, 24), rng.choice([1, 2]), rng.randint(1, 16),
                      rng.choice([16, 20, 32, 64, 80, 128]), 0, 0,
                      page=rng.choice([16, 32]), dtype=rng.choice(["bfloat16", "float32"]))
        most = max(1, LARGEST_COPY // (_page_elems(case) * _itemsize(case)))
        case["pairs"] = _spread(rng, 1, min(most, 64 if job == "fork" else 2500))
        case["pages"] = 2 * case["pairs"] + rng.randint(1, 50)
    del case["name"]
    return case


def _itemsize(case):
    return 4 if case["dtype"] == "float32" else 2


def _page_elems(case):
    return case["entries"] * case["planes"] * case["heads"] * case["page"] * case["dim"]


def work(case):
    if case["kind"] == "rules":
        rows, vocab = case["rows"], case["vocab"]
        per_row = 8 * vocab + 12 * case["bias"]
        if case["penalties"]:
            per_row += vocab // 4 + 4 * case["generated"]
        if case["grammar"]:
            per_row += vocab // 8
        return {"bytes": rows * per_row, "flops": 0}
    if case["kind"] == "history":
        per_slot = 4 * case["vocab"] + case["vocab"] // 4
        return {"bytes": case["slots"] * (per_slot + 4 * (case["prompt"] + case["generated"]) + 16),
                "flops": 0}
    if case["kind"] == "logprobs":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 12 + 8 * case["top"]),
                "flops": 4 * case["rows"] * case["vocab"]}
    share = _filled_share(case)
    return {"bytes": int(2 * case["pairs"] * _page_elems(case) * _itemsize(case) * share),
            "flops": 0}


def _filled_share(case):
    return 0.5 if case["job"] == "fork" else 1.0


# -- inputs ---------------------------------------------------------------------------------


def _words(vocab):
    return -(-vocab // 32)


def _pack(bits):
    """[rows, vocab] truth values as [rows, words] int32: bit v % 32 of word v // 32."""
    rows, vocab = bits.shape
    full = torch.zeros(rows, _words(vocab) * 32, dtype=torch.bool, device=bits.device)
    full[:, :vocab] = bits
    weight = (1 << torch.arange(32, device=bits.device, dtype=torch.int64))
    words = (full.view(rows, -1, 32) * weight).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _unpack(words, vocab):
    shift = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words.unsqueeze(-1) >> shift) & 1).flatten(1)[:, :vocab] != 0


def _text(gen, n, vocab):
    """n token ids, a few of them often, most seldom."""
    u = torch.rand(n, generator=gen, device=DEV)
    return (u ** 3 * vocab).long().clamp_(0, vocab - 1).to(torch.int32)


def _ragged(gen, n, mean):
    """n lengths between half and one and a half times the mean."""
    u = torch.rand(n, generator=gen, device=DEV)
    return ((0.5 + u) * mean).round().long().tolist()


def _text_of(case, gen, slots):
    """Tokens of the slots behind one another, where each begins, how many are of its prompt."""
    prompt = [max(1, n) for n in _ragged(gen, slots, case["prompt"])]
    generated = _ragged(gen, slots, case["generated"])
    ends = torch.tensor([p + g for p, g in zip(prompt, generated)]).cumsum(0).tolist()
    return _text(gen, ends[-1], case["vocab"]), [0] + ends, prompt


def _logits(gen, rows, vocab):
    x = torch.randn(rows, vocab, generator=gen, device=DEV) * 2.5
    ids = torch.randint(0, vocab, (rows, 4), generator=gen, device=DEV)
    lift = torch.randn(rows, 4, generator=gen, device=DEV) * 4.0
    return x.scatter_(1, ids, x.gather(1, ids) + lift)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)        # noqa: E731
    if case["kind"] == "rules":
        rows, vocab = case["rows"], case["vocab"]
        tokens, start, n_prompt = _text_of(case, gen, rows)
        counts = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV)
        prompt = torch.zeros(rows, vocab, dtype=torch.bool, device=DEV)
        owner = torch.repeat_interleave(
            torch.arange(rows, device=DEV),
            torch.tensor([b - a for a, b in zip(start, start[1:])], device=DEV))
        place = torch.arange(start[-1], device=DEV) - torch.tensor(start, device=DEV)[owner]
        is_prompt = place < torch.tensor(n_prompt, device=DEV)[owner]
        ids = tokens.long()
        prompt[owner[is_prompt], ids[is_prompt]] = True
        counts.index_put_((owner[~is_prompt], ids[~is_prompt]),
                          torch.ones((), dtype=torch.int32, device=DEV), accumulate=True)
        slots = torch.randperm(rows, generator=gen, device=DEV).to(torch.int32)
        s = dict(logits=_logits(gen, rows, vocab), prompt=_pack(prompt),
                 output=_pack(counts > 0), counts=counts,
                 slots=slots if case["penalties"] else torch.full_like(slots, -1),
                 repetition=1.0 + 0.5 * torch.rand(rows, generator=gen, device=DEV),
                 presence=torch.rand(rows, generator=gen, device=DEV),
                 frequency=0.5 * torch.rand(rows, generator=gen, device=DEV),
                 out=torch.empty(rows, vocab, device=DEV))
        if case["bias"]:
            n = case["bias"]
            # distinct ids of a row: a random offset into steps through the vocabulary
            step = vocab // n
            first = torch.randint(0, vocab, (rows, 1), generator=gen, device=DEV)
            ids = (first + step * torch.arange(n, device=DEV)) % vocab
            s["bias_start"] = ints([i * n for i in range(rows + 1)])
            s["bias_ids"] = ids.flatten().to(torch.int32)
            s["bias_values"] = torch.randn(rows * n, generator=gen, device=DEV) * 5.0
        if case["grammar"]:
            s["mask"] = _pack(torch.rand(rows, vocab, generator=gen, device=DEV) > MASKED)
            s["mask_row"] = torch.randperm(rows, generator=gen, device=DEV).to(torch.int32)
        return s
    if case["kind"] == "history":
        n, vocab = case["slots"], case["vocab"]
        tokens, start, n_prompt = _text_of(case, gen, n)
        zeros = lambda w: torch.zeros(n, w, dtype=torch.int32, device=DEV)     # noqa: E731
        return dict(tokens=tokens, start=ints(start), n_prompt=ints(n_prompt),
                    slots=torch.randperm(n, generator=gen, device=DEV).to(torch.int32),
                    sampled=_text(gen, n, vocab), prompt=zeros(_words(vocab)),
                    output=zeros(_words(vocab)), counts=zeros(vocab))
    if case["kind"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        logits = _logits(gen, rows, vocab)
        # most tokens are likely ones, as sampled ones are; some are any
        tokens = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.7,
                             logits.argmax(1),
                             torch.randint(0, vocab, (rows,), generator=gen, device=DEV))
        return dict(logits=logits, tokens=tokens.to(torch.int32),
                    logprob=torch.empty(rows, device=DEV),
                    rank=torch.empty(rows, dtype=torch.int32, device=DEV),
                    top_ids=torch.empty(rows, top, dtype=torch.int32, device=DEV) if top else None,
                    top_logprobs=torch.empty(rows, top, device=DEV) if top else None)
    dtype = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    shape = (case["planes"], case["heads"], case["page"], case["dim"])
    src = torch.empty(case["entries"], case["pages"], *shape, dtype=dtype, device=DEV)
    src.normal_(generator=gen)
    pairs = case["pairs"]
    order = torch.randperm(case["pages"], generator=gen, device=DEV).tolist()
    if case["job"] == "fork":
        # some requests' last pages, several copies of each; half a page is filled on average
        parents = max(1, pairs // 7)
        rows = torch.randint(1, case["page"], (parents,), generator=gen, device=DEV).tolist()
        return dict(src=src, dst=src, src_pages=[order[i % parents] for i in range(pairs)],
                    dst_pages=order[parents:parents + pairs],
                    rows=[rows[i % parents] for i in range(pairs)])
    dst = torch.zeros(case["entries"], pairs + pairs // 5 + 1, *shape, dtype=dtype, device=DEV)
    return dict(src=src, dst=dst, src_pages=order[:pairs], dst_pages=list(range(pairs)), rows=None)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        from hetero_serve_b200.kernels.ops import CudaOps, TokenHistory
        state["ops"] = CudaOps()
        if "counts" in state:
            state["history"] = TokenHistory(state["prompt"], state["output"], state["counts"])
    return state


# -- one pass ---------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _run_own(s, case):
    ops = s["ops"]
    if case["kind"] == "rules":
        ops.logit_rules(s["out"], s["logits"], s["history"], s["slots"], s["repetition"],
                        s["presence"], s["frequency"], bias_start=s.get("bias_start"),
                        bias_ids=s.get("bias_ids"), bias_values=s.get("bias_values"),
                        mask=s.get("mask"), mask_row=s.get("mask_row"))
        return s["out"]
    if case["kind"] == "history":
        ops.history_begin(s["history"], s["slots"], s["tokens"], s["start"], s["n_prompt"])
        ops.history_add(s["history"], s["slots"], s["sampled"])
        return [s["prompt"], s["output"], s["counts"]]
    if case["kind"] == "logprobs":
        ops.token_logprobs(s["logprob"], s["rank"], s["logits"], s["tokens"],
                           top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
        return [s["logprob"], s["rank"]] + ([s["top_ids"], s["top_logprobs"]] if case["top"] else [])
    ops.copy_pages(s["dst"], s["src"], s["dst_pages"], s["src_pages"], s["rows"])
    return s["dst"]


def _run_plain(s, case):
    if case["kind"] == "rules":
        return _plain_rules(s, case)
    if case["kind"] == "history":
        return _plain_history(s, case["vocab"])
    if case["kind"] == "logprobs":
        return _plain_logprobs(s, case["top"])
    return _plain_pages(s)


def _plain_rules(s, case):
    x, vocab = s["logits"], case["vocab"]
    if case["penalties"]:
        slots = s["slots"].long()
        output = _unpack(s["output"][slots], vocab)
        seen = _unpack(s["prompt"][slots], vocab) | output
        r = s["repetition"].unsqueeze(1)
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        c = torch.where(output, s["counts"][slots], 0).float()
        x = x - (s["frequency"].unsqueeze(1) * c + s["presence"].unsqueeze(1) * output.float())
    if "bias_ids" in s:
        n = s["bias_start"].diff().long()
        row = torch.repeat_interleave(torch.arange(len(n), device=x.device), n,
                                      output_size=s["bias_ids"].shape[0])
        x = x.index_put((row, s["bias_ids"].long()), s["bias_values"], accumulate=True)
    if "mask" in s:
        allowed = _unpack(s["mask"][s["mask_row"].long()], vocab)
        x = torch.where(allowed, x, -math.inf)
    return x


def _plain_history(s, vocab):
    slots, start = s["slots"].long(), s["start"].long()
    n = start.diff()
    owner = torch.repeat_interleave(torch.arange(len(n), device=n.device), n,
                                    output_size=s["tokens"].shape[0])
    place = torch.arange(len(owner), device=n.device) - start[owner]
    is_prompt = (place < s["n_prompt"][owner]).to(torch.int32)
    ids = s["tokens"].long()
    prompt = torch.zeros_like(s["counts"])
    prompt.index_put_((slots[owner], ids), is_prompt, accumulate=True)
    counts = s["counts"]
    counts.zero_()
    counts.index_put_((slots[owner], ids), 1 - is_prompt, accumulate=True)
    counts.index_put_((slots, s["sampled"].long()), torch.ones_like(s["sampled"]), accumulate=True)
    s["prompt"].copy_(_pack(prompt > 0))
    s["output"].copy_(_pack(counts > 0))
    return [s["prompt"], s["output"], counts]


def _plain_logprobs(s, top):
    x, t = s["logits"], s["tokens"].long().unsqueeze(1)
    m = x.amax(1, keepdim=True)
    log_sum = torch.log(torch.exp(x - m).sum(1, keepdim=True))
    mine = x.gather(1, t)
    index = torch.arange(x.shape[1], device=x.device)
    before = (x > mine) | ((x == mine) & (index < t))
    out = [((mine - m) - log_sum).squeeze(1), before.sum(1).to(torch.int32)]
    if top:
        # the order of the bits of a float is that of its value once negative ones are flipped;
        # below them the index, so that equal logits come in the order of their indices
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits >= 0, bits, -2147483648 - bits - 1) * 2 ** 32 + (2 ** 31 - index)
        best = key.topk(top, dim=1).indices
        out += [best.to(torch.int32), (x.gather(1, best) - m) - log_sum]
    return out


def _plain_pages(s):
    dst, src = s["dst"], s["src"]
    d = torch.tensor(s["dst_pages"], device=dst.device)
    taken = src[:, torch.tensor(s["src_pages"], device=dst.device)]
    if s["rows"] is not None:
        rows = torch.tensor(s["rows"], device=dst.device)
        filled = torch.arange(src.shape[-2], device=dst.device) < rows[:, None]
        taken = torch.where(filled[None, :, None, None, :, None], taken, dst[:, d])
    dst[:, d] = taken
    return dst


# -- the definitions in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "pages":
        return None                  # copies, not computed
    s = _inputs(case, seed)
    if case["kind"] == "rules":
        return _exact_rules(s, case)
    if case["kind"] == "history":
        return _exact_history(s, case)
    out = torch.empty(case["rows"], dtype=torch.float64, device=DEV)
    top = torch.empty(case["rows"], case["top"], dtype=torch.float64, device=DEV)
    for r in range(case["rows"]):
        row = s["logits"][r].double()
        log_total = torch.logsumexp(row, 0)
        out[r] = row[s["tokens"][r].long()] - log_total
        if case["top"]:
            top[r] = row.sort(descending=True).values[:case["top"]] - log_total
    return [out, None] + ([None, top] if case["top"] else [])


def _exact_history(s, case):
    """Request by request, on the host: whole numbers."""
    vocab = case["vocab"]
    prompt, output, counts = ([None] * case["slots"] for _ in range(3))
    tokens, start, first = s["tokens"].cpu(), s["start"].tolist(), s["n_prompt"].tolist()
    for k, slot in enumerate(s["slots"].tolist()):
        text = tokens[start[k]:start[k + 1]].long()
        said = torch.cat([text[first[k]:], s["sampled"][k:k + 1].cpu().long()])
        counts[slot] = torch.bincount(said, minlength=vocab)
        for words, ids in ((prompt, text[:first[k]]), (output, said)):
            flags = torch.bincount(ids, minlength=_words(vocab) * 32).clamp(max=1).view(-1, 32)
            value = sum(flags[:, i] << i for i in range(31))
            words[slot] = value - (flags[:, 31] << 31)
    return [torch.stack(x).to(DEV) for x in (prompt, output, counts)]


def _exact_rules(s, case):
    """Row by row: the tokens that stand in the record, one after another, then the others."""
    out = s["logits"].double()
    vocab = case["vocab"]
    bit = torch.arange(vocab, device=DEV)

    def has(words):
        return (words.long()[bit // 32] >> (bit % 32)) % 2 == 1

    for r in range(case["rows"]):
        row = out[r]
        slot = int(s["slots"][r])
        if slot >= 0:
            said = torch.nonzero(has(s["output"][slot])).flatten()
            known = torch.nonzero(has(s["prompt"][slot]) | has(s["output"][slot])).flatten()
            by = s["repetition"][r].double()
            v = row[known]
            row[known] = torch.clamp(v, min=0) / by + torch.clamp(v, max=0) * by
            row[said] -= s["frequency"][r].double() * s["counts"][slot][said].double()
            row[said] -= s["presence"][r].double()
        if "bias_ids" in s:
            a, b = int(s["bias_start"][r]), int(s["bias_start"][r + 1])
            row[s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        if "mask" in s:
            row[~has(s["mask"][int(s["mask_row"][r])])] = -math.inf
    return out
