"""An oracle for what requests may ask of their answers: greedy decoding over the plain model's
logits with penalties, biases and a grammar written as plain dictionary code, and scores."""

from __future__ import annotations

import math
import random
from collections import Counter

import torch


def ruled(row, prompt, output, *, repetition_penalty=1.0, presence_penalty=0.0,
          frequency_penalty=0.0, logit_bias=None, grammar=None):
    row = row.double().clone()
    said = Counter(output)
    for t in set(prompt) | set(output):
        row[t] = row[t] / repetition_penalty if row[t] > 0 else row[t] * repetition_penalty
    for t, c in said.items():
        row[t] -= frequency_penalty * c + presence_penalty
    for t, b in (logit_bias or {}).items():
        row[t] += b
    if grammar is not None:
        allowed = grammar.allowed(tuple(output))
        if allowed is not None:
            keep = torch.full_like(row, -math.inf)
            keep[list(allowed)] = row[list(allowed)]
            row = keep
    return row


def greedy(logits_of, prompt, n, **rules):
    """Tokens, and for each the gap to the next best (how close the call was)."""
    out, gaps = [], []
    while len(out) < n:
        row = ruled(logits_of(prompt + out)[-1], prompt, out, **rules)
        if bool((row == -math.inf).all()):
            break
        best = torch.topk(row, 2).values
        gaps.append(float(best[0] - best[1]))
        out.append(int(row.argmax()))
    return out, gaps


class Alternating:
    """A grammar that looks at what was said: even and odd token ids in turn, in every form a
    grammar may answer in, and any token in every fourth place."""

    def __init__(self, vocab):
        self.vocab = vocab

    def ids(self, output):
        n = len(output)
        if n % 4 == 3:
            return None
        first = 0 if not output else 1 - output[-1] % 2
        return range(first, self.vocab, 2)

    def allowed(self, output):
        import numpy as np
        from hetero_serve_b200.sampling import mask_words
        ids = self.ids(output)
        if ids is None or len(output) % 4 == 0:
            return ids
        flags = np.zeros(self.vocab, dtype=bool)
        flags[list(ids)] = True
        return flags if len(output) % 4 == 1 else mask_words(flags, self.vocab)


class Plain:
    """The same grammar for the oracle: ids."""

    def __init__(self, grammar):
        self.grammar = grammar

    def allowed(self, output):
        return self.grammar.ids(output)


# -- many requests of every kind, submitted while others run, over a cache that changes its size -----

ENGINES = (dict(num_blocks=40, max_batch=8, max_prefill_tokens=64, pipeline=False),
           dict(num_blocks=40, max_batch=8, max_prefill_tokens=24, policy="mixed"),
           dict(num_blocks=10, max_batch=4, max_prefill_tokens=16, policy="mixed", prefix_cache=False),
           dict(num_blocks=10, max_batch=3, max_prefill_tokens=16))


def any_requests(rng, vocab):
    from hetero_serve_b200 import OneOf
    out = []
    for i in range(rng.randint(2, 6)):
        r = dict(prompt_ids=[rng.randrange(vocab) for _ in range(rng.choice([1, 2, 15, 16, 17, 30]))],
                 max_new_tokens=rng.randint(1, 16), temperature=rng.choice([0, 0.8]),
                 seed=rng.randrange(1000), top_k=rng.choice([0, 5]), stop_at_eos=False, req_id=f"q{i}")
        if rng.random() < 0.5:
            r.update(repetition_penalty=1.3, frequency_penalty=0.2, presence_penalty=0.1)
        if rng.random() < 0.3:
            r.update(logit_bias={rng.randrange(vocab): rng.choice([-math.inf, 2.0]) for _ in range(5)})
        if rng.random() < 0.3:
            r.update(grammar=rng.choice([Alternating(vocab), OneOf([[1, 2, 3], [1, 5], [7]])]))
        if rng.random() < 0.4:
            r.update(logprobs=rng.choice([0, 2, 9]))
        if rng.random() < 0.4:
            r.update(samples=rng.randint(2, 4))
        out.append(r)
    return out


def run_through(eng, requests, rng):
    """Every answer with its alternatives and its end, and its scores; the cache is resized and text
    scored meanwhile."""
    from hetero_serve_b200 import Request
    from hetero_serve_b200.cache import OutOfPages
    vocab, seqs, todo = eng.model.spec.vocab_size, [], list(requests)
    while todo or eng.has_work():
        if todo and (rng.random() < 0.4 or not eng.has_work()):
            seqs.append(eng.submit_nowait(Request(**todo.pop(0))))
        try:
            if rng.random() < 0.05:
                eng.resize_cache(rng.randint(10, 40))
            if rng.random() < 0.04:
                eng.score([rng.randrange(vocab) for _ in range(rng.randint(2, 40))], rng.choice([0, 3]))
        except OutOfPages:
            pass
        eng.step()
        eng.runner.manager.check()
    assert eng.runner.manager.free_slots() == eng.config.live_requests
    answers = [s for q in seqs for s in (q, *q.siblings)]
    return ([(s.output_ids, [[t for t, _ in x.top] for x in s.scores], s.finish_reason) for s in answers],
            torch.tensor([x.logprob for s in answers for x in s.scores]))
