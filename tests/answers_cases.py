"""An oracle for what requests may ask of their answers: greedy decoding over the plain model's
logits with penalties, biases and a grammar written as plain dictionary code, and scores."""

from __future__ import annotations

import math
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
