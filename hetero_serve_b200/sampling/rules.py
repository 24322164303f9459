"""What a request may say: penalties for tokens it repeats, biases of single tokens, and
grammars that rule tokens out.

The arithmetic is :meth:`CudaOps.logit_rules`'s, in this order: a token seen in the prompt or
answer has its logit divided by ``repetition`` (multiplied where it is not positive); one
generated c > 0 times loses ``frequency * c + presence``; a biased token gains its bias; a token
that the grammar rules out becomes -inf.

A *grammar* is any object with ``allowed(output_ids)``: asked before every token with the tokens
generated so far, it says which may come next — ``None`` (any), a packed mask (an array of
``ceil(vocab / 32)`` 32-bit words, bit v % 32 of word v // 32), an array of truth values over the
vocabulary, or token ids (anything else that yields whole numbers; 32-bit arrays are masks).  An
answer that allows nothing ends the request (``finish_reason == "grammar"``), and so does a grammar
that raises or answers with anything else (``"grammar_error"``; the record's ``error`` says what).
"""

from __future__ import annotations

import math
import operator
from dataclasses import dataclass, field
from typing import Mapping, Sequence

import numpy as np


# The largest number a rule may hold.  Steps hold them in 32 bits: up to here a finite logit stays
# finite under any of them, and so does its quotient by a temperature (1e8 * 1e20 + 1e7 * 1e20, for
# the largest logits and counts there are, is ten decades below the largest number of 32 bits).
LARGEST = 1e20


def is_whole(n) -> bool:
    """Whether ``n`` is a whole number (a truth value is none)."""
    return isinstance(n, (int, np.integer)) and not isinstance(n, bool)


@dataclass(frozen=True, eq=False)
class LogitRules:
    """The numbers of a request's rules; ValueError for numbers no request can mean (beyond
    ``LARGEST``; a finite bias below ``-LARGEST`` counts as that)."""

    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Mapping[int, float] = field(default_factory=dict)
    # the biases as arrays, as a step packs them
    bias_ids: np.ndarray = field(init=False, repr=False)
    bias_values: np.ndarray = field(init=False, repr=False)
    _ruled_words: np.ndarray | None = field(init=False, repr=False, default=None)

    def __post_init__(self):
        if not 1 / LARGEST <= self.repetition <= LARGEST:
            raise ValueError(f"repetition penalty {self.repetition}: between {1 / LARGEST} and "
                             f"{LARGEST}")
        for name in ("presence", "frequency"):
            if not abs(getattr(self, name)) <= LARGEST:
                raise ValueError(f"{name} penalty {getattr(self, name)}: at most {LARGEST} either way")
        for token, value in self.bias.items():
            if not is_whole(token) or not 0 <= token < 2 ** 31:
                raise ValueError(f"bias of {token!r}, which is no token id")
            if not value <= LARGEST:
                raise ValueError(f"bias {value} of token {token}: -inf, or a number up to {LARGEST}")
        values = (v if v == -math.inf else max(v, -LARGEST) for v in self.bias.values())
        for name, kind, of in (("bias_ids", np.int32, self.bias.keys()),
                               ("bias_values", np.float32, values)):
            object.__setattr__(self, name, np.fromiter(of, dtype=kind, count=len(self.bias)))

    @property
    def ruled_out(self) -> list[int]:
        """The tokens whose bias is -inf."""
        return self.bias_ids[np.isneginf(self.bias_values)].tolist()

    def leave(self, words: np.ndarray, vocab: int) -> np.ndarray:
        """A packed mask without the tokens whose bias is -inf."""
        out = self._ruled_words                    # packed once: steps ask for every row
        if out is None or len(out) != len(words):
            out = mask_words(self.ruled_out, vocab)
            object.__setattr__(self, "_ruled_words", out)
        return words & ~out

    @property
    def penalises(self) -> bool:
        """Whether the record of the request's tokens is needed."""
        return self.repetition != 1.0 or self.presence != 0.0 or self.frequency != 0.0

    @property
    def neutral(self) -> bool:
        return not self.penalises and not len(self.bias_ids)

    def check(self, vocab: int | None = None) -> None:
        """ValueError for a bias of a token the vocabulary does not have, and for biases that rule
        all of it out."""
        if vocab is None or not len(self.bias_ids):
            return
        if int(self.bias_ids.max()) >= vocab:
            raise ValueError(f"bias of token {int(self.bias_ids.max())}: the vocabulary has {vocab}")
        if len(self.bias_ids) >= vocab and len(self.ruled_out) >= vocab:
            raise ValueError("the biases leave no token")


def _token(t) -> int:
    if isinstance(t, (bool, np.bool_)) or str(getattr(t, "dtype", "")) == "torch.bool":
        raise ValueError("truth values outside an array: which tokens are meant?")
    return operator.index(t)              # (a fraction, or text, is no token id either)


def mask_words(allowed, vocab: int) -> np.ndarray | None:
    """What a grammar's ``allowed`` answered as packed int32 words (None: any token)."""
    if allowed is None:
        return None
    words = -(-vocab // 32)
    if isinstance(allowed, np.ndarray) and allowed.dtype != bool and allowed.ndim == 1 \
            and allowed.dtype.itemsize == 4 and allowed.dtype.kind in "iu":
        if allowed.shape[0] != words:
            raise ValueError(f"a mask of {allowed.shape[0]} words for {vocab} tokens ({words} words)")
        out = allowed.astype(np.uint32, copy=True)
        if vocab % 32:
            out[-1] &= np.uint32((1 << (vocab % 32)) - 1)
        return out.view(np.int32)
    flags = np.zeros(words * 32, dtype=bool)
    if isinstance(allowed, np.ndarray) and allowed.dtype == bool:
        if allowed.shape != (vocab,):
            raise ValueError(f"truth values of shape {allowed.shape} for {vocab} tokens")
        flags[:vocab] = allowed
    else:
        if isinstance(allowed, np.ndarray) and allowed.ndim == 1 and allowed.dtype.kind in "iu":
            ids = allowed.astype(np.int64)
        else:
            ids = np.fromiter((_token(t) for t in allowed), dtype=np.int64)
        if ids.size and (ids.min() < 0 or ids.max() >= vocab):
            raise ValueError(f"a grammar allows a token outside [0, {vocab})")
        flags[ids] = True
    return np.packbits(flags, bitorder="little").view(np.int32)


class OneOf:
    """The grammar of a choice: the answer is one of the given token sequences, and then
    ``end`` (the end-of-sequence token, say) if one is given."""

    def __init__(self, sequences: Sequence[Sequence[int]], end: int | None = None):
        if not sequences or any(len(s) == 0 for s in sequences):
            raise ValueError("a choice needs sequences, none of them empty")
        self._root: dict = {}
        self._end = end
        for s in sequences:
            node = self._root
            for t in s:
                node = node.setdefault(int(t), {})
            node[None] = True                      # a sequence ends here

    def allowed(self, output_ids: Sequence[int]) -> list[int]:
        node = self._root
        for t in output_ids:
            if t not in node:
                return []
            node = node[t]
        ids = [t for t in node if t is not None]
        if None in node and self._end is not None:
            ids.append(self._end)
        return ids
