"""Sampling.  Token selection runs on the device inside the step (``ops.sample``:
argmax, temperature, top-k; ``csrc/sampling.cu``).  This module holds the host-side
statement of the same rule, used to document and cross-check it, and what a request may ask for
before the draw (``rules.py``: penalties, biases, grammars).
"""

from .rule import philox4x32_10, uniform_for_position
from .rules import LogitRules, OneOf, is_whole, mask_words

__all__ = ["LogitRules", "OneOf", "is_whole", "mask_words", "philox4x32_10", "uniform_for_position"]
