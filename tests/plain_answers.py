"""Plain twins (float64, loops) of the operations around a step's answers: rules on logits and the
record of tokens they go by, log-probabilities, copies of cache pages.  Signatures are those of
``CudaOps``; with them the engine runs on CPU tensors."""

from __future__ import annotations

import math

import torch

from plain_ops import PlainOps

WORD = 32


def set_bit(words, v):
    value = (int(words[v // WORD]) & 0xFFFFFFFF) | (1 << (v % WORD))
    words[v // WORD] = value - (1 << 32) if value >= 1 << 31 else value


def pack(flags):
    """[rows, vocab] truth values as int32 words, bit v % 32 of word v // 32."""
    rows, vocab = flags.shape
    out = torch.zeros(rows, -(-vocab // WORD), dtype=torch.int32)
    for r, v in torch.nonzero(flags.cpu()).tolist():
        set_bit(out[r], v)
    return out


def bits_set(words):
    """The indices of the set bits of one row of words."""
    return [WORD * i + b for i, word in enumerate(words.tolist()) if word
            for b in range(WORD) if (word >> b) & 1]


class PlainAnswerOps(PlainOps):
    def history_begin(self, history, slots, tokens, start, n_prompt):
        n, vocab = history.counts.shape
        for k in range(slots.shape[0]):
            slot = int(slots[k])
            if not 0 <= slot < n:
                continue
            for t in history.tensors():
                t[slot] = 0
            a, b = int(start[k]), int(start[k + 1])
            for i in range(a, b):
                v = int(tokens[i])
                if not 0 <= v < vocab:
                    continue
                if i < a + int(n_prompt[k]):
                    set_bit(history.prompt[slot], v)
                else:
                    set_bit(history.output[slot], v)
                    history.counts[slot, v] += 1

    def history_add(self, history, slots, tokens):
        n, vocab = history.counts.shape
        for k in range(slots.shape[0]):
            slot, v = int(slots[k]), int(tokens[k])
            if 0 <= slot < n and 0 <= v < vocab:
                set_bit(history.output[slot], v)
                history.counts[slot, v] += 1

    def logit_rules(self, out, logits, history=None, slots=None, repetition=None, presence=None,
                    frequency=None, *, bias_start=None, bias_ids=None, bias_values=None, mask=None,
                    mask_row=None):
        rows, vocab = logits.shape
        y = logits.double().clone()
        for w in range(rows):
            slot = -1 if history is None else int(slots[w])
            if history is not None and 0 <= slot < history.counts.shape[0]:
                said = set(bits_set(history.output[slot]))
                for v in said | set(bits_set(history.prompt[slot])):
                    if v >= vocab:
                        continue
                    r = float(repetition[w])
                    y[w, v] = y[w, v] / r if y[w, v] > 0 else y[w, v] * r
                    if v in said:
                        c = int(history.counts[slot, v])
                        y[w, v] -= float(frequency[w]) * c + (float(presence[w]) if c else 0.0)
            if bias_start is not None:
                listed = {}
                for j in range(int(bias_start[w]), int(bias_start[w + 1])):
                    listed[int(bias_ids[j])] = float(bias_values[j])
                for v, b in listed.items():
                    if 0 <= v < vocab:
                        y[w, v] += b
            if mask is not None and 0 <= int(mask_row[w]) < mask.shape[0]:
                kept = [v for v in bits_set(mask[int(mask_row[w])]) if v < vocab]
                ruled = torch.full((vocab,), -math.inf, dtype=torch.float64)
                ruled[kept] = y[w, kept]
                y[w] = ruled
        out.copy_(y.to(out.dtype))

    def token_logprobs(self, logprob, rank, logits, tokens, top_ids=None, top_logprobs=None):
        rows, vocab = logits.shape
        for w in range(rows):
            x = logits[w].double()
            empty = bool((x == -math.inf).all())
            m = x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).max()
            lp = x if empty else (x - m) - torch.log(torch.exp(x - m).sum())
            # larger first, equal ones by index, NaN behind everything
            index, nan = torch.arange(vocab), (x != x).cpu()
            real = index[~nan]
            by = torch.cat([real[torch.sort(x.cpu()[~nan], descending=True, stable=True).indices],
                            index[nan]]).tolist()
            t = int(tokens[w])
            if 0 <= t < vocab:
                logprob[w], rank[w] = lp[t].to(logprob.dtype), by.index(t)
            else:
                logprob[w], rank[w] = math.nan, -1
            if top_ids is not None:
                for n in range(top_ids.shape[1]):
                    top_ids[w, n] = by[n]
                    top_logprobs[w, n] = lp[by[n]].to(top_logprobs.dtype)

    def copy_pages(self, dst, src, dst_pages, src_pages, rows=None):
        for i, (d, s) in enumerate(zip(dst_pages, src_pages)):
            n = dst.shape[4] if rows is None else int(rows[i])
            dst[:, d, :, :, :n] = src[:, s, :, :, :n]
