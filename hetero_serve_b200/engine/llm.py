"""The Python entry point: a model folder in, generated token ids out.

    engine = LLMEngine("path/to/model", dtype="bfloat16", num_blocks=512)
    record = engine.submit(Request(prompt_ids=[...], max_new_tokens=32))
    outputs = engine.generate([[...], [...]], max_new_tokens=16, temperature=0.8, seed=1)
    answers = engine.submit_samples(Request(prompt_ids=[...], samples=8, temperature=0.8, logprobs=0))
    scores = engine.score([...], alternatives=5)

``Request`` and ``RequestRecord`` carry the reference's names
(heteroserve/sched/router.py:36-44, heteroserve/metrics.py:31-68); ``submit`` is the
reference's ``Router.submit(Request) -> RequestRecord`` (router.py:404-406) without the
processes and sockets in between.  ``submit_nowait`` / ``step`` / ``has_work`` expose the
continuous-batching loop for callers that feed requests while others run.
"""

from __future__ import annotations

import tempfile
import itertools
from dataclasses import replace
from pathlib import Path
from typing import Sequence

import torch

from ..cache import OutOfPages
from ..config import EngineConfig, preset
from ..kernels.ops import MAX_ALTERNATIVES
from ..sampling import is_whole
from ..weights import write_model_dir
from .loading import TORCH_DTYPES, load_model
from .metrics import RequestRecord, summarise
from .scheduler import Request, Scheduler, SequenceState
from .step import Runner, StepEntry, StepError, TokenLogprobs

_scored = itertools.count()


class LLMEngine:
    def __init__(self, model_dir: str | Path, config: EngineConfig | None = None, *, ops=None,
                 **overrides):
        cfg = config or EngineConfig()
        if overrides:
            cfg = replace(cfg, **overrides)
        self.config = cfg
        self.model, self.model_config = load_model(model_dir, cfg.dtype, cfg.device)
        spec = self.model.spec
        self.runner = Runner(
            self.model, num_pages=cfg.num_blocks, page_size=cfg.block_size,
            max_requests=cfg.live_requests, dtype=TORCH_DTYPES[cfg.dtype], device=cfg.device,
            ops=ops, prefix_cache=cfg.prefix_cache, cuda_graphs=cfg.cuda_graphs,
            fused_decode=cfg.fused_decode)
        limit = self.runner.max_positions
        max_ctx = min(cfg.max_ctx or limit, limit)
        self.scheduler = Scheduler(
            self.runner.manager, self._run_step, max_batch=cfg.max_batch,
            max_prefill_tokens=cfg.max_prefill_tokens, max_ctx=max_ctx,
            eos_token_id=spec.eos_token_id, policy=cfg.policy, vocab_size=spec.vocab_size,
            pipeline=cfg.pipeline, fork_fn=self.runner.fork)
        self._tmp = None

    # -- construction --------------------------------------------------------------
    @classmethod
    def from_dir(cls, model_dir, **kw) -> "LLMEngine":
        return cls(model_dir, **kw)

    @classmethod
    def random(cls, model: str | dict, seed: int = 0, *, store_dtype: str | None = None,
               **kw) -> "LLMEngine":
        """Random-weights mode: write a model folder for a preset name or a config.json
        dictionary (``model``) and a seed into a temporary folder, then load it like any other;
        ``config=EngineConfig(...)`` or single engine options go through as for the constructor."""
        raw = preset(model) if isinstance(model, str) else dict(model)
        tmp = tempfile.TemporaryDirectory(prefix="hetero_serve_b200-")
        dtype = kw.get("dtype", (kw.get("config") or EngineConfig()).dtype)
        write_model_dir(tmp.name, raw, seed, store_dtype or ("bfloat16" if str(dtype).startswith("b") else "float32"))
        eng = cls(tmp.name, **kw)
        eng._tmp = tmp
        return eng

    # -- the loop -------------------------------------------------------------------
    def _run_step(self, entries: list[StepEntry]):
        """Launch a step with device sampling.  The copy of its tokens to the host is enqueued
        behind it; the scheduler asks for them (``tokens_host``) when it needs them — with
        ``pipeline``, after it has launched the following step."""
        res = self.runner.step(entries, sample=True)
        res.start_fetch()
        return res

    def submit_nowait(self, request: Request) -> SequenceState:
        return self.scheduler.add(request)

    def has_work(self) -> bool:
        return self.scheduler.has_work()

    def step(self) -> list[RequestRecord]:
        """One scheduler iteration; returns the records of requests whose end became known in
        it (with ``pipeline`` that is one call after the step that produced their last token)."""
        return [RequestRecord.of(s) for s in self.scheduler.step()]

    def run_until_done(self) -> list[RequestRecord]:
        out: list[RequestRecord] = []
        while self.scheduler.has_work():
            out.extend(self.step())
        return out

    def submit(self, request: Request) -> RequestRecord:
        """Run until this request has finished (others in flight advance too; of several samples
        this is the first: see :meth:`submit_samples`)."""
        seq = self.submit_nowait(request)
        while seq.state != "done":
            self.step()
        return RequestRecord.of(seq)

    def submit_samples(self, request: Request) -> list[RequestRecord]:
        """Run until every answer to this request's prompt has finished (``request.samples`` of
        them, in the order of their seeds; others in flight advance too)."""
        seq = self.submit_nowait(request)
        answers = [seq, *seq.siblings]
        while any(s.state != "done" for s in answers):
            self.step()
        return [RequestRecord.of(s) for s in answers]

    def score(self, token_ids: Sequence[int], alternatives: int = 0) -> list[TokenLogprobs]:
        """Score given text: the log-probability and rank of every token but the first behind the
        ones before it, with the likeliest ``alternatives`` at its place.  Runs beside live
        requests, in portions of the engine's token budget, and needs a state slot and pages for
        the text meanwhile (:class:`OutOfPages` otherwise).  Text with a token outside the
        vocabulary, or longer than the model, is refused (:class:`StepError`)."""
        runner, text = self.runner, [int(t) for t in token_ids]
        vocab = self.model.spec.vocab_size
        most = min(MAX_ALTERNATIVES, vocab)
        if not (is_whole(alternatives) and 0 <= alternatives <= most):
            raise ValueError(f"{alternatives} alternatives: between 0 and {most}")
        # Steps take FROM_DEVICE in a portion's first place, and never see the last token.
        bad = [t for t in text if not 0 <= t < vocab]
        if bad:
            raise StepError(f"token id {bad[0]} is outside [0, {vocab})")
        if len(text) - 1 > runner.max_positions:
            raise StepError(f"{len(text)} tokens to score: the model has "
                            f"{runner.max_positions} positions, and the last token needs none")
        name, out = ("score", next(_scored)), []
        with runner._on_device():
            runner.open(name)
            try:
                for at in range(0, len(text) - 1, self.config.max_prefill_tokens):
                    part = text[at:min(at + self.config.max_prefill_tokens, len(text) - 1)]
                    res = runner.step([StepEntry(name, part, want=range(len(part)))])
                    out += self._scores(res.logits, text[at + 1:at + 1 + len(part)], alternatives)
            finally:
                runner.close(name)
        return out

    def _scores(self, logits, tokens, alternatives) -> list[TokenLogprobs]:
        n, dev = len(tokens), logits.device
        given = torch.tensor(tokens, dtype=torch.int32, device=dev)
        logprob = torch.empty(n, device=dev)
        rank = torch.empty(n, dtype=torch.int32, device=dev)
        ids = torch.empty(n, alternatives, dtype=torch.int32, device=dev)
        lps = torch.empty(n, alternatives, device=dev)
        self.runner.ops.token_logprobs(logprob, rank, logits, given,
                                       *((ids, lps) if alternatives else ()))
        self.runner.check_status()
        return [TokenLogprobs(lp, r, list(zip(i, p))) for lp, r, i, p in
                zip(logprob.tolist(), rank.tolist(), ids.tolist(), lps.tolist())]

    def resize_cache(self, num_blocks: int) -> None:
        """Make the cache smaller or larger while requests live: their pages move to the lowest
        numbers of pools of the new size, published prefixes as far as they fit.  Raises
        :class:`OutOfPages`, with nothing changed, where the live requests' pages do not fit, or a
        smaller pool would not hold a request that waits.  The longest request the engine takes
        stays what it was."""
        for pool, n, promised in zip(self.runner.manager.pools, self.runner.pool_sizes(num_blocks),
                                     self.scheduler.pages_promised()):
            if n < min(promised, pool.num_pages):
                raise OutOfPages(f"a waiting request needs {promised} pages: they do not fit {n}")
        self.runner.resize_cache(num_blocks)
        self.config = replace(self.config, num_blocks=num_blocks)

    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 32,
                 temperature: float = 0.0, top_k: int = 0, seed: int = 0,
                 stop_at_eos: bool = True, **options) -> list[list[int]]:
        """Generate for several prompts at once; returns the new token ids of each.  ``options``
        are further fields of :class:`Request` (penalties, ``logit_bias``; one answer a prompt)."""
        if options.get("samples", 1) != 1:
            raise ValueError("generate gives one answer a prompt: see submit_samples")
        seqs = [self.submit_nowait(Request(list(p), max_new_tokens, temperature, top_k,
                                           seed + i, stop_at_eos, **options))
                for i, p in enumerate(prompts)]
        self.run_until_done()
        return [list(s.output_ids) for s in seqs]

    def state_message(self) -> dict:
        msg = self.scheduler.state_message()
        msg["engine"] = f"hetero_serve_b200/{self.config.dtype}"
        msg["device"] = self.config.device
        return msg

    def summarise(self, records: list[RequestRecord], wall_s: float) -> dict:
        return summarise(records, wall_s)
