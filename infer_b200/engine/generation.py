"""The engine as the scheduler sees it (step function + sampler), and the Python entry point ``LLM``.

Option names follow the reference where it has them: ``slots``, ``max_seq``, ``budget_mb``
(src/main_serve_bench.cpp:15-27; kernels/batch_gpu.h:38-40), ``max_new``, ``temperature``, ``seed``, ``eos_id``
(src/scheduler.h:36-87), ``top_k`` / ``top_p`` (src/sampler.h:16-25).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Dict, Hashable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..sampling.sampler import Sampler
from .. import ops
from .engine import Engine, OutOfPages, StepEntry
from .scheduler import (BatchEngine, BatchItem, Completed, Request, SampleParams, Scheduler, SchedulerConfig, TokenScore)


class PendingTokens:
    """Sampled token ids on their way to the host."""

    def __init__(self, rids, host, event, asked=None, scores=None):
        self.rids, self._host, self._event = rids, host, event
        self._asked, self._scores = asked, scores       # per row the alternatives that were asked for (None: no score); ops.TokenLogprobs on the host

    def result(self) -> Dict[Hashable, int]:
        if self._event is None:
            return {}
        self._event.synchronize()
        return {rid: int(t) for rid, t in zip(self.rids, self._host.tolist())}

    @property
    def scores(self) -> Dict[Hashable, TokenScore]:
        """How likely each token was, for the requests that asked."""
        if self._scores is None:
            return {}
        self._event.synchronize()
        logprob, entropy, ids, best = (t.tolist() for t in self._scores)
        return {rid: TokenScore(logprob[i], entropy[i], [(t, p) for t, p in zip(ids[i][:int(n)], best[i][:int(n)]) if t >= 0])
                for i, (rid, n) in enumerate(zip(self.rids, self._asked)) if n is not None}


class GenerationEngine(BatchEngine):
    """Runs a planned batch as ONE step and samples on the device; only token ids cross to the host."""

    def __init__(self, engine: Engine):
        self.engine = engine
        self.sampler = Sampler(engine.rt.device)       # for callers that sample from logits themselves
        self.max_seq_len = engine.max_seq_len
        self.max_requests = engine.cache.n_slots
        self._pinned, self._flip = {}, 0

    def capacity_tokens(self) -> int:
        return min(self.engine.cache.pages_total()) * self.engine.cache.page_size if self.engine.cache.groups else 1 << 60

    def add_request(self, rid) -> None:
        self.engine.add_request(rid)

    def end_request(self, rid) -> None:
        self.engine.end_request(rid)

    def can_run(self, wanted) -> bool:
        return self.engine.cache.can_reserve(list(wanted))

    def has_room(self, prompt_len: int) -> bool:
        need = -(-prompt_len // self.engine.cache.page_size) + 1
        return all(f >= need for f in self.engine.cache.pages_free())

    def tokens_that_fit(self, wanted, rid, n: int) -> int:
        cache = self.engine.cache
        lo, hi = 0, n
        while lo < hi:                                  # largest m <= n with can_reserve(wanted + (rid, m))
            mid = (lo + hi + 1) // 2
            if cache.can_reserve(list(wanted) + [(rid, mid)]):
                lo = mid
            else:
                hi = mid - 1
        return lo

    def run_async(self, batch: Sequence[BatchItem]) -> "PendingTokens":
        """Enqueues the step, the sampling and the copy of the sampled ids to pinned host memory, and returns at
        once. Every sampled token also stays on the device (engine.next_tokens[slot]); a later decode item may pass
        FEEDBACK_TOKEN instead of the id."""
        entries = [StepEntry(b.rid, b.tokens, [len(b.tokens) - 1] if b.sample is not None else []) for b in batch]
        rows = [b for b in batch if b.sample is not None]
        # the sampling kernel's inputs travel in the step's one packed buffer and the kernel runs inside the step
        # (inside its CUDA graph when the shape is captured): one copy in, one launch, one copy out per step
        if any(b.sample.logprobs is not None for b in rows):
            return self._run_scored(entries, rows)
        ids = self.engine.step(entries, sample=[(b.sample, b.position) for b in rows])
        if not rows:
            return PendingTokens([], None, None)
        # Pinned buffers for the ids take turns (four per batch size): a buffer comes round again only after the
        # result of the step that used it last has been read, which waits on that step's event.
        self._flip = (self._flip + 1) % 4
        key = (len(rows), self._flip)
        slot = self._pinned.get(key)
        if slot is None:
            slot = self._pinned[key] = (torch.empty(len(rows), dtype=torch.int32).pin_memory(), torch.cuda.Event())
        host, event = slot
        event.synchronize()                     # the copy that wrote this buffer last has landed (no-op if never used)
        host.copy_(ids, non_blocking=True)
        event.record()
        return PendingTokens([b.rid for b in rows], host, event)

    def _run_scored(self, entries, rows: Sequence[BatchItem]) -> "PendingTokens":
        """As ``run_async`` where a request wants to know how likely its tokens are: the step leaves its logits, and the sampler and the log
        probabilities read them behind it (the same sampler on the same logits: the same tokens)."""
        asked = [b.sample.logprobs for b in rows]
        slots = [self.engine.cache.slot(b.rid) for b in rows]
        logits = self.engine.step(entries)
        with torch.cuda.device(self.engine.rt.device):
            ids = self.sampler.sample(logits, [b.sample for b in rows], [b.position for b in rows], self.engine.next_tokens, slots)
            scores = ops.token_logprobs(logits, ids, max(int(n) for n in asked if n is not None))
            copies = []
            for t in (ids, *scores):
                host = torch.empty(t.shape, dtype=t.dtype, pin_memory=True)
                host.copy_(t, non_blocking=True)
                copies.append(host)
            event = torch.cuda.Event()
            event.record()
        return PendingTokens([b.rid for b in rows], copies[0], event, asked, ops.TokenLogprobs(*copies[1:]))

    def run(self, batch: Sequence[BatchItem]) -> Dict[Hashable, int]:
        return self.run_async(batch).result()

    def pages_in_use(self) -> int:
        return max(self.engine.cache.pages_in_use(), default=0)

    def pages_total(self) -> int:
        return max(self.engine.cache.pages_total(), default=0)


@dataclass
class PromptScore:
    """Place i is behind the prompt's id i: ``logprobs[i]`` is the log probability of id i + 1 there, ``entropies[i]`` the entropy (nats) of the
    distribution, ``top_ids[i]`` and ``top_logprobs[i]`` the likeliest tokens (id -1 where there is none)."""
    logprobs: np.ndarray
    entropies: np.ndarray
    top_ids: np.ndarray
    top_logprobs: np.ndarray

    @property
    def perplexity(self) -> float:
        """exp of the mean negative log probability (1 for a prompt of one id)."""
        return float(np.exp(-np.mean(self.logprobs, dtype=np.float64))) if len(self.logprobs) else 1.0


class LLM:
    """Python entry point: a model folder in, token ids out.

        llm = LLM("/path/to/model", dtype="bfloat16", slots=8, max_seq=4096)
        outs = llm.generate([[1, 2, 3], [4, 5]], max_new=16)                    # greedy
        outs = llm.generate(prompts, max_new=16, temperature=0.8, seed=7)      # seeded sampling
        (ids, scores), = llm.generate([[1, 2, 3]], max_new=16, logprobs=5)      # how likely each token was, with five alternatives
        score, = llm.score([[1, 2, 3, 4]], top=5)                               # the same of given tokens
    """

    def __init__(self, model: str, dtype="bfloat16", device: str = "cuda:0", slots: int = 8, max_seq: int = 4096,
                 budget_mb: int = 0, max_batch_tokens: int = 512, page_size: int = 16, eos_id: Optional[int] = None,
                 kernels: Optional[Dict[str, str]] = None, weights=None, spec=None, overlap: bool = True,
                 kv_blocks: int = 0):
        """slots: live requests; max_seq: per-sequence cap; budget_mb: size of the page pool in MiB, or kv_blocks: its
        size in pages (both 0 = reserve slots x max_seq, as the reference does, kernels/batch_gpu.cu:92-95);
        max_batch_tokens: the token budget of a step, which is also the largest prompt portion. ``spec`` + ``weights``
        may replace the folder."""
        from ..config.registry import load_config
        from ..weights.binder import load_weights
        if spec is None:
            arch, typed = load_config(model)
            spec = arch.to_spec(typed)
            weights = load_weights(model, spec)
        self.engine = Engine(spec, weights, dtype=dtype, device=device,
                             max_tokens=int(kv_blocks) * page_size if kv_blocks else slots * max_seq,
                             max_requests=slots, page_size=page_size, max_seq_len=max_seq, kernels=kernels,
                             cache_budget_bytes=int(budget_mb) << 20)
        self.batch_engine = GenerationEngine(self.engine)
        default_eos = eos_id if eos_id is not None else (spec.eos_token_id if spec.eos_token_id is not None else -1)
        self.scheduler_config = SchedulerConfig(eos_id=default_eos, max_batch_tokens=max_batch_tokens, overlap=overlap)
        self._next_id = 0

    def new_scheduler(self, **overrides) -> Scheduler:
        cfg = SchedulerConfig(**{**self.scheduler_config.__dict__, **overrides})
        return Scheduler(self.batch_engine, cfg)

    def generate(self, prompts: Sequence[Sequence[int]], max_new: int = 16, temperature: float = 0.0, seed: int = 0,
                 top_k: int = 0, top_p: float = 1.0, eos_id: Optional[int] = None,
                 on_token: Optional[Callable[[Hashable, int], None]] = None, logprobs: Optional[int] = None):
        """Generates up to max_new tokens for every prompt (lists of token ids); returns the new ids per prompt
        (eos included if hit). With ``logprobs`` = n (0 to 20) it returns (ids, scores) per prompt instead: a ``TokenScore`` for each id, of the
        model's own distribution (before temperature and filters), with the n likeliest tokens."""
        if logprobs is not None and not 0 <= int(logprobs) <= 20:
            raise ValueError(f"logprobs takes 0 to 20 alternatives, not {logprobs}")
        sch = self.new_scheduler(on_token=on_token)
        ids = []
        for p in prompts:
            rid = self._next_id
            self._next_id += 1
            ids.append(rid)
            sch.submit(Request(rid, [int(t) for t in p], max_new, 0,
                               SampleParams(temperature, seed, top_k, top_p, None if logprobs is None else int(logprobs)), eos_id))
        sch.run_until_idle()
        done = {c.id: c for c in sch.completed}
        self.last_scheduler = sch
        return [done[i].tokens if logprobs is None else (done[i].tokens, done[i].scores) for i in ids]

    def score(self, prompts: Sequence[Sequence[int]], top: int = 0) -> List["PromptScore"]:
        """How likely the model finds given token ids: for each prompt of n ids a ``PromptScore`` of n - 1 places. Prompts run in portions under the
        token budget, several in a step; the logits are not stored (of a 32-bit model a portion's are for the moment)."""
        prompts = [[int(t) for t in p] for p in prompts]
        V = self.engine.spec.vocab_size
        for i, p in enumerate(prompts):
            if not p:
                raise ValueError(f"prompt {i} is empty")
            if len(p) - 1 > self.engine.max_seq_len:
                raise ValueError(f"prompt {i}: {len(p) - 1} positions exceed the limit of {self.engine.max_seq_len}")
            if min(p) < 0 or max(p) >= V:
                raise ValueError(f"prompt {i}: a token id is outside the vocabulary [0, {V})")
        if not 0 <= int(top) <= 20:
            raise ValueError(f"0 to 20 alternatives can be asked for, not {top}")
        eng, budget = self.engine, self.scheduler_config.max_batch_tokens
        waiting = [i for i, p in enumerate(prompts) if len(p) > 1]
        fed: Dict[int, int] = {}                          # prompts in work -> ids in the cache
        names = {}
        parts: List[list] = [[] for _ in prompts]         # per prompt (step's result, first row, rows)
        try:
            while waiting or fed:
                # a prompt starts when all that is left of those in work and all of it have pages
                while waiting and len(eng.cache.requests) < eng.cache.n_slots:
                    i = waiting[0]
                    names[i] = ("score", self._next_id)
                    eng.add_request(names[i])
                    left = [(names[j], len(prompts[j]) - 1 - n) for j, n in fed.items()]
                    if not eng.cache.can_reserve(left + [(names[i], len(prompts[i]) - 1)]):
                        eng.end_request(names.pop(i))
                        break
                    self._next_id += 1
                    fed[i] = 0
                    waiting.pop(0)
                if not fed:
                    raise OutOfPages(f"prompt {waiting[0]} ({len(prompts[waiting[0]])} tokens) does not fit the free pages and slots")
                entries, asked, room = [], [], budget
                for i, n in list(fed.items()):
                    m = min(len(prompts[i]) - 1 - n, room)
                    if m == 0:
                        break
                    entries.append((i, m))
                    asked += prompts[i][n + 1:n + 1 + m]
                    room -= m
                r = eng.step_logprobs([StepEntry(names[i], prompts[i][fed[i]:fed[i] + m], range(m)) for i, m in entries], asked, int(top))
                row = 0
                for i, m in entries:
                    parts[i].append((r, row, m))
                    row += m
                    fed[i] += m
                    if fed[i] == len(prompts[i]) - 1:
                        eng.end_request(names.pop(i))
                        del fed[i]
        finally:
            for name in names.values():
                eng.end_request(name)
        eng.check_status()
        host: Dict[int, tuple] = {}                       # a step's result is copied once
        out = []
        for got in parts:
            rows = []
            for r, row, m in got:
                if id(r) not in host:
                    host[id(r)] = tuple(t.cpu().numpy() for t in r)
                rows.append(tuple(a[row:row + m] for a in host[id(r)]))
            empty = (np.zeros(0, np.float32), np.zeros(0, np.float32), np.zeros((0, int(top)), np.int32), np.zeros((0, int(top)), np.float32))
            out.append(PromptScore(*(np.concatenate([x[k] for x in rows]) if rows else empty[k] for k in range(4))))
        return out
