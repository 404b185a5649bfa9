"""Continuous-batching inference engine.

Scheduler (one `step()` = one decode batch plus prefill chunks):
  * running sequences each get one decode token per step (up to
    max_num_seqs); a sequence whose next token needs a new KV block takes one,
    and if none is free the most recently admitted running sequence is
    preempted (its blocks freed, it returns to the head of the queue and is
    recomputed later);
  * waiting requests are admitted in (priority, arrival) order while the
    step's token budget (max_num_batched_tokens) and free KV blocks allow;
    long prompts are split into chunks (chunked prefill) so one huge prompt
    does not stall the decode batch;
  * prompt blocks already in the prefix cache are not recomputed;
  * a request for n samples becomes n requests when its prompt is computed: the
    others fork its block table (full blocks shared, the partial one copied on the
    device) and sample their first token from the same logits;
  * penalties, biases and grammar masks change the logits of the requests that
    have any before sampling; each such request holds a row of the runner's
    table of token counts while it runs.

Reference: ContinuousBatching (include/nn/inference.hpp:89-170, FIFO admit to
max_batch), DynamicBatcher / PriorityScheduler
(include/api/serving_production.hpp:24-106) and SpeculativeDecoding's greedy
sampling (include/nn/inference.hpp:13-86).
"""
from __future__ import annotations

import itertools
import time
from collections import deque
from dataclasses import dataclass, field, replace
from typing import Callable, Dict, List, Optional, Sequence

import numpy as np
import torch

from ..config import ServeConfig, TransformerConfig
from ..models.params import FlatParams
from ..ops import serving as SV
from .kv_cache import BlockManager
from .model_runner import ModelRunner, PrefillItem


@dataclass
class SamplingParams:
    max_tokens: int = 16
    temperature: float = 0.0
    top_p: float = 1.0
    stop_token_ids: tuple = ()
    # token sequences that end generation when the output ends with one (the
    # server's OpenAI `stop` strings, tokenized); the server leaves them out of the text
    stop_sequences: tuple = ()
    seed: Optional[int] = None
    # logits before sampling (ops/logits.py): z / r or z * r for tokens of the prompt or
    # output, - frequency * count - presence for generated ones, + bias per token id,
    # and -inf for all but the allowed tokens: a fixed set, or a grammar called with
    # the tokens generated so far (it returns the ids allowed next, None = all; none at
    # all ends the request with reason "stop" and without a token; an exception or an id
    # outside the vocabulary ends it with reason "error", Request.error says why)
    repetition_penalty: float = 1.0
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    logit_bias: Optional[Dict[int, float]] = None
    allowed_token_ids: Optional[Sequence[int]] = None
    grammar: Optional[Callable[[List[int]], Optional[Sequence[int]]]] = None
    n: int = 1  # samples of the prompt; the request's own is the first (Request.samples: the others' ids)

    @property
    def penalised(self) -> bool:
        return self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0 or self.presence_penalty != 0.0

    @property
    def adjusts(self) -> bool:
        return self.penalised or bool(self.logit_bias) or self.allowed_token_ids is not None or self.grammar is not None

    @property
    def banned(self) -> List[int]:
        """Tokens with a bias of -inf."""
        return [t for t, b in (self.logit_bias or {}).items() if b < -3.4028235e38]

    def allowed(self, output: List[int]) -> Optional[Sequence[int]]:
        """The token ids that may come next (None = all)."""
        ids = self.grammar(output) if self.grammar is not None else None
        if ids is None or self.allowed_token_ids is None:
            return self.allowed_token_ids if ids is None else ids
        fixed = set(self.allowed_token_ids)
        return [t for t in ids if t in fixed]


def _token_ids(ids, vocab: int) -> np.ndarray:
    """Token ids (any iterable of integers, a set among them) as int64 [n]; ValueError where one
    is no id of the vocabulary."""
    a = np.asarray(ids if isinstance(ids, (list, tuple, np.ndarray)) else list(ids))
    if a.size and not (a.ndim == 1 and a.dtype.kind in "iu" and a.min() >= 0 and a.max() < vocab):
        raise ValueError(f"token ids must be integers in [0, {vocab})")
    return a.astype(np.int64, copy=False).reshape(-1)


def _mix64(a: int, b: int) -> int:
    """splitmix64 finaliser of a + golden-ratio * (b + 1): a 64-bit seed per (stream, index)."""
    z = (int(a) + 0x9E3779B97F4A7C15 * (int(b) + 1)) & 0xFFFFFFFFFFFFFFFF
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & 0xFFFFFFFFFFFFFFFF
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & 0xFFFFFFFFFFFFFFFF
    return z ^ (z >> 31)


def _ends_with_any(out: List[int], seqs) -> bool:
    for sq in seqs:
        n = len(sq)
        if n and len(out) >= n and tuple(out[-n:]) == tuple(sq):
            return True
    return False


@dataclass
class Request:
    req_id: int
    prompt: List[int]
    params: SamplingParams
    priority: int = 0
    arrival: float = 0.0
    output: List[int] = field(default_factory=list)
    table: List[int] = field(default_factory=list)
    computed: int = 0           # tokens whose K/V are in the cache
    prefill_len: int = 0        # tokens to prefill before decoding (all but a pending last token)
    cached_prefix: int = 0
    first_token_time: Optional[float] = None
    scheduled_time: Optional[float] = None  # first admission to the running set (queue time ends)
    token_times: List[float] = field(default_factory=list)
    finished: bool = False
    finish_reason: Optional[str] = None
    error: Optional[str] = None  # what went wrong (finish_reason "error")
    on_token: Optional[Callable[["Request", int], None]] = None
    on_finish: Optional[Callable[["Request"], None]] = None  # called once, however the request ends
    samples: List[int] = field(default_factory=list)  # ids of the other samples (params.n > 1)
    forks: int = 0              # continuations made of this request, its samples among them
    counts_row: int = -1        # row of the runner's token counts
    # params.allowed_token_ids (without a grammar) and logit_bias as the runner packs them, once
    fixed_mask: Optional[object] = None
    fixed_bias: Optional[object] = None

    @property
    def tokens(self) -> List[int]:
        return self.prompt + self.output

    # O(1) forms of len(tokens) and tokens[-1] for the per-step paths
    @property
    def n_tokens(self) -> int:
        return len(self.prompt) + len(self.output)

    @property
    def last_token(self) -> int:
        return self.output[-1] if self.output else self.prompt[-1]

    @property
    def in_prefill(self) -> bool:
        return self.computed < self.prefill_len


class LLMEngine:
    def __init__(self, cfg: TransformerConfig, params: FlatParams, serve: Optional[ServeConfig] = None, *,
                 device="cuda", kv_dtype: str = "fp8", weights: str = "none", group_size: int = 128,
                 clock: Callable[[], float] = time.perf_counter, runner=None):
        """runner: an already built runner (e.g. the tensor-parallel
        serve.tp_runner.RunnerProxy on rank 0); params is then unused."""
        self.cfg = cfg
        self.sc = serve or ServeConfig()
        self.runner = runner if runner is not None else ModelRunner(
            cfg, params, device, kv_dtype=kv_dtype, weights=weights, group_size=group_size,
            num_blocks=self.sc.num_kv_blocks, block_size=self.sc.block_size,
            max_model_len=self.sc.max_model_len)
        if self.sc.cuda_graphs and hasattr(self.runner, "enable_graphs"):
            self.runner.enable_graphs(self.sc.max_num_seqs)
        self.blocks = BlockManager(self.runner.num_blocks, self.sc.block_size,
                                   self.sc.enable_prefix_caching)
        self.waiting: deque = deque()
        self.running: List[Request] = []
        self.ids = itertools.count()
        self.clock = clock
        self.finished: Dict[int, Request] = {}
        self.stats = {"prompt_tokens": 0, "generated_tokens": 0, "preemptions": 0, "steps": 0,
                      "prefill_tokens_computed": 0}
        self._seed = 1234
        self._counts_free: List[int] = []  # unused rows of the runner's token counts
        self._counts_rows = 0
        # when a list: one (schedule_s, prefill_s, decode_s, prefill_tokens,
        # decode_seqs) record per step, host clock; the prefill and decode
        # phases each end with the device read of their sampled tokens
        self.step_log: Optional[list] = None

    # ---------------------------------------------------------- requests
    def add_request(self, prompt: List[int], params: Optional[SamplingParams] = None, priority: int = 0,
                    on_token=None, arrival: Optional[float] = None, on_finish=None) -> int:
        """Queue a prompt; returns the request's id.  on_token(request, token) is called for each token,
        on_finish(request) once when the request has ended, which it can do without another token (an abort,
        a grammar that allows none).  Its further samples (params.n > 1) call both too."""
        if not prompt:
            raise ValueError("empty prompt")
        if len(prompt) + (params.max_tokens if params else 16) > self.sc.max_model_len:
            raise ValueError("prompt + max_tokens exceeds max_model_len")
        if params is not None:
            self._check_params(params)
        r = Request(next(self.ids), list(prompt), params or SamplingParams(), priority,
                    self.clock() if arrival is None else arrival, on_token=on_token, on_finish=on_finish)
        self.stats["prompt_tokens"] += len(prompt)
        # priority first (lower value = sooner), FIFO within a priority: every
        # request, priority 0 included, goes in front of the first waiting
        # request with a larger priority value
        idx = next((k for k, w in enumerate(self.waiting) if w.priority > priority), len(self.waiting))
        self.waiting.insert(idx, r)
        return r.req_id

    def _check_params(self, p: SamplingParams) -> None:
        if p.temperature > 0 and not getattr(self.runner, "supports_top_p", False):
            if p.top_p < 1.0:
                raise ValueError("top_p < 1 is not supported by this runner (tensor-parallel serving samples "
                                 "from vocabulary slices); use top_p = 1")
            if p.seed is not None:
                raise ValueError("per-request seeds are not supported by this runner (tensor-parallel serving)")
        if p.adjusts and not getattr(self.runner, "supports_adjust", False):
            raise ValueError("penalties, biases and grammars are not supported by this runner (tensor-parallel serving "
                             "samples from vocabulary slices)")
        # the kernel's numbers are fp32, and it multiplies by the reciprocal of the repetition penalty
        most = float(np.finfo(np.float32).max)
        if not (2.0 ** -126 <= p.repetition_penalty <= 2.0 ** 126 and abs(p.frequency_penalty) <= most and abs(p.presence_penalty) <= most):
            raise ValueError("penalties must be finite in fp32, repetition_penalty in [2^-126, 2^126]")
        if not all(b <= most for b in (p.logit_bias or {}).values()):  # -inf bans a token
            raise ValueError("logit_bias: values must be finite in fp32, or -inf")
        V = self.cfg.vocab_size
        if any(not 0 <= t < V for t in p.logit_bias or ()):
            raise ValueError(f"logit_bias and allowed_token_ids take token ids in [0, {V})")
        if p.allowed_token_ids is not None:
            if not len(p.allowed_token_ids):
                raise ValueError("allowed_token_ids must not be empty")
            ids = _token_ids(p.allowed_token_ids, V)
            if p.banned and set(ids.tolist()) <= set(p.banned):
                raise ValueError("logit_bias bans every token of allowed_token_ids")
        if not 1 <= p.n <= self.sc.max_num_seqs:
            raise ValueError(f"n must be in [1, {self.sc.max_num_seqs}]")

    def abort_request(self, req_id: int) -> bool:
        """Drop a request that has not finished (its client went away): its KV
        blocks are freed and it leaves the waiting / running queues.  Returns
        False when the request is unknown or already finished."""
        for r in list(self.running):
            if r.req_id == req_id:
                self._release(r)
                self.running.remove(r)
                self._finish(r, "abort")
                return True
        for r in list(self.waiting):
            if r.req_id == req_id:
                if r.table:
                    self.blocks.free_seq(r.table)
                self.waiting.remove(r)
                self._finish(r, "abort")
                return True
        return False

    def _finish(self, r: Request, reason: Optional[str]) -> None:
        r.finished, r.finish_reason = True, reason
        self.finished[r.req_id] = r
        if r.on_finish:
            r.on_finish(r)

    # ------------------------------------------------------------ forks, pages
    def fork_request(self, req_id: int, params: Optional[SamplingParams] = None, on_token=None, on_finish=None) -> int:
        """Continue a running request a second time from where it is now: a new
        request with the same tokens so far, whose KV blocks are shared with the
        first's (the partly filled one copied).  params: the new one's (default:
        the same with another seed; its max_tokens counts the tokens so far too)."""
        r = next((x for x in self.running if x.req_id == req_id), None)
        if r is None or r.in_prefill or not r.output:
            raise ValueError("fork_request: the request is not running, or has no token yet")
        if params is not None:
            if params.n != 1:
                raise ValueError("fork_request: n must be 1")
            if len(r.prompt) + params.max_tokens > self.sc.max_model_len:
                raise ValueError("prompt + max_tokens exceeds max_model_len")
            if params.max_tokens <= len(r.output):
                raise ValueError(f"fork_request: max_tokens counts the {len(r.output)} tokens generated so far")
            self._check_params(params)
        return self._fork(r, r.n_tokens - 1, params, on_token, on_finish).req_id

    def _fork(self, r: Request, computed: int, params: Optional[SamplingParams], on_token, on_finish) -> Request:
        """A copy of r whose first `computed` tokens are in the cache; it runs at once
        where there is room, else it waits and is recomputed (from the prefix cache)."""
        rid = next(self.ids)
        r.forks += 1
        if params is None:
            # another seed for each, the same ones whenever the request is made again
            seed = None if r.params.seed is None else _mix64(r.params.seed, r.forks) >> 1
            params = replace(r.params, n=1, seed=seed)
        # a sample of the prompt arrived with it; a fork midway arrives now, and its latencies are
        # those of its own tokens (the tokens so far have no time in it)
        c = Request(rid, list(r.prompt), params, r.priority, self.clock() if r.output else r.arrival, output=list(r.output),
                    cached_prefix=computed, on_token=on_token, on_finish=on_finish)
        if hasattr(self.runner, "copy_pages") and len(self.running) < self.sc.max_num_seqs:
            try:
                c.table, copies = self.blocks.fork(r.table, computed)
            except MemoryError:
                pass
            else:
                self.runner.copy_pages(copies)
                c.prefill_len = c.computed = computed
                c.scheduled_time = c.arrival if r.output else r.scheduled_time
                self.running.append(c)
                return c
        # ahead of its own priority's requests (its prompt is in the prefix cache), behind lower values
        idx = next((k for k, w in enumerate(self.waiting) if w.priority >= c.priority), len(self.waiting))
        self.waiting.insert(idx, c)
        return c

    def compact(self) -> int:
        """Move the KV blocks in use to the lowest block ids (between steps);
        returns how many moved."""
        if not hasattr(self.runner, "copy_pages"):
            raise ValueError("compact is not supported by this runner")
        moves = self.blocks.compact([r.table for r in self.running] + [r.table for r in self.waiting])
        self.runner.copy_pages(moves)
        return len(moves)

    def _release(self, r: Request) -> None:
        """What a request holds while it runs: its KV blocks and its counts row."""
        self.blocks.free_seq(r.table)
        if r.counts_row >= 0:
            self._counts_free.append(r.counts_row)
            r.counts_row = -1

    def has_work(self) -> bool:
        return bool(self.waiting or self.running)

    # ---------------------------------------------------------- scheduling
    def _preempt(self, r: Request) -> None:
        """Free a running request's blocks; it is recomputed when readmitted
        (prompt and generated tokens, except the last one, which decode feeds)."""
        self._release(r)
        r.computed = 0
        self.running.remove(r)
        self.waiting.appendleft(r)
        self.stats["preemptions"] += 1

    def _schedule(self):
        decode: List[Request] = []
        preempted = set()  # request ids preempted during this pass
        for r in list(self.running):
            if r.in_prefill or r.req_id in preempted:
                continue
            while True:
                try:
                    self.blocks.append_slot(r.table, r.n_tokens - 1)
                    break
                except MemoryError:
                    victims = [x for x in self.running if x is not r]
                    if not victims:
                        raise
                    preempted.add(victims[-1].req_id)
                    self._preempt(victims[-1])
            decode.append(r)
        if preempted:
            decode = [r for r in decode if r.req_id not in preempted]
        budget = max(self.sc.max_num_batched_tokens - len(decode), 1)
        prefill: List[Request] = [r for r in self.running if r.in_prefill]
        admitted_tokens = sum(r.prefill_len - r.computed for r in prefill)
        while (self.waiting and len(self.running) < self.sc.max_num_seqs
               and admitted_tokens < budget):
            r = self.waiting[0]
            seq = r.tokens if not r.output else r.tokens[:-1]
            try:
                r.table, cached = self.blocks.allocate(seq)
            except MemoryError:
                break
            self.waiting.popleft()
            if r.scheduled_time is None:
                r.scheduled_time = self.clock()
            r.prefill_len = len(seq)
            r.computed = cached
            r.cached_prefix = cached
            self.running.append(r)
            prefill.append(r)
            admitted_tokens += r.prefill_len - cached
        items = []
        for r in prefill:
            if budget <= 0:
                break
            n = min(r.prefill_len - r.computed, budget)
            chunk = r.tokens[r.computed:r.computed + n]
            slots = self.blocks.slots_for(r.table, 0, r.computed + n)
            last = r.computed + n == r.prefill_len
            items.append((r, PrefillItem(r.req_id, chunk, r.computed, slots, last and not r.output)))
            budget -= n
        return decode, items

    # ---------------------------------------------------------------- step
    def _emit(self, r: Request, tok: Optional[int], now: float) -> None:
        if tok is None:  # its grammar allows no token, or failed
            self._release(r)
            self.running.remove(r)
            self._finish(r, "stop" if r.error is None else "error")
            return
        r.output.append(tok)
        r.token_times.append(now)
        if r.first_token_time is None:
            r.first_token_time = now
        self.stats["generated_tokens"] += 1
        if tok in r.params.stop_token_ids or _ends_with_any(r.output, r.params.stop_sequences):
            r.finished, r.finish_reason = True, "stop"
        elif len(r.output) >= r.params.max_tokens:
            r.finished, r.finish_reason = True, "length"
        if r.on_token:
            r.on_token(r, tok)
        if r.finished:
            self._release(r)
            self.running.remove(r)
            self._finish(r, r.finish_reason)

    def _adjust(self, reqs: List[Request], logits: torch.Tensor, allowed: List) -> torch.Tensor:
        """Penalties, biases and masks of the requests that have any; a request new to
        the counts table (or back in it) gets its row written from its tokens."""
        if not any(r.params.adjusts for r in reqs):
            return logits
        fresh = [r for r in reqs if r.params.penalised and r.counts_row < 0]
        for r in fresh:
            if not self._counts_free:  # one row per running request is enough
                self._counts_free += range(self._counts_rows, self._counts_rows + self.sc.max_num_seqs)
                self._counts_rows += self.sc.max_num_seqs
            r.counts_row = self._counts_free.pop()
        if fresh:
            self.runner.set_counts([r.counts_row for r in fresh], [(r.prompt, r.output) for r in fresh], self._counts_rows)
        ps = [r.params for r in reqs]
        return self.runner.adjust_logits(
            logits, [r.counts_row if r.params.penalised else -1 for r in reqs],
            [(p.repetition_penalty, p.frequency_penalty, p.presence_penalty) for p in ps],
            [self._packed_bias(r) for r in reqs], [self._packed_mask(r, a) for r, a in zip(reqs, allowed)])

    def _packed_mask(self, r: Request, allowed):
        if allowed is None:
            return None
        pack = getattr(self.runner, "pack_allowed", None) or np.ndarray.tolist
        if r.params.grammar is not None:
            return pack(allowed)
        if r.fixed_mask is None:
            r.fixed_mask = pack(_token_ids(allowed, self.cfg.vocab_size))
        return r.fixed_mask

    def _packed_bias(self, r: Request):
        pack = getattr(self.runner, "pack_bias", None)
        if not r.params.logit_bias or pack is None:
            return r.params.logit_bias
        if r.fixed_bias is None:
            r.fixed_bias = pack(r.params.logit_bias)
        return r.fixed_bias

    def _allowed(self, r: Request) -> Optional[Sequence[int]]:
        """The token ids that may come next (None = all; an array where a grammar names them).  A grammar is the caller's code: where it
        fails, its request alone ends (_emit), without a token."""
        if r.params.grammar is None:
            return r.params.allowed_token_ids
        try:
            ids = r.params.allowed(r.output)
            if ids is None:
                return None
            ids = _token_ids(ids, self.cfg.vocab_size)
            banned = r.params.banned
            return ids[~np.isin(ids, banned)] if banned else ids  # banned ones are no choice: none left ends the request
        except Exception as e:
            r.error = f"grammar: {type(e).__name__}: {e}"
            return _token_ids((), 0)

    def _sample(self, reqs: List[Request], logits: torch.Tensor) -> List[Optional[int]]:
        allowed = [self._allowed(r) for r in reqs]
        tok = self._draw(reqs, self._adjust(reqs, logits, allowed))
        if any(r.counts_row >= 0 for r in reqs):
            self.runner.add_counts([r.counts_row for r in reqs], tok)
        return [t if a is None or len(a) else None for t, a in zip(tok.tolist(), allowed)]

    def _draw(self, reqs: List[Request], logits: torch.Tensor) -> torch.Tensor:
        temps = [r.params.temperature for r in reqs]
        if all(t <= 0 for t in temps):
            return self.runner.sample(logits, None, 0)
        else:
            self._seed += 1
            kw = {}
            top_ps = [r.params.top_p for r in reqs]
            if any(p < 1.0 for p, t in zip(top_ps, temps) if t > 0):
                kw["top_ps"] = top_ps
            if any(r.params.seed is not None for r, t in zip(reqs, temps) if t > 0):
                # a seeded request's draw k uses (its seed, k), whatever its batch row
                kw["row_seeds"] = [_mix64(r.params.seed, len(r.output)) if r.params.seed is not None
                                   else _mix64(self._seed, i) for i, r in enumerate(reqs)]
            return self.runner.sample(logits, temps, self._seed, **kw)

    def step(self) -> List[Request]:
        """Run one scheduling step; returns requests that finished during it."""
        t0 = self.clock() if self.step_log is not None else 0.0
        decode, items = self._schedule()
        self.stats["steps"] += 1
        done_before = set(self.finished)
        t1 = self.clock() if self.step_log is not None else 0.0
        n_pre = sum(len(it.tokens) for _, it in items)
        if items:
            seq_ids, logits = self.runner.prefill([it for _, it in items])
            for r, it in items:
                r.computed += len(it.tokens)
                self.stats["prefill_tokens_computed"] += len(it.tokens)
                if not r.in_prefill:
                    self.blocks.register_full_blocks(r.tokens, r.table, r.prefill_len)
            if seq_ids:
                by_id = {r.req_id: r for r, _ in items}
                reqs = [by_id[i] for i in seq_ids]
                if any(r.params.n > 1 for r in reqs):
                    reqs, logits = self._spread(reqs, logits)
                toks = self._sample(reqs, logits)
                now = self.clock()
                for r, t in zip(reqs, toks):
                    self._emit(r, t, now)
        t2 = self.clock() if self.step_log is not None else 0.0
        if decode:
            live = {x.req_id for x in self.running}
            decode = [r for r in decode if not r.finished and r.req_id in live]
        if decode:
            toks_in = [r.last_token for r in decode]
            pos = [r.n_tokens - 1 for r in decode]
            bs = self.blocks.block_size
            slots = [r.table[p // bs] * bs + p % bs for r, p in zip(decode, pos)]
            logits = self.runner.decode(toks_in, pos, slots, [r.table for r in decode])
            toks = self._sample(decode, logits)
            now = self.clock()
            for r, t in zip(decode, toks):
                self._emit(r, t, now)
        if self.step_log is not None:
            t3 = self.clock()
            self.step_log.append((t1 - t0, t2 - t1, t3 - t2, n_pre, len(decode)))
        return [self.finished[i] for i in self.finished if i not in done_before]

    def _spread(self, reqs: List[Request], logits: torch.Tensor):
        """Prompts just computed whose requests want several samples: the others are
        forked and take the same row of logits (those that have to wait for room
        are left to their own turn)."""
        out, rows = [], []
        for k, r in enumerate(reqs):
            out.append(r)
            rows.append(k)
            if r.params.n > 1 and not r.samples:
                for _ in range(r.params.n - 1):
                    c = self._fork(r, r.prefill_len, None, r.on_token, r.on_finish)
                    r.samples.append(c.req_id)
                    if c.table:
                        out.append(c)
                        rows.append(k)
        return out, logits.index_select(0, torch.tensor(rows, device=logits.device))

    def generate(self, prompts: List[List[int]], params: Optional[SamplingParams] = None) -> List:
        """The outputs of the prompts; with params.n > 1, the list of its samples for each prompt."""
        ids = [self.add_request(p, params) for p in prompts]
        while any(i not in self.finished or any(j not in self.finished for j in self.finished[i].samples) for i in ids):
            self.step()
        if params is not None and params.n > 1:
            return [[self.finished[j].output for j in [i] + self.finished[i].samples] for i in ids]
        return [self.finished[i].output for i in ids]
