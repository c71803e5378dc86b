"""The generation loop over batches of requests.

Per sequence the order is that of MythEclipse/llm's loop
(apps/engine/src/generate.rs:78-127): prefill; then sample from the current
logits; a stop token ends the sequence without being emitted or fed; else emit,
stop if the context is full, and feed the token for the next logits. Here a
batch of requests with unequal prompts starts together (one prefill step),
every live sequence then advances by one token per step, sequences that end
leave the batch (their slot goes back to the cache) and the rest go on; when
the batch is empty the next batch starts. Stop reasons and the timing fields
are those of generate.rs:20-49,129-160. Who is live, who goes on and who leaves
for which reason is decided by the native host library
(`csrc/host/generation.cpp`); this module owns slots, steps, sampling, timing
and callbacks.

With `share_prefix`, neighbouring requests whose prompts begin alike begin together: what they
have in common is prefilled once and forked (equal prompts as a whole: several samples of one
prompt), and the steps read the shared pages once.
"""
from __future__ import annotations

import time
from array import array
from ctypes import byref, c_int, c_void_p
from dataclasses import dataclass, field

import torch

from .. import native
from ..cache import PAGE
from ..errors import ContextFull, FormatError
from ..sampling import BatchSampler, SamplingParams
from .step import Entry


@dataclass
class GenerationRequest:
    prompt: list
    max_tokens: int = 256
    params: SamplingParams = field(default_factory=SamplingParams)
    stop_tokens: tuple = ()


@dataclass
class GenerationResult:
    tokens: list
    stop_reason: str                 # 'eos', 'max_tokens', 'cancelled', 'context_full'
    prompt_tokens: int
    generated_tokens: int = 0
    prefill_ms: float = 0.0
    ttft_ms: float = 0.0
    decode_ms: float = 0.0
    total_ms: float = 0.0
    tokens_per_second: float = 0.0


def plan_batches(requests, fits, max_batch: int) -> list:
    """Cut the requests, in their order, into batches: a batch takes requests
    while it has fewer than `max_batch` and `fits(list of final lengths)` says
    the cache can hold them all to their end. A request that does not fit even
    alone is an error."""
    batches, current, lengths = [], [], []
    for index, final_length in requests:
        if current and (len(current) >= max_batch or not fits(lengths + [final_length])):
            batches.append(current)
            current, lengths = [], []
        if not fits([final_length]):
            raise ContextFull(final_length if isinstance(final_length, int) else final_length[0], 0)
        current.append(index)
        lengths.append(final_length)
    if current:
        batches.append(current)
    return batches


class _Prompts:
    """How the prompts of neighbouring requests begin alike. `twin[i]`: prompt i is the one before it. The others fall into runs
    of neighbours that start with the same `common` tokens, whole pages that leave each of them at least a token (0: a prompt alone)."""

    def __init__(self, prompts):
        self.twin = [i > 0 and prompts[i] == prompts[i - 1] for i in range(len(prompts))]
        alone = [i for i, t in enumerate(self.twin) if not t]
        try:
            tokens = array("i", [t for i in alone for t in prompts[i]])
        except (OverflowError, TypeError) as error:
            raise FormatError(f"token ids must be 32-bit integers ({error})") from None
        n = len(alone)
        first, common, runs = (c_int * (n + 1))(), (c_int * n)(), c_int()
        native.check(native.lib().llmh_prompt_runs(n, native.ints(len(prompts[i]) for i in alone),
                                                   (c_int * len(tokens)).from_buffer(tokens), PAGE, first, common, byref(runs)))
        self.run, self.common = [0] * len(prompts), [0] * len(prompts)
        for k in range(runs.value):
            for j in range(first[k], first[k + 1]):
                self.run[alone[j]], self.common[alone[j]] = k, common[k]
        for i, t in enumerate(self.twin):
            if t:
                self.run[i], self.common[i] = self.run[i - 1], self.common[i - 1]
        self.lengths = [len(p) for p in prompts]

    def shared(self, i: int) -> int:
        """Positions (whole pages) of request i's prompt that are pages of the request before it."""
        if self.twin[i]:
            return self.lengths[i] // PAGE * PAGE
        return self.common[i] if i > 0 and self.run[i] == self.run[i - 1] else 0


def _start(engine, reqs, batch, prompts, slots):
    """Prefill a batch: a slot a request is put into `slots`, and the logits of every prompt's last token are returned. `prompts`: what the
    prompts have in common (a _Prompts of all requests; `batch` are their indices), or None."""
    if prompts is None:
        slots += engine.acquire(len(reqs))
        return engine.step([Entry(slot, r.prompt, [len(r.prompt) - 1]) for slot, r in zip(slots, reqs)])
    alone = [b for b, i in enumerate(batch) if b == 0 or not prompts.twin[i]]
    runs = []                                            # of prompts that begin alike
    for b in alone:
        if runs and prompts.run[batch[b]] == prompts.run[batch[runs[-1][0]]]:
            runs[-1].append(b)
        else:
            runs.append([b])
    firsts = engine.acquire(len(runs))
    slots += firsts
    common = [prompts.common[batch[members[0]]] if len(members) > 1 else 0 for members in runs]
    begun = [Entry(first, reqs[members[0]].prompt[:n], []) for first, members, n in zip(firsts, runs, common) if n]
    if begun:
        engine.step(begun)
    slot_of, done = {}, {}
    for first, members, n in zip(firsts, runs, common):
        forks = engine.fork(first, len(members) - 1) if n else []
        slots += forks
        # (a run of several prompts has a page in common at least)
        slot_of.update(zip(members, [first] + forks))
        done.update((b, n) for b in members)
    logits = engine.step([Entry(slot_of[b], reqs[b].prompt[done[b]:], [len(reqs[b].prompt) - done[b] - 1]) for b in alone])
    rows = []
    for k, b in enumerate(alone):                        # equal prompts: the rest of them
        end = alone[k + 1] if k + 1 < len(alone) else len(reqs)
        rows += [k] * (end - b)
        if end - b > 1:
            children = engine.fork(slot_of[b], end - b - 1)
            slots += children
            slot_of.update(zip(range(b + 1, end), children))
    slots[:] = [slot_of[b] for b in range(len(reqs))]
    return logits if len(alone) == len(reqs) else logits[torch.tensor(rows, dtype=torch.long, device=logits.device)]


def generate(engine, requests, max_batch: int | None = None, on_token=None, cancel=None, share_prefix: bool = False) -> list:
    """Run every request to its end and return one GenerationResult each, in
    the order of the requests. `on_token(request index, token)` is called for
    every emitted token; `cancel()` returning True ends all live sequences with
    reason 'cancelled'. `share_prefix`: what the prompts of neighbouring requests have
    in common at their beginning is prefilled and held once (see the module text)."""
    requests = list(requests)
    context = engine.max_seq_len
    for i, r in enumerate(requests):
        if len(r.prompt) == 0:
            raise FormatError(f"request {i} has an empty prompt")
        if len(r.prompt) > context:
            raise ContextFull(len(r.prompt), context)
        r.params.check(engine.vocab)
    results = [None] * len(requests)
    final = [(i, min(len(r.prompt) + max(r.max_tokens, 0), context)) for i, r in enumerate(requests)]
    fits, prompts = engine.cache.can_hold, None
    if share_prefix and requests:
        prompts = _Prompts([list(r.prompt) for r in requests])
        final = [(i, (length, prompts.shared(i))) for i, length in final]

        def fits(items):                                 # (a batch's first sequence has nobody to share with)
            return engine.cache.can_hold_shared([n for n, _ in items], [0] + [shared for _, shared in items[1:]])
    batches = plan_batches(final, fits, max_batch or engine.max_slots)
    for batch in batches:
        _run_batch(engine, requests, batch, results, on_token, cancel, prompts)
    return results


_REASONS = ("eos", "max_tokens", "cancelled", "context_full")       # codes of csrc/host/generation.cpp


class _Schedule:
    """The batch's decisions, kept by the native host library (`csrc/host/generation.cpp`):
    who is live, who goes on, who leaves and why."""

    def __init__(self, reqs, max_seq_len: int):
        n = len(reqs)
        self.n = n
        stops = [int(t) for r in reqs for t in r.stop_tokens]
        handle = c_void_p()
        native.check(native.lib().llmh_generation_create(
            n, native.ints(int(r.max_tokens) for r in reqs), native.ints(len(r.stop_tokens) for r in reqs),
            native.ints(stops), int(max_seq_len), byref(handle)))
        self._handle = handle
        self._a, self._b, self._c, self._d = ((c_int * max(n, 1))() for _ in range(4))

    def __del__(self):
        if getattr(self, "_handle", None):
            native.lib().llmh_generation_destroy(self._handle)
            self._handle = None

    def live(self) -> list:
        return list(self._a[:native.lib().llmh_generation_live(self._handle, self._a)])

    def drop_exhausted(self):
        """(rows of the live list that stay, sequences that leave with 'max_tokens')."""
        kept, done = c_int(), c_int()
        native.check(native.lib().llmh_generation_drop_exhausted(self._handle, self._a, byref(kept), self._b,
                                                                 byref(done)))
        return list(self._a[:kept.value]), list(self._b[:done.value])

    def plan_onward(self, lengths) -> list:
        count = c_int()
        native.check(native.lib().llmh_generation_plan_onward(self._handle, native.ints(lengths), self._a,
                                                              byref(count)))
        return list(self._a[:count.value])

    def take_tokens(self, tokens):
        """(emitted flag per live row, [(sequence, reason)] that leave, rows of the planned step that stay)."""
        done, going = c_int(), c_int()
        native.check(native.lib().llmh_generation_take_tokens(
            self._handle, native.ints(tokens), self._a, self._b, self._c, byref(done), self._d, byref(going)))
        finished = [(self._b[i], _REASONS[self._c[i]]) for i in range(done.value)]
        return list(self._a[:len(tokens)]), finished, list(self._d[:going.value])

    def cancel(self) -> list:
        done = c_int()
        native.check(native.lib().llmh_generation_cancel(self._handle, self._a, byref(done)))
        return list(self._a[:done.value])


def _run_batch(engine, requests, batch, results, on_token, cancel, prompts=None) -> None:
    started = time.perf_counter()
    slots = []
    reqs = [requests[i] for i in batch]
    emitted = [[] for _ in batch]
    reason = ["max_tokens"] * len(batch)
    first_token_at = [None] * len(batch)
    sampler = BatchSampler([r.params for r in reqs], engine.vocab, engine.device)
    schedule = _Schedule(reqs, engine.max_seq_len)
    released = set()

    def finish(b, why):
        reason[b] = why
        if b not in released:
            engine.release([slots[b]])
            released.add(b)

    # ids travel device -> pinned host memory while the next step is already queued
    on_gpu = str(getattr(engine, "device", "cpu")).startswith("cuda")
    # (and behind them the sampler's refusal flags, read with every step's ids)
    staging = torch.empty(2 * len(batch), dtype=torch.int32, pin_memory=on_gpu)
    flags = staging[len(batch):]
    copied = torch.cuda.Event() if on_gpu else None

    try:
        live = schedule.live()
        logits = _start(engine, reqs, batch, prompts, slots)
        prefill_done = None
        while live:
            if cancel is not None and cancel():
                for b in schedule.cancel():
                    finish(b, "cancelled")
                break
            # sequences that may not emit anything leave before sampling
            rows, exhausted = schedule.drop_exhausted()
            if exhausted:
                for b in exhausted:
                    finish(b, "max_tokens")
                logits = logits[rows] if rows else logits[:0]
                live = schedule.live()
                if not live:
                    break
            sampled = sampler.sample(logits, live)               # int32 on the device
            staging[:len(live)].copy_(sampled, non_blocking=True)
            if not sampler.all_greedy:
                flags.copy_(sampler.status, non_blocking=True)
            if copied is not None:
                copied.record()
            # Who goes on is known before the ids are: everyone whose limits allow one more
            # token. Their next step is queued now, fed with the ids on the device; a
            # sequence that turns out to have drawn a stop token simply drops that step.
            onward = schedule.plan_onward([engine.length(slots[b]) for b in live])
            next_logits = None
            if onward:
                feed = sampled if len(onward) == len(live) else sampled[
                    torch.tensor(onward, dtype=torch.long, device=sampled.device)]
                next_logits = engine.step([Entry(slots[live[k]], [0], [0]) for k in onward],
                                          device_tokens=feed)
            if copied is not None:
                copied.synchronize()                             # the ids, not the queued step
            tokens = staging[:len(live)].tolist()
            sampler.check_status(flags)
            engine.check()
            now = time.perf_counter()
            if prefill_done is None:
                prefill_done = now
            counts, finished, going_rows = schedule.take_tokens(tokens)
            for b, token, counted in zip(live, tokens, counts):
                if not counted:
                    continue
                emitted[b].append(token)
                if first_token_at[b] is None:
                    first_token_at[b] = now
                if on_token is not None:
                    on_token(batch[b], token)
            for b, why in finished:
                finish(b, why)
            live = schedule.live()
            if live:
                logits = next_logits if len(going_rows) == len(onward) else next_logits[going_rows]
    finally:
        # (a prefill that failed has taken some of the slots)
        engine.release([slot for b, slot in enumerate(slots) if b not in released])
    ended = time.perf_counter()
    for b, index in enumerate(batch):
        n = len(emitted[b])
        first = first_token_at[b] if first_token_at[b] is not None else ended
        total_ms = (ended - started) * 1e3
        ttft_ms = (first - started) * 1e3
        decode_ms = max(total_ms - ttft_ms, 0.0)
        results[index] = GenerationResult(
            tokens=emitted[b], stop_reason=reason[b], prompt_tokens=len(reqs[b].prompt),
            generated_tokens=n, prefill_ms=((prefill_done or ended) - started) * 1e3,
            ttft_ms=ttft_ms, decode_ms=decode_ms, total_ms=total_ms,
            tokens_per_second=((n - 1) * 1e3 / decode_ms) if n > 1 and decode_ms > 0 else 0.0)
