"""Batched continuous decoding of many requests on the resident decoder.

The reference scheduler (glm_vx/scheduler.py:40-243) runs one model owner
thread that interleaves requests, one token of one request per model call
(scheduler.py:160-166), each call a host round trip per kernel.  Here the
owner thread drives a ResidentDecoder (gpu/decoder.py) whose B slots decode
together: every step advances every occupied slot by one token on the device
-- the next prompt token of a slot still in its prompt, the token chosen last
step otherwise -- and the host reads back B token ids (and, for sampled
requests only, their logits rows).  A request is admitted into a free slot,
whose caches are emptied first; it leaves its slot at EOS or max_tokens.

Interface kept from the reference: submit(tokens, max_tokens, temperature,
seed) -> Request with an `events` queue of {"type": "token", "token_id"} and
a final {"type": "done", "reason", ...}; cancel(req); status(); close();
BusyError when admission capacity is exhausted; the same ValueError texts.
Greedy requests take the device argmax; temperature > 0 samples on the host
from the row's logits exactly as the reference's _sample does
(scheduler.py:113-120).  The prefix cache and batched prefill of the
reference are not rebuilt (a prompt runs through the decode steps, one
token per step, which is the reference's prefill_token semantics).

Beyond the reference, a request may bring its own low-rank adapter (a decoder
with an AdapterBank, gpu/adapters.py) and its own rules for what it may say
(a decoder with LogitRules, gpu/rules.py): penalties for repeated tokens,
per-token biases, and a mask of allowed tokens, fixed or given anew for each
token by a function of the tokens generated so far (a grammar).  They are
applied on the device; a request whose rules leave no token ends with reason
'exhausted'.
"""
from collections import deque
from dataclasses import dataclass, field
import queue
import sys
import threading
import time
import uuid

import numpy as np

from .rules import allowed_tokens, to_f32


class BusyError(Exception):
    pass


@dataclass
class Request:
    tokens: tuple
    max_tokens: int
    temperature: float = 0.0
    seed: int = 0
    id: str = field(default_factory=lambda: 'cmpl-' + uuid.uuid4().hex)
    events: queue.Queue = field(default_factory=queue.Queue)
    cancelled: threading.Event = field(default_factory=threading.Event)
    cursor: int = 0
    generated: int = 0
    next_token: int | None = None
    created: float = field(default_factory=time.monotonic)
    first_token_at: float | None = None
    rng: object = None
    finished: bool = False
    reservation: int = 0
    slot: int = -1
    decode_seconds: float = 0.0
    adapter: int | None = None
    adapter_load: int = 0
    rules: dict = field(default_factory=dict)
    allowed: object = None
    output: list = field(default_factory=list)


class BatchScheduler:
    """Continuous batching over `decoder.B` slots of a ResidentDecoder."""

    def __init__(self, decoder, *, token_budget=None, max_pending_events=64):
        if type(max_pending_events) is not int or max_pending_events < 2:
            raise ValueError('at least two pending events required')
        self.decoder = decoder
        self.config = decoder.config
        self.slots = [None] * decoder.B
        self.token_budget = int(token_budget if token_budget is not None else decoder.B * decoder.capacity)
        self.max_pending_events = max_pending_events
        self.lock = threading.Condition()
        self.pending = deque()
        self.reserved = 0
        self.count = 0
        self.closed = False
        self.steps = 0
        self.error = None
        # Every slot advances one cache row per step, occupied or not: an
        # idle slot is emptied before it would reach the cache capacity.
        self.slot_len = [0] * decoder.B
        self.thread = threading.Thread(target=self._run, name='glm-vx-b200-decoder', daemon=True)
        self.thread.start()

    # ---------------------------------------------------------- admission
    def submit(self, tokens, max_tokens, temperature=0.0, seed=0, *, adapter=None, repetition_penalty=1.0,
               presence_penalty=0.0, frequency_penalty=0.0, logit_bias=None, allowed=None):
        """adapter: a loaded slot of the decoder's bank; should the adapter be
        unloaded or replaced, the request ends with reason 'error'.
        logit_bias: {token: value to add, -inf to ban}.  allowed: the tokens
        that may be said, as a boolean array over the vocabulary or token ids
        (copied here), or a function from the list of tokens generated so far
        to such a mask (or None: all)."""
        cfg = self.config
        if not isinstance(tokens, list) or not tokens or any(type(t) is not int or not 0 <= t < cfg['vocab_size']
                                                             for t in tokens):
            raise ValueError('prompt must be a nonempty array of valid token IDs')
        if type(max_tokens) is not int or max_tokens < 1:
            raise ValueError('max_tokens must be a positive integer')
        if not isinstance(temperature, (int, float)) or isinstance(temperature, bool) or \
                not 0 <= temperature <= sys.float_info.max:
            raise ValueError('temperature must be finite and nonnegative')
        if type(seed) is not int or seed < 0:
            raise ValueError('seed must be a nonnegative integer')
        rules, allowed = self._rules(repetition_penalty, presence_penalty, frequency_penalty, logit_bias, allowed)
        load = 0
        if adapter is not None:
            bank = getattr(self.decoder, 'adapters', None)
            if bank is not None and type(adapter) is int and 0 <= adapter < bank.slots:
                load = bank.loaded[adapter]
            if not load:
                raise ValueError('adapter must be a loaded slot of the decoder\'s adapter bank')
        amount = len(tokens) + max_tokens
        if amount > min(cfg.get('max_position_embeddings', 2**31 - 1), self.decoder.capacity):
            raise ValueError('request exceeds context limit')
        req = Request(tuple(tokens), max_tokens, float(temperature), seed, adapter=adapter,
                      adapter_load=load, rules=rules, allowed=allowed)
        req.reservation = amount
        req.rng = np.random.default_rng(seed)
        req.events = queue.Queue(maxsize=min(max_tokens + 2, self.max_pending_events))
        with self.lock:
            if self.closed:
                raise BusyError('scheduler is closed')
            if self.count >= len(self.slots) or self.reserved + amount > self.token_budget:
                raise BusyError('admission capacity exhausted')
            self.reserved += amount
            self.count += 1
            self.pending.append(req)
            self.lock.notify()
        return req

    def _rules(self, repetition, presence, frequency, bias, allowed):
        """The request's rules as LogitRules.set takes them ({}: none), and
        `allowed` as a mask of its own (an iterable is read once, an array may
        change) or the function that it is."""
        rules = getattr(self.decoder, 'rules', None)
        numbers = {'repetition_penalty': repetition, 'presence_penalty': presence, 'frequency_penalty': frequency}
        for name, value in numbers.items():
            if not isinstance(value, (int, float)) or isinstance(value, bool) or not np.isfinite(to_f32(value)):
                raise ValueError(f'{name} must be finite')
        if not to_f32(repetition) > 0:
            raise ValueError('repetition_penalty must be positive')
        bias = dict(bias or {})
        vocab = self.config['vocab_size']
        for token, value in bias.items():
            if type(token) is not int or not 0 <= token < vocab:
                raise ValueError('logit_bias must name valid token IDs')
            if not isinstance(value, (int, float)) or isinstance(value, bool) or not to_f32(value) < np.inf:
                raise ValueError('logit_bias values must be finite or -inf')
        if (repetition, presence, frequency) == (1.0, 0.0, 0.0) and not bias and allowed is None:
            return {}, None
        if rules is None:
            raise ValueError('the decoder has no logit rules')
        if len(bias) > rules.max_bias:
            raise ValueError(f'logit_bias names more than {rules.max_bias} tokens')
        if allowed is not None and not callable(allowed):
            allowed = allowed_tokens(allowed, vocab)
        return {'repetition': float(repetition), 'presence': float(presence), 'frequency': float(frequency),
                'bias': {token: float(to_f32(value)) for token, value in bias.items()}}, allowed

    def cancel(self, req):
        req.cancelled.set()
        with self.lock:
            self.lock.notify_all()

    def status(self):
        with self.lock:
            return {'active_requests': self.count, 'reserved_tokens': self.reserved, 'slots': len(self.slots),
                    'token_budget': self.token_budget, 'max_pending_events': self.max_pending_events,
                    'steps': self.steps, 'error': self.error}

    def close(self, timeout=10):
        with self.lock:
            self.closed = True
            self.lock.notify_all()
        self.thread.join(timeout=timeout)
        if self.thread.is_alive():
            raise TimeoutError('decoder worker is still stopping')

    # -------------------------------------------------------------- worker
    def _finish(self, req, reason, error=None):
        if req.finished:
            return
        req.finished = True
        if 0 <= req.slot < len(self.slots) and self.slots[req.slot] is req:
            self.slots[req.slot] = None
            self._vacate(req)
        with self.lock:
            self.reserved -= req.reservation
            self.count -= 1
            self.lock.notify_all()
        try:
            req.events.put_nowait({'type': 'done', 'reason': reason, 'error': error, 'prompt_tokens': len(req.tokens),
                                   'completion_tokens': req.generated, 'cached_prompt_tokens': 0,
                                   'timings': {'prefill_seconds': 0.0, 'decode_seconds': req.decode_seconds,
                                               'prefix_seconds': 0.0}})
        except queue.Full:
            pass

    def _replaced(self, req):
        """Whether the request's adapter is no longer the one it was submitted
        with; then it has ended.  Seen after a step, no load or unload met it."""
        if req.adapter is None or self.decoder.adapters.loaded[req.adapter] == req.adapter_load:
            return False
        self._finish(req, 'error', 'the adapter was unloaded or replaced')
        return True

    def _vacate(self, req):
        """Takes the request's adapter and rules from its slot, which is stepped
        with the others while it is idle."""
        try:
            if req.adapter is not None:
                self.decoder.set_adapter(req.slot)
            if req.rules:
                self.decoder.rules.clear(req.slot)
        except Exception as exc:  # the slot's next request does it again, or fails by it
            self.error = str(exc)

    def _fail(self, exc, requests):
        """Ends the requests that the decoder's failure `exc` leaves without a result."""
        self.error = str(exc)
        for req in requests:
            self._finish(req, 'error', str(exc))

    def _sample(self, logits, req):
        logits = np.asarray(logits, dtype=np.float32)
        # a request's own rules may take tokens out (-inf); anything else that is not finite is an error
        fine = np.isfinite(logits) | (logits == -np.inf if req.rules else False)
        if logits.shape != (self.config['vocab_size'],) or not np.all(fine):
            raise ValueError('nonfinite or invalid logits')
        scaled = (logits.astype(np.float64) - float(np.max(logits))) / req.temperature
        probs = np.exp(scaled)
        probs /= probs.sum()
        return int(req.rng.choice(len(probs), p=probs))

    def _admit(self):
        with self.lock:
            while not self.pending and not self.closed and not any(self.slots):
                self.lock.wait()
            arrivals = list(self.pending)
            self.pending.clear()
            closed = self.closed
        for req in arrivals:
            free = self.slots.index(None)
            req.slot = free
            self.slots[free] = req
            try:
                self.decoder.reset_slot(free)
                self.slot_len[free] = 0
                if getattr(self.decoder, 'adapters', None) is not None:
                    self.decoder.set_adapter(free, req.adapter)
                if self._replaced(req):
                    continue
                if req.rules:
                    fixed = req.allowed if not callable(req.allowed) else None
                    self.decoder.rules.set(free, prompt=len(req.tokens), allowed=fixed, **req.rules)
            except ValueError as exc:  # the adapter was unloaded meanwhile, or the like: this request's own failure
                self._finish(req, 'error', str(exc))
            except Exception as exc:  # the device's, which the other requests meet in their next step
                self._fail(exc, [req])
        for b, r in enumerate(self.slots):
            if r is None and self.slot_len[b] >= self.decoder.capacity - 1:
                try:
                    self.decoder.reset_slot(b)
                    self.slot_len[b] = 0
                except Exception as exc:  # its cache would run over in a step of the others
                    self._fail(exc, [r for r in self.slots if r is not None])
        return closed

    def _run(self):
        dec, eos = self.decoder, self.config.get('eos_token_id', [])
        eos = [eos] if isinstance(eos, int) else list(eos or [])
        while True:
            closed = self._admit()
            for req in [r for r in self.slots if r is not None]:
                if closed or req.cancelled.is_set():
                    self._finish(req, 'cancelled')
                elif req.events.qsize() >= req.events.maxsize - 1:
                    self._finish(req, 'backpressure', 'client output queue is full')
            for r in [r for r in self.slots if r is not None and callable(r.allowed)]:
                if r.cursor + 1 >= len(r.tokens):  # the coming step's choice is used
                    try:
                        self.decoder.rules.allow(r.slot, r.allowed(list(r.output)))
                    except Exception as exc:  # the request's own function failed, or its mask is none
                        self._finish(r, 'error', str(exc))
            active = [r for r in self.slots if r is not None]
            if closed and not active:
                return
            if not active:
                continue
            try:
                feed = [0] * len(self.slots)
                for r in active:
                    feed[r.slot] = r.tokens[r.cursor] if r.cursor < len(r.tokens) else r.next_token
                t0 = time.perf_counter()
                dec.set_tokens(feed)
                dec.step()
                chosen = dec.read_tokens()
                sampled = [r for r in active if r.temperature > 0 and r.cursor + 1 >= len(r.tokens)]
                logits = dec.read_logits() if sampled else None
                dt = time.perf_counter() - t0
                self.steps += 1
                self.slot_len = [n + 1 for n in self.slot_len]
            except Exception as exc:  # the device or a bounded wait failed: every active request ends
                self._fail(exc, active)
                continue
            for r in active:
                if self._replaced(r):
                    continue
                r.decode_seconds += dt
                if r.cursor < len(r.tokens):
                    r.cursor += 1
                    if r.cursor < len(r.tokens):
                        continue  # still inside the prompt: this step's output is not sampled
                if chosen[r.slot] < 0:  # no logit above -inf: by its rules, or the model's
                    self._finish(r, *(('exhausted', 'no token is allowed') if r.rules else
                                      ('error', 'nonfinite logits')))
                    continue
                try:
                    token = self._sample(logits[r.slot], r) if r.temperature > 0 else int(chosen[r.slot])
                except ValueError as exc:  # nothing to sample from: rules can sum up to an infinite logit
                    self._finish(r, 'error', str(exc))
                    continue
                r.output.append(token)
                r.generated += 1
                r.next_token = token
                if r.first_token_at is None:
                    r.first_token_at = time.monotonic()
                r.events.put_nowait({'type': 'token', 'token_id': token})
                reason = 'stop' if token in eos else 'length' if r.generated >= r.max_tokens else None
                if reason:
                    self._finish(r, reason)


def collect(req, timeout=60.0):
    """Drain a request's events: (token ids, done event)."""
    tokens = []
    while True:
        ev = req.events.get(timeout=timeout)
        if ev['type'] == 'token':
            tokens.append(ev['token_id'])
        else:
            return tokens, ev
