"""What each sequence of a batch may say next: penalties, biases, grammar masks.

`LogitRules` holds, for the B sequences of a decoder, on the device: the
tokens each has been fed (prompt, then output), its repetition, presence and
frequency penalties, its per-token biases and a mask of the tokens its
grammar allows.  `select` turns a step's logits into the ones these rules
leave and picks the largest, in one kernel that a captured step replays
(glmvx_logits_select): setting a sequence's rules or its mask between steps
needs no new capture and no logits on the host.

The reference takes the model's logits as they are (glm_vx/generate.py:96,
glm_vx/scheduler.py:113-120); this has no counterpart there.
"""
import operator

import numpy as np

from . import runtime as rt

MAX_BIAS = 2047


def to_f32(value):
    """The value as a float32, infinite beyond its range (whole numbers too)."""
    with np.errstate(over='ignore'):
        try:
            return np.float32(value)
        except OverflowError:
            return np.float32(np.inf if value > 0 else -np.inf)


def allowed_tokens(allowed, vocab):
    """A new boolean array [vocab], True where token v is allowed: from such an
    array, or an array or iterable of token ids."""
    allowed = np.asarray(allowed if isinstance(allowed, np.ndarray) else list(allowed))
    if allowed.dtype == np.bool_:
        if allowed.shape != (vocab,):
            raise ValueError(f'a mask has one truth value for each of {vocab} tokens')
        return allowed.copy()
    if allowed.size and (allowed.dtype.kind not in 'iu' or allowed.min() < 0 or allowed.max() >= vocab):
        raise ValueError('allowed token ids must be in the vocabulary')
    keep = np.zeros(vocab, bool)
    keep[allowed.astype(np.int64).reshape(-1)] = True
    return keep


def pack_mask(allowed, vocab):
    """uint32 words, bit v % 32 of word v // 32 set where token v is allowed
    (`allowed` as in allowed_tokens)."""
    words, keep = (vocab + 31) // 32, allowed_tokens(allowed, vocab)
    return np.packbits(np.pad(keep, (0, 32 * words - vocab)), bitorder='little').view('<u4').astype(np.uint32)


class LogitRules:
    """Rules of `batch` sequences over `vocab` tokens, with histories of up to
    `capacity` tokens (what is fed after that is not remembered) and up to
    `max_bias` biased tokens each.  A sequence without rules gets the plain
    argmax (-1 when nothing is above -inf)."""

    def __init__(self, backend, batch, vocab, capacity, max_bias=512):
        self.batch, self.vocab = int(batch), int(vocab)
        self.capacity, self.max_bias = int(capacity), int(max_bias)
        if min(self.batch, self.vocab, self.capacity) < 1 or not 1 <= self.max_bias <= MAX_BIAS:
            raise ValueError(f'batch, vocabulary and capacity must be positive, max_bias 1..{MAX_BIAS}')
        if self.capacity > (1 << 20) - 2:
            raise ValueError('histories hold up to 2^20 - 2 tokens')
        self.backend, self.lib = backend, backend.lib
        backend._begin()
        B, W = self.batch, (self.vocab + 31) // 32
        self.words = W
        self._masked = [None] * B  # whether sequence b has a mask (None: not yet said)
        sizes = (('history', 4 * B * self.capacity), ('lens', 4 * B), ('prompts', 4 * B), ('penalties', 12 * B),
                 ('bias_ids', 4 * B * self.max_bias), ('bias_values', 4 * B * self.max_bias), ('bias_lens', 4 * B),
                 ('masks', 4 * B * W), ('mask_rows', 4 * B))
        with backend.device.lock:  # no other thread captures a step on the stream meanwhile
            self._bufs = {name: rt.DeviceBuffer(nbytes) for name, nbytes in sizes}
        for b in range(B):
            self.clear(b)

    def _put(self, name, array, item, width=1):
        """`array` into element `item` of buffer `name` (elements of `width` words)."""
        s = self.backend.stream
        with self.backend.device.lock:  # no other thread captures a step on the stream meanwhile
            s.synchronize()  # a step in flight still reads what is there
            self._bufs[name].upload(np.ascontiguousarray(array), s.handle, 4 * item * width)
            s.synchronize()

    def _sequence(self, b):
        if not 0 <= b < self.batch:
            raise ValueError('sequence outside the batch')
        self.backend._begin()
        return b

    def restart(self):
        """Every history is empty; the rules stay."""
        self.backend._begin()
        self._put('lens', np.zeros(self.batch, np.int32), 0)

    def clear(self, b):
        """Sequence b has no history and no rules."""
        self._put('lens', np.zeros(1, np.int32), self._sequence(b))
        self.set(b)

    def set(self, b, prompt=0, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
        """Sequence b's rules from now on: the first `prompt` fed tokens are its
        prompt (they count for the repetition penalty only); tokens seen are
        divided (positive logits) or multiplied by `repetition`, output tokens
        lose `frequency` per occurrence and `presence` once; `bias` {token:
        value} is added (-inf bans); `allowed` as in allowed_tokens (None:
        all)."""
        self._sequence(b)
        values = np.array([to_f32(v) for v in (repetition, presence, frequency)])
        if not np.isfinite(values).all() or values[0] <= 0:
            raise ValueError('penalties must be finite, the repetition penalty positive')
        if int(prompt) < 0:
            raise ValueError('prompt length must be nonnegative')
        try:
            bias = {operator.index(t): to_f32(v) for t, v in dict(bias or {}).items()}
        except TypeError as exc:
            raise ValueError('biased tokens must be whole numbers') from exc
        if len(bias) > self.max_bias:
            raise ValueError(f'more than {self.max_bias} biased tokens')
        if any(not 0 <= t < self.vocab for t in bias):
            raise ValueError('biased tokens must be in the vocabulary')
        biases = np.array(list(bias.values()), np.float32)
        if np.isnan(biases).any() or (biases == np.inf).any():
            raise ValueError('biases must be finite or -inf')
        words = None if allowed is None else pack_mask(allowed, self.vocab)
        self._put('prompts', np.array([min(int(prompt), 2**31 - 1)], np.int32), b)
        self._put('penalties', values, b, 3)
        if bias:
            self._put('bias_ids', np.array(list(bias), np.int32), b, self.max_bias)
            self._put('bias_values', biases, b, self.max_bias)
        self._put('bias_lens', np.array([len(bias)], np.int32), b)
        self._mask(b, words)

    def allow(self, b, allowed):
        """Replaces sequence b's mask alone (a grammar's next state; None: all)."""
        self._sequence(b)
        self._mask(b, None if allowed is None else pack_mask(allowed, self.vocab))

    def _mask(self, b, words):
        if words is not None:
            self._put('masks', words, b, self.words)
        if self._masked[b] is not (words is not None):
            self._put('mask_rows', np.array([-1 if words is None else b], np.int32), b)
            self._masked[b] = words is not None

    def history(self, b):
        """The tokens sequence b has been fed."""
        self._sequence(b)
        lens = np.empty(self.batch, np.int32)
        with self.backend.device.lock:
            self.backend.stream.synchronize()
            self._bufs['lens'].download(lens, self.backend.stream.handle)
            self.backend.stream.synchronize()
            row = np.empty(int(lens[b]), np.int32)
            if row.size:
                self._bufs['history'].download(row, self.backend.stream.handle, 4 * b * self.capacity)
                self.backend.stream.synchronize()
        return row

    def select(self, tokens, logits, stream=None):
        """One step's choice, device addresses: tokens int32 [batch], the tokens
        just fed, become the chosen ones (-1: nothing is allowed); logits f32
        [batch][vocab] become the ones the rules leave."""
        d = {name: buf.ptr for name, buf in self._bufs.items()}
        rt.check(self.lib, self.lib.glmvx_logits_select(
            tokens, logits, self.vocab, logits, self.vocab, self.batch, self.vocab, tokens, d['history'], self.capacity,
            d['lens'], d['prompts'], d['penalties'], d['bias_ids'], d['bias_values'], d['bias_lens'], self.max_bias,
            d['masks'], d['mask_rows'], self.batch, self.backend.stream.handle if stream is None else stream),
            'glmvx_logits_select')

    def close(self):
        with self.backend.device.lock:
            if self._bufs:
                self.backend.stream.synchronize()
            for buf in self._bufs.values():
                buf.close()
            self._bufs = {}
