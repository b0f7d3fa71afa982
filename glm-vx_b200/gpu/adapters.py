"""Low-rank adapters of many requests, resident beside a model's projections.

A serving batch holds rows of different users; each may bring a low-rank
change of some projections, y += scale * B (A x), instead of its own copy of
the model.  `AdapterBank` keeps up to `slots` such adapters on the device,
for every projection they may change one stack of A [slots][max_rank][cols]
and one of B [slots][rows][max_rank], and adds them to a projection's output
for a whole batch at once, each row by its own adapter (glmvx_lora_add).
Nothing about the adapters is part of a captured step but the stacks'
addresses: loading, replacing or dropping one needs no new capture.

The reference serves one set of weights (glm_vx/model.py:178-324); this has
no counterpart there.  gpu/decoder.py `ResidentDecoder(adapters=bank)` adds
the bank to its projections, gpu/serving.py `submit(adapter=slot)` picks one
for a request.
"""

import itertools
import threading

import numpy as np

from . import runtime as rt
from .rules import to_f32

MAX_RANK = 256
# Storage of the stacks: GGML kind -> (bytes of a weight, name).
KINDS = {0: (4, 'F32'), 1: (2, 'F16'), 30: (2, 'BF16')}
ATTENTION_PARTS = ('q_a_proj', 'q_b_proj', 'kv_a_proj_with_mqa', 'o_proj')
MLP_PARTS = ('gate_proj', 'up_proj', 'down_proj')


def projection_shapes(config, layers=None):
    """{projection name: (rows, cols)} of the projections of a GLM-MoE-DSA
    model that an adapter may change: the attention projections of every
    layer and the MLP of the dense ones (the indexer's, the routed experts'
    and kv_b, which the decoder absorbs into the queries, stay as they are)."""
    from .decoder import _layer_types
    n = int(config['num_hidden_layers'])
    H, heads = int(config['hidden_size']), int(config['num_attention_heads'])
    q_lora, rot = int(config['q_lora_rank']), int(config['qk_rope_head_dim'])
    attention = {'q_a_proj': (q_lora, H), 'q_b_proj': (heads * (int(config['qk_nope_head_dim']) + rot), q_lora),
                 'kv_a_proj_with_mqa': (int(config['kv_lora_rank']) + rot, H),
                 'o_proj': (H, heads * int(config['v_head_dim']))}
    shapes = {}
    mlp_types = _layer_types(config, n)[1]
    for i in range(int(n if layers is None else layers)):
        for part in ATTENTION_PARTS:
            shapes[f'model.layers.{i}.self_attn.{part}'] = attention[part]
        if mlp_types[i] == 'dense':
            I = int(config['intermediate_size'])
            for part, shape in zip(MLP_PARTS, ((I, H), (I, H), (H, I))):
                shapes[f'model.layers.{i}.mlp.{part}'] = shape
    return shapes


def to_kind(values, kind):
    """A float32 array rounded once (nearest, ties to even) to the kind's
    storage: float32, float16, or BF16 as its uint16 bit patterns."""
    values = np.ascontiguousarray(values, np.float32)
    if kind == 0:
        return values
    if kind == 1:
        with np.errstate(over='ignore'):
            half = values.astype(np.float16)
        if not np.isfinite(half).all():
            raise ValueError('adapter weights exceed the F16 range')
        return half
    bits = values.view(np.uint32).astype(np.uint64)
    rounded = (bits + 0x7fff + (bits >> 16 & 1)) >> 16
    if ((rounded & 0x7f80) == 0x7f80).any():
        raise ValueError('adapter weights exceed the BF16 range')
    return rounded.astype(np.uint16)


class AdapterBank:
    """Up to `slots` adapters of ranks up to `max_rank` for the projections
    `shapes` ({name: (rows, cols)}), stored as GGML `kind` 0 (F32), 1 (F16) or
    30 (BF16), for calls of up to `max_tokens` rows.

    The calls of one bank share its workspace, so they belong on one stream
    (the backend's by default).

    loaded[slot] is False while the slot is empty or about to change, else the
    number of the load that filled it, another one each time: equal before
    and after a step, it stood still meanwhile."""

    _loads = itertools.count(1)

    def __new__(cls, *args, **kwargs):
        bank = super().__new__(cls)
        bank._changing = threading.RLock()  # one load or unload at a time: a slot is one adapter's as a whole
        return bank

    def __init__(self, backend, shapes, slots, max_rank, kind=30, max_tokens=64):
        self.shapes = {str(k): (int(r), int(c)) for k, (r, c) in dict(shapes).items()}
        self.slots, self.max_rank, self.kind, self.max_tokens = int(slots), int(max_rank), int(kind), int(max_tokens)
        if not self.shapes or any(min(s) < 1 for s in self.shapes.values()):
            raise ValueError('an adapter bank needs projections with positive shapes')
        if self.slots < 1 or not 1 <= self.max_rank <= MAX_RANK or not 1 <= self.max_tokens <= 1 << 20:
            raise ValueError(f'slots and max_tokens must be positive, max_rank 1..{MAX_RANK}')
        if self.slots > 1 << 24 or any(max(s) > 1 << 22 for s in self.shapes.values()):
            raise ValueError('a bank has at most 2^24 slots, and projections of at most 2^22 rows and columns')
        if self.kind not in KINDS:
            raise ValueError('adapters are stored as kind 0 (F32), 1 (F16) or 30 (BF16)')
        self.backend, self.lib = backend, backend.lib
        backend._begin()
        self._bufs = []
        self._stacks = {}
        self.loaded = [False] * self.slots
        size = KINDS[self.kind][0]
        stream = backend.stream.handle
        with backend.device.lock:  # no other thread captures a step on the stream meanwhile
            for name, (rows, cols) in self.shapes.items():
                a = self._dev(self.slots * self.max_rank * cols * size)
                b = self._dev(self.slots * self.max_rank * rows * size)
                ranks, scales = self._dev(4 * self.slots), self._dev(4 * self.slots)
                rt.call('glmvx_memset', ranks.ptr, 0, 4 * self.slots, stream)
                rt.call('glmvx_memset', scales.ptr, 0, 4 * self.slots, stream)
                self._stacks[name] = (a, b, ranks, scales)
            need = int(self.lib.glmvx_lora_workspace_bytes(self.max_tokens, self.slots, self.max_rank))
            self._workspace, self._workspace_bytes = self._dev(need), need
            backend.stream.synchronize()

    def _dev(self, nbytes):
        buf = rt.DeviceBuffer(max(int(nbytes), 256))
        self._bufs.append(buf)
        return buf

    def _slot(self, slot):
        if type(slot) is not int or not 0 <= slot < self.slots:
            raise ValueError('adapter slot outside the bank')
        return slot

    def _put(self, buf, array, offset):
        with self.backend.device.lock:  # no other thread captures a step on the stream meanwhile
            self.backend.stream.synchronize()  # steps in flight still read what is there
            buf.upload(array, self.backend.stream.handle, offset)
            self.backend.stream.synchronize()

    def load(self, slot, weights, scale=1.0):
        """Fills `slot` with an adapter: weights {name: (A [r, cols], B [rows,
        r])} with 0 <= r <= max_rank, the same scale (alpha / r of the usual
        convention) for all of them; projections without an entry are left
        as the model has them.  Steps that run meanwhile see the slot empty,
        then with the projections that are already there."""
        slot = self._slot(slot)
        scale = to_f32(scale)
        if not np.isfinite(scale):
            raise ValueError('adapter scale must be finite')
        ready = {}
        for name, pair in weights.items():
            if name not in self.shapes:
                raise ValueError(f'{name} is not a projection of the bank')
            rows, cols = self.shapes[name]
            a, b = (np.asarray(v, np.float32) for v in pair)
            r = a.shape[0] if a.ndim == 2 else -1
            if a.shape != (r, cols) or b.shape != (rows, r):
                raise ValueError(f'{name}: A {a.shape} and B {b.shape} do not fit ({rows}, {cols})')
            if r > self.max_rank:
                raise ValueError(f'{name}: rank {r} exceeds {self.max_rank}')
            if not (np.isfinite(a).all() and np.isfinite(b).all()):
                raise ValueError(f'{name}: nonfinite adapter weights')
            wide = np.zeros((rows, self.max_rank), np.float32)
            wide[:, :r] = b
            ready[name] = (r, to_kind(a, self.kind), to_kind(wide, self.kind))
        with self._changing:
            self.unload(slot)
            for name, (r, a, b) in ready.items():
                sa, sb, ranks, scales = self._stacks[name]
                size = KINDS[self.kind][0]
                rows, cols = self.shapes[name]
                if r:
                    self._put(sa, a, slot * self.max_rank * cols * size)
                    self._put(sb, b, slot * self.max_rank * rows * size)
                self._put(scales, np.array([scale]), 4 * slot)
                self._put(ranks, np.array([r], np.int32), 4 * slot)
            self.loaded[slot] = next(self._loads)

    def unload(self, slot):
        """Empties `slot`: rows that still name it are left as the model has them."""
        slot = self._slot(slot)
        with self._changing:
            self.backend._begin()
            self.loaded[slot] = False
            for _, _, ranks, _ in self._stacks.values():
                self._put(ranks, np.zeros(1, np.int32), 4 * slot)

    def add(self, name, y, x, ids, tokens, stream=None):
        """y[t] += the adapter ids[t]'s change of projection `name` at x[t], t <
        tokens: device addresses of f32 [tokens][rows], f32 [tokens][cols] and
        int32 [tokens] (-1: none)."""
        rows, cols = self.shapes[name]
        if not 0 <= tokens <= self.max_tokens:
            raise ValueError('more tokens than the bank was made for')
        a, b, ranks, scales = self._stacks[name]
        rt.check(self.lib, self.lib.glmvx_lora_add(
            y, rows, x, cols, ids, self.kind, a.ptr, b.ptr, ranks.ptr, scales.ptr, tokens, rows, cols, self.slots,
            self.max_rank, self._workspace.ptr, self._workspace_bytes,
            self.backend.stream.handle if stream is None else stream), 'glmvx_lora_add')

    def close(self):
        with self.backend.device.lock:
            if self._bufs:
                self.backend.stream.synchronize()
            for buf in self._bufs:
                buf.close()
            self._bufs = []
