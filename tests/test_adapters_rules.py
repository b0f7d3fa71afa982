"""Adapter banks, logit rules and the scheduler's use of them, without a GPU:
argument checks, storage rounding, masks, and the serving loop over a decoder
that applies the rules in NumPy."""
from types import SimpleNamespace

import numpy as np
import pytest

from gpu.adapters import AdapterBank, projection_shapes, to_kind
from gpu.rules import LogitRules, pack_mask
from gpu.serving import BatchScheduler, collect

CONFIG = dict(num_hidden_layers=2, hidden_size=64, num_attention_heads=2, q_lora_rank=32, kv_lora_rank=32,
              qk_nope_head_dim=16, qk_rope_head_dim=8, v_head_dim=16, intermediate_size=96, vocab_size=50,
              mlp_layer_types=['dense', 'sparse'])


class NoDevice:
    """A backend whose device must not be reached."""
    lib = None

    def _begin(self):
        raise AssertionError('the device was reached')


def test_projection_shapes():
    shapes = projection_shapes(CONFIG)
    assert shapes['model.layers.0.self_attn.q_a_proj'] == (32, 64)
    assert shapes['model.layers.1.self_attn.q_b_proj'] == (48, 32)
    assert shapes['model.layers.0.self_attn.kv_a_proj_with_mqa'] == (40, 64)
    assert shapes['model.layers.1.self_attn.o_proj'] == (64, 32)
    assert shapes['model.layers.0.mlp.down_proj'] == (64, 96)
    assert not any(name.startswith('model.layers.1.mlp') for name in shapes)
    assert not any(name.startswith('model.layers.1') for name in projection_shapes(CONFIG, layers=1))


@pytest.mark.parametrize('change,message', [
    (dict(shapes={}), 'projections'), (dict(shapes={'a': (0, 4)}), 'positive'), (dict(slots=0), 'positive'),
    (dict(max_rank=0), 'max_rank'), (dict(max_rank=257), 'max_rank'), (dict(max_tokens=0), 'positive'),
    (dict(kind=8), 'kind')])
def test_bank_refusals(change, message):
    args = dict(shapes={'a': (4, 4)}, slots=2, max_rank=4, kind=30, max_tokens=4)
    args.update(change)
    with pytest.raises(ValueError, match=message):
        AdapterBank(NoDevice(), **args)


def bank_without_device():
    bank = AdapterBank.__new__(AdapterBank)
    bank.shapes, bank.slots, bank.max_rank, bank.kind, bank.max_tokens = {'a': (6, 4)}, 2, 3, 30, 4
    bank.backend, bank.loaded, bank._bufs = NoDevice(), [False, False], []
    return bank


@pytest.mark.parametrize('slot,weights,scale,message', [
    (2, {}, 1.0, 'slot'), (-1, {}, 1.0, 'slot'), (True, {}, 1.0, 'slot'), (0, {}, np.inf, 'scale'),
    (0, {'b': (np.zeros((1, 4)), np.zeros((6, 1)))}, 1.0, 'not a projection'),
    (0, {'a': (np.zeros((1, 5)), np.zeros((6, 1)))}, 1.0, 'fit'),
    (0, {'a': (np.zeros((2, 4)), np.zeros((6, 1)))}, 1.0, 'fit'),
    (0, {'a': (np.zeros(4), np.zeros((6, 1)))}, 1.0, 'fit'),
    (0, {'a': (np.zeros((4, 4)), np.zeros((6, 4)))}, 1.0, 'rank 4'),
    (0, {'a': (np.full((1, 4), np.nan), np.zeros((6, 1)))}, 1.0, 'nonfinite'),
    (0, {'a': (np.full((1, 4), 3.4e38), np.zeros((6, 1)))}, 1.0, 'BF16')])
def test_load_refusals(slot, weights, scale, message):
    with pytest.raises(ValueError, match=message):
        bank_without_device().load(slot, weights, scale)


@pytest.mark.parametrize('part', ['adapters', 'rules'])
def test_a_decoder_refuses_what_belongs_to_another_backend(part):
    from gpu.decoder import ResidentDecoder
    config = dict(CONFIG, index_n_heads=2, index_head_dim=16, index_topk=8, indexer_types=['full', 'full'])
    theirs = dict(adapters=SimpleNamespace(backend=NoDevice(), shapes={}, max_tokens=2, slots=2),
                  rules=SimpleNamespace(backend=NoDevice(), batch=2, vocab=50))
    with pytest.raises(ValueError, match='backend'):
        ResidentDecoder(NoDevice(), config, None, batch=2, capacity=8, **{part: theirs[part]})


class CountingLock:
    depth = 0

    def __enter__(self):
        self.depth += 1

    def __exit__(self, *exc):
        self.depth -= 1


class QuietBackend:
    """A backend that only notes whether the device's lock was held."""

    def __init__(self):
        self.device, self.held = SimpleNamespace(lock=CountingLock()), []
        self.stream = SimpleNamespace(handle=0, synchronize=self._note)

    def _note(self, *args):
        self.held.append(self.device.lock.depth > 0)

    def _begin(self):
        pass

    def buffer(self):
        return SimpleNamespace(ptr=0, upload=self._note)


def test_what_is_put_into_place_waits_for_a_capture(monkeypatch):
    """Loading an adapter or a rule works on the stream that another thread may be capturing a step on: both hold the
    device's lock."""
    from gpu import decoder
    from gpu import runtime as rt
    backend = QuietBackend()
    bank = bank_without_device()
    bank.backend, bank._stacks = backend, {'a': tuple(backend.buffer() for _ in range(4))}
    bank.load(0, {'a': (np.zeros((1, 4)), np.zeros((6, 1)))})
    assert len(backend.held) >= 12 and all(backend.held)
    backend.held.clear()
    rules = LogitRules.__new__(LogitRules)
    rules.backend, rules.batch, rules.vocab, rules.max_bias, rules.words = backend, 2, 50, 4, 2
    rules._masked = [None, None]
    rules._bufs = {n: backend.buffer() for n in ('lens', 'prompts', 'penalties', 'bias_ids', 'bias_values', 'bias_lens',
                                                 'masks', 'mask_rows')}
    rules.set(1, bias={3: 1.0}, allowed=[1, 2])
    assert len(backend.held) >= 12 and all(backend.held)
    backend.held.clear()
    dec = decoder.ResidentDecoder.__new__(decoder.ResidentDecoder)
    dec.backend, dec._graph, dec._step_launches, dec._bufs = backend, None, backend._note, []
    monkeypatch.setattr(rt, 'Graph', lambda stream: SimpleNamespace(begin=backend._note, end=backend._note))
    dec.step_graph()
    assert backend.held == [True] * 3 and backend.device.lock.depth == 0


def test_storage_rounding():
    x = np.array([1.0, 1 + 2.0**-8, 1 + 3 * 2.0**-8, -1 - 2.0**-8 - 2.0**-20, 2.0**-130, 0.0], np.float32)
    got = (to_kind(x, 30).astype(np.uint32) << 16).view(np.float32)
    assert got[:4].tolist() == [1.0, 1.0, 1 + 2.0**-6, -1 - 2.0**-7]
    assert np.all(np.abs(got - x) <= np.abs(x) * 2.0**-8 + 2.0**-133)
    half = to_kind(x, 1).astype(np.float32)
    assert np.all(np.abs(half - x) <= np.abs(x) * 2.0**-11 + 2.0**-25)
    assert to_kind(x, 0).tobytes() == x.tobytes()
    with pytest.raises(ValueError, match='F16'):
        to_kind(np.float32([7e4]), 1)


def test_pack_mask():
    keep = np.zeros(70, bool)
    keep[[0, 31, 32, 69]] = True
    words = pack_mask(keep, 70)
    assert words.dtype == np.uint32 and words.tolist() == [1 | 1 << 31, 1, 1 << 5]
    assert pack_mask([0, 31, 32, 69, 69], 70).tolist() == words.tolist()
    assert pack_mask(np.array([69]), 70).tolist() == [0, 0, 32]
    assert pack_mask([], 70).tolist() == [0, 0, 0] and pack_mask(set(), 70).tolist() == [0, 0, 0]
    for bad in (np.zeros(69, bool), [70], [-1], [0.5]):
        with pytest.raises(ValueError):
            pack_mask(bad, 70)


@pytest.mark.parametrize('change,message', [
    (dict(batch=0), 'positive'), (dict(vocab=0), 'positive'), (dict(capacity=0), 'positive'),
    (dict(max_bias=0), 'max_bias'), (dict(max_bias=2048), 'max_bias'), (dict(capacity=2**20 - 1), '2\\^20')])
def test_rules_refusals(change, message):
    args = dict(batch=2, vocab=10, capacity=8, max_bias=4)
    args.update(change)
    with pytest.raises(ValueError, match=message):
        LogitRules(NoDevice(), **args)


class HostRules:
    """LogitRules' interface over NumPy."""

    def __init__(self, batch, vocab):
        self.batch, self.vocab, self.max_bias = batch, vocab, 4
        self.rows = [None] * batch
        for b in range(batch):
            self.clear(b)

    def clear(self, b):
        self.rows[b] = dict(history=[], prompt=0, repetition=1.0, presence=0.0, frequency=0.0, bias={}, allowed=None)

    def set(self, b, **rules):
        self.rows[b].update(rules)

    def allow(self, b, allowed):
        if allowed is not None:
            pack_mask(allowed, self.vocab)
        self.rows[b]['allowed'] = allowed

    def select(self, fed, logits):
        chosen = []
        for b, row in enumerate(self.rows):
            row['history'].append(int(fed[b]))
            l = logits[b].astype(np.float64)
            for t in set(row['history']):
                l[t] = l[t] / row['repetition'] if l[t] > 0 else l[t] * row['repetition']
            said = row['history'][row['prompt']:]
            for t in set(said):
                l[t] -= said.count(t) * row['frequency'] + row['presence']
            for t, v in row['bias'].items():
                l[t] += v
            if row['allowed'] is not None:
                words = pack_mask(row['allowed'], self.vocab)
                v = np.arange(self.vocab)
                l[(words[v // 32] >> (v % 32).astype(np.uint32)) & 1 == 0] = -np.inf
            logits[b] = l
            chosen.append(int(np.argmax(l)) if l.max() > -np.inf else -1)
        return chosen


class HostDecoder:
    """A decoder whose logits depend on the fed token and the sequence's adapter alone."""

    def __init__(self, batch, vocab, rules=True, slots=0):
        self.B, self.capacity, self.config = batch, 64, dict(vocab_size=vocab)
        self.table = np.random.default_rng(3).normal(size=(4, vocab, vocab)).astype(np.float32)
        self.rules = HostRules(batch, vocab) if rules else None
        self.adapters = None
        if slots:
            self.adapters = bank_without_device()
            self.adapters.slots, self.adapters.loaded = slots, [True] * slots
        self.adapter = [None] * batch

    def reset_slot(self, b):
        if self.rules:
            self.rules.clear(b)

    def set_adapter(self, b, slot=None):
        if slot is not None and not self.adapters.loaded[slot]:
            raise ValueError('no adapter is loaded there')
        self.adapter[b] = slot

    def set_tokens(self, tokens):
        self.fed = list(tokens)

    def step(self):
        self.logits = np.stack([self.table[0 if a is None else 1 + a, t] for a, t in zip(self.adapter, self.fed)])
        self.chosen = self.rules.select(self.fed, self.logits) if self.rules else self.logits.argmax(1).tolist()

    def read_tokens(self):
        return np.array(self.chosen, np.int32)

    def read_logits(self):
        return self.logits.copy()


@pytest.fixture
def serve():
    made = []

    def start(*args, **kwargs):
        made.append(BatchScheduler(HostDecoder(*args, **kwargs)))
        return made[-1]

    yield start
    for sched in made:
        sched.close()


def greedy(table, token, n):
    out = []
    for _ in range(n):
        token = int(np.argmax(table[token]))
        out.append(token)
    return out


def test_requests_keep_to_their_own_rules_and_adapters(serve):
    sched = serve(4, 50, slots=2)
    table = sched.decoder.table
    plain = sched.submit([7, 8], 6)
    other = sched.submit([7, 8], 6, adapter=1)
    first = greedy(table[0], 8, 1)[0]
    banned = sched.submit([7, 8], 6, logit_bias={first: float('-inf')})
    fixed = sched.submit([7, 8], 6, allowed=[3, 4])
    assert collect(plain)[0] == greedy(table[0], 8, 6)
    assert collect(other)[0] == greedy(table[2], 8, 6)
    assert first not in collect(banned)[0]
    assert set(collect(fixed)[0]) <= {3, 4}
    again = [sched.submit([7, 8], 6) for _ in range(4)]  # the slots' rules and adapters left with their requests
    assert all(collect(r)[0] == greedy(table[0], 8, 6) for r in again)


def test_penalties_stop_a_loop(serve):
    sched = serve(2, 50)
    for t in range(50):
        sched.decoder.table[0, t, 5] = 50.0
        sched.decoder.table[0, t, 6] = 49.0
    assert collect(sched.submit([1], 4))[0] == [5, 5, 5, 5]
    assert collect(sched.submit([1], 4, frequency_penalty=0.6))[0] == [5, 5, 6, 5]
    assert collect(sched.submit([1], 4, presence_penalty=2.0))[0] == [5, 6, 5, 5]
    assert collect(sched.submit([5], 2, repetition_penalty=1.5))[0] == [6, 5]
    assert collect(sched.submit([5], 2, presence_penalty=2.0))[0] == [5, 6]  # the prompt is not output


def test_a_grammar_is_asked_before_each_token(serve):
    sched = serve(2, 50)
    asked = []

    def grammar(output):
        asked.append(list(output))
        return None if len(output) == 3 else [10 + len(output)]

    tokens, done = collect(sched.submit([1, 2, 3], 4, allowed=grammar))
    assert tokens[:3] == [10, 11, 12] and done['reason'] == 'length'
    assert asked == [[], [10], [10, 11], [10, 11, 12]]


def test_a_request_without_a_token_left_ends_alone(serve):
    sched = serve(2, 50)
    fine = sched.submit([4], 5)
    tokens, done = collect(sched.submit([4], 5, allowed=lambda output: [9] if not output else []))
    assert tokens == [9] and done['reason'] == 'exhausted'
    assert collect(fine)[0] == greedy(sched.decoder.table[0], 4, 5)


@pytest.mark.parametrize('grammar', [lambda output: 1 // 0, lambda output: [50], lambda output: np.zeros(7, bool)])
def test_a_failing_grammar_ends_its_request_alone(serve, grammar):
    sched = serve(2, 50)
    fine = sched.submit([4], 5)
    tokens, done = collect(sched.submit([4], 5, allowed=grammar))
    assert tokens == [] and done['reason'] == 'error' and done['error']
    assert collect(fine)[0] == greedy(sched.decoder.table[0], 4, 5)
    assert sched.status()['error'] is None and sched.status()['active_requests'] == 0


def test_an_adapter_unloaded_before_admission_ends_its_request_alone(serve):
    sched = serve(1, 50, slots=1)
    hold = sched.decoder.adapters.loaded
    with sched.lock:  # the worker admits after this block
        req = sched.submit([4], 3, adapter=0)
        hold[0] = False
    assert collect(req)[1]['reason'] == 'error'
    assert collect(sched.submit([4], 3))[0] == greedy(sched.decoder.table[0], 4, 3)


def test_sampling_keeps_to_the_mask(serve):
    sched = serve(1, 50)
    tokens, _ = collect(sched.submit([4], 20, temperature=2.0, seed=5, allowed=[3, 30, 31]))
    assert set(tokens) <= {3, 30, 31} and len(set(tokens)) > 1
    assert collect(sched.submit([4], 20, temperature=2.0, seed=5, allowed=[3, 30, 31]))[0] == tokens


def test_submit_refusals(serve):
    sched = serve(1, 50, slots=2)
    sched.decoder.adapters.loaded[1] = False
    bad = [dict(adapter=2), dict(adapter=-1), dict(adapter=1), dict(adapter=True), dict(repetition_penalty=0),
           dict(repetition_penalty=-1.0), dict(repetition_penalty=float('nan')), dict(presence_penalty='1'),
           dict(frequency_penalty=float('inf')), dict(frequency_penalty=1e60), dict(logit_bias={50: 1.0}),
           dict(logit_bias={-1: 1.0}), dict(logit_bias={True: 1.0}), dict(logit_bias={1: float('inf')}),
           dict(logit_bias={1: float('nan')}), dict(logit_bias={i: 1.0 for i in range(5)}), dict(allowed=[50]),
           dict(allowed=np.zeros(49, bool))]
    for change in bad:
        with pytest.raises(ValueError), np.errstate(over='ignore'):
            sched.submit([1], 2, **change)
    assert sched.status()['active_requests'] == 0
    plain = serve(1, 50, rules=False)
    for change in (dict(repetition_penalty=1.1), dict(logit_bias={1: 1.0}), dict(allowed=[1])):
        with pytest.raises(ValueError, match='no logit rules'):
            plain.submit([1], 2, **change)
    with pytest.raises(ValueError, match='adapter'):
        plain.submit([1], 2, adapter=0)
    assert len(collect(plain.submit([1], 2, repetition_penalty=1, logit_bias={}))[0]) == 2


@pytest.mark.parametrize('rules', [dict(frequency_penalty=-3e38, logit_bias={4: 3e38}),
                                   dict(presence_penalty=-3e38, logit_bias={4: 3e38})])
def test_a_request_whose_logits_overflow_ends_alone(serve, rules):
    """Finite rules can sum up to an infinite logit, which cannot be sampled: that request ends, the others go on."""
    sched = serve(2, 50)
    sched.decoder.table[0, 4, 4] = 50.0  # 4 says 4, so that its penalties count
    with np.errstate(over='ignore'):
        fine = sched.submit([7, 8], 6)
        tokens, done = collect(sched.submit([4], 6, temperature=1.0, **rules), timeout=5)
        assert done['reason'] == 'error' and 'nonfinite' in done['error']
        assert collect(fine, timeout=5)[0] == greedy(sched.decoder.table[0], 8, 6)
        assert sched.thread.is_alive() and sched.status()['active_requests'] == 0
        assert collect(sched.submit([7, 8], 6), timeout=5)[0] == greedy(sched.decoder.table[0], 8, 6)


def test_a_failing_admission_ends_its_request_alone(serve):
    """What the device or the decoder raises while a request is put into its slot ends that request."""
    from gpu.runtime import CUDAError
    sched = serve(2, 50)
    clear = sched.decoder.rules.clear

    def fails(b):
        raise CUDAError('glmvx_stream_synchronize', 700, 'as if')

    sched.decoder.rules.clear = fails
    tokens, done = collect(sched.submit([4], 3), timeout=5)
    assert tokens == [] and done['reason'] == 'error' and 'as if' in done['error']
    assert sched.thread.is_alive() and sched.status()['active_requests'] == 0 and 'as if' in sched.status()['error']
    sched.decoder.rules.clear = clear
    assert collect(sched.submit([4], 3), timeout=5)[0] == greedy(sched.decoder.table[0], 4, 3)


def test_a_failing_reset_of_an_idle_slot_ends_what_runs(serve):
    """An idle slot is emptied before its cache is full; where that fails, the requests of the step end with the
    device's error, and the worker stays."""
    from gpu.runtime import CUDAError
    sched = serve(2, 50)
    reset, failed = sched.decoder.reset_slot, []

    def fails(b):
        if b == 1:
            failed.append(b)
            raise CUDAError('glmvx_memset', 700, 'as if')
        reset(b)

    sched.decoder.reset_slot = fails
    for _ in range(2):  # slot 1 stays idle for more steps than a sequence has room for
        tokens, done = collect(sched.submit([4], 40), timeout=5)
    assert failed and done['reason'] == 'error' and 'as if' in done['error'] and len(tokens) < 40
    sched.decoder.reset_slot = reset
    assert collect(sched.submit([4], 3), timeout=5)[0] == greedy(sched.decoder.table[0], 4, 3)


@pytest.mark.parametrize('allowed', [lambda: iter([3, 4]), lambda: (t for t in [3, 4]), lambda: map(int, '34'),
                                     lambda: {3: 'x', 4: 'y'}.keys()])
def test_allowed_tokens_that_can_be_read_once(serve, allowed):
    sched = serve(2, 50)
    tokens, done = collect(sched.submit([7], 4, allowed=allowed()))
    assert len(tokens) == 4 and set(tokens) <= {3, 4} and done['reason'] == 'length'


@pytest.mark.parametrize('boolean', [False, True])
def test_a_mask_is_the_one_that_was_submitted(serve, boolean):
    """What the caller does to its array or list after submit() counts for nothing."""
    sched = serve(2, 50)
    mask = [3, 4]
    if boolean:
        mask = np.zeros(50, bool)
        mask[[3, 4]] = True
    with sched.lock:  # the worker admits after this block
        req = sched.submit([7], 4, allowed=mask)
        if boolean:
            mask[:] = False
            mask[9] = True
        else:
            mask[:] = [9]
    assert set(collect(req)[0]) <= {3, 4}


def test_numbers_beyond_every_range(serve):
    """Whole numbers that no float holds are refused, or stand for a ban, as floats beyond float32 do."""
    sched = serve(1, 50)
    big = 10 ** 400
    for change in (dict(repetition_penalty=big), dict(presence_penalty=-big), dict(frequency_penalty=big),
                   dict(logit_bias={1: big}), dict(logit_bias={1: 1e39}), dict(temperature=big)):
        with pytest.raises(ValueError):
            sched.submit([1], 2, **change)
    first = greedy(sched.decoder.table[0], 4, 1)[0]
    for ban in (-big, -1e39, float('-inf')):
        tokens, done = collect(sched.submit([4], 1, logit_bias={first: ban}))
        assert done['reason'] == 'length' and tokens != [first]


@pytest.mark.parametrize('change,message', [
    (dict(repetition=10 ** 400), 'finite'), (dict(presence=-10 ** 400), 'finite'), (dict(frequency=1e39), 'finite'),
    (dict(bias={3: 10 ** 400}), 'biases'), (dict(bias={3: float('nan')}), 'biases'), (dict(prompt=-1), 'prompt'),
    (dict(bias={1.5: 1.0}), 'biased tokens'), (dict(bias={'1': 1.0}), 'biased tokens'),
    (dict(bias={50: 1.0}), 'biased tokens'), (dict(bias={-1: 1.0}), 'biased tokens'),
    (dict(bias={i: 0.0 for i in range(5)}), 'more than 4'), (dict(repetition=0.0), 'positive')])
def test_rules_that_cannot_be_set(change, message):
    backend = QuietBackend()
    rules = LogitRules.__new__(LogitRules)
    rules.backend, rules.batch, rules.vocab, rules.max_bias, rules._bufs = backend, 2, 50, 4, {}
    with pytest.raises(ValueError, match=message):
        rules.set(1, **change)
    assert not backend.held  # nothing was put into place


def test_a_prompt_longer_than_any_history():
    """All that is fed is prompt, as with any prompt that is not yet at its end."""
    backend, put = QuietBackend(), {}
    rules = LogitRules.__new__(LogitRules)
    rules.backend, rules.batch, rules.vocab, rules.max_bias, rules._masked = backend, 2, 50, 4, [False, False]
    rules._put = lambda name, array, item, width=1: put.__setitem__(name, np.array(array))
    rules.set(1, prompt=10 ** 12, bias={np.int64(7): -10 ** 400})
    assert put['prompts'].tolist() == [2 ** 31 - 1] and put['prompts'].dtype == np.int32
    assert put['bias_ids'].tolist() == [7] and put['bias_values'].tolist() == [-np.inf]


@pytest.mark.parametrize('remembered,refused', [(7, True), (8, False), (9, False)])
def test_rules_remember_as_much_as_a_sequence_holds(remembered, refused):
    """Past its capacity a history stops growing and the penalties no longer follow the output: a decoder whose
    sequences are longer than that is refused."""
    from gpu.decoder import ResidentDecoder
    config = dict(CONFIG, index_n_heads=2, index_head_dim=16, index_topk=8, indexer_types=['full', 'full'])
    backend = NoDevice()
    rules = SimpleNamespace(backend=backend, batch=2, vocab=50, capacity=remembered)
    with pytest.raises(ValueError if refused else Exception) as raised:
        ResidentDecoder(backend, config, None, batch=2, capacity=8, rules=rules)
    assert ('histories' in str(raised.value)) == refused


def test_a_sequence_that_nothing_is_left_to_stays_at_its_end():
    """generate() goes on with the others; the ended row keeps -1 whatever its later steps would choose."""
    from gpu.decoder import ResidentDecoder
    dec = ResidentDecoder.__new__(ResidentDecoder)
    dec.B, steps, choices = 3, [], [[5, 6, 7], [5, -1, 8], [-1, 3, 9], [4, -1, 2]]
    dec.reset = dec.check = lambda: None
    dec.set_tokens, dec.step = lambda tokens: None, lambda: steps.append('step')
    dec.read_tokens = lambda: np.array(choices[steps.count('step') - 1], np.int32)
    out, _ = dec.generate([[1], [2], [3]], 4)
    assert out.tolist() == [[5, 5, -1, -1], [6, -1, -1, -1], [7, 8, 9, 2]]


@pytest.mark.parametrize('how', ['length', 'exhausted', 'cancelled', 'error'])
def test_a_finished_request_leaves_nothing_in_its_slot(serve, how):
    """An idle slot is stepped with the others: it reads no adapter's weights, no mask and no history any more."""
    sched = serve(2, 50, slots=2)
    dec = sched.decoder
    if how == 'error':
        allowed = lambda output: 1 // 0 if output else None
    else:
        allowed = (lambda output: [] if output else [3]) if how == 'exhausted' else [3, 4]
    req = sched.submit([4], 30, adapter=1, frequency_penalty=0.5, logit_bias={7: 2.0}, allowed=allowed)
    if how == 'cancelled':
        req.events.get(timeout=5)
        sched.cancel(req)
    assert collect(req, timeout=5)[1]['reason'] in (how, 'length')
    assert dec.adapter == [None, None]
    clean = HostRules(1, 50).rows[0]
    assert [dict(row, history=[]) for row in dec.rules.rows] == [clean, clean]


def test_a_slot_that_cannot_be_vacated_is_noted(serve):
    sched = serve(1, 50, slots=1)
    put = sched.decoder.set_adapter

    def fails(b, slot=None):
        if slot is None:
            raise RuntimeError('as if')
        put(b, slot)

    sched.decoder.set_adapter = fails
    tokens, done = collect(sched.submit([4], 3, adapter=0), timeout=5)
    assert len(tokens) == 3 and done['reason'] == 'length' and sched.status()['error'] == 'as if'
    sched.decoder.set_adapter = put
    assert collect(sched.submit([4], 3), timeout=5)[0] == greedy(sched.decoder.table[0], 4, 3)


def test_a_slot_is_empty_before_its_weights_change():
    """Whoever compares a slot's load before and after a step sees every change that the step may have met."""
    backend = QuietBackend()
    bank = bank_without_device()
    seen = []
    buffer = lambda: SimpleNamespace(ptr=0, upload=lambda *args: seen.append(list(bank.loaded)))
    bank.backend, bank._stacks = backend, {'a': tuple(buffer() for _ in range(4))}
    weights = {'a': (np.zeros((1, 4)), np.zeros((6, 1)))}
    bank.load(0, weights)
    first = bank.loaded[0]
    bank.load(1, weights)
    assert first and bank.loaded[0] == first and bank.loaded[1] not in (False, first)
    seen.clear()
    bank.load(0, weights)
    assert bank.loaded[0] not in (False, first, bank.loaded[1]) and seen and not any(s[0] for s in seen)
    seen.clear()
    bank.unload(1)
    assert not bank.loaded[1] and seen and not any(s[1] for s in seen)


def test_an_adapter_replaced_before_admission_ends_its_request_alone(serve):
    """A request runs with the adapter that was there when it was submitted, not with what its slot holds later."""
    sched = serve(2, 50, slots=1)
    loaded = sched.decoder.adapters.loaded
    loaded[0] = 11
    with sched.lock:  # the worker admits after this block
        req, fine = sched.submit([4], 3, adapter=0), sched.submit([4], 3)
        loaded[0] = 12
    tokens, done = collect(req, timeout=5)
    assert tokens == [] and done['reason'] == 'error' and 'replaced' in done['error']
    assert collect(fine, timeout=5)[0] == greedy(sched.decoder.table[0], 4, 3)
    assert collect(sched.submit([4], 3, adapter=0), timeout=5)[0] == greedy(sched.decoder.table[1], 4, 3)


@pytest.mark.parametrize('left', [False, 12])
@pytest.mark.parametrize('prompt', [1, 9])
def test_an_adapter_replaced_while_it_is_used_ends_its_request_alone(serve, left, prompt):
    """No token comes from a step that a load or an unload may have met, be it in the prompt."""
    sched = serve(2, 50, slots=1)
    loaded, step, steps = sched.decoder.adapters.loaded, sched.decoder.step, []
    loaded[0] = 11

    def meets_a_load():
        steps.append(len(steps))
        if len(steps) == 5:
            loaded[0] = left
        step()

    sched.decoder.step = meets_a_load
    with sched.lock:
        req, fine = sched.submit([4] * prompt, 20, adapter=0), sched.submit([4], 8)
    tokens, done = collect(req, timeout=5)
    assert done['reason'] == 'error' and 'replaced' in done['error']
    assert tokens == greedy(sched.decoder.table[1], 4, 4 if prompt == 1 else 0)
    assert collect(fine, timeout=5)[0] == greedy(sched.decoder.table[0], 4, 8)
    assert sched.status()['error'] is None


class HeldLock:
    """An RLock that knows how deep it is held."""

    def __init__(self):
        import threading
        self.lock, self.depth = threading.RLock(), 0

    def __enter__(self):
        self.lock.acquire()
        self.depth += 1

    def __exit__(self, *exc):
        self.depth -= 1
        self.lock.release()


def test_banks_and_rules_are_made_and_closed_outside_captures(monkeypatch):
    """What they issue on the stream (and their memory's release) would join or end another thread's capture: all of
    it holds the device's lock.  So does the capture of one layer's attention."""
    from gpu import decoder
    from gpu import runtime as rt
    backend = QuietBackend()
    backend.device.lock = HeldLock()
    backend.lib = SimpleNamespace(glmvx_lora_workspace_bytes=lambda *args: 64)

    class Buffer:
        ptr = 0

        def __init__(self, nbytes):
            backend._note()

        def upload(self, *args):
            backend._note()

        close = upload

    monkeypatch.setattr(rt, 'DeviceBuffer', Buffer)
    monkeypatch.setattr(rt, 'call', lambda name, *args: backend._note())
    bank = AdapterBank(backend, {'a': (6, 4), 'b': (4, 4)}, 2, 3)
    rules = LogitRules(backend, 2, 50, 8)
    assert len(backend.held) >= 40 and all(backend.held)
    backend.held.clear()
    bank.close()
    rules.close()
    assert len(backend.held) >= 19 and all(backend.held)
    backend.held.clear()
    dec = decoder.ResidentDecoder.__new__(decoder.ResidentDecoder)
    dec.backend, dec.layers, dec.n, dec.x, dec.hidden, dec.eps, dec._bufs = backend, [{'in_norm': 0}], 0, 0, 4, 0, []
    dec._rmsnorm = dec._attention = backend._note
    monkeypatch.setattr(rt, 'Graph', lambda stream: SimpleNamespace(begin=backend._note, end=backend._note))
    dec.attention_graph()
    assert backend.held == [True] * 4 and backend.device.lock.depth == 0


def test_two_loads_of_one_slot_do_not_mix():
    """The slot holds one of the two adapters as a whole, and an unload between the two does not empty half of it."""
    import threading
    import time
    bank, order = bank_without_device(), []
    bank.backend, bank.shapes = QuietBackend(), {n: (6, 4) for n in 'abcd'}
    bank._stacks = {n: 'ABrs' for n in bank.shapes}

    def put(buf, array, offset):
        order.append(threading.current_thread().name)
        time.sleep(0.002)

    bank._put = put
    weights = {n: (np.ones((1, 4)), np.ones((6, 1))) for n in bank.shapes}
    threads = [threading.Thread(target=bank.load, args=(0, weights), name=f'load {i}') for i in range(2)]
    threads.append(threading.Thread(target=bank.unload, args=(0,), name='unload'))
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join(10)
    assert len(order) == 2 * (4 + 16) + 4
    assert sum(a != b for a, b in zip(order, order[1:])) == 2, order


@pytest.mark.parametrize('scale', [1e39, -1e39, pytest.param(10 ** 400, id='10^400'), float('nan'),
                                   float('-inf')])
def test_scales_beyond_float32_are_refused(scale):
    with pytest.raises(ValueError, match='scale must be finite'):
        bank_without_device().load(0, {}, scale)


@pytest.mark.parametrize('change', [dict(slots=(1 << 24) + 1), dict(shapes={'a': ((1 << 22) + 1, 4)}),
                                    dict(shapes={'a': (4, (1 << 22) + 1)})])
def test_banks_that_no_call_takes_are_refused(change):
    args = dict(shapes={'a': (4, 4)}, slots=2, max_rank=4)
    args.update(change)
    with pytest.raises(ValueError, match='at most'):
        AdapterBank(NoDevice(), **args)


def test_a_row_without_a_finite_logit_ends_its_request_alone(serve):
    """A decoder with rules chooses -1 there for a request without rules too: no token, and nothing to feed."""
    sched = serve(2, 50)
    sched.decoder.table[0, 4, :] = -np.inf
    sched.decoder.table[0, 7, 7] = 50.0
    with sched.lock:
        req, fine = sched.submit([4], 5), sched.submit([7], 5)
    tokens, done = collect(req, timeout=5)
    assert tokens == [] and done['reason'] == 'error'
    assert collect(fine, timeout=5)[0] == [7] * 5
    assert sched.status()['error'] is None
