"""The resident decoder and the scheduler with adapters and logit rules: a small
all-F32 GLM-MoE-DSA model (dense MLPs), whose merged weights W + s B A are the
check of the adapters and whose plain logits are the check of the rules."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

CONFIG = dict(num_hidden_layers=2, hidden_size=128, num_attention_heads=4, q_lora_rank=64, kv_lora_rank=32,
              qk_nope_head_dim=16, qk_rope_head_dim=8, v_head_dim=16, intermediate_size=192, vocab_size=300,
              index_n_heads=4, index_head_dim=16, index_topk=64, mlp_layer_types=['dense', 'dense'],
              indexer_types=['full', 'full'], rms_norm_eps=1e-5, rope_parameters={'rope_theta': 10000},
              eos_token_id=[])
PROMPTS = [[3, 250, 17, 17], [9, 9, 120, 44], [200, 1, 2, 299]]


class Source:
    """Random F32 weights, with optional (A, B, scale) changes merged in."""

    def __init__(self, changes=None, seed=5):
        from gpu.adapters import projection_shapes
        c, rng = CONFIG, np.random.default_rng(seed)
        H = c['hidden_size']
        self.dense, self.packed = {}, {}

        def matrix(name, rows, cols, scale=1.0):
            return (scale * rng.normal(size=(rows, cols)) / np.sqrt(cols)).astype(np.float32)

        self.dense['model.embed_tokens.weight'] = rng.normal(size=(c['vocab_size'], H)).astype(np.float32)
        self.packed['lm_head'] = matrix('lm_head', c['vocab_size'], H, 3.0)
        self.dense['model.norm.weight'] = np.ones(H, np.float32)
        for name, (rows, cols) in sorted(projection_shapes(c).items()):
            self.packed[name] = matrix(name, rows, cols)
        for i in range(c['num_hidden_layers']):
            p = f'model.layers.{i}'
            a = p + '.self_attn'
            for name, n in ((p + '.input_layernorm', H), (p + '.post_attention_layernorm', H),
                            (a + '.q_a_layernorm', c['q_lora_rank']), (a + '.kv_a_layernorm', c['kv_lora_rank']),
                            (a + '.indexer.k_norm', c['index_head_dim'])):
                self.dense[name + '.weight'] = (1 + 0.1 * rng.normal(size=n)).astype(np.float32)
            self.dense[a + '.indexer.k_norm.bias'] = np.zeros(c['index_head_dim'], np.float32)
            heads = c['num_attention_heads'] * (c['qk_nope_head_dim'] + c['v_head_dim'])
            self.dense[a + '.kv_b_proj.weight'] = matrix('kv_b', heads, c['kv_lora_rank'])
            self.packed[a + '.indexer.wq_b'] = matrix('wq_b', c['index_n_heads'] * c['index_head_dim'],
                                                      c['q_lora_rank'])
            self.packed[a + '.indexer.wk'] = matrix('wk', c['index_head_dim'], H)
            self.packed[a + '.indexer.weights_proj'] = matrix('w', c['index_n_heads'], H)
        for name, (a, b) in (changes or {}).items():
            w = self.packed[name].astype(np.float64)
            self.packed[name] = (w + SCALE * b.astype(np.float64) @ a.astype(np.float64)).astype(np.float32)

    def packed_tensor(self, name):
        w = self.packed[name.removesuffix('.weight')]  # KeyError for what is dense
        return w.reshape(-1).view(np.uint8), 0, w.shape

    def dense_tensor(self, name):
        return self.dense[name]


SCALE = 1.5


def adapter(seed, names, rank):
    from gpu.adapters import projection_shapes
    shapes, rng = projection_shapes(CONFIG), np.random.default_rng(seed)
    return {name: ((rng.normal(size=(rank, shapes[name][1])) / np.sqrt(shapes[name][1])).astype(np.float32),
                   (0.3 * rng.normal(size=(shapes[name][0], rank)) / np.sqrt(rank)).astype(np.float32))
            for name in names}


def all_names():
    from gpu.adapters import projection_shapes
    return list(projection_shapes(CONFIG))


def decoder(backend, source=None, **kwargs):
    from gpu.decoder import ResidentDecoder
    return ResidentDecoder(backend, CONFIG, source or Source(), batch=len(PROMPTS), capacity=40, **kwargs)


def run(dec, steps=6):
    """Logits [steps][B][vocab] while the prompts and then fixed tokens are fed."""
    dec.reset()
    out = []
    for s in range(steps):
        dec.set_tokens([p[s] if s < len(p) else 10 * s + b for b, p in enumerate(PROMPTS)])
        dec.step()
        out.append(dec.read_logits())
    dec.check()
    return np.stack(out)


@pytest.fixture(scope='module')
def plain_logits(gpu_backend):
    dec = decoder(gpu_backend)
    try:
        return run(dec)
    finally:
        dec.close()


def test_each_sequence_runs_with_its_own_adapter(gpu_backend, plain_logits):
    """Rows with adapter 0, none, and 2 equal the rows of models with those
    changes merged into their weights.  Both run in f32; the longest sums have
    192 products (off by at most 192 * 2^-24 = 1.2e-5 of their absolute terms),
    ten projections and two attentions deep: 3e-4 of the row's norm covers the
    sum of the layers' worst cases."""
    from gpu.adapters import AdapterBank, projection_shapes
    first, third = adapter(1, all_names(), 8), adapter(2, all_names()[::2], 3)
    bank = AdapterBank(gpu_backend, projection_shapes(CONFIG), slots=4, max_rank=8, kind=0, max_tokens=len(PROMPTS))
    bank.load(0, first, SCALE)
    bank.load(2, third, SCALE)
    dec = decoder(gpu_backend, adapters=bank)
    merged = [decoder(gpu_backend, Source(first)), None, decoder(gpu_backend, Source(third))]
    try:
        assert run(dec).tobytes() == plain_logits.tobytes()  # no sequence has one yet: nothing changed
        dec.set_adapter(0, 0)
        dec.set_adapter(2, 2)
        got = run(dec)
        for b, model in enumerate(merged):
            want = (plain_logits if model is None else run(model))[:, b]
            off = np.linalg.norm(got[:, b] - want, axis=-1) / np.linalg.norm(want, axis=-1)
            assert (off <= (0 if model is None else 3e-4)).all(), (b, off)
            if model is not None:
                assert (np.linalg.norm(want - plain_logits[:, b], axis=-1) > 0.05 * np.linalg.norm(want, axis=-1)).all()
        # the captured step follows what is loaded: adapter 0 replaced by 2's weights, 2 dropped
        bank.load(0, third, SCALE)
        bank.unload(2)
        again = run(dec)
        want = run(merged[2])
        off = np.linalg.norm(again[:, 0] - want[:, 0], axis=-1) / np.linalg.norm(want[:, 0], axis=-1)
        assert (off <= 3e-4).all()
        assert again[:, 1:].tobytes() == plain_logits[:, 1:].tobytes()
        dec.set_adapter(0)
        assert run(dec).tobytes() == plain_logits.tobytes()
        with pytest.raises(ValueError, match='loaded'):
            dec.set_adapter(0, 2)
        with pytest.raises(ValueError, match='slot outside'):
            dec.set_adapter(3, 0)
    finally:
        for d in [dec] + [m for m in merged if m]:
            d.close()
        bank.close()


@pytest.mark.parametrize('kind,step', [(1, 2.0**-11), (30, 2.0**-8)])
def test_stored_kinds(gpu_backend, plain_logits, kind, step):
    """F16 and BF16 banks hold each weight rounded once, off by at most `step` of
    itself, or below the smallest normal F16 by half its steps' 2^-24: the
    decoder equals the merged model of the rounded weights (the bound above)."""
    from gpu.adapters import AdapterBank, projection_shapes, to_kind
    change = adapter(3, all_names(), 5)

    def rounded(v):
        s = to_kind(v, kind)
        w = s.astype(np.float32) if kind == 1 else (s.astype(np.uint32) << 16).view(np.float32)
        assert np.all(np.abs(w - v) <= step * np.abs(v) + 2.0**-25)
        return w

    bank = AdapterBank(gpu_backend, projection_shapes(CONFIG), slots=1, max_rank=8, kind=kind, max_tokens=64)
    bank.load(0, change, SCALE)
    dec = decoder(gpu_backend, adapters=bank)
    model = decoder(gpu_backend, Source({n: (rounded(a), rounded(b)) for n, (a, b) in change.items()}))
    try:
        for b in range(len(PROMPTS)):
            dec.set_adapter(b, 0)
        got, want = run(dec), run(model)
        assert (np.linalg.norm(got - want, axis=-1) <= 3e-4 * np.linalg.norm(want, axis=-1)).all()
    finally:
        dec.close()
        model.close()
        bank.close()


def test_an_adapter_loaded_while_the_step_is_captured(gpu_backend, plain_logits):
    """Another thread's load waits for the capture's end: the graph holds the step alone, the adapter is there after."""
    import threading
    import time
    from gpu.adapters import AdapterBank, projection_shapes
    bank = AdapterBank(gpu_backend, projection_shapes(CONFIG), slots=1, max_rank=4, kind=0, max_tokens=len(PROMPTS))
    weights = adapter(3, all_names(), 4)
    loader = threading.Thread(target=bank.load, args=(0, weights, SCALE))
    dec = decoder(gpu_backend, adapters=bank)
    launches = dec._step_launches

    def captured():
        loader.start()
        time.sleep(0.3)
        assert loader.is_alive() and not bank.loaded[0]
        launches()

    dec._step_launches = captured
    try:
        assert run(dec).tobytes() == plain_logits.tobytes()
        loader.join(10)
        assert bank.loaded[0]
        dec.set_adapter(1, 0)
        got = run(dec)
        assert run(dec).tobytes() == got.tobytes()
        assert np.delete(got, 1, axis=1).tobytes() == np.delete(plain_logits, 1, axis=1).tobytes()
        assert (np.linalg.norm(got[:, 1] - plain_logits[:, 1], axis=-1) > 0.01).all()
    finally:
        dec.close()
        bank.close()


def test_decoder_refuses_what_does_not_fit(gpu_backend):
    from gpu.adapters import AdapterBank
    from gpu.rules import LogitRules
    for shapes, tokens, message in (({'model.layers.0.self_attn.q_a_proj': (64, 64)}, 64, 'not a projection'),
                                    ({'model.layers.5.self_attn.q_a_proj': (64, 128)}, 64, 'not a projection'),
                                    ({'model.layers.0.self_attn.q_a_proj': (64, 128)}, 2, 'fewer')):
        bank = AdapterBank(gpu_backend, shapes, 1, 4, max_tokens=tokens)
        with pytest.raises(ValueError, match=message):
            decoder(gpu_backend, adapters=bank)
        with pytest.raises(ValueError, match='more tokens'):
            bank.add(next(iter(shapes)), 0, 0, 0, tokens + 1)
        bank.close()
    rules = LogitRules(gpu_backend, 2, CONFIG['vocab_size'], 8)
    with pytest.raises(ValueError, match='rules'):
        decoder(gpu_backend, rules=rules)
    rules.close()


def expected(row, history, prompt, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
    """The rules in f32, one rounding an operation."""
    l = row.copy()
    f = np.float32
    for t in set(history):
        l[t] = l[t] / f(repetition) if l[t] > 0 else l[t] * f(repetition)
    said = history[prompt:]
    for t in set(said):
        l[t] = l[t] - f(said.count(t)) * f(frequency) - f(presence)
    for t, v in (bias or {}).items():
        l[t] += f(v)
    if allowed is not None:
        keep = np.zeros(len(l), bool)
        keep[list(allowed)] = True
        l[~keep] = -np.inf
    return l


def test_rules_in_the_captured_step(gpu_backend, plain_logits):
    from gpu.rules import LogitRules
    rules = LogitRules(gpu_backend, len(PROMPTS), CONFIG['vocab_size'], capacity=40, max_bias=8)
    dec = decoder(gpu_backend, rules=rules)
    sets = [dict(prompt=4, repetition=1.3, presence=0.5, frequency=0.25),
            dict(prompt=2, repetition=0.7, frequency=-0.5, bias={9: -np.inf, 120: 30.0, 7: -1.5},
                 allowed=range(0, 300, 3)),
            {}]
    try:
        assert run(dec).tobytes() == plain_logits.tobytes()  # rules that say nothing
        for b, s in enumerate(sets):
            rules.set(b, **s)
        dec.reset()
        fed = [[] for _ in PROMPTS]
        for s in range(6):
            tokens = [p[s] if s < len(p) else 10 * s + b for b, p in enumerate(PROMPTS)]
            dec.set_tokens(tokens)
            dec.step()
            logits, chosen = dec.read_logits(), dec.read_tokens()
            for b, t in enumerate(tokens):
                fed[b].append(t)
                want = expected(plain_logits[s, b], fed[b], **{'prompt': 0, **sets[b]})
                assert np.array_equal(logits[b], want), (s, b)
                assert chosen[b] == int(np.argmax(want))
        assert [rules.history(b).tolist() for b in range(3)] == fed
        rules.allow(1, [])
        rules.allow(0, [5, 6])
        dec.set_tokens([1, 2, 3])
        dec.step()
        assert dec.read_tokens()[1] == -1 and dec.read_tokens()[0] in (5, 6)
        dec.reset_slot(0)
        assert rules.history(0).size == 0 and rules.history(1).size == 7
        dec.check()
    finally:
        dec.close()
        rules.close()


def test_scheduler_serves_different_users_at_once(gpu_backend):
    """Requests with and without adapters and rules in one batch say what each says alone."""
    from gpu.adapters import AdapterBank, projection_shapes
    from gpu.rules import LogitRules
    from gpu.serving import BatchScheduler, collect
    bank = AdapterBank(gpu_backend, projection_shapes(CONFIG), slots=2, max_rank=8, max_tokens=len(PROMPTS))
    bank.load(1, adapter(4, all_names(), 8), SCALE)
    rules = LogitRules(gpu_backend, len(PROMPTS), CONFIG['vocab_size'], capacity=40)
    dec = decoder(gpu_backend, adapters=bank, rules=rules)
    sched = BatchScheduler(dec)
    asks = [dict(), dict(adapter=1, frequency_penalty=0.5),
            dict(repetition_penalty=1.5, allowed=lambda out: range(100) if len(out) % 2 else range(100, 300))]
    try:
        alone = [collect(sched.submit(list(p), 8, **a)) for p, a in zip(PROMPTS, asks)]
        together = [sched.submit(list(p), 8, **a) for p, a in zip(PROMPTS, asks)]
        assert [collect(r)[0] for r in together] == [tokens for tokens, _ in alone]
        assert all(done['reason'] == 'length' for _, done in alone)
        assert [t < 100 for t in alone[2][0]] == [False, True] * 4
        assert collect(sched.submit(list(PROMPTS[1]), 8))[0] != alone[1][0]
        tokens, done = collect(sched.submit(list(PROMPTS[0]), 8, allowed=[]))
        assert tokens == [] and done['reason'] == 'exhausted'
        sampled, _ = collect(sched.submit(list(PROMPTS[0]), 8, temperature=1.5, seed=3, allowed=[7, 8, 9]))
        assert set(sampled) <= {7, 8, 9}
        assert sched.status()['error'] is None
    finally:
        sched.close()
        dec.check()
        dec.close()
        rules.close()
        bank.close()


def test_generate_with_a_sequence_that_nothing_is_left_to(gpu_backend):
    """The ended row returns -1 from then on, nothing is reported and the other rows say what they say without rules."""
    from gpu.rules import LogitRules
    plain = decoder(gpu_backend)
    rules = LogitRules(gpu_backend, len(PROMPTS), CONFIG['vocab_size'], capacity=40)
    dec = decoder(gpu_backend, rules=rules)
    try:
        want, logits = plain.generate(PROMPTS, 6, with_logits=True)
        rules.set(1, allowed=[])
        got, seen = dec.generate(PROMPTS, 6, with_logits=True)
        assert got[1].tolist() == [-1] * 6 and (seen[1] == -np.inf).all()
        assert np.array_equal(got[[0, 2]], want[[0, 2]])
        assert seen[[0, 2]].tobytes() == logits[[0, 2]].tobytes()
        rules.set(1, prompt=4, frequency=3e38, allowed=[7])  # twice 3e38 is infinite: 7 may be said two times
        got, _ = dec.generate(PROMPTS, 6)
        assert got[1].tolist() == [7, 7, -1, -1, -1, -1]
        assert np.array_equal(got[[0, 2]], want[[0, 2]])
        rules.set(1)
        assert np.array_equal(dec.generate(PROMPTS, 6)[0], want)
    finally:
        dec.close()
        plain.close()
        rules.close()


@pytest.mark.parametrize('max_tokens', [600, 4096])
def test_a_bank_of_prompts_takes_every_number_of_tokens(gpu_backend, max_tokens):
    """One workspace, made for the most tokens, holds fewer ones' call.  Against 64 bits: a sum of K products is off by
    (K / 8 + 40) * 2^-23 + 3 * 2^-22 of its absolute terms at most (test_gpu_lora.py says why), which is 29 * 2^-22 for
    96 and 24 * 2^-22 for 8: 64 * 2^-22 holds both and what they make of one another."""
    from gpu import runtime as rt
    from gpu.adapters import AdapterBank
    rng = np.random.default_rng(max_tokens)
    rows, cols, rank, slots = 40, 96, 8, 16
    bank = AdapterBank(gpu_backend, {'p': (rows, cols)}, slots, rank, kind=0, max_tokens=max_tokens)
    weights = [(rng.normal(size=(rank, cols)).astype(np.float32), rng.normal(size=(rows, rank)).astype(np.float32))
               for _ in range(slots)]
    for i, pair in enumerate(weights):
        bank.load(i, {'p': pair}, 0.5)
    x, y = rng.normal(size=(max_tokens, cols)).astype(np.float32), np.zeros((max_tokens, rows), np.float32)
    ids = rng.integers(-1, slots, max_tokens).astype(np.int32)
    bufs = [rt.DeviceBuffer(v.nbytes) for v in (y, x, ids)]
    want, mass = np.zeros((max_tokens, rows)), np.zeros((max_tokens, rows))
    for i, (a, b) in enumerate(weights):
        mine = ids == i
        want[mine] = 0.5 * (x[mine].astype(np.float64) @ a.T.astype(np.float64)) @ b.T.astype(np.float64)
        mass[mine] = 0.5 * (np.abs(x[mine]) @ np.abs(a.T)) @ np.abs(b.T)
    try:
        for buf, v in zip(bufs, (y, x, ids)):
            buf.upload(v, gpu_backend.stream.handle)
        for tokens in sorted({1, 64, 65, 100, max_tokens // 2 + 1, max_tokens - 96, max_tokens - 1, max_tokens}):
            bufs[0].upload(y, gpu_backend.stream.handle)
            bank.add('p', *(buf.ptr for buf in bufs), tokens)
            got = np.empty_like(y)
            bufs[0].download(got, gpu_backend.stream.handle)
            gpu_backend.stream.synchronize()
            assert (np.abs(got[:tokens] - want[:tokens]) <= 64 * 2.0 ** -22 * mass[:tokens]).all()
            assert not got[tokens:].any()
    finally:
        for buf in bufs:
            buf.close()
        bank.close()


def test_a_bank_made_while_the_step_is_captured(gpu_backend, plain_logits):
    """Another thread's new bank and rules wait for the capture's end, and so does their closing."""
    import threading
    import time
    from gpu.adapters import AdapterBank, projection_shapes
    from gpu.rules import LogitRules
    made = []

    def make():
        made.append(AdapterBank(gpu_backend, projection_shapes(CONFIG), slots=2, max_rank=4))
        made.append(LogitRules(gpu_backend, 2, 50, 8))

    maker = threading.Thread(target=make)
    closer = threading.Thread(target=lambda: [part.close() for part in made])
    decs = [decoder(gpu_backend), decoder(gpu_backend)]
    for dec, thread in zip(decs, (maker, closer)):
        launches = dec._step_launches

        def captured(thread=thread, launches=launches):
            thread.start()
            time.sleep(0.3)
            assert thread.is_alive()
            launches()

        dec._step_launches = captured
    try:
        for dec, thread in zip(decs, (maker, closer)):
            assert run(dec).tobytes() == plain_logits.tobytes()
            thread.join(10)
            assert not thread.is_alive() and len(made) == 2
            assert run(dec).tobytes() == plain_logits.tobytes()
    finally:
        for dec in decs:
            dec.close()


def test_a_served_adapter_that_is_replaced(gpu_backend):
    """Its request ends with an error, its neighbours say what they say alone, and the slot is left as a plain one."""
    import threading
    from gpu.adapters import AdapterBank, projection_shapes
    from gpu.rules import LogitRules
    from gpu.serving import BatchScheduler, collect
    bank = AdapterBank(gpu_backend, projection_shapes(CONFIG), slots=2, max_rank=8, max_tokens=len(PROMPTS))
    bank.load(0, adapter(5, all_names(), 8), SCALE)
    rules = LogitRules(gpu_backend, len(PROMPTS), CONFIG['vocab_size'], capacity=40)
    dec = decoder(gpu_backend, adapters=bank, rules=rules)
    sched = BatchScheduler(dec)
    said, loaded = threading.Event(), threading.Event()

    def pause(output):  # the worker waits here for the load, between two steps
        if len(output) == 3:
            said.set()
            loaded.wait(10)
        return None

    try:
        alone = collect(sched.submit(list(PROMPTS[0]), 12))[0]
        mine = collect(sched.submit(list(PROMPTS[1]), 12, adapter=0))[0]
        with sched.lock:
            fine, ends = sched.submit(list(PROMPTS[0]), 12), sched.submit(list(PROMPTS[1]), 12, adapter=0,
                                                                          allowed=pause)
        assert said.wait(10)
        bank.load(0, adapter(6, all_names(), 8), SCALE)
        loaded.set()
        tokens, done = collect(ends)
        assert done['reason'] == 'error' and 'replaced' in done['error'] and tokens == mine[:3]
        assert collect(fine)[0] == alone
        ids = np.zeros(len(PROMPTS), np.int32)
        dec.adapter_ids.download(ids, gpu_backend.stream.handle)
        gpu_backend.stream.synchronize()
        assert (ids == -1).all()
        assert collect(sched.submit(list(PROMPTS[1]), 12, adapter=0))[0] != mine
        bank.unload(0)
        with pytest.raises(ValueError, match='adapter'):
            sched.submit(list(PROMPTS[1]), 12, adapter=0)
        assert collect(sched.submit(list(PROMPTS[0]), 12))[0] == alone and sched.status()['error'] is None
    finally:
        loaded.set()
        sched.close()
        dec.check()
        dec.close()
        rules.close()
        bank.close()
