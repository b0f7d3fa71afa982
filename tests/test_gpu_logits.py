"""glmvx_logits_select against the formula: bit for bit in f32 with one
rounding per operation, and in 64 bits.

Tolerance against 64 bits: at most five roundings (the quotient or product,
c * frequency, two differences, the bias), each off by at most 2^-24 of a
value that is no larger than the sum of the absolute terms."""
import numpy as np
import pytest

from gpu import runtime as rt

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, rows, vocab, cap=0, lens=None, prompts=None, fed=None, penalties=False, bias=0, bias_lens=None,
                 masks=0, mask_rows=None, pad=0, out_pad=0, seed=0, share=None):
        rng = np.random.default_rng(seed)
        self.rows, self.vocab, self.cap, self.out_pad = rows, vocab, cap, out_pad
        self.logits = (3 * rng.normal(size=(rows, vocab + pad))).astype(np.float32)
        self.history = self.lens = self.prompts = self.fed = self.penalties = None
        self.bias_ids = self.bias_values = self.bias_lens = self.masks = self.mask_rows = None
        if cap:
            self.history = (rng.random((rows, cap)) ** 3 * vocab).astype(np.int32)
            self.lens = np.asarray(rng.integers(0, cap + 1, rows) if lens is None else lens, np.int32)
            if prompts is not False:
                self.prompts = np.asarray(self.lens // 2 if prompts is None else prompts, np.int32)
            if fed is not False:
                self.fed = np.asarray(rng.integers(0, vocab, rows) if fed is None else fed, np.int32)
        if penalties:
            self.penalties = np.stack([rng.uniform(0.8, 2, rows), rng.uniform(-1, 1, rows), rng.uniform(-1, 1, rows)],
                                      1).astype(np.float32)
        if bias:
            self.bias_ids = rng.integers(0, vocab, (rows, bias)).astype(np.int32)
            self.bias_values = (10 * rng.normal(size=(rows, bias))).astype(np.float32)
            self.bias_lens = np.asarray(rng.integers(0, bias + 1, rows) if bias_lens is None else bias_lens, np.int32)
        if masks:
            share = rng.random(masks) if share is None else share
            keep = rng.random((masks, (vocab + 31) // 32, 32)) < np.reshape(share, (-1, 1, 1))
            self.masks = (keep.astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)
            self.mask_rows = np.asarray(rng.integers(-1, masks, rows) if mask_rows is None else mask_rows, np.int32)

    def want(self, dtype):
        """(logits, selected, history, lens, sum of absolute terms) with every operation in `dtype`."""
        rows, vocab = self.rows, self.vocab
        out, mass = np.empty((rows, vocab), dtype), np.empty((rows, vocab))
        selected = np.empty(rows, np.int32)
        history = None if self.history is None else self.history.copy()
        lens = None if self.lens is None else self.lens.copy()
        with np.errstate(all='ignore'):
            for b in range(rows):
                l = self.logits[b, :vocab].astype(dtype)
                told = []
                if history is not None:
                    n = int(np.clip(lens[b], 0, self.cap))
                    told = history[b, :n].tolist()
                    if self.fed is not None and 0 <= self.fed[b] < vocab:
                        told.append(int(self.fed[b]))
                        if n < self.cap:
                            history[b, n], lens[b] = self.fed[b], n + 1
                m = np.abs(l.astype(np.float64))
                if self.penalties is not None:
                    rep, pres, freq = self.penalties[b].astype(dtype)
                    prompt = int(self.prompts[b]) if self.prompts is not None else 0
                    seen, count = np.zeros(vocab, bool), np.zeros(vocab, np.int64)
                    for i, v in enumerate(told):
                        if 0 <= v < vocab:
                            seen[v] = True
                            count[v] += i >= prompt
                    l = np.where(seen, np.where(l > 0, l / rep, l * rep), l)
                    m = np.abs(l.astype(np.float64)) + count * abs(float(freq)) + (count > 0) * abs(float(pres))
                    l = np.where(count > 0, l - count.astype(dtype) * freq - pres, l)
                if self.bias_ids is not None:
                    n = int(np.clip(self.bias_lens[b], 0, self.bias_ids.shape[1]))
                    for v, w in dict(zip(self.bias_ids[b, :n].tolist(), self.bias_values[b, :n])).items():
                        if 0 <= v < vocab:
                            l[v] += dtype(w)
                            m[v] += abs(float(w))
                if self.masks is not None and self.mask_rows[b] >= 0:
                    if self.mask_rows[b] < len(self.masks):
                        v = np.arange(vocab)
                        keep = (self.masks[self.mask_rows[b]][v // 32] >> (v % 32).astype(np.uint32)) & 1 > 0
                    else:
                        keep = np.zeros(vocab, bool)
                    l = np.where(keep, l, dtype(-np.inf))
                top = int(np.argmax(l))
                out[b], mass[b], selected[b] = l, m, -1 if l[top] == -np.inf else top
        return out, selected, history, lens, mass

    def run(self, backend, in_place=False, stream=None):
        s = stream or backend.stream
        keep = {}

        def up(v):
            if v is None:
                return None
            buf = rt.DeviceBuffer(v.nbytes)
            buf.upload(v, s.handle)
            keep[id(v)] = buf
            return buf.ptr

        logits = up(self.logits)
        stride = self.logits.shape[1] if in_place else self.vocab + self.out_pad
        host = self.logits.copy() if in_place else np.full((self.rows, stride), 7.0, np.float32)
        out = keep[id(self.logits)] if in_place else rt.DeviceBuffer(host.nbytes)
        if not in_place:
            out.upload(host, s.handle)
        sel = rt.DeviceBuffer(4 * self.rows)
        rt.call('glmvx_logits_select', sel.ptr, out.ptr, stride, logits, self.logits.shape[1], self.rows, self.vocab,
                up(self.fed), up(self.history), self.cap, up(self.lens), up(self.prompts), up(self.penalties),
                up(self.bias_ids), up(self.bias_values), up(self.bias_lens),
                0 if self.bias_ids is None else self.bias_ids.shape[1], up(self.masks), up(self.mask_rows),
                0 if self.masks is None else len(self.masks), s.handle)
        got = {'out': host, 'selected': np.empty(self.rows, np.int32)}
        out.download(got['out'], s.handle)
        sel.download(got['selected'], s.handle)
        for n in ('history', 'lens'):
            v = getattr(self, n)
            if v is not None:
                got[n] = np.empty_like(v)
                keep[id(v)].download(got[n], s.handle)
        s.synchronize()
        for buf in list(keep.values()) + [sel] + ([] if in_place else [out]):
            buf.close()
        return got

    def check(self, backend, in_place=False):
        before = self.logits.copy()
        got = self.run(backend, in_place)
        l, selected, history, lens, _ = self.want(np.float32)
        assert got['selected'].tolist() == selected.tolist()
        assert np.array_equal(got['out'][:, :self.vocab], l, equal_nan=True)
        rest = got['out'][:, self.vocab:]
        assert np.array_equal(rest, before[:, self.vocab:] if in_place else np.full_like(rest, 7.0))
        if history is not None:
            assert got['history'].tolist() == history.tolist() and got['lens'].tolist() == lens.tolist()
        exact, _, _, _, mass = self.want(np.float64)
        fine = np.isfinite(exact)
        assert (np.abs(got['out'][:, :self.vocab][fine] - exact[fine]) <= 5 * 2.0 ** -24 * mass[fine]).all()
        return got


@pytest.mark.parametrize('in_place', [False, True])
@pytest.mark.parametrize('rows,vocab,cap,bias,masks,pad', [
    (1, 1, 1, 1, 1, 0), (1, 31, 5, 2, 2, 0), (2, 32, 9, 0, 2, 1), (3, 33, 0, 3, 0, 0), (5, 512, 700, 40, 3, 4),
    (4, 8191, 64, 2047, 2, 0), (7, 8193, 33, 5, 4, 3), (17, 32003, 300, 31, 3, 13), (2, 154880, 3000, 300, 2, 0),
    (65, 1000, 50, 7, 5, 0), (1, 700001, 20, 3, 1, 0)])
def test_all_rules(gpu_backend, rows, vocab, cap, bias, masks, pad, in_place):
    Case(rows, vocab, cap, penalties=cap > 0, bias=bias, masks=masks, pad=pad, out_pad=2, seed=rows).check(
        gpu_backend, in_place)


@pytest.mark.parametrize('what', [
    dict(), dict(penalties=True, cap=40), dict(bias=9), dict(masks=2), dict(cap=40), dict(penalties=True),
    dict(penalties=True, cap=40, fed=False), dict(penalties=True, cap=40, prompts=False), dict(cap=40, masks=3)])
def test_each_rule_alone(gpu_backend, what):
    Case(6, 1234, seed=4, **what).check(gpu_backend)


def test_nothing_given_is_the_argmax(gpu_backend):
    case = Case(9, 5000, seed=2)
    got = case.check(gpu_backend)
    assert got['selected'].tolist() == case.logits.argmax(1).tolist()
    assert got['out'][:, :5000].tobytes() == case.logits.tobytes()


def test_history_edges(gpu_backend):
    """Empty and full histories, prompts longer than the history, fed tokens of no row, skipped ids, lengths
    outside the capacity."""
    case = Case(8, 300, cap=12, lens=[0, 12, 5, 0, 12, 3, -4, 40], prompts=[0, 12, 99, 3, -5, 3, 0, 6],
                fed=[5, 7, 9, 250, -1, -9, 8, 8], penalties=True, seed=6)
    case.history[2, :3] = [-1, 300, 2**31 - 1]
    case.history[5, 0] = -2**31
    got = case.run(gpu_backend)
    l, selected, history, lens, _ = case.want(np.float32)
    assert np.array_equal(got['out'][:, :300], l) and got['selected'].tolist() == selected.tolist()
    assert got['history'].tolist() == history.tolist()
    assert got['lens'][:6].tolist() == [1, 12, 6, 1, 12, 3]


def test_one_token_many_times(gpu_backend):
    """A history of one token, and every bias entry on one token: the count is whole, the last entry holds."""
    case = Case(3, 100, cap=5000, lens=[5000, 4999, 2500], prompts=[0, 2000, 2500], fed=[4, 4, 4], penalties=True,
                bias=2047, bias_lens=[2047, 1000, 0], seed=8)
    case.history[:] = 4
    case.bias_ids[:] = 4
    case.check(gpu_backend)


def test_rows_with_nothing_left(gpu_backend):
    """No allowed token, allowed tokens at -inf only, a ban by bias, a row of -inf: -1 and no other row touched."""
    case = Case(6, 200, bias=1, bias_lens=[0, 0, 1, 0, 0, 0], masks=3, mask_rows=[0, 1, 1, -1, 2, -1],
                share=[0.0, 0.0, 1.0], seed=9)
    case.masks[1, 0] = 1 << 7
    case.logits[1, 7] = -np.inf
    case.bias_ids[2], case.bias_values[2] = 7, -np.inf
    case.logits[3, :] = -np.inf
    case.logits[5, :] = np.finfo(np.float32).min
    got = case.check(gpu_backend)
    assert got['selected'].tolist() == [-1, -1, -1, -1, int(np.argmax(case.logits[4])), 0]


def test_what_is_not_finite(gpu_backend):
    """NaN and infinities: the first allowed NaN is taken, a masked one leaves no trace, -0.0 and 0.0 tie."""
    case = Case(6, 64, masks=1, mask_rows=[-1, 0, -1, -1, 0, -1], share=[1.0], seed=10)
    case.masks[0, 0] = ~np.uint32(1 << 20)
    case.logits[0, [20, 50]] = np.nan
    case.logits[1, 20], case.logits[1, 40] = np.nan, np.inf
    case.logits[2, [9, 33]] = np.inf
    case.logits[3, :] = -1
    case.logits[3, 30], case.logits[3, 40] = -0.0, 0.0
    case.logits[4, 20] = np.inf
    case.logits[5, [3, 60]] = 50.0
    got = case.check(gpu_backend)
    assert got['selected'][[0, 1, 2, 3, 5]].tolist() == [20, 40, 9, 30, 3]


@pytest.mark.parametrize('vocab', [100, 20000])
def test_bad_ids_are_reported(gpu_backend, vocab):
    """A fed token outside the vocabulary counts for nothing; a mask that is not there allows nothing."""
    gpu_backend.device.check_device_error()
    case = Case(2, vocab, cap=4, lens=[1, 1], fed=[vocab, 3], penalties=True, seed=11)
    case.check(gpu_backend)
    with pytest.raises(rt.CUDAError, match='device error word 3'):
        gpu_backend.device.check_device_error()
    got = Case(2, vocab, masks=2, mask_rows=[2, 1], share=[1.0, 1.0], seed=12).check(gpu_backend)
    assert got['selected'][0] == -1 and got['selected'][1] >= 0
    with pytest.raises(rt.CUDAError, match='device error word 3'):
        gpu_backend.device.check_device_error()


def test_the_mask_bits_behind_the_vocabulary_count_for_nothing(gpu_backend):
    case = Case(1, 70, masks=1, mask_rows=[0], share=[0.0], seed=13)
    case.masks[0, 2] = 0xffffffff << 6 & 0xffffffff
    assert case.check(gpu_backend)['selected'].tolist() == [-1]


def test_captured_steps_feed_themselves(gpu_backend):
    """selected is fed: replays of one captured call walk on, each choice joining the history."""
    rows, vocab, cap, steps = 3, 900, 6, 8
    case = Case(rows, vocab, cap=cap, lens=[0, 2, 6], prompts=[0, 1, 0], fed=[1, 2, 3], penalties=True, seed=14)
    case.penalties[:] = [1.3, 0.7, 2.5]
    s = gpu_backend.stream
    host = {n: getattr(case, n) for n in ('logits', 'fed', 'history', 'lens', 'prompts', 'penalties')}
    dev = {n: rt.DeviceBuffer(v.nbytes) for n, v in host.items()}
    out = rt.DeviceBuffer(4 * rows * vocab)
    g = rt.Graph(s)
    g.begin()
    try:
        rt.call('glmvx_logits_select', dev['fed'].ptr, out.ptr, vocab, dev['logits'].ptr, vocab, rows, vocab,
                dev['fed'].ptr, dev['history'].ptr, cap, dev['lens'].ptr, dev['prompts'].ptr, dev['penalties'].ptr,
                None, None, None, 0, None, None, 0, s.handle)
    finally:
        g.end()
    for n, v in host.items():
        dev[n].upload(v, s.handle)
    for _ in range(steps):
        g.launch()
        l, selected, case.history, case.lens, _ = case.want(np.float32)
        got = np.empty(rows, np.int32)
        dev['fed'].download(got, s.handle)
        s.synchronize()
        assert got.tolist() == selected.tolist()
        case.fed = selected
    left = np.empty_like(case.history)
    dev['history'].download(left, s.handle)
    s.synchronize()
    assert left.tolist() == case.history.tolist()
    g.close()
    for b in list(dev.values()) + [out]:
        b.close()


@pytest.mark.parametrize('rows,vocab,cap,bias', [(1, 700001, 100000, 3), (2, 400000, 60000, 2047), (3, 1300000, 8, 1)])
def test_vocabularies_that_go_in_passes(gpu_backend, rows, vocab, cap, bias):
    """Histories as long as the vocabulary's share of a CTA: the rules do not fit shared memory at once."""
    Case(rows, vocab, cap, lens=[cap, cap - 1, 0][:rows], penalties=True, bias=bias, masks=2,
         seed=vocab).check(gpu_backend)


@pytest.mark.parametrize('vocab', [4, 124, 128, 132, 2048, 2052, 6148])
def test_vocabularies_around_the_blocks(gpu_backend, vocab):
    """One block of tokens and its neighbours, whole groups of four and not, in rows beside one another."""
    for v in (vocab - 1, vocab):
        Case(5, v, cap=30, penalties=True, bias=4, masks=3, pad=4 if v == vocab else 1, seed=v).check(gpu_backend, True)


def test_many_rows(gpu_backend):
    """More rows than run at once, each with a CTA of its own."""
    Case(700, 1000, cap=12, penalties=True, bias=2, masks=4, seed=20).check(gpu_backend)


@pytest.mark.parametrize('vocab', [64, 63])
def test_a_ban_holds_whatever_the_logit_is(gpu_backend, vocab):
    """-inf as a bias is the end of a token, also of one whose logit is infinite or no number, by itself or by its
    penalties; with other biases those stay what the sum makes of them."""
    case = Case(4, vocab, cap=4, lens=[2, 2, 0, 0], prompts=[0, 0, 0, 0], fed=[9, 9, -1, -1], penalties=True, bias=2,
                bias_lens=[1, 1, 2, 2], seed=30)
    case.history[:, :] = 9
    case.penalties[:] = [1, 0, 0]
    case.penalties[0] = [1e-38, 0, 0]  # 30 / 1e-38
    case.penalties[1] = [1, 0, -3e38]  # three times
    case.bias_ids[:] = [9, 5]
    case.bias_values[:] = -np.inf
    case.bias_values[2, 1] = 1.0
    case.logits[:, 9], case.logits[2, 5] = 30.0, np.inf
    case.logits[3, 9], case.logits[3, 5] = np.nan, np.inf
    got = case.run(gpu_backend)
    assert (got['out'][:, 9] == -np.inf).all() and got['out'][2, 5] == np.inf and got['out'][3, 5] == -np.inf
    rest = np.delete(np.arange(vocab), [5, 9])
    assert np.array_equal(got['out'][:, rest], case.logits[:, rest])
    want = [int(np.argmax(np.where(np.arange(vocab) == 9, -np.inf, case.logits[b, :vocab]))) for b in (0, 1)]
    assert got['selected'][:3].tolist() == want + [5] and got['selected'][3] == rest[np.argmax(case.logits[3, rest])]
