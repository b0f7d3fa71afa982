"""glmvx_lora_add against the formula in 64 bits.

Tolerance: h = A x and y + s B h are sums of f32 products.  A chain of n
roundings is off by at most n * 2^-23 of the sum of the absolute terms (2^-24
a rounding; tensor cores may cut instead of rounding, which doubles it).  The
kernels add at least eight products per link of a chain, so a sum of K has at
most K / 8 links, plus 40 for joining the parts; an operand may stand as two
TF32 parts, off by 2^-22 of itself and, where both stand so, by another 2^-22
for the product of the small parts, so 3 * 2^-22 covers both."""
import numpy as np
import pytest

from gpu import runtime as rt

pytestmark = pytest.mark.gpu

KINDS = {0: (np.float32, 4), 1: (np.float16, 2), 30: (np.uint16, 2)}


def pack(kind, v):
    """v (f32) as the kind's storage, and the f64 values that storage stands for."""
    if kind == 30:  # BF16: the upper half of the f32 pattern
        bits = (np.ascontiguousarray(v, np.float32).view(np.uint32) >> 16).astype(np.uint16)
        return bits, (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    s = v.astype(KINDS[kind][0])
    return s, s.astype(np.float64)


class Case:
    """One call's host data; junk fills what the contract says is not read."""

    def __init__(self, tokens, rows, cols, adapters, max_rank, kind, ids=None, ranks=None, y_pad=0, x_pad=0, seed=0):
        rng = np.random.default_rng(seed)
        self.dims = (tokens, rows, cols, adapters, max_rank)
        self.kind = kind
        self.ids = np.asarray(rng.integers(-1, adapters, tokens) if ids is None else ids, np.int32)
        self.ranks = np.asarray(rng.integers(0, max_rank + 1, adapters) if ranks is None else ranks, np.int32)
        self.scales = rng.uniform(0.5, 2.0, adapters).astype(np.float32)
        self.x = rng.normal(size=(tokens, cols + x_pad)).astype(np.float32)
        self.y = rng.normal(size=(tokens, rows + y_pad)).astype(np.float32)
        a = (rng.normal(size=(adapters, max_rank, cols)) / np.sqrt(cols)).astype(np.float32)
        b = rng.normal(size=(adapters, rows, max_rank)).astype(np.float32)
        for i, r in enumerate(np.clip(self.ranks, 0, max_rank)):
            a[i, r:] = np.nan
            b[i, :, r:] = np.nan
        self.a, self.a64 = pack(kind, a)
        self.b, self.b64 = pack(kind, b)

    def want(self):
        """(y in 64 bits, how far each element may be off)."""
        tokens, rows, cols, adapters, max_rank = self.dims
        y = self.y[:, :rows].astype(np.float64)
        tol = np.zeros_like(y)
        for t in range(tokens):
            i = self.ids[t]
            if not 0 <= i < adapters:
                continue
            r = int(np.clip(self.ranks[i], 0, max_rank))
            x = self.x[t, :cols].astype(np.float64)
            a, b, s = self.a64[i, :r], self.b64[i, :, :r], float(self.scales[i])
            h, mass = a @ x, np.abs(a) @ np.abs(x)
            part = 3 * 2.0 ** -22
            h_off = mass * ((cols / 8 + 40) * 2.0 ** -23 + part)
            d_mass = np.abs(b) @ (np.abs(h) + h_off)
            tol[t] = s * (np.abs(b) @ h_off + d_mass * ((r / 8 + 40) * 2.0 ** -23 + part))
            y[t] += s * (b @ h)
            tol[t] += np.abs(y[t]) * 2.0 ** -24  # the sum with y
        return y, tol

    def run(self, backend, stream=None, repeat=1, offset=0):
        """The call on device copies; returns y with its padding.  `offset` shifts x, y, a and b by that many
        elements inside their buffers, off the 16-byte boundary."""
        lib, s = backend.lib, stream or backend.stream
        tokens, rows, cols, adapters, max_rank = self.dims
        need = lib.glmvx_lora_workspace_bytes(tokens, adapters, max_rank)
        keep, at = [], {}
        for name, v in (('x', self.x), ('y', self.y), ('a', self.a), ('b', self.b), ('ids', self.ids),
                        ('ranks', self.ranks), ('scales', self.scales)):
            shift = offset * v.itemsize if name in 'xyab' else 0
            buf = rt.DeviceBuffer(v.nbytes + shift + 16)
            buf.upload(v, s.handle, shift)
            keep.append(buf)
            at[name] = buf.ptr + shift
            if name == 'y':
                y_buf, y_shift = buf, shift
        ws = rt.DeviceBuffer(need)
        rt.call('glmvx_memset', ws.ptr, 0xff, need, s.handle)  # NaN: nothing of it may count
        for _ in range(repeat):
            rt.call('glmvx_lora_add', at['y'], self.y.shape[1], at['x'], self.x.shape[1], at['ids'], self.kind,
                    at['a'], at['b'], at['ranks'], at['scales'], tokens, rows, cols, adapters, max_rank, ws.ptr, need,
                    s.handle)
        out = np.empty_like(self.y)
        y_buf.download(out, s.handle, y_shift)
        s.synchronize()
        for buf in keep + [ws]:
            buf.close()
        return out

    def check(self, backend, **how):
        out = self.run(backend, **how)
        rows = self.dims[1]
        want, tol = self.want()
        off = np.abs(out[:, :rows].astype(np.float64) - want)
        assert (off <= tol).all(), (np.max(off / np.maximum(tol, 1e-300)), np.argwhere(off > tol)[:4])
        assert out[:, rows:].tobytes() == self.y[:, rows:].tobytes(), 'the padding behind the rows changed'
        ranks = np.clip(self.ranks, 0, self.dims[4])
        still = [t for t, i in enumerate(self.ids) if not 0 <= i < self.dims[3] or ranks[i] == 0]
        assert out[still].tobytes() == self.y[still].tobytes(), 'a row without an adapter changed'
        return out


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('tokens,rows,cols,adapters,max_rank', [
    (1, 1, 1, 1, 1), (1, 576, 6144, 2, 8), (2, 33, 31, 3, 3), (7, 130, 257, 4, 16), (8, 64, 64, 1, 17),
    (9, 1001, 515, 9, 13), (17, 96, 2048, 40, 64), (64, 256, 1024, 64, 16), (64, 512, 512, 1, 32),
    (65, 100, 100, 5, 100), (129, 72, 200, 2, 256), (300, 160, 96, 7, 24), (1000, 40, 56, 70, 5)])
def test_against_64_bits(gpu_backend, kind, tokens, rows, cols, adapters, max_rank):
    Case(tokens, rows, cols, adapters, max_rank, kind, seed=tokens + rows).check(gpu_backend)


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('y_pad,x_pad,offset', [(4, 8, 0), (3, 5, 0), (1, 0, 1), (0, 0, 3), (0, 4, 4)])
def test_strides_and_alignment(gpu_backend, kind, y_pad, x_pad, offset):
    Case(21, 136, 160, 4, 16, kind, y_pad=y_pad, x_pad=x_pad, seed=7).check(gpu_backend, offset=offset)
    Case(200, 136, 160, 4, 16, kind, y_pad=y_pad, x_pad=x_pad, seed=8).check(gpu_backend, offset=offset)


@pytest.mark.parametrize('ids', [[-1] * 12, [2] * 12, [0, 1, 2] * 4, [-7] + [1] * 11, [2] + [-1] * 11])
def test_spreads(gpu_backend, ids):
    Case(12, 300, 128, 3, 8, 30, ids=ids, ranks=[8, 5, 3]).check(gpu_backend)


def test_ranks_outside_the_bank_are_clamped(gpu_backend):
    Case(6, 64, 64, 3, 8, 1, ids=[0, 1, 2, 0, 1, 2], ranks=[-4, 99, 0]).check(gpu_backend)


@pytest.mark.parametrize('tokens', [5, 500])
def test_an_unknown_adapter_is_reported_and_its_row_stays(gpu_backend, tokens):
    ids = np.zeros(tokens, np.int32)
    ids[3] = 2
    case = Case(tokens, 64, 64, 2, 8, 30, ids=ids, ranks=[8, 8])
    gpu_backend.device.check_device_error()
    case.check(gpu_backend)
    with pytest.raises(rt.CUDAError, match='device error word 3'):
        gpu_backend.device.check_device_error()
    gpu_backend.device.check_device_error()


@pytest.mark.parametrize('tokens,kind', [(13, 30), (13, 0), (400, 1)])
def test_a_token_does_not_depend_on_the_others(gpu_backend, tokens, kind):
    """The same token alone-by-adapter, among others of its adapter, and shuffled: the same bits, every time."""
    case = Case(tokens, 96, 320, 5, 16, kind, ranks=[16, 7, 1, 16, 12], seed=3)
    out = case.run(gpu_backend)
    assert case.run(gpu_backend).tobytes() == out.tobytes()
    order = np.random.default_rng(1).permutation(tokens)
    case.ids, case.x, case.y = case.ids[order], case.x[order], case.y[order]
    assert case.run(gpu_backend).tobytes() == out[order].tobytes()
    others = case.ids != case.ids[0]
    case.ids[others] = -1
    alone = case.run(gpu_backend)
    assert alone[~others].tobytes() == out[order][~others].tobytes()


@pytest.mark.parametrize('tokens', [4, 300])
def test_what_is_not_finite_stays_in_its_row(gpu_backend, tokens):
    case = Case(tokens, 80, 96, 2, 8, 30, ids=np.arange(tokens) % 2, ranks=[8, 4])
    clean = case.run(gpu_backend)
    case.x[1, 5], case.x[2, 0], case.y[3, 7] = np.nan, np.inf, -np.inf
    out = case.run(gpu_backend)
    assert np.isnan(out[1]).all() and not np.isfinite(out[2]).any()
    assert out[3, 7] == -np.inf and np.array_equal(np.delete(out[3], 7), np.delete(clean[3], 7))
    rest = np.delete(np.arange(tokens), [1, 2, 3])
    assert out[rest].tobytes() == clean[rest].tobytes()


def test_calls_add_up_and_replay(gpu_backend):
    """Two calls in a row add twice; a captured call replays on what the buffers then hold, beside a call on
    another stream with its own workspace."""
    case = Case(10, 128, 256, 3, 8, 1, ranks=[8, 8, 8], seed=5)
    twice = case.run(gpu_backend, repeat=2)
    first = case.run(gpu_backend)
    step = first.astype(np.float64) - case.y
    assert np.allclose(twice - first.astype(np.float64), step, rtol=0, atol=8 * 2.0 ** -24 * np.abs(twice).max())
    s, other = gpu_backend.stream, rt.Stream()
    tokens, rows, cols, adapters, max_rank = case.dims
    need = gpu_backend.lib.glmvx_lora_workspace_bytes(tokens, adapters, max_rank)
    bufs = {n: rt.DeviceBuffer(v.nbytes) for n, v in (('x', case.x), ('y', case.y), ('z', case.y), ('a', case.a),
                                                      ('b', case.b), ('ids', case.ids), ('ranks', case.ranks),
                                                      ('scales', case.scales))}
    ws = [rt.DeviceBuffer(need), rt.DeviceBuffer(need)]

    def issue(y, w, stream):
        rt.call('glmvx_lora_add', bufs[y].ptr, rows, bufs['x'].ptr, cols, bufs['ids'].ptr, 1, bufs['a'].ptr,
                bufs['b'].ptr, bufs['ranks'].ptr, bufs['scales'].ptr, tokens, rows, cols, adapters, max_rank,
                ws[w].ptr, need, stream.handle)

    try:
        g = rt.Graph(s)
        g.begin()
        try:
            issue('y', 0, s)
        finally:
            g.end()
        for n in ('x', 'a', 'b', 'ids', 'ranks', 'scales'):
            bufs[n].upload(getattr(case, n), s.handle)
        bufs['y'].upload(case.y, s.handle)
        bufs['z'].upload(case.y, s.handle)
        s.synchronize()
        for _ in range(2):
            g.launch()
            issue('z', 1, other)
        s.synchronize()
        other.synchronize()
        for n in 'yz':
            got = np.empty_like(case.y)
            bufs[n].download(got)
            assert got.tobytes() == twice.tobytes()
        case.ids = np.full(tokens, -1, np.int32)  # the graph reads the ids when it runs
        bufs['ids'].upload(case.ids, s.handle)
        g.launch()
        s.synchronize()
        bufs['y'].download(got)
        assert got.tobytes() == twice.tobytes()
        g.close()
    finally:
        other.close()
        for b in list(bufs.values()) + ws:
            b.close()


def test_long_rows(gpu_backend):
    """The widths of a served model's projections, a decode batch and a prompt."""
    Case(64, 6144, 2048, 16, 16, 30, seed=1).check(gpu_backend)
    Case(3, 576, 6144, 2, 64, 1, seed=2).check(gpu_backend)
    Case(700, 576, 2048, 3, 32, 30, ids=np.sort(np.arange(700) % 3), seed=3).check(gpu_backend)


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('max_rank,cols,rows', [(8, 512, 256), (12, 520, 260), (20, 1000, 132), (24, 768, 64),
                                                (40, 64, 1028), (64, 2056, 8), (256, 264, 36), (48, 24, 4)])
def test_ranks_and_widths_on_both_sides_of_the_tiles(gpu_backend, kind, max_rank, cols, rows):
    """Ranks and widths that end inside a chunk, with vector loads and without, few and many tokens."""
    for tokens in (6, 70):
        Case(tokens, rows, cols, 3, max_rank, kind, ids=np.arange(tokens) % 4 - 1,
             ranks=[max_rank, max(1, max_rank // 2 + 1), 1], seed=tokens + cols).check(gpu_backend)


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('max_rank,cols,rows', [(1, 31, 5), (16, 512, 256), (19, 515, 130), (33, 1000, 132),
                                                (64, 64, 1028), (256, 264, 36)])
def test_few_tokens_in_one_launch_and_in_two(gpu_backend, kind, max_rank, cols, rows):
    """The number of tiles there may be (tokens, or an eighth of them and one an adapter) decides: from 19 on, two
    launches; both with ranks that differ and adapters that several tiles share."""
    for tokens, adapters in ((18, 40), (19, 40), (64, 3), (64, 90)):
        rng = np.random.default_rng(tokens + adapters)
        ids = np.where(rng.random(tokens) < 0.5, rng.integers(-1, 3, tokens), rng.integers(0, adapters, tokens))
        Case(tokens, rows, cols, adapters, max_rank, kind, ids=ids, seed=tokens + cols).check(gpu_backend)


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('offset', [0, 1, 2, 4])
@pytest.mark.parametrize('max_rank,cols,rows', [(12, 1028, 64), (14, 1026, 66), (15, 257, 63), (36, 516, 68),
                                                (37, 1025, 65), (60, 300, 4), (38, 10, 2), (3, 9, 1)])
def test_rows_on_every_boundary(gpu_backend, kind, offset, max_rank, cols, rows):
    """Rows that start on 8, 4 and 2 bytes, stacks that do not start on 4: what is read by the word stays inside the
    stack (its last adapter's last row is used) and what it brings along does not count (NaN behind the ranks)."""
    for tokens in (5, 70):
        Case(tokens, rows, cols, 3, max_rank, kind, ids=np.arange(tokens) % 3, ranks=[max_rank - 2, 1, max_rank],
             seed=tokens + cols).check(gpu_backend, offset=offset)
    Case(40, rows, cols, 30, max_rank, kind, ids=np.arange(40) % 30, seed=cols).check(gpu_backend, offset=offset)


@pytest.mark.parametrize('tokens,adapters,max_rank,cols,rows', [(1, 1, 16, 8192, 8192), (1, 1, 16, 8192, 8196),
                                                                (9, 2, 64, 4096, 64), (9, 2, 64, 4088, 8)])
def test_adapters_around_the_size_for_one_launch(gpu_backend, tokens, adapters, max_rank, cols, rows):
    Case(tokens, rows, cols, adapters, max_rank, 30, ids=np.arange(tokens) % adapters, ranks=[max_rank] * adapters,
         seed=rows).check(gpu_backend)


@pytest.mark.parametrize('kind', [0, 30])
def test_a_token_of_two_launches_does_not_depend_on_the_others(gpu_backend, kind):
    case = Case(40, 96, 320, 50, 16, kind, ids=np.arange(40) % 7, ranks=[16, 7, 1, 16, 12] * 10, seed=4)
    out = case.run(gpu_backend)
    case.ids[case.ids != 3] = -1
    alone = case.run(gpu_backend)
    assert alone[3::7].tobytes() == out[3::7].tobytes()


def test_many_adapters_and_many_tokens(gpu_backend):
    """More adapters than the plan counts in shared memory, more tokens than its threads keep."""
    Case(200, 8, 16, 5000, 2, 1, seed=1).check(gpu_backend)
    ids = np.random.default_rng(2).integers(-1, 3, 6000)
    Case(6000, 12, 16, 3, 4, 30, ids=ids, ranks=[4, 0, 3], seed=2).check(gpu_backend)
    Case(5000, 4, 8, 1, 1, 0, ids=np.zeros(5000), ranks=[1], seed=3).check(gpu_backend)


def test_a_captured_call_of_many_tokens_replays(gpu_backend):
    """The plan is made anew by each replay: ids written between two replays count in the second."""
    case = Case(300, 64, 128, 6, 8, 30, ranks=[8] * 6, seed=9)
    tokens, rows, cols, adapters, max_rank = case.dims
    s, other = gpu_backend.stream, case.ids[::-1].copy()
    need = gpu_backend.lib.glmvx_lora_workspace_bytes(tokens, adapters, max_rank)
    bufs = {n: rt.DeviceBuffer(getattr(case, n).nbytes) for n in ('x', 'y', 'a', 'b', 'ids', 'ranks', 'scales')}
    ws = rt.DeviceBuffer(need)
    g = rt.Graph(s)
    g.begin()
    try:
        rt.call('glmvx_lora_add', bufs['y'].ptr, rows, bufs['x'].ptr, cols, bufs['ids'].ptr, 30, bufs['a'].ptr,
                bufs['b'].ptr, bufs['ranks'].ptr, bufs['scales'].ptr, tokens, rows, cols, adapters, max_rank, ws.ptr,
                need, s.handle)
    finally:
        g.end()
    try:
        for n, buf in bufs.items():
            buf.upload(getattr(case, n), s.handle)
        first = case.run(gpu_backend)
        for ids, start in ((case.ids, case.y), (other, first)):
            case.ids, case.y = ids, start
            bufs['ids'].upload(ids, s.handle)
            g.launch()
            got = np.empty_like(case.y)
            bufs['y'].download(got, s.handle)
            s.synchronize()
            assert got.tobytes() == case.run(gpu_backend).tobytes()
    finally:
        g.close()
        for buf in list(bufs.values()) + [ws]:
            buf.close()


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('tokens,adapters,cols', [(4, 2, 96), (40, 50, 96), (300, 3, 96), (5, 2, 31), (70, 2, 2100)])
def test_infinities_are_the_formulas(gpu_backend, kind, tokens, adapters, cols):
    """An infinite x makes what the formula makes of it: h and y infinite with its sign, NaN where signs or a zero meet
    it.  Values next to the largest finite one stay finite and as exact as others."""
    rank, rows = 3, 72
    ids = np.arange(tokens) % adapters
    ids[:4] = 0, 1, 0, 1
    case = Case(tokens, rows, cols, adapters, rank, kind, ids=ids, ranks=[1 + 2 * (i % 2) for i in range(adapters)],
                seed=cols)
    a, b = case.a64.copy(), case.b64.copy()
    a[0, 0, 7] = 1.5  # one TF32 part holds it
    a[1, :, 5] = np.abs(a[1, :, 5])  # h of one sign
    a[0, 0, 3] = 0.0
    a[1, :, 11:13] *= 2.0 ** -7
    b[1, :20] = np.abs(b[1, :20])  # ranks of one sign: infinite; mixed: NaN
    case.a, case.a64 = pack(kind, a.astype(np.float32))
    case.b, case.b64 = pack(kind, b.astype(np.float32))
    big = np.finfo(np.float32).max
    case.x[0, 7], case.x[1, 5], case.x[2, 3], case.x[3, 11:13] = np.inf, -np.inf, np.inf, (big, -big / 8)
    with np.errstate(all='ignore'):
        out = case.run(gpu_backend)[:, :rows].astype(np.float64)
        want, tol = case.want()
    assert np.isinf(want).any() and np.isnan(want).any()
    assert np.array_equal(np.isnan(out), np.isnan(want))
    assert np.array_equal(out[np.isinf(want)], want[np.isinf(want)])
    fine = np.isfinite(want)
    assert (np.abs(want[3][fine[3]]) > 1e30).any()
    assert (np.abs(out[fine] - want[fine]) <= tol[fine]).all()


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('tokens', [4, 40, 300])
@pytest.mark.parametrize('rank', [16, 256])
def test_long_sums_do_not_drift(gpu_backend, kind, tokens, rank):
    """The norm of the whole change's error, which a bound for every element is too wide to see.

    A tensor core cuts what an addition leaves over: half of 2^-23 of the sum at the mean, toward zero.  Through 64
    normal products, eight at a time, the sum grows as the root of their number; 0.8 sqrt(8 i) for i = 1 .. 8, added
    up, is 36 of a product's size where the sum itself has 8: 4.5 * 2^-24 of it, for each of the m products of parts
    that a step adds one after another (2; 3 with F32 weights).  Chains end there and go on as rounded sums, whose
    errors are of one sign with what they cut: A's 6144 columns lose that share of h, B's ranks that of y (a quarter of
    the ranks an eighth: 16 are cut to 1.1 * 2^-24).  The parts leave 2^-23 of x and of h over."""
    rows, cols, adapters = 256, 6144, 3
    ids = np.arange(tokens) % adapters
    case = Case(tokens, rows, cols, adapters, rank, kind, ids=ids, ranks=[rank] * adapters, seed=rank)
    case.y[:] = 0
    want, _ = case.want()
    off = np.linalg.norm(case.run(gpu_backend) - want) / np.linalg.norm(want)
    m = 3 if kind == 0 else 2
    assert off <= m * (4.5 + (4.5 if rank >= 64 else 1.1)) * 2.0 ** -24 + 2.0 ** -22, off


@pytest.mark.parametrize('kind', [0, 1, 30])
@pytest.mark.parametrize('max_rank', [64, 65, 72, 128, 136, 255])
def test_ranks_around_the_chains(gpu_backend, kind, max_rank):
    """Stacks of up to 64 ranks and of more, whose adapters end before, at and after a multiple of 64."""
    ranks = [min(r, max_rank) for r in (1, 63, 64, 65, 127, 128, 129, 192, 255)]
    for tokens, cols, rows in ((9, 96, 132), (70, 100, 67)):
        Case(tokens, rows, cols, 9, max_rank, kind, ids=np.arange(tokens) % 9, ranks=ranks,
             seed=max_rank).check(gpu_backend)
    case = Case(3, 64, 64, 3, max_rank, kind, ids=[2, 0, 2], ranks=ranks[-3:], seed=max_rank)
    assert case.check(gpu_backend).tobytes() == case.run(gpu_backend).tobytes()


@pytest.mark.parametrize('tokens,adapters,used', [(1 << 20, 1, 1), (1 << 20, 3, 2), (3000, 1 << 20, 1 << 20),
                                                  (40, 1 << 24, 1 << 24)])
def test_the_largest_numbers_of_tokens_and_adapters(gpu_backend, tokens, adapters, used):
    """Against 64 bits: sums of 8 and 1 products, off by (8 / 8 + 40) * 2^-23 + 3 * 2^-22 of their terms each."""
    rows, cols, s = 4, 8, gpu_backend.stream
    rng = np.random.default_rng(tokens)
    ids = rng.integers(adapters - used, adapters, tokens).astype(np.int32)
    ids[::7] = -1
    x = rng.normal(size=(tokens, cols)).astype(np.float32)
    a, b = (rng.normal(size=(adapters, n)).astype(np.float16) for n in (cols, rows))
    need = gpu_backend.lib.glmvx_lora_workspace_bytes(tokens, adapters, 1)
    host = dict(y=np.zeros((tokens, rows), np.float32), x=x, ids=ids, a=a, b=b, ranks=np.ones(adapters, np.int32),
                scales=np.full(adapters, 2.0, np.float32), ws=np.full(need, 0xff, np.uint8))
    dev = {n: rt.DeviceBuffer(v.nbytes) for n, v in host.items()}
    try:
        for n, v in host.items():
            dev[n].upload(v, s.handle)
        rt.call('glmvx_lora_add', dev['y'].ptr, rows, dev['x'].ptr, cols, dev['ids'].ptr, 1, dev['a'].ptr,
                dev['b'].ptr, dev['ranks'].ptr, dev['scales'].ptr, tokens, rows, cols, adapters, 1, dev['ws'].ptr,
                need, s.handle)
        out = np.empty_like(host['y'])
        dev['y'].download(out, s.handle)
        s.synchronize()
    finally:
        for buf in dev.values():
            buf.close()
    at, has = np.maximum(ids, 0), (ids >= 0)[:, None]
    h = np.einsum('tc,tc->t', x.astype(np.float64), a[at].astype(np.float64))[:, None]
    mass = np.einsum('tc,tc->t', np.abs(x).astype(np.float64), np.abs(a[at]).astype(np.float64))[:, None]
    want = np.where(has, 2 * h * b[at].astype(np.float64), 0.0)
    off = 41 * 2.0 ** -23 + 3 * 2.0 ** -22
    tol = np.where(has, 2 * (2 * off + off * off) * mass * np.abs(b[at]).astype(np.float64), 0.0)
    assert (np.abs(out - want) <= tol).all()
