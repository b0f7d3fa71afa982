"""What glmvx_lora_add refuses, checked before any CUDA call (no GPU needed)."""
import pytest

from gpu import runtime as rt

GOOD = dict(y=4096, y_stride=64, x=8192, x_stride=32, ids=256, kind=30, a=256, b=256, ranks=256, scales=256,
            tokens=2, rows=64, cols=32, adapters=3, max_rank=8, workspace=256, workspace_bytes=1 << 20, stream=None)


def call(**change):
    args = dict(GOOD, **change)
    lib = rt.library()
    return lib.glmvx_lora_add(*args.values()), lib.glmvx_last_error().decode()


@pytest.mark.parametrize('change,code,message', [
    (dict(tokens=-1), -1, 'dimensions'), (dict(tokens=(1 << 20) + 1), -1, 'dimensions'),
    (dict(rows=0), -1, 'dimensions'), (dict(cols=0), -1, 'dimensions'), (dict(adapters=0), -1, 'dimensions'),
    (dict(adapters=(1 << 24) + 1), -1, 'dimensions'),
    (dict(rows=(1 << 22) + 1), -1, 'dimensions'), (dict(cols=(1 << 22) + 1), -1, 'dimensions'),
    (dict(max_rank=0), -1, 'max_rank'), (dict(max_rank=257), -1, 'max_rank'), (dict(kind=8), -4, 'kind'),
    (dict(kind=-1), -4, 'kind'), (dict(y_stride=63), -1, 'strides'), (dict(x_stride=31), -1, 'strides'),
    (dict(y=None), -1, 'null'), (dict(x=None), -1, 'null'), (dict(ids=None), -1, 'null'), (dict(a=None), -1, 'null'),
    (dict(b=None), -1, 'null'), (dict(ranks=None), -1, 'null'), (dict(scales=None), -1, 'null'),
    (dict(workspace=None), -1, 'null'), (dict(y=4098), -1, 'misaligned'), (dict(x=8193), -1, 'misaligned'),
    (dict(ids=258), -1, 'misaligned'), (dict(a=257), -1, 'misaligned'), (dict(kind=0, b=258), -1, 'misaligned'),
    (dict(workspace=264), -1, 'misaligned'), (dict(workspace_bytes=2 * 8 * 4 - 1), -1, 'workspace')])
def test_refusals(change, code, message):
    got, text = call(**change)
    assert got == code and message in text, (got, text)


def test_no_tokens_is_no_work():
    assert call(tokens=0, y=None, x=None, ids=None)[0] == 0


def test_workspace_size():
    size = rt.library().glmvx_lora_workspace_bytes
    assert size(1, 1, 1) > 0 and size(0, 1, 1) > 0
    assert size(64, 4, 16) >= 64 * 16 * 4
    for bad in ((-1, 1, 1), ((1 << 20) + 1, 1, 1), (1, 0, 1), (1, (1 << 24) + 1, 1), (1, 1, 0), (1, 1, 257)):
        assert size(*bad) < 0


@pytest.mark.parametrize('adapters,max_rank', [(1, 1), (16, 32), (24, 64), (4, 16), (300, 256)])
def test_a_workspace_does_for_fewer_tokens_too(adapters, max_rank):
    """A bank asks once, for the most tokens it takes."""
    size = rt.library().glmvx_lora_workspace_bytes
    need = [size(t, adapters, max_rank) for t in [*range(1, 20000), *range(20000, 1 << 20, 4097), 1 << 20]]
    assert all(a <= b for a, b in zip(need, need[1:]))
    # h holds at least a part of every token
    assert need[-1] >= 4 * max_rank << 20
