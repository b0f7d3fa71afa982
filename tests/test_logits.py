"""What glmvx_logits_select refuses, checked before any CUDA call (no GPU needed)."""
import pytest

from gpu import runtime as rt

GOOD = dict(selected=256, out=4096, out_stride=100, logits=8192, logits_stride=100, rows=2, vocab=100, fed=256,
            history=256, history_capacity=16, history_lens=256, prompt_lens=256, penalties=256, bias_ids=256,
            bias_values=256, bias_lens=256, bias_capacity=4, masks=256, mask_rows=256, mask_count=3, stream=None)


def call(**change):
    args = dict(GOOD, **change)
    lib = rt.library()
    return lib.glmvx_logits_select(*args.values()), lib.glmvx_last_error().decode()


@pytest.mark.parametrize('change,message', [
    (dict(rows=-1), 'dimensions'), (dict(vocab=0), 'dimensions'), (dict(vocab=2**30 + 1), 'dimensions'),
    (dict(rows=2**24 + 1), 'dimensions'), (dict(selected=None), 'null'),
    (dict(out=None), 'null'), (dict(logits=None), 'null'), (dict(out_stride=99), 'strides'),
    (dict(logits_stride=99), 'strides'), (dict(out=8192, out_stride=101), 'in place'),
    (dict(history=None), 'history'), (dict(history_lens=None), 'history'),
    (dict(history=None, history_lens=None, prompt_lens=None), 'history'),
    (dict(history=None, history_lens=None, fed=None), 'history'), (dict(history_capacity=0), 'capacity'),
    (dict(history_capacity=2**20 - 1), 'capacity'), (dict(bias_ids=None), 'biases'),
    (dict(bias_values=None), 'biases'), (dict(bias_lens=None), 'biases'), (dict(bias_capacity=0), 'bias capacity'),
    (dict(bias_capacity=2048), 'bias capacity'), (dict(masks=None), 'masks'), (dict(mask_rows=None), 'masks'),
    (dict(mask_count=0), 'no masks'), (dict(out=4097), 'misaligned'), (dict(masks=258), 'misaligned')])
def test_refusals(change, message):
    code, text = call(**change)
    assert code == -1 and message in text, (code, text)


def test_no_rows_is_no_work():
    assert call(rows=0, out=None, logits=None)[0] == 0
