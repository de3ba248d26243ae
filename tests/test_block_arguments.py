"""Workspaces and strides of the operators of a policy's blocks, without a device."""

import pytest
import torch

from conftest import PRODUCT
from cuju_amd import layers, library

SPAN = 128


def attention(time, batch=1, heads=1, key_size=8, value_size=8, checkpoints=0, d_decay=0, of_head=0):
    return layers._ATTENTION.pack(0, batch, time, 1, heads, key_size, value_size, of_head, 1.0, *[0] * 22, checkpoints, *[0] * 8, d_decay, 0, 0)


@pytest.mark.parametrize('key_size, value_size', [(1, 1), (3, 3), (5, 7), (8, 8), (128, 128)])
@pytest.mark.parametrize('time', [384, 385, 512, 513, 3000])
def test_workspaces_of_joined_spans(time, key_size, value_size):
    # Behind the memories of odd sizes, factors of eight bytes lie where eight bytes may.
    lib = library.load(PRODUCT)
    for batch, heads in ((1, 1), (3, 1), (1, 5)):
        joined = batch * heads * ((time - 1) // SPAN)
        sizes = dict(batch=batch, heads=heads, key_size=key_size, value_size=value_size)
        memories = -(-joined * key_size * value_size // 2) * 8
        assert lib.cuju_linear_attention_forward_workspace(attention(time, **sizes)) == memories + 8 * joined
        assert lib.cuju_linear_attention_forward_workspace(attention(time, checkpoints=64, **sizes)) == 8 * joined
        plain = lib.cuju_linear_attention_backward_workspace(attention(time, **sizes))
        assert plain % 8 == 0 and plain >= 4 * joined * key_size * value_size + 8 * joined
        # Decays: dots and products by slices of 16 keys, and whether a span has a step that nearly forgets.
        spans, slices = batch * heads * (-(-time // SPAN)), -(-key_size // 16)
        learnt = lib.cuju_linear_attention_backward_workspace(attention(time, d_decay=64, **sizes))
        assert learnt >= plain + 4 * slices * (2 * batch * heads * time + spans) + spans
        assert lib.cuju_linear_attention_backward_workspace(attention(time, d_decay=64, of_head=1, **sizes)) >= learnt + 8 * spans


def test_rows_that_lie_in_no_two_axes():
    x = torch.zeros(4, 3, 5, 8)
    # Five rows 8 apart, four times 120 apart, before an axis of one row: two strides where there is room for one.
    moved = x[:, :1].transpose(1, 2)
    assert moved.shape == (4, 5, 1, 8) and layers._row_strides(moved) is None
    for each in (moved, x.transpose(0, 2), x[:, ::2], x[:, :2]):
        rows = layers._in_rows(each)
        assert layers._row_strides(rows) is not None and torch.equal(rows, each)
