"""Linear attention where digits are lost first: memories and scores that differ from each other in their last bits.

Every product here and every sum of some of them is a number of 24 bits, and the results have few: in 32 bits nothing is
rounded, in any order, and the results are exact in all types. In 16 bits the last digits of 1 + 2^-8 + n 2^-20 would be lost.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
SMALL, ONE = 2.0 ** -20, 1 + 2.0 ** -8
# batch, heads, key size, value size: loose, whole and full tiles, few heads and many.
SIZES = [(127, 1, 5, 3), (127, 1, 20, 24), (127, 1, 32, 32), (127, 2, 64, 64), (1270, 2, 64, 64), (1270, 1, 128, 64), (254, 1, 96, 48)]


def zeros(batch, time, heads, key_size, value_size, dtype):
    query, key = (torch.zeros(batch, time, heads, key_size, dtype=dtype, device='cuda') for _ in range(2))
    value = torch.zeros(batch, time, heads, value_size, dtype=dtype, device='cuda')
    return query, key, value, torch.zeros(batch, time, heads, device='cuda'), torch.zeros(batch, heads, key_size, value_size, device='cuda')


def counts(batch):
    """1 to 31 along the batch: five digits, which every type holds."""
    return 1 + torch.arange(batch, device='cuda') % 31


def attend(query, key, value, decay, state):
    from cuju_amd import layers
    return layers.linear_attention(query, key, value, decay, state=state, scale=1.0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', SIZES)
def test_a_memory_of_24_bits(sizes, dtype):
    # (one + n small) - one of two rows of the memory, at every step.
    batch, heads, key_size, value_size = sizes
    query, key, value, decay, state = zeros(batch, 40, heads, key_size, value_size, dtype)
    n = counts(batch)
    query[..., 0], query[..., key_size - 1] = 1, -1
    state[:, :, 0], state[:, :, key_size - 1] = ONE + n[:, None, None] * SMALL, ONE
    output, last = attend(query, key, value, decay, state)
    assert torch.equal(output.float(), (n * SMALL)[:, None, None, None].expand(output.shape))
    assert torch.equal(last, state)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', SIZES)
def test_scores_of_24_bits(sizes, dtype):
    # The scores one + n small and one of two steps with the later ones, whose values are 1 and -1.
    batch, heads, key_size, value_size = sizes
    query, key, value, decay, state = zeros(batch, 40, heads, key_size, value_size, dtype)
    n = counts(batch)
    query[..., 0], query[..., 1], query[..., key_size - 1] = 1, 2.0 ** -4, 2.0 ** -10
    key[:, [3, 20], :, 0], key[:, [3, 20], :, 1] = 1, 2.0 ** -4
    key[:, 3, :, key_size - 1] = n[:, None] * 2.0 ** -10
    value[:, 3], value[:, 20] = 1, -1
    output, _ = attend(query, key, value, decay, state)
    assert not bool(output[:, :3].any())
    assert torch.equal(output[:, 20:].float(), (n * SMALL)[:, None, None, None].expand(batch, 20, heads, value_size))


@pytest.mark.parametrize('learnt', [False, True])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', SIZES)
def test_gradients_of_24_bits(sizes, dtype, learnt):
    # Whether the decay is learnt does not matter to the other gradients' digits.
    batch, heads, key_size, value_size = sizes
    query, key, value, decay, state = zeros(batch, 40, heads, key_size, value_size, dtype)
    n = counts(batch)
    exact = (n * SMALL)[:, None, None, None]
    key[:, 7, :, 0], key[:, 7, :, key_size - 1] = 1, -1
    value[:, 9, :, 0], value[:, 9, :, value_size - 1] = 1, -1
    d_output, d_last = torch.zeros_like(value), torch.zeros_like(state)
    d_output[:, 30, :, 0], d_output[:, 30, :, value_size - 1] = 1, -1
    # Two rows of the last memory's gradient for dv, and two columns for dk; two columns of the first memory for dq.
    rows, columns = d_last.clone(), d_last.clone()
    rows[:, :, 0], rows[:, :, key_size - 1] = ONE + n[:, None, None] * SMALL, ONE
    columns[..., 0], columns[..., value_size - 1] = ONE + n[:, None, None] * SMALL, ONE

    def gradients(d_last, d_output, state, *, k=key, v=value):
        leaves = [x.detach().requires_grad_() for x in (query, k, v)]
        gates = decay.detach().requires_grad_(learnt)
        return torch.autograd.grad(attend(*leaves, gates, state), leaves, [d_output, d_last])

    none = torch.zeros_like(value)
    *_, d_value = gradients(rows, none, state)
    assert torch.equal(d_value[:, 7].float(), exact[:, 0].expand(batch, heads, value_size))
    _, d_key, _ = gradients(columns, none, state)
    assert torch.equal(d_key[:, 9].float(), exact[:, 0].expand(batch, heads, key_size))
    d_query, _, _ = gradients(torch.zeros_like(d_last), d_output, columns, k=torch.zeros_like(key), v=torch.zeros_like(value))
    assert torch.equal(d_query[:, 30].float(), exact[:, 0].expand(batch, heads, key_size))
