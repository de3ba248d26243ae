"""The policy operators against their definitions in 64 bits (tests/layer_oracle.py).

Tolerances, in the 2-norm relative to the result. In 32 bits a value is a chain of at most four
products that each sum up to 144 terms; with rounding errors of 2^-24 of either sign a product adds
sqrt(144) 2^-24 = 7e-7, the chain under 3e-6, and a gradient, which takes two such chains, under 6e-6. A
result that is rounded once to bfloat16 or float16 is off by at most 2^-8 or 2^-11 more.
"""

import pytest
import torch

from layer_oracle import delta_rule as exact_rule
from layer_oracle import group_norm as exact_norm

pytestmark = pytest.mark.gpu

VALUES, GRADIENTS = 3e-6, 6e-6
ROUNDING = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(found, exact, bound, terms=0.0):
    """`terms`: the size of what the result is a small difference of, if it is one."""
    found = found.detach().cpu()
    exact = exact.reshape(found.shape)
    assert bool(torch.isfinite(found).all())
    error, size = float((found.double() - exact).norm()), float(exact.norm())
    allowed = bound * max(size, terms) + ROUNDING[found.dtype] * size
    assert error <= allowed + 1e-30, f'{error:.3g} off, {allowed:.3g} allowed'


def inputs(batch, time, key_heads, heads, key_size, value_size, dtype=torch.float32, seed=0, episode=0, state=True):
    """Unit keys that keep a direction of their own, decays of all reaches, and a memory."""
    generator = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=generator)

    def directions():
        x = normal(batch, time, key_heads, key_size) + normal(batch, 1, key_heads, key_size)
        return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)

    given = {'query': directions().to(dtype), 'key': directions().to(dtype),
             'value': normal(batch, time, heads, value_size).to(dtype),
             'decay': -torch.logspace(-3, 0.3, heads) * torch.nn.functional.softplus(normal(batch, time, heads)),
             'beta': torch.sigmoid(normal(batch, time, heads)),
             'state': normal(batch, heads, key_size, value_size) if state else None,
             'resets': torch.rand(batch, time, generator=generator) < 1 / episode if episode else None}
    return {name: x.cuda() if x is not None else None for name, x in given.items()}


def rule(given, **changes):
    from cuju_amd import layers
    given = {**given, **changes}
    return layers.delta_rule(given['query'], given['key'], given['value'], given['decay'], given['beta'],
                             state=given['state'], resets=given['resets'])


def learn(given, d_output=None, d_last=None, seed=5):
    """Outputs and gradients of a training pass, and the outputs' gradients it was given."""
    generator = torch.Generator().manual_seed(seed)
    names = [n for n in ('query', 'key', 'value', 'decay', 'beta', 'state') if given[n] is not None]
    leaves = {n: given[n].detach().requires_grad_() for n in names}
    output, last = rule(given, **leaves)
    if d_output is None:
        d_output = torch.randn(output.shape, generator=generator).to(output.dtype).cuda()
    if d_last is None:
        d_last = torch.randn(last.shape, generator=generator).cuda()
    found = torch.autograd.grad([output, last], list(leaves.values()), [d_output, d_last])
    return {'output': output, 'last': last, **{'d_' + n: g for n, g in zip(names, found)}}, d_output, d_last


def learn_close(given):
    found, d_output, d_last = learn(given)
    exact = exact_rule(**given, d_output=d_output, d_last=d_last)
    for name, x in found.items():
        if x.numel():
            close(x, exact[name], GRADIENTS if name.startswith('d_') else VALUES)
    return found


# batch, time, key heads, heads, key size, value size, steps of an episode
RULES = [
    (1, 1, 1, 1, 1, 1, 0),
    (3, 1, 2, 2, 64, 64, 0),
    (2, 15, 1, 3, 16, 33, 0),
    (2, 16, 2, 4, 32, 16, 4),
    (2, 17, 3, 3, 33, 48, 0),
    (3, 63, 1, 2, 64, 64, 9),
    (2, 64, 2, 2, 64, 128, 30),
    (2, 65, 2, 2, 96, 65, 0),
    (1, 129, 1, 4, 128, 128, 50),
    (5, 200, 2, 2, 40, 72, 3),
    (2, 130, 1, 1, 100, 20, 1),
]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', RULES)
def test_delta_rule_and_its_gradients(sizes, dtype):
    learn_close(inputs(*sizes[:6], dtype=dtype, seed=sum(sizes), episode=sizes[6], state=sizes[1] % 2 == 1))


@pytest.mark.parametrize('heads', [300, 1100])
def test_delta_rule_of_many_heads(heads):
    # Wide and narrow pieces of the memory, as few or many heads get them.
    for value_size in (16, 30, 64, 100):
        given = inputs(heads, 20, 1, 1, 24, value_size, seed=heads + value_size, episode=15)
        output, last = rule(given)
        exact = exact_rule(**given)
        close(output, exact[0], VALUES)
        close(last, exact[1], VALUES)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', [(1, 1, 1, 1, 1), (7, 2, 6, 40, 72), (5, 3, 3, 64, 64), (3, 1, 2, 128, 128),
                                   (9, 2, 2, 17, 5), (4, 1, 1, 100, 30)])
def test_a_step_is_one_step_of_the_rule(sizes, dtype):
    from cuju_amd import layers
    batch, key_heads, heads, key_size, value_size = sizes
    given = inputs(batch, 1, key_heads, heads, key_size, value_size, dtype=dtype, seed=sum(sizes))
    for resets in (None, torch.arange(batch, device='cuda') % 2 == 0):
        state = given['state'].clone()
        at = [given[n].squeeze(1) for n in ('query', 'key', 'value', 'decay', 'beta')]
        output = layers.delta_rule_step(*at, state, resets=resets)
        exact = exact_rule(**{**given, 'resets': resets[:, None] if resets is not None else None})
        close(output, exact[0][:, 0], VALUES)
        close(state, exact[1], VALUES)


def test_steps_one_by_one_follow_the_rule():
    from cuju_amd import layers
    given = inputs(6, 70, 2, 4, 64, 64, seed=3, episode=20)
    state = given['state'].clone()
    outputs = [layers.delta_rule_step(*[given[n][:, t] for n in ('query', 'key', 'value', 'decay', 'beta')], state,
                                      resets=given['resets'][:, t]) for t in range(70)]
    exact = exact_rule(**given)
    close(torch.stack(outputs, 1), exact[0], VALUES)
    close(state, exact[1], VALUES)


def test_a_memory_carried_over_pieces_is_the_whole():
    given = inputs(3, 90, 2, 2, 64, 48, seed=4, episode=25)
    state, outputs = given['state'], []
    for low, high in ((0, 1), (1, 30), (30, 30), (30, 90)):
        piece = {n: x[:, low:high] for n, x in given.items() if n != 'state'}
        output, state = rule(piece, state=state)
        outputs.append(output)
    exact = exact_rule(**given)
    close(torch.cat(outputs, 1), exact[0], VALUES)
    close(state, exact[1], VALUES)


def test_repeated_keys():
    # The same unit key at every step with beta 1 and no decay: the triangular system is all ones,
    # the case that powers of it would lose. Each value is then written over the last.
    given = inputs(2, 80, 1, 2, 64, 32, seed=6, state=False)
    given['key'] = given['key'][:, :1].expand(-1, 80, -1, -1)
    given['decay'] = torch.zeros_like(given['decay'])
    given['beta'] = torch.ones_like(given['beta'])
    found, d_output, d_last = learn(given)
    exact = exact_rule(**given, d_output=d_output, d_last=d_last)
    # The memory is key value^T of the last value whatever it kept, so the decays' true gradients are
    # zero: a sum of terms of the size of the memory times its gradient cancels.
    terms = float(exact['last'].norm()) * float(d_last.double().norm())
    for name, x in found.items():
        close(x, exact[name], GRADIENTS if name.startswith('d_') else VALUES, terms if name == 'd_decay' else 0.0)


@pytest.mark.parametrize('decay', [0.0, -30.0, -200.0, -1e30, -float('inf')])
def test_extreme_decays(decay):
    given = inputs(2, 70, 2, 2, 32, 32, seed=7)
    given['decay'][:, 5::9] = decay
    given['decay'][0, 40:44] = decay
    found, d_output, d_last = learn(given)
    # The definition with a factor of 0 where 32 bits have none.
    exact = exact_rule(**{**given, 'decay': given['decay'].clamp_min(-700)}, d_output=d_output, d_last=d_last)
    for name, x in found.items():
        close(x, exact[name], GRADIENTS if name.startswith('d_') else VALUES)


def test_gates_of_zero_and_keys_of_zero():
    given = inputs(2, 40, 1, 2, 32, 32, seed=8)
    given['beta'][:, ::3] = 0
    given['key'][:, 7:9] = 0
    learn_close(given)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_nothing_crosses_a_reset(bad):
    from cuju_amd import layers
    given = inputs(3, 60, 1, 2, 48, 40, seed=9)
    resets = torch.zeros(3, 60, dtype=torch.bool, device='cuda')
    resets[0, 0] = resets[1, 21] = resets[2, 37] = True
    given['resets'] = resets
    spoilt = {n: x.clone() for n, x in given.items()}
    spoilt['state'][:] = bad
    for b, t in ((1, 21), (2, 37)):
        for name in ('query', 'key', 'value', 'decay', 'beta'):
            spoilt[name][b, :t] = bad
    found, clean = rule(spoilt), rule(given)
    for b, t in ((0, 0), (1, 21), (2, 37)):
        assert torch.equal(found[0][b, t:], clean[0][b, t:])
        assert torch.equal(found[1][b], clean[1][b])
    # The gradients of the steps after.
    spoilt_learnt, d_output, d_last = learn(spoilt)
    clean_learnt, _, _ = learn(given, d_output, d_last)
    for b, t in ((0, 0), (1, 21), (2, 37)):
        for name in ('query', 'key', 'value', 'decay', 'beta'):
            assert torch.equal(spoilt_learnt['d_' + name][b, t:], clean_learnt['d_' + name][b, t:]), name
    assert not bool(spoilt_learnt['d_state'][0].any())
    state = torch.full_like(given['state'], bad)
    output = layers.delta_rule_step(*[given[n][:, 0] for n in ('query', 'key', 'value', 'decay', 'beta')], state,
                                    resets=torch.ones(3, dtype=torch.bool, device='cuda'))
    assert bool(torch.isfinite(output).all()) and bool(torch.isfinite(state).all())


def test_strides_and_alignment():
    given = inputs(4, 50, 2, 2, 32, 32, seed=10, episode=20)
    wanted, d_output, d_last = learn(given)
    # An axis of time first, one packed tensor of queries, keys and values, and an odd offset.
    packed = torch.zeros(50, 4, 2, 3 * 32 + 1, device='cuda')
    views = {}
    for i, name in enumerate(('query', 'key', 'value')):
        views[name] = packed[..., 1 + 32 * i:1 + 32 * (i + 1)].transpose(0, 1)
        views[name].copy_(given[name])
    views['decay'] = given['decay'].transpose(0, 1).contiguous().transpose(0, 1)
    views['resets'] = given['resets'].transpose(0, 1).contiguous().transpose(0, 1).to(torch.uint8)
    found, _, _ = learn({**given, **views}, d_output, d_last)
    for name in wanted:
        assert torch.equal(found[name], wanted[name]), name
    # Gradients that come as views: time first, and one value for all.
    moved, _, _ = learn(given, d_output.transpose(0, 1).contiguous().transpose(0, 1), d_last)
    for name in wanted:
        assert torch.equal(moved[name], wanted[name]), name
    one = torch.ones((), device='cuda')
    found, _, _ = learn(given, one.expand(d_output.shape), one.expand(d_last.shape))
    wanted, _, _ = learn(given, torch.ones_like(d_output), torch.ones_like(d_last))
    for name in wanted:
        assert torch.equal(found[name], wanted[name]), name


def test_broadcast_inputs():
    # One query and key for the whole batch: their gradients are the batch's sum.
    given = inputs(3, 33, 2, 2, 32, 32, seed=11)
    query, key = (given[n][:1].clone().requires_grad_() for n in ('query', 'key'))
    output, last = rule(given, query=query.expand(3, -1, -1, -1), key=key.expand(3, -1, -1, -1))
    d_output, d_last = torch.randn_like(output), torch.randn_like(last)
    found = torch.autograd.grad([output, last], [query, key], [d_output, d_last])
    given['query'], given['key'] = query.detach().expand(3, -1, -1, -1), key.detach().expand(3, -1, -1, -1)
    exact = exact_rule(**given, d_output=d_output, d_last=d_last)
    for x, name in zip(found, ('d_query', 'd_key')):
        close(x, exact[name].sum(0, keepdim=True), GRADIENTS)


def test_only_one_output_is_learnt_from():
    given = inputs(2, 70, 1, 2, 32, 32, seed=12)
    for which in (0, 1):
        leaf = given['value'].clone().requires_grad_()
        outputs = rule(given, value=leaf)
        d = torch.randn_like(outputs[which])
        found, = torch.autograd.grad(outputs[which], leaf, d)
        zeros = [torch.zeros_like(x) for x in outputs]
        zeros[which] = d
        close(found, exact_rule(**given, d_output=zeros[0], d_last=zeros[1])['d_value'], GRADIENTS)


def test_gates_in_other_types():
    from cuju_amd import layers
    given = inputs(2, 20, 1, 2, 32, 32, dtype=torch.bfloat16, seed=13)
    decay = given['decay'].to(torch.bfloat16).requires_grad_()
    beta = given['beta'].double().requires_grad_()
    output, last = rule(given, decay=decay, beta=beta)
    d_output, d_last = torch.randn_like(output), torch.randn_like(last)
    found = torch.autograd.grad([output, last], [decay, beta], [d_output, d_last])
    assert found[0].dtype == torch.bfloat16 and found[1].dtype == torch.double
    exact = exact_rule(**{**given, 'decay': decay, 'beta': beta.float()}, d_output=d_output, d_last=d_last)
    close(found[0], exact['d_decay'], GRADIENTS)
    close(found[1].float(), exact['d_beta'], GRADIENTS)
    scaled = layers.delta_rule(given['query'], given['key'], given['value'], decay.detach(), beta.detach(), scale=3.0)[0]
    close(scaled, exact_rule(given['query'], given['key'], given['value'], decay, beta.float(), scale=3.0)[0], VALUES)


def test_empty_batches_and_times():
    from cuju_amd import layers
    for batch, time in ((0, 5), (3, 0), (0, 0)):
        given = inputs(batch, time, 1, 2, 32, 16, seed=14)
        found, d_output, d_last = learn(given)
        assert found['output'].shape == (batch, time, 2, 16) and found['d_query'].shape == (batch, time, 1, 32)
        assert torch.equal(found['last'], given['state'])
        assert torch.equal(found['d_state'], d_last)
    given = inputs(3, 0, 1, 2, 32, 16, state=False)
    assert not bool(rule(given)[1].any())
    empty = inputs(0, 1, 1, 2, 32, 16)
    output = layers.delta_rule_step(*[empty[n][:, 0] for n in ('query', 'key', 'value', 'decay', 'beta')], empty['state'])
    assert output.shape == (0, 2, 16)


def test_offsets_past_32_bits():
    # Two sequences of one allocation, 2^31 elements and some apart.
    given = inputs(2, 20, 1, 1, 32, 32, dtype=torch.bfloat16, seed=15, episode=9)
    apart = (1 << 31) + 64
    room = torch.empty(apart + 20 * 32, dtype=torch.bfloat16, device='cuda')
    wanted, d_output, d_last = learn(given)
    for name in ('query', 'key', 'value'):
        view = room.as_strided((2, 20, 1, 32), (apart, 32, 32, 1))
        view.copy_(given[name])
        found, _, _ = learn({**given, name: view}, d_output, d_last)
        for n in wanted:
            assert torch.equal(found[n], wanted[n]), (name, n)


def test_calls_repeat_bit_for_bit():
    given = inputs(30, 100, 2, 4, 64, 64, dtype=torch.bfloat16, seed=16, episode=30)
    first, d_output, d_last = learn(given)
    for _ in range(3):
        again, _, _ = learn(given, d_output, d_last)
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_gradients_against_differences():
    # A central difference along a direction, h = 2^-6: rounding leaves 64 * 2 * 3e-6 of the loss's
    # terms, the third derivative h^2 of them: 1e-3 of the size of the terms.
    given = inputs(2, 37, 1, 2, 24, 24, seed=17, episode=15)
    found, d_output, d_last = learn(given)
    generator = torch.Generator().manual_seed(1)

    def loss(changed):
        output, last = rule({**given, **changed})
        return float((output.double() * d_output.double()).sum() + (last.double() * d_last.double()).sum())

    for name in ('query', 'key', 'value', 'decay', 'beta', 'state'):
        x = given[name]
        along = torch.randn(x.shape, generator=generator).cuda()
        along /= along.norm()
        h = 2.0 ** -6
        difference = (loss({name: x + h * along}) - loss({name: x - h * along})) / (2 * h)
        slope = float((found['d_' + name].double() * along.double()).sum())
        size = float(found['d_' + name].double().norm())
        assert abs(difference - slope) <= 1e-3 * size + 1e-3 * abs(slope), name


def test_on_another_stream_and_in_a_graph():
    from cuju_amd import layers
    given = inputs(4, 40, 1, 2, 64, 64, dtype=torch.bfloat16, seed=18, episode=10)
    x = torch.randn(2, 6, 8, 16, device='cuda')
    wanted, norm = rule(given), layers.group_norm(x, 4, activation='silu')
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        found, again = rule(given), layers.group_norm(x, 4, activation='silu')
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(found[0], wanted[0]) and torch.equal(found[1], wanted[1]) and torch.equal(norm, again)

    at = [given[n][:, 0] for n in ('query', 'key', 'value', 'decay', 'beta')]
    state = given['state'].clone()
    with torch.cuda.stream(side):
        layers.delta_rule_step(*at, state.clone()), rule(given), layers.group_norm(x, 4, activation='silu')
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        output = layers.delta_rule_step(*at, state)
        replayed = rule(given)
        normed = layers.group_norm(x, 4, activation='silu')
    eager = given['state'].clone()
    state.copy_(given['state'])
    for _ in range(4):
        graph.replay()
        expected = layers.delta_rule_step(*at, eager)
        torch.cuda.synchronize()
        assert torch.equal(output, expected) and torch.equal(state, eager)
        assert torch.equal(replayed[0], wanted[0]) and torch.equal(replayed[1], wanted[1])
        assert torch.equal(normed, norm)


# --------------------------------------------------------------------------------------- group norm

def norm_learn(x, groups, weight, bias, activation, dy, epsilon=1e-5):
    from cuju_amd import layers
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
    given = iter(leaves)
    args = [next(given) if t is not None else None for t in (x, weight, bias)]
    y = layers.group_norm(args[0], groups, args[1], args[2], epsilon=epsilon, activation=activation)
    found = dict(zip([n for n, t in (('dx', x), ('d_weight', weight), ('d_bias', bias)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    return {'y': y, **found}


def norm_inputs(shape, dtype, seed):
    generator = torch.Generator().manual_seed(seed)
    channels = shape[-1]
    x = torch.randn(*shape, generator=generator) * (0.5 + torch.rand(channels, generator=generator))
    x = (x + torch.randn(channels, generator=generator)).to(dtype)
    weight = 1 + 0.3 * torch.randn(channels, generator=generator)
    bias = 0.3 * torch.randn(channels, generator=generator)
    dy = torch.randn(*shape, generator=generator).to(dtype)
    return [t.cuda() for t in (x, weight, bias, dy)]


# Shape and groups: single values, odd channels, one and many groups, maps held by one workgroup, by
# several, and by none.
NORMS = [
    ((1, 1), 1), ((2, 3, 5), 5), ((3, 7, 7, 6), 2), ((2, 9, 13, 40), 5), ((4, 16, 16, 64), 16), ((2, 12, 12, 30), 10),
    ((1, 72, 96, 16), 4), ((3, 36, 48, 64), 8), ((2, 72, 96, 32), 1), ((1, 72, 96, 32), 8), ((1, 200, 210, 24), 3),
    ((2, 5, 5, 1024), 2), ((1, 31, 17, 700), 7), ((65, 4), 2),
]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape, groups', NORMS)
def test_group_norm_and_its_gradients(shape, groups, dtype):
    x, weight, bias, dy = norm_inputs(shape, dtype, sum(shape) + groups)
    for activation in ('none', 'silu'):
        found = norm_learn(x, groups, weight, bias, activation, dy)
        exact = exact_norm(x, groups, weight, bias, activation=activation, dy=dy)
        for name, each in found.items():
            close(each, exact[name], GRADIENTS, exact['terms'] if name == 'dx' else 0.0)


def test_group_norm_with_relu():
    # No value within 32-bit rounding of the corner.
    x, weight, bias, dy = norm_inputs((3, 8, 8, 16), torch.float32, 1)
    z = exact_norm(x, 4, weight, bias)
    assert float(z.abs().min()) > 1e-5
    found = norm_learn(x, 4, weight, bias, 'relu', dy)
    exact = exact_norm(x, 4, weight, bias, activation='relu', dy=dy)
    for name, each in found.items():
        close(each, exact[name], GRADIENTS)


def test_group_norm_without_weights():
    x, weight, bias, dy = norm_inputs((2, 10, 10, 24), torch.bfloat16, 2)
    for w, b in ((None, None), (weight, None), (None, bias), (weight.to(torch.bfloat16), bias.double())):
        found = norm_learn(x, 3, w, b, 'silu', dy)
        exact = exact_norm(x, 3, w, b, activation='silu', dy=dy)
        for name, each in found.items():
            close(each.float() if each.dtype == torch.double else each, exact[name], GRADIENTS)


@pytest.mark.parametrize('pixels', [50, 40000])
def test_group_norm_far_from_zero_and_without_spread(pixels):
    from cuju_amd import layers
    generator = torch.Generator().manual_seed(3)
    # A mean 1,000 times the deviation: the deviation is 2^-14 of the values' size, so the mean's
    # rounding of 2^-24 of it is 2^-10 / sqrt(pixels) of a deviation at most; the inputs are exact.
    x = (1024 + torch.randn(2, pixels, 16, generator=generator)).cuda()
    y = layers.group_norm(x, 4)
    close(y, exact_norm(x, 4), 2.0 ** -10)
    flat = torch.full((2, pixels, 16), 3.25, device='cuda')
    assert float(layers.group_norm(flat, 4).abs().max()) <= 1e-3
    found = norm_learn(flat, 4, None, None, 'silu', torch.ones_like(flat))
    assert bool(torch.isfinite(found['dx']).all())


def test_group_norm_keeps_maps_and_groups_apart():
    from cuju_amd import layers
    for shape in ((3, 6, 6, 16), (3, 120, 120, 16)):
        x, weight, bias, dy = norm_inputs(shape, torch.float32, 4)
        wanted = layers.group_norm(x, 4, weight, bias, activation='silu')
        spoilt = x.clone()
        spoilt[1, 2, 3, 5] = float('nan')
        found = layers.group_norm(spoilt, 4, weight, bias, activation='silu')
        assert bool(torch.isnan(found[1, :, :, 4:8]).all())
        found[1, :, :, 4:8] = wanted[1, :, :, 4:8]
        assert torch.equal(found, wanted)


def test_group_norm_of_extreme_values():
    from cuju_amd import layers
    x = torch.zeros(1, 64, 8, device='cuda')
    x[0, 0] = 1e4
    weight = torch.full((8,), 200.0, device='cuda')
    for activation in ('silu', 'relu'):
        found = norm_learn(x, 2, weight, None, activation, torch.ones_like(x))
        assert all(bool(torch.isfinite(t).all()) for t in found.values())
    close(layers.group_norm(x, 2, weight, activation='silu'), exact_norm(x, 2, weight, activation='silu'), GRADIENTS)


def test_group_norm_strides_alignment_and_empty_maps():
    from cuju_amd import layers
    x, weight, bias, dy = norm_inputs((3, 8, 6, 16), torch.bfloat16, 5)
    wanted = layers.group_norm(x, 4, weight, bias)
    nchw = x.permute(0, 3, 1, 2).contiguous()
    assert torch.equal(layers.group_norm(nchw.permute(0, 2, 3, 1), 4, weight, bias), wanted)
    last = nchw.to(memory_format=torch.channels_last)
    assert torch.equal(layers.group_norm(last.permute(0, 2, 3, 1), 4, weight, bias), wanted)
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device='cuda')[1:].view(x.shape)
    odd.copy_(x)
    torch.testing.assert_close(layers.group_norm(odd, 4, weight, bias), wanted)
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8)):
        x = torch.empty(shape, device='cuda', requires_grad=True)
        weight = torch.ones(8, device='cuda', requires_grad=True)
        y = layers.group_norm(x, 2, weight)
        dx, d_weight = torch.autograd.grad(y, [x, weight], torch.ones_like(y))
        assert y.shape == shape and dx.shape == shape and not bool(d_weight.any())


def test_group_norm_gradients_against_differences():
    # As for the delta rule; h = 2^-5 of a step that moves every value.
    x, weight, bias, dy = norm_inputs((2, 9, 9, 12), torch.float32, 6)
    from cuju_amd import layers
    found = norm_learn(x, 3, weight, bias, 'silu', dy)
    generator = torch.Generator().manual_seed(2)
    for name, at in (('dx', 0), ('d_weight', 1), ('d_bias', 2)):
        args = [x, weight, bias]
        along = torch.randn(args[at].shape, generator=generator).cuda()
        along /= along.norm()
        h = 2.0 ** -5

        def loss(sign):
            moved = list(args)
            moved[at] = args[at] + sign * h * along
            y = layers.group_norm(moved[0], 3, moved[1], moved[2], activation='silu')
            return float((y.double() * dy.double()).sum())

        difference = (loss(1) - loss(-1)) / (2 * h)
        slope = float((found[name].double() * along.double()).sum())
        assert abs(difference - slope) <= 2e-3 * float(found[name].double().norm()), name


def test_group_norm_repeats_bit_for_bit():
    x, weight, bias, dy = norm_inputs((40, 20, 20, 32), torch.bfloat16, 7)
    first = norm_learn(x, 8, weight, bias, 'silu', dy)
    again = norm_learn(x, 8, weight, bias, 'silu', dy)
    assert all(torch.equal(first[n], again[n]) for n in first)


# ------------------------------------------------------------------------------------ torch.compile

def test_compiled_calls_equal_eager_ones():
    from cuju_amd import layers
    torch._dynamo.reset()
    given = inputs(3, 70, 1, 2, 32, 32, seed=19, episode=20)

    def train(q, k, v, decay, beta, state, resets, x, weight):
        normed = layers.group_norm(x, 2, weight, activation='silu')
        output, last = layers.delta_rule(q, k, v, decay, beta, state=state, resets=resets)
        return output, last, normed

    def act(q, k, v, decay, beta, state):
        return layers.delta_rule_step(q, k, v, decay, beta, state)

    x, weight = torch.randn(2, 5, 8, device='cuda'), torch.rand(8, device='cuda')
    names = ('query', 'key', 'value', 'decay', 'beta', 'state')

    def play(train):
        leaves = [given[n].clone().requires_grad_() for n in names] + [given['resets'], x.clone().requires_grad_(),
                                                                      weight.clone().requires_grad_()]
        outputs = train(*leaves)
        loss = sum((y.float() * (1 + i)).sum() for i, y in enumerate(outputs))
        loss.backward()
        return [*outputs, *[t.grad for t in leaves if t.requires_grad]]

    for found, wanted in zip(play(torch.compile(train, fullgraph=True, backend='aot_eager')), play(train)):
        assert torch.equal(found, wanted)
    at = [given[n][:, 0] for n in names[:5]]
    states = [given['state'].clone() for _ in range(2)]
    compiled = torch.compile(act, fullgraph=True, backend='aot_eager')
    for _ in range(2):
        assert torch.equal(compiled(*at, states[0]), act(*at, states[1]))
    assert torch.equal(*states)


# ---------------------------------------------------------------------------------------- refusals

def test_refusals():
    from cuju_amd import ArgumentError, ChoiceError, layers
    given = inputs(2, 4, 2, 4, 32, 32)

    def refused(**changes):
        with pytest.raises(ArgumentError):
            rule(given, **changes)

    refused(query=given['query'].cpu())
    refused(key=given['key'].cpu())
    refused(query=given['query'].double())
    refused(key=given['key'].half())
    refused(key=given['key'][..., :16])
    refused(value=given['value'][:, :3])
    refused(value=given['value'][:, :, :3], decay=given['decay'][..., :3], beta=given['beta'][..., :3])
    refused(decay=given['decay'][..., :1])
    refused(decay=given['decay'].int())
    refused(beta=given['beta'][:1])
    refused(state=given['state'][:1])
    refused(resets=torch.zeros(2, 5, dtype=torch.bool, device='cuda'))
    refused(resets=torch.zeros(2, 4, device='cuda'))
    refused(query=given['query'][:, 0])
    wide = torch.zeros(2, 4, 2, 129, device='cuda')
    refused(query=wide, key=wide, state=None)
    at = [given[n][:, 0] for n in ('query', 'key', 'value', 'decay', 'beta')]
    for state in (None, given['state'].half(), given['state'].transpose(-1, -2), given['state'][:1]):
        with pytest.raises(ArgumentError):
            layers.delta_rule_step(*at, state)
    with pytest.raises(ArgumentError):
        layers.delta_rule_step(at[0].requires_grad_(), *at[1:], given['state'])
    x = torch.zeros(2, 3, 8, device='cuda')
    for bad in (lambda: layers.group_norm(x.cpu(), 2), lambda: layers.group_norm(x.double(), 2),
                lambda: layers.group_norm(x, 3), lambda: layers.group_norm(x, 0),
                lambda: layers.group_norm(x, 2, torch.ones(7, device='cuda')),
                lambda: layers.group_norm(x, 2, torch.ones(8)),
                lambda: layers.group_norm(x, 2, torch.ones(8, dtype=torch.int32, device='cuda')),
                lambda: layers.group_norm(x[0, 0], 2)):
        with pytest.raises(ArgumentError):
            bad()
    with pytest.raises(ChoiceError):
        layers.group_norm(x, 2, activation='gelu')
    y = layers.group_norm(x.requires_grad_(), 2)
    dx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# ------------------------------------------------- tracers, modes and transforms besides torch.compile

def small_calls():
    """Calls of each operator as functions of tensors, with tensors for them."""
    from cuju_amd import layers
    given = inputs(2, 40, 1, 2, 16, 16, seed=20)
    names = ('query', 'key', 'value', 'decay', 'beta', 'state')
    x, weight = torch.randn(2, 5, 8, device='cuda'), torch.rand(8, device='cuda')

    def norm(x, weight):
        return layers.group_norm(x, 2, weight, activation='silu')

    def rule(q, k, v, decay, beta, state):
        return layers.delta_rule(q, k, v, decay, beta, state=state)

    def step(q, k, v, decay, beta, state):
        state = state.clone()
        return layers.delta_rule_step(q, k, v, decay, beta, state), state

    return [(norm, (x, weight)), (rule, tuple(given[n] for n in names)),
            (step, (*[given[n][:, 0] for n in names[:5]], given['state']))]


def outputs_of(call, tensors):
    found = call(*tensors)
    return found if isinstance(found, (tuple, list)) else (found,)


def gradients_of(call):
    def learnt(*tensors):
        leaves = [x.detach().requires_grad_() for x in tensors]
        outputs = outputs_of(call, leaves)
        return torch.autograd.grad(outputs, leaves, [torch.ones_like(y) for y in outputs])
    return learnt


@pytest.mark.parametrize('which', range(3))
def test_traced_graphs_compute(which):
    from torch.fx.experimental.proxy_tensor import make_fx
    call, tensors = small_calls()[which]
    other = [x * 0.5 for x in tensors]
    for each in (call, gradients_of(call)) if which < 2 else (call,):
        graph = make_fx(lambda *t: each(*t))(*tensors)
        for found, wanted in zip(outputs_of(graph, other), outputs_of(each, other)):
            assert torch.equal(found, wanted)
    traced = torch.jit.trace(call, tensors, check_trace=False)
    for found, wanted in zip(outputs_of(traced, other), outputs_of(call, other)):
        assert torch.equal(found, wanted)


def test_modes_see_the_gradients():
    from torch.utils._python_dispatch import TorchDispatchMode
    names = []

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, function, types, args=(), kwargs=None):
            names.append(function.name())
            return function(*args, **(kwargs or {}))

    for call, tensors in small_calls()[:2]:
        wanted = gradients_of(call)(*tensors)
        with Seen():
            found = gradients_of(call)(*tensors)
        assert all(torch.equal(a, b) for a, b in zip(found, wanted))
    assert [n for n in names if n.startswith('cuju_amd')] == [
        'cuju_amd::group_norm', 'cuju_amd::group_norm_backward', 'cuju_amd::delta_rule', 'cuju_amd::delta_rule_backward']


def test_transforms():
    (norm, (x, weight)), (rule, given), _ = small_calls()
    maps = torch.randn(3, *x.shape, device='cuda')
    found = torch.func.vmap(norm, (0, None))(maps, weight)
    assert torch.equal(found, torch.stack([norm(each, weight) for each in maps]))
    assert torch.equal(torch.func.functionalize(norm)(x, weight), norm(x, weight))
    assert all(torch.equal(a, b) for a, b in zip(torch.func.functionalize(rule)(*given), rule(*given)))
    # Gradients of function transforms are not there, and say so.
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: norm(x, weight).sum())(x)


def test_compiled_by_the_default_backend():
    from cuju_amd import layers
    torch._dynamo.reset()
    given = inputs(3, 40, 1, 2, 32, 32, seed=21)
    at = [given[n][:, 0] for n in ('query', 'key', 'value', 'decay', 'beta')]
    states = [given['state'].clone() for _ in range(2)]

    def act(q, k, v, decay, beta, state):
        return layers.delta_rule_step(q, k, v, decay, beta, state)

    compiled = torch.compile(act, fullgraph=True)
    for _ in range(2):
        assert torch.equal(compiled(*at, states[0]), act(*at, states[1]))
    assert torch.equal(*states)
    x, weight = torch.randn(2, 5, 8, device='cuda'), torch.rand(8, device='cuda')
    norm = torch.compile(lambda x, weight: layers.group_norm(x, 2, weight, activation='silu'), fullgraph=True)
    found, wanted = ([t.detach().requires_grad_() for t in (x, weight)] for _ in range(2))
    y, expected = norm(*found), layers.group_norm(wanted[0], 2, wanted[1], activation='silu')
    assert torch.equal(y, expected)
    y.backward(torch.ones_like(y)), expected.backward(torch.ones_like(y))
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(found, wanted))


# ------------------------------------------------------------------------- group norm: extreme values

@pytest.mark.parametrize('bad', [float('inf'), -float('inf'), float('nan')])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(2, 6, 6, 16), (2, 150, 150, 16), (1, 40, 40, 700)])
def test_an_infinity_leaves_its_group_nothing(shape, dtype, bad):
    # The mean is infinite, so no value has a difference from it: the whole group is NaN, whatever the activation, in
    # maps that are held, that are cut, and whose groups have a kernel for their statistics.
    from cuju_amd import layers
    x, weight, bias, dy = norm_inputs(shape, dtype, 8)
    each = shape[-1] // 4
    spoilt = x.clone()
    spoilt[0, 3, 2, each + 1] = bad
    for activation in ('none', 'relu', 'silu'):
        wanted = layers.group_norm(x, 4, weight, bias, activation=activation)
        found = norm_learn(spoilt, 4, weight, bias, activation, dy)
        for name, clean in (('y', wanted), ('dx', norm_learn(x, 4, weight, bias, activation, dy)['dx'])):
            result = found[name].clone()
            assert bool(torch.isnan(result[0, ..., each:2 * each]).all()), (name, activation)
            result[0, ..., each:2 * each] = clean[0, ..., each:2 * each]
            assert torch.equal(result, clean), (name, activation)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('far', [30.0, 1000.0])
@pytest.mark.parametrize('shape', [(2, 8, 8, 16), (1, 72, 96, 32), (2, 72, 96, 16), (1, 512, 512, 16), (1, 40, 40, 700)])
def test_a_pixel_that_stands_out(shape, far, dtype):
    # A corner many deviations from the rest, in maps that are held and that are cut: as exact as without it, for
    # squares are taken about a mean.
    x, weight, bias, dy = norm_inputs(shape, dtype, 9)
    for at in ((0, 0), (shape[1] - 1, shape[2] // 2)):
        spoilt = x.clone()
        spoilt[:, at[0], at[1]] = far
        found = norm_learn(spoilt, 4, weight, bias, 'silu', dy)
        exact = exact_norm(spoilt, 4, weight, bias, activation='silu', dy=dy)
        for name, each in found.items():
            close(each, exact[name], VALUES if name == 'y' else GRADIENTS, exact['terms'] if name == 'dx' else 0.0)


# Maps, pixels, channels and groups: an update's small maps (4,096 matches of 64 steps), acting for 16,384 matches of
# 11 agents, and maps that are cut and whose many groups have a kernel for their statistics.
@pytest.mark.parametrize('sizes', [(262144, 3, 64, 16), (180224, 2, 32, 32), (16500, 33, 256, 256)])
def test_group_norm_of_many_maps_and_groups(sizes):
    from cuju_amd import layers
    maps, pixels, channels, groups = sizes
    x = torch.randn(maps, pixels, channels, device='cuda', dtype=torch.bfloat16)
    dy = torch.randn(maps, pixels, channels, device='cuda', dtype=torch.bfloat16)
    weight, bias = torch.rand(channels, device='cuda') + 0.5, torch.randn(channels, device='cuda')
    found = norm_learn(x, groups, weight, bias, 'silu', dy)
    # The first, some and the last against the definition, and all against calls of half the maps.
    some = torch.tensor([0, 1, maps // 3, maps - 2, maps - 1], device='cuda')
    exact = exact_norm(x[some], groups, weight, bias, activation='silu', dy=dy[some])
    close(found['y'][some], exact['y'], VALUES)
    close(found['dx'][some], exact['dx'], GRADIENTS, exact['terms'])
    half = maps // 2
    parts = [norm_learn(x[at], groups, weight, bias, 'silu', dy[at]) for at in (slice(0, half), slice(half, None))]
    assert torch.equal(found['y'], torch.cat([p['y'] for p in parts]))
    assert torch.equal(found['dx'], torch.cat([p['dx'] for p in parts]))
    for name in ('d_weight', 'd_bias'):
        close(found[name], sum(p[name].double() for p in parts).cpu(), GRADIENTS)


@pytest.mark.parametrize('shape', [(3, 8, 8, 16), (2, 72, 96, 16)])
def test_group_norm_gradients_that_are_asked_for(shape, monkeypatch):
    from cuju_amd import layers
    x, weight, bias, dy = norm_inputs(shape, torch.float32, 10)
    wanted = norm_learn(x, 4, weight, bias, 'silu', dy)
    given, packed, call = {'dx': x, 'd_weight': weight, 'd_bias': bias}, [], layers._call
    monkeypatch.setattr(layers, '_call', lambda *a: (packed.append(layers._NORM.unpack(a[1])), call(*a)))
    for asked in (('dx',), ('dx', 'd_weight'), ('d_bias',), ('d_weight', 'd_bias')):
        leaves = [t.detach().requires_grad_(name in asked) for name, t in given.items()]
        y = layers.group_norm(leaves[0], 4, leaves[1], leaves[2], activation='silu')
        y.backward(dy)
        for name, leaf in zip(given, leaves):
            assert torch.equal(leaf.grad, wanted[name]) if name in asked else leaf.grad is None
        # No sums of channels that nobody wants.
        assert [bool(p) for p in packed[-1][-2:]] == ['d_weight' in asked, 'd_bias' in asked]


# --------------------------------------------------------------- delta rule: steps that are not finite

def spoil(x, steps, bad):
    """`x` with one of its values at the given (sequence, step) places not finite."""
    x = x.clone()
    for i, (b, t) in enumerate(steps):
        at = x[b, t].view(-1)
        at[(7 * i + 3) % at.numel()] = bad
    return x


# Sequence and step: in a first chunk, in a later one, two in one chunk, in the first and in the last step.
SPOILT = [(1, 5), (2, 21), (3, 18), (3, 27), (4, 0), (5, 40)]


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('name', ['query', 'key', 'value', 'decay', 'beta'])
@pytest.mark.parametrize('heads, key_size, value_size, dtype', [
    (2, 48, 40, torch.float32), (2, 128, 128, torch.float32), (3, 33, 21, torch.float16), (190, 64, 64, torch.bfloat16),
    (190, 16, 32, torch.float16)])
def test_outputs_before_a_step_that_is_not_finite(heads, key_size, value_size, dtype, name, bad):
    # As in the definition, and in acting: it reaches its own step and the later ones of its episode, no step before.
    given = inputs(6, 41, 1, heads, key_size, value_size, dtype=dtype, seed=22)
    given['resets'] = torch.zeros(6, 41, dtype=torch.bool, device='cuda')
    given['resets'][2, 30] = given['resets'][3, 25] = True
    given[name] = spoil(given[name], SPOILT, bad)
    output, last = rule(given)
    exact = exact_rule(**given)
    for found, wanted in ((output, exact[0]), (last, exact[1])):
        finite = torch.isfinite(wanted)
        assert torch.equal(torch.isfinite(found).cpu(), finite)
        zero = torch.zeros((), dtype=torch.double)
        close(torch.where(finite, found.cpu(), zero.to(found.dtype)), torch.where(finite, wanted, zero), VALUES)


@pytest.mark.parametrize('step', [0, 15, 16, 31, 32, 40, 63, 64, 95, 99])
def test_outputs_before_a_step_that_is_not_finite_in_training(step):
    # With the memories kept for the gradients, from which the outputs are found again.
    given = inputs(3, 100, 1, 2, 48, 40, seed=29)
    given['value'][1, step, 1, 7] = given['key'][2, step, 0, 3] = float('nan')
    output, last = rule(given, value=given['value'].clone().requires_grad_())
    exact = exact_rule(**given)
    for found, wanted in ((output, exact[0]), (last, exact[1])):
        found, finite = found.detach().cpu(), torch.isfinite(wanted)
        assert torch.equal(torch.isfinite(found), finite)
        close(torch.where(finite, found, 0.0), torch.where(finite, wanted, 0.0), VALUES)


def test_a_memory_that_is_not_finite_reaches_its_columns():
    given = inputs(3, 50, 1, 2, 32, 48, seed=23)
    given['state'][1, 1, 3, 17] = float('nan')
    given['state'][2] = float('nan')
    given['resets'] = torch.zeros(3, 50, dtype=torch.bool, device='cuda')
    given['resets'][2, 44] = True
    output, last = rule(given)
    exact = exact_rule(**given)
    for found, wanted in ((output, exact[0]), (last, exact[1])):
        finite = torch.isfinite(wanted)
        assert torch.equal(torch.isfinite(found).cpu(), finite)
        close(torch.where(finite, found.cpu(), 0.0), torch.where(finite, wanted, 0.0), VALUES)


@pytest.mark.parametrize('bad', [0.0, float('nan')])
def test_a_memory_put_down_where_it_was_taken(bad):
    # The library takes one buffer for the memory before and after.
    from cuju_amd import layers
    given = inputs(3, 50, 1, 2, 32, 48, seed=30)
    given['value'][1, 21, 0, 5] = bad
    wanted, last = rule(given)
    memory, output = given['state'].clone(), torch.empty_like(given['value'])
    layers._call('cuju_delta_rule_forward',
                 layers._rule(given['query'], given['key'], given['value'], given['decay'], given['beta'], memory, None,
                              32 ** -0.5, output, memory), memory.device)
    assert torch.equal(output.nan_to_num(nan=1e30), wanted.nan_to_num(nan=1e30))
    # Of the sequence that is played again the memory is that of single steps.
    assert torch.equal(memory[::2], last[::2]) and torch.equal(torch.isnan(memory[1]), torch.isnan(last[1]))
    close(memory[1].nan_to_num(nan=0.0), last[1].nan_to_num(nan=0.0).double().cpu(), VALUES)


def test_a_sequence_of_nothing_finite_ends():
    # Long ones are passed over once their memory is lost.
    given = inputs(8, 2000, 2, 2, 64, 64, dtype=torch.bfloat16, seed=24)
    given['key'] = torch.full_like(given['key'], float('nan'))
    output, last = rule(given)
    assert bool(torch.isnan(output).all()) and bool(torch.isnan(last).all())


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_a_later_episode_does_not_reach_an_earlier_one(bad):
    given = inputs(3, 60, 1, 2, 48, 40, seed=25)
    given['resets'] = torch.zeros(3, 60, dtype=torch.bool, device='cuda')
    starts = ((0, 32), (1, 21), (2, 37))
    for b, t in starts:
        given['resets'][b, t] = True
    spoilt = {n: x.clone() for n, x in given.items()}
    for b, t in starts:
        for name in ('query', 'key', 'value', 'decay', 'beta'):
            spoilt[name][b, t:] = bad
    clean, d_output, d_last = learn(given)
    bad_d_output, bad_d_last = d_output.clone(), torch.full_like(d_last, bad)
    for b, t in starts:
        bad_d_output[b, t:] = bad
    found, _, _ = learn(spoilt, bad_d_output, bad_d_last)
    for b, t in starts:
        for name in ('output', 'd_query', 'd_key', 'd_value', 'd_decay', 'd_beta'):
            assert torch.equal(found[name][b, :t], clean[name][b, :t]), name
    assert torch.equal(found['d_state'], clean['d_state'])


# ------------------------------------------------------- kernels that many heads and other sizes choose

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('key_size, value_size', [(32, 64), (32, 32), (64, 64), (64, 72), (64, 128), (96, 64), (128, 128), (128, 100)])
def test_gradients_of_many_heads(key_size, value_size, dtype):
    # Enough heads for the widest pieces of the memory, with last pieces that are not whole, kept memories and resets.
    # Heads are independent, so some stand for all.
    given = inputs(1100, 70, 1, 1, key_size, value_size, dtype=dtype, seed=26 + key_size + value_size, episode=25)
    found, d_output, d_last = learn(given)
    some = torch.cat([torch.arange(0, 1100, 61), torch.tensor([1023, 1024, 1099])])
    exact = exact_rule(**{n: x[some.cuda()] for n, x in given.items()}, d_output=d_output[some.cuda()], d_last=d_last[some.cuda()])
    for name, x in found.items():
        assert bool(torch.isfinite(x).all()), name
        close(x[some.cuda()], exact[name], GRADIENTS if name.startswith('d_') else VALUES)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('value_size', [4, 12, 16, 20, 32, 48])
def test_a_step_of_few_columns(value_size, dtype):
    from cuju_amd import layers
    for key_size in (32, 64, 128):
        given = inputs(9, 1, 1, 2, key_size, value_size, dtype=dtype, seed=27 + key_size + value_size)
        state = given['state'].clone()
        output = layers.delta_rule_step(*[given[n].squeeze(1) for n in ('query', 'key', 'value', 'decay', 'beta')], state)
        exact = exact_rule(**given)
        close(output, exact[0][:, 0], VALUES)
        close(state, exact[1], VALUES)


@pytest.mark.parametrize('shape, groups', [((2, 26, 26, 64), 8), ((3, 30, 20, 48), 2), ((2, 36, 36, 24), 2)])
def test_group_norm_of_maps_in_two_slabs(shape, groups):
    x, weight, bias, dy = norm_inputs(shape, torch.float32, 11)
    found = norm_learn(x, groups, weight, bias, 'silu', dy)
    exact = exact_norm(x, groups, weight, bias, activation='silu', dy=dy)
    for name, each in found.items():
        close(each, exact[name], GRADIENTS, exact['terms'] if name == 'dx' else 0.0)


# ---------------------------------------------------------------------- training in a graph, recomputed

def test_gradients_in_a_graph():
    given = inputs(4, 70, 1, 2, 32, 40, dtype=torch.bfloat16, seed=28, episode=20)
    x, weight, bias, dy = norm_inputs((3, 72, 96, 16), torch.bfloat16, 12)

    def train():
        found, d_output, d_last = learn(given, given_d[0], given_d[1])
        return [*found.values(), *norm_learn(x, 4, weight, bias, 'silu', dy).values()]

    _, *given_d = learn(given)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = train()
    for scale in (1.0, 0.5, -2.0):
        for each in (*given_d, dy):
            each.mul_(scale)
        wanted = train()
        for each in found:
            each.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(found, wanted))


def test_selective_recomputation():
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    seen = []

    def policy(context, operator, *args, **kwargs):
        if operator.name().startswith('cuju_amd'):
            seen.append(operator.name())
            return CheckpointPolicy.MUST_SAVE
        return CheckpointPolicy.PREFER_RECOMPUTE

    def recomputed(call):
        return lambda *t: checkpoint(lambda *u: call(*u), *t, use_reentrant=False,
                                     context_fn=lambda: create_selective_checkpoint_contexts(policy))

    for call, tensors in small_calls()[:2]:
        found, wanted = (gradients_of(each)(*tensors) for each in (recomputed(call), call))
        assert all(torch.equal(a, b) for a, b in zip(found, wanted))
    assert {'cuju_amd::group_norm', 'cuju_amd::delta_rule'} <= set(seen)
