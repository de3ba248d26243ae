"""Linear attention with decays against its definition in 64 bits (tests/block_oracle.py).

Tolerances, in the 2-norm. An element of the memory is a sum of at most 400 steps and an output one of at most 160
terms. Rounding errors of 2^-24 of a sum's parts, of either sign, leave it off by 2^-24 of the 2-norm of its terms times the
root of their number, which is more than that of its own size where terms cancel: (sqrt(400) + sqrt(160)) 2^-24 =
2e-6, and with the factors' 2^-23 under 3e-6 of the terms. A gradient takes two such chains, under 6e-6. A result rounded
once to bfloat16 or float16 is off by at most 2^-8 or 2^-11 of its size, and its products may take memories and
scores to 16 bits, 2^-15 of the terms. A decay's gradient is a sum over at most 128 steps of the differences of two such
dots: the 2-norm of the sums of errors is at most sqrt(128) times that of the errors, 12 x 6e-6 of all dots' terms.
"""

import pytest
import torch

from block_oracle import attention as exact_attention
from block_oracle import attention_terms

pytestmark = pytest.mark.gpu

VALUES, GRADIENTS = 3e-6, 6e-6
ROUNDING = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
PIECES = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -15, torch.float16: 2.0 ** -15}
DECAYS = 12 * GRADIENTS
TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = 'query', 'key', 'value', 'decay', 'state'


def close(found, exact, bound, terms):
    """`terms`: the 2-norm of the terms that the result is a sum of."""
    found = found.detach()
    exact = exact.reshape(found.shape)
    assert bool(torch.isfinite(found).all())
    error, size = float((found.double() - exact).norm()), float(exact.norm())
    allowed = (bound + PIECES[found.dtype]) * max(terms, size) + ROUNDING[found.dtype] * size
    assert error <= allowed + 1e-30, f'{error:.3g} off, {allowed:.3g} allowed'


def bound_of(name):
    return DECAYS if name == 'd_decay' else GRADIENTS if name.startswith('d_') else VALUES


def all_close(found, exact, terms, names=None):
    for name in names or found:
        if found[name].numel():
            close(found[name], exact[name], bound_of(name), terms[name])


def forward_close(found, given, **changes):
    """Outputs and last memory of a call on `given`."""
    given = {**given, **changes}
    all_close(dict(zip(('output', 'last'), found)), dict(zip(('output', 'last'), exact_attention(**given))), attention_terms(**given))


def inputs(batch, time, key_heads, heads, key_size, value_size, dtype=torch.float32, seed=0, episode=0, state=True, fixed=False):
    """Unit keys that keep a direction of their own, decays of all reaches, and a memory."""
    generator = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=generator)

    def directions():
        x = normal(batch, time, key_heads, key_size) + normal(batch, 1, key_heads, key_size)
        return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)

    reach = torch.logspace(-3, 0.3, heads)
    given = {'query': directions().to(dtype), 'key': directions().to(dtype),
             'value': normal(batch, time, heads, value_size).to(dtype),
             'decay': -reach if fixed else -reach * torch.nn.functional.softplus(normal(batch, time, heads)),
             'state': normal(batch, heads, key_size, value_size) if state else None,
             'resets': torch.rand(batch, time, generator=generator) < 1 / episode if episode else None}
    return {name: x.cuda() if x is not None else None for name, x in given.items()}


def attend(given, **changes):
    from cuju_amd import layers
    given = {**given, **changes}
    return layers.linear_attention(given['query'], given['key'], given['value'], given['decay'], state=given['state'],
                                   resets=given['resets'])


def learn(given, d_output=None, d_last=None, seed=5):
    """Outputs and gradients of a training pass, and the outputs' gradients it was given."""
    generator = torch.Generator().manual_seed(seed)
    leaves = {n: given[n].detach().requires_grad_() for n in NAMES if given[n] is not None}
    output, last = attend(given, **leaves)
    if d_output is None:
        d_output = torch.randn(output.shape, generator=generator).to(output.dtype).cuda()
    if d_last is None:
        d_last = torch.randn(last.shape, generator=generator).cuda()
    found = torch.autograd.grad([output, last], list(leaves.values()), [d_output, d_last])
    return {'output': output, 'last': last, **{'d_' + n: g for n, g in zip(leaves, found)}}, d_output, d_last


def learn_close(given):
    found, d_output, d_last = learn(given)
    d = {'d_output': d_output, 'd_last': d_last}
    all_close(found, exact_attention(**given, **d), attention_terms(**given, **d))
    return found


def step_of(given, t=0):
    """The arguments of a step."""
    return [given[n][:, t] if n != 'decay' or given[n].dim() == 3 else given[n] for n in ('query', 'key', 'value', 'decay')]


# batch, time, key heads, heads, key size, value size, steps of an episode
SIZES = [
    (1, 1, 1, 1, 1, 1, 0),
    (3, 1, 2, 2, 64, 64, 0),
    (2, 15, 1, 3, 16, 33, 0),
    (2, 16, 2, 4, 32, 16, 4),
    (2, 17, 3, 3, 33, 48, 0),
    (2, 31, 1, 1, 20, 100, 7),
    (2, 32, 1, 2, 64, 64, 0),
    (3, 33, 1, 2, 64, 64, 9),
    (2, 64, 2, 2, 64, 128, 30),
    (2, 128, 2, 2, 96, 65, 0),
    (1, 129, 1, 4, 128, 128, 50),
    (5, 200, 2, 2, 40, 72, 3),
    (2, 130, 1, 1, 100, 20, 1),
    (1, 385, 1, 2, 64, 32, 0),
    (2, 300, 2, 6, 48, 80, 20),
]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', SIZES)
def test_values_and_gradients(sizes, dtype):
    learn_close(inputs(*sizes[:6], dtype=dtype, seed=sum(sizes), episode=sizes[6], state=sizes[1] % 2 == 1))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', [(2, 40, 1, 3, 32, 32, 9), (3, 260, 2, 4, 64, 64, 100), (1, 129, 1, 1, 20, 24, 0)])
def test_a_decay_of_each_head(sizes, dtype):
    given = inputs(*sizes[:6], dtype=dtype, seed=sum(sizes), episode=sizes[6], fixed=True)
    assert given['decay'].shape == (sizes[3],)
    found = learn_close(given)
    # The same as one that is given for every step.
    wide = {**given, 'decay': given['decay'].expand(sizes[0], sizes[1], sizes[3])}
    for name, x in learn(wide)[0].items():
        if name != 'd_decay':
            assert torch.equal(x, found[name]), name


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('key_size, value_size', [(16, 16), (32, 64), (32, 32), (64, 64), (64, 72), (64, 128), (96, 64), (128, 128), (128, 100)])
def test_many_heads(key_size, value_size, dtype):
    # Wide pieces of the memory, as many heads get them.
    learn_close(inputs(600, 40, 1, 2, key_size, value_size, dtype=dtype, seed=key_size + value_size, episode=15))


@pytest.mark.parametrize('heads', [300, 1100])
def test_many_heads_forward(heads):
    for value_size in (16, 30, 64, 100):
        given = inputs(heads, 20, 1, 1, 24, value_size, seed=heads + value_size, episode=15)
        forward_close(attend(given), given)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('time', [255, 256, 257, 400])
@pytest.mark.parametrize('batch', [1, 130])
def test_long_sequences_of_few_and_many_heads(batch, time, dtype):
    given = inputs(batch, time, 1, 1, 32, 128, dtype=dtype, seed=time + batch, episode=150)
    forward_close(attend(given), given)
    learn_close(given)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', [(1, 1, 1, 1, 1), (7, 2, 6, 40, 72), (5, 3, 3, 64, 64), (3, 1, 2, 128, 128),
                                   (9, 2, 2, 17, 5), (4, 1, 1, 100, 30), (3, 2, 2, 64, 16), (3, 2, 2, 64, 32)])
def test_a_step_is_one_step(sizes, dtype):
    from cuju_amd import layers
    batch, key_heads, heads, key_size, value_size = sizes
    for fixed in (False, True):
        given = inputs(batch, 1, key_heads, heads, key_size, value_size, dtype=dtype, seed=sum(sizes), fixed=fixed)
        for resets in (None, torch.arange(batch, device='cuda') % 2 == 0):
            state = given['state'].clone()
            output = layers.linear_attention_step(*step_of(given), state, resets=resets)
            forward_close((output[:, None], state), given, resets=resets[:, None] if resets is not None else None)


def test_steps_one_by_one_follow_the_whole():
    from cuju_amd import layers
    given = inputs(6, 70, 2, 4, 64, 64, seed=3, episode=20)
    state = given['state'].clone()
    outputs = [layers.linear_attention_step(*step_of(given, t), state, resets=given['resets'][:, t]) for t in range(70)]
    forward_close((torch.stack(outputs, 1), state), given)


def test_a_memory_carried_over_pieces_is_the_whole():
    given = inputs(3, 90, 2, 2, 64, 48, seed=4, episode=25)
    state, outputs = given['state'], []
    for low, high in ((0, 1), (1, 30), (30, 30), (30, 90)):
        piece = {n: x[:, low:high] for n, x in given.items() if n != 'state'}
        output, state = attend(piece, state=state)
        outputs.append(output)
    forward_close((torch.cat(outputs, 1), state), given)


@pytest.mark.parametrize('decay', [0.0, 0.01, -30.0, -200.0, -1e30, -float('inf')])
def test_extreme_decays(decay):
    given = inputs(2, 150, 2, 2, 32, 32, seed=7)
    given['decay'][:, 5::9] = decay
    given['decay'][0, 40:44] = decay
    given['decay'][1, 127:129] = decay
    found, d_output, d_last = learn(given)
    # The definition with a factor of 0 where 32 bits have none.
    given = {**given, 'decay': given['decay'].clamp_min(-700), 'd_output': d_output, 'd_last': d_last}
    all_close(found, exact_attention(**given), attention_terms(**given))


def test_factors_past_one():
    # Memories that grow by e^20 on the way, and by e^80 at one step of a head that holds nothing yet. (e^100 is 3e43, more
    # than 32 bits hold, 3.4e38: times a memory of zeros it is no number.)
    given = inputs(2, 50, 1, 2, 32, 32, seed=8, state=False)
    given['decay'][:] = 0.4
    given['decay'][:, 0] = 80.0
    learn_close(given)


def test_keys_and_values_of_zero():
    given = inputs(2, 40, 1, 2, 32, 32, seed=8)
    given['value'][:, ::3] = 0
    given['key'][:, 7:9] = 0
    learn_close(given)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_nothing_crosses_a_reset(bad, dtype):
    from cuju_amd import layers
    given = inputs(4, 160, 1, 2, 48, 40, dtype=dtype, seed=9)
    resets = torch.zeros(4, 160, dtype=torch.bool, device='cuda')
    resets[0, 0] = resets[1, 21] = resets[2, 37] = resets[3, 140] = True
    given['resets'] = resets
    places = ((0, 0), (1, 21), (2, 37), (3, 140))
    spoilt = {n: x.clone() for n, x in given.items()}
    spoilt['state'][:] = bad
    for b, t in places:
        for name in ('query', 'key', 'value', 'decay'):
            spoilt[name][b, :t] = bad
    wanted, d_output, d_last = learn(given)
    exact = exact_attention(**given, d_output=d_output, d_last=d_last)
    terms = attention_terms(**given, d_output=d_output, d_last=d_last)
    for found in (learn(spoilt, d_output, d_last)[0], dict(zip(('output', 'last'), attend(spoilt)))):
        for b, t in places:
            for name, x in found.items():
                if name != 'd_state':
                    low = 0 if name == 'last' else t
                    close(x[b][low:], exact[name][b][low:], bound_of(name), terms[name])
    found = learn(spoilt, d_output, d_last)[0]
    assert not bool(found['d_state'][0].any())
    # Neither backwards: what comes after a reset does not reach the gradients before it.
    late = {n: x.clone() for n, x in given.items()}
    for b, t in places[1:]:
        for name in ('query', 'key', 'value', 'decay'):
            late[name][b, t:] = bad
    found = learn(late, d_output, d_last)[0]
    for b, t in places[1:]:
        for name in ('output', 'd_query', 'd_key', 'd_value', 'd_decay'):
            close(found[name][b, :t], exact[name][b, :t], bound_of(name), terms[name])
        close(found['d_state'][b], exact['d_state'][b], GRADIENTS, terms['d_state'])
    state = torch.full_like(given['state'], bad)
    output = layers.linear_attention_step(*step_of(given), state, resets=torch.ones(4, dtype=torch.bool, device='cuda'))
    assert bool(torch.isfinite(output).all()) and bool(torch.isfinite(state).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('name', ['query', 'key', 'value', 'decay'])
@pytest.mark.parametrize('heads, time', [(7, 100), (7, 300), (700, 70)])
def test_outputs_before_a_step_that_is_not_finite(heads, time, name, bad, dtype):
    given = inputs(heads, time, 1, 1, 32, 64, dtype=dtype, seed=23)
    wanted = attend(given)[0]
    steps = [0, 15, 16, 31, 50, min(128, time - 2), time - 1]
    spoilt = given[name].clone()
    for b, t in enumerate(steps):
        spoilt[b, t, 0] = bad
    output = attend(given, **{name: spoilt})[0]
    exact, terms = exact_attention(**given)[0], attention_terms(**given)['output']
    for b, t in enumerate(steps):
        if t:
            close(output[b, :t], exact[b, :t], VALUES, terms)
        if name == 'query':
            assert not bool(torch.isfinite(output[b, t]).any())
            if t + 1 < time:
                close(output[b, t + 1:], exact[b, t + 1:], VALUES, terms)
        else:
            assert not bool(torch.isfinite(output[b, t:]).any())
    if heads > len(steps):
        assert torch.equal(output[len(steps):], wanted[len(steps):])


def test_a_column_that_is_not_finite_stays_one():
    # An infinity in one column of the values reaches that column alone.
    given = inputs(3, 70, 1, 1, 32, 64, seed=24)
    spoilt = given['value'].clone()
    spoilt[1, 20, 0, 5] = float('inf')
    output, last = attend(given, value=spoilt)
    exact, terms = exact_attention(**given), attention_terms(**given)
    others = [c for c in range(64) if c != 5]
    close(output[..., others], exact[0][..., others], VALUES, terms['output'])
    close(last[..., others], exact[1][..., others], VALUES, terms['last'])
    assert not bool(torch.isfinite(output[1, 20:, 0, 5]).any())
    close(output[1, :20, 0, 5], exact[0][1, :20, 0, 5], VALUES, terms['output'])


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
    d = {'d_output': d_output, 'd_last': d_last}
    all_close(found, exact_attention(**given, **d), attention_terms(**given, **d))
    # Gradients that come as views: time first, and one value for all.
    moved, _, _ = learn(given, d_output.transpose(0, 1).contiguous().transpose(0, 1), d_last)
    for name in wanted:
        assert torch.equal(moved[name], wanted[name]), name
    one = torch.ones((), device='cuda')
    found, _, _ = learn(given, one.expand(d_output.shape), one.expand(d_last.shape))
    wanted, _, _ = learn(given, torch.ones_like(d_output), torch.ones_like(d_last))
    for name in wanted:
        assert torch.equal(found[name], wanted[name]), name


def test_a_step_with_strides():
    from cuju_amd import layers
    given = inputs(5, 3, 2, 4, 32, 24, seed=10)
    packed = torch.zeros(5, 4, 100, device='cuda')
    value = packed[..., 1:25]
    value.copy_(given['value'][:, 1])
    state, decay = given['state'].clone(), torch.stack([given['decay'][:, 1]] * 3, -1)[..., 1]
    resets = torch.zeros(5, 2, dtype=torch.uint8, device='cuda')
    resets[2] = 1
    output = layers.linear_attention_step(given['query'][:, 1], given['key'][:, 1], value, decay, state, resets=resets[:, 1])
    piece = {n: x[:, 1:2] for n, x in given.items() if n not in ('state', 'resets')}
    forward_close((output[:, None], state), {**piece, 'state': given['state'], 'resets': resets[:, 1:]})


def test_broadcast_inputs():
    # One query and key for the whole batch: their gradients are the batch's sum.
    given = inputs(3, 33, 2, 2, 32, 32, seed=11)
    query, key = (given[n][:1].clone().requires_grad_() for n in ('query', 'key'))
    output, last = attend(given, query=query.expand(3, -1, -1, -1), key=key.expand(3, -1, -1, -1))
    d_output, d_last = torch.randn_like(output), torch.randn_like(last)
    found = torch.autograd.grad([output, last], [query, key], [d_output, d_last])
    given['query'], given['key'] = query.detach().expand(3, -1, -1, -1), key.detach().expand(3, -1, -1, -1)
    d = {'d_output': d_output, 'd_last': d_last}
    exact, terms = exact_attention(**given, **d), attention_terms(**given, **d)
    for x, name in zip(found, ('d_query', 'd_key')):
        close(x, exact[name].sum(0, keepdim=True), GRADIENTS, terms[name])


@pytest.mark.parametrize('time', [70, 140])
def test_only_one_output_is_learnt_from(time):
    given = inputs(2, time, 1, 2, 32, 32, seed=12)
    for which in (0, 1):
        leaf, decay = (given[n].clone().requires_grad_() for n in ('value', 'decay'))
        outputs = attend(given, value=leaf, decay=decay)
        d = torch.randn_like(outputs[which])
        found = torch.autograd.grad(outputs[which], [leaf, decay], d)
        zeros = [torch.zeros_like(x) for x in outputs]
        zeros[which] = d
        d = {'d_output': zeros[0], 'd_last': zeros[1]}
        all_close(dict(zip(('d_value', 'd_decay'), found)), exact_attention(**given, **d), attention_terms(**given, **d))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', [(2, 70, 1, 3, 32, 48), (40, 140, 2, 2, 64, 64)])
def test_a_decay_that_is_not_learnt(sizes, dtype):
    given = inputs(*sizes, dtype=dtype, seed=13, episode=40)
    leaves = {n: given[n].clone().requires_grad_() for n in ('query', 'key', 'value', 'state')}
    output, last = attend(given, **leaves)
    d_output, d_last = torch.randn_like(output), torch.randn_like(last)
    found = torch.autograd.grad([output, last], list(leaves.values()), [d_output, d_last])
    d = {'d_output': d_output, 'd_last': d_last}
    all_close({'d_' + n: x for n, x in zip(leaves, found)}, exact_attention(**given, **d), attention_terms(**given, **d))


def test_gates_in_other_types():
    from cuju_amd import layers
    given = inputs(2, 20, 1, 2, 32, 32, dtype=torch.bfloat16, seed=13)
    for decay in (given['decay'].to(torch.bfloat16), given['decay'].double(), given['decay'][0, 0].half(), given['decay'][0, 0].double()):
        decay.requires_grad_()
        output, last = attend(given, decay=decay)
        d_output, d_last = torch.randn_like(output), torch.randn_like(last)
        found, = torch.autograd.grad([output, last], [decay], [d_output, d_last])
        assert found.dtype == decay.dtype and found.shape == decay.shape
        held = {**given, 'decay': decay.float(), 'd_output': d_output, 'd_last': d_last}
        all_close({'d_decay': found if found.dtype != torch.double else found.float()}, exact_attention(**held), attention_terms(**held))
        scaled = layers.linear_attention(given['query'], given['key'], given['value'], decay.detach(), scale=3.0)
        forward_close(scaled, given, decay=decay.float(), state=None, scale=3.0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('scale', [-0.7, 0.0])
def test_scales_that_are_not_positive(scale, dtype):
    from cuju_amd import layers
    given = inputs(2, 300, 1, 2, 32, 48, dtype=dtype, seed=29, episode=25)
    leaves = {n: given[n].detach().requires_grad_() for n in NAMES}
    output, last = layers.linear_attention(*[leaves[n] for n in NAMES[:4]], state=leaves['state'], resets=given['resets'], scale=scale)
    forward_close((output, last), given, scale=scale)
    d_output, d_last = torch.randn_like(output), torch.randn_like(last)
    found = torch.autograd.grad([output, last], list(leaves.values()), [d_output, d_last])
    d = {'d_output': d_output, 'd_last': d_last, 'scale': scale}
    all_close({'d_' + n: x for n, x in zip(leaves, found)}, exact_attention(**given, **d), attention_terms(**given, **d))


def test_empty_batches_and_times():
    from cuju_amd import layers
    for batch, time in ((0, 5), (3, 0), (0, 0)):
        for fixed in (False, True):
            given = inputs(batch, time, 1, 2, 32, 16, seed=14, fixed=fixed)
            found, d_output, d_last = learn(given)
            assert found['output'].shape == (batch, time, 2, 16) and found['d_query'].shape == (batch, time, 1, 32)
            assert torch.equal(found['last'], given['state'])
            assert torch.equal(found['d_state'], d_last)
            assert found['d_decay'].shape == given['decay'].shape and not bool(found['d_decay'].any())
    given = inputs(3, 0, 1, 2, 32, 16, state=False)
    assert not bool(attend(given)[1].any())
    empty = inputs(0, 1, 1, 2, 32, 16)
    output = layers.linear_attention_step(*step_of(empty), empty['state'])
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
    # Two steps of one. They are too far apart to be played together, and one after the other their sums are taken in another
    # order: the bounds of rounding hold, not equality.
    given = inputs(1, 2, 1, 1, 32, 32, dtype=torch.bfloat16, seed=15)
    _, d_output, d_last = learn(given)
    d = {'d_output': d_output, 'd_last': d_last}
    for name in ('query', 'key', 'value'):
        view = room.as_strided((1, 2, 1, 32), (32, apart, 32, 1))
        view.copy_(given[name])
        found, _, _ = learn({**given, name: view}, d_output, d_last)
        all_close(found, exact_attention(**given, **d), attention_terms(**given, **d))


@pytest.mark.parametrize('dtype', TYPES)
def test_the_widest_steps_that_are_played_together(dtype):
    stride = (1 << 26) // dtype.itemsize - 8
    given = inputs(1, 60, 1, 1, 64, 32, dtype=dtype, seed=30, episode=25)
    room = torch.empty(60 * stride, dtype=dtype, device='cuda')
    wanted, d_output, d_last = learn(given)
    for name in ('query', 'key', 'value'):
        size = given[name].shape[-1]
        view = room.as_strided((1, 60, 1, size), (size, stride, size, 1))
        view.copy_(given[name])
        found, _, _ = learn({**given, name: view}, d_output, d_last)
        for n in wanted:
            assert torch.equal(found[n], wanted[n]), (name, n)


def test_calls_repeat_bit_for_bit():
    for fixed in (False, True):
        given = inputs(30, 200, 2, 4, 64, 64, dtype=torch.bfloat16, seed=16, episode=30, fixed=fixed)
        first, d_output, d_last = learn(given)
        for _ in range(3):
            again, _, _ = learn(given, d_output, d_last)
            for name in first:
                assert torch.equal(first[name], again[name]), name


@pytest.mark.parametrize('fixed', [False, True])
def test_gradients_against_differences(fixed):
    # A central difference along a direction, h = 2^-6: rounding leaves 64 * 2 * 3e-6 of the loss's
    # terms, the third derivative h^2 of them: 1e-3 of the size of the terms.
    given = inputs(2, 140, 1, 2, 24, 24, seed=17, episode=50, fixed=fixed)
    found, d_output, d_last = learn(given)
    generator = torch.Generator().manual_seed(1)

    def loss(changed):
        output, last = attend({**given, **changed})
        return float((output.double() * d_output.double()).sum() + (last.double() * d_last.double()).sum())

    for name in NAMES:
        x = given[name]
        along = torch.randn(x.shape, generator=generator).cuda()
        along /= along.norm()
        h = 2.0 ** -6 if name != 'decay' or not fixed else 2.0 ** -12
        difference = (loss({name: x + h * along}) - loss({name: x - h * along})) / (2 * h)
        slope = float((found['d_' + name].double() * along.double()).sum())
        size = float(found['d_' + name].double().norm())
        # The decay of a head moves every step: a smaller step, and what rounding leaves of a loss of that size.
        extra = 2.0 ** 12 * 3e-6 * float(d_output.norm()) if h < 2.0 ** -6 else 0.0
        assert abs(difference - slope) <= 1e-3 * size + 1e-3 * abs(slope) + extra, name


def test_on_another_stream_and_in_a_graph():
    from cuju_amd import layers
    given = inputs(4, 300, 1, 2, 64, 64, dtype=torch.bfloat16, seed=18, episode=40)
    wanted = attend(given)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        found = attend(given)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(found[0], wanted[0]) and torch.equal(found[1], wanted[1])
    at, state = step_of(given), given['state'].clone()
    with torch.cuda.stream(side):
        layers.linear_attention_step(*at, state.clone()), attend(given)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        output = layers.linear_attention_step(*at, state)
        replayed = attend(given)
    # A second graph of the same pool: its workspaces are its own.
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        second = attend(given)
    eager = given['state'].clone()
    state.copy_(given['state'])
    for _ in range(4):
        graphs[0].replay()
        expected = layers.linear_attention_step(*at, eager)
        torch.cuda.synchronize()
        assert torch.equal(output, expected) and torch.equal(state, eager)
        assert torch.equal(replayed[0], wanted[0]) and torch.equal(replayed[1], wanted[1])
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(second[0], wanted[0]) and torch.equal(second[1], wanted[1])


@pytest.mark.parametrize('fixed', [False, True])
def test_gradients_in_a_graph(fixed):
    given = inputs(4, 150, 1, 2, 32, 40, dtype=torch.bfloat16, seed=28, episode=40, fixed=fixed)
    _, *given_d = learn(given)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        learn(given, *given_d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = list(learn(given, *given_d)[0].values())
    for scale in (1.0, 0.5, -2.0):
        for each in given_d:
            each.mul_(scale)
        wanted = list(learn(given, *given_d)[0].values())
        for each in found:
            each.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(found, wanted))


# ------------------------------------------------------------ torch.compile, tracers, modes, refusals

@pytest.mark.parametrize('fixed', [False, True])
def test_compiled_calls_equal_eager_ones(fixed):
    from cuju_amd import layers
    torch._dynamo.reset()
    given = inputs(3, 140, 1, 2, 32, 32, seed=19, episode=20, fixed=fixed)

    def train(q, k, v, decay, state, resets):
        return layers.linear_attention(q, k, v, decay, state=state, resets=resets)

    def act(q, k, v, decay, state):
        return layers.linear_attention_step(q, k, v, decay, state)

    def play(train):
        leaves = [given[n].clone().requires_grad_() for n in NAMES] + [given['resets']]
        outputs = train(*leaves)
        sum((y.float() * (1 + i)).sum() for i, y in enumerate(outputs)).backward()
        return [*outputs, *[t.grad for t in leaves if t.requires_grad]]

    for found, wanted in zip(play(torch.compile(train, fullgraph=True, backend='aot_eager')), play(train)):
        assert torch.equal(found, wanted)
    states = [given['state'].clone() for _ in range(2)]
    compiled = torch.compile(act, fullgraph=True, backend='aot_eager')
    for _ in range(2):
        assert torch.equal(compiled(*step_of(given), states[0]), act(*step_of(given), states[1]))
    assert torch.equal(*states)


def small_call():
    from cuju_amd import layers
    given = inputs(2, 40, 1, 2, 16, 16, seed=20)
    return (lambda q, k, v, decay, state: layers.linear_attention(q, k, v, decay, state=state)), tuple(given[n] for n in NAMES)


def gradients_of(call):
    def learnt(*tensors):
        leaves = [x.detach().requires_grad_() for x in tensors]
        outputs = call(*leaves)
        return torch.autograd.grad(outputs, leaves, [torch.ones_like(y) for y in outputs])
    return learnt


def test_traced_graphs_compute():
    from torch.fx.experimental.proxy_tensor import make_fx
    call, tensors = small_call()
    other = [x * 0.5 for x in tensors]
    for each in (call, gradients_of(call)):
        graph = make_fx(lambda *t: each(*t))(*tensors)
        assert all(torch.equal(a, b) for a, b in zip(graph(*other), each(*other)))


def test_modes_see_the_gradients():
    from torch.utils._python_dispatch import TorchDispatchMode
    names = []

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, function, types, args=(), kwargs=None):
            names.append(function.name())
            return function(*args, **(kwargs or {}))

    call, tensors = small_call()
    wanted = gradients_of(call)(*tensors)
    with Seen():
        found = gradients_of(call)(*tensors)
    assert all(torch.equal(a, b) for a, b in zip(found, wanted))
    assert [n for n in names if n.startswith('cuju_amd')] == ['cuju_amd::linear_attention', 'cuju_amd::linear_attention_backward']


def test_refusals():
    from cuju_amd import ArgumentError, layers
    given = inputs(2, 4, 2, 4, 32, 32)

    def refused(**changes):
        with pytest.raises(ArgumentError):
            attend(given, **changes)

    refused(query=given['query'].cpu())
    refused(key=given['key'].cpu())
    refused(decay=given['decay'].cpu())
    refused(decay=given['decay'][0, 0].cpu())
    refused(query=given['query'].double())
    refused(key=given['key'].half())
    refused(key=given['key'][..., :16])
    refused(value=given['value'][:, :3])
    refused(value=given['value'][:, :, :3], decay=given['decay'][..., :3])
    refused(decay=given['decay'][..., :1])
    refused(decay=given['decay'][0, 0, :3])
    refused(decay=given['decay'][0])
    refused(decay=given['decay'].int())
    refused(decay=given['decay'][0, 0].int())
    refused(state=given['state'][:1])
    refused(resets=torch.zeros(2, 5, dtype=torch.bool, device='cuda'))
    refused(resets=torch.zeros(2, 4, device='cuda'))
    refused(query=given['query'][:, 0])
    wide = torch.zeros(2, 4, 2, 129, device='cuda')
    refused(query=wide, key=wide, state=None)
    at = step_of(given)
    for state in (None, given['state'].half(), given['state'].transpose(-1, -2), given['state'][:1]):
        with pytest.raises(ArgumentError):
            layers.linear_attention_step(*at, state)
    with pytest.raises(ArgumentError):
        layers.linear_attention_step(at[0].requires_grad_(), *at[1:], given['state'])
    value = given['value'].requires_grad_()
    gradient, = torch.autograd.grad(attend(given, value=value)[0].sum(), value, create_graph=True)
    with pytest.raises(RuntimeError):
        gradient.sum().backward()
