"""The norms of rows against their definitions in 64 bits (tests/block_oracle.py).

Tolerances, in the 2-norm relative to the result. In 32 bits a value is a product of at most ten factors, each rounded by
2^-24, with the root of a sum of squares in which a value meets at most 16 + 9 others one after the other, and a
sigmoid whose exponential is 8 x 2^-24 off for arguments up to 8: (10 + 25 / 2 + 8) 2^-24 = 1.8e-6 at worst, so under 2e-6. A
gradient takes two such chains, under 4e-6, and may be a small difference of larger terms, of which it is that. A result
rounded once to bfloat16 or float16 is off by at most 2^-8 or 2^-11 more.
"""

import pytest
import torch

from block_oracle import rows as exact_rows

pytestmark = pytest.mark.gpu

VALUES, GRADIENTS = 2e-6, 4e-6
ROUNDING = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(found, exact, bound, terms=0.0):
    found = found.detach()
    assert found.shape == exact.shape
    assert bool(torch.isfinite(found).all())
    error, size = float((found.double() - exact).norm()), float(exact.norm())
    allowed = bound * max(size, terms) + ROUNDING[found.dtype] * size
    assert error <= allowed + 1e-30, f'{error:.3g} off, {allowed:.3g} allowed'


def inputs(shape, dtype, seed=0):
    """Rows of their own levels, a gate, and vectors."""
    generator = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=generator)

    size = shape[-1]
    given = {'x': 2 * normal(*shape), 'block': normal(*shape) * normal(*shape[:-1], 1).exp(), 'gates': normal(*shape),
             'd_stream': normal(*shape), 'd_normed': normal(*shape)}
    given = {n: x.to(dtype).cuda() for n, x in given.items()}
    return {**given, **{n: (1 + 0.3 * normal(size)).cuda() for n in ('after', 'scale', 'before')}}


def call(given, names, activation='silu', epsilon=1e-6, **changes):
    """The outputs of the call that takes the inputs `names`, as a dictionary."""
    from cuju_amd import layers
    given = {**{n: given[n] for n in names}, **changes}
    if 'x' not in names:
        return {'stream': layers.rms_norm(given['block'], given.get('after'), given.get('gates'), epsilon=epsilon, activation=activation)}
    stream, normed = layers.residual_norm(given['x'], given['block'], given.get('before'), after=given.get('after'),
                                          gate=given.get('gates'), scale=given.get('scale', 1.0), epsilon=epsilon, activation=activation)
    return {'stream': stream, 'normed': normed}


def learn(given, names, activation='silu', of=('stream', 'normed'), **changes):
    """Outputs and gradients of a training pass that learns from the outputs `of`."""
    given = {**given, **changes}
    leaves = {n: given[n].detach().requires_grad_() for n in names}
    outputs = call(given, names, activation, **leaves)
    of = [n for n in of if n in outputs]
    found = torch.autograd.grad([outputs[n] for n in of], list(leaves.values()), [given['d_' + n] for n in of])
    return {**outputs, **{'d_' + n.replace('gates', 'gate'): g for n, g in zip(leaves, found)}}


def exact(given, names, activation='silu', of=('stream', 'normed'), epsilon=1e-6):
    return exact_rows(**{n: given[n] for n in names}, epsilon=epsilon, activation=activation,
                      norm_block='x' not in names or 'after' in names,
                      **{'d_' + n: given['d_' + n] for n in of if 'x' in names or n == 'stream'})


def learn_close(given, names, activation='silu', **options):
    found, wanted = learn(given, names, activation, **options), exact(given, names, activation, **options)
    for name, x in found.items():
        if not name.startswith('d_'):
            close(x, wanted[name], VALUES)
        else:
            close(x, wanted[name], GRADIENTS, wanted['terms'] if name in ('d_x', 'd_block') else 0.0)
    return found


ALL = ('x', 'block', 'gates', 'after', 'scale', 'before')
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 3, 8), (11, 4, 64), (33, 31), (9, 100), (4, 129), (37, 256), (6, 5, 257), (10, 512), (7, 1001),
          (5, 1024), (3, 1500), (5, 2048), (2, 3, 2049), (4, 4096), (3, 5001), (2, 8191), (3, 8192)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_rms_norm(shape, dtype):
    learn_close(inputs(shape, dtype, seed=sum(shape)), ('block', 'after', 'gates'))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_residual_norm(shape, dtype):
    learn_close(inputs(shape, dtype, seed=sum(shape)), ALL)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('activation', ['none', 'sigmoid', 'silu'])
@pytest.mark.parametrize('names', [('block',), ('block', 'after'), ('block', 'gates'), ('x', 'block'), ('x', 'block', 'before'),
                                   ('x', 'block', 'after'), ('x', 'block', 'gates'), ('x', 'block', 'gates', 'scale'),
                                   ('x', 'block', 'gates', 'after', 'before')])
def test_what_a_call_may_leave_out(names, activation, dtype):
    learn_close(inputs((13, 3, 72), dtype, seed=len(names)), names, activation)


@pytest.mark.parametrize('rows, size', [(50000, 64), (5000, 100), (3000, 1000), (2500, 2000), (2100, 4100)])
def test_many_rows(rows, size):
    # More rows than workgroups take at a time.
    given = inputs((rows, size), torch.bfloat16, seed=size)
    learn_close(given, ALL)
    learn_close(given, ('block', 'after', 'gates'))


@pytest.mark.parametrize('of', [('stream',), ('normed',)])
def test_only_one_output_is_learnt_from(of):
    given = inputs((9, 200), torch.float32, seed=3)
    # The norm's weight has no part in the stream.
    learn_close(given, ALL if of == ('normed',) else ALL[:-1], of=of)


@pytest.mark.parametrize('names', [('x',), ('block',), ('gates',), ('after',), ('scale',), ('before',), ('x', 'scale')])
def test_gradients_that_are_asked_for(names):
    given = inputs((40, 96), torch.float32, seed=4)
    leaves = {n: given[n].clone().requires_grad_() for n in names}
    outputs = call(given, ALL, **leaves)
    found = torch.autograd.grad(list(outputs.values()), list(leaves.values()), [given['d_' + n] for n in outputs])
    wanted = learn(given, ALL)
    for name, x in zip(names, found):
        assert torch.equal(x, wanted['d_' + name.replace('gates', 'gate')])


def test_scales_of_one_value():
    from cuju_amd import layers
    given = inputs((20, 48), torch.float32, seed=5)
    scale = torch.tensor(0.7, device='cuda', requires_grad=True)
    outputs = layers.residual_norm(given['x'], given['block'], scale=scale)
    found, = torch.autograd.grad(outputs, [scale], [given['d_stream'], given['d_normed']])
    wide = {**given, 'scale': torch.full((48,), 0.7, device='cuda')}
    wanted = exact(wide, ('x', 'block', 'scale'))
    for x, name in zip(outputs, ('stream', 'normed')):
        close(x, wanted[name], VALUES)
        assert torch.equal(x, layers.residual_norm(given['x'], given['block'], scale=float(scale.detach()))[name == 'normed'])
    close(found, wanted['d_scale'].sum(), GRADIENTS, float(wanted['d_scale'].norm()))


def test_strides_and_alignment():
    for size in (64, 65):
        given = inputs((6, 5, size), torch.bfloat16, seed=size)
        wanted = learn(given, ALL)
        # Heads of one projection at an odd offset, time before the batch, and one gate for all.
        packed = torch.zeros(6, 5 * 3 * size + 1, dtype=torch.bfloat16, device='cuda')
        views = {n: packed[:, 1 + 5 * size * i:1 + 5 * size * (i + 1)].unflatten(1, (5, size)) for i, n in enumerate(('x', 'block', 'gates'))}
        for name, view in views.items():
            view.copy_(given[name])
        found = learn(given, ALL, **views)
        assert all(torch.equal(found[n], wanted[n]) for n in wanted)
        moved = {n: given[n].transpose(0, 1).contiguous().transpose(0, 1) for n in ('x', 'block', 'gates', 'd_stream', 'd_normed')}
        found = learn(given, ALL, **moved)
        assert all(torch.equal(found[n], wanted[n]) for n in wanted)
        # Values that are not side by side, and an axis more.
        apart = {n: given[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ('x', 'block', 'gates')}
        found = learn(given, ALL, **apart)
        assert all(torch.equal(found[n], wanted[n]) for n in wanted)
        deep = {n: given[n].view(2, 3, 5, size) for n in ('x', 'block', 'gates', 'd_stream', 'd_normed')}
        deep['x'] = deep['x'].transpose(0, 1).contiguous().transpose(0, 1)
        found = learn(given, ALL, **deep)
        assert all(torch.equal(found[n].reshape(wanted[n].shape), wanted[n]) for n in wanted)
        one = given['gates'][:1, :1].clone().requires_grad_()
        y = call(given, ALL, gates=one.expand(6, 5, size))
        whole = call(given, ALL, gates=one.detach().expand(6, 5, size).contiguous())
        assert all(torch.equal(y[n], whole[n]) for n in y)
        d_one, = torch.autograd.grad(y['stream'], one, given['d_stream'])
        assert d_one.shape == one.shape


def test_vectors_of_rows():
    from cuju_amd import layers
    given = inputs((300,), torch.float32, seed=6)
    learn_close(given, ALL)
    column = given['block'].new_zeros(300, 2)[:, 1]
    column.copy_(given['block'])
    assert torch.equal(layers.rms_norm(column), layers.rms_norm(given['block']))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [40, 300, 3000])
def test_rows_of_zeros_and_large_values(size, dtype):
    given = inputs((6, size), dtype, seed=7)
    given['block'][0] = 0
    given['x'][1] = 0
    given['block'][1] = 0
    given['block'][2] *= 1000
    given['x'][3] *= 1000
    found = learn(given, ALL)
    wanted = exact(given, ALL)
    for row in range(6):
        for name in ('stream', 'normed', 'd_x', 'd_block', 'd_gate'):
            # A row of zeros has an inverse of 1000, and the gradient of what becomes of it that size: two of them one behind
            # the other reach 1e6, and past the largest number of the type, 65,504 in float16, the rounded result is infinite.
            x, y = found[name][row], wanted[name][row]
            held = y.abs() < torch.finfo(dtype).max
            assert torch.equal(x[~held].double(), y[~held].sign() * float('inf'))
            close(x[held], y[held], GRADIENTS, float((1000.0 if row < 2 else 0.0) * given['d_normed'].double().norm()))


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('name', ['x', 'block', 'gates'])
@pytest.mark.parametrize('size', [40, 600, 3000])
def test_a_row_that_is_not_finite_stays_one(size, name, bad):
    given = inputs((9, size), torch.bfloat16, seed=8)
    spoilt = given[name].clone()
    spoilt[4, 17] = bad
    found, wanted = learn(given, ALL, **{name: spoilt}), learn(given, ALL)
    others = [0, 1, 2, 3, 5, 6, 7, 8]
    for n in ('stream', 'normed', 'd_x', 'd_block', 'd_gate'):
        assert torch.equal(found[n][others], wanted[n][others])
    if name != 'block':
        columns = [c for c in range(size) if c != 17]
        assert torch.equal(found['stream'][4, columns], wanted['stream'][4, columns])
    elif bad != bad:
        assert not bool(torch.isfinite(found['stream'][4]).any())


def test_empty_rows():
    from cuju_amd import layers
    given = inputs((0, 4, 32), torch.bfloat16)
    for names in (ALL, ('block', 'after', 'gates')):
        found = learn(given, names)
        assert found['stream'].shape == (0, 4, 32)
        assert not any(bool(found[n].any()) for n in found)
    assert layers.rms_norm(torch.zeros(3, 0, 8, device='cuda')).shape == (3, 0, 8)


def test_offsets_past_32_bits():
    from cuju_amd import layers
    given = inputs((2, 3, 64), torch.bfloat16, seed=9)
    apart = (1 << 31) + 64
    room = torch.empty(apart + 3 * 64, dtype=torch.bfloat16, device='cuda')
    wanted = learn(given, ALL)
    for name in ('x', 'block', 'gates'):
        view = room.as_strided((2, 3, 64), (apart, 64, 1))
        view.copy_(given[name])
        found = learn(given, ALL, **{name: view})
        assert all(torch.equal(found[n], wanted[n]) for n in wanted)
    # More values than 32 bits count.
    rows = room[:(1 << 31) + 64].view(-1, 64)
    rows[:] = 1
    rows[-1] = torch.arange(64, device='cuda')
    y = layers.rms_norm(rows)
    assert torch.equal(y[-1], layers.rms_norm(rows[-1].clone())) and torch.equal(y[-2], layers.rms_norm(rows[0].clone()))


def test_weights_in_other_types():
    given = inputs((10, 64), torch.bfloat16, seed=10)
    given.update(after=given['after'].bfloat16(), scale=given['scale'].double(), before=given['before'].half())
    found = learn(given, ALL)
    assert [found['d_' + n].dtype for n in ('after', 'scale', 'before')] == [torch.bfloat16, torch.double, torch.half]
    wanted = exact({**given, 'scale': given['scale'].float()}, ALL)
    for name in ('stream', 'normed'):
        close(found[name], wanted[name], VALUES)


def test_calls_repeat_bit_for_bit():
    given = inputs((30000, 96), torch.bfloat16, seed=11)
    first = learn(given, ALL)
    for _ in range(3):
        again = learn(given, ALL)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_gradients_against_differences():
    # A central difference along a direction, h = 2^-6: rounding leaves 64 x 2e-6 of the loss's terms, the third derivative
    # h^2 of them: 1e-3 of the size of the terms.
    given = inputs((40, 130), torch.float32, seed=12)
    found = learn(given, ALL)
    generator = torch.Generator().manual_seed(1)

    def loss(**changes):
        outputs = call(given, ALL, **changes)
        return sum(float((outputs[n].double() * given['d_' + n].double()).sum()) for n in outputs)

    for name in ALL:
        x = given[name]
        along = torch.randn(x.shape, generator=generator).cuda()
        along /= along.norm()
        h = 2.0 ** -6
        difference = (loss(**{name: x + h * along}) - loss(**{name: x - h * along})) / (2 * h)
        gradient = found['d_' + name.replace('gates', 'gate')].double()
        slope = float((gradient * along.double()).sum())
        assert abs(difference - slope) <= 1e-3 * float(gradient.norm()) + 1e-3 * abs(slope), name


def test_on_another_stream_and_in_a_graph():
    given = inputs((70, 4, 64), torch.bfloat16, seed=13)
    wanted = learn(given, ALL)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        found = learn(given, ALL)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(found[n], wanted[n]) for n in wanted)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = learn(given, ALL)
    for scale in (1.0, 0.5, -2.0):
        given['block'].mul_(scale)
        given['d_normed'].mul_(scale)
        wanted = learn(given, ALL)
        for x in replayed.values():
            x.detach().fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(replayed[n], wanted[n]) for n in wanted)


def small_calls():
    from cuju_amd import layers
    given = inputs((6, 5, 40), torch.float32, seed=14)

    def norm(block, after, gates):
        return (layers.rms_norm(block, after, gates),)

    def block(x, block, gates, after, scale, before):
        return layers.residual_norm(x, block, before, after=after, gate=gates, scale=scale)

    return [(norm, [given[n] for n in ('block', 'after', 'gates')]), (block, [given[n] for n in ALL])]


def gradients_of(call):
    def learnt(*tensors):
        leaves = [x.detach().requires_grad_() for x in tensors]
        outputs = call(*leaves)
        return torch.autograd.grad(outputs, leaves, [torch.ones_like(y) for y in outputs])
    return learnt


@pytest.mark.parametrize('which', range(2))
def test_compiled_and_traced_calls(which):
    from torch.fx.experimental.proxy_tensor import make_fx
    torch._dynamo.reset()
    call, tensors = small_calls()[which]
    other = [x * 0.5 for x in tensors]
    for each in (call, gradients_of(call)):
        graph = make_fx(lambda *t: each(*t))(*tensors)
        assert all(torch.equal(a, b) for a, b in zip(graph(*other), each(*other)))
    compiled = torch.compile(call, fullgraph=True, backend='aot_eager')
    assert all(torch.equal(a, b) for a, b in zip(gradients_of(compiled)(*other), gradients_of(call)(*other)))
    maps = torch.stack([tensors[0], other[0]])
    found = torch.func.vmap(lambda x: call(x, *tensors[1:]))(maps)
    for i in range(2):
        assert all(torch.equal(a[i], b) for a, b in zip(found, call(maps[i], *tensors[1:])))


def test_modes_see_the_gradients():
    from torch.utils._python_dispatch import TorchDispatchMode
    names = []

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, function, types, args=(), kwargs=None):
            names.append(function.name())
            return function(*args, **(kwargs or {}))

    for call, tensors in small_calls():
        wanted = gradients_of(call)(*tensors)
        with Seen():
            found = gradients_of(call)(*tensors)
        assert all(torch.equal(a, b) for a, b in zip(found, wanted))
    assert [n for n in names if n.startswith('cuju_amd')] == ['cuju_amd::row_norm', 'cuju_amd::row_norm_backward'] * 2


def test_refusals():
    from cuju_amd import ArgumentError, ChoiceError, layers
    x, weight = torch.zeros(2, 3, 8, device='cuda'), torch.ones(8, device='cuda')
    for bad in (lambda: layers.rms_norm(x.cpu()), lambda: layers.rms_norm(x.double()), lambda: layers.rms_norm(x, weight[:7]),
                lambda: layers.rms_norm(x, weight.cpu()), lambda: layers.rms_norm(x, weight.int()),
                lambda: layers.rms_norm(x, weight, x[:1]), lambda: layers.rms_norm(x, weight, x.half()),
                lambda: layers.rms_norm(x, weight, x.cpu()), lambda: layers.rms_norm(x[0, 0, 0]),
                lambda: layers.rms_norm(torch.zeros(2, 0, device='cuda')), lambda: layers.rms_norm(torch.zeros(2, 8193, device='cuda')),
                lambda: layers.residual_norm(x, x[:1]), lambda: layers.residual_norm(x, x.half()), lambda: layers.residual_norm(x, None),
                lambda: layers.residual_norm(x, x, scale=weight[:7]), lambda: layers.residual_norm(x, x, scale=weight.cpu()),
                lambda: layers.residual_norm(x, x, weight[:7]), lambda: layers.residual_norm(x, x, after=weight[None]),
                lambda: layers.residual_norm(x, x, gate=x[..., :4])):
        with pytest.raises(ArgumentError):
            bad()
    for bad in (lambda: layers.rms_norm(x, gate=x, activation='relu'), lambda: layers.residual_norm(x, x, gate=x, activation=None)):
        with pytest.raises(ChoiceError):
            bad()
    y = layers.rms_norm(x.requires_grad_())
    dx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
