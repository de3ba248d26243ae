"""Clipped gradients against their definition in 64 bits (tests/block_oracle.py).

The norm is a sum in 64 bits, rounded once to 32: off by at most 2^-24. A clipped value is a product with a factor that is
rounded once, and is rounded itself: off by 2 x 2^-24 in 32 bits, and by 2^-8 or 2^-11 more in bfloat16 or float16. (A
factor below 2^-100 is a power of two, which rounds nothing that is not too small, and a rest that is rounded once.)
"""

import pytest
import torch

from block_oracle import clip as exact_clip

pytestmark = pytest.mark.gpu

ROUNDING = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def clip(gradients, most, **options):
    from cuju_amd import layers
    return layers.clip_gradients(gradients, most, **options)


def gradients_of(shapes, dtypes, seed=0, scale=0.1):
    generator = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(*shape, generator=generator)).to(dtypes[i % len(dtypes)]).cuda() for i, shape in enumerate(shapes)]


def clip_close(gradients, most, **options):
    norm, exact = exact_clip(gradients, most, **options)
    found = clip(gradients, most, **options)
    assert found.shape == () and found.dtype == torch.float32
    # Rounded to 32 bits, a norm past their largest number, (2 - 2^-23) 2^127, is an infinity.
    if norm >= 2.0 ** 128:
        assert float(found) == float('inf')
    else:
        assert abs(float(found) - norm) <= 2.0 ** -24 * norm
    for x, wanted in zip(gradients, exact):
        error, allowed = (x.double() - wanted).abs(), (2.0 ** -23 + ROUNDING[x.dtype]) * wanted.abs()
        # Of numbers too small for all their digits the last digit.
        assert bool((error <= allowed + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps).all())


POLICY = [(64, 256), (64,), (32, 288), (256, 768), (256,), (9, 256), (9,), (4,), (20, 384), (20,), (1,), (1, 1)]


@pytest.mark.parametrize('dtypes', [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize('most', [0.0, 1e-3, 1.0, 1e6, float('inf')])
def test_a_policys_gradients(dtypes, most):
    clip_close(gradients_of(POLICY, dtypes, seed=1), most)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [1, 3, 7, 8, 9, 255, 256, 1023, 1024, 4096, 8191, 8192, 8193, 100003, 1 << 20, (1 << 24) + 5])
def test_sizes(size, dtype):
    clip_close(gradients_of([(size,)], [dtype], seed=size), 0.01)


@pytest.mark.parametrize('count', [127, 128, 129, 300])
def test_many_tensors(count):
    shapes = [(1 + 37 * i % 1000,) for i in range(count)]
    clip_close(gradients_of(shapes, TYPES, seed=count), 0.5)


def test_large_tensors():
    clip_close(gradients_of([(5000, 5001), (3,), (7001, 999)], [torch.bfloat16, torch.float32], seed=2), 1.0)


def test_below_the_most_nothing_changes():
    gradients = gradients_of(POLICY, TYPES, seed=3)
    before = [g.clone() for g in gradients]
    for most in (1e4, float('inf')):
        clip(gradients, most)
        assert all(torch.equal(a, b) for a, b in zip(gradients, before))


def test_places_in_a_buffer():
    # Tensors side by side at odd offsets; what lies between and behind them stays.
    for dtype in TYPES:
        room = torch.full((3000,), 7.0, dtype=dtype, device='cuda')
        views = [room[1:2], room[3:40], room[41:1001].view(2, 480), room[1003:2999]]
        for view, g in zip(views, gradients_of([v.shape for v in views], [dtype], seed=4)):
            view.copy_(g)
        clip_close(views, 0.1)
        assert bool((room[[0, 2, 40, 1001, 1002, 2999]] == 7).all())


def test_orders_of_axes():
    maps = torch.randn(4, 3, 5, 6).cuda().to(memory_format=torch.channels_last)
    turned = torch.randn(7, 9).cuda().t()
    one = torch.randn(5, 1, 3).cuda().transpose(0, 2)
    clip_close([maps, turned, one, torch.randn(1, 4).cuda()[:, 1:2]], 0.3)


def test_values_of_all_sizes():
    # Squares that 32 bits do not hold, and numbers too small to have squares there.
    large = torch.tensor([3e30, -4e30], device='cuda')
    assert abs(float(clip([large], 1.0)) - 5e30) <= 2.0 ** -23 * 5e30
    torch.testing.assert_close(large.cpu(), torch.tensor([0.6, -0.8]), rtol=2.0 ** -22, atol=0)
    small = torch.tensor([3e-30, -4e-30], device='cuda')
    assert abs(float(clip([small], 1.0)) - 5e-30) <= 2.0 ** -23 * 5e-30
    clip_close([torch.tensor([6e4, 1.0, 6e-8], device='cuda').half()], 0.5)


@pytest.mark.parametrize('most', [1.0, 1e-6, 1e-25])
def test_factors_below_the_range_of_floats(most):
    clip_close([torch.full((7,), 3e38, device='cuda'), torch.full((5,), 1e38, dtype=torch.bfloat16, device='cuda'),
                torch.full((5,), 6e4, dtype=torch.float16, device='cuda')], most)


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_norms_that_are_not_finite(bad):
    gradients = gradients_of(POLICY, TYPES, seed=5)
    gradients[3][5, 5] = bad
    kept = [g.clone() for g in gradients]
    norm = clip(gradients, float('inf'))
    assert torch.equal(torch.isnan(norm), torch.tensor(bad != bad, device='cuda')) and not bool(torch.isfinite(norm))
    assert all(torch.equal(a, b) or bad != bad for a, b in zip(gradients, kept))
    clip(gradients, 1.0)
    if bad != bad:
        assert all(bool(torch.isnan(g).all()) for g in gradients)
    else:
        assert bool(torch.isnan(gradients[3][5, 5])) and all(not bool(g.any()) for i, g in enumerate(gradients) if i != 3)


def test_nothing_and_zeros():
    empty, zeros = torch.zeros(0, 3, device='cuda'), torch.zeros(5, device='cuda')
    assert float(clip([empty], 1.0)) == 0 and float(clip([zeros, empty, None], 1.0)) == 0
    assert not bool(zeros.any())
    one = torch.tensor(2.0, device='cuda')
    assert float(clip(one, 1.0, epsilon=0.0)) == 2 and float(one) == 1


def test_as_torch_does():
    parameters = [torch.nn.Parameter(g) for g in gradients_of(POLICY, [torch.float32], seed=6)]
    for p, g in zip(parameters, gradients_of(POLICY, [torch.float32], seed=7, scale=1.0)):
        p.grad = g
    mine = [p.grad.clone() for p in parameters] + [None]
    wanted = torch.nn.utils.clip_grad_norm_(parameters, 1.0)
    found = clip(mine, 1.0)
    # Two norms in 32 bits, one of them summed there over 300,000 squares.
    torch.testing.assert_close(found, wanted, rtol=1e-5, atol=0)
    for a, b in zip(mine, parameters):
        torch.testing.assert_close(a, b.grad, rtol=1e-5, atol=0)


def test_in_place_writes_are_seen():
    x = torch.ones(3, device='cuda', requires_grad=True)
    y = x * 2
    z = y * y
    with torch.no_grad():
        clip([y.detach()], 0.1)
    with pytest.raises(RuntimeError, match='modified'):
        z.sum().backward()


def test_calls_repeat_bit_for_bit():
    gradients = gradients_of([(3000, 1000), (5,), (999, 77)], TYPES, seed=8)
    copies = [[g.clone() for g in gradients] for _ in range(4)]
    norms = [clip(each, 0.5) for each in copies]
    for norm, each in zip(norms, copies):
        assert torch.equal(norm, norms[0]) and all(torch.equal(a, b) for a, b in zip(each, copies[0]))


def test_on_another_stream_and_in_a_graph():
    gradients = gradients_of(POLICY, TYPES, seed=9)
    given = [g.clone() for g in gradients]
    wanted = [g.clone() for g in gradients]
    norm = clip(wanted, 0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        found = clip(gradients, 0.5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(found, norm) and all(torch.equal(a, b) for a, b in zip(gradients, wanted))
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        replayed = clip(gradients, 0.5)
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        again = clip(gradients, 0.25)
    for scale in (1.0, 3.0, 0.5):
        for g, x, w in zip(gradients, given, wanted):
            g.copy_(x * scale), w.copy_(x * scale)
        graphs[0].replay()
        norm = clip(wanted, 0.5)
        torch.cuda.synchronize()
        assert torch.equal(replayed, norm) and all(torch.equal(a, b) for a, b in zip(gradients, wanted))
        graphs[1].replay()
        norm = clip(wanted, 0.25)
        torch.cuda.synchronize()
        assert torch.equal(again, norm) and all(torch.equal(a, b) for a, b in zip(gradients, wanted))


def test_compiled_calls_equal_eager_ones():
    torch._dynamo.reset()
    gradients = gradients_of(POLICY[:4], TYPES, seed=10)
    copies = [[g.clone() for g in gradients] for _ in range(2)]

    def update(a, b, c, d):
        return clip([a, b, c, d], 0.5)

    compiled = torch.compile(update, fullgraph=True, backend='aot_eager')
    for _ in range(2):
        assert torch.equal(compiled(*copies[0]), update(*copies[1]))
        assert all(torch.equal(a, b) for a, b in zip(*copies))


def test_refusals():
    from cuju_amd import ArgumentError
    g = torch.ones(4, 6, device='cuda')
    for bad in ([], [None], [g.cpu()], [g, g.cpu()], [g.double()], [g.int()], [g, g], [g, g[1]], [g[1:], g[:2]], [g[:, :3]],
                [g[:1].expand(4, 6)], [g.to_sparse()], [g, 1.0], [g.clone().requires_grad_()]):
        with pytest.raises(ArgumentError):
            clip(bad, 0.5)
    for most, epsilon in ((-1.0, 0.0), (float('nan'), 0.0), (1.0, -1.0), (1.0, float('nan'))):
        with pytest.raises(ArgumentError):
            clip([g], most, epsilon=epsilon)
    assert bool((g == 1).all())
