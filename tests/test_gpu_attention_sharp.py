"""The gradients of log decays at steps that nearly forget, one by one, against the definition (tests/block_oracle.py).

Such a gradient is smaller than those around it by the step's factor, and a bound on a tensor's norm does not see it. Each is a sum
of what passes its step, and its bound is relative to the 2-norm of the terms of that sum alone: memories and their gradients
are within 3e-6 of their terms' 2-norm each, a sum of pairs of steps within sqrt(128 + 128) 2^-24 = 1e-6, and factors, of
exponents below 2^7 that are held in 32 bits on the way to each, within 2^-18 ln 2 = 2.6e-6, two of them; under 13e-6, four times of
which no single value of random rounding errors exceeds.
"""

import pytest
import torch

from block_oracle import attention as exact_attention
from test_gpu_attention import NAMES, TYPES, inputs, learn, learn_close

pytestmark = pytest.mark.gpu

BOUND = 4 * 13e-6
SPAN = 128


def exact_decays(given, d_output, d_last):
    """The gradients of the decays of all steps and the 2-norms of their terms."""
    wide = given['decay'].expand(*given['value'].shape[:3])
    square = lambda x: x.detach().double().square() if x is not None else None  # noqa: E731
    scale = given['query'].shape[-1] ** -0.5
    exact = exact_attention(given['query'], given['key'], given['value'], wide, given['state'], given['resets'], scale, d_output, d_last)
    squares = exact_attention(*[square(given[n]) for n in ('query', 'key', 'value')], 2 * wide.double(), square(given['state']),
                              given['resets'], scale ** 2, square(d_output), square(d_last))
    return exact['d_decay'], squares['d_decay'].sqrt()


def each_close(given, where):
    """Checks the gradients at `where`, one by one."""
    found, d_output, d_last = learn(given)
    exact, terms = exact_decays(given, d_output, d_last)
    error, allowed = (found['d_decay'].double() - exact).abs(), BOUND * terms
    assert bool(torch.isfinite(found['d_decay']).all())
    worst = (error / allowed.clamp_min(1e-300))[where].max()
    assert bool((error <= allowed)[where].all()), f'{float(worst):.3g} times the bound'
    return found


def spans_of(where):
    """All steps of the spans in which `where` is true."""
    wide = torch.zeros_like(where)
    for low in range(0, where.shape[1], SPAN):
        wide[:, low:low + SPAN] = where[:, low:low + SPAN].any(1, keepdim=True)
    return wide


SIZES = [(2, 1, 1, 1, 8, 8, 0), (2, 17, 3, 3, 33, 48, 5), (2, 128, 1, 2, 64, 64, 0), (2, 130, 1, 1, 100, 20, 40), (1, 129, 1, 4, 128, 128, 0),
         (2, 300, 2, 6, 48, 80, 100), (2, 400, 1, 3, 7, 5, 90), (3, 150, 2, 2, 32, 16, 0)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes', SIZES)
@pytest.mark.parametrize('decay', [-4.5, -10.0, -15.0, -30.0, -80.0])
def test_steps_that_nearly_forget(decay, sizes, dtype):
    given = inputs(*sizes[:6], dtype=dtype, seed=sum(sizes), episode=sizes[6])
    given['decay'].clamp_(min=-0.5)
    time = sizes[1]
    sharp = torch.zeros(given['decay'].shape, dtype=torch.bool, device='cuda')
    for t in {0, time // 2, max(time - 3, 0), min(127, time - 1), min(128, time - 1)}:
        sharp[0, t, 0] = True
    sharp[-1, time // 3] = True
    given['decay'][sharp] = decay
    each_close(given, spans_of(sharp))


@pytest.mark.parametrize('state', [False, True])
@pytest.mark.parametrize('decay', [-5.0, -40.0])
def test_every_step_nearly_forgets(decay, state):
    given = inputs(3, 200, 1, 2, 40, 24, seed=1, episode=30, state=state)
    given['decay'][:] = decay
    each_close(given, torch.ones_like(given['decay'], dtype=torch.bool))


@pytest.mark.parametrize('dtype', TYPES)
def test_a_head_that_nearly_forgets(dtype):
    # One decay of a head: the sum of its steps, next to heads that remember.
    given = inputs(3, 260, 1, 3, 32, 40, dtype=dtype, seed=2, episode=100, fixed=True)
    given['decay'][:] = torch.tensor([-0.01, -6.0, -25.0])
    found, d_output, d_last = learn(given)
    exact, terms = exact_decays(given, d_output, d_last)
    error, allowed = (found['d_decay'].double() - exact.sum((0, 1))).abs(), BOUND * terms.square().sum((0, 1)).sqrt()
    assert bool((error <= allowed)[1:].all())
    learn_close(given)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('name', ['query', 'key', 'value', 'decay', 'state'])
def test_other_episodes_beside_a_value_that_is_not_finite(name, bad):
    # Three episodes in a span; the value is in the first one, or in the last.
    for low, high in ((0, 40), (80, 128)):
        given = inputs(2, 140, 1, 2, 32, 32, seed=3)
        given['resets'] = torch.zeros(2, 140, dtype=torch.bool, device='cuda')
        given['resets'][:, [40, 80, 130]] = True
        given['decay'].clamp_(min=-0.5)
        sharp = torch.zeros_like(given['decay'], dtype=torch.bool)
        sharp[:, [20, 60, 100]] = True
        given['decay'][sharp] = -12.0
        _, d_output, d_last = learn(given)
        exact, terms = exact_decays(given, d_output, d_last)
        if name == 'state':
            given['state'][:, 0, 3, 5] = bad
            low, high = 0, 40
        else:
            given[name][:, low + 9, 0] = bad
        found = learn(given, d_output, d_last)[0]['d_decay']
        for first, last in ((0, 40), (40, 80), (80, 128)):
            if first != low:
                error = (found[:, first:last].double() - exact[:, first:last]).abs()
                assert bool((error <= BOUND * terms[:, first:last])[sharp[:, first:last]].all())
        assert not bool(found[:, [40, 80, 130]].any())


@pytest.mark.parametrize('time', [1, 100, 300])
def test_a_first_step_that_nothing_comes_before(time):
    # Whatever its decay, there is nothing to forget.
    found, *_ = learn(inputs(3, time, 1, 2, 32, 32, seed=7, state=False))
    assert not bool(found['d_decay'][:, 0].any())


def test_strides_streams_and_graphs():
    given = inputs(4, 200, 2, 4, 32, 32, dtype=torch.bfloat16, seed=4, episode=60)
    given['decay'][:, 50] = -9.0
    wanted, *given_d = learn(given)
    # An axis of time first, and an odd offset: loads of single elements.
    packed = torch.zeros(200, 4, 8, 2 * 32 + 1, dtype=torch.bfloat16, device='cuda')
    views = {}
    for i, name in enumerate(('query', 'key')):
        views[name] = packed[:, :, :2, 1 + 32 * i:1 + 32 * (i + 1)].transpose(0, 1)
        views[name].copy_(given[name])
    sharp = torch.zeros_like(given['decay'], dtype=torch.bool)
    sharp[:, 50] = True
    each_close({**given, **views}, spans_of(sharp))
    for _ in range(2):
        assert all(torch.equal(x, wanted[n]) for n, x in learn(given, *given_d)[0].items())
    # An eager graph of the same leaves ends before the capture.
    del wanted
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        learn(given, *given_d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = list(learn(given, *given_d)[0].values())
    for decay in (-9.0, -0.5, -20.0):
        # Whether a span has such a step is seen at every replay.
        given['decay'][:, 50] = decay
        wanted = list(learn(given, *given_d)[0].values())
        for each in found:
            each.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(found, wanted))


def test_only_the_last_memory_is_learnt_from():
    given = inputs(2, 140, 1, 2, 32, 32, seed=6)
    given['decay'][:, 70] = -11.0
    leaves = [given[n].detach().requires_grad_() for n in NAMES]
    from cuju_amd import layers
    _, last = layers.linear_attention(*leaves[:4], state=leaves[4])
    d_last = torch.randn(last.shape, generator=torch.Generator().manual_seed(2)).cuda()
    found, = torch.autograd.grad(last, leaves[3], d_last)
    exact, terms = exact_decays(given, torch.zeros_like(given['value']), d_last)
    # One head has forgotten its steps by e^-110 at the end. 32 bits hold no factor F below 2^-126, and what passes a step is at
    # most F |S| |D|, with unit keys |S| at most |state| and the sum of all |value|.
    lost = 2.0 ** -126 * float((given['state'].norm() + given['value'].norm(dim=-1).sum()) * d_last.norm())
    assert bool(((found.double() - exact).abs() <= BOUND * terms + lost)[:, 70].all())
