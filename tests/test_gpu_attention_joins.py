"""Linear attention over spans that are joined: factors past one, whose products leave the range of 32 bits though no memory does,
and more spans than a join takes at a time. The definition is that of block_oracle.py, the bounds are test_gpu_attention.py's and,
where a decay is the same at many steps, another: every step's factor is within 2^-23 of the exponential, those of equal decays
err alike, and steps that are played one by one multiply them all. A memory is a product of at most `time` of them, so
time 2^-23 of its terms.
"""

import pytest
import torch

from block_oracle import attention as exact_attention
from block_oracle import attention_terms
from test_gpu_attention import all_close, attend, bound_of, close, forward_close, inputs, learn

pytestmark = pytest.mark.gpu


def grown(batch, time, first, later, **options):
    """Sequences whose log decays are `later` but for those at the steps `first`."""
    given = inputs(batch, time, 1, 2, 32, 32, seed=time + batch, **options)
    given['decay'][:] = later
    for t, decay in first.items():
        given['decay'][:, t] = decay
    return given


def grown_close(found, exact, terms, time):
    for name, x in found.items():
        close(x, exact[name], bound_of(name) + (12 if name == 'd_decay' else 1) * time * 2.0 ** -23, terms[name])


# Growth of a memory that holds nothing yet, by more than 3e38 with the growth of the steps after it.
# float16 holds what is written afterwards alone.
GROWTH = [({0: 80.0}, 0.1, torch.float32), ({0: 50.0, 1: 50.0}, 0.0, torch.float32), ({0: 80.0}, 0.1, torch.bfloat16),
          ({0: 50.0, 1: 50.0}, 0.0, torch.bfloat16), ({0: 70.0, 1: 20.0, 2: -20.0}, 0.0, torch.bfloat16), ({0: 88.0}, 0.01, torch.float16)]


@pytest.mark.parametrize('time', [129, 400])
@pytest.mark.parametrize('first, later, dtype', GROWTH)
def test_growth_of_an_empty_memory(first, later, time, dtype):
    # Few heads, whose steps are cut and joined, and more, whose steps are not: both are the definition.
    for batch in (1, 300):
        given = grown(batch, time, first, later, dtype=dtype, state=False)
        grown_close(dict(zip(('output', 'last'), attend(given))), dict(zip(('output', 'last'), exact_attention(**given))),
                    attention_terms(**given), time)
        leaves = [given[n].detach().requires_grad_() for n in ('query', 'key', 'value', 'decay')]
        output, last = attend({**given, **dict(zip(('query', 'key', 'value', 'decay'), leaves))})
        d_output = torch.randn(output.shape, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        # The last memory has no gradient: the joined one is empty, too.
        found = torch.autograd.grad(output, leaves, d_output)
        exact = exact_attention(**given, d_output=d_output)
        grown_close(dict(zip(('d_query', 'd_key', 'd_value', 'd_decay'), found)), exact,
                    attention_terms(**given, d_output=d_output), time)


def test_growth_of_a_memory_of_next_to_nothing():
    # By e^120, more than 32 bits hold, in two steps of one span: 1e-30 becomes 1e22.
    given = grown(1, 400, {140: 60.0, 141: 60.0}, 0.0)
    given['state'] *= 1e-30
    given['key'][:, :142] = 0
    forward_close(attend(given), given)
    # Backwards, of the gradient of the last memory, past steps that write nothing.
    given = grown(1, 400, {300: 60.0, 301: 60.0}, 0.0, state=False)
    given['value'][:, :302] = 0
    given['state'] = torch.zeros(1, 2, 32, 32, device='cuda')
    found, d_output, d_last = learn(given, torch.zeros(1, 400, 2, 32, device='cuda'), 1e-30 * torch.randn(1, 2, 32, 32, device='cuda'))
    d = {'d_output': d_output, 'd_last': d_last}
    all_close(found, exact_attention(**given, **d), attention_terms(**given, **d))


def test_a_factor_that_is_infinite():
    # exp(inf) times a memory of zeros is no number, in the definition as here; later episodes have their own.
    given = grown(1, 400, {130: float('inf')}, 0.0, state=False)
    given['key'][:, :131] = 0
    given['resets'] = torch.zeros(1, 400, dtype=torch.bool, device='cuda')
    given['resets'][:, 260] = True
    output, last = attend(given)
    assert not bool(output[:, :130].any()) and not bool(torch.isfinite(output[:, 130:260]).any())
    whole = {n: x[:, 260:] for n, x in given.items() if n != 'state'}
    forward_close((output[:, 260:], last), {**whole, 'state': None})


@pytest.mark.parametrize('time, dtype', [(1152, torch.float32), (1153, torch.float32), (1300, torch.bfloat16), (1300, torch.float16),
                                         (3000, torch.bfloat16)])
@pytest.mark.parametrize('episode', [0, 700])
def test_more_spans_than_a_join_takes_at_a_time(episode, time, dtype):
    # 9 and more joined memories, 8 at a time. An element of the memory, and of its gradient, is a sum of up to 3,000 steps:
    # sqrt(3000 / 400) of the bounds of 400.
    given = inputs(2, time, 1, 1, 16, 16, dtype=dtype, seed=time, episode=episode)
    given['decay'] *= 0.02
    wider = (time / 400) ** 0.5
    found = dict(zip(('output', 'last'), attend(given)))
    exact, terms = dict(zip(('output', 'last'), exact_attention(**given))), attention_terms(**given)
    for name, x in found.items():
        close(x, exact[name], wider * bound_of(name), terms[name])
    found, d_output, d_last = learn(given)
    d = {'d_output': d_output, 'd_last': d_last}
    exact, terms = exact_attention(**given, **d), attention_terms(**given, **d)
    for name, x in found.items():
        close(x, exact[name], wider * bound_of(name), terms[name])


def test_long_sequences_repeat_and_are_captured():
    given = inputs(2, 1300, 1, 1, 16, 16, dtype=torch.bfloat16, seed=2, episode=700)
    wanted = attend(given)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(attend(given), wanted))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = attend(given)
    for scale in (1.0, -0.5, 2.0):
        given['value'].mul_(scale)
        wanted = attend(given)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, wanted))
