"""A policy's block of all its operators together against 64 bits, and the example policy with residual blocks and the memory
that only adds: what acting answered, an update's pass answers again, and it learns from it."""

import importlib.util
import os

import pytest
import torch

from block_oracle import attention as exact_attention
from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def example():
    spec = importlib.util.spec_from_file_location('recurrent_policy', os.path.join(ROOT, 'examples', 'recurrent_policy.py'))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def learner_of(example, **changes):
    return example.Learner('academy_3_vs_1_with_keeper_l3_r0', 4, **{'steps': 21, 'dtype': torch.float32, 'memory': 'linear', 'blocks': 2,
                                                                     **changes})


# The two passes differ by the order of 32-bit sums: products of at most 768 terms (768 x 2^-24 = 4.6e-5 at worst
# and some 2e-6 in the mean), ten of them in a row, and a memory whose errors do not grow.
SAME = 2e-5


@pytest.mark.parametrize('changes', [{}, {'memory': 'delta'}, {'blocks': 0}])
def test_an_update_sees_what_acting_answered(example, changes):
    learner = learner_of(example, **changes)
    learner.play()  # so that the next segment starts with a memory
    segment = learner.play()
    with torch.no_grad():
        logits, values = learner.policy.learn(segment['maps'], segment['memory'], segment['resets'])
    for found, acted in ((logits, segment['logits']), (values, segment['values'])):
        assert found.shape == acted.shape
        assert float((found - acted).norm()) <= SAME * float(acted.norm())


def test_resets_clear_both_alike(example):
    learner = learner_of(example)
    segment = learner.play()
    agents = learner.agents
    resets = torch.rand(21, agents, generator=torch.Generator().manual_seed(1)).cuda() < 0.2
    before = torch.randn(learner.memory.shape, generator=torch.Generator().manual_seed(2)).cuda()
    memory = before.clone()
    acted = torch.stack([learner.policy.act(segment['maps'][t], memory, resets[t])[0] for t in range(21)])
    with torch.no_grad():
        found, _ = learner.policy.learn(segment['maps'], before, resets)
    assert float((found - acted).norm()) <= SAME * float(acted.norm())
    # An agent that starts anew answers as if nothing had been before.
    fresh = learner.policy.act(segment['maps'][0], torch.zeros_like(before), torch.zeros_like(resets[0]))[0]
    anew = learner.policy.act(segment['maps'][0], before.clone(), torch.ones_like(resets[0]))[0]
    assert torch.equal(fresh, anew)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('changes', [{}, {'memory': 'delta'}, {'blocks': 0}])
def test_an_update_learns(example, changes, dtype):
    learner = learner_of(example, dtype=dtype, **changes)
    before = {name: x.detach().clone() for name, x in learner.policy.named_parameters()}
    for _ in range(2):
        result = learner.update(learner.play())
        assert all(bool(torch.isfinite(x)) for x in result.values())
    gradients = [x.grad for x in learner.policy.parameters()]
    assert float(torch.stack([g.double().square().sum() for g in gradients]).sum().sqrt()) <= 1 + 1e-5
    for name, x in learner.policy.named_parameters():
        assert bool(torch.isfinite(x.grad).all()) and float(x.grad.norm()) > 0, name
        assert not torch.equal(x.detach(), before[name]), name


def test_unknown_memories_are_refused(example):
    with pytest.raises(ValueError):
        example.Policy(memory='none')


# A block in 32 bits is a chain of ten products and norms, each off by under 3e-6 of its terms (768 of them); the gradients
# pass through twice as many: 20 x 3e-6, and as much again where terms cancel. Where an episode starts they cancel without such a
# bound: a head's answer there is (q.k) v, its norm does not depend on q.k, and so the gradients of q and k are differences of
# two terms of size 1 / |q.k|, which leaves 2^-24 / |q.k| of them. That much any arithmetic in 32 bits is off, so the
# gradients may be off by four times what the plain formulas in 32 bits are.
BLOCK = 1.2e-4


@pytest.mark.parametrize('time', [40, 150])
@pytest.mark.parametrize('fixed', [False, True])
def test_a_block_of_all_operators(fixed, time):
    from cuju_amd import layers
    generator = torch.Generator().manual_seed(time)
    batch, heads, size, width = 6, 4, 32, 96

    def normal(*shape):
        return torch.randn(*shape, generator=generator).cuda()

    parameters = {'x': normal(batch, time, width), 'begun': 1 + 0.2 * normal(width), 'projection': 0.1 * normal(4 * heads * size, width),
                  'decay': -normal(heads).abs() if fixed else -normal(batch, time, heads).abs(), 'memory': normal(batch, heads, size, size),
                  'answered': 1 + 0.2 * normal(size), 'out': 0.1 * normal(width, heads * size), 'after': 1 + 0.2 * normal(width),
                  'scale': 0.3 * normal(width), 'next': 1 + 0.2 * normal(width)}
    resets = torch.rand(batch, time, generator=generator).cuda() < 0.05
    d_stream, d_normed = normal(batch, time, width), normal(batch, time, width)

    def split(normed, projection):
        return (normed @ projection.t()).unflatten(-1, (4, heads, size)).unbind(2)

    def run(p):
        normed = layers.rms_norm(p['x'], p['begun'])
        query, key, value, gate = split(normed, p['projection'])
        read, last = layers.linear_attention(query, key, value, p['decay'], state=p['memory'], resets=resets)
        outcome = layers.rms_norm(read, p['answered'], gate).flatten(-2) @ p['out'].t()
        return (*layers.residual_norm(p['x'], outcome, p['next'], after=p['after'], scale=p['scale']), last)

    def plain(p):
        norm = lambda x: x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
        query, key, value, gate = split(norm(p['x']) * p['begun'], p['projection'])
        memory, answers = p['memory'], []
        decay = p['decay'].expand(batch, time, heads).exp() * ~resets[..., None]
        for t in range(time):
            memory = memory * decay[:, t, :, None, None] + key[:, t, :, :, None] * value[:, t, :, None, :]
            answers.append(size ** -0.5 * (memory * query[:, t, :, :, None]).sum(-2))
        read = norm(torch.stack(answers, 1)) * p['answered'] * torch.nn.functional.silu(gate)
        stream = p['x'] + p['scale'] * (norm(read.flatten(-2) @ p['out'].t()) * p['after'])
        return stream, norm(stream) * p['next'], memory

    results = []
    for call, kind in ((run, torch.float32), (plain, torch.double), (plain, torch.float32)):
        leaves = {n: x.detach().to(kind).requires_grad_() for n, x in parameters.items()}
        outputs = call(leaves)
        gradients = torch.autograd.grad(outputs[:2], list(leaves.values()), [d_stream.to(kind), d_normed.to(kind)])
        results.append((outputs, dict(zip(leaves, gradients))))
    for found, wanted in zip(*(r[0] for r in results[:2])):
        found, wanted = found.detach(), wanted.detach()
        assert float((found.double() - wanted).norm()) <= BLOCK * float(wanted.norm())
    errors = 0.0
    for name, wanted in results[1][1].items():
        off, plainly = (float((results[i][1][name].double() - wanted).norm()) for i in (0, 2))
        allowed = max(BLOCK * float(wanted.norm()), 4 * plainly)
        assert off <= allowed, name
        errors += allowed
    # The update's gradients are clipped together.
    gradients = list(results[0][1].values())
    norm = layers.clip_gradients(gradients, 0.5)
    wanted = sum(float(g.square().sum()) for g in results[1][1].values()) ** 0.5
    assert abs(float(norm) - wanted) <= errors
    assert abs(sum(float(g.double().square().sum()) for g in gradients) ** 0.5 - 0.5) <= 1e-5


def test_the_memory_of_a_replay_is_that_of_acting():
    # Segment after segment, as a match is played: the memory carried on, against the whole match in 64 bits.
    from cuju_amd import layers
    generator = torch.Generator().manual_seed(3)
    query, key, value = (torch.randn(3, 200, 2, 32, generator=generator).cuda() / 5 for _ in range(3))
    decay = -torch.rand(2, generator=generator).cuda()
    acted, memory = [], torch.zeros(3, 2, 32, 32, device='cuda')
    for t in range(200):
        acted.append(layers.linear_attention_step(query[:, t], key[:, t], value[:, t], decay, memory))
    output, last = layers.linear_attention(query, key, value, decay)
    wanted, final = exact_attention(query, key, value, decay)
    for found in (torch.stack(acted, 1), output):
        assert float((found.double() - wanted).norm()) <= 3e-6 * float(wanted.norm())
    for found in (memory, last):
        assert float((found.double() - final).norm()) <= 3e-6 * float(final.norm())
