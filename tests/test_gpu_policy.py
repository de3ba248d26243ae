"""The recurrent policy of `examples/recurrent_policy.py`: what acting answered, an update's pass over the
segment answers again, and it learns from it."""

import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def example():
    spec = importlib.util.spec_from_file_location('recurrent_policy', os.path.join(ROOT, 'examples', 'recurrent_policy.py'))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def learner_of(example, **changes):
    return example.Learner('academy_3_vs_1_with_keeper_l3_r0', 4, **{'steps': 21, 'dtype': torch.float32, **changes})


# The two passes differ by the order of 32-bit sums: products of at most 768 terms (768 x 2^-24 = 4.6e-5 at worst
# and some 2e-6 in the mean), five of them in a row, and a memory whose errors do not grow.
SAME = 1e-5


def test_an_update_sees_what_acting_answered(example):
    learner = learner_of(example)
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
def test_an_update_learns(example, dtype):
    learner = learner_of(example, dtype=dtype)
    before = {name: x.detach().clone() for name, x in learner.policy.named_parameters()}
    for _ in range(2):
        result = learner.update(learner.play())
        assert all(bool(torch.isfinite(x)) for x in result.values())
    for name, x in learner.policy.named_parameters():
        assert bool(torch.isfinite(x.grad).all()) and float(x.grad.norm()) > 0, name
        assert not torch.equal(x.detach(), before[name]), name
