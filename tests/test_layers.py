"""The policy operators without a device: the layout of their arguments, the library's own refusals
(made before any launch), the package's, and the oracle of their tests against torch's autograd."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import layer_oracle
from conftest import PRODUCT, ROOT
from cuju_amd import ArgumentError, layers


def test_argument_structs_are_the_headers(tmp_path):
    compiler = shutil.which('gcc') or shutil.which('cc')
    if compiler is None:
        pytest.skip('no C compiler')
    source = tmp_path / 'sizes.c'
    source.write_text('#include <stdio.h>\n#include "cuju_amd.h"\nint main(void) { printf("%zu %zu %zu %zu %zu\\n", '
                      'sizeof(struct cuju_delta_rule), offsetof(struct cuju_delta_rule, state), '
                      'offsetof(struct cuju_delta_rule, d_state), sizeof(struct cuju_group_norm), '
                      'offsetof(struct cuju_group_norm, dy)); }\n')
    subprocess.run([compiler, '-I', os.path.join(ROOT, 'include'), str(source), '-o', str(tmp_path / 'sizes')], check=True)
    found = subprocess.run([str(tmp_path / 'sizes')], capture_output=True, text=True, check=True).stdout.split()
    # The packed structs, cut before the members named above.
    import struct
    cut = [layers._RULE.size, struct.calcsize('@7if3P2PP17q'), struct.calcsize('@7if3P2PP17q4PP3qP3P2P'),
           layers._NORM.size, struct.calcsize('@6if3P3P')]
    assert [int(x) for x in found] == cut


def test_the_library_refuses_before_any_launch():
    from cuju_amd import library
    lib = library.load(PRODUCT)

    def rule(type=0, batch=1, time=1, key_heads=1, heads=1, key_size=8, value_size=8, state=0):
        return layers._RULE.pack(type, batch, time, key_heads, heads, key_size, value_size, 1.0, *[0] * 6, *[0] * 17,
                                 state, *[0] * 3, 0, 0, 0, 0, 0, *[0] * 3, *[0] * 2, 0, 0)

    for function in ('cuju_delta_rule_step', 'cuju_delta_rule_forward', 'cuju_delta_rule_backward'):
        call = getattr(lib, function)
        for bad, message in ((rule(type=3), b'type'), (rule(heads=3, key_heads=2), b'multiple'),
                             (rule(key_size=129), b'sizes'), (rule(value_size=0), b'sizes'),
                             (rule(batch=1 << 23), b'2^23'), (rule(batch=-1), b'multiple'), (rule(), b'expected')):
            assert call(bad, None) == -1
            assert message in lib.cuju_last_error()
        assert call(None, None) == -1
        # Nothing to do.
        assert call(rule(batch=0), None) == 0
    assert lib.cuju_delta_rule_step(rule(time=2), None) == -1

    def norm(type=0, batch=1, pixels=4, channels=8, groups=2, activation=0):
        return layers._NORM.pack(type, batch, pixels, channels, groups, activation, 1e-5, *[0] * 10)

    for call in (lib.cuju_group_norm_forward, lib.cuju_group_norm_backward):
        for bad in (norm(type=-1), norm(groups=3), norm(activation=3), norm(batch=1 << 21, groups=2), norm(), None):
            assert call(bad, None) == -1
            assert lib.cuju_last_error()
        assert call(norm(batch=0), None) == 0 and call(norm(pixels=0), None) == 0
    assert lib.cuju_group_norm_workspace(norm()) >= 2 * 8 * 4
    assert lib.cuju_group_norm_workspace(norm(groups=3)) == 0


def test_the_library_refuses_what_its_indexes_do_not_reach():
    from cuju_amd import library
    lib = library.load(PRODUCT)

    def rule(batch=1, time=1, heads=1):
        return layers._RULE.pack(0, batch, time, 1, heads, 8, 8, 1.0, *[0] * 39)

    def norm(batch=1, pixels=1, channels=1, groups=1):
        return layers._NORM.pack(0, batch, pixels, channels, groups, 0, 1e-5, *[0] * 10)

    for call in (lib.cuju_delta_rule_step, lib.cuju_delta_rule_forward, lib.cuju_delta_rule_backward):
        for bad in (rule(time=1 << 30), rule(heads=1 << 16), rule(batch=1 << 20, heads=8)):
            assert call(bad, None) == -1 and b'2^' in lib.cuju_last_error()
    for call in (lib.cuju_group_norm_forward, lib.cuju_group_norm_backward):
        for bad in (norm(pixels=1 << 20, channels=1 << 10), norm(channels=1 << 24), norm(batch=1 << 22),
                    norm(batch=1 << 15, channels=1 << 14)):
            assert call(bad, None) == -1 and b'2^' in lib.cuju_last_error()


def test_tensors_of_another_device_are_refused():
    x = torch.zeros(1, 2, 1, 8)
    gate = torch.zeros(1, 2, 1)
    with pytest.raises(ArgumentError):
        layers.delta_rule(x, x, x, gate, gate)
    with pytest.raises(ArgumentError):
        layers.delta_rule_step(x[:, 0], x[:, 0], x[:, 0], gate[:, 0], gate[:, 0], torch.zeros(1, 1, 8, 8))
    with pytest.raises(ArgumentError):
        layers.group_norm(torch.zeros(1, 4, 8), 2)


def test_the_rules_oracle_has_autograds_gradients():
    generator = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, dtype=torch.double)

    batch, time, key_heads, heads, key_size, value_size = 2, 9, 2, 4, 5, 3
    given = {'query': normal(batch, time, key_heads, key_size), 'key': 0.3 * normal(batch, time, key_heads, key_size),
             'value': normal(batch, time, heads, value_size), 'decay': -normal(batch, time, heads).abs(),
             'beta': normal(batch, time, heads).sigmoid(), 'state': normal(batch, heads, key_size, value_size)}
    resets = torch.rand(batch, time, generator=generator) < 0.2
    leaves = {name: x.clone().requires_grad_() for name, x in given.items()}
    memory, outputs = leaves['state'], []
    for t in range(time):
        k, q = (leaves[n][:, t].repeat_interleave(2, 1) for n in ('key', 'query'))
        memory = memory * (leaves['decay'][:, t].exp() * ~resets[:, t, None])[..., None, None]
        wrote = leaves['beta'][:, t, :, None] * (leaves['value'][:, t] - (memory * k[..., None]).sum(-2))
        memory = memory + k[..., None] * wrote[..., None, :]
        outputs.append(0.7 * (memory * q[..., None]).sum(-2))
    output = torch.stack(outputs, 1)
    d_output, d_last = normal(*output.shape), normal(*memory.shape)
    gradients = torch.autograd.grad([output, memory], list(leaves.values()), [d_output, d_last])
    found = layer_oracle.delta_rule(**given, resets=resets, scale=0.7, d_output=d_output, d_last=d_last)
    torch.testing.assert_close(found['output'], output.detach())
    torch.testing.assert_close(found['last'], memory.detach())
    for name, gradient in zip(leaves, gradients):
        torch.testing.assert_close(found['d_' + name], gradient)


@pytest.mark.parametrize('activation', ['none', 'relu', 'silu'])
def test_the_norms_oracle_is_torchs(activation):
    generator = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 4, 6, generator=generator, dtype=torch.double, requires_grad=True)
    weight = torch.randn(6, generator=generator, dtype=torch.double, requires_grad=True)
    bias = torch.randn(6, generator=generator, dtype=torch.double, requires_grad=True)
    z = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 3, weight, bias).permute(0, 2, 3, 1)
    y = {'none': lambda z: z, 'relu': torch.relu, 'silu': torch.nn.functional.silu}[activation](z)
    dy = torch.randn(y.shape, generator=generator, dtype=torch.double)
    gradients = torch.autograd.grad(y, [x, weight, bias], dy)
    found = layer_oracle.group_norm(x, 3, weight, bias, activation=activation, dy=dy)
    for name, wanted in zip(('y', 'dx', 'd_weight', 'd_bias'), (y.detach(), *gradients)):
        torch.testing.assert_close(found[name], wanted)


# ------------------------------------------------- who else sees a call: modes, tracers and transforms

def fake_inputs(time=3):
    """Inputs of the delta rule without memory behind them."""
    lead = (2, time) if time else (2,)
    query, key = (torch.empty(*lead, 1, 8, device='cuda') for _ in range(2))
    decay, beta = (torch.empty(*lead, 2, device='cuda') for _ in range(2))
    return query, key, torch.empty(*lead, 2, 4, device='cuda'), decay, beta, torch.empty(2, 2, 8, 4, device='cuda')


@pytest.fixture
def fake(monkeypatch):
    """Tensors without memory, and a failure instead of a launch."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    def launched(*_):
        raise AssertionError('launched for tensors without memory')

    monkeypatch.setattr(layers, '_call', launched)
    return FakeTensorMode()


def rule_of(query, key, value, decay, beta, state):
    return layers.delta_rule(query, key, value, decay, beta, state=state)


def norm_of(x, weight):
    return layers.group_norm(x, 2, weight)


def test_tensors_without_memory_are_not_launched_for(fake):
    with fake:
        x, weight = torch.empty(2, 3, 8, device='cuda'), torch.empty(8, device='cuda')
        given, step = fake_inputs(), fake_inputs(time=0)
        found = (norm_of(x, weight), *rule_of(*given), layers.delta_rule_step(*step))
        assert [tuple(y.shape) for y in found] == [(2, 3, 8), (2, 3, 2, 4), (2, 2, 8, 4), (2, 2, 4)]
        weight.requires_grad_()
        assert norm_of(x, weight).requires_grad
    # Neither outside of the mode that made them.
    assert norm_of(x, weight).shape == x.shape and rule_of(*given)[1].shape == (2, 2, 8, 4)
    assert layers.delta_rule_step(*step).shape == (2, 2, 4)


def test_tracers_and_modes_see_the_operators(fake):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, function, types, args=(), kwargs=None):
            self.names.append(function.name())
            return function(*args, **(kwargs or {}))

    with fake:
        x, weight = torch.empty(2, 3, 8, device='cuda'), torch.empty(8, device='cuda')
        given, step = fake_inputs(), fake_inputs(time=0)
        for call, tensors, name in ((norm_of, (x, weight), 'group_norm'), (rule_of, given, 'delta_rule'),
                                    (layers.delta_rule_step, step, 'delta_rule_step')):
            with Seen() as seen:
                call(*tensors)
            assert [n for n in seen.names if n.startswith('cuju_amd')] == [f'cuju_amd::{name}']
            traced = [node.target.name() for node in make_fx(lambda *t: call(*t))(*tensors).graph.nodes
                      if node.op == 'call_function' and hasattr(node.target, 'name')]
            assert [n for n in traced if n.startswith('cuju_amd')] == [f'cuju_amd::{name}']


def test_functional_tensors_are_not_launched_for(fake):
    with fake:
        x, weight = torch.empty(2, 3, 8, device='cuda'), torch.empty(8, device='cuda')
        assert torch.func.functionalize(norm_of)(x, weight).shape == x.shape
        assert torch.func.functionalize(rule_of)(*fake_inputs())[0].shape == (2, 3, 2, 4)


def test_forward_mode_derivatives_are_refused(fake):
    from torch.autograd import forward_ad
    with fake:
        x, weight = torch.empty(2, 3, 8, device='cuda'), torch.empty(8, device='cuda')
        for call, tensors in ((norm_of, (x, weight)), (rule_of, fake_inputs()),
                              (layers.delta_rule_step, fake_inputs(time=0))):
            for which in range(len(tensors)):
                with forward_ad.dual_level():
                    call(*tensors)
                    duals = list(tensors)
                    duals[which] = forward_ad.make_dual(tensors[which], torch.empty_like(tensors[which]))
                    with pytest.raises(ArgumentError, match='forward-mode'):
                        call(*duals)
        with pytest.raises(ArgumentError, match='forward-mode'):
            torch.func.jvp(norm_of, (x, weight), (x, weight))


def test_tensors_that_are_missing_are_refused(fake):
    with fake:
        for call, tensors in ((layers.delta_rule, fake_inputs()[:5]), (layers.delta_rule_step, fake_inputs(time=0))):
            for which in range(len(tensors)):
                for bad in (None, 1.0):
                    with pytest.raises(ArgumentError):
                        call(*tensors[:which], bad, *tensors[which + 1:])
        with pytest.raises(ArgumentError):
            layers.group_norm(None, 2)


def test_group_norm_takes_the_maps_of_an_update(fake):
    # 4,096 matches of 64 steps, acting for 16,384 matches of 11 agents, and the last batch before the refusals.
    with fake:
        for maps, channels, groups in ((262144, 64, 16), (180224, 64, 32), ((1 << 22) - 1, 64, 64)):
            x = torch.empty(maps, 3, channels, device='cuda', dtype=torch.bfloat16)
            assert layers.group_norm(x, groups).shape == x.shape
        with pytest.raises(ArgumentError, match='maps'):
            layers.group_norm(torch.empty(1 << 22, 1, 1, device='cuda'), 1)
