"""The operators of a policy's blocks without a device: the layout of their arguments, the library's own refusals
(made before any launch), the package's, and the oracle of their tests against torch's autograd."""

import array
import os
import shutil
import struct
import subprocess

import pytest
import torch

import block_oracle
from conftest import PRODUCT, ROOT
from cuju_amd import ArgumentError, layers, library

# The structs of the header, the packed ones, and members before which their formats are cut.
STRUCTS = {
    'cuju_linear_attention': ('_ATTENTION', {'query': '@8if', 'state': '@8if5P14q', 'd_output': '@8if5P14q4P', 'd_query': '@8if5P14q4PP3qP'}),
    'cuju_row_norm': ('_ROWS', {'rows': '@5i2f', 'after': '@5i2fq3P6q', 'd_stream': '@5i2fq3P6q6P', 'workspace': '@5i2fq3P6q6P8P'}),
    'cuju_gradients': ('_GRADIENTS', {'gradients': '@q', 'most': '@qP', 'norm': '@qP2d'}),
}


@pytest.mark.parametrize('name', list(STRUCTS))
def test_argument_structs_are_the_headers(name, tmp_path):
    compiler = shutil.which('gcc') or shutil.which('cc')
    if compiler is None:
        pytest.skip('no C compiler')
    packed, members = STRUCTS[name]
    source = tmp_path / 'sizes.c'
    printed = ''.join(f'printf("%zu ", offsetof(struct {name}, {member})); ' for member in members)
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "cuju_amd.h"\n'
                      f'int main(void) {{ printf("%zu ", sizeof(struct {name})); {printed}}}\n')
    subprocess.run([compiler, '-I', os.path.join(ROOT, 'include'), str(source), '-o', str(tmp_path / 'sizes')], check=True)
    found = subprocess.run([str(tmp_path / 'sizes')], capture_output=True, text=True, check=True).stdout.split()
    # A member starts where the format before it ends, filled up to a pointer.
    cut = [(struct.calcsize(each) + 7) // 8 * 8 for each in members.values()]
    assert [int(x) for x in found] == [getattr(layers, packed).size, *cut]


def attention(type=0, batch=1, time=1, key_heads=1, heads=1, key_size=8, value_size=8):
    return layers._ATTENTION.pack(type, batch, time, key_heads, heads, key_size, value_size, 0, 1.0, *[0] * 34)


def test_the_library_refuses_before_any_launch():
    lib = library.load(PRODUCT)
    for function in ('cuju_linear_attention_step', 'cuju_linear_attention_forward', 'cuju_linear_attention_backward'):
        call = getattr(lib, function)
        for bad, message in ((attention(type=3), b'type'), (attention(heads=3, key_heads=2), b'multiple'),
                             (attention(key_size=129), b'sizes'), (attention(value_size=0), b'sizes'),
                             (attention(batch=1 << 23), b'2^23'), (attention(batch=-1), b'multiple'), (attention(), b'expected'),
                             (attention(time=1 << 24), b'2^24'), (attention(heads=1 << 16), b'2^16')):
            assert call(bad, None) == -1
            assert message in lib.cuju_last_error()
        assert call(None, None) == -1
        # Nothing to do.
        assert call(attention(batch=0), None) == 0
    assert lib.cuju_linear_attention_step(attention(time=2), None) == -1
    for function in ('cuju_linear_attention_forward_workspace', 'cuju_linear_attention_backward_workspace'):
        assert getattr(lib, function)(attention(heads=3, key_heads=2)) == 0
    # Memories between spans, for few heads and long sequences alone.
    assert lib.cuju_linear_attention_forward_workspace(attention(time=400)) >= 3 * 8 * 8 * 4
    assert lib.cuju_linear_attention_forward_workspace(attention(time=300)) == 0
    assert lib.cuju_linear_attention_forward_workspace(attention(time=400, batch=4096)) == 0


def test_the_library_refuses_norms_and_gradients():
    lib = library.load(PRODUCT)

    def norm(type=0, size=8, inner=1, activation=0, rows=4):
        return layers._ROWS.pack(type, size, inner, activation, 1, 1e-6, 1.0, rows, *[0] * 24)

    for call in (lib.cuju_row_norm_forward, lib.cuju_row_norm_backward):
        for bad in (norm(type=3), norm(size=0), norm(size=8193), norm(inner=0), norm(activation=3), norm(rows=-1), norm(), None):
            assert call(bad, None) == -1
            assert lib.cuju_last_error()
        assert call(norm(rows=0), None) == 0
    assert lib.cuju_row_norm_workspace(norm()) >= 4 * 3 * 8 * 4 and lib.cuju_row_norm_workspace(norm(size=0)) == 0

    def gradients(*each, most=1.0, epsilon=1e-6, norm=64):
        table = array.array('q', [x for one in each for x in one])
        return layers._GRADIENTS.pack(len(each), table.buffer_info()[0], most, epsilon, norm, 0), table

    for bad, message in ((gradients((64, 4, 3)), b'type'), (gradients((64, -1, 0)), b'values'), (gradients((64, 1 << 44, 0)), b'values'),
                         (gradients((0, 4, 0)), b'data'), (gradients((64, 4, 0), most=-1.0), b'at least'),
                         (gradients((64, 4, 0), epsilon=float('nan')), b'at least'), (gradients((64, 4, 0), norm=0), b'norm'),
                         (gradients((64, 4, 0)), b'workspace')):
        assert lib.cuju_clip_gradients(bad[0], None) == -1
        assert message in lib.cuju_last_error()
    assert lib.cuju_clip_gradients(None, None) == -1
    # Tensors that share memory, with a workspace that no launch reaches.
    for each in (((64, 4, 0), (64, 4, 0)), ((64, 4, 0), (76, 1, 1)), ((128, 100, 1), (64, 100, 2))):
        given, table = gradients(*each)
        assert lib.cuju_clip_gradients(given[:-8] + struct.pack('@P', 64), None) == -1
        assert b'overlap' in lib.cuju_last_error()
    # A sum for each workgroup: 40 KB in tiles of 32, and as many as are launched at most for each 128 tensors.
    given, table = gradients((64, 10000, 0))
    assert lib.cuju_clip_gradients_workspace(given) == 8 * 2
    given, table = gradients(*[(64, 1 << 24, 0)] * 129)
    assert lib.cuju_clip_gradients_workspace(given) == 8 * 2 * 1024


def test_tensors_of_another_device_are_refused():
    for bad in (lambda: layers.rms_norm(torch.zeros(2, 8)), lambda: layers.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8)),
                lambda: layers.clip_gradients([torch.zeros(3)], 1.0), lambda: layers.clip_gradients([], 1.0),
                lambda: layers.clip_gradients([None], 1.0)):
        with pytest.raises(ArgumentError):
            bad()
    x, gate = torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1)
    for decay in (gate, gate[0, 0]):
        with pytest.raises(ArgumentError):
            layers.linear_attention(x, x, x, decay)
        with pytest.raises(ArgumentError):
            layers.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], decay if decay.dim() == 1 else decay[:, 0], torch.zeros(1, 1, 8, 8))


@pytest.mark.parametrize('fixed', [False, True])
def test_attentions_oracle_has_autograds_gradients(fixed):
    generator = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, dtype=torch.double)

    batch, time, key_heads, heads, key_size, value_size = 2, 9, 2, 4, 5, 3
    given = {'query': normal(batch, time, key_heads, key_size), 'key': normal(batch, time, key_heads, key_size),
             'value': normal(batch, time, heads, value_size),
             'decay': -normal(heads).abs() if fixed else -normal(batch, time, heads).abs(),
             'state': normal(batch, heads, key_size, value_size)}
    resets = torch.rand(batch, time, generator=generator) < 0.2
    leaves = {name: x.clone().requires_grad_() for name, x in given.items()}
    memory, outputs = leaves['state'], []
    decay = leaves['decay'].expand(batch, time, heads)
    for t in range(time):
        k, q = (leaves[n][:, t].repeat_interleave(2, 1) for n in ('key', 'query'))
        memory = memory * (decay[:, t].exp() * ~resets[:, t, None])[..., None, None]
        memory = memory + k[..., None] * leaves['value'][:, t, :, None, :]
        outputs.append(0.7 * (memory * q[..., None]).sum(-2))
    output = torch.stack(outputs, 1)
    d_output, d_last = normal(*output.shape), normal(*memory.shape)
    gradients = torch.autograd.grad([output, memory], list(leaves.values()), [d_output, d_last])
    found = block_oracle.attention(**given, resets=resets, scale=0.7, d_output=d_output, d_last=d_last)
    torch.testing.assert_close(found['output'], output.detach())
    torch.testing.assert_close(found['last'], memory.detach())
    for name, gradient in zip(leaves, gradients):
        torch.testing.assert_close(found['d_' + name], gradient)


@pytest.mark.parametrize('names', [('block',), ('block', 'after', 'gates'), ('x', 'block'), ('x', 'block', 'gates', 'after', 'scale', 'before')])
@pytest.mark.parametrize('activation', ['none', 'sigmoid', 'silu'])
def test_the_norms_oracle_has_autograds_gradients(names, activation):
    generator = torch.Generator().manual_seed(1)
    leaves = {n: torch.randn(*((3, 2, 5) if n in ('x', 'block', 'gates') else (5,)), generator=generator, dtype=torch.double,
                             requires_grad=True) for n in names}
    norm = lambda x: x / (x.square().mean(-1, keepdim=True) + 1e-3).sqrt()  # noqa: E731
    h = norm(leaves['block']) if 'x' not in names or 'after' in names else leaves['block']
    h = h * leaves.get('after', 1)
    if 'gates' in names:
        z = leaves['gates']
        h = h * {'none': z, 'sigmoid': z.sigmoid(), 'silu': torch.nn.functional.silu(z)}[activation]
    outputs = {'stream': h}
    if 'x' in names:
        outputs['stream'] = leaves['x'] + leaves.get('scale', 1) * h
        outputs['normed'] = norm(outputs['stream']) * leaves.get('before', 1)
    d = {'d_' + n: torch.randn(h.shape, generator=generator, dtype=torch.double) for n in outputs}
    gradients = torch.autograd.grad(list(outputs.values()), list(leaves.values()), list(d.values()))
    found = block_oracle.rows(**leaves, epsilon=1e-3, activation=activation, norm_block='x' not in names or 'after' in names, **d)
    for name, x in outputs.items():
        torch.testing.assert_close(found[name], x.detach())
    for name, x in zip(leaves, gradients):
        torch.testing.assert_close(found['d_' + name.replace('gates', 'gate')], x)


def test_rows_that_lie_in_two_axes():
    x = torch.zeros(4, 3, 5, 8)
    assert layers._row_strides(x) == (40, 8) and layers._row_strides(x[0, 0]) == (8, 0) and layers._row_strides(x[0, 0, 0]) == (0, 0)
    assert layers._row_strides(x.transpose(1, 2)) is None and layers._row_strides(x.transpose(2, 3)) is None
    assert layers._row_strides(x[:, :1].transpose(1, 2)) == (120, 0 + 120) or layers._row_strides(x[:, :1].transpose(1, 2)) is None
    assert layers._row_strides(x[:, 1]) == (120, 8) and layers._row_strides(x[1].transpose(0, 1)) == (8, 40)
    assert layers._row_strides(x[:1, :1, :1].expand(4, 3, 5, 8)) == (0, 0)
    assert layers._row_strides(x[..., :1]) == (40, 8) and layers._row_strides(x[0, ..., 1:]) == (40, 8)


# ------------------------------------------------- who else sees a call: modes, tracers and transforms

@pytest.fixture
def fake(monkeypatch):
    """Tensors without memory, and a failure instead of a launch."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    def launched(*_):
        raise AssertionError('launched for tensors without memory')

    monkeypatch.setattr(layers, '_call', launched)
    return FakeTensorMode()


def attention_inputs(time=300, fixed=False):
    lead = (2, time) if time else (2,)
    query, key = (torch.empty(*lead, 1, 8, device='cuda') for _ in range(2))
    decay = torch.empty(*(() if fixed else lead), 2, device='cuda')
    return query, key, torch.empty(*lead, 2, 4, device='cuda'), decay, torch.empty(2, 2, 8, 4, device='cuda')


def attend(query, key, value, decay, state):
    return layers.linear_attention(query, key, value, decay, state=state)


# Each operator's name, a call of it, and inputs.
CALLS = {
    'linear_attention': (attend, attention_inputs),
    'linear_attention_step': (layers.linear_attention_step, lambda: attention_inputs(time=0)),
    'row_norm': (lambda x, block, gate, scale: layers.residual_norm(x, block, gate=gate, scale=scale),
                 lambda: (*(torch.empty(2, 3, 8, device='cuda') for _ in range(3)), torch.empty(8, device='cuda'))),
    'clip_gradients': (lambda *gradients: layers.clip_gradients(gradients, 1.0),
                       lambda: (torch.empty(2, 3, device='cuda'), torch.empty(4, device='cuda', dtype=torch.bfloat16))),
}
# Arguments that may be None.
FREE = {'linear_attention': (4,), 'row_norm': (2, 3), 'clip_gradients': (0, 1)}


@pytest.mark.parametrize('fixed', [False, True])
def test_attention_without_memory(fake, fixed):
    with fake:
        given, step = attention_inputs(fixed=fixed), attention_inputs(0, fixed)
        assert [tuple(x.shape) for x in attend(*given)] == [(2, 300, 2, 4), (2, 2, 8, 4)]
        assert layers.linear_attention_step(*step).shape == (2, 2, 4)
        leaves = [x.requires_grad_() for x in given]
        assert all(x.requires_grad for x in attend(*leaves))


@pytest.mark.parametrize('name', list(CALLS))
def test_tracers_and_modes_see_the_operators(fake, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, function, types, args=(), kwargs=None):
            self.names.append(function.name())
            return function(*args, **(kwargs or {}))

    call, make = CALLS[name]
    with fake:
        tensors = make()
        with Seen() as seen:
            call(*tensors)
        assert [n for n in seen.names if n.startswith('cuju_amd')] == [f'cuju_amd::{name}']
        traced = [node.target.name() for node in make_fx(lambda *t: call(*t))(*tensors).graph.nodes
                  if node.op == 'call_function' and hasattr(node.target, 'name')]
        assert [n for n in traced if n.startswith('cuju_amd')] == [f'cuju_amd::{name}']


@pytest.mark.parametrize('name', list(CALLS))
def test_forward_mode_derivatives_are_refused(fake, name):
    from torch.autograd import forward_ad
    call, make = CALLS[name]
    with fake:
        tensors = make()
        for which in range(len(tensors)):
            with forward_ad.dual_level():
                call(*tensors)
                duals = list(tensors)
                duals[which] = forward_ad.make_dual(tensors[which], torch.empty_like(tensors[which]))
                with pytest.raises(ArgumentError, match='forward-mode'):
                    call(*duals)


@pytest.mark.parametrize('name', list(CALLS))
def test_tensors_that_are_missing_are_refused(fake, name):
    call, make = CALLS[name]
    with fake:
        tensors = make()
        for which in range(len(tensors)):
            for bad in (None, 1.0):
                if bad is None and which in FREE.get(name, ()) or bad and (name, which) in (('linear_attention', 4), ('row_norm', 3)):
                    continue
                with pytest.raises(ArgumentError):
                    call(*tensors[:which], bad, *tensors[which + 1:])
