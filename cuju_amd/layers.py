"""Operators of a policy that learns from a batch, as hand-written kernels for the MI355X.

* `delta_rule`: the gated delta rule over many steps, a recurrent memory with gradients. Its
  `resets` take a batch's `done`, so a memory never reaches over the end of an episode.
* `delta_rule_step`: one step of it for acting, with the memory updated in place.
* `group_norm`: group norm with an activation over channels-last maps, such as an encoder of super
  mini-maps makes, with gradients.

All run on the current stream of their tensors' device, wait for nothing, and can be captured in a
HIP graph. Under `torch.compile`, tracers, dispatch modes and function transforms, and for tensors of a
subclass, they are the operators `cuju_amd::delta_rule`, `cuju_amd::delta_rule_step` and
`cuju_amd::group_norm` with their backward operators. Element types
are float32, bfloat16 and float16; sums, statistics and memories are held in 32 bits whatever the
type. There is no implementation for another device. Gradients are those of reverse mode, of first
order; forward-mode derivatives are refused.
"""

from __future__ import annotations

import functools
import struct

import torch
from torch.autograd import forward_ad

from .errors import ArgumentError, ChoiceError, from_library
from .library import load

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {'none': 0, 'relu': 1, 'silu': 2}
# Key and value sizes, heads of a sequence and of a batch, and steps, that the delta rule's kernels take.
MOST_SIZE = 128
MOST_HEADS, MOST_HEADS_OF_BATCH = (1 << 16) - 1, (1 << 23) - 1
MOST_STEPS = (1 << 30) - 1
# Steps between two memories that the forward pass keeps for the backward pass.
SEGMENT = 32

# `struct cuju_delta_rule` and `struct cuju_group_norm` (include/cuju_amd.h).
_RULE = struct.Struct('@7if3P2PP17q4PP3qP3P2PPP')
_NORM = struct.Struct('@6if3P3P2P2P')


def _pointer(tensor) -> int:
    return 0 if tensor is None else tensor.data_ptr()


@functools.lru_cache(maxsize=None)
def _library():
    return load()


def _call(function, packed: bytes, device: torch.device) -> None:
    lib = _library()
    # The handle alone: a Stream object around it would be a tenth of a small call's time.
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if device.index == torch._C._cuda_getDevice():
        status = getattr(lib, function)(packed, stream)
    else:
        with torch.cuda.device(device):
            status = getattr(lib, function)(packed, stream)
    if status != 0:
        raise from_library(lib.cuju_last_error().decode())


_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}
_compiling = torch.compiler.is_compiling
_dispatch_modes, _tracing_state = torch._C._len_torch_dispatch_stack, torch._C._get_tracing_state
_transform_level = torch._C._functorch.maybe_current_level


def _operator(name: str, direct, *tensors):
    """`direct`, which launches without a way through torch's dispatcher, or the operator that it is
    registered as where something else has to see the call: a compiler, a tracer, a dispatch mode, a
    function transform or a subclass of tensors."""
    if (_compiling() or _dispatch_modes() or _tracing_state() is not None or _transform_level() is not None
            or not _PLAIN.issuperset(map(type, tensors))):
        return getattr(torch.ops.cuju_amd, name)
    return direct


def _shape(name: str, tensor: torch.Tensor, shape: tuple) -> None:
    if tensor.shape != shape:
        raise ArgumentError(f'expected {name} of the shape {shape}, found {tuple(tensor.shape)}')


def _device(first: str, tensor: torch.Tensor, names: tuple, others: tuple) -> None:
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise ArgumentError(f'expected {first} on a HIP device')
    device, kind = tensor.device, torch.Tensor
    for other in others:
        if other is not None and (not isinstance(other, kind) or other.device != device):
            name = names[[each is other for each in others].index(True)]
            raise ArgumentError(f'expected {name} on the device of {first}')
    if forward_ad._current_level >= 0 and any(x is not None and forward_ad.unpack_dual(x).tangent is not None
                                              for x in (tensor, *others)):
        raise ArgumentError('there are no forward-mode derivatives: expected tensors without a tangent')


def _learns(*tensors) -> bool:
    """Whether a call on these tensors has gradients."""
    if torch.is_grad_enabled():
        for tensor in tensors:
            if tensor is not None and tensor.requires_grad:
                return True
    return False


def _gate(name: str, tensor: torch.Tensor) -> torch.Tensor:
    """`tensor`, of a floating type, in 32 bits."""
    if not tensor.is_floating_point():
        raise ArgumentError(f'expected {name} of a floating type, found {tensor.dtype}')
    return tensor.float()


def _flat(tensor: torch.Tensor) -> torch.Tensor:
    """`tensor` with neighbouring values of its last axis side by side."""
    return tensor if tensor.stride(-1) == 1 or tensor.shape[-1] == 1 else tensor.contiguous()


# ----------------------------------------------------------------------------------- the delta rule

def _rule(q, k, v, decay, beta, state, resets, scale, output=None, last=None, checkpoints=None, d_output=None, d_last=None,
          gradients=(None,) * 6, workspace=None) -> bytes:
    """The arguments of a call; tensors are [batch, time, head, size], packed for the library."""
    batch, time, key_heads, key_size = q.shape
    heads, value_size = v.shape[2:]
    sb, st = resets.stride() if resets is not None else (0, 0)
    d_strides = d_output.stride()[:3] if d_output is not None else (0, 0, 0)
    return _RULE.pack(TYPES[q.dtype], batch, time, key_heads, heads, key_size, value_size, scale,
                      q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), beta.data_ptr(), _pointer(resets),
                      *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *decay.stride(), *beta.stride(), sb, st,
                      _pointer(state), _pointer(output), _pointer(last), _pointer(checkpoints),
                      _pointer(d_output), *d_strides, _pointer(d_last),
                      *[_pointer(g) for g in gradients], _pointer(workspace))


@functools.lru_cache(maxsize=256)
def _rule_workspace(kind, batch, time, key_heads, key_size, heads, value_size) -> int:
    """Bytes of workspace of a backward pass of these sizes."""
    return _library().cuju_delta_rule_workspace(
        _RULE.pack(kind, batch, time, key_heads, heads, key_size, value_size, 0.0, *[0] * 39))


_OTHERS = 'key', 'value', 'decay', 'beta', 'state', 'resets'


def _check_rule(query, key, value, decay, beta, state, resets, steps):
    """The checked arguments as the kernels take them; `steps`: whether they have a time axis."""
    axes = 4 if steps else 3
    if key is None or value is None or decay is None or beta is None:
        raise ArgumentError('expected a key, value, decay and beta')
    _device('query', query, _OTHERS, (key, value, decay, beta, state, resets))
    dtype = query.dtype
    if dtype not in TYPES:
        raise ArgumentError(f'expected query of float32, bfloat16 or float16, found {dtype}')
    if key.dtype != dtype or value.dtype != dtype:
        raise ArgumentError(f'expected key and value of {dtype}, found {key.dtype} and {value.dtype}')
    if query.dim() != axes or value.dim() != axes:
        raise ArgumentError(f'expected query and value of {axes} axes, found {query.dim()} and {value.dim()}')
    shape = query.shape
    *lead, key_heads, key_size = shape
    heads, value_size = value.shape[-2:]
    _shape('key', key, shape)
    _shape('value', value, (*lead, heads, value_size))
    gates = (*lead, heads)
    _shape('decay', decay, gates)
    _shape('beta', beta, gates)
    if key_heads < 1 or heads < 1 or heads % key_heads:
        raise ArgumentError(f'expected heads that are a multiple of the {key_heads} key heads, found {heads}')
    if not 1 <= key_size <= MOST_SIZE or not 1 <= value_size <= MOST_SIZE:
        raise ArgumentError(f'expected key and value sizes from 1 to {MOST_SIZE}, found {key_size} and {value_size}')
    if heads > MOST_HEADS or lead[0] * heads > MOST_HEADS_OF_BATCH or lead[-1] > MOST_STEPS:
        raise ArgumentError(f'expected at most {MOST_HEADS} heads, {MOST_HEADS_OF_BATCH} in the batch, and {MOST_STEPS} '
                            f'steps, found the shape {tuple(value.shape)}')
    if decay.dtype != torch.float32:
        decay = _gate('decay', decay)
    if beta.dtype != torch.float32:
        beta = _gate('beta', beta)
    if state is not None:
        _shape('state', state, (lead[0], heads, key_size, value_size))
    if resets is not None:
        _shape('resets', resets, tuple(lead))
        if resets.dtype == torch.bool:
            resets = resets.view(torch.uint8)
        elif resets.dtype != torch.uint8:
            raise ArgumentError(f'expected resets of bool or uint8, found {resets.dtype}')
    return _flat(query), _flat(key), _flat(value), decay, beta, resets


def _rule_forward(q, k, v, decay, beta, state, resets, scale, train):
    batch, time = q.shape[:2]
    heads, value_size = v.shape[2:]
    output = v.new_empty((batch, time, heads, value_size))
    last = torch.empty((batch, heads, q.shape[3], value_size), dtype=torch.float32, device=v.device)
    kept = max(time - 1, 0) // SEGMENT if train else 0
    checkpoints = torch.empty((batch, heads, kept, q.shape[3], value_size), dtype=torch.float32, device=v.device)
    if batch:
        _call('cuju_delta_rule_forward', _rule(q, k, v, decay, beta, state, resets, scale, output, last,
                                               checkpoints if kept else None), v.device)
    return output, last, checkpoints


def _rule_backward(q, k, v, decay, beta, state, resets, scale, checkpoints, d_output, d_last):
    batch, _, _, key_size = q.shape
    heads = v.shape[2]
    dense = [x.new_empty(x.shape) for x in (q, k, v, decay, beta)]
    d_state = torch.empty((batch, heads, key_size, v.shape[3]), dtype=torch.float32, device=v.device)
    if batch:
        size = _rule_workspace(TYPES[q.dtype], *q.shape, *v.shape[2:])
        workspace = torch.empty(size, dtype=torch.uint8, device=v.device) if size else None
        _call('cuju_delta_rule_backward',
              _rule(q, k, v, decay, beta, state, resets, scale, checkpoints=checkpoints if checkpoints.numel() else None,
                    d_output=d_output, d_last=d_last, gradients=(*dense, d_state), workspace=workspace), v.device)
    return (*dense, d_state)


def _rule_step(q, k, v, decay, beta, state, resets, scale):
    batch, heads, value_size = v.shape
    output = v.new_empty((batch, heads, value_size))
    if batch:
        sb = resets.stride(0) if resets is not None else 0
        qb, qh = q.stride()[:2]
        kb, kh = k.stride()[:2]
        vb, vh = v.stride()[:2]
        db, dh = decay.stride()
        bb, bh = beta.stride()
        _call('cuju_delta_rule_step',
              _RULE.pack(TYPES[q.dtype], batch, 1, q.shape[1], heads, q.shape[2], value_size, scale,
                         q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), beta.data_ptr(), _pointer(resets),
                         qb, 0, qh, kb, 0, kh, vb, 0, vh, db, 0, dh, bb, 0, bh, sb, 0,
                         state.data_ptr(), output.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), v.device)
    torch.autograd.graph.increment_version(state)
    return output


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, beta, state, resets, scale):
        run = _operator('delta_rule', _rule_forward, q, k, v, decay, beta, state, resets)
        output, last, checkpoints = run(q, k, v, decay, beta, state, resets, scale, True)
        ctx.save_for_backward(q, k, v, decay, beta, state, resets, checkpoints)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return output, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output, d_last):
        q, k, v, decay, beta, state, resets, checkpoints = ctx.saved_tensors
        d_output = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if d_output is None else _flat(d_output)
        d_last = d_last.contiguous() if d_last is not None else None
        run = _operator('delta_rule_backward', _rule_backward, q, k, v, decay, beta, state, resets, checkpoints, d_output, d_last)
        *dense, d_state = run(q, k, v, decay, beta, state, resets, ctx.scale, checkpoints, d_output, d_last)
        return (*dense, d_state if state is not None else None, None, None)


def delta_rule(query, key, value, decay, beta, *, state=None, resets=None, scale=None):
    """The gated delta rule over many steps: `(output, last)`.

    Each head keeps a matrix S [key size, value size], from `state` or zeros. At each step it is
    cleared where `resets` is true, scaled by `exp(decay)`, and written:
    `u = beta * (value - S^T key)`, `S += key u^T`; the output is `scale * S^T query`.

    * `query`, `key`: [batch, time, key heads, key size]; `value`: [batch, time, heads, value size], all
      of one type. Head h reads the key head `h // (heads / key heads)`. Keys are taken as they are:
      the rule is stable for `beta * |key|^2` up to 2, as with keys of unit length and beta up to 1.
    * `decay` (the logarithm of the factor, so at most 0 in use; -inf keeps nothing) and `beta`:
      [batch, time, heads], of any floating type, held in 32 bits.
    * `state`: [batch, heads, key size, value size], in 32 bits.
    * `resets`: [batch, time], bool or uint8: true where an episode starts. Nothing before such a step,
      not even an infinity, reaches its outputs, the later ones or their gradients. Each costs about as
      much as 16 steps (32 in the backward pass), for the steps between two are worked on together.
    * `scale`: by default 1 / sqrt(key size).

    `output` is [batch, time, heads, value size] in the inputs' type, `last` the memory after the last
    step in 32 bits. Sizes go up to 128, strides are free (an axis of time before the batch is a
    transposed view). Gradients reach every floating input; they are the same on every call. A NaN or an
    infinity reaches the outputs of its own step and of later ones, as in the definition; in the memory an
    infinity becomes a NaN. It may reach all gradients of its episode, and none of another.
    """
    q, k, v, decay, beta, resets = _check_rule(query, key, value, decay, beta, state, resets, True)
    if state is not None:
        state = state.float().contiguous()
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if _learns(q, k, v, decay, beta, state):
        return _DeltaRule.apply(q, k, v, decay, beta, state, resets, scale)
    run = _operator('delta_rule', _rule_forward, q, k, v, decay, beta, state, resets)
    output, last, _ = run(q, k, v, decay, beta, state, resets, scale, False)
    return output, last


def delta_rule_step(query, key, value, decay, beta, state, *, resets=None, scale=None):
    """One step of the gated delta rule, as in acting: returns the output and updates `state` in place.

    As `delta_rule` without the axis of time: `query` and `key` [batch, key heads, key size], `value`
    [batch, heads, value size], `decay` and `beta` [batch, heads], `resets` [batch]; `state` is a
    contiguous float32 tensor [batch, heads, key size, value size]. A memory that is reset is not read.
    It has no gradients: an update learns through `delta_rule`.
    """
    q, k, v, decay, beta, resets = _check_rule(query, key, value, decay, beta, state, resets, False)
    if state is None or state.dtype != torch.float32 or not state.is_contiguous():
        raise ArgumentError('expected state as a contiguous float32 tensor, which the step updates')
    if _learns(q, k, v, decay, beta, state):
        raise ArgumentError('delta_rule_step has no gradients: call it under torch.no_grad(), or call delta_rule')
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    run = _operator('delta_rule_step', _rule_step, q, k, v, decay, beta, state, resets)
    return run(q, k, v, decay, beta, state, resets, scale)


# --------------------------------------------------------------------------------------- group norm

def _norm(x, groups, weight, bias, epsilon, activation, y=None, stats=None, workspace=None, dy=None, dx=None, d_weight=None,
          d_bias=None) -> bytes:
    batch, channels = x.shape[0], x.shape[-1]
    pixels = x.numel() // (batch * channels) if batch else 0
    return _NORM.pack(TYPES[x.dtype], batch, pixels, channels, groups, activation, epsilon, x.data_ptr(),
                      _pointer(weight), _pointer(bias), _pointer(y), _pointer(stats), _pointer(workspace),
                      _pointer(dy), _pointer(dx), _pointer(d_weight), _pointer(d_bias))


@functools.lru_cache(maxsize=256)
def _norm_bytes(kind, batch, pixels, channels, groups) -> int:
    """Bytes of workspace of a pass over maps of these sizes."""
    return _library().cuju_group_norm_workspace(_NORM.pack(kind, batch, pixels, channels, groups, 0, 0.0, *[0] * 10))


def _norm_workspace(x, groups):
    batch, channels = x.shape[0], x.shape[-1]
    return torch.empty(_norm_bytes(TYPES[x.dtype], batch, x.numel() // (batch * channels), channels, groups),
                       dtype=torch.uint8, device=x.device)


def _norm_forward(x, weight, bias, groups, epsilon, activation):
    y = torch.empty_like(x)
    stats = torch.empty((x.shape[0], groups, 2), dtype=torch.float32, device=x.device)
    if x.numel():
        workspace = _norm_workspace(x, groups)
        _call('cuju_group_norm_forward', _norm(x, groups, weight, bias, epsilon, activation, y, stats, workspace), x.device)
    return y, stats


def _norm_backward(x, weight, bias, stats, dy, groups, epsilon, activation, of_weight, of_bias):
    """The gradients of x, weight and bias; those of weight and bias are empty where they are not asked for."""
    dx = torch.empty_like(x)
    d_weight, d_bias = (torch.empty(x.shape[-1] if asked else 0, dtype=torch.float32, device=x.device)
                        for asked in (of_weight, of_bias))
    if x.numel():
        workspace = _norm_workspace(x, groups)
        _call('cuju_group_norm_backward',
              _norm(x, groups, weight, bias, epsilon, activation, None, stats, workspace, dy, dx,
                    d_weight if of_weight else None, d_bias if of_bias else None), x.device)
    else:
        d_weight.zero_()
        d_bias.zero_()
    return dx, d_weight, d_bias


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, epsilon, activation):
        run = _operator('group_norm', _norm_forward, x, weight, bias)
        y, stats = run(x, weight, bias, groups, epsilon, activation)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.options = groups, epsilon, activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        run = _operator('group_norm_backward', _norm_backward, x, weight, bias, stats, dy)
        _, of_weight, of_bias, *_ = ctx.needs_input_grad
        dx, d_weight, d_bias = run(x, weight, bias, stats, dy.contiguous(), *ctx.options, of_weight, of_bias)
        return dx, d_weight if of_weight else None, d_bias if of_bias else None, None, None, None


def group_norm(x, groups, weight=None, bias=None, *, epsilon=1e-5, activation='none'):
    """Group norm with an activation over channels-last maps `x` [batch, ..., channels].

    The channels are cut into `groups` equal runs; each is normalised over its channels and all axes
    between the batch and the channels, then scaled by `weight` and shifted by `bias` ([channels], held
    in 32 bits, by default ones and zeros), then passed through `activation`: 'none', 'relu' or
    'silu'. The output has the type and shape of `x`, contiguous. A NCHW tensor of torch's channels-last
    memory format is such a map as `x.permute(0, 2, 3, 1)`, without a copy. Gradients reach `x`,
    `weight` and `bias`; they are the same on every call.
    """
    _device('x', x, ('weight', 'bias'), (weight, bias))
    if x.dtype not in TYPES:
        raise ArgumentError(f'expected x of float32, bfloat16 or float16, found {x.dtype}')
    if x.dim() < 2 or x.shape[-1] < 1:
        raise ArgumentError(f'expected x of a batch axis and channels, found the shape {tuple(x.shape)}')
    channels = x.shape[-1]
    if not isinstance(groups, int) or groups < 1 or channels % groups:
        raise ArgumentError(f'expected groups that divide the {channels} channels, found {groups}')
    if activation not in ACTIVATIONS:
        raise ChoiceError(f"expected the activation 'none', 'relu' or 'silu', found {activation!r}")
    for name, each in (('weight', weight), ('bias', bias)):
        if each is not None:
            _shape(name, each, (channels,))
            if not each.is_floating_point():
                raise ArgumentError(f'expected {name} of a floating type, found {each.dtype}')
    batch = x.shape[0]
    if x.numel() // (batch or 1) >= 1 << 30 or channels >= 1 << 24:
        raise ArgumentError(f'expected fewer than 2^30 values and 2^24 channels in a map, found the shape {tuple(x.shape)}')
    if batch >= 1 << 22 or batch * channels >= 1 << 29:
        raise ArgumentError(f'expected fewer than 2^22 maps and 2^29 channels in the batch, found the shape {tuple(x.shape)}')
    x = x.contiguous()
    weight = weight.float().contiguous() if weight is not None else None
    bias = bias.float().contiguous() if bias is not None else None
    options = groups, float(epsilon), ACTIVATIONS[activation]
    if _learns(x, weight, bias):
        return _GroupNorm.apply(x, weight, bias, *options)
    run = _operator('group_norm', _norm_forward, x, weight, bias)
    return run(x, weight, bias, *options)[0]


# -------------------------------------------------------------------------- operators of torch.compile

_NAMESPACE = torch.library.Library('cuju_amd', 'FRAGMENT')
_INPUTS = 'Tensor query, Tensor key, Tensor value, Tensor decay, Tensor beta'
_NAMESPACE.define(f'delta_rule({_INPUTS}, Tensor? state, Tensor? resets, float scale, bool train) -> '
                  '(Tensor, Tensor, Tensor)')
_NAMESPACE.define(f'delta_rule_backward({_INPUTS}, Tensor? state, Tensor? resets, float scale, Tensor checkpoints, '
                  'Tensor d_output, Tensor? d_last) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)')
_NAMESPACE.define(f'delta_rule_step({_INPUTS}, Tensor(a!) state, Tensor? resets, float scale) -> Tensor')
_NAMESPACE.define('group_norm(Tensor x, Tensor? weight, Tensor? bias, int groups, float epsilon, int activation) -> '
                  '(Tensor, Tensor)')
_NAMESPACE.define('group_norm_backward(Tensor x, Tensor? weight, Tensor? bias, Tensor stats, Tensor dy, int groups, '
                  'float epsilon, int activation, bool of_weight, bool of_bias) -> (Tensor, Tensor, Tensor)')
_NAMESPACE.impl('delta_rule', _rule_forward, 'CUDA')
_NAMESPACE.impl('delta_rule_backward', _rule_backward, 'CUDA')
_NAMESPACE.impl('delta_rule_step', _rule_step, 'CUDA')
_NAMESPACE.impl('group_norm', _norm_forward, 'CUDA')
_NAMESPACE.impl('group_norm_backward', _norm_backward, 'CUDA')


@torch.library.register_fake('cuju_amd::delta_rule')
def _(query, key, value, decay, beta, state, resets, scale, train):
    batch, time, _, key_size = query.shape
    heads, value_size = value.shape[2:]
    kept = max(time - 1, 0) // SEGMENT if train else 0
    return (value.new_empty(value.shape), decay.new_empty((batch, heads, key_size, value_size)),
            decay.new_empty((batch, heads, kept, key_size, value_size)))


@torch.library.register_fake('cuju_amd::delta_rule_backward')
def _(query, key, value, decay, beta, state, resets, scale, checkpoints, d_output, d_last):
    batch, _, _, key_size = query.shape
    return (*[x.new_empty(x.shape) for x in (query, key, value, decay, beta)],
            decay.new_empty((batch, value.shape[2], key_size, value.shape[3])))


@torch.library.register_fake('cuju_amd::delta_rule_step')
def _(query, key, value, decay, beta, state, resets, scale):
    return value.new_empty(value.shape)


@torch.library.register_fake('cuju_amd::group_norm')
def _(x, weight, bias, groups, epsilon, activation):
    return x.new_empty(x.shape), x.new_empty((x.shape[0], groups, 2), dtype=torch.float32)


@torch.library.register_fake('cuju_amd::group_norm_backward')
def _(x, weight, bias, stats, dy, groups, epsilon, activation, of_weight, of_bias):
    sums = (x.new_empty((x.shape[-1] if asked else 0,), dtype=torch.float32) for asked in (of_weight, of_bias))
    return x.new_empty(x.shape), *sums
