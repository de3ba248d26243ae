"""Operators of a policy that learns from a batch, as hand-written kernels for the MI355X.

* `delta_rule`: the gated delta rule over many steps, a recurrent memory with gradients. Its
  `resets` take a batch's `done`, so a memory never reaches over the end of an episode.
* `delta_rule_step`: one step of it for acting, with the memory updated in place.
* `linear_attention`, `linear_attention_step`: a memory that only adds and forgets, in the same two forms.
* `group_norm`: group norm with an activation over channels-last maps, such as an encoder of super
  mini-maps makes, with gradients.
* `rms_norm`: the root-mean-square norm of rows with a gate, such as a memory's answers take, with gradients.
* `residual_norm`: a block's end and the next one's start in one pass, with gradients: the block's output
  normed, gated, scaled and added to the stream, and the stream's norm.
* `clip_gradients`: the global norm of an update's gradients, which are clipped by it in place.

All run on the current stream of their tensors' device, wait for nothing, and can be captured in a
HIP graph; a backward pass only while no eager graph of the same leaves is alive (torch ties a leaf to the
stream of the first graph that uses it), so let such outputs go first. Under `torch.compile`, tracers,
dispatch modes and function transforms, and for tensors of a subclass, they are operators of torch's
namespace `cuju_amd`, of their own names (both norms of rows are `cuju_amd::row_norm`) with their backward
operators. Element types are float32, bfloat16 and float16; sums, statistics and memories are held in 32
bits whatever the type. There is no implementation for another device. Gradients are those of reverse mode, of first
order; forward-mode derivatives are refused.
"""

from __future__ import annotations

import array
import functools
import struct

import torch
from torch.autograd import forward_ad

from .errors import ArgumentError, ChoiceError, LibraryError, from_library
from .library import load

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {'none': 0, 'relu': 1, 'silu': 2}
# Activations of a gate, and values of a row, that the norms of rows take.
GATES = {'none': 0, 'sigmoid': 1, 'silu': 2}
MOST_ROW = 8192
# Key and value sizes, heads of a sequence and of a batch, and steps, that the delta rule's kernels take.
MOST_SIZE = 128
MOST_HEADS, MOST_HEADS_OF_BATCH = (1 << 16) - 1, (1 << 23) - 1
MOST_STEPS = (1 << 30) - 1
# Steps between two memories that the forward pass keeps for the backward pass: of the delta rule, of linear attention.
SEGMENT, SPAN = 32, 128
# Steps that linear attention's kernels take.
MOST_SPANNED_STEPS = (1 << 24) - 1

# `struct cuju_delta_rule`, `struct cuju_linear_attention` and `struct cuju_group_norm` (include/cuju_amd.h).
_RULE = struct.Struct('@7if3P2PP17q4PP3qP3P2PPP')
_ATTENTION = struct.Struct('@8if5P14q4PP3qP5PP')
_NORM = struct.Struct('@6if3P3P2P2P')
# `struct cuju_row_norm`, `struct cuju_gradients` and the number of words of a `struct cuju_gradient`.
_ROWS = struct.Struct('@5i2fq3P6q3P3P2P3P3PP')
_GRADIENTS = struct.Struct('@qP2d2P')


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
    contiguous float32 tensor [batch, heads, key size, value size]. It is read whether it is reset or not, but
    what a memory that is reset held does not matter, infinities and NaN included.
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


# --------------------------------------------------------------------------------- linear attention

def _attention(q, k, v, decay, state, resets, scale, output=None, last=None, checkpoints=None, d_output=None, d_last=None,
               gradients=(None,) * 5, workspace=0, of_head=False) -> bytes:
    """The arguments of a call; tensors are [batch, time, head, size], packed for the library."""
    batch, time, key_heads, key_size = q.shape
    heads, value_size = v.shape[2:]
    return _ATTENTION.pack(TYPES[q.dtype], batch, time, key_heads, heads, key_size, value_size, of_head, scale,
                           q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), _pointer(resets),
                           *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *_decay_strides(decay),
                           *(resets.stride() if resets is not None else (0, 0)),
                           _pointer(state), _pointer(output), _pointer(last), _pointer(checkpoints),
                           _pointer(d_output), *(d_output.stride()[:3] if d_output is not None else (0, 0, 0)), _pointer(d_last),
                           *[_pointer(g) for g in gradients], workspace)


def _decay_strides(decay) -> tuple:
    return decay.stride() if decay.dim() == 3 else (0, 0, decay.stride(0))


@functools.lru_cache(maxsize=256)
def _attention_bytes(function, kind, batch, time, key_heads, key_size, heads, value_size, of_head, kept, of_decay) -> int:
    """Bytes of workspace of a pass of these sizes; `kept`, `of_decay`: whether it has checkpoints and the decay's gradient."""
    return getattr(_library(), function)(
        _ATTENTION.pack(kind, batch, time, key_heads, heads, key_size, value_size, of_head, 0.0, *[0] * 22, int(kept), *[0] * 8,
                        int(of_decay), 0, 0))


def _attention_workspace(function, q, v, of_head, kept, of_decay):
    size = _attention_bytes(function, TYPES[q.dtype], *q.shape, *v.shape[2:], of_head, kept, of_decay)
    return torch.empty(size, dtype=torch.uint8, device=q.device) if size else None


def _attention_forward(q, k, v, decay, state, resets, scale, train):
    batch, time, _, key_size = q.shape
    heads, value_size = v.shape[2:]
    output = v.new_empty((batch, time, heads, value_size))
    last = torch.empty((batch, heads, key_size, value_size), dtype=torch.float32, device=v.device)
    kept = max(time - 1, 0) // SPAN if train else 0
    checkpoints = torch.empty((batch, heads, kept, key_size, value_size), dtype=torch.float32, device=v.device)
    if batch:
        workspace = _attention_workspace('cuju_linear_attention_forward_workspace', q, v, False, kept > 0, False)
        _call('cuju_linear_attention_forward',
              _attention(q, k, v, decay, state, resets, scale, output, last, checkpoints if kept else None,
                         workspace=_pointer(workspace)), v.device)
    return output, last, checkpoints


def _attention_backward(q, k, v, decay, state, resets, scale, checkpoints, d_output, d_last, of_decay):
    """The gradients; the decay's is empty where it is not asked for."""
    batch, _, _, key_size = q.shape
    heads = v.shape[2]
    dense = [x.new_empty(x.shape) for x in (q, k, v)]
    d_decay = decay.new_empty(decay.shape if of_decay else 0)
    d_state = torch.empty((batch, heads, key_size, v.shape[3]), dtype=torch.float32, device=v.device)
    if batch:
        of_head = decay.dim() == 1
        workspace = _attention_workspace('cuju_linear_attention_backward_workspace', q, v, of_head, checkpoints.numel() > 0, of_decay)
        _call('cuju_linear_attention_backward',
              _attention(q, k, v, decay, state, resets, scale, checkpoints=checkpoints if checkpoints.numel() else None,
                         d_output=d_output, d_last=d_last, gradients=(*dense, d_decay if of_decay else None, d_state),
                         workspace=_pointer(workspace), of_head=of_head), v.device)
    elif decay.dim() == 1:
        d_decay.zero_()
    return (*dense, d_decay, d_state)


def _attention_step(q, k, v, decay, state, resets, scale):
    batch, heads, value_size = v.shape
    output = v.new_empty((batch, heads, value_size))
    if batch:
        qb, qh = q.stride()[:2]
        kb, kh = k.stride()[:2]
        vb, vh = v.stride()[:2]
        db, dh = decay.stride() if decay.dim() == 2 else (0, decay.stride(0))
        _call('cuju_linear_attention_step',
              _ATTENTION.pack(TYPES[q.dtype], batch, 1, q.shape[1], heads, q.shape[2], value_size, 0, scale,
                              q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), _pointer(resets),
                              qb, 0, qh, kb, 0, kh, vb, 0, vh, db, 0, dh, resets.stride(0) if resets is not None else 0, 0,
                              state.data_ptr(), output.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), v.device)
    torch.autograd.graph.increment_version(state)
    return output


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, state, resets, scale):
        run = _operator('linear_attention', _attention_forward, q, k, v, decay, state, resets)
        output, last, checkpoints = run(q, k, v, decay, state, resets, scale, True)
        ctx.save_for_backward(q, k, v, decay, state, resets, checkpoints)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return output, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output, d_last):
        q, k, v, decay, state, resets, checkpoints = ctx.saved_tensors
        d_output = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if d_output is None else _flat(d_output)
        d_last = d_last.contiguous() if d_last is not None else None
        run = _operator('linear_attention_backward', _attention_backward, q, k, v, decay, state, resets, checkpoints, d_output, d_last)
        of_decay = ctx.needs_input_grad[3]
        *dense, d_decay, d_state = run(q, k, v, decay, state, resets, ctx.scale, checkpoints, d_output, d_last, of_decay)
        return (*dense, d_decay if of_decay else None, d_state if state is not None else None, None, None)


def _check_attention(query, key, value, decay, state, resets, steps):
    """The checked arguments as the kernels take them; `steps`: whether they have a time axis. A decay of heads alone stays so."""
    if key is None or value is None or decay is None:
        raise ArgumentError('expected a key, value and decay')
    gates = decay
    of_heads = isinstance(decay, torch.Tensor) and decay.dim() == 1
    if of_heads and isinstance(value, torch.Tensor) and value.dim() > 1:
        _shape('decay', decay, tuple(value.shape[-2:-1]))
        decay = _gate('decay', decay)
        gates = decay.expand(value.shape[:-1])
    # A memory that does not forget has every gate of the rule but beta.
    q, k, v, gates, _, resets = _check_rule(query, key, value, gates, gates, state, resets, steps)
    if steps and q.shape[1] > MOST_SPANNED_STEPS:
        raise ArgumentError(f'expected at most {MOST_SPANNED_STEPS} steps, found the shape {tuple(value.shape)}')
    return q, k, v, decay if of_heads else gates, resets


def linear_attention(query, key, value, decay, *, state=None, resets=None, scale=None):
    """Linear attention with decays over many steps: `(output, last)`.

    Each head keeps a matrix S [key size, value size], from `state` or zeros. At each step it is
    cleared where `resets` is true, scaled by `exp(decay)`, and written: `S += key value^T`; the output
    is `scale * S^T query`. It is the memory of `delta_rule` that only adds, and costs about half as much.

    * `query`, `key`: [batch, time, key heads, key size]; `value`: [batch, time, heads, value size], all
      of one type. Head h reads the key head `h // (heads / key heads)`.
    * `decay` (the logarithm of the factor, so at most 0 in use; -inf keeps nothing): [batch, time,
      heads], or [heads] for one that is the same at every step, of any floating type, held in 32 bits. From 89 on the
      factor leaves the range of 32 bits, and a memory of zeros times it is no number.
    * `state`: [batch, heads, key size, value size], in 32 bits.
    * `resets`: [batch, time], bool or uint8: true where an episode starts. Nothing before such a step,
      not even an infinity, reaches its outputs, the later ones or their gradients.
    * `scale`: by default 1 / sqrt(key size).

    `output` is [batch, time, heads, value size] in the inputs' type, `last` the memory after the last
    step in 32 bits. Sizes go up to 128, strides are free (an axis of time before the batch is a
    transposed view). Gradients reach every floating input; they are the same on every call. Memories, scores and sums
    have 32 bits whatever the type, also where an output or a gradient is rounded to 16. The gradient of a log decay is
    found from the products of queries and keys with their gradients at the same 128 steps, and is some times 2^-24 of
    those off; where one of the 128 has a log decay below -4, each is a sum of its own and as much of that off.
    Such steps cost more: about as much as the rest of the backward pass where every 128 have one. A NaN or an
    infinity reaches the outputs of its own step and of later ones, as in the definition; in the memory an
    infinity may become a NaN. It may reach all gradients of its episode, and none of another.
    """
    q, k, v, decay, resets = _check_attention(query, key, value, decay, state, resets, True)
    if state is not None:
        state = state.float().contiguous()
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if _learns(q, k, v, decay, state):
        return _LinearAttention.apply(q, k, v, decay, state, resets, scale)
    run = _operator('linear_attention', _attention_forward, q, k, v, decay, state, resets)
    output, last, _ = run(q, k, v, decay, state, resets, scale, False)
    return output, last


def linear_attention_step(query, key, value, decay, state, *, resets=None, scale=None):
    """One step of linear attention with decays, as in acting: returns the output and updates `state` in place.

    As `linear_attention` without the axis of time: `query` and `key` [batch, key heads, key size],
    `value` [batch, heads, value size], `decay` [batch, heads] or [heads], `resets` [batch]; `state` is a
    contiguous float32 tensor [batch, heads, key size, value size]. It is read whether it is reset or not, but
    what a memory that is reset held does not matter, infinities and NaN included.
    It has no gradients: an update learns through `linear_attention`.
    """
    q, k, v, decay, resets = _check_attention(query, key, value, decay, state, resets, False)
    if state is None or state.dtype != torch.float32 or not state.is_contiguous():
        raise ArgumentError('expected state as a contiguous float32 tensor, which the step updates')
    if _learns(q, k, v, decay, state):
        raise ArgumentError('linear_attention_step has no gradients: call it under torch.no_grad(), or call linear_attention')
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    run = _operator('linear_attention_step', _attention_step, q, k, v, decay, state, resets)
    return run(q, k, v, decay, state, resets, scale)


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


# ------------------------------------------------------------------------------------ norms of rows

def _row_strides(tensor) -> tuple | None:
    """The strides of `tensor`'s rows, [all axes but the last two][the last but one]; None if it is not made of such rows."""
    *lead, size = tensor.shape
    *strides, last = tensor.stride() or (1,)
    if size != 1 and last != 1:
        return None
    if len(lead) < 2:
        return strides[0] if lead else 0, 0
    step, outer = 0, None
    for stride, count in zip(reversed(strides[:-1]), reversed(lead[:-1])):
        if count == 1:
            continue
        if outer is None:
            step = stride
        elif stride != outer:
            return None
        outer = stride * count
    return step, strides[-1]


def _in_rows(tensor):
    return tensor if tensor is None or tensor.is_contiguous() or _row_strides(tensor) is not None else tensor.contiguous()


def _rows(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block, stream=None, normed=None, stats=None,
          d_stream=None, d_normed=None, gradients=(None,) * 6, workspace=None) -> bytes:
    """The arguments of a call, packed for the library."""
    shape = block.shape
    size, inner = shape[-1], shape[-2] if len(shape) > 2 else 1
    strides = []
    for tensor in (x, block, gate):
        strides += _row_strides(tensor) if tensor is not None else (0, 0)
    return _ROWS.pack(TYPES[block.dtype], size, inner, activation, norm_block, epsilon, scale, block.numel() // size,
                      _pointer(x), block.data_ptr(), _pointer(gate), *strides, _pointer(after), _pointer(scales), _pointer(before),
                      _pointer(stream), _pointer(normed), _pointer(stats), _pointer(d_stream), _pointer(d_normed),
                      *[_pointer(g) for g in gradients], _pointer(workspace))


@functools.lru_cache(maxsize=256)
def _rows_bytes(kind, rows, size) -> int:
    """Bytes of workspace of a backward pass over rows of these sizes."""
    return _library().cuju_row_norm_workspace(_ROWS.pack(kind, size, 1, 0, 0, 0.0, 0.0, rows, *[0] * 24))


def _rows_forward(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block, train):
    """The stream, its norm (empty where there is no `x`) and statistics (empty where there is no training)."""
    stream = block.new_empty(block.shape)
    normed = block.new_empty(block.shape if x is not None else 0)
    rows = block.numel() // block.shape[-1]
    stats = torch.empty((rows, 2) if train else 0, dtype=torch.float32, device=block.device)
    if rows:
        _call('cuju_row_norm_forward', _rows(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block, stream,
                                             normed if x is not None else None, stats if train else None), block.device)
    return stream, normed, stats


def _rows_backward(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block, stats, d_stream, d_normed, asked):
    """The gradients of the six tensors; empty where they are not asked for."""
    size = block.shape[-1]
    maps = [block.new_empty(block.shape if of else 0) for of in asked[:3]]
    sums = [torch.empty(size if of else 0, dtype=torch.float32, device=block.device) for of in asked[3:]]
    if block.numel():
        workspace = None
        if any(asked[3:]):
            workspace = torch.empty(_rows_bytes(TYPES[block.dtype], block.numel() // size, size), dtype=torch.uint8, device=block.device)
        gradients = [each if of else None for each, of in zip((*maps, *sums), asked)]
        _call('cuju_row_norm_backward', _rows(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block, stats=stats,
                                              d_stream=d_stream, d_normed=d_normed, gradients=gradients, workspace=workspace),
              block.device)
    else:
        for each in sums:
            each.zero_()
    return (*maps, *sums)


class _RowNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, gate, after, scales, before, *options):
        run = _operator('row_norm', _rows_forward, x, block, gate, after, scales, before)
        stream, normed, stats = run(x, block, gate, after, scales, before, *options, True)
        ctx.save_for_backward(x, block, gate, after, scales, before, stats)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return (stream, normed) if x is not None else stream

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_stream, d_normed=None):
        *inputs, stats = ctx.saved_tensors
        d_stream, d_normed = (d.contiguous() if d is not None else None for d in (d_stream, d_normed))
        run = _operator('row_norm_backward', _rows_backward, *inputs, stats, d_stream, d_normed)
        asked = list(ctx.needs_input_grad[:6])
        found = run(*inputs, *ctx.options, stats, d_stream, d_normed, asked)
        return (*[each if of else None for each, of in zip(found, asked)], None, None, None, None)


def _row_norm(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block):
    if activation not in GATES:
        raise ChoiceError(f"expected the activation 'none', 'sigmoid' or 'silu', found {activation!r}")
    if block.dtype not in TYPES:
        raise ArgumentError(f'expected rows of float32, bfloat16 or float16, found {block.dtype}')
    if block.dim() < 1 or not 1 <= block.shape[-1] <= MOST_ROW:
        raise ArgumentError(f'expected rows of 1 to {MOST_ROW} values, found the shape {tuple(block.shape)}')
    if block.dim() > 2 and block.shape[-2] >= 1 << 31:
        raise ArgumentError(f'expected fewer than 2^31 rows on an axis, found the shape {tuple(block.shape)}')
    for name, each in (('x', x), ('gate', gate)):
        if each is not None:
            _shape(name, each, block.shape)
            if each.dtype != block.dtype:
                raise ArgumentError(f'expected {name} of {block.dtype}, found {each.dtype}')
    vectors = []
    for name, each in (('the weight after the block', after), ('scale', scales), ('weight', before)):
        if each is not None:
            _shape(name, each, block.shape[-1:])
            each = _gate(name, each).contiguous()
        vectors.append(each)
    inputs = _in_rows(x), _in_rows(block), _in_rows(gate), *vectors
    options = float(scale), float(epsilon), GATES[activation], norm_block
    if _learns(*inputs):
        return _RowNorm.apply(*inputs, *options)
    run = _operator('row_norm', _rows_forward, *inputs)
    stream, normed, _ = run(*inputs, *options, False)
    return (stream, normed) if x is not None else stream


def rms_norm(x, weight=None, gate=None, *, epsilon=1e-6, activation='silu'):
    """The root-mean-square norm of the rows of `x` [..., size], with a gate: `weight * x / sqrt(mean(x^2) + epsilon) *
    activation(gate)`.

    `weight` ([size], held in 32 bits) is by default ones; `gate` has the shape and type of `x`, and `activation`
    is 'none', 'sigmoid' or 'silu' of it. Rows are runs of the last axis, of up to 8192 values: for a norm of
    each head that is the head's. The output has the type and shape of `x`, contiguous. Strides are free; what does
    not lie in rows is copied. Gradients reach `x`, `weight` and `gate`; they are the same on every call.
    """
    _device('x', x, ('weight', 'gate'), (weight, gate))
    return _row_norm(None, x, gate, weight, None, None, 1.0, epsilon, activation, True)


def residual_norm(x, block, weight=None, *, after=None, gate=None, scale=None, epsilon=1e-6, activation='sigmoid'):
    """A block's end and the next block's start: `(stream, normed)`, with rows along the last axis.

    The block's output is normed by its root mean square and multiplied by `after`, where that is given, and
    multiplied by `activation(gate)`, where there is a gate. `stream = x + scale * output`, and
    `normed = weight * stream / sqrt(mean(stream^2) + epsilon)`.

    * `x`, `block`, `gate`: [..., size] of one shape and type, with a size of up to 8192. Strides are free; what does not
      lie in rows is copied.
    * `weight`, `after`: [size], held in 32 bits; `weight` is by default ones. A norm after the block without a
      weight takes ones.
    * `scale`: a number, by default 1, or a tensor [size] or [] that may be learnt.
    * `activation`: 'none', 'sigmoid' or 'silu', of the gate.

    Both outputs have the type and shape of `x`, contiguous; `normed` is of the stream before it is rounded to that
    type. Gradients reach every tensor; they are the same on every call.
    """
    learnt = scale if isinstance(scale, torch.Tensor) else None
    _device('x', x, ('block', 'weight', 'after', 'gate', 'scale'), (block, weight, after, gate, learnt))
    if block is None:
        raise ArgumentError('expected a block')
    if learnt is not None and learnt.dim() == 0 and x.dim():
        learnt = learnt.expand(x.shape[-1])
    number = 1.0 if learnt is not None or scale is None else scale
    return _row_norm(x, block, gate, after, learnt, weight, number, epsilon, activation, after is not None)


# --------------------------------------------------------------------------------- clipped gradients

def _dense(tensor) -> bool:
    """Whether `tensor`'s values lie side by side in memory, in any order of its axes."""
    if tensor.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(tensor.stride(), tensor.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _clip(gradients, most, epsilon):
    device = gradients[0].device
    norm = torch.empty((), dtype=torch.float32, device=device)
    table = array.array('q')
    for each in gradients:
        table.extend((each.data_ptr(), each.numel(), TYPES[each.dtype]))
    address, _ = table.buffer_info()
    size = _library().cuju_clip_gradients_workspace(_GRADIENTS.pack(len(gradients), address, most, epsilon, 0, 0))
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    try:
        _call('cuju_clip_gradients', _GRADIENTS.pack(len(gradients), address, most, epsilon, norm.data_ptr(), _pointer(workspace)), device)
    except LibraryError as error:
        # The library looks whether tensors overlap.
        raise ArgumentError(str(error)) from None
    torch.autograd.graph.increment_version(gradients)
    return norm


def clip_gradients(gradients, most, *, epsilon=1e-6):
    """Clips the gradients of an update by their global norm, in place, and returns the norm they had.

    `gradients` is a tensor or some of them, of float32, bfloat16 or float16, mixed at will, on one device; None
    among them (a parameter that has no gradient) is passed over. The norm is the root of the sum of all squares,
    summed in 64 bits in an order that is always the same. Every value is multiplied by
    `min(1, most / (norm + epsilon))`; gradients below `most` are not written, and with `most` of infinity none
    are. A norm that is not finite spreads, as in the formula. The values of a tensor have to lie side by side
    in memory, and no two tensors may share any. The norm is a float32 tensor [] on the device, and nothing waits for it; one
    past the range of float32 is returned as infinity, and clips by its value.
    """
    gradients = [gradients] if isinstance(gradients, torch.Tensor) else [each for each in gradients if each is not None]
    if not gradients:
        raise ArgumentError('expected a gradient')
    most, epsilon = float(most), float(epsilon)
    if not most >= 0 or not epsilon >= 0:
        raise ArgumentError(f'expected a norm and an epsilon of at least 0, found {most} and {epsilon}')
    _device('gradients', gradients[0], ('all gradients',) * len(gradients), tuple(gradients))
    for each in gradients:
        if each.dtype not in TYPES:
            raise ArgumentError(f'expected gradients of float32, bfloat16 or float16, found {each.dtype}')
        if each.layout != torch.strided or not _dense(each):
            raise ArgumentError(f'expected gradients whose values lie side by side, found one of the shape {tuple(each.shape)}')
    if _learns(*gradients):
        raise ArgumentError('clip_gradients has no gradients of its own: call it under torch.no_grad()')
    return _operator('clip_gradients', _clip, *gradients)(gradients, most, epsilon)


# -------------------------------------------------------------------------- operators of torch.compile

_NAMESPACE = torch.library.Library('cuju_amd', 'FRAGMENT')
_INPUTS = 'Tensor query, Tensor key, Tensor value, Tensor decay, Tensor beta'
_NAMESPACE.define(f'delta_rule({_INPUTS}, Tensor? state, Tensor? resets, float scale, bool train) -> '
                  '(Tensor, Tensor, Tensor)')
_NAMESPACE.define(f'delta_rule_backward({_INPUTS}, Tensor? state, Tensor? resets, float scale, Tensor checkpoints, '
                  'Tensor d_output, Tensor? d_last) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)')
_NAMESPACE.define(f'delta_rule_step({_INPUTS}, Tensor(a!) state, Tensor? resets, float scale) -> Tensor')
_NAMESPACE.define('linear_attention(Tensor query, Tensor key, Tensor value, Tensor decay, Tensor? state, Tensor? resets, '
                  'float scale, bool train) -> (Tensor, Tensor, Tensor)')
_NAMESPACE.define('linear_attention_backward(Tensor query, Tensor key, Tensor value, Tensor decay, Tensor? state, Tensor? resets, '
                  'float scale, Tensor checkpoints, Tensor d_output, Tensor? d_last, bool of_decay) -> '
                  '(Tensor, Tensor, Tensor, Tensor, Tensor)')
_NAMESPACE.define('linear_attention_step(Tensor query, Tensor key, Tensor value, Tensor decay, Tensor(a!) state, Tensor? resets, '
                  'float scale) -> Tensor')
_NAMESPACE.define('group_norm(Tensor x, Tensor? weight, Tensor? bias, int groups, float epsilon, int activation) -> '
                  '(Tensor, Tensor)')
_NAMESPACE.define('group_norm_backward(Tensor x, Tensor? weight, Tensor? bias, Tensor stats, Tensor dy, int groups, '
                  'float epsilon, int activation, bool of_weight, bool of_bias) -> (Tensor, Tensor, Tensor)')
_ROW_INPUTS = ('Tensor? x, Tensor block, Tensor? gate, Tensor? after, Tensor? scales, Tensor? before, float scale, float epsilon, '
               'int activation, bool norm_block')
_NAMESPACE.define(f'row_norm({_ROW_INPUTS}, bool train) -> (Tensor, Tensor, Tensor)')
_NAMESPACE.define(f'row_norm_backward({_ROW_INPUTS}, Tensor stats, Tensor? d_stream, Tensor? d_normed, bool[] asked) -> '
                  '(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)')
_NAMESPACE.define('clip_gradients(Tensor(a!)[] gradients, float most, float epsilon) -> Tensor')
_NAMESPACE.impl('delta_rule', _rule_forward, 'CUDA')
_NAMESPACE.impl('delta_rule_backward', _rule_backward, 'CUDA')
_NAMESPACE.impl('delta_rule_step', _rule_step, 'CUDA')
_NAMESPACE.impl('linear_attention', _attention_forward, 'CUDA')
_NAMESPACE.impl('linear_attention_backward', _attention_backward, 'CUDA')
_NAMESPACE.impl('linear_attention_step', _attention_step, 'CUDA')
_NAMESPACE.impl('group_norm', _norm_forward, 'CUDA')
_NAMESPACE.impl('group_norm_backward', _norm_backward, 'CUDA')
_NAMESPACE.impl('row_norm', _rows_forward, 'CUDA')
_NAMESPACE.impl('row_norm_backward', _rows_backward, 'CUDA')
_NAMESPACE.impl('clip_gradients', _clip, 'CUDA')


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


@torch.library.register_fake('cuju_amd::linear_attention')
def _(query, key, value, decay, state, resets, scale, train):
    batch, time, _, key_size = query.shape
    heads, value_size = value.shape[2:]
    kept = max(time - 1, 0) // SPAN if train else 0
    return (value.new_empty(value.shape), decay.new_empty((batch, heads, key_size, value_size)),
            decay.new_empty((batch, heads, kept, key_size, value_size)))


@torch.library.register_fake('cuju_amd::linear_attention_backward')
def _(query, key, value, decay, state, resets, scale, checkpoints, d_output, d_last, of_decay):
    batch, _, _, key_size = query.shape
    return (*[x.new_empty(x.shape) for x in (query, key, value)], decay.new_empty(decay.shape if of_decay else (0,)),
            decay.new_empty((batch, value.shape[2], key_size, value.shape[3])))


@torch.library.register_fake('cuju_amd::linear_attention_step')
def _(query, key, value, decay, state, resets, scale):
    return value.new_empty(value.shape)


@torch.library.register_fake('cuju_amd::group_norm')
def _(x, weight, bias, groups, epsilon, activation):
    return x.new_empty(x.shape), x.new_empty((x.shape[0], groups, 2), dtype=torch.float32)


@torch.library.register_fake('cuju_amd::group_norm_backward')
def _(x, weight, bias, stats, dy, groups, epsilon, activation, of_weight, of_bias):
    sums = (x.new_empty((x.shape[-1] if asked else 0,), dtype=torch.float32) for asked in (of_weight, of_bias))
    return x.new_empty(x.shape), *sums


@torch.library.register_fake('cuju_amd::row_norm')
def _(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block, train):
    rows = block.numel() // block.shape[-1]
    return (block.new_empty(block.shape), block.new_empty(block.shape if x is not None else (0,)),
            block.new_empty((rows, 2) if train else (0,), dtype=torch.float32))


@torch.library.register_fake('cuju_amd::row_norm_backward')
def _(x, block, gate, after, scales, before, scale, epsilon, activation, norm_block, stats, d_stream, d_normed, asked):
    maps = (block.new_empty(block.shape if of else (0,)) for of in asked[:3])
    return *maps, *(block.new_empty((block.shape[-1] if of else 0,), dtype=torch.float32) for of in asked[3:])


@torch.library.register_fake('cuju_amd::clip_gradients')
def _(gradients, most, epsilon):
    return gradients[0].new_empty((), dtype=torch.float32)
