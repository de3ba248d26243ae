"""The definitions of the policy operators in 64 bits, step by step, for the tests: values and
gradients written out, on the CPU."""

import torch


def delta_rule(query, key, value, decay, beta, state=None, resets=None, scale=None, d_output=None, d_last=None):
    """`(output, last)` of the gated delta rule, or with `d_output` a dictionary of them and all gradients.
    A step that is reset starts from zeros, whatever the memory held."""
    query, key, value, decay, beta = (x.detach().cpu().double() for x in (query, key, value, decay, beta))
    batch, time, key_heads, key_size = query.shape
    heads, value_size = value.shape[2:]
    group = heads // key_heads
    scale = key_size ** -0.5 if scale is None else scale
    q, k = query.repeat_interleave(group, 2), key.repeat_interleave(group, 2)
    if state is None:
        memory = torch.zeros(batch, heads, key_size, value_size, dtype=torch.double)
    else:
        memory = state.detach().cpu().double()
    cleared = torch.zeros(batch, time, dtype=torch.bool) if resets is None else resets.cpu().bool()
    output = torch.zeros(batch, time, heads, value_size, dtype=torch.double)
    held, errors = [], []
    for t in range(time):
        memory = memory * decay[:, t].exp()[..., None, None]
        memory = torch.where(cleared[:, t, None, None, None], torch.zeros_like(memory), memory)
        error = value[:, t] - torch.einsum('bhkv,bhk->bhv', memory, k[:, t])
        held.append(memory)
        errors.append(error)
        memory = memory + torch.einsum('bhk,bhv->bhkv', k[:, t], beta[:, t, :, None] * error)
        output[:, t] = scale * torch.einsum('bhkv,bhk->bhv', memory, q[:, t])
    if d_output is None:
        return output, memory
    d_output = d_output.detach().cpu().double()
    d_memory = torch.zeros_like(memory) if d_last is None else d_last.detach().cpu().double()
    d_q, d_k, d_v, d_decay, d_beta = (torch.zeros_like(x) for x in (q, k, value, decay, beta))
    for t in reversed(range(time)):
        written = beta[:, t, :, None] * errors[t]
        after = held[t] + torch.einsum('bhk,bhv->bhkv', k[:, t], written)
        d_q[:, t] = scale * torch.einsum('bhkv,bhv->bhk', after, d_output[:, t])
        d_memory = d_memory + scale * torch.einsum('bhk,bhv->bhkv', q[:, t], d_output[:, t])
        d_written = torch.einsum('bhkv,bhk->bhv', d_memory, k[:, t])
        d_error = beta[:, t, :, None] * d_written
        d_beta[:, t] = (d_written * errors[t]).sum(-1)
        d_v[:, t] = d_error
        d_k[:, t] = (torch.einsum('bhkv,bhv->bhk', d_memory, written) - torch.einsum('bhkv,bhv->bhk', held[t], d_error))
        d_memory = d_memory - torch.einsum('bhk,bhv->bhkv', k[:, t], d_error)
        d_decay[:, t] = (d_memory * held[t]).sum((-2, -1))
        d_memory = d_memory * decay[:, t].exp()[..., None, None]
        d_memory = torch.where(cleared[:, t, None, None, None], torch.zeros_like(d_memory), d_memory)

    def shared(x):
        return x.reshape(batch, time, key_heads, group, key_size).sum(3)

    return {'output': output, 'last': memory, 'd_query': shared(d_q), 'd_key': shared(d_k), 'd_value': d_v,
            'd_decay': d_decay, 'd_beta': d_beta, 'd_state': d_memory}


def group_norm(x, groups, weight=None, bias=None, epsilon=1e-5, activation='none', dy=None):
    """`y`, or with `dy` a dictionary of it and all gradients."""
    shape = x.shape
    channels = shape[-1]
    x = x.detach().cpu().double().reshape(shape[0], -1, channels)
    weight = torch.ones(channels, dtype=torch.double) if weight is None else weight.detach().cpu().double()
    bias = torch.zeros(channels, dtype=torch.double) if bias is None else bias.detach().cpu().double()
    part = x.reshape(shape[0], -1, groups, channels // groups)
    mean = part.mean((1, 3), keepdim=True)
    inverse = 1 / (((part - mean) ** 2).mean((1, 3), keepdim=True) + epsilon).sqrt()
    xh = ((part - mean) * inverse).reshape(x.shape)
    z = xh * weight + bias
    sigmoid = 1 / (1 + (-z).exp())
    y = {'none': z, 'relu': z.clamp_min(0), 'silu': z * sigmoid}[activation]
    if dy is None:
        return y.reshape(shape)
    slope = {'none': torch.ones_like(z), 'relu': (z > 0).double(), 'silu': sigmoid * (1 + z * (1 - sigmoid))}[activation]
    dz = dy.detach().cpu().double().reshape(x.shape) * slope
    inner = (dz * weight).reshape(part.shape)
    xh = xh.reshape(part.shape)
    dx = inverse * (inner - inner.mean((1, 3), keepdim=True) - xh * (inner * xh).mean((1, 3), keepdim=True))
    # `terms`: the size of the three terms whose difference dx is.
    return {'y': y.reshape(shape), 'dx': dx.reshape(shape), 'terms': float((inverse * inner).norm()), 'd_weight': (dz * xh.reshape(x.shape)).sum((0, 1)),
            'd_bias': dz.sum((0, 1))}
