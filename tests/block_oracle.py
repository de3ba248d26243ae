"""The definitions of the operators of a policy's blocks in 64 bits, for the tests: values and gradients written
out, where the tensors are."""

import torch


def attention(query, key, value, decay, state=None, resets=None, scale=None, d_output=None, d_last=None):
    """`(output, last)` of linear attention with decays, or with `d_output` a dictionary of them, all gradients, and
    `dots`, the sum of the products of queries and keys with their gradients, each without its own step's, and of the
    last memory with its gradient. A step that is reset starts from zeros, whatever the memory held."""
    query, key, value, decay = (x.detach().double() for x in (query, key, value, decay))
    batch, time, key_heads, key_size = query.shape
    heads, value_size = value.shape[2:]
    group, of_heads = heads // key_heads, decay.dim() == 1
    decay = decay.expand(batch, time, heads)
    scale = key_size ** -0.5 if scale is None else scale
    q, k = query.repeat_interleave(group, 2), key.repeat_interleave(group, 2)
    memory = value.new_zeros(batch, heads, key_size, value_size)
    if state is not None:
        memory = state.detach().double()
    cleared = torch.zeros(batch, time, dtype=torch.bool, device=value.device) if resets is None else resets.bool()
    output = value.new_zeros(batch, time, heads, value_size)
    held = []
    for t in range(time):
        memory = torch.where(cleared[:, t, None, None, None], 0.0, memory * decay[:, t].exp()[..., None, None])
        held.append(memory)
        memory = memory + k[:, t, :, :, None] * value[:, t, :, None, :]
        output[:, t] = scale * (memory * q[:, t, :, :, None]).sum(-2)
    if d_output is None:
        return output, memory
    d_output = d_output.detach().double()
    last, d_memory = memory, torch.zeros_like(memory) if d_last is None else d_last.detach().double()
    d_q, d_k, d_v, d_decay = (torch.zeros_like(x) for x in (q, k, value, decay))
    dots = (last * d_memory).sum()
    for t in reversed(range(time)):
        after = held[t] + k[:, t, :, :, None] * value[:, t, :, None, :]
        d_q[:, t] = scale * (after * d_output[:, t, :, None, :]).sum(-1)
        dots = dots + ((d_memory * value[:, t, :, None, :]).sum(-1) * k[:, t]).sum()
        dots = dots + (scale * (held[t] * d_output[:, t, :, None, :]).sum(-1) * q[:, t]).sum()
        d_memory = d_memory + scale * q[:, t, :, :, None] * d_output[:, t, :, None, :]
        d_k[:, t] = (d_memory * value[:, t, :, None, :]).sum(-1)
        d_v[:, t] = (d_memory * k[:, t, :, :, None]).sum(-2)
        d_decay[:, t] = (d_memory * held[t]).sum((-2, -1))
        d_memory = torch.where(cleared[:, t, None, None, None], 0.0, d_memory * decay[:, t].exp()[..., None, None])

    def shared(x):
        return x.reshape(batch, time, key_heads, group, key_size).sum(3)

    return {'output': output, 'last': last, 'd_query': shared(d_q), 'd_key': shared(d_k), 'd_value': d_v,
            'd_decay': d_decay.sum((0, 1)) if of_heads else d_decay, 'd_state': d_memory, 'dots': dots}


def attention_terms(query, key, value, decay, state=None, resets=None, scale=None, d_output=None, d_last=None):
    """The 2-norms of all terms that the results of `attention` are sums of, by name: the square of a term is the same
    product of the squared inputs. That of `d_decay` is of the dots that it is a sum of."""
    squares = [x.detach().double().square() for x in (query, key, value)]
    square = lambda x: x.detach().double().square() if x is not None else None  # noqa: E731
    scale = query.shape[-1] ** -0.5 if scale is None else scale
    if d_output is None:
        d_output = torch.zeros_like(value)
    found = attention(*squares, 2 * decay.detach().double(), square(state), resets, scale ** 2, square(d_output), square(d_last))
    found['d_decay'] = found['dots']
    return {name: float(x.sum()) ** 0.5 for name, x in found.items() if name != 'dots'}


def gate(x, activation):
    """The factor of a gate and its derivative."""
    s = torch.sigmoid(x)
    return {'none': (x, torch.ones_like(x)), 'sigmoid': (s, s * (1 - s)), 'silu': (x * s, s * (1 + x * (1 - s)))}[activation]


def unit(x, epsilon):
    """`(x inverse, inverse)` for the inverse of the root mean square of the rows."""
    inverse = 1 / ((x * x).mean(-1, keepdim=True) + epsilon).sqrt()
    return x * inverse, inverse


def rows(block, x=None, gates=None, after=None, scale=None, before=None, epsilon=1e-6, activation='silu', norm_block=True,
         d_stream=None, d_normed=None):
    """A dictionary of the outputs of a norm of rows, and with the outputs' gradients of all gradients. Those that are
    the differences of like terms come with the terms' size."""
    double = lambda t: t.detach().double() if t is not None else None  # noqa: E731
    block, x, gates, after, scale, before = (double(t) for t in (block, x, gates, after, scale, before))
    ones, columns = block.new_ones(block.shape[-1]), lambda t: t.reshape(-1, t.shape[-1]).sum(0)  # noqa: E731
    after, scale, before = (ones if t is None else t for t in (after, scale, before))
    factor, slope = gate(gates, activation) if gates is not None else (torch.ones_like(block), None)
    u, inner = unit(block, epsilon) if norm_block else (block, torch.ones_like(block[..., :1]))
    h = after * factor * u
    found = {}
    if x is not None:
        h = x + scale * h
        e, outer = unit(h, epsilon)
        found['normed'] = before * e
    found['stream'] = h
    if d_stream is None and d_normed is None:
        return found
    dh = double(d_stream) if d_stream is not None else torch.zeros_like(h)
    if x is not None:
        dy = double(d_normed) if d_normed is not None else torch.zeros_like(h)
        found['d_before'] = columns(dy * e)
        de = dy * before
        found['terms'] = float((outer * de).norm())
        dh = dh + outer * (de - e * (de * e).mean(-1, keepdim=True))
        found['d_x'] = dh
        found['d_scale'] = columns(dh * after * factor * u)
    found['d_after'] = columns(dh * scale * factor * u)
    if gates is not None:
        found['d_gate'] = dh * scale * after * u * slope
    du = dh * scale * after * factor
    found['terms'] = max(found.get('terms', 0.0), float((inner * du).norm()))
    found['d_block'] = inner * (du - u * (du * u).mean(-1, keepdim=True)) if norm_block else du
    return found


def clip(gradients, most, epsilon=1e-6):
    """The global norm and the clipped gradients."""
    gradients = [g.detach().double() for g in gradients]
    norm = sum(float((g * g).sum()) for g in gradients) ** 0.5
    factor = min(1.0, most / (norm + epsilon))
    return norm, [g * factor for g in gradients]
