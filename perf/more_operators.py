"""What the operators of a deeper policy in `cuju_amd.layers` are measured on.

A case is one operator and one kind of call:

* "act": one step of linear attention with decays for every agent of a batch, the state updated in place;
* "replay": linear attention over a stretch of steps, forward;
* "learn": the same with every gradient;
* "norm", "norm learn": the root-mean-square norm of rows with a gate, forward and with every gradient;
* "block", "block learn": a block's output normed, gated, scaled and added to the residual stream, and the
  stream's norm for the next block, forward and with every gradient;
* "clip": the norm of all gradients of an update, and the gradients clipped by it, in place.

The plain form (`own` false) is elementary torch operations in 32 bits; sums of log decays and of the squares of
many gradients are in 64.
"""

import torch

own = False

TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
BYTES = {'float32': 4, 'bfloat16': 2, 'float16': 2}
EPSILON = 1e-6


def _attention(**given):
    case = dict(call='act', batch=1, time=1, key_heads=4, heads=4, key_size=64, value_size=64, dtype='bfloat16',
                initial=True, fixed=False, episode=0)
    case.update(given)
    return case


def _norm(**given):
    case = dict(call='norm', rows=1, heads=1, size=64, dtype='bfloat16', gate='silu')
    case.update(given)
    return case


def _block(**given):
    case = dict(call='block', rows=1, size=256, dtype='bfloat16', after=True, gate='sigmoid', scaled=True)
    case.update(given)
    return case


def _clip(**given):
    case = dict(call='clip', layers=1, width=64, half=False, most=1.0)
    case.update(given)
    return case


def listed():
    return [
        # Acting in one match with all eleven players of a side: latency alone.
        _attention(name='act 11v11 x1', batch=11, episode=3000),
        # Acting in the headline workload: 16,384 matches of 11 agents.
        _attention(name='act 11v11 x16384', batch=180224, key_heads=2, heads=2, episode=3000),
        # Reading a whole match of 3,000 steps again, for its values, with wide heads.
        _attention(name='replay match x1', call='replay', batch=11, time=3000, key_heads=2, heads=4, key_size=128,
                   value_size=128, initial=False),
        # One update of a small training batch: 64 matches of 4 agents, 128 steps.
        _attention(name='learn 5v5 x64', call='learn', batch=256, time=128, episode=3000),
        # One update on the 4,096-match workload with one agent, 64 steps.
        _attention(name='learn 11v11 x4096', call='learn', batch=4096, time=64, episode=3000),
        # A ragged one in 32 bits: heads that share keys, one decay learnt for each, episodes that end often.
        _attention(name='learn ragged', call='learn', batch=37, time=301, key_heads=2, heads=6, key_size=48,
                   value_size=80, dtype='float32', fixed=True, episode=20),
        # What the memories of one match's agents answer, normed and gated by head: latency alone.
        _norm(name='norm 11v11 x1', rows=11, heads=4),
        # The same in the update on 4,096 matches of 64 steps.
        _norm(name='norm learn x4096', call='norm learn', rows=262144, heads=4),
        # A block's end and the next one's norm in that update, with everything that it may have.
        _block(name='block learn x4096', call='block learn', rows=262144),
        # Odd rows in 32 bits, with the plainest block.
        _block(name='block learn ragged', call='block learn', rows=5003, size=1001, dtype='float32', after=False,
               gate='', scaled=False),
        # The gradients of a policy of two blocks, in 32 bits: latency alone.
        _clip(name='clip policy', layers=2, width=256),
        # Those of a large one, in 32 and 16 bits.
        _clip(name='clip large', layers=7, width=4096, half=True),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm from `low` to `high`."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    call = rng.choice(('act', 'replay', 'learn', 'learn', 'norm', 'norm learn', 'block', 'block learn', 'clip'))
    dtype = rng.choice(('bfloat16', 'bfloat16', 'float16', 'float32'))
    if call == 'clip':
        return _clip(layers=_spread(rng, 1, 6), width=_spread(rng, 16, 4096), half=rng.random() < 0.5,
                     most=rng.choice((0.5, 1.0, 1e9)))
    if call.startswith('norm'):
        size, heads = _spread(rng, 8, 4096), rng.choice((1, 1, 2, 4, 6))
        return _norm(call=call, rows=_spread(rng, 1, min(262144, 60_000_000 // (size * heads))), heads=heads, size=size,
                     dtype=dtype, gate=rng.choice(('silu', 'sigmoid', 'none', '')))
    if call.startswith('block'):
        size = _spread(rng, 8, 8192)
        return _block(call=call, rows=_spread(rng, 1, min(262144, 60_000_000 // size)), size=size, dtype=dtype,
                      after=rng.random() < 0.6, gate=rng.choice(('silu', 'sigmoid', 'none', '', '')),
                      scaled=rng.random() < 0.6)
    key_heads = rng.choice((1, 2, 3, 4))
    heads = key_heads * rng.choice((1, 1, 2, 3))
    key_size = rng.choice((16, 24, 32, 40, 64, 64, 96, 128))
    value_size = rng.choice((16, 32, 64, 64, 72, 100, 128))
    size = heads * key_size * value_size
    if call == 'act':
        time, most = 1, 700_000_000 // size
    else:
        time = _spread(rng, 1, 600 if call == 'learn' else 3000)
        most = max(1, 4_000_000_000 // (size * time))
    return _attention(call=call, batch=_spread(rng, 1, min(most, 32768)), time=time, key_heads=key_heads, heads=heads,
                      key_size=key_size, value_size=value_size, dtype=dtype,
                      initial=call == 'act' or rng.random() < 0.7, fixed=rng.random() < 0.4,
                      episode=rng.choice((0, 20, 400, 3000)))


def _shapes(case):
    """The shapes of a policy's parameters: in each block two norms' weights, the memory's projections and rates, and
    two products with their shifts."""
    width = case['width']
    block = [(width,), (3 * width + width // 8 + 1, width), (width // 8 + 1,), (width, width), (width,), (2 * width, width),
             (2 * width,), (width, 2 * width)]
    return block * case['layers']


def prepare(case, seed):
    generator = torch.Generator(device='cuda')
    generator.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device='cuda')

    state = {'case': case}
    if case['call'] == 'clip':
        # Gradients lie side by side in a buffer of each type, as they do where ranks add them up together.
        shapes = _shapes(case)
        counts = [torch.Size(shape).numel() for shape in shapes]
        kinds = [torch.bfloat16 if case['half'] and len(shape) > 1 else torch.float32 for shape in shapes]
        state['buffers'] = {}
        for kind in sorted(set(kinds), key=str):
            total = sum(n for n, each in zip(counts, kinds) if each == kind)
            state['buffers'][str(kind)] = (0.02 * normal(total)).to(kind)
        state['gradients'], used = [], dict.fromkeys(state['buffers'], 0)
        for shape, count, kind in zip(shapes, counts, kinds):
            at = used[str(kind)]
            state['gradients'].append(state['buffers'][str(kind)][at:at + count].view(shape))
            used[str(kind)] = at + count
        state['most'] = case['most']
        return state

    kind = TYPES[case['dtype']]
    learn = case['call'].endswith('learn')
    if case['call'].startswith('norm'):
        shape = (case['rows'], case['heads'], case['size'])
        # What memories answer: every row has its own level, from next to nothing to some units.
        state['x'] = (normal(*shape) * torch.exp(2 * normal(*shape[:2], 1))).to(kind)
        state['weight'] = 1 + 0.2 * normal(case['size'])
        state['gate'] = normal(*shape).to(kind) if case['gate'] else None
        if learn:
            state['dy'] = (0.01 * normal(*shape)).to(kind)
        return state
    if case['call'].startswith('block'):
        shape = (case['rows'], case['size'])
        state['x'] = (3 * normal(*shape)).to(kind)
        state['block'] = normal(*shape).to(kind)
        state['gate'] = normal(*shape).to(kind) if case['gate'] else None
        state['after'] = 1 + 0.2 * normal(case['size']) if case['after'] else None
        state['scale'] = 0.5 + 0.2 * normal(case['size']) if case['scaled'] else None
        state['before'] = 1 + 0.2 * normal(case['size'])
        if learn:
            state['d_stream'], state['d_normed'] = ((0.01 * normal(*shape)).to(kind) for _ in range(2))
        return state

    batch, time, key_heads, heads = case['batch'], case['time'], case['key_heads'], case['heads']
    key_size, value_size = case['key_size'], case['value_size']

    def directions(count):
        # Unit vectors that keep a direction of their own through a match: one step is like the next.
        x = normal(batch, time, count, key_size).add_(normal(batch, 1, count, key_size))
        return x.div_(x.norm(dim=-1, keepdim=True)).to(kind)

    state['query'] = directions(key_heads)
    state['key'] = directions(key_heads)
    state['value'] = normal(batch, time, heads, value_size).to(kind)
    # Memories from a few steps to some thousand, by head.
    reach = torch.logspace(-3.0, -0.3, heads, device='cuda')
    if case['fixed']:
        state['decay'] = -reach
    else:
        state['decay'] = -reach * torch.nn.functional.softplus(normal(batch, time, heads))
    state['resets'] = None
    if case['episode']:
        state['resets'] = torch.rand(batch, time, generator=generator, device='cuda') < 1 / case['episode']
    state['state'] = 0.3 * normal(batch, heads, key_size, value_size) if case['initial'] else None
    if case['call'] == 'act':
        for name in ('query', 'key', 'value', 'resets') + (() if case['fixed'] else ('decay',)):
            state[name] = state[name].squeeze(1) if state[name] is not None else None
    if learn:
        state['d_output'] = normal(batch, time, heads, value_size).mul_(0.01).to(kind)
        state['d_state'] = 0.01 * normal(batch, heads, key_size, value_size)
    return state


def run(state):
    case = state['case']
    if case['call'] == 'clip':
        # The most that is left falls a little from update to update, so that gradients clipped before are clipped again.
        most, state['most'] = state['most'], state['most'] * 0.999
        return {'norm': _clip_gradients(state['gradients'], most), **state['buffers']}
    if case['call'] == 'act':
        return {'output': _step(state), 'state': state['state']}
    if case['call'] == 'replay':
        return dict(zip(('output', 'last'), _attend(*(state[n] for n in ('query', 'key', 'value', 'decay', 'state', 'resets')))))
    if case['call'] == 'learn':
        return _learn(state, ('query', 'key', 'value', 'decay', 'state'), ('output', 'last'), ('d_output', 'd_state'),
                      lambda q, k, v, decay, first: _attend(q, k, v, decay, first, state['resets']))
    if case['call'] == 'norm':
        return _rms_norm(state['x'], state['weight'], state['gate'], case['gate'])
    if case['call'] == 'norm learn':
        return _learn(state, ('x', 'weight', 'gate'), ('y',), ('dy',),
                      lambda x, weight, gate: (_rms_norm(x, weight, gate, case['gate']),))
    names = 'x', 'block', 'after', 'gate', 'scale', 'before'
    if case['call'] == 'block':
        return dict(zip(('stream', 'normed'), _residual_norm(*(state[n] for n in names), case['gate'])))
    return _learn(state, names, ('stream', 'normed'), ('d_stream', 'd_normed'),
                  lambda *inputs: _residual_norm(*inputs, case['gate']))


def _learn(state, names, outputs, gradients, call):
    """One training pass of `call`: its outputs and the gradients of every input."""
    inputs = {name: state[name].detach().requires_grad_() if state[name] is not None else None for name in names}
    results = call(*inputs.values())
    learnt = {name: x for name, x in inputs.items() if x is not None}
    found = torch.autograd.grad(results, list(learnt.values()), [state[name] for name in gradients])
    return {**{name: x.detach() for name, x in zip(outputs, results)},
            **{'grad_' + name: x for name, x in zip(learnt, found)}}


def _clip_gradients(gradients, most):
    if own:
        from cuju_amd import layers
        return layers.clip_gradients(gradients, most, epsilon=EPSILON)
    norm = torch.stack([g.double().square().sum() for g in gradients]).sum().sqrt().float()
    factor = (most / (norm + EPSILON)).clamp(max=1)
    for gradient in gradients:
        gradient.copy_(gradient.float() * factor)
    return norm


def _step(state):
    query, key, value, decay, memory, resets = (state[n] for n in ('query', 'key', 'value', 'decay', 'state', 'resets'))
    if own:
        from cuju_amd import layers
        return layers.linear_attention_step(query, key, value, decay, memory, resets=resets)
    kind, group = value.dtype, memory.shape[1] // key.shape[1]
    query, key = query.float().repeat_interleave(group, 1), key.float().repeat_interleave(group, 1)
    kept = decay.exp()
    if resets is not None:
        kept = kept * ~resets[:, None]
    memory.mul_(kept[..., None, None]).add_(key[..., :, None] * value.float()[..., None, :])
    return (torch.matmul(query[..., None, :], memory).squeeze(-2) * query.shape[-1] ** -0.5).to(kind)


def _attend(query, key, value, decay, memory, resets):
    if own:
        from cuju_amd import layers
        return layers.linear_attention(query, key, value, decay, state=memory, resets=resets)
    batch, time, heads, value_size = value.shape
    key_size, kind = key.shape[-1], value.dtype
    chunk = min(64, 1 << (time - 1).bit_length())
    count = -(-time // chunk)
    short = count * chunk - time

    def split(x):
        """[batch, time, heads, ...] as [batch, heads, chunk, step, ...], filled with zeros."""
        x = x.repeat_interleave(heads // x.shape[2], 2)
        x = torch.cat([x, x.new_zeros(batch, short, *x.shape[2:])], 1) if short else x
        return x.reshape(batch, count, chunk, *x.shape[2:]).movedim(3, 1)

    query, key, value = split(query.float()), split(key.float()), split(value.float())
    decay = split(decay.expand(batch, time, heads).double())
    ends = split(resets[..., None].double().expand(-1, -1, heads)) if resets is not None else torch.zeros_like(decay)

    def kept(later, earlier, seen):
        """The factors between two places, given as the sums of log decays and of resets up to them."""
        same = (later[1][..., :, None] == earlier[1][..., None, :]) & seen
        return (later[0][..., :, None] - earlier[0][..., None, :]).masked_fill(~same, -torch.inf).exp().float()

    within = decay.cumsum(-1), ends.cumsum(-1)
    lower = torch.ones(chunk, chunk, dtype=torch.bool, device=value.device).tril()
    between = kept(within, within, lower)
    whole = within[0].masked_fill(within[1] != 0, -torch.inf).exp().float()
    # The memory before each chunk and after the last: the first one, and what the chunks before have written.
    written = (between[..., -1, :, None] * key).transpose(-1, -2) @ value
    totals = tuple(torch.nn.functional.pad(x[..., -1].cumsum(-1), (1, 0)) for x in within)
    earlier = torch.ones(count + 1, count + 1, dtype=torch.bool, device=value.device).tril()
    if memory is None:
        memory = value.new_zeros(batch, heads, key_size, value_size)
    held = torch.cat([memory[:, :, None], written], 2).flatten(3)
    memories = (kept(totals, totals, earlier) @ held).unflatten(-1, (key_size, value_size))
    scores = (query @ key.transpose(-1, -2)) * between
    output = key_size ** -0.5 * (whole[..., None] * (query @ memories[:, :, :-1]) + scores @ value)
    output = output.reshape(batch, heads, count * chunk, value_size)[:, :, :time]
    return output.transpose(1, 2).to(kind), memories[:, :, -1]


def _gate(x, name):
    return x * x.sigmoid() if name == 'silu' else x.sigmoid() if name == 'sigmoid' else x


def _rms_norm(x, weight, gate, name):
    if own:
        from cuju_amd import layers
        if gate is None:
            return layers.rms_norm(x, weight, epsilon=EPSILON)
        return layers.rms_norm(x, weight, gate, epsilon=EPSILON, activation=name)
    kind, x = x.dtype, x.float()
    y = x * (x.square().mean(-1, keepdim=True) + EPSILON).rsqrt() * weight
    return (y * _gate(gate.float(), name) if gate is not None else y).to(kind)


def _residual_norm(x, block, after, gate, scale, before, name):
    if own:
        from cuju_amd import layers
        options = {'activation': name} if gate is not None else {}
        return layers.residual_norm(x, block, before, after=after, gate=gate, scale=scale, epsilon=EPSILON, **options)
    kind, x, block = x.dtype, x.float(), block.float()
    if after is not None:
        block = block * (block.square().mean(-1, keepdim=True) + EPSILON).rsqrt() * after
    if gate is not None:
        block = block * _gate(gate.float(), name)
    stream = x + (block * scale if scale is not None else block)
    normed = stream * (stream.square().mean(-1, keepdim=True) + EPSILON).rsqrt() * before
    return stream.to(kind), normed.to(kind)


def work(case):
    if case['call'] == 'clip':
        # Each gradient is read for the norm; those that are clipped are written.
        counts = [(torch.Size(s).numel(), 2 if case['half'] and len(s) > 1 else 4) for s in _shapes(case)]
        values = sum(n for n, _ in counts)
        clipped = 0.02 * values ** 0.5 > case['most']
        return {'bytes': sum(n * size for n, size in counts) * (2 if clipped else 1) + 4, 'flops': values * (3 if clipped else 2)}
    size, learn = BYTES[case['dtype']], case['call'].endswith('learn')
    if case['call'].startswith('norm'):
        values = case['rows'] * case['heads'] * case['size']
        maps = 2 + bool(case['gate'])
        # Forward: a row and its gate in, the row out. Backward: the row's gradient in, a gradient for each input.
        return {'bytes': values * size * (maps + (maps if learn else 0)) + 4 * case['size'] * (2 if learn else 1),
                'flops': values * (25 if learn else 8)}
    if case['call'].startswith('block'):
        values = case['rows'] * case['size']
        inputs = 2 + bool(case['gate'])
        vectors = 1 + case['after'] + case['scaled']
        return {'bytes': values * size * (inputs + 2 + (inputs + 2 if learn else 0)) + 4 * case['size'] * vectors * (2 if learn else 1),
                'flops': values * (40 if learn else 15)}
    batch = case['batch']
    tokens = batch * case['time']
    keys = tokens * case['key_heads'] * case['key_size'] * size
    values = tokens * case['heads'] * case['value_size'] * size
    gates = 4 * case['heads'] * (1 if case['fixed'] else tokens)
    states = batch * case['heads'] * case['key_size'] * case['value_size']
    total = 2 * keys + 2 * values + gates + (tokens if case['episode'] else 0)
    total += 4 * states * (2 if case['initial'] else 1)
    # A step scales the memory, adds a product to it and reads it once: 5 operations a value of it.
    flops = 5 * tokens * case['heads'] * case['key_size'] * case['value_size']
    if learn:
        total += 2 * keys + 2 * values + gates + 4 * states * (2 if case['initial'] else 1)
        flops *= 3
    return {'bytes': total, 'flops': flops}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case['call'] == 'clip':
            norm = sum(float(torch.linalg.vector_norm(x.double())) ** 2 for x in state['buffers'].values()) ** 0.5
            factor = min(1.0, case['most'] / (norm + EPSILON))
            return {'norm': torch.tensor(norm, dtype=torch.double), **{name: x.double() * factor for name, x in state['buffers'].items()}}
        if case['call'].startswith('norm'):
            return _exact_norm(case, state)
        if case['call'].startswith('block'):
            return _exact_block(case, state)
        return _exact_attention(case, state)


def _exact_gate(x, name):
    """The gate's factor and its derivative."""
    s = 1 / (1 + (-x).exp())
    if name == 'silu':
        return x * s, s * (1 + x * (1 - s))
    return (s, s * (1 - s)) if name == 'sigmoid' else (x, torch.ones_like(x))


def _exact_norm(case, state):
    x, weight = state['x'].double(), state['weight'].double()
    inverse = 1 / ((x * x).sum(-1, keepdim=True) / case['size'] + EPSILON).sqrt()
    unit = x * inverse
    factor, slope = _exact_gate(state['gate'].double(), case['gate']) if case['gate'] else (torch.ones_like(x), None)
    y = unit * weight * factor
    if case['call'] == 'norm':
        return y
    dy = state['dy'].double()
    found = {'y': y, 'grad_weight': (dy * unit * factor).sum((0, 1))}
    if case['gate']:
        found['grad_gate'] = dy * unit * weight * slope
    d_unit = dy * weight * factor
    found['grad_x'] = inverse * (d_unit - unit * (d_unit * unit).sum(-1, keepdim=True) / case['size'])
    return found


def _exact_block(case, state):
    size = case['size']
    x, block, before = (state[n].double() for n in ('x', 'block', 'before'))
    scale = state['scale'].double() if case['scaled'] else torch.ones_like(before)
    after = state['after'].double() if case['after'] else torch.ones_like(before)
    factor, slope = _exact_gate(state['gate'].double(), case['gate']) if case['gate'] else (torch.ones_like(x), None)
    if case['after']:
        inner = 1 / ((block * block).sum(-1, keepdim=True) / size + EPSILON).sqrt()
    else:
        inner = torch.ones_like(block[:, :1])
    unit = block * inner
    stream = x + scale * factor * after * unit
    outer = 1 / ((stream * stream).sum(-1, keepdim=True) / size + EPSILON).sqrt()
    even = stream * outer
    found = {'stream': stream, 'normed': even * before}
    if case['call'] == 'block':
        return found
    d_normed = state['d_normed'].double()
    found['grad_before'] = (d_normed * even).sum(0)
    d_even = d_normed * before
    d_stream = state['d_stream'].double() + outer * (d_even - even * (d_even * even).sum(-1, keepdim=True) / size)
    found['grad_x'] = d_stream
    if case['scaled']:
        found['grad_scale'] = (d_stream * factor * after * unit).sum(0)
    if case['gate']:
        found['grad_gate'] = d_stream * scale * after * unit * slope
    if case['after']:
        found['grad_after'] = (d_stream * scale * factor * unit).sum(0)
    d_unit = d_stream * scale * factor * after
    if case['after']:
        d_unit = inner * (d_unit - unit * (d_unit * unit).sum(-1, keepdim=True) / size)
    found['grad_block'] = d_unit
    return found


def _exact_attention(case, state):
    if case['call'] == 'act':
        for name in ('query', 'key', 'value', 'resets') + (() if case['fixed'] else ('decay',)):
            state[name] = state[name].unsqueeze(1) if state[name] is not None else None
    decay = state['decay'].expand(case['batch'], case['time'], case['heads'])
    # Pieces of the batch whose memories of every step fit in some GB.
    kept = case['heads'] * case['key_size'] * case['value_size'] * (case['time'] if case['call'] == 'learn' else 8)
    piece = max(1, 1_000_000_000 // kept)
    tensors = {**{name: x for name, x in state.items() if name != 'case' and x is not None}, 'decay': decay}
    pieces = [_exact_piece(case, {name: x[at:at + piece] for name, x in tensors.items()})
              for at in range(0, case['batch'], piece)]
    found = {name: torch.cat([part[name] for part in pieces]) for name in pieces[0]}
    if case['fixed'] and case['call'] == 'learn':
        found['grad_decay'] = found['grad_decay'].sum((0, 1))
    return found


def _exact_piece(case, given):
    """Step by step from the definition, and its gradients backwards through the steps."""
    group = case['heads'] // case['key_heads']
    query, key = (given[name].double().repeat_interleave(group, 2) for name in ('query', 'key'))
    value = given['value'].double()
    kept = given['decay'].double().exp()
    if 'resets' in given:
        kept = torch.where(given['resets'][..., None], 0.0, kept)
    count, time, heads, _ = value.shape
    scale = case['key_size'] ** -0.5
    if 'state' in given:
        memory = given['state'].double()
    else:
        memory = value.new_zeros(count, heads, case['key_size'], case['value_size'])
    learn = case['call'] == 'learn'
    outputs, before = [], []
    for t in range(time):
        memory = memory * kept[:, t, :, None, None]
        if learn:
            before.append(memory)
        memory = memory + key[:, t, :, :, None] * value[:, t, :, None, :]
        outputs.append(scale * (memory * query[:, t, :, :, None]).sum(-2))
    output = torch.stack(outputs, 1)
    if case['call'] == 'act':
        return {'output': output[:, 0], 'state': memory}
    found = {'output': output, 'last': memory}
    if not learn:
        return found
    d_output, d_memory = given['d_output'].double(), given['d_state'].double()
    d_query, d_key, d_value = torch.empty_like(query), torch.empty_like(key), torch.empty_like(value)
    d_decay = torch.empty_like(kept)
    for t in reversed(range(time)):
        k, d_out = key[:, t, :, :, None], d_output[:, t, :, None, :]
        after = before[t] + k * value[:, t, :, None, :]
        d_query[:, t] = scale * (after * d_out).sum(-1)
        d_memory = d_memory + scale * query[:, t, :, :, None] * d_out
        d_value[:, t] = (d_memory * k).sum(-2)
        d_key[:, t] = (d_memory * value[:, t, :, None, :]).sum(-1)
        d_decay[:, t] = (d_memory * before[t]).sum((-2, -1))
        d_memory = d_memory * kept[:, t, :, None, None]

    def shared(x):
        return x.view(count, time, case['key_heads'], group, -1).sum(3)

    found.update(grad_query=shared(d_query), grad_key=shared(d_key), grad_value=d_value, grad_decay=d_decay)
    if 'state' in given:
        found['grad_state'] = d_memory
    return found
