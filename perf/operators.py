"""What the policy operators of `cuju_amd.layers` are measured on.

A case is one operator and one kind of call:

* "act": one step of the gated delta rule for every agent of a batch, the state updated in place;
* "replay": the rule over a stretch of steps, forward;
* "learn": the same with every gradient;
* "norm": group norm with an activation over channels-last maps, forward;
* "norm learn": the same with every gradient.

The plain form (`own` false) is elementary torch operations in 32 bits.
"""

import torch

own = False

TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
BYTES = {'float32': 4, 'bfloat16': 2, 'float16': 2}
EPSILON = 1e-5


def _rule(**given):
    case = dict(call='act', batch=1, time=1, key_heads=4, heads=4, key_size=64, value_size=64, dtype='bfloat16',
                initial=True, episode=0)
    case.update(given)
    return case


def _norm(**given):
    case = dict(call='norm', batch=1, height=72, width=96, channels=16, groups=4, dtype='bfloat16',
                activation='silu')
    case.update(given)
    return case


def listed():
    return [
        # Acting in one match with all eleven players of a side: latency alone.
        _rule(name='act 11v11 x1', batch=11, episode=3000),
        # Acting in the 5-a-side workload, 64 matches of 4 agents, with odd heads in 32 bits.
        _rule(name='act 5v5 x64', batch=256, key_heads=2, heads=6, key_size=40, value_size=72, dtype='float32',
              episode=3000),
        # Acting in the headline workload: 16,384 matches of 11 agents.
        _rule(name='act 11v11 x16384', batch=180224, key_heads=2, heads=2, episode=3000),
        # Reading a whole match of 3,000 steps again, for its values, with wide heads.
        _rule(name='replay match x1', call='replay', batch=11, time=3000, key_heads=2, heads=4, key_size=128,
              value_size=128, initial=False),
        # The steps before a training segment, that bring the memory up to date: 400-step drills.
        _rule(name='replay drills x2048', call='replay', batch=2048, time=40, value_size=128, dtype='float16',
              episode=400),
        # One update of a small training batch: 64 matches of 4 agents, 128 steps.
        _rule(name='learn 5v5 x64', call='learn', batch=256, time=128, episode=3000),
        # One update on the 4,096-match workload with one agent, 64 steps.
        _rule(name='learn 11v11 x4096', call='learn', batch=4096, time=64, episode=3000),
        # A ragged one in 32 bits, heads that share keys, episodes that end often.
        _rule(name='learn ragged', call='learn', batch=37, time=77, key_heads=2, heads=6, key_size=48, value_size=80,
              dtype='float32', episode=20),
        # The encoder of one drill's three agents at full resolution: latency alone.
        _norm(name='norm drill x1', batch=3, activation='relu'),
        # The encoder of 200 drills of three agents at full resolution.
        _norm(name='norm drills x200', batch=600, channels=32, groups=8),
        # The same matches after a halving convolution, in training.
        _norm(name='norm learn x200', call='norm learn', batch=600, height=36, width=48, channels=64, groups=16),
        # A small odd map in 32 bits, in training.
        _norm(name='norm learn ragged', call='norm learn', batch=77, height=9, width=13, channels=40, groups=5,
              dtype='float32'),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm from `low` to `high`."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    call = rng.choice(('act', 'replay', 'learn', 'learn', 'norm', 'norm learn'))
    dtype = rng.choice(('bfloat16', 'bfloat16', 'float16', 'float32'))
    if call.startswith('norm'):
        height, width = _spread(rng, 3, 72), _spread(rng, 3, 96)
        groups = rng.choice((1, 2, 4, 8, 16, 5))
        channels = groups * rng.choice((1, 2, 4, 8, 6, 3))
        most = max(1, 60_000_000 // (height * width * channels))
        # The derivative of relu jumps at 0, where rounding alone decides: gradients go by the smooth ones.
        activation = rng.choice(('silu', 'none') if call == 'norm learn' else ('silu', 'relu', 'none'))
        return _norm(call=call, batch=_spread(rng, 1, min(most, 4096)), height=height, width=width,
                     channels=channels, groups=groups, dtype=dtype, activation=activation)
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
    return _rule(call=call, batch=_spread(rng, 1, min(most, 32768)), time=time, key_heads=key_heads, heads=heads,
                 key_size=key_size, value_size=value_size, dtype=dtype, initial=call == 'act' or rng.random() < 0.7,
                 episode=rng.choice((0, 20, 400, 3000)))


def prepare(case, seed):
    generator = torch.Generator(device='cuda')
    generator.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device='cuda')

    kind = TYPES[case['dtype']]
    batch = case['batch']
    state = {'case': case}
    if case['call'].startswith('norm'):
        shape = (batch, case['height'], case['width'], case['channels'])
        # A convolution's outputs: every channel has its own level and spread.
        state['x'] = (normal(*shape).mul_(0.5 + normal(case['channels']).abs_())
                      .add_(normal(case['channels']))).to(kind)
        state['weight'] = 1 + 0.2 * normal(case['channels'])
        state['bias'] = 0.2 * normal(case['channels'])
        if case['call'] == 'norm learn':
            state['dy'] = normal(*shape).mul_(0.01).to(kind)
        return state

    time, key_heads, heads = case['time'], case['key_heads'], case['heads']
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
    state['decay'] = -reach * torch.nn.functional.softplus(normal(batch, time, heads))
    state['beta'] = torch.sigmoid(normal(batch, time, heads))
    state['resets'] = None
    if case['episode']:
        state['resets'] = torch.rand(batch, time, generator=generator, device='cuda') < 1 / case['episode']
    state['state'] = 0.3 * normal(batch, heads, key_size, value_size) if case['initial'] else None
    if case['call'] == 'act':
        for name in ('query', 'key', 'value', 'decay', 'beta', 'resets'):
            state[name] = state[name].squeeze(1) if state[name] is not None else None
    if case['call'] == 'learn':
        state['d_output'] = normal(batch, time, heads, value_size).mul_(0.01).to(kind)
        state['d_state'] = 0.01 * normal(batch, heads, key_size, value_size)
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from cuju_amd import layers
    case = state['case']
    if case['call'] == 'act':
        output = layers.delta_rule_step(state['query'], state['key'], state['value'], state['decay'], state['beta'],
                                        state['state'], resets=state['resets'])
        return {'output': output, 'state': state['state']}
    if case['call'] == 'replay':
        output, last = layers.delta_rule(state['query'], state['key'], state['value'], state['decay'], state['beta'],
                                         state=state['state'], resets=state['resets'])
        return {'output': output, 'state': last}
    if case['call'] == 'learn':
        return _learn(state, lambda q, k, v, decay, beta, first: layers.delta_rule(
            q, k, v, decay, beta, state=first, resets=state['resets']))
    if case['call'] == 'norm':
        return layers.group_norm(state['x'], case['groups'], state['weight'], state['bias'], epsilon=EPSILON,
                                 activation=case['activation'])
    return _norm_learn(state, lambda x, weight, bias: layers.group_norm(
        x, case['groups'], weight, bias, epsilon=EPSILON, activation=case['activation']))


def _plain(state):
    case = state['case']
    if case['call'] == 'act':
        return _plain_step(state)
    if case['call'] == 'replay':
        return dict(zip(('output', 'state'), _plain_rule(state['query'], state['key'], state['value'], state['decay'],
                                                         state['beta'], state['state'], state['resets'])))
    if case['call'] == 'learn':
        return _learn(state, lambda q, k, v, decay, beta, first: _plain_rule(q, k, v, decay, beta, first,
                                                                             state['resets']))
    if case['call'] == 'norm':
        return _plain_norm(state['x'], state['weight'], state['bias'], case)
    return _norm_learn(state, lambda x, weight, bias: _plain_norm(x, weight, bias, case))


def _learn(state, rule):
    """One training pass of `rule`: its outputs and the gradients of every input."""
    names = ['query', 'key', 'value', 'decay', 'beta'] + (['state'] if state['state'] is not None else [])
    inputs = [state[name].detach().requires_grad_() for name in names]
    first = inputs[5] if len(inputs) > 5 else None
    output, last = rule(*inputs[:5], first)
    gradients = torch.autograd.grad([output, last], inputs, [state['d_output'], state['d_state']])
    return {'output': output.detach(), 'last': last.detach(),
            **{'d_' + name: gradient for name, gradient in zip(names, gradients)}}


def _norm_learn(state, norm):
    inputs = [state[name].detach().requires_grad_() for name in ('x', 'weight', 'bias')]
    y = norm(*inputs)
    dx, d_weight, d_bias = torch.autograd.grad(y, inputs, state['dy'])
    return {'y': y.detach(), 'dx': dx, 'd_weight': d_weight, 'd_bias': d_bias}


def _plain_step(state):
    query, key, value = state['query'].float(), state['key'].float(), state['value'].float()
    memory = state['state']
    group = memory.shape[1] // key.shape[1]
    query, key = query.repeat_interleave(group, 1), key.repeat_interleave(group, 1)
    kept = state['decay'].exp()
    if state['resets'] is not None:
        kept = kept * ~state['resets'][:, None]
    memory.mul_(kept[..., None, None])
    seen = torch.matmul(key[..., None, :], memory).squeeze(-2)
    memory.add_(key[..., :, None] * (state['beta'][..., None] * (value - seen))[..., None, :])
    output = torch.matmul(query[..., None, :], memory).squeeze(-2) * query.shape[-1] ** -0.5
    return {'output': output.to(state['value'].dtype), 'state': memory}


def _unit_lower_inverse(a):
    """The inverse of I + a for a strictly lower `a`, from blocks of one row to the whole."""
    count = a.shape[-1]
    inverse = torch.eye(count, device=a.device).expand(a.shape).contiguous()
    size = 1
    while size < count:
        at = torch.arange(0, count, 2 * size, device=a.device)[:, None] + torch.arange(size, device=a.device)
        low, high = at[:, :, None] + size, at[:, None, :]
        first = inverse[..., at[:, :, None], high]
        second = inverse[..., low, high + size]
        inverse[..., low, high] = -second @ (a[..., low, high] @ first)
        size *= 2
    return inverse


def _plain_rule(query, key, value, decay, beta, memory, resets):
    batch, time, heads, value_size = value.shape
    key_size, kind = key.shape[-1], value.dtype
    chunk = 64
    while chunk > 1 and chunk // 2 >= time:
        chunk //= 2
    count = -(-time // chunk)

    def split(x):
        """[batch, time, heads, ...] as [batch, heads, chunk, step, ...] in 32 bits, filled with zeros."""
        x = x.float().repeat_interleave(heads // x.shape[2], 2)
        short = count * chunk - time
        x = torch.cat([x, x.new_zeros(batch, short, *x.shape[2:])], 1) if short else x
        return x.reshape(batch, count, chunk, *x.shape[2:]).movedim(3, 1)

    query, key, value, decay, beta = (split(x) for x in (query, key, value, decay, beta))
    ends = split(resets[..., None].expand(-1, -1, heads)) if resets is not None else torch.zeros_like(decay)
    reach, part = decay.cumsum(-1), ends.cumsum(-1)
    lower = torch.ones(chunk, chunk, dtype=torch.bool, device=value.device).tril()
    same = (part[..., :, None] == part[..., None, :]) & lower
    between = (reach[..., :, None] - reach[..., None, :]).masked_fill(~same, -torch.inf).exp()
    whole = reach.masked_fill(part != 0, -torch.inf).exp()
    after = between[..., -1, :]

    a = (beta[..., None] * (key @ key.transpose(-1, -2)) * between).tril(-1)
    with torch.no_grad():
        inverse = _unit_lower_inverse(a)
    # One step of Newton's iteration: the value stays, and it has the inverse's derivative.
    inverse = 2 * inverse - inverse @ (inverse + a @ inverse)
    told = inverse @ (beta[..., None] * value)
    asked = inverse @ ((beta * whole)[..., None] * key)
    scale = key_size ** -0.5
    mixed = scale * (query @ key.transpose(-1, -2)) * between
    query = (scale * whole)[..., None] * query
    key = (after[..., None] * key).transpose(-1, -2)

    if memory is None:
        memory = value.new_zeros(batch, heads, key_size, value_size)
    outputs = []
    for n in range(count):
        new = told[:, :, n] - asked[:, :, n] @ memory
        outputs.append(query[:, :, n] @ memory + mixed[:, :, n] @ new)
        memory = whole[:, :, n, -1, None, None] * memory + key[:, :, n] @ new
    output = torch.stack(outputs, 2).reshape(batch, heads, count * chunk, value_size)[:, :, :time]
    return output.transpose(1, 2).to(kind), memory


def _plain_norm(x, weight, bias, case):
    kind = x.dtype
    batch, channels, groups = x.shape[0], x.shape[-1], case['groups']
    x = x.float().reshape(batch, -1, groups, channels // groups)
    mean = x.mean((1, 3), keepdim=True)
    centred = x - mean
    scaled = centred * ((centred * centred).mean((1, 3), keepdim=True) + EPSILON).rsqrt()
    z = scaled.reshape(batch, case['height'], case['width'], channels) * weight + bias
    if case['activation'] == 'silu':
        z = z * z.sigmoid()
    elif case['activation'] == 'relu':
        z = z.clamp_min(0)
    return z.to(kind)


def work(case):
    batch, size = case['batch'], BYTES[case['dtype']]
    if case['call'].startswith('norm'):
        values = batch * case['height'] * case['width'] * case['channels']
        # Forward: the map in and out, its sums and its values. Backward: two maps more (dy, dx).
        learn = case['call'] == 'norm learn'
        return {'bytes': values * size * (4 if learn else 2) + 4 * case['channels'] * (4 if learn else 2),
                'flops': values * (30 if learn else 10)}
    tokens = batch * case['time']
    keys = tokens * case['key_heads'] * case['key_size'] * size
    values = tokens * case['heads'] * case['value_size'] * size
    gates = tokens * case['heads'] * 4
    states = batch * case['heads'] * case['key_size'] * case['value_size']
    total = 2 * keys + 2 * values + 2 * gates + (tokens if case['episode'] else 0)
    total += 4 * states * (2 if case['initial'] else 1)
    # A step reads the memory twice and writes a product to it: 6 operations a value of it, and its decay.
    flops = 7 * tokens * case['heads'] * case['key_size'] * case['value_size']
    if case['call'] == 'learn':
        total += 2 * keys + 2 * values + 2 * gates + 4 * states * (2 if case['initial'] else 1)
        flops *= 3
    return {'bytes': total, 'flops': flops}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case['call'].startswith('norm'):
            return _exact_norm(case, state)
        return _exact_rule(case, state)


def _exact_norm(case, state):
    count, groups = case['batch'], case['groups']
    x = state['x'].double().view(count, -1, groups, case['channels'] // groups)
    weight, bias = (state[name].double().view(groups, -1) for name in ('weight', 'bias'))
    variance, mean = torch.var_mean(x, (1, 3), unbiased=False, keepdim=True)
    inverse = 1 / (variance + EPSILON).sqrt()
    x = (x - mean).mul_(inverse)
    z = x * weight + bias
    if case['activation'] == 'silu':
        gate = 1 / (1 + (-z).exp())
        slope = gate * (1 + z * (1 - gate))
        y = z * gate
    elif case['activation'] == 'relu':
        slope = (z > 0).double()
        y = z * slope
    else:
        slope = torch.ones_like(z)
        y = z
    y = y.view(state['x'].shape)
    if case['call'] == 'norm':
        return y
    dz = state['dy'].double().view(z.shape) * slope
    d_bias, d_weight = dz.sum((0, 1)), (dz * x).sum((0, 1))
    dz = dz * weight
    dx = inverse * (dz - dz.mean((1, 3), keepdim=True) - x * (dz * x).mean((1, 3), keepdim=True))
    return {'y': y, 'dx': dx.view(y.shape), 'd_weight': d_weight.flatten(), 'd_bias': d_bias.flatten()}


def _exact_rule(case, state):
    if case['call'] == 'act':
        for name in ('query', 'key', 'value', 'decay', 'beta', 'resets'):
            state[name] = state[name].unsqueeze(1) if state[name] is not None else None
    # Pieces of the batch whose memories of every step fit in some GB.
    kept = case['heads'] * case['key_size'] * case['value_size'] * (case['time'] if case['call'] == 'learn' else 8)
    piece = max(1, 1_000_000_000 // kept)
    tensors = {name: x for name, x in state.items() if name != 'case' and x is not None}
    pieces = [_exact_piece(case, {name: x[at:at + piece] for name, x in tensors.items()})
              for at in range(0, case['batch'], piece)]
    return {name: torch.cat([part[name] for part in pieces]) for name in pieces[0]}


def _exact_piece(case, given):
    """The rule step by step from its definition, and its gradients backwards through the steps."""
    group = case['heads'] // case['key_heads']
    query, key = (given[name].double().repeat_interleave(group, 2) for name in ('query', 'key'))
    value, beta = given['value'].double(), given['beta'].double()
    kept = given['decay'].double().exp()
    if 'resets' in given:
        kept = torch.where(given['resets'][..., None], 0.0, kept)
    count, time, heads, value_size = value.shape
    scale = case['key_size'] ** -0.5
    if 'state' in given:
        memory = given['state'].double()
    else:
        memory = value.new_zeros(count, heads, case['key_size'], value_size)
    learn = case['call'] == 'learn'
    outputs, before, errors = [], [], []
    for t in range(time):
        memory = memory * kept[:, t, :, None, None]
        error = value[:, t] - (memory * key[:, t, :, :, None]).sum(-2)
        if learn:
            before.append(memory)
            errors.append(error)
        memory = memory + key[:, t, :, :, None] * (beta[:, t, :, None] * error)[:, :, None, :]
        outputs.append(scale * (memory * query[:, t, :, :, None]).sum(-2))
    output = torch.stack(outputs, 1)
    if case['call'] == 'act':
        return {'output': output[:, 0], 'state': memory}
    if not learn:
        return {'output': output, 'state': memory}
    last = memory
    d_output, d_memory = given['d_output'].double(), given['d_state'].double()
    d_query, d_key, d_value = torch.empty_like(query), torch.empty_like(key), torch.empty_like(value)
    d_decay, d_beta = torch.empty_like(beta), torch.empty_like(beta)
    for t in reversed(range(time)):
        q, k, d_out = query[:, t, :, :, None], key[:, t, :, :, None], d_output[:, t, :, None, :]
        written = (beta[:, t, :, None] * errors[t])[:, :, None, :]
        after = before[t] + k * written
        d_query[:, t] = scale * (after * d_out).sum(-1)
        d_memory = d_memory + scale * q * d_out
        d_written = (d_memory * k).sum(-2)
        d_error = beta[:, t, :, None] * d_written
        d_beta[:, t] = (d_written * errors[t]).sum(-1)
        d_value[:, t] = d_error
        d_key[:, t] = (d_memory * written).sum(-1) - (before[t] * d_error[:, :, None, :]).sum(-1)
        d_memory = d_memory - k * d_error[:, :, None, :]
        d_decay[:, t] = (d_memory * before[t]).sum((-2, -1))
        d_memory = d_memory * kept[:, t, :, None, None]

    def shared(x):
        return x.view(count, time, case['key_heads'], group, -1).sum(3)

    found = {'output': output, 'last': last, 'd_query': shared(d_query), 'd_key': shared(d_key), 'd_value': d_value,
             'd_decay': d_decay, 'd_beta': d_beta}
    if 'state' in given:
        found['d_state'] = d_memory
    return found
