"""A recurrent policy that acts in and learns from a batch of matches, all on the device.

Each agent's super mini-map goes through two patch layers, normalised by `layers.group_norm`, and what
it shows is kept in a memory, `layers.delta_rule`. Acting plays the memory on by one step at a time
(`layers.delta_rule_step`, in place); an update plays the whole segment again with gradients, from the
memory at its start. The matches' `done` flags clear the memories in both. The update's gradients are clipped
by `layers.clip_gradients`.

The memory may be one that only adds and forgets, `layers.linear_attention`, whose answers are normed and
gated by head (`layers.rms_norm`), and what is seen may go through residual blocks, each of which ends in
`layers.residual_norm`:

    python examples/recurrent_policy.py --environments 256 --updates 20
    python examples/recurrent_policy.py --environments 256 --updates 20 --memory linear --blocks 2
"""

from __future__ import annotations

import argparse
import os
import sys
import time

import torch
from torch import nn
from torch.nn import functional

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import cuju_amd
from cuju_amd import layers

ACTIONS = 19


def patches(x: torch.Tensor, size: int) -> torch.Tensor:
    """Maps [n, height, width, channels] as maps of their `size` x `size` patches."""
    n, height, width, channels = x.shape
    x = x.reshape(n, height // size, size, width // size, size, channels).transpose(2, 3)
    return x.reshape(n, height // size, width // size, size * size * channels)


class Block(nn.Module):
    """Two products over what the stream holds, whose outcome is normed, scaled and added to the stream."""

    def __init__(self, width: int):
        super().__init__()
        self.up, self.down = nn.Linear(width, 2 * width), nn.Linear(2 * width, width)
        self.after, self.scale, self.next = (nn.Parameter(torch.full((width,), x)) for x in (1.0, 0.1, 1.0))

    def forward(self, stream: torch.Tensor, normed: torch.Tensor) -> tuple:
        """The stream after the block, and its norm for the next one."""
        outcome = self.down(functional.silu(self.up(normed)))
        return layers.residual_norm(stream, outcome, self.next, after=self.after, scale=self.scale)


class Policy(nn.Module):
    """Maps [.., 72, 96, channels] to logits and a value, with a memory of `heads` matrices an agent: of the delta rule,
    or 'linear'. What is seen goes through `blocks` residual blocks."""

    def __init__(self, channels: int = 4, heads: int = 4, size: int = 32, width: int = 64, memory: str = 'delta', blocks: int = 0):
        super().__init__()
        if memory not in ('delta', 'linear'):
            raise ValueError(f"expected the memory 'delta' or 'linear', found {memory!r}")
        self.heads, self.size, self.linear = heads, size, memory == 'linear'
        self.first = nn.Linear(8 * 8 * channels, width // 2, bias=False)
        self.second = nn.Linear(3 * 3 * width // 2, width, bias=False)
        self.scales = nn.ParameterList([torch.ones(width // 2), torch.ones(width)])
        self.shifts = nn.ParameterList([torch.zeros(width // 2), torch.zeros(width)])
        self.seen = nn.Linear(3 * 4 * width, 4 * width)
        # A query, a key, a value and two gates a head; decays start out spread over short and long memories.
        self.projection = nn.Linear(4 * width, heads * (3 * size + 2))
        self.rates = nn.Parameter(torch.linspace(-5, 0, heads))
        self.head = nn.Linear(4 * width + heads * size, ACTIONS + 1)
        if self.linear:
            # What lets a head's answer through, and its norm's weight.
            self.gate, self.answered = nn.Linear(4 * width, heads * size), nn.Parameter(torch.ones(size))
        self.blocks = nn.ModuleList([Block(4 * width) for _ in range(blocks)])
        if blocks:
            self.begun = nn.Parameter(torch.ones(4 * width))

    def encode(self, maps: torch.Tensor) -> torch.Tensor:
        """Features [n, features] of uint8 maps [n, 72, 96, channels]."""
        x = self.first(patches(maps, 8).to(self.first.weight.dtype) / 255)
        x = layers.group_norm(x, 8, self.scales[0], self.shifts[0], activation='silu')
        x = self.second(patches(x, 3))
        x = layers.group_norm(x, 8, self.scales[1], self.shifts[1], activation='silu')
        stream = functional.silu(self.seen(x.flatten(1)))
        if not self.blocks:
            return stream
        normed = layers.rms_norm(stream, self.begun)
        for block in self.blocks:
            stream, normed = block(stream, normed)
        return normed

    def inputs(self, features: torch.Tensor) -> tuple:
        """What the memory takes, of features [.., features]."""
        lead = features.shape[:-1]
        query, key, value, gates = self.projection(features).split(
            [self.heads * self.size] * 3 + [self.heads * 2], dim=-1)
        query, key, value = (x.reshape(*lead, self.heads, self.size) for x in (query, key, value))
        rate, beta = gates.float().reshape(*lead, 2, self.heads).unbind(-2)
        # Under autocast the norms come in 32 bits.
        query, key = (functional.normalize(x, dim=-1).to(value.dtype) for x in (query, key))
        return (query, key, value, -functional.softplus(rate + self.rates), torch.sigmoid(beta))

    def outputs(self, features: torch.Tensor, read: torch.Tensor) -> tuple:
        if self.linear:
            gate = self.gate(features).unflatten(-1, (self.heads, self.size))
            read = layers.rms_norm(read, self.answered, gate.to(read.dtype), activation='silu')
        out = self.head(torch.cat([features, read.flatten(-2)], dim=-1)).float()
        return out[..., :ACTIONS], out[..., ACTIONS]

    def memory(self, agents: int, device) -> torch.Tensor:
        return torch.zeros(agents, self.heads, self.size, self.size, device=device)

    @torch.no_grad()
    def act(self, maps: torch.Tensor, memory: torch.Tensor, resets: torch.Tensor) -> tuple:
        """Logits and values of one step of maps [agents, 72, 96, channels]; plays `memory` on in place."""
        features = self.encode(maps)
        query, key, value, decay, beta = self.inputs(features)
        if self.linear:
            read = layers.linear_attention_step(query, key, beta[..., None].to(value.dtype) * value, decay, memory, resets=resets)
        else:
            read = layers.delta_rule_step(query, key, value, decay, beta, memory, resets=resets)
        return self.outputs(features, read)

    def learn(self, maps: torch.Tensor, memory: torch.Tensor, resets: torch.Tensor) -> tuple:
        """The same of maps [steps, agents, 72, 96, channels] from the memory before them, with gradients."""
        features = self.encode(maps.flatten(0, 1)).unflatten(0, maps.shape[:2])
        # The memory takes [agents, steps, ..]: views, without a copy.
        query, key, value, decay, beta = (x.transpose(0, 1) for x in self.inputs(features))
        if self.linear:
            value = beta[..., None].to(value.dtype) * value
            read, _ = layers.linear_attention(query, key, value, decay, state=memory, resets=resets.t())
        else:
            read, _ = layers.delta_rule(query, key, value, decay, beta, state=memory, resets=resets.t())
        return self.outputs(features, read.transpose(0, 1))


class Learner:
    """Plays a batch and updates its policy, one segment of `steps` steps after another."""

    def __init__(self, scenario: str, environments: int, steps: int = 32, device: str = 'cuda:0', seed: int = 0,
                 dtype: torch.dtype = torch.bfloat16, rate: float = 3e-4, memory: str = 'delta', blocks: int = 0):
        self.batch = cuju_amd.BatchEnvironment(scenario, environment_count=environments, seed=seed, device=device,
                                               representation='extracted', rewards='scoring,checkpoints')
        torch.manual_seed(seed)
        self.policy = Policy(memory=memory, blocks=blocks).to(device)
        # The maps' large products run in `dtype`; the parameters and the memory stay in 32 bits.
        self.cast = torch.autocast('cuda', dtype=dtype, enabled=dtype != torch.float32)
        self.optimizer = torch.optim.Adam(self.policy.parameters(), lr=rate)
        self.steps, self.agents = steps, environments * self.batch.agents
        self.maps = self.batch.reset()
        self.memory = self.policy.memory(self.agents, device)
        self.resets = torch.ones(self.agents, dtype=torch.bool, device=device)

    def play(self) -> dict:
        """One segment of steps: what the update needs, each [steps, agents, ..], and the memory before it."""
        kept = {name: [] for name in ('maps', 'resets', 'actions', 'logits', 'values', 'rewards', 'done')}
        before = self.memory.clone()
        for _ in range(self.steps):
            maps = self.maps.flatten(0, 1).clone()
            with self.cast:
                logits, values = self.policy.act(maps, self.memory, self.resets)
            actions = torch.multinomial(logits.softmax(-1), 1)[:, 0]
            self.maps, reward, done, _ = self.batch.step(actions.view(-1, self.batch.agents).int())
            done = done.repeat_interleave(self.batch.agents)
            step = (maps, self.resets, actions, logits, values, reward.flatten().clone(), done)
            for name, x in zip(kept, step):
                kept[name].append(x)
            # The maps of an ended match are already the next episode's.
            self.resets = done
        return {'memory': before, **{name: torch.stack(x) for name, x in kept.items()}}

    def update(self, segment: dict, discount: float = 0.993, smoothing: float = 0.95) -> dict:
        """One step of an advantage actor-critic on a played segment."""
        with torch.no_grad(), self.cast:
            # The value after the segment, of a memory that acting keeps for itself.
            _, after = self.policy.act(self.maps.flatten(0, 1), self.memory.clone(), self.resets)
        values, going = segment['values'], (~segment['done']).float()
        advantages, carried = torch.empty_like(values), torch.zeros_like(after)
        for t in reversed(range(self.steps)):
            carried = (segment['rewards'][t] + going[t] * discount * (after + smoothing * carried)) - values[t]
            advantages[t], after = carried, values[t]
        with self.cast:
            logits, found = self.policy.learn(segment['maps'], segment['memory'], segment['resets'])
        chosen = logits.log_softmax(-1).gather(-1, segment['actions'][..., None])[..., 0]
        entropy = torch.distributions.Categorical(logits=logits).entropy().mean()
        scaled = (advantages - advantages.mean()) / (advantages.std() + 1e-6)
        loss = -(chosen * scaled).mean() + 0.5 * (found - advantages - values).square().mean() - 0.01 * entropy
        self.optimizer.zero_grad()
        loss.backward()
        norm = layers.clip_gradients([x.grad for x in self.policy.parameters()], 1.0)
        self.optimizer.step()
        return {'loss': loss.detach(), 'entropy': entropy.detach(), 'norm': norm}


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split('\n')[0])
    parser.add_argument('--scenario', default='academy_3_vs_1_with_keeper_l3_r0')
    parser.add_argument('--environments', type=int, default=256)
    parser.add_argument('--steps', type=int, default=32, help='steps of a segment')
    parser.add_argument('--updates', type=int, default=20)
    parser.add_argument('--memory', default='delta', choices=('delta', 'linear'))
    parser.add_argument('--blocks', type=int, default=0, help='residual blocks over what is seen')
    parser.add_argument('--device', default='cuda:0')
    arguments = parser.parse_args()
    learner = Learner(arguments.scenario, arguments.environments, arguments.steps, arguments.device, memory=arguments.memory,
                      blocks=arguments.blocks)
    for number in range(arguments.updates):
        begin = time.perf_counter()
        segment = learner.play()
        torch.cuda.synchronize()
        played = time.perf_counter()
        result = learner.update(segment)
        loss, entropy = float(result['loss']), float(result['entropy'])
        print(f'update {number}: reward {float(segment["rewards"].sum()) / learner.agents:.4f} an agent, '
              f'{int(segment["done"].sum()) // learner.batch.agents} episodes, loss {loss:.4f}, entropy {entropy:.3f}, '
              f'{learner.steps * arguments.environments / (played - begin):.0f} steps/s played, '
              f'{1e3 * (time.perf_counter() - played):.1f} ms to update', flush=True)


if __name__ == '__main__':
    main()
