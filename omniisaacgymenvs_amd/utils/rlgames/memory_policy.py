"""A policy with a memory on top of utils/rlgames/memory_ops.py: what a task such as ShadowHandOpenAI_LSTM (utils/task_util.py) is
driven with, its state kept per env on the device and cleared by the envs' own ``reset_buf``.

``MemoryPolicy.step`` takes one observation per env between two ``env.step`` calls; ``MemoryPolicy.forward`` takes whole rollouts, with
the same weights and the same results, and is differentiable.  The projections are torch's; norm and memory are the HIP kernels.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn

from .memory_ops import MAX_HEAD_DIM, MAX_WIDTH, decay_attention, decay_attention_step, layer_norm


class LayerNorm(nn.Module):
    """``layer_norm`` with a weight and a bias of its own."""

    def __init__(self, width: int, eps: float = 1e-5):
        super().__init__()
        self.weight, self.bias, self.eps = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width)), eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)


class MemoryBlock(nn.Module):
    """x + out(memory(norm(x))): linear attention over the env's own past, every head with a decay of its own."""

    def __init__(self, width: int, heads: int):
        super().__init__()
        if heads < 1 or width < 1 or width % heads:
            raise ValueError(f"MemoryBlock: width {width} is not a multiple of {heads} heads")
        if width > MAX_WIDTH or width // heads > MAX_HEAD_DIM:
            raise ValueError(f"MemoryBlock: width {width} over {heads} heads; heads are 1 to {MAX_HEAD_DIM} wide, all of them {MAX_WIDTH}")
        self.heads, self.head_dim = heads, width // heads
        self.norm = LayerNorm(width)
        self.qkv = nn.Linear(width, 3 * width, bias=False)
        self.out = nn.Linear(width, width, bias=False)
        # memories from 4 to 512 steps long
        self.register_buffer("decay", 1 - torch.exp2(-2 - 7 * torch.arange(heads, dtype=torch.float32) / max(heads - 1, 1)))

    def _apply(self, fn, recurse: bool = True):
        """``.half()``, ``.to(torch.bfloat16)``: the decays stay in 32 bits (0.998 would be 1 in bf16) and move with the weights."""
        decay = self.decay
        super()._apply(fn, recurse)
        if self.decay.dtype is not torch.float32:
            self.decay = decay.to(self.decay.device)
        return self

    def _heads(self, x: torch.Tensor):
        qkv = self.qkv(self.norm(x)).unflatten(-1, (3, self.heads, self.head_dim))
        return qkv.unbind(-3)

    def step(self, x: torch.Tensor, state: torch.Tensor, resets: Optional[torch.Tensor]) -> torch.Tensor:
        return x + self.out(decay_attention_step(*self._heads(x), self.decay, state, resets).flatten(-2))

    def forward(self, x, state, resets, lengths) -> Tuple[torch.Tensor, torch.Tensor]:
        o, state = decay_attention(*self._heads(x), self.decay, state, resets, lengths)
        return x + self.out(o.flatten(-2)), state


class MemoryPolicy(nn.Module):
    """Observations -> action means in (-1, 1) and values, through ``layers`` memory blocks.  Runs in fp32, cast to fp16 or bf16 (with
    observations of that type), or under autocast."""

    def __init__(self, num_observations: int, num_actions: int, width: int = 256, heads: int = 4, layers: int = 1):
        super().__init__()
        if layers < 1:
            raise ValueError(f"MemoryPolicy: {layers} layers")
        self.encoder = nn.Linear(num_observations, width)
        self.blocks = nn.ModuleList(MemoryBlock(width, heads) for _ in range(layers))
        self.norm = LayerNorm(width)
        self.mu, self.value = nn.Linear(width, num_actions), nn.Linear(width, 1)

    def initial_state(self, num_envs: int) -> torch.Tensor:
        """(layers, N, heads, head_dim, head_dim), empty memories; in 32 bits whatever the policy's type."""
        b = self.blocks[0]
        return torch.zeros(len(self.blocks), num_envs, b.heads, b.head_dim, b.head_dim, dtype=torch.float32, device=b.decay.device)

    def _read(self, x):
        x = self.norm(x)
        return torch.tanh(self.mu(x)), self.value(x).squeeze(-1)

    @torch.no_grad()
    def step(self, obs: torch.Tensor, state: torch.Tensor, resets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One step of every env: (N, num_observations) -> action means (N, num_actions), values (N,).  ``state`` is updated in place;
        envs that ``resets`` (the flags that came with ``obs``) marks start from an empty one."""
        x = self.encoder(obs)
        for i, block in enumerate(self.blocks):
            x = block.step(x, state[i], resets)
        return self._read(x)

    def forward(self, obs: torch.Tensor, state: Optional[torch.Tensor] = None, resets: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """A rollout: obs (N, T, num_observations) with its resets (N, T) -> action means (N, T, num_actions), values (N, T) and
        the state behind it; ``state`` is the one in front of it (None: empty) and is left alone.  Rows from ``lengths`` on read
        no memory."""
        x, states = self.encoder(obs), []
        for i, block in enumerate(self.blocks):
            x, s = block(x, None if state is None else state[i], resets, lengths)
            states.append(s)
        return (*self._read(x), torch.stack(states))
