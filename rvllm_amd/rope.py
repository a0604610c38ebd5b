"""RoPE angle tables for rvkv_attn_prep.

rope_cos_sin follows src/model.rs:224-250: theta_j = rope_theta **
(-2 j / head_dim), divided by factors[j] when Llama-3 frequency factors are
given; angle[i, j] = positions[i] * theta_j; the tables are cos and sin of
the angles, f32 [n, head_dim / 2], computed on the host. The reference builds
it once per forward for that forward's positions; the engine backend builds it
once for all positions of the context and gathers a forward's rows on the GPU.
Every layer shares them.
"""
from __future__ import annotations

import numpy as np


def rope_cos_sin(rope_theta: float, head_dim: int, positions,
                 factors=None):
    half = head_dim // 2
    # Every step is an f32 operation of the reference; pow, cos and sin are
    # evaluated in f64 and rounded once, which gives the correctly rounded
    # f32 result.
    expo = (np.float32(-2.0) * np.arange(half, dtype=np.float32)
            / np.float32(head_dim))
    theta = np.power(np.float64(np.float32(rope_theta)),
                     expo.astype(np.float64)).astype(np.float32)
    if factors is not None:
        theta = theta / np.asarray(factors, np.float32)
    pos = np.asarray(positions).astype(np.float32).reshape(-1, 1)
    angle = (pos * theta.reshape(1, half)).astype(np.float64)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def rope_inv_freq(rope_theta: float, rot_dim: int, factors=None):
    """f32 [rot_dim / 2] frequencies for rope_append: rope_theta ** (-2 j /
    rot_dim), divided by factors[j] (a number, or one per frequency) where a
    model scales them for longer contexts."""
    inv = float(rope_theta) ** (-np.arange(0, rot_dim, 2, dtype=np.float64)
                                / rot_dim)
    if factors is not None:
        inv = inv / np.asarray(factors, np.float64)
    return inv.astype(np.float32)


def rope_yarn(rope_theta: float, rot_dim: int, factor: float,
              original_context: int, beta_fast: float = 32.0,
              beta_slow: float = 1.0):
    """(inv_freq, attn_factor) scaled as YaRN does (Peng et al., 2023): a
    frequency that turns more than beta_fast times over the original context
    stays, one that turns fewer than beta_slow times is divided by factor, and
    those between are mixed linearly in their index; the rotation is scaled by
    0.1 ln(factor) + 1."""
    inv = float(rope_theta) ** (-np.arange(0, rot_dim, 2, dtype=np.float64)
                                / rot_dim)

    def index_of(turns):
        # theta ** (-2 j / d) * context = 2 pi turns, solved for j
        return (rot_dim * np.log(original_context / (2 * np.pi * turns))
                / (2 * np.log(float(rope_theta))))

    low = max(np.floor(index_of(beta_fast)), 0)
    high = min(np.ceil(index_of(beta_slow)), rot_dim - 1)
    slow = np.clip((np.arange(rot_dim // 2) - low) / max(high - low, 1e-3),
                   0, 1)
    inv = inv * (1 - slow) + inv / factor * slow
    return inv.astype(np.float32), 0.1 * float(np.log(factor)) + 1.0
