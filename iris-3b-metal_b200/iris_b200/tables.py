"""Position tables computed once per resolution on the host, then kept on the device.

They must match the reference bit for bit (the token-position mapping is an
integer layout), so they are evaluated with the same fp32 torch arithmetic:

* ``rope_2d`` / ``rope_1d``: ``src/iris3b/nn/rope.py:19-89``; cos/sin split as
  ``RopeTable.from_complex`` does (``src/iris_metal/model.py:55-65``);
* ``sincos_pos_embed_2d``: ``src/iris3b/nn/embeddings.py:269-288`` (float64,
  stored as float32).

``rope_table`` (the text side's tables, with scaling for long contexts) is this
build's own and evaluated in float64.
"""

from __future__ import annotations

import math

import torch


def rope_2d(head_dim: int, height: int, width: int, theta: float, scale: float, aspect: str) -> torch.Tensor:
    """Complex64 ``[height*width, head_dim/2]``: frequency pairs interleaved (x, y),
    tokens row-major."""
    n_pairs = head_dim // 4
    freqs = 1.0 / theta ** (torch.arange(0, head_dim, 4)[:n_pairs].float() / head_dim)
    if aspect == "square":
        xs, ys = torch.linspace(0, scale, width), torch.linspace(0, scale, height)
    elif aspect == "isotropic":
        step = scale / max(max(height, width) - 1, 1)
        xs, ys = torch.arange(width).float() * step, torch.arange(height).float() * step
    else:
        raise ValueError(f"unknown rope aspect mode '{aspect}'")
    xc = torch.polar(torch.ones(width, n_pairs), torch.outer(xs, freqs))
    yc = torch.polar(torch.ones(height, n_pairs), torch.outer(ys, freqs))
    grid = torch.stack([xc[None, :, :].expand(height, width, -1), yc[:, None, :].expand(height, width, -1)], dim=-1)
    return grid.reshape(height * width, 2 * n_pairs)


def rope_1d(head_dim: int, length: int, theta: float) -> torch.Tensor:
    freqs = 1.0 / theta ** (torch.arange(0, head_dim, 2)[: head_dim // 2].float() / head_dim)
    angles = torch.outer(torch.arange(length).float(), freqs)
    return torch.polar(torch.ones_like(angles), angles)


def rope_table(
    rotary: int,
    length: int,
    theta: float = 10000.0,
    *,
    scaling: str | None = None,
    factor: float = 1.0,
    trained_length: int | None = None,
    fast_turns: float = 32.0,
    slow_turns: float = 1.0,
    device=None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """FP32 ``(cos, sin)`` ``[length, rotary / 2]`` of the angles ``p * theta^(-2i / rotary)``
    for :func:`iris_b200.kernels.rope`, evaluated in float64 (a far position's angle
    has lost its fraction in float32) and rounded once.

    ``scaling`` stretches a model trained on fewer positions by ``factor``: ``"linear"``
    divides every angle; ``"ntk"`` raises ``theta`` by ``factor^(rotary / (rotary - 2))``, so
    that the slowest pair is divided by ``factor`` and the fastest is kept; ``"ramp"``
    keeps pairs that turn at least ``fast_turns`` times over ``trained_length``
    positions, divides those that turn at most ``slow_turns`` times, blends linearly
    in the pair's index between (from the whole index at or before the one end, pair 0
    at the earliest, to the one at or behind the other), and multiplies both tables by
    ``0.1 ln(factor) + 1``."""
    if rotary < 2 or rotary % 2 or length < 1 or theta <= 1 or factor < 1:
        raise ValueError("rope_table needs an even rotary width, a positive length, theta > 1 and factor >= 1")
    if scaling not in (None, "linear", "ntk", "ramp"):
        raise ValueError(f"unknown rope scaling {scaling!r}")
    if scaling is None and factor != 1:
        raise ValueError("rope_table: a factor needs a scaling")
    magnitude = 1.0
    if scaling == "ntk":
        if rotary == 2:
            raise ValueError("rope_table: ntk scaling needs more than one pair")
        theta = theta * factor ** (rotary / (rotary - 2))
    freqs = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "ramp":
        if trained_length is None or trained_length < 1 or not fast_turns > slow_turns > 0:
            raise ValueError("rope_table: ramp scaling needs trained_length and fast_turns > slow_turns > 0")

        def pair(turns: float) -> float:  # the (fractional) pair that turns so often over trained_length
            return rotary * math.log(trained_length / (2 * math.pi * turns)) / (2 * math.log(theta))

        first = max(math.floor(pair(fast_turns)), 0)
        last = math.ceil(pair(slow_turns))  # may lie behind the last pair: then none is divided in full
        index = torch.arange(rotary // 2, dtype=torch.float64)
        divided = ((index - first) / max(last - first, 1)).clamp(0, 1)
        divided[trained_length * freqs <= 2 * math.pi * slow_turns] = 1  # every pair, where they start so slowly
        freqs = freqs / factor * divided + freqs * (1 - divided)
        magnitude = 0.1 * math.log(factor) + 1
    angles = torch.outer(torch.arange(length, dtype=torch.float64), freqs)
    return tuple((f * magnitude).float().contiguous().to(device) for f in (angles.cos(), angles.sin()))


def cos_sin(*tables: torch.Tensor, device) -> tuple[torch.Tensor, torch.Tensor]:
    """Concatenated complex tables -> contiguous FP32 (cos, sin) ``[N, head_dim/2]``."""
    cis = torch.view_as_real(torch.cat(tables))
    return cis[..., 0].contiguous().to(device), cis[..., 1].contiguous().to(device)


def sincos_pos_embed_2d(embed_dim: int, height: int, width: int) -> torch.Tensor:
    """``[H*W, dim]``: channels ``[sin | cos](x * w_i)`` then ``[sin | cos](y * w_i)``,
    ``w_i = 10000^(-i / (dim / 4))``, evaluated in float64."""
    quarter = embed_dim // 4
    omega = 1.0 / 10000.0 ** (torch.arange(quarter, dtype=torch.float64) / quarter)
    ys, xs = torch.meshgrid(torch.arange(height, dtype=torch.float64), torch.arange(width, dtype=torch.float64),
                            indexing="ij")  # fmt: skip
    ax = torch.outer(xs.reshape(-1), omega)
    ay = torch.outer(ys.reshape(-1), omega)
    return torch.cat([ax.sin(), ax.cos(), ay.sin(), ay.cos()], dim=1).float()
