"""Rotary positions on several axes (time, height, width): what ``native.rotary`` is given, and its plain form.

A head of ``dim`` channels has ``dim / 2`` pairs at most; each axis owns a run of them (``sections``).  Video models give
time a little more than height and width: 22 + 21 + 21 pairs of a 128-channel head."""
from __future__ import annotations

import torch


def rotary_frequencies(sections, *, theta: float = 10000.0, per_axis: bool = True, device=None) -> torch.Tensor:
    """float64 [sum(sections)] radians per position.  ``per_axis``: every axis has the frequencies ``theta ** (-i / n)``
    of its own ``n`` pairs (video models); otherwise one series over all pairs is dealt to the axes in order (image and
    text models that extend a text model's rotation)."""
    sections = tuple(int(s) for s in sections)
    if not sections or min(sections) < 0 or sum(sections) == 0:
        raise ValueError("sections must be the non-negative pairs of each axis.")
    counts = sections if per_axis else (sum(sections),)
    series = [theta ** (-torch.arange(n, dtype=torch.float64) / n) for n in counts if n]
    return torch.cat(series).to(device)


def even_sections(dim: int, axes: int = 3) -> tuple[int, ...]:
    """Pairs of each axis for a whole head of ``dim`` channels: equal shares, the remainder on the first axis."""
    share = dim // 2 // axes
    return (dim // 2 - share * (axes - 1),) + (share,) * (axes - 1)


def grid_positions(*extents: int, start=None, device=None) -> torch.Tensor:
    """int32 [tokens, axes] positions of a clip whose tokens lie in raster order (last axis fastest), ``start`` added."""
    if not extents or min(extents) < 0:
        raise ValueError("extents must be the non-negative lengths of each axis.")
    axes = [torch.arange(n, dtype=torch.int32, device=device) for n in extents]
    grid = torch.stack(torch.meshgrid(*axes, indexing="ij"), dim=-1).reshape(-1, len(extents))
    return grid if start is None else grid + torch.as_tensor(start, dtype=torch.int32, device=device)


def rotary_reference(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections,
                     layout: str = "interleaved", norm: str | None = None, weight=None, eps: float = 1e-6) -> torch.Tensor:
    """``native.rotary`` of one tensor [batch, tokens, heads, dim] in plain torch (fp32, angles in fp64)."""
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(int(n))], device=x.device)
    angles = positions.double()[..., axis] * inv_freq
    angles = angles if angles.ndim == 3 else angles[None]
    cos, sin = angles.cos().float()[:, :, None], angles.sin().float()[:, :, None]
    v = x.float()
    if norm is not None:
        axes = (-1,) if norm == "head" else (-2, -1)
        v = v * torch.rsqrt(v.square().mean(dim=axes, keepdim=True) + eps)
        if weight is not None:
            v = v * weight.float().reshape(x.shape[2:] if norm == "token" else x.shape[3:])
    pairs = inv_freq.numel()
    if layout == "interleaved":
        a, b = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = v[..., :pairs], v[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((turned, v[..., 2 * pairs:]), dim=-1).to(x.dtype)
