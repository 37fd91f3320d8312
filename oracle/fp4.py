"""Oracles of the rotated cache writes and of the 4-bit cache, in float64 on the CPU,
element by element from the definitions."""

from __future__ import annotations

import math

import torch

EXPONENTS = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}


def rotate(x, positions, cos_sin, halves):
    """x [tokens, heads, dim] with the leading dims of cos_sin's angles turned, in
    float64; rows whose position is outside cos_sin stay."""
    out = x.detach().double().cpu().clone()
    cos_sin = cos_sin.double().cpu()
    half = cos_sin.shape[1]
    for t, position in enumerate(positions.tolist()):
        if not 0 <= position < cos_sin.shape[0]:
            continue
        c, s = cos_sin[position, :, 0], cos_sin[position, :, 1]
        first = torch.arange(half) if halves else torch.arange(half) * 2
        second = first + half if halves else first + 1
        a, b = out[t][:, first].clone(), out[t][:, second].clone()
        out[t][:, first] = a * c - b * s
        out[t][:, second] = b * c + a * s
    return out


def nearest(x, dtype):
    """The values [..., dim] that a 4-bit cache holds of float32 values x [..., dim]
    written from `dtype`."""
    low, high = EXPONENTS[dtype]
    x = x.detach().double().cpu()
    out = torch.empty_like(x)
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    borders = [(a + b) / 2 for a, b in zip(grid, grid[1:])]
    for g in range(0, x.shape[-1], 32):
        part = x[..., g:g + 32]
        top = part.abs().amax(-1)
        exponent = torch.full(top.shape, float(low), dtype=torch.float64)
        for e in range(low, high):
            exponent = torch.where(top > 7 * 2.0 ** e, float(e + 1), exponent)
        y = part * torch.exp2(-exponent)[..., None]
        size = torch.zeros_like(y)
        for i, border in enumerate(borders):
            up = y.abs() >= border if i % 2 else y.abs() > border  # a tie: the even code
            size = torch.where(up, grid[i + 1], size)
        value = torch.where(y < 0, -size, size) * torch.exp2(exponent)[..., None]
        out[..., g:g + 32] = torch.where(torch.isfinite(top)[..., None], value, math.nan)
    return out


def decode(cache, head_dim):
    """(keys, values) [pages, page_size, kv_heads, head_dim] of a 4-bit cache's bytes."""
    cache = cache.cpu()
    pages, heads, size, _ = cache.shape
    groups = -(-head_dim // 32)
    flat = cache.reshape(pages, heads, -1)
    code = size * 16 * groups
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    grid = torch.cat((grid, -grid))
    out = []
    for which in range(2):
        codes = flat[:, :, which * code:(which + 1) * code].reshape(pages, heads, size, -1)
        at = 2 * code + which * 4 * size
        scales = flat[:, :, at:at + 4 * size].reshape(pages, heads, size, 4)[..., :groups]
        nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        scale = torch.exp2(scales.double() - 127)
        scale = torch.where(scales == 255, math.nan, scale)
        value = grid[nibbles.long()].unflatten(-1, (groups, 32)) * scale[..., None]
        out.append(value.flatten(-2)[..., :head_dim].transpose(1, 2))
    return tuple(out)
