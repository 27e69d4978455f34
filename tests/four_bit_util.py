"""The cache of 4 bits an element in 64 bits: blocks, pools, and attention over them, written from the definition and element by
element where the kernels work in words."""
from __future__ import annotations

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantised(x: torch.Tensor) -> torch.Tensor:
    """The values that blocks of 32 elements along the last axis are kept as (float64)."""
    blocks = x.double().reshape(*x.shape[:-1], -1, 32)
    top = blocks.abs().amax(dim=-1, keepdim=True)
    unit = torch.full_like(top, 2.0 ** -126)
    for power in range(-125, 128):
        unit = torch.where(top > 7.0 * unit, torch.full_like(unit, 2.0 ** power), unit)
    levels = LEVELS.to(x.device)
    off = (blocks.abs()[..., None] / unit[..., None] - levels).abs()
    nearest = off.amin(dim=-1, keepdim=True)
    even = torch.arange(8, device=x.device) % 2
    chosen = torch.where(off == nearest, even, 2).argmin(dim=-1)          # of two equally near levels the one with the even code
    out = torch.copysign(levels[chosen] * unit, blocks)
    return torch.where(torch.isfinite(blocks).all(dim=-1, keepdim=True), out, math.nan).reshape(x.shape)


def codes_of(values: torch.Tensor):
    """(codes, powers) of values that are already numbers of the format: any power that holds a block does."""
    blocks = values.double().reshape(*values.shape[:-1], -1, 32)
    top = blocks.abs().amax(dim=-1, keepdim=True)
    nan = torch.isnan(blocks).any(dim=-1, keepdim=True)
    power = torch.where(top > 0, torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2, -126.0)
    for _ in range(3):                                                     # the smallest that gives whole codes
        a = blocks.abs() / 2.0 ** power
        fits = ((a[..., None] - LEVELS.to(values.device)).abs().amin(dim=-1) == 0).all(dim=-1, keepdim=True)
        power = torch.where(fits | nan | (top == 0), power, power + 1)
    a = blocks.abs() / 2.0 ** power
    code = (a[..., None] - LEVELS.to(values.device)).abs().argmin(dim=-1) + 8 * torch.signbit(blocks)
    powers = torch.where(nan, 255.0, power + 127).squeeze(-1)
    return torch.where(nan, 0, code).reshape(values.shape).to(torch.uint8), powers.to(torch.uint8)


def pools_of(k: torch.Tensor, v: torch.Tensor):
    """The four tensors of a cache whose pages hold ``k`` and ``v`` ``[pages, heads, tokens, dim]`` (numbers of the format)."""
    pages, heads, tokens, dim = k.shape
    pack = lambda codes: (codes[..., 0::2] | (codes[..., 1::2] << 4))     # noqa: E731
    kc, kp = codes_of(k)
    vc, vp = codes_of(v)
    return (pack(kc).reshape(pages, heads, tokens, dim // 32, 16).permute(0, 1, 3, 2, 4).contiguous(), kp.contiguous(),
            pack(vc).reshape(pages, heads, tokens // 4, 4, dim // 8, 4).permute(0, 1, 2, 4, 3, 5).contiguous(),
            vp.reshape(pages, heads, tokens // 4, 4, dim // 32).permute(0, 1, 2, 4, 3).contiguous())


def held(pools, page: int, head: int, token: int):
    """(key, value) float64 that a cache holds at one place, read element by element."""
    kc, kp, vc, vp = pools
    dim = kc.shape[2] * 32
    e = torch.arange(dim, device=kc.device)
    number = lambda code, power: torch.where(power == 255, math.nan, LEVELS.to(kc.device)[(code & 7).long()] * torch.where((code & 8) > 0, -1.0, 1.0)  # noqa: E731
                                             * 2.0 ** (power.double() - 127))
    k = number((kc[page, head, e // 32, token, e % 32 // 2] >> (4 * (e % 2))) & 15, kp[page, head, token, e // 32])
    v = number((vc[page, head, token // 4, e // 8, token % 4, e % 8 // 2] >> (4 * (e % 2))) & 15, vp[page, head, token // 4, e // 32, token % 4])
    return k, v


def attended(q, k, v, position: int, scale: float, window: int = 0):
    """One row's attention in 64 bits: q [q_heads, dim], k and v [keys, kv_heads, dim] -> (out, sum p |v|, sqrt(sum p^2 v^2), sqrt(sum p^2),
    largest sum |q k| of a score), the last four for the tolerances."""
    heads, dim = q.shape
    group = heads // k.shape[1]
    first = max(0, position - window + 1) if window else 0
    if position < 0:
        return tuple(torch.zeros(heads, dim, dtype=torch.float64, device=q.device) for _ in range(5))
    q, k, v = q.double(), k[first:position + 1].double(), v[first:position + 1].double()
    k, v = (x.repeat_interleave(group, dim=1).transpose(0, 1) for x in (k, v))
    scores = (k @ q[:, :, None]).squeeze(-1) * scale
    p = torch.softmax(scores, dim=-1)
    size = (k.abs() @ q.abs()[:, :, None]).squeeze(-1).amax(dim=-1) * scale
    mix = lambda w, x: (w[:, None, :] @ x).squeeze(1)                      # noqa: E731
    return (mix(p, v), mix(p, v.abs()), mix(p * p, v * v).sqrt(), (p * p).sum(-1).sqrt()[:, None].expand(-1, dim), size[:, None].expand(-1, dim))
