"""Weights in 4 bits and their products from the definition, in 64 bits on the CPU."""
from __future__ import annotations

import torch

VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def pad(n):
    return -(-n // 128) * 128


def weights(E, N, K, seed=0, low=118, high=123):
    """(codes, scales) drawn evenly, zeros beyond K."""
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (E, N, pad(K)), generator=gen, dtype=torch.uint8)
    codes[..., K:] = 0
    scales = torch.randint(low, high, (E, N, pad(K) // 32), generator=gen, dtype=torch.uint8)
    return pack(codes), scales


def pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def values(data, scales, K):
    codes = torch.stack([data & 15, data >> 4], -1).flatten(-2).long()
    v = VALUES[codes & 7] * torch.where(codes >= 8, -1.0, 1.0).double()
    s = 2.0 ** (scales.double() - 127)
    s = torch.where(scales == 255, float("nan"), s)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)[..., :K]


def quantize(x):
    """(codes, scales): for each 32 the smallest power of two (from 2^-127) with which none passes 6; nearest,
    ties to the code whose last bit is 0."""
    K = x.shape[-1]
    p = torch.zeros(*x.shape[:-1], pad(K), dtype=torch.float64)
    p[..., :K] = x.double()
    b = p.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 6.0) / 6))
    # the logarithm's rounding cannot put a power of two on the wrong side unnoticed
    e = torch.where(top > 6 * 2.0 ** e, e + 1, e)
    e = torch.where(top <= 6 * 2.0 ** (e - 1), e - 1, e)
    e = torch.where(top > 0, e.clamp_min(-127), 0.0)
    bad = ~torch.isfinite(b).all(-1)
    v = (b / 2.0 ** e.unsqueeze(-1)).nan_to_num(0.0)
    dist = (v.abs().unsqueeze(-1) - VALUES).abs()
    near = dist.min(-1, keepdim=True).values
    even = torch.arange(8) % 2 == 0
    order = torch.where(dist == near, torch.where(even, 0, 1), 2)
    code = order.argmin(-1).to(torch.uint8) | torch.where(torch.signbit(v), 8, 0).to(torch.uint8)
    code = torch.where(bad.unsqueeze(-1), 0, code).to(torch.uint8)
    scale = torch.where(bad, 255.0, e + 127).to(torch.uint8)
    return pack(code.flatten(-2)), scale


def linear(x, w, offsets, rows=None, bias=None, gelu=False, R=None):
    """(out, sum of |x w|), [R, N]: zeros for rows of no expert."""
    E, N, K = w.shape
    R = (x.shape[0] if rows is None else len(rows)) if R is None else R
    out, size = torch.zeros(R, N, dtype=torch.float64), torch.zeros(R, N, dtype=torch.float64)
    for e in range(E):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if a >= b:
            continue
        at = torch.arange(a, b) if rows is None else rows[a:b].long()
        here = (at >= 0) & (at < x.shape[0])
        xe = x.double()[at.clamp(0, x.shape[0] - 1)] * here.unsqueeze(1)
        y = xe @ w[e].t()
        size[a:b] = xe.abs() @ w[e].abs().t()
        if bias is not None:
            y = y + bias[e].double()
            size[a:b] += bias[e].double().abs()
        out[a:b] = y * 0.5 * torch.erfc(-y / 2.0 ** 0.5) if gelu else y
    return out, size
