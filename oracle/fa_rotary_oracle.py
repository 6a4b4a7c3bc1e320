"""Rotary tables and the rotation from their definitions, in 64 bits on the CPU."""
import math

import torch


def frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=0, low=1.0, high=32.0):
    out = []
    for i in range(rotary_dim // 2):
        b = base * factor ** (rotary_dim / (rotary_dim - 2)) if scaling == "ntk" else base
        f = b ** (-2.0 * i / rotary_dim)
        if scaling == "linear":
            f /= factor
        if scaling == "by_parts":
            g = min(max((original_length * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = f * (g + (1 - g) / factor)
        out.append(f)
    return out


def table(positions, rotary_dim, attention_factor=1.0, **how):
    """cos, sin (n, rotary_dim / 2) of a list of positions."""
    f = frequencies(rotary_dim, **how)
    # whole turns are taken out in integers where the product would lose bits
    cos = [[attention_factor * math.cos(math.remainder(p * w, 2 * math.pi)) for w in f] for p in positions]
    sin = [[attention_factor * math.sin(math.remainder(p * w, 2 * math.pi)) for w in f] for p in positions]
    return torch.tensor(cos, dtype=torch.float64), torch.tensor(sin, dtype=torch.float64)


def turn(x, cos, sin, interleaved):
    """x (..., H, D) in 64 bits by cos, sin (..., rd / 2) of its rows."""
    x = x.double().clone()
    rd = 2 * cos.shape[-1]
    for i in range(rd // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rd // 2)
        c, s = cos[..., i, None].double(), sin[..., i, None].double()
        u, v = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = u * c - v * s, v * c + u * s
    return x
