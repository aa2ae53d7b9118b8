"""Microscaled 4-bit numbers and AdamW's 8-bit moments on the CPU, in float64, element by element."""
import math

import numpy as np
import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
LOWEST = -120


def exponent(t):
    """floor(log2 |t|), far below every scale for zero."""
    _, e = np.frexp(np.abs(t.double().numpy()))
    return torch.from_numpy(np.where(t.numpy() != 0, e - 1, -5000).astype(np.int64))


def quantize(t):
    """codes (.., blocks, 32) as whole numbers 0..15 and scales (.., blocks) as bytes, of (.., c)."""
    t = t.detach().cpu()
    pad = -t.shape[-1] % 32
    x = torch.nn.functional.pad(t.double(), (0, pad)).reshape(*t.shape[:-1], -1, 32)
    odd = ~torch.isfinite(x).all(-1)
    x = torch.where(odd.unsqueeze(-1), torch.zeros_like(x), x)
    e = (exponent(x.abs().amax(-1)) - 2).clamp(min=LOWEST)
    y = x.abs() * torch.exp2(-e.double()).unsqueeze(-1)
    code = torch.zeros_like(y, dtype=torch.int64)
    for i, m in enumerate(MIDDLES):
        code += (y > m) if i % 2 == 0 else (y >= m)
    code |= (x < 0).long() << 3
    return code, torch.where(odd, torch.full_like(e, 255), e + 127)


def values(code, scale, c):
    """(.., c) in float64"""
    size = GRID[code & 7] * torch.where(code >= 8, -1.0, 1.0).double()
    power = torch.where(scale == 255, torch.full_like(scale, 0).double() * math.nan, torch.exp2(scale.double() - 127))
    return (size * power.unsqueeze(-1)).flatten(-2)[..., :c]


def rounded(t):
    """What (.., c) is as such numbers."""
    return values(*quantize(t), t.shape[-1])


def operand(x, a, k, d, bs_last):
    """(a, d, n, k) of a tensor with a*k*d features."""
    x = x.detach().cpu()
    x = x.reshape(a, k, d, -1).permute(0, 2, 3, 1) if bs_last else x.reshape(-1, a, k, d).permute(1, 3, 0, 2)
    return x.contiguous()


def tensor(t, shape, bs_last):
    a, d, n, k = t.shape
    return (t.permute(0, 3, 1, 2) if bs_last else t.permute(2, 0, 3, 1)).reshape(shape)


def unpacked(codes):
    """(.., 16 blocks) bytes as (.., blocks, 32) codes."""
    codes = codes.cpu().long()
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32))


def act(name, z):
    if name in (None, "none"):
        return z
    return z * torch.sigmoid(z) if name == "silu" else torch.nn.functional.gelu(z)


def product(x, w, bias, pattern, name, gated, bs_last):
    """y in float64 of operands x (a, d, n, c) and w (a, d, rows, c), as (a, d, n, b); differentiable."""
    a, b, c, d = pattern
    z = x @ w.transpose(2, 3)
    if bias is not None:
        z = z + bias.reshape(a, -1, d).permute(0, 2, 1).unsqueeze(2)
    if not gated:
        return act(name, z)
    return act(name, z[..., :b]) * z[..., b:]


# -- AdamW ---------------------------------------------------------------------------------------------


def _mix(x):
    x = ((x ^ x >> 16) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ x >> 15) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ x >> 16


def dither(n, seed, tensor, step):
    key = _mix((_mix((seed + tensor) & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    h = _mix(torch.arange(n, dtype=torch.int64) ^ key)
    return (h & 0xFFFF).double() / 65536, (h >> 16).double() / 65536


def decode_moments(m, v, scales):
    n = m.numel()
    s = torch.exp2(scales.cpu().double() - 127).repeat_interleave(32, 1)[:, :n]
    x = m.cpu().reshape(-1).view(torch.float8_e4m3fn).float().double()
    y = (v.cpu().reshape(-1).to(torch.int32) << 7).to(torch.int16).view(torch.float16).double()
    return x * s[0], y * s[1]


def _down_or_up(y, r, least):
    q = exponent(y).clamp(min=least) - 3
    step = torch.exp2(q.double())
    return torch.floor(y / step + r) * step


def encode_moments(m, v, r, s):
    n = m.numel()
    pad = -n % 32
    finite_m, finite_v = m.abs() < 2.0 ** 128, v < 2.0 ** 128
    x, y = (torch.nn.functional.pad(torch.where(f, t, torch.zeros_like(t)), (0, pad)).reshape(-1, 32) for t, f in ((m, finite_m), (v, finite_v)))
    em = (exponent(x.abs().amax(1)) - 7).clamp(min=LOWEST)
    ev = (exponent(y.amax(1)) - 14).clamp(min=LOWEST)
    x, y = x * torch.exp2(-em.double()).unsqueeze(1), y * torch.exp2(-ev.double()).unsqueeze(1)
    r, s = (torch.nn.functional.pad(t, (0, pad)).reshape(-1, 32) for t in (r, s))
    x = torch.copysign(_down_or_up(x.abs(), r, -6), x).flatten()[:n]
    y = torch.where(y > 0, _down_or_up(y, s, -14).clamp(min=2.0 ** -17), torch.zeros_like(y)).flatten()[:n]
    cm = x.float().to(torch.float8_e4m3fn).view(torch.uint8)
    cv = (y.to(torch.float16).view(torch.int16) >> 7).to(torch.uint8)
    cm = torch.where(finite_m, cm, torch.full_like(cm, 0x7f))
    cv = torch.where(finite_v, cv, torch.where(torch.isnan(v), 0xfc, 0xf8).to(torch.uint8))
    return cm, cv, torch.stack([em + 127, ev + 127]).to(torch.uint8)


def adamw(w, g, m, v, step, lr, betas, eps, decay, grad_scale):
    """(w, m, v) of one step in float64."""
    g = g.cpu().double().reshape(-1) * grad_scale
    m = m * betas[0] + g * (1 - betas[0])
    v = v * betas[1] + g * g * (1 - betas[1])
    hat = (v / (1 - betas[1] ** step)).sqrt()
    return w.cpu().double().reshape(-1) * (1 - lr * decay) - lr / (1 - betas[0] ** step) * m / (hat + eps), m, v
