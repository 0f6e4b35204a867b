"""The 8-bit cache in plain 64-bit arithmetic: rows to codes and scales, and attention over them."""
import math

import torch

FLOOR = 2.0 ** -120


def quantise(x):
    """[..., width] of any type -> (codes as float64, scales float32): the nearest whole number to x / scale, ties to even."""
    x = x.double()
    amax = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    scale = torch.where(fine, (amax / 127).clamp_min(FLOOR), torch.full_like(amax, math.nan)).float()
    codes = torch.round(x / scale.double()[..., None])
    return torch.where(fine[..., None], codes, torch.zeros_like(codes)), scale


def seen_keys(p, window, keep):
    """Positions that the query at p sees."""
    first = max(0, p - window + 1) if window > 0 else (p - p % -window if window < 0 else 0)
    kept = min(keep, first) if window else 0
    return list(range(kept)) + list(range(first, p + 1))


def attend(q, k, v, p, keys, scale, slope=0.0, rate=None, sink=None, cap=0.0, temp=None):
    """One query over the keys at the positions ``keys`` (k and v: float64 [tokens, width] by position).  Returns the result, the
    sum of weight * |v| per entry, and the largest sum of |q_i k_i| * scale: what roundings are measured by."""
    if not keys:
        z = torch.zeros(v.shape[1], dtype=torch.float64)
        return z, z, 0.0
    at = torch.tensor(keys)
    factor = scale * (1.0 if temp is None else 1.0 + temp[0] * math.log((p + 1) // temp[1] + 1))
    s = (k[at] @ q) * factor
    size = ((k[at].abs() @ q.abs()) * abs(factor)).max().item()
    if cap > 0:
        s = cap * torch.tanh(s / cap)
    if slope:
        back = (p - at).double()
        s = s - slope * (back if rate is None else torch.log1p(rate * back))
    top = s.max() if sink is None else torch.maximum(s.max(), torch.tensor(sink, dtype=torch.float64))
    e = torch.exp(s - top)
    norm = e.sum() + (0 if sink is None else math.exp(sink - top))
    w = e / norm
    return w @ v[at], w @ v[at].abs(), size


def tolerance(dtype, ref, weighted, size, width, n_keys):
    """A bound on the kernel's error.  A 32-bit score of ``width`` terms is off by at most (width + 8) 2^-23 times the sum of their
    magnitudes (sums on the tensor cores may be cut instead of rounded: a whole step each), which moves a weight by twice that; the sums over
    ``n_keys`` weights by (n_keys + 64) 2^-23 of sum w |v|.  With bfloat16 rows a weight is rounded once (2^-8) and the result once (2^-8 of itself)."""
    moved = 2 * (width + 8) * 2.0 ** -23 * size + (n_keys + 64) * 2.0 ** -23
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    return weighted * (moved + half) + ref.abs() * half + 1e-30


def gpt_attention(h, c_attn_w, c_attn_b, c_proj_w, c_proj_b, n_head):
    """``plain_gpt.attention`` with keys and values as an 8-bit cache holds them."""
    T, d = h.shape
    q, k, v = (x.reshape(T, n_head, d // n_head) for x in (h @ c_attn_w + c_attn_b).split(d, dim=1))
    k, v = (codes * scale.double()[..., None] for codes, scale in (quantise(k), quantise(v)))
    out = [attend(q[p, i], k[:, i], v[:, i], p, list(range(p + 1)), (d // n_head) ** -0.5)[0] for p in range(T) for i in range(n_head)]
    return torch.stack(out).reshape(T, d) @ c_proj_w + c_proj_b
