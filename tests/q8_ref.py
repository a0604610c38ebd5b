"""Plain 64-bit forms of the 8-bit paged cache's operators (test
infrastructure), on the CPU, and the tolerances they are compared with."""
from __future__ import annotations

import math

import numpy as np
import torch


def i32(a, device="cuda"):
    arr = np.ascontiguousarray(np.asarray(a, np.uint32)).view(np.int32)
    return torch.from_numpy(arr.copy()).to(device)


def rotate(x, pos, inv_freq, interleaved, factor, norm=None, eps=1e-6):
    """x [rows, heads, hd] -> f64, normed and rotated, pair by pair."""
    x = x.double().cpu().clone()
    hd = x.shape[-1]
    if norm is not None:
        x = (x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + eps)
             * norm.double().cpu())
    if inv_freq is None:
        return x
    inv = inv_freq.double().cpu()
    n = inv.numel()
    ang = torch.as_tensor(np.asarray(pos, np.float64))[:, None] * inv
    c = (torch.cos(ang) * factor)[:, None]
    s = (torch.sin(ang) * factor)[:, None]
    p = torch.arange(n)
    i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + n)
    a, b = x[..., i].clone(), x[..., j].clone()
    x[..., i], x[..., j] = a * c - b * s, a * s + b * c
    return x


def quantise(x):
    """x [..., hd] f64 -> (codes int8, scale f32 [...]); a row that is not
    finite: scale NaN, codes 0."""
    top = x.abs().amax(-1)
    fin = torch.isfinite(x).all(-1)
    scale = (top / 127).to(torch.float32)
    scale = torch.where(fin, scale, math.nan)
    s = scale.double()[..., None]
    code = torch.round(x / s).clamp(-127, 127)
    return torch.where(s > 0, code, 0).to(torch.int8), scale


def attend(q, k, v, seen, scale):
    """q [rows, H, hd], k, v [keys, kv, hd], seen [rows, keys]; f64. Returns
    the result and a bound of what an f32-accurate kernel may be off by.

    With u = 2^-24, per (row, head): q is held as two f16 parts, to 2u of its
    largest value, or as a fixed-point number below 127/128 2^23: off by half a
    unit and by u of itself, half a unit again, and the largest value is above
    127/128 2^22 units, so to 1 / (127/128 2^22) < 5u of it. A score's hd + 4
    products and sums round by u each, so it is off by at most ds = scale (5u
    max|q| sum|k| + (hd + 4) u sum|q k|) and a weight by ds relative to it, in the sum and in the
    products. A weight is cut to two f16 parts of 10 bits and more: 2^-20 = 16u
    of itself, or the smallest f16 step, 2u of the largest value. Sums over m
    keys round by m u, twice. With the largest weight 1, the weights' sum l is
    at least 1:  |err| <= max|v| (2 ds + 16u + 2u m / l + 2 m u)."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    H, kv, hd = q.shape[1], k.shape[1], q.shape[2]
    rows, n = q.shape[0], k.shape[0]
    u = 2.0 ** -24
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape[:2], dtype=torch.float64)
    if n == 0:
        return out, tol
    for h in range(H):
        kh, vh, qh = k[:, h * kv // H], v[:, h * kv // H], q[:, h]
        s = (qh @ kh.T) * scale
        s = torch.where(seen, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        w = torch.where(seen, w, 0.0)
        l = w.sum(-1, keepdim=True)
        out[:, h] = torch.where(l > 0, (w @ vh) / l.clamp(min=1e-300), 0.0)
        ka = kh.abs()
        ds = scale * (5 * u * qh.abs().amax(-1, keepdim=True) * ka.sum(-1)
                      + (hd + 4) * u * (qh.abs() @ ka.T))
        ds = torch.where(seen, ds, 0.0).amax(-1)
        vmax = torch.where(seen, vh.abs().amax(-1)[None], 0.0).amax(-1)
        m = seen.sum(-1).double()
        tol[:, h] = vmax * (2 * ds + 16 * u + 2 * u * m
                            / l[:, 0].clamp(min=1) + 2 * m * u)
    return out, tol


def check_close(got, want, tol, what=""):
    """Element by element within tol (per row and head) and the type's final
    rounding; f32 results besides to 1e-5 in the 2-norm: the errors above add
    up as random ones, of which sqrt(4096) u = 4e-6 is the largest part."""
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    room = tol[..., None] + half * want.abs() + 2.0 ** -25
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (err / room).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: error {worst:.3g} times its bound"
    norm = want.norm().item()
    if got.dtype == torch.float32 and norm > 0:
        rel = (got.double() - want).norm().item() / norm
        assert rel <= 1e-5, f"{what}: relative error {rel:.3g}"
