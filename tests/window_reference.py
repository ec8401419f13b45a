"""Windowed attention and its gradients from their formulas in 64 bits, with bounds on what the kernels' roundings may add."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(n, left, right, sinks, mask, device):
    """[B or 1, N, N]: which keys a query sees."""
    far = torch.arange(n, device=device)[None, :] - torch.arange(n, device=device)[:, None]
    seen = (far <= right) & ((far >= -left) | (torch.arange(n, device=device)[None, :] < sinks))
    return seen[None] if mask is None else seen[None] & mask[:, None, :]


def reference(q, k, v, left, right, sinks=0, rel_bias=None, mask=None, scale=None, grad=None):
    """{name: (value, bound, size)} of o and, with ``grad``, of dq, dk, dv and drel_bias.  q, k, v [B, H, N, D]; entries that mask hides, and rows of q and
    grad that see nothing, are taken as zeros.

    The bounds.  u is half a step of the 16-bit type.  Logits: fp32 sums of exact products, at most 2^-22 of the sum of magnitudes off, and
    the exponentials and sums after them some 2^-21 more: relative error e of p.  o: p rounded (u, and in fp16 half of the
    smallest step), the result rounded.  dS: p off by e, delta by what o is off, and rounded for its two products."""
    dtype, device, n = q.dtype, q.device, q.shape[2]
    u, tiny = half_step(dtype), torch.finfo(dtype).smallest_normal * half_step(dtype)
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    scale = q.shape[3] ** -0.5 if scale is None else scale
    seen = visible(n, left, right, sinks, mask, device)[:, None]
    some = seen.any(-1, keepdim=True)
    q = torch.where(some, q.double(), 0.0)
    there = mask[:, None, :, None] if mask is not None else torch.ones(1, 1, 1, 1, dtype=torch.bool, device=device)
    k, v = (torch.where(there, t.double(), 0.0).repeat_interleave(group, 1) for t in (k, v))
    logits, size = scale * q @ k.transpose(-1, -2), scale * q.abs() @ k.abs().transpose(-1, -2)
    if rel_bias is not None:
        r = rel_bias.shape[1] // 2
        at = (torch.arange(n, device=device)[None, :] - torch.arange(n, device=device)[:, None]).clamp(-r, r) + r
        logits, size = logits + rel_bias.double()[:, at], size + rel_bias.double().abs()[:, at]
    logits = logits.masked_fill(~seen, -math.inf)
    p = torch.where(some, torch.softmax(torch.where(some, logits, 0.0), -1), 0.0)
    e = 2.0 ** -20 * (1 + torch.where(seen, size, 0.0).amax(-1, keepdim=True))
    o = p @ v
    weight = p * (u + e) + tiny * seen
    bound_o = weight @ v.abs() + u * o.abs() + tiny
    out = {"o": (o, bound_o, o)}
    if grad is None:
        return out
    g = torch.where(some, grad.double(), 0.0)
    shared = lambda t: t.unflatten(1, (heads // group, group)).sum(2)  # noqa: E731
    dv, bound_dv = shared(p.transpose(-1, -2) @ g), shared(weight.transpose(-1, -2) @ g.abs())
    dp, dp_size = g @ v.transpose(-1, -2), g.abs() @ v.abs().transpose(-1, -2)
    delta, delta_size = (g * o).sum(-1, keepdim=True), (g.abs() * o.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    off = p * ((g.abs() * bound_o).sum(-1, keepdim=True) + 2.0 ** -21 * (dp_size + delta_size)) + e * ds.abs()
    rounded = off + u * ds.abs() + tiny * seen
    # The terms of dS before they cancel: a query that sees one key has dS = 0, but dP - delta of a rounded o is half a step of delta off.
    # So the norm of the error of dQ and dK is measured by these: the roundings of dS, of o in delta and of the result each are at most u of them.
    terms = p * (dp.abs() + delta.abs())
    for name, value, bound, size in (("dq", scale * ds @ k, scale * rounded @ k.abs(), scale * terms @ k.abs()),
                                     ("dk", shared(scale * ds.transpose(-1, -2) @ q), shared(scale * rounded.transpose(-1, -2) @ q.abs()),
                                      shared(scale * terms.transpose(-1, -2) @ q.abs()))):
        out[name] = (value, bound + u * value.abs() + tiny, size)
    out["dv"] = (dv, bound_dv + u * dv.abs() + tiny, dv)
    if rel_bias is not None:
        flat = at.flatten()
        put = lambda t: torch.zeros(heads, 2 * r + 1, dtype=torch.float64, device=device).index_add_(1, flat, t.sum(0).flatten(1))  # noqa: E731
        value, sums = put(ds), put(ds.abs())
        # summed in fp32: by rows and tiles, chains of some hundreds at most
        out["drel_bias"] = (value, put(off) + 2.0 ** -15 * sums + half_step(rel_bias.dtype) * value.abs() + 1e-30, sums)
    return out


def check(got, want, dtype):
    """Every entry within its bound; and the whole within two half steps of the norm of its terms (each result has two or three independent roundings of at
    most u, on the average below u / sqrt 3)."""
    for name, (value, bound, size) in want.items():
        x = got[name].double()
        assert x.shape == value.shape, name
        assert bool(torch.isfinite(x).all()), name
        over = (x - value).abs() - bound
        assert bool((over <= 0).all()), (name, float(over.max()), int((over > 0).sum()))
        if name != "drel_bias":
            assert float((x - value).norm()) <= 2 * half_step(dtype) * float(size.norm()) + 1e-6, (name, float((x - value).norm() / size.norm()))
