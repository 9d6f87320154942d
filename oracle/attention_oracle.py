"""Attention in 64 bits, with bounds on what a kernel may be off.

``attention`` and ``gradients`` follow the definition for one sequence:
q [Lq, H, d], k and v [Lk, Hk, d], ``see`` a [Lq, Lk] truth table (or [H, Lq,
Lk]).  A row that sees nothing is zero and has no gradient.

``bounds`` gives, element by element, how far a result of a kernel may be from
these: it follows each rounding of the kernel's arithmetic through the formula
with absolute values.  u = half a step of fp32, w = half a step of the tensors'
type (what weights and score gradients are rounded to before they enter a
product; 0 in fp32), d and L the lengths of the sums:

* scores:  e_s = (d + 4) u scale |q|.|k|, as an error of the exponent, plus the
  exponential's own 2^-21; weights are off by 2 e_s (numerator and sum) + w;
* out:     P (2 e_s + w + (L + 8) u) |v|, and w |out| for the result's rounding;
* delta:   |g|.tol(out), dP: (d + 4) u |g|.|v|;  dS = P (dP - delta) is off by
  |dS| (2 e_s + w) + P (tol(dP) + tol(delta)) and so on.
"""
from __future__ import annotations

import torch


def _heads(x, h):
    """[L, Hk, d] -> [H, L, d] in 64 bits, the heads of a group side by side."""
    x = x.detach().double().transpose(0, 1)
    return x.repeat_interleave(h // x.shape[0], dim=0)


def weights(q, k, see, scale):
    """(P [H, Lq, Lk], lse [H, Lq])."""
    h = q.shape[1]
    s = torch.matmul(_heads(q, h), _heads(k, h).transpose(1, 2)) * scale
    s = torch.where(see, s, torch.full_like(s, float("-inf")))
    lse = torch.logsumexp(s, dim=-1) if s.shape[-1] else s.new_full(s.shape[:-1], float("-inf"))
    p = torch.where(see & torch.isfinite(lse)[..., None], torch.exp(s - lse[..., None]), torch.zeros_like(s))
    return p, lse


def _masked(x, see):
    """Rows of k or v no query sees, set to zero: they may hold anything."""
    any_row = see.reshape(-1, see.shape[-1]).any(dim=0)
    return torch.where(any_row[:, None, None], x.detach().double(), torch.zeros((), dtype=torch.float64, device=x.device))


def attention(q, k, v, see, scale):
    """(out [Lq, H, d], lse [H, Lq])."""
    k, v = _masked(k, see), _masked(v, see)
    p, lse = weights(q, k, see, scale)
    return torch.matmul(p, _heads(v, q.shape[1])).transpose(0, 1), lse


def _fold(x, hk):
    """[H, L, d] -> [L, Hk, d]: the sum over the heads of a group."""
    h, n, d = x.shape
    return x.reshape(hk, h // hk, n, d).sum(1).transpose(0, 1)


def gradients(q, k, v, g, see, scale):
    """(dq, dk, dv) for the gradient g [Lq, H, d] of the output."""
    h, hk = q.shape[1], k.shape[1]
    k, v = _masked(k, see), _masked(v, see)
    p, _ = weights(q, k, see, scale)
    gh, qh, kh, vh = (_heads(x, h) for x in (g, q, k, v))
    out = torch.matmul(p, vh)
    ds = p * (torch.matmul(gh, vh.transpose(1, 2)) - (gh * out).sum(-1, keepdim=True))
    return ((torch.matmul(ds, kh) * scale).transpose(0, 1), _fold(torch.matmul(ds.transpose(1, 2), qh) * scale, hk),
            _fold(torch.matmul(p.transpose(1, 2), gh), hk))


def bounds(q, k, v, see, scale, dtype, g=None, kv_error=0.0, weight_step=None, grad_steps=None):
    """Tolerances of out, or with g of (out, dq, dk, dv).  kv_error: a relative error that k
    and v already carry on their way into the products.  weight_step: the error of a weight that
    is too small for its type, grad_steps: of (P, dS) in the gradients' products; by default fp16's
    smallest step, and nothing in the other types, whose exponents reach as far as fp32's."""
    u = 2.0**-24
    w = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    r = torch.finfo(dtype).eps / 2
    h, hk, d, n = q.shape[1], k.shape[1], q.shape[2], k.shape[0]
    k, v = _masked(k, see), _masked(v, see)
    p, _ = weights(q, k, see, scale)
    qh, kh, vh = (_heads(x, h) for x in (q, k, v))
    dot = torch.matmul(qh.abs(), kh.abs().transpose(1, 2)) * abs(scale)
    e_s = torch.where(see, ((d + 4) * u + kv_error) * dot, torch.zeros_like(dot)).amax(-1, keepdim=True) + 2.0**-21
    e_p = 2 * e_s + w
    sums = (n + 8) * u
    out = torch.matmul(p, vh)
    tol = torch.matmul(p * (e_p + sums + kv_error), vh.abs()) + r * out.abs()
    # a result below the type's normal range is rounded to its smallest step; a weight too
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    tiny = step if dtype == torch.float16 else 0.0
    if weight_step is None:
        weight_step = tiny
    p_step, ds_step = (tiny, tiny) if grad_steps is None else grad_steps
    low = weight_step * torch.matmul(see.double().expand_as(p), vh.abs())
    tol = tol + step + low
    if g is None:
        return tol.transpose(0, 1)
    gh = _heads(g, h)
    dp = torch.matmul(gh, vh.transpose(1, 2))
    ds = p * (dp - (gh * out).sum(-1, keepdim=True))
    t_delta = (gh.abs() * tol).sum(-1, keepdim=True) + (d + 4) * u * (gh * out).abs().sum(-1, keepdim=True)
    t_dp = (d + 4) * u * torch.matmul(gh.abs(), vh.abs().transpose(1, 2))
    t_ds = ds.abs() * e_p + p * (t_dp + t_delta) + ds_step * see
    m = q.shape[0]
    t_dq = abs(scale) * torch.matmul(t_ds + sums * ds.abs(), kh.abs())
    t_dk = abs(scale) * torch.matmul((t_ds + (m + 8) * u * ds.abs()).transpose(1, 2), qh.abs())
    t_dv = torch.matmul((p * (e_p + (m + 8) * u) + p_step * see).transpose(1, 2), gh.abs())
    dq, dk, dv = gradients(q, k, v, g, see, scale)
    return (tol.transpose(0, 1), t_dq.transpose(0, 1) + r * dq.abs() + step, _fold(t_dk, hk) + r * dk.abs() + step,
            _fold(t_dv, hk) + r * dv.abs() + step)


def quantise(x):
    """(codes as the values they stand for, scales) of an e4m3 cache row: 64 bits, ties to even."""
    x = x.detach().double()
    m = x.abs().amax(-1).clamp_min(2.0**-100)
    y = x * 448.0 / m[..., None]  # a tie stays one: the product is exact
    size = y.abs().clamp_min(2.0**-6)
    e = torch.frexp(size).exponent - 1
    step = torch.ldexp(torch.ones_like(size), e - 3)
    return torch.round(y / step) * step, m / 448.0
