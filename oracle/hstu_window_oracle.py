"""Oracle of `hstu_window`: HSTU attention over a sliding window with sinks, its gradients, and how far a correct kernel may
be from them.

THIS IS TEST INFRASTRUCTURE, NOT PRODUCT CODE (see oracle/hstu_oracle.py for who may import it).

Everything is computed in 64 bits, sequence by sequence, from the definition: the row at position p = i + (len_k - len_q)
sees the keys j <= p with p - j < window or j < sink; a target row (group > 0) counts its window from the end of the history
and sees the targets of its own group up to itself.

The tolerances count roundings (u = half a step of the element type, 2^-24 of a 32-bit sum):
  x = alpha q.k      off by (dim + 4) 2^-24 alpha |q|.|k|
  silu(x)            that times 1.1 (its slope), and what the approximation leaves: tanh.approx is 2^-11 off relative to tanh,
                     so silu = x (1 + tanh(x / 2)) / 2 is |x| 2^-12; the form with exp2 and a reciprocal 2^-20 relative
  P                  one rounding to the element type before the product that consumes it; below the type's normal range
                     that is half of its smallest step instead (fp16: 2^-25, which small P and dS do reach)
  sums over keys     n 2^-24 of the sum of magnitudes; the result one rounding
and the same for dS = dP f(x), f = scale alpha sg (1 + x (1 - sg)), whose slope in sg is at most scale alpha (1 + |x|).
"""
from __future__ import annotations

import torch


def window_mask(len_q, len_k, tgt, group, window, sink, device="cpu"):
    """Boolean [len_q, len_k]."""
    i = torch.arange(len_q, device=device)[:, None]
    j = torch.arange(len_k, device=device)[None, :]
    p, hist = i + len_k - len_q, len_k - tgt
    see = (j <= p) & ((p - j < window) | (j < sink)) if window else j <= p
    if tgt > 0 and group > 0:
        ti, tj = i - (len_q - tgt), j - hist
        old = tj < 0
        if window:
            old = old & ((hist - j < window) | (j < sink))
        same = (tj >= 0) & (tj <= ti) & (ti // group == tj // group)
        see = torch.where(ti >= 0, old | same, see)
    return see


def attention(q, k, v, see, alpha, scale, dtype, grad=None, tanh=False, staged=False, unit=None, behind=False):
    """One sequence: q [lq, hq, d], k, v [lk, hk, .] -> {"out": (value, tolerance)} and with grad also dq, dk, dv.
    staged: k and v may have been rounded to the element type on their way, one rounding each: u relative, and below the type's
    normal range half of its smallest step.  Such a cache's blocks may differ by any power of two, and that shows how tensor
    cores add: the products of 16 keys and the accumulator are shifted to the largest exponent among them and cut off some 25
    bits below it, and a P of zero has the exponent of one there.  So a masked value v costs the rows that do not see it up to
    2^-25 |v| for its group of 16 keys (seen as errors that are multiples of 2^-17 beside hidden values of 256).
    unit: [keys, hk], the scales of the values (value = number * scale).  A kernel may round P * scale instead of P, to fp16
    relative to the row's largest: half a smallest step is then 2^-25 of that largest, for every number.
    behind: P and dS are rounded without the scale, which the sums take: so is half a smallest step."""
    u = torch.finfo(dtype).eps / 2
    hq, hk = q.shape[1], k.shape[1]
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))                     # [heads, rows, dim]
    kk, vv = (t.repeat_interleave(hq // hk, 0) for t in (k, v))
    f32, tiny = 2.0 ** -24, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    step = tiny * abs(scale) if behind else tiny
    x = alpha * q @ kk.transpose(1, 2)
    xerr = (q.shape[2] + 4) * f32 * abs(alpha) * (q.abs() @ kk.abs().transpose(1, 2))
    if staged:
        xerr = xerr + (u + f32) * abs(alpha) * (q.abs() @ kk.abs().transpose(1, 2)) + tiny * abs(alpha) * q.abs().sum(2, keepdim=True)
    sg = torch.sigmoid(x)
    approx = x.abs() * 2.0 ** -12 if tanh else (x * sg).abs() * 2.0 ** -20
    perr = torch.where(see, abs(scale) * (1.1 * (xerr + approx) + (u + 4 * f32) * (x * sg).abs()) + step, 0.0)
    p = torch.where(see, x * sg * scale, 0.0)
    out = p @ vv
    n = k.shape[1] + 4
    got = {"out": (out, u * out.abs() + perr @ vv.abs() + (n * f32 + (u if staged else 0)) * (p.abs() @ vv.abs()) +
                   (tiny * p.abs().sum(2, keepdim=True) + (n // 16 + 1) * 2.0 ** -25 * vv.abs().amax(1, keepdim=True)
                    if staged and vv.shape[1] else 0.0))}
    if unit is not None and vv.shape[1] and dtype == torch.float16:
        scales = unit.double().t().repeat_interleave(hq // hk, 0)
        most = (p.abs() * scales[:, None, :]).amax(2, keepdim=True)
        got["out"] = got["out"][0], got["out"][1] + 2.0 ** -25 * most * (vv.abs() / scales[..., None]).sum(1, keepdim=True)
    if grad is not None:
        g = grad.double().transpose(0, 1)
        dp = g @ vv.transpose(1, 2)
        dperr = (v.shape[2] + 4) * f32 * (g.abs() @ vv.abs().transpose(1, 2))
        f = scale * alpha * sg * (1 + x * (1 - sg))
        sgerr = 0.25 * xerr + (2.0 ** -12 if tanh else sg * 2.0 ** -20)
        ferr = abs(scale * alpha) * ((1 + x.abs()) * 1.1 * sgerr + xerr * 0.3) + 8 * f32 * f.abs()
        ds = torch.where(see, dp * f, 0.0)
        dserr = torch.where(see, u * (dp * f).abs() + dp.abs() * ferr + dperr * f.abs() + dperr * ferr + step, 0.0)
        m = q.shape[1] * (hq // hk) + 4
        dq = ds @ kk
        got["dq"] = dq, u * dq.abs() + dserr @ kk.abs() + n * f32 * (ds.abs() @ kk.abs())
        for name, a, aerr, b in (("dk", ds, dserr, q), ("dv", p, perr, g)):
            shared = lambda t: t.unflatten(0, (hk, hq // hk)).sum(1)   # noqa: E731
            val = shared(a.transpose(1, 2) @ b)
            got[name] = val, u * val.abs() + shared(aerr.transpose(1, 2) @ b.abs()) + m * f32 * shared(a.abs().transpose(1, 2) @ b.abs())
    return {name: (a.transpose(0, 1), b.transpose(0, 1)) for name, (a, b) in got.items()}


def hstu_window(q, k, v, window, sink=0, max_seq_len=0, max_seq_len_k=0, silu_scale=0.0, seq_offset=None, seq_offset_k=None,
                num_target=None, target_group_size=0, alpha=1.0, grad=None, tanh=False):
    """{"out", "dq", "dk", "dv"}: (value in 64 bits, tolerance), packed like the operator's tensors."""
    offq = [int(t) for t in seq_offset]
    offk = [int(t) for t in seq_offset_k] if seq_offset_k is not None else offq
    scale = silu_scale or 1.0 / max_seq_len
    got = {"out": [torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device=q.device) for _ in range(2)]}
    if grad is not None:
        got |= {n: [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2)]
                for n, t in (("dq", q), ("dk", k), ("dv", v))}
    for b in range(len(offq) - 1):
        rows, keys = slice(offq[b], offq[b + 1]), slice(offk[b], offk[b + 1])
        t = int(num_target[b]) if num_target is not None else 0
        see = window_mask(offq[b + 1] - offq[b], offk[b + 1] - offk[b], t, target_group_size, window, sink, q.device)
        one = attention(q[rows], k[keys], v[keys], see, alpha, scale, q.dtype, grad[rows] if grad is not None else None, tanh,
                        behind=q.dtype == torch.float16)
        for name, pair in one.items():
            for full, part in zip(got[name], pair):
                full[rows if name in ("out", "dq") else keys] = part
    return {name: tuple(pair) for name, pair in got.items()}
