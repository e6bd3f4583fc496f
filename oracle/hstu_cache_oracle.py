"""Oracle of the paged cache in 8 bits: `hstu_cache_append`, bit for bit, and `hstu_paged_8bit` in 64 bits.

THIS IS TEST INFRASTRUCTURE, NOT PRODUCT CODE (see oracle/hstu_oracle.py for who may import it).
"""
from __future__ import annotations

import math

import torch

from . import hstu_window_oracle as WO

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def numbers(x, held):
    """The 8-bit numbers nearest to x (fp32; ties to even, beyond the largest the largest, NaN: itself or 0)."""
    most = MOST[held]
    if held == torch.int8:
        return torch.nan_to_num(x, nan=0.0, posinf=most, neginf=-most).round().clamp(-most, most).to(held)
    return x.clamp(-most, most).to(held)


def block_scale(x, held):
    """The smallest power of two from 2^-100 on that the finite values of x fit."""
    x = x[torch.isfinite(x)].abs()
    amax = x.max().item() if x.numel() else 0.0
    if amax == 0.0:
        return 2.0 ** -100
    e = math.frexp(amax)[1] - 9          # amax < 2^(e + 9)
    while amax > MOST[held] * 2.0 ** e:
        e += 1
    while e > -100 and amax <= MOST[held] * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** max(e, -100)


def append(k, v, kv_cache, kv_scale, seq_offset, page_offsets, page_ids, last_page_len, num_target=None):
    """(kv_cache, kv_scale) after the call, new tensors; CPU tensors throughout."""
    cache, scale, held = kv_cache.clone(), kv_scale.clone(), kv_cache.dtype
    page, block = cache.shape[2], cache.shape[2] // scale.shape[2]
    off, po, ids = seq_offset.tolist(), page_offsets.tolist(), page_ids.tolist()
    for b in range(len(off) - 1):
        fresh = off[b + 1] - off[b] - (int(num_target[b]) if num_target is not None else 0)
        pages = po[b + 1] - po[b]
        cached = (pages - 1) * page + int(last_page_len[b]) if pages else 0
        start = cached - fresh
        for blk in range(start // block, (cached + block - 1) // block if fresh else 0):
            base, r0, r1 = blk * block, max(blk * block, start), min(cached, (blk + 1) * block)
            pid, at = ids[po[b] + base // page], base % page
            for which, x in ((0, k), (1, v)):
                rows = x[off[b] + r0 - start:off[b] + r1 - start].float()          # [n, heads, dim]
                for h in range(rows.shape[1]):
                    s = torch.tensor(block_scale(rows[:, h], held))
                    old = scale[pid, which, at // block, h].clone()
                    if r0 > base:
                        if s > old:
                            kept = cache[pid, which, at:at + r0 - base, h].float() * (old / s)
                            cache[pid, which, at:at + r0 - base, h] = numbers(kept, held)
                        else:
                            s = old
                    scale[pid, which, at // block, h] = s
                    cache[pid, which, at + r0 - base:at + r1 - base, h] = numbers(rows[:, h] / s, held)
    return cache, scale


def paged(q, k, v, kv_cache, kv_scale, max_seq_len, max_seq_len_k=0, silu_scale=0.0, seq_offset=None, seq_offset_k=None,
          page_offsets=None, page_ids=None, last_page_len=None, num_target=None, target_group_size=0, alpha=1.0, window=0,
          num_sink=0, tanh=None):
    """(value in 64 bits, tolerance).  tanh: whether SiLU may come from tanh.approx, by default where the framework's kernels take
    that form - bf16, heads of 64 and 128."""
    if tanh is None:
        tanh = q.dtype == torch.bfloat16 and q.shape[2] in (64, 128)
    off, off_k, po, ids = (t.tolist() for t in (seq_offset, seq_offset_k, page_offsets, page_ids))
    page, per_page = kv_cache.shape[2], kv_scale.shape[2]
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(len(off) - 1):
        t = int(num_target[b]) if num_target is not None else 0
        n = off_k[b + 1] - off_k[b] - t
        mine = ids[po[b]:po[b + 1]]
        rows = slice(off[b], off[b + 1])
        kv = []
        unit = torch.ones(n + t, k.shape[1], device=q.device)
        unit[:n] = kv_scale[mine, 1].repeat_interleave(page // per_page, 1).flatten(0, 1)[:n]
        for which, new in ((0, k), (1, v)):
            x = kv_cache[mine, which].float().double().flatten(0, 1) * \
                kv_scale[mine, which].double().repeat_interleave(page // per_page, 1).flatten(0, 1)[..., None]
            kv.append(torch.cat((x[:n], new[off[b + 1] - t:off[b + 1]].double())))
        see = WO.window_mask(off[b + 1] - off[b], off_k[b + 1] - off_k[b], t, target_group_size, window, num_sink, q.device)
        one = WO.attention(q[rows], *kv, see, alpha, silu_scale or 1.0 / max_seq_len, q.dtype, tanh=tanh, staged=True, unit=unit)
        out[rows], tol[rows] = one["out"]
    return out, tol
