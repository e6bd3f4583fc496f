"""What the windowed attention and the 8-bit cache are timed on: the calls a recommendation model with long histories
makes when it trains, ranks and appends to its cache.

Five kinds of case, each a pass through the public entry points:

  window   `hstu_window`: attention in which a row sees the last `window` keys and the first `sink` ones, inference
  train    the same with its gradients: one attention layer's part of a training step
  append   `hstu_cache_append`: new keys and values into a paged cache of 8-bit rows with a scale per block of tokens and head
  step     `hstu_cache_append` and `hstu_paged_8bit` behind it: one serving step of users whose histories lie in such a cache
  rank     `hstu_paged_8bit` alone: candidates against cached histories

A case is a dict of plain values.  Its sequence lengths come from the case alone (so that its work is known); the seed
decides which user has which length, and every value.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_MOST = {"e4m3": 448.0, "int8": 127.0}


def _window(kind, dtype="bf16", batch=32, heads=4, kv_heads=None, dim_qk=128, dim_v=128, lo=256, hi=1024, targets=0, group=1,
            window=256, sink=4, lengths_seed=0, **more):
    return dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads or heads, dim_qk=dim_qk, dim_v=dim_v,
                lengths="uniform", lo=lo, hi=hi, mu=0.0, sigma=0.0, targets=targets, group=group, window=window, sink=sink,
                lengths_seed=lengths_seed, **more)


def _cached(kind, dtype="bf16", held="e4m3", batch=128, heads=8, kv_heads=None, dim=128, lengths="uniform", lo=200, hi=2048,
            mu=0.0, sigma=0.0, new_rows=1, targets=0, page=128, block=32, window=0, sink=0, lengths_seed=0, **more):
    return dict(kind=kind, dtype=dtype, held=held, batch=batch, heads=heads, kv_heads=kv_heads or heads, dim=dim, lengths=lengths,
                lo=lo, hi=hi, mu=mu, sigma=sigma, new_rows=new_rows, targets=targets, page=page, block=block, window=window,
                sink=sink, lengths_seed=lengths_seed, **more)


def listed():
    return [
        # One small online request: 8 users of at most 200 events with their candidates; latency is what counts.
        _window("window", name="window_request", batch=8, dim_qk=64, dim_v=64, lo=20, hi=200, targets=16, window=64),
        # An ordinary inference batch: 32 histories of 256 to 1024 events, a quarter of the longest one visible.
        _window("window", name="window_mid"),
        # The longest histories, which are what a window is for.
        _window("window", name="window_long", batch=16, lo=4096, hi=8192, window=512, sink=16),
        # A training step with candidates behind every history.
        _window("train", name="window_train_mid", targets=32, window=128, sink=8),
        # A training step on long histories, the largest case of all.
        _window("train", name="window_train_long", batch=16, heads=8, lo=1024, hi=4096, window=512),
        # A training step in fp32 with shared key heads, as in a numerics study of a small model.
        _window("train", "fp32", name="window_train_fp32", batch=16, heads=2, kv_heads=1, dim_qk=64, dim_v=64, lo=50, hi=500,
                window=100),
        # The histories of 256 users written into an empty cache.
        _cached("append", name="append_histories", batch=256, heads=4, dim=64, lengths="lognormal", lo=64, hi=2048,
                mu=math.log(600), sigma=0.6, new_rows=2048),
        # The smallest serving step: 4 users, one new event each, the other two types.
        _cached("step", "fp16", "int8", name="step_few", batch=4, heads=4, dim=64, lo=20, hi=200, page=32, block=16),
        # One new event of each of 128 users, 8 heads of 128.
        _cached("step", name="step_batch"),
        # One new event of 4 users with the longest histories the operators take: few rows, a long axis.
        _cached("step", name="step_long", batch=4, lo=14000, hi=20000, block=64),
        # The same for 512 users whose model sees a window and the first events.
        _cached("step", name="step_window", batch=512, heads=4, lo=1024, hi=8192, window=1024, sink=16),
        # Ranking: 4096 users, mostly short, 16 new events and up to 64 candidates as queries.
        _cached("rank", name="rank_serving", batch=4096, heads=4, dim=64, lengths="lognormal", lo=8, hi=2048, mu=math.log(200),
                sigma=0.8, new_rows=16, targets=64),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "train", "train", "append", "step", "step", "rank"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    heads = rng.choice([2, 4, 8])
    kv_heads = rng.choice([heads, heads, heads // 2])
    sink = rng.choice([0, 1, 4, _spread(rng, 1, 200)])
    if kind in ("window", "train"):
        if rng.random() < 0.2:
            dtype = "fp32"
        dims = rng.choice([(64, 64), (128, 128), (128, 128), (32, 32), (64, 128), (96, 96)])
        hi = _spread(rng, 60, 8000 if kind == "window" else 4000)
        if dtype == "fp32":
            hi = min(hi, 1500)
        # as many sequences as the dense form of the scores leaves room for
        most = (4e9 if kind == "window" else 1.6e9) if dtype != "fp32" else 3e7
        batch = max(1, min(_spread(rng, 1, 512), int(most / (heads * hi * hi))))
        lo = max(1, int(hi * rng.choice([0.05, 0.25, 0.5])))
        return _window(kind, dtype, batch, heads, kv_heads, dims[0], dims[1], lo, hi, targets=rng.choice([0, _spread(rng, 1, 64)]),
                       group=rng.choice([1, 1, 3]), window=_spread(rng, 1, hi), sink=sink, lengths_seed=rng.randrange(1 << 20))
    held = rng.choice(["e4m3", "e4m3", "int8"])
    dim = rng.choice([64, 128, 128, 32, 96])
    page = rng.choice([32, 64, 128, 256])
    block = rng.choice([b for b in (8, 16, 32, 64, 128) if page % b == 0])
    hi = _spread(rng, 40, 2048 if kind != "step" else 16000)
    lo = max(1, int(hi * rng.choice([0.05, 0.25, 0.5])))
    queries = {"append": hi, "step": 4, "rank": 80}[kind]
    new = {"append": _spread(rng, 1, hi), "step": rng.choice([1, 1, 4]), "rank": _spread(rng, 1, 16)}[kind]
    batch = max(1, min(_spread(rng, 1, 2048), int(1e9 / (hi * kv_heads * dim)), int(2e9 / (hi * heads * queries)) if kind != "append" else 2048))
    window = rng.choice([0, 0, _spread(rng, 1, hi)]) if kind != "append" else 0
    return _cached(kind, dtype, held, batch, heads, kv_heads, dim, lo=lo, hi=hi, new_rows=new,
                   targets=_spread(rng, 1, 64) if kind == "rank" else 0, page=page, block=block, window=window,
                   sink=sink if window else 0, lengths_seed=rng.randrange(1 << 20))


# ------------------------------------------------------------------------------------------------ lengths and work
def _lengths(case):
    """(rows, targets among them) of the sequences of a case, in the order they are drawn in."""
    rng = np.random.default_rng(case["lengths_seed"])
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    if case["lengths"] == "lognormal":
        ls = np.clip(np.rint(rng.lognormal(case["mu"], case["sigma"], n)), lo, hi).astype(np.int64)
    else:
        ls = rng.integers(lo, hi + 1, n).astype(np.int64)
    ts = np.minimum(rng.integers(1, case["targets"] + 1, n), ls - 1) if case["targets"] else np.zeros(n, np.int64)
    return ls, np.maximum(ts, 0).astype(np.int64)


def _cached_lengths(case):
    """(cached rows, new rows among them, targets) of every user."""
    ls, ts = _lengths(case)
    cached = np.maximum(ls - ts, 1)
    return cached, np.minimum(cached, case["new_rows"]), ts


def _seen(position, window, sink):
    """How many keys a history row at this position sees."""
    if not window:
        return position + 1
    return np.minimum(position + 1, window) + np.minimum(sink, np.maximum(0, position + 1 - window))


def _pairs(case, first, hist, ts):
    """Visible (row, key) pairs: history rows first .. hist of each sequence, then its targets."""
    window, sink, group = case["window"], case["sink"], case.get("group", 1)
    rows = sum(int(_seen(np.arange(a, h), window, sink).sum()) for a, h in zip(first, hist))
    return rows + sum(int((_seen(h, window, sink) - 1) * t + (np.arange(t) % group + 1).sum()) for h, t in zip(hist, ts))


def work(case):
    hq, hk = case["heads"], case["kv_heads"]
    if case["kind"] in ("window", "train"):
        es, dq, dv = _BYTES[case["dtype"]], case["dim_qk"], case["dim_v"]
        ls, ts = _lengths(case)
        pairs, tokens = _pairs(case, np.zeros_like(ls), ls - ts, ts), int(ls.sum())
        qkv = tokens * (hq * dq + hk * (dq + dv))
        if case["kind"] == "train":
            return {"bytes": float(es * (2 * qkv + 2 * tokens * hq * dv)), "flops": 2.0 * hq * (4 * dq + 3 * dv) * pairs}
        return {"bytes": float(es * (qkv + tokens * hq * dv)), "flops": 2.0 * hq * (dq + dv) * pairs}
    dim, es = case["dim"], _BYTES[case["dtype"]]
    cached, new, ts = _cached_lengths(case)
    scales = 4.0 / case["block"] / dim
    appended = float(2 * hk * dim * int(new.sum())) * (es + 1 + scales)
    if case["kind"] == "append":
        return {"bytes": appended, "flops": float(4 * hk * dim * int(new.sum()))}
    visible = cached
    if case["window"]:   # of the cached rows: what any row of the user's sees
        visible = np.minimum(cached, case["window"] + new - 1 + np.minimum(case["sink"], cached))
    rows = int((new + ts).sum())
    bytes_ = float(2 * hk * dim * int(visible.sum())) * (1 + scales) + es * float(rows * hq * 2 * dim + int(ts.sum()) * hk * 2 * dim)
    return {"bytes": bytes_ + (appended if case["kind"] == "step" else 0.0),
            "flops": 4.0 * hq * dim * _pairs(case, cached - new, cached, ts)}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype = _DTYPES[case["dtype"]]
    hq, hk = case["heads"], case["kv_heads"]
    order = rng.permutation(case["batch"])

    def rnd(*shape, scale=0.5, grad=False):
        return torch.empty(*shape, device=dev, dtype=dtype).normal_(0.0, scale, generator=gen).requires_grad_(grad)

    def offsets(counts):
        return torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)).to(dev)

    def index(values):
        return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int64)).to(dev)

    if case["kind"] in ("window", "train"):
        dq, dv = case["dim_qk"], case["dim_v"]
        ls, ts = (a[order] for a in _lengths(case))
        tokens, grad = int(ls.sum()), case["kind"] == "train"
        state = dict(kind=case["kind"], q=rnd(tokens, hq, dq, grad=grad), k=rnd(tokens, hk, dq, grad=grad),
                     v=rnd(tokens, hk, dv, grad=grad), max_seq_len=case["hi"], seq_offset=offsets(ls),
                     num_target=index(ts) if case["targets"] else None, group=case["group"] if case["targets"] else 0,
                     alpha=dq ** -0.5, window=case["window"], sink=case["sink"])
        if grad:
            state["grad_out"] = rnd(tokens, hq, dv)
        return state

    dim, page, block = case["dim"], case["page"], case["block"]
    cached, new, ts = (a[order] for a in _cached_lengths(case))
    count = (cached + page - 1) // page
    pages, rows = int(count.sum()) + 2, int((new + ts).sum())
    held, most = _DTYPES[case["held"]], _MOST[case["held"]]
    # A cache that was filled earlier, block by block; what the new rows' places hold is left over from other users.  Heads
    # differ in size, as they do in a trained model.
    x = torch.empty(pages, 2, page // block, block, hk, dim, device=dev).normal_(0.0, 0.5, generator=gen)
    x *= torch.exp2(torch.arange(hk, device=dev) % 4 - 2.0)[:, None]
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(3, 5)) / most)))
    x /= scale[:, :, :, None, :, None]
    cache = (x if held.is_floating_point else x.round()).clamp(-most, most).to(held).view(pages, 2, page, hk, dim)
    del x
    return dict(kind=case["kind"], q=rnd(rows, hq, dim), k=rnd(rows, hk, dim), v=rnd(rows, hk, dim), cache=cache,
                scale=scale.contiguous(), max_q=int((new + ts).max()), max_k=int((cached + ts).max()), seq_offset=offsets(new + ts),
                seq_offset_k=offsets(cached + ts), page_offsets=offsets(count), page_ids=index(rng.permutation(pages)[: pages - 2]),
                last_page_len=index(cached - (count - 1) * page), num_target=index(ts) if case["targets"] else None,
                group=1 if case["targets"] else 0, alpha=dim ** -0.5, window=case["window"], sink=case["sink"])


# ------------------------------------------------------------------------------------------------ the plain form
def _visible(lq, lk, tgt, group, window, sink, nq, nk):
    """[batch, nq, nk]: whether row i sees key j.  A history row at position p sees the keys up to p of which it is less than
    `window` away, and the first `sink` ones; a target counts its window from the end of the history, and sees the targets of
    its own group up to itself."""
    i = torch.arange(nq, device=lq.device)[None, :, None]
    j = torch.arange(nk, device=lq.device)[None, None, :]
    lq, lk, tgt = lq[:, None, None], lk[:, None, None], tgt[:, None, None]
    position, hist, nth = i + lk - lq, lk - tgt, i - (lq - tgt)
    target = nth >= 0 if group else torch.zeros_like(nth, dtype=torch.bool)
    at = torch.where(target, hist, position)
    past = torch.where(target, j < hist, j <= position)
    if window:
        past &= (at - j < window) | (j < sink)
    if group:
        past |= target & (j >= hist) & (j <= position) & (nth // group == (j - hist) // group)
    return past & (i < lq) & (j < lk)


def _padded(x, offset, n):
    """[tokens, heads, dim] -> [batch, heads, n, dim] in 32 bits; rows behind a sequence's end hold anything finite."""
    at = (offset[:-1, None] + torch.arange(n, device=x.device)).clamp(max=x.shape[0] - 1)
    return x.float()[at].transpose(1, 2)


def _packed(x, offset, tokens):
    """The other way round."""
    b = torch.repeat_interleave(torch.arange(offset.numel() - 1, device=x.device), offset.diff(), output_size=tokens)
    return x[b, :, torch.arange(tokens, device=x.device) - offset[b]]


def _attend(q, k, v, see, alpha, scale):
    """[batch, heads, rows, dim] each; one key head per query head."""
    x = (q @ k.transpose(2, 3)).mul_(alpha)
    p = torch.exp(-x).add_(1.0).reciprocal_().mul_(x).mul_(scale)
    return p.masked_fill_(~see[:, None], 0.0) @ v


def _attend_gradients(q, k, v, g, see, alpha, scale):
    x = (q @ k.transpose(2, 3)).mul_(alpha)
    s = torch.exp(-x).add_(1.0).reciprocal_()
    see = see[:, None]
    dv = (x * s).mul_(scale).masked_fill_(~see, 0.0).transpose(2, 3) @ g
    # d silu(x) / dx = s (1 + x (1 - s))
    d = x.mul_(1.0 - s).add_(1.0).mul_(s)
    del s
    d.mul_(g @ v.transpose(2, 3)).mul_(scale * alpha).masked_fill_(~see, 0.0)
    return d @ k, d.transpose(2, 3) @ q, dv


def _plain_window(s):
    n, dtype = s["max_seq_len"], s["q"].dtype
    lengths = s["seq_offset"].diff()
    tgt = s["num_target"] if s["num_target"] is not None else torch.zeros_like(lengths)
    see = _visible(lengths, lengths, tgt, s["group"], s["window"], s["sink"], n, n)
    tokens, ratio = s["q"].shape[0], s["q"].shape[1] // s["k"].shape[1]
    q, k, v = (_padded(s[name].detach(), s["seq_offset"], n) for name in ("q", "k", "v"))
    k, v = k.repeat_interleave(ratio, 1), v.repeat_interleave(ratio, 1)
    out = _packed(_attend(q, k, v, see, s["alpha"], 1.0 / n), s["seq_offset"], tokens).to(dtype)
    if s["kind"] == "window":
        return out
    dq, dk, dv = _attend_gradients(q, k, v, _padded(s["grad_out"], s["seq_offset"], n), see, s["alpha"], 1.0 / n)
    dk, dv = dk.unflatten(1, (-1, ratio)).sum(2), dv.unflatten(1, (-1, ratio)).sum(2)
    return [out] + [_packed(d, s["seq_offset"], tokens).to(dtype) for d in (dq, dk, dv)]


def _rows_of_cache(s, n):
    """(page, row inside it) of each user's first n cached rows, [batch, n]; any page where there is none."""
    j = torch.arange(n, device=s["cache"].device)
    page = s["cache"].shape[2]
    slot = (s["page_offsets"][:-1, None] + j // page).clamp(max=s["page_ids"].numel() - 1)
    return s["page_ids"][slot], (j % page).expand(slot.shape)


def _plain_append(s):
    """New rows into the cache.  A block's scale is the smallest power of two that its rows fit, and never shrinks; rows the
    block holds already are held anew when it grows."""
    cache, scale = s["cache"].view(torch.uint8), s["scale"]
    pages, _, page, hk, dim = cache.shape
    block, held = page // scale.shape[2], s["cache"].dtype
    most = _MOST["e4m3" if held.is_floating_point else "int8"]
    tgt = s["num_target"] if s["num_target"] is not None else torch.zeros_like(s["last_page_len"])
    count = s["seq_offset"].diff() - tgt                     # new rows of each user
    cached = s["seq_offset_k"].diff() - tgt
    start = cached - count
    tokens = s["k"].shape[0]
    b = torch.repeat_interleave(torch.arange(count.numel(), device=cache.device), s["seq_offset"].diff(), output_size=tokens)
    nth = torch.arange(tokens, device=cache.device) - s["seq_offset"][b]
    is_new = nth < count[b]                                  # (targets are not kept: their place is one past the cache's end)
    at = start[b] + nth
    slot = (s["page_offsets"][b] + at // page).clamp(max=s["page_ids"].numel() - 1)
    where = torch.where(is_new, s["page_ids"][slot], pages)
    row = at % page
    x = torch.stack((s["k"], s["v"]), 1).float()             # [tokens, 2, heads, dim]
    # scales: what the new rows need, and what a block that holds rows already has
    need = torch.zeros(pages + 1, scale.shape[2], 2, hk, device=cache.device)
    need.index_put_((where, row // block), torch.zeros((), device=cache.device))
    flat = where * scale.shape[2] + row // block
    need = need.view(-1, 2, hk).index_reduce_(0, flat, x.abs().amax(-1), "amax").view_as(need)
    m, e = torch.frexp(need)
    e = e - (9 if held.is_floating_point else 7) + (m > (0.875 if held.is_floating_point else 0.9921875))
    need = torch.exp2(torch.where(need > 0, e, -100).clamp(min=-100).float())
    first_at = start // block * block                        # the block of each user's first new row
    part = (start > first_at) & (count > 0)
    fslot = (s["page_offsets"][:-1] + first_at // page).clamp(max=s["page_ids"].numel() - 1)
    fpage, fblock = s["page_ids"][fslot], first_at % page // block
    old = scale[fpage, :, fblock]                            # [batch, 2, heads]
    both = torch.where(part[:, None, None], torch.maximum(need[fpage, fblock], old), need[fpage, fblock])
    need[torch.where(count > 0, fpage, pages), fblock] = both
    # the rows those blocks hold already
    r = torch.arange(block, device=cache.device)
    rows = first_at[:, None] % page + r
    keep = part[:, None] & (first_at[:, None] + r < start[:, None])
    kept = cache[fpage[:, None], :, rows].view(held).float() * (old / both)[:, None, :, :, None]
    kept = _held(kept, most, held)
    padded = torch.cat((cache, torch.empty_like(cache[:1])))   # (one page more, for what is not kept)
    padded[torch.where(keep, fpage[:, None], pages), :, rows] = kept
    padded[where, :, row] = _held(x / need[where, row // block][..., None], most, held)
    cache.copy_(padded[:pages])
    new_scale = torch.cat((scale, torch.empty_like(scale[:1])))
    new_scale[where, :, row // block] = need[where, row // block]
    scale.copy_(new_scale[:pages])


def _held(x, most, held):
    return (x if held.is_floating_point else x.round()).clamp(-most, most).to(held).view(torch.uint8)


def _plain_paged(s):
    dtype, nq, nk = s["q"].dtype, s["max_q"], s["max_k"]
    lq, lk = s["seq_offset"].diff(), s["seq_offset_k"].diff()
    tgt = s["num_target"] if s["num_target"] is not None else torch.zeros_like(lq)
    page, block = s["cache"].shape[2], s["cache"].shape[2] // s["scale"].shape[2]
    where, row = _rows_of_cache(s, nk)
    # targets come from the call's own keys and values
    own_row = (s["seq_offset"][1:, None] - lk[:, None] + torch.arange(nk, device=lk.device)).clamp(0, s["k"].shape[0] - 1)
    cached = (torch.arange(nk, device=lk.device) < (lk - tgt)[:, None])[:, :, None, None]
    ratio = s["q"].shape[1] // s["k"].shape[1]

    def operand(which, new):
        x = s["cache"].view(torch.uint8)[where, which, row].view(s["cache"].dtype).float()
        x *= s["scale"][where, which, row // block][..., None]
        return torch.where(cached, x, new.float()[own_row]).transpose(1, 2).repeat_interleave(ratio, 1)

    see = _visible(lq, lk, tgt, s["group"], s["window"], s["sink"], nq, nk)
    q = _padded(s["q"], s["seq_offset"], nq)
    out = _attend(q, operand(0, s["k"]), operand(1, s["v"]), see, s["alpha"], 1.0 / nq)
    return _packed(out, s["seq_offset"], s["q"].shape[0]).to(dtype)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        import ops_rec_b200 as ops_rec
        attention = ops_rec.ascendc.attention
    if s["kind"] in ("window", "train"):
        if not own:
            return _plain_window(s)
        out = attention.hstu_window(s["q"], s["k"], s["v"], s["window"], s["sink"], s["max_seq_len"], 0, 0.0, s["seq_offset"],
                                    None, s["num_target"], s["group"], s["alpha"])
        if s["kind"] == "window":
            return out
        return [out] + list(torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["grad_out"]))
    out = None
    if s["kind"] != "rank":
        if own:
            attention.hstu_cache_append(s["k"], s["v"], s["cache"], s["scale"], s["seq_offset"], s["page_offsets"], s["page_ids"],
                                        s["last_page_len"], s["num_target"])
        else:
            _plain_append(s)
    if s["kind"] != "append":
        if own:
            out = attention.hstu_paged_8bit(s["q"], s["k"], s["v"], s["cache"], s["scale"], s["max_q"], s["max_k"], 0.0,
                                            s["seq_offset"], s["seq_offset_k"], s["page_offsets"], s["page_ids"],
                                            s["last_page_len"], s["num_target"], s["group"], s["alpha"], s["window"], s["sink"])
        else:
            out = _plain_paged(s)
    if s["kind"] == "rank":
        return out
    # the cache's numbers and their scales, as they are held
    return {"cache": s["cache"], "scale": s["scale"]} | ({} if out is None else {"out": out})


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attention(q, k, v, tgt, group, window, sink, alpha, scale):
    """One sequence, [rows, heads, dim] in 64 bits; key heads are shared by neighbouring query heads."""
    lq, lk = q.shape[0], k.shape[0]
    hist = lk - tgt
    j = torch.arange(lk, device=q.device)
    end = torch.arange(lq, device=q.device) + (lk - lq) + 1      # one past the last key of a row, targets left aside
    low = end - window if window else torch.full_like(end, -(1 << 60))
    if group and tgt:
        low[lq - tgt:] = hist + 1 - window if window else -(1 << 60)
        end[lq - tgt:] = hist
    see = (j < end[:, None]) & ((j >= low[:, None]) | (j < sink))
    if group and tgt:
        t = torch.arange(tgt, device=q.device)
        see[lq - tgt:, hist:] = (t[:, None] >= t) & (t[:, None] // group == t // group)
    k, v = (x.repeat_interleave(q.shape[1] // x.shape[1], 1) for x in (k, v))
    x = torch.einsum("ihd,jhd->hij", q, k) * alpha
    return torch.einsum("hij,jhd->ihd", torch.where(see, torch.nn.functional.silu(x) * scale, 0.0), v)


def exact(case, seed):
    s = prepare(case, seed)
    off = s["seq_offset"].tolist()
    tgt = s["num_target"].tolist() if s["num_target"] is not None else [0] * (len(off) - 1)
    if case["kind"] in ("window", "train"):
        train = case["kind"] == "train"
        leaves = [s[n].detach().double().requires_grad_(train) for n in ("q", "k", "v")]
        got = [torch.empty(s["q"].shape[0], case["heads"], case["dim_v"], dtype=torch.float64, device=leaves[0].device)]
        got += [torch.empty_like(x) for x in leaves] if train else []
        for a, b, t in zip(off, off[1:], tgt):
            one = [x.detach()[a:b].requires_grad_(train) for x in leaves]
            out = _exact_attention(*one, t, s["group"], s["window"], s["sink"], s["alpha"], 1.0 / s["max_seq_len"])
            got[0][a:b] = out.detach()
            if train:
                for full, g in zip(got[1:], torch.autograd.grad(out, one, s["grad_out"][a:b].double())):
                    full[a:b] = g
        return got if train else got[0]
    cache, scale = s["cache"].double(), s["scale"].double()
    off_k, po, ids = s["seq_offset_k"].tolist(), s["page_offsets"].tolist(), s["page_ids"].tolist()
    page, per_page = cache.shape[2], scale.shape[2]
    block, bits = page // per_page, {"e4m3": (9, 0.875), "int8": (7, 127 / 128)}[case["held"]]
    k, v = s["k"].double(), s["v"].double()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=cache.device)
    for b in range(len(off) - 1):
        n_cached = off_k[b + 1] - off_k[b] - tgt[b]
        mine = torch.tensor(ids[po[b]:po[b + 1]], device=cache.device)
        value = cache[mine].transpose(0, 1).reshape(2, len(mine) * page, *cache.shape[3:])
        factor = scale[mine].transpose(0, 1).reshape(2, len(mine) * per_page, -1)
        if case["kind"] != "rank":
            new = off[b + 1] - off[b] - tgt[b]
            begin = n_cached - new
            fresh = torch.stack((k[off[b]:off[b] + new], v[off[b]:off[b] + new]))
            first = begin // block
            held = torch.zeros(2, (n_cached + block - 1) // block - first, block, *cache.shape[3:], dtype=torch.float64, device=cache.device)
            flat = held.flatten(1, 2)                       # from the first touched block on
            lead = begin - first * block
            flat[:, lead:lead + new] = fresh
            big = held.abs().amax(dim=(2, 4))
            m, e = torch.frexp(big)
            want = torch.ldexp(torch.ones_like(big), torch.where(big > 0, e - bits[0] + (m > bits[1]).int(), -100).clamp(min=-100))
            if lead:
                before = factor[:, first].clone()
                want[:, 0] = torch.maximum(want[:, 0], before)
                flat[:, :lead] = value[:, first * block:begin] * before[:, None, :, None]
            x = (held / want[:, :, None, :, None]).flatten(1, 2)[:, :lead + new]
            # (powers of two: the quotients are those of 32 bits, and are rounded once)
            x = x.float().to(torch.float8_e4m3fn).double() if case["held"] == "e4m3" else x.round()
            value[:, first * block:n_cached] = x
            factor[:, first:first + want.shape[1]] = want
            cache[mine] = value.view(2, len(mine), page, *cache.shape[3:]).transpose(0, 1)
            scale[mine] = factor.view(2, len(mine), per_page, -1).transpose(0, 1)
        if case["kind"] != "append":
            kk, vv = (value[w, :n_cached] * factor[w].repeat_interleave(block, 0)[:n_cached, :, None] for w in (0, 1))
            kk, vv = torch.cat((kk, k[off[b + 1] - tgt[b]:off[b + 1]])), torch.cat((vv, v[off[b + 1] - tgt[b]:off[b + 1]]))
            out[off[b]:off[b + 1]] = _exact_attention(s["q"][off[b]:off[b + 1]].double(), kk, vv, tgt[b], s["group"], s["window"],
                                                      s["sink"], s["alpha"], 1.0 / s["max_q"])
    if case["kind"] == "rank":
        return out
    # (a cache of whole numbers has no other value than the one that run() returns)
    whole = {"cache": cache if case["held"] == "e4m3" else cache.to(torch.int8), "scale": scale}
    return whole | ({} if case["kind"] == "append" else {"out": out})
