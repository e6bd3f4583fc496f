"""hstu_cache_append and hstu_paged_8bit: refusals (CPU), the numbers and scales bit for bit and the attention against 64 bits
with tolerances that count roundings (GPU; oracle/hstu_cache_oracle.py, oracle/hstu_window_oracle.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

import ops_rec_b200 as ops_rec
from oracle import hstu_cache_oracle as CO
from ops_rec_b200 import cabi

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
append_op = ops_rec.ascendc.attention.hstu_cache_append
paged_op = ops_rec.ascendc.attention.hstu_paged_8bit


# ------------------------------------------------------------------------------------------------------- CPU
def test_oracle_scales_and_numbers():
    assert CO.block_scale(torch.tensor([448.0]), E4M3) == 1.0 and CO.block_scale(torch.tensor([448.1]), E4M3) == 2.0
    assert CO.block_scale(torch.tensor([127.0, -3]), INT8) == 1.0 and CO.block_scale(torch.tensor([-127.1]), INT8) == 2.0
    assert CO.block_scale(torch.tensor([0.0, float("nan"), float("inf")]), E4M3) == 2.0 ** -100
    x = torch.tensor([float("nan"), float("inf"), -1e9, 2.5, 3.5, 0.0])
    assert CO.numbers(x, INT8).tolist() == [0, 127, -127, 2, 4, 0]
    e = CO.numbers(x, E4M3).float()
    assert e[0].isnan() and e[1:].tolist() == [448, -448, 2.5, 3.5, 0]


def meta(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_operators_on_meta_tensors_and_their_refusals():
    k, cache, scale = meta(10, 2, 64), meta(6, 2, 32, 2, 64, dtype=E4M3), meta(6, 2, 2, 2, dtype=FP32)
    i = lambda n: meta(n, dtype=torch.int64)   # noqa: E731
    table = (i(3), i(3), i(6), i(2))
    append_op(k, k, cache, scale, *table)
    q = meta(10, 4, 64)
    at = lambda *a, **kw: paged_op(q, *a, 8, 32, 0.0, i(3), i(3), *table[1:], **kw)   # noqa: E731
    assert at(k, k, cache, scale).shape == (10, 4, 64)
    for bad, needle in ((dict(kv_cache=meta(6, 2, 32, 2, 64)), "float8_e4m3fn or int8"),
                        (dict(kv_cache=meta(6, 2, 32, 2, 32, dtype=E4M3)), "must be .pages, 2"),
                        (dict(kv_cache=meta(6, 1, 32, 2, 64, dtype=INT8)), "must be .pages, 2"),
                        (dict(kv_scale=meta(6, 2, 5, 2, dtype=FP32)), "kv_scale must be"),
                        (dict(kv_scale=meta(6, 2, 2, 2, dtype=BF16)), "kv_scale must be"),
                        (dict(kv_scale=meta(6, 2, 2, 1, dtype=FP32)), "kv_scale must be")):
        args = dict(kv_cache=cache, kv_scale=scale) | bad
        with pytest.raises(RuntimeError, match=needle):
            append_op(k, k, args["kv_cache"], args["kv_scale"], *table)
        with pytest.raises(RuntimeError, match=needle):
            at(k, k, args["kv_cache"], args["kv_scale"])
    with pytest.raises(RuntimeError, match="must be contiguous"):
        append_op(k, k, meta(6, 2, 2, 32, 64, dtype=E4M3).transpose(2, 3), scale, *table)
    with pytest.raises(RuntimeError, match="one shape and dtype"):
        append_op(k, k[:5], cache, scale, *table)
    with pytest.raises(RuntimeError, match="no gradients"):
        append_op(meta(10, 2, 64).requires_grad_(), k, cache, scale, *table)
    c = torch.zeros(4, 1, 64, dtype=BF16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        append_op(c, c, torch.zeros(1, 2, 32, 1, 64, dtype=INT8), torch.zeros(1, 2, 1, 1), *(torch.tensor([0, 4]),) * 4)


@pytest.mark.parametrize("change,code,needle", [
    (dict(struct_bytes=4), -2, "struct_bytes"), (dict(dtype=7), -2, "bf16, fp16 or fp32"), (dict(held=2), -2, "e4m3 or int8"),
    (dict(page_size=0), -2, "page_size"), (dict(block=12), -2, "whole blocks"), (dict(block=0), -2, "whole blocks"),
    (dict(batch=0), -2, "at least two element"), (dict(index_bytes=2), -2, "int32 or int64"), (dict(heads_k=17), -2, "head count"),
    (dict(dim=513), -2, "head dim"), (dict(dim=0), -2, "head dim"), (dict(num_pages=0), -2, "must not be empty"),
    (dict(total=-1), -2, "too many"), (dict(total=1 << 40), -2, "too many"), (dict(total=1 << 30, block=1), -2, "too many"),
    (dict(k=0x7F0000000001), -2, "not aligned"), (dict(kv_scale=0x7F0000000002), -2, "not aligned"),
    (dict(k=None), -1, "null"), (dict(page_ids=None), -1, "null"), (dict(kv_scale=None), -1, "null"),
])
def test_append_entry_point_refuses(change, code, needle):
    lib, at = cabi.load(), 0x7F0000000000
    a = cabi.HstuCacheAppendArgs(C.sizeof(cabi.HstuCacheAppendArgs), 0, 0, 32, 16, 2, 64, 8, 4, 0, 100, 10, 10, *(at,) * 9, None)
    for name, value in change.items():
        setattr(a, name, value)
    assert lib.hstu_cache_append(C.byref(a), None) == code and needle in lib.hstu_last_error().decode()
    assert lib.hstu_cache_append(None, None) == -1


@pytest.mark.parametrize("change,needle", [
    (dict(struct_bytes=4), "struct_bytes"), (dict(held=3), "e4m3 or int8"), (dict(block=5), "whole blocks"),
    (dict(window=-1), "window expect at least 0"), (dict(num_sink=-1), "num_sink expect"), (dict(mask_type=2), "takes no mask"),
    (dict(attn_bias=0x7F0000000000), "takes no attn_bias"), (dict(num_context=0x7F0000000000), "takes no num_context"),
    (dict(dim_v=64), "must equal dim_v"), (dict(num_pages=0), "must not be empty"),
    (dict(num_target=0x7F0000000000), "targetGroupSize must be greater"), (dict(num_page_ids=1 << 40), "too large"),
])
def test_paged_entry_point_refuses(change, needle):
    from tests.test_cabi_boundary import _args
    lib, at, n = cabi.load(), 0x7F0000000000, C.c_uint64()
    p = cabi.HstuPagedArgs(C.sizeof(cabi.HstuPagedArgs), 32, _args(), at, at, at, at, None, 10, 10)
    a = cabi.HstuPaged8Args(C.sizeof(cabi.HstuPaged8Args), 0, 16, 0, 0, 0, at, p)
    assert lib.hstu_paged_8bit_fwd_get_workspace_size(C.byref(a), C.byref(n)) == 0
    assert lib.hstu_paged_8bit_fwd(C.byref(a), None, 0, None) < 0
    for name, value in change.items():
        setattr(next(s for s in (a, a.paged, a.paged.base) if hasattr(s, name)), name, value)
    assert lib.hstu_paged_8bit_fwd_get_workspace_size(C.byref(a), C.byref(n)) == -2
    assert needle in lib.hstu_last_error().decode()


# ------------------------------------------------------------------------------------------------------- GPU
def make(cached, new, targets=None, hq=4, hk=2, d=64, dtype=BF16, held=E4M3, page=32, block=16, seed=0, index=torch.int64, spare=3):
    """A serving batch: users of `cached` rows, the last `new` of them new, with `targets` candidates; the cache holds what an
    earlier life of its pages left, and the rows in front of the new ones."""
    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    cached, new = np.asarray(cached), np.asarray(new)
    ts = np.asarray(targets) if targets is not None else np.zeros_like(cached)
    count = (cached + page - 1) // page
    pages, rows = int(count.sum()) + spare, int((new + ts).sum())
    rnd = lambda *s: (torch.randn(*s, generator=gen) * 0.5).to(dtype)   # noqa: E731
    off = lambda n: torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=index)   # noqa: E731
    x = torch.randn(pages, 2, page, hk, d, generator=gen) * torch.exp2(torch.arange(hk) % 4 - 2.0)[:, None]
    scale = torch.empty(pages, 2, page // block, hk)
    cache = torch.empty(x.shape, dtype=held)
    amax = x.unflatten(2, (-1, block)).abs().amax((3, 5))
    scale = torch.exp2(torch.ceil(torch.log2(amax / CO.MOST[held])))
    cache = CO.numbers((x.unflatten(2, (-1, block)) / scale[:, :, :, None, :, None]).flatten(2, 3), held)
    ids = rng.permutation(pages)[:pages - spare] if pages > spare else np.zeros(1, np.int64)   # (no user has a page)
    args = dict(q=rnd(rows, hq, d), k=rnd(rows, hk, d), v=rnd(rows, hk, d), kv_cache=cache, kv_scale=scale,
                max_seq_len=max(int((new + ts).max()), 1), max_seq_len_k=max(int((cached + ts).max()), 1), seq_offset=off(new + ts),
                seq_offset_k=off(cached + ts), page_offsets=off(count), page_ids=torch.tensor(ids, dtype=index),
                last_page_len=torch.tensor(np.where(count > 0, cached - (count - 1) * page, 0), dtype=index), alpha=d ** -0.5)
    if targets is not None:
        args |= dict(num_target=torch.tensor(ts, dtype=index), target_group_size=1)
    return args


TABLE = ("k", "v", "kv_cache", "kv_scale", "seq_offset", "page_offsets", "page_ids", "last_page_len")


def table(args, cuda=True):
    got = {n: args[n] for n in TABLE} | ({"num_target": args["num_target"]} if "num_target" in args else {})
    return {n: t.cuda() for n, t in got.items()} if cuda else got


def on_gpu(args):
    return {n: t.cuda() if torch.is_tensor(t) else t for n, t in args.items()}


def check_append(args, label=""):
    want_cache, want_scale = CO.append(**table(args, False))
    t = table(args)
    st = cabi.hstu_cache_append(**t, return_status=True)
    assert st == 0, label
    assert torch.equal(t["kv_scale"].cpu(), want_scale), label
    assert torch.equal(t["kv_cache"].cpu().view(torch.uint8), want_cache.view(torch.uint8)), label
    return t["kv_cache"], t["kv_scale"]


def check_paged(args, window=0, sink=0, label="", **kw):
    cu = on_gpu(args)
    want, tol = CO.paged(**cu, window=window, num_sink=sink)
    out, st = cabi.hstu_paged_8bit_forward(**cu, window=window, num_sink=sink, return_status=True, **kw)
    assert st == 0 and torch.isfinite(out.float()).all(), label
    far = (out.double() - want).abs() - tol - torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    assert (far <= 0).all(), (label, far.max().item(), (far > 0).float().mean().item())
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("d,page,block", [(64, 32, 16), (128, 128, 32), (8, 24, 8), (96, 64, 64), (20, 10, 5), (320, 16, 1)])
def test_append_bit_for_bit(dtype, held, d, page, block):
    cached = [1, 0, 130, 75, page, page + 1, 300, 2 * page]
    new = [1, 0, 130, 3, page, 1, 211, 0]
    args = make(cached, new, [3, 2, 0, 9, 1, 0, 5, 4], hk=3, hq=3, d=d, dtype=dtype, held=held, page=page, block=block, seed=d)
    check_append(args)
    # larger rows behind the ones a block holds: their scale grows, the old rows are rounded anew
    args["k"], args["v"] = args["k"] * 37, args["v"] * 0.01
    check_append(args)


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
def test_append_of_extreme_values(held):
    args = make([70, 40, 33], [70, 1, 20], dtype=BF16, held=held, seed=1)
    k, v = args["k"], args["v"]
    k[3, 0, 5], k[4, 1, 7], v[6, 0, 1] = float("inf"), float("-inf"), float("nan")
    k[16:32] = 0                                     # a block of zeros
    v[16:32] = float("nan")                          # and one of nothing finite
    k[40] = torch.finfo(BF16).max
    v[41] = 1e-38
    k[50, :, ::2] = 448 * 2.0 ** -3                  # on the border of a scale
    k[51, :, ::2] = 127 * 2.0 ** -5
    check_append(args)
    args["k"] = args["k"].float()
    args["v"] = args["v"].float() * 1e-4
    check_append(args)


@pytest.mark.gpu
def test_append_row_by_row_and_what_stays_untouched():
    args = make([50, 9], [0, 0], seed=2)
    t = table(args)
    cache, scale = t["kv_cache"], t["kv_scale"]
    for n in range(1, 40):                           # one row of each user a step, growing; pages were handed out beforehand
        step = make([50 + n, 9 + n], [1, 1], seed=100 + n, index=torch.int32 if n % 2 else torch.int64, spare=6)
        ids = torch.arange(8)[torch.randperm(8, generator=torch.Generator().manual_seed(3))]
        po = step["page_offsets"]
        per = [ids[:po[1]], ids[4:4 + po[2] - po[1]]]
        step["page_ids"] = torch.cat(per).to(po.dtype)
        if n == 1:
            cache = torch.zeros(9, 2, 32, 2, 64, dtype=E4M3)
            scale = torch.full((9, 2, 2, 2), 2.0 ** -20)
        step["kv_cache"], step["kv_scale"] = cache.cpu(), scale.cpu()
        step["k"], step["v"] = step["k"] * 1.2 ** n, step["v"] * 1.2 ** n
        cache, scale = check_append(step, n)


@pytest.mark.gpu
def test_append_flags_what_does_not_fit_and_writes_nothing_there():
    args = make([60, 45, 100], [10, 5, 30], seed=3)
    clean = CO.append(**table(args, False))
    first = args["page_ids"][args["page_offsets"][0]:args["page_offsets"][1]].tolist()
    for name, change, bit in (("last_page_len", torch.tensor([40, 0, 0]), cabi.ST_BAD_PAGES),      # beyond the page
                              ("page_ids", torch.tensor([0, 10 ** 6, 0, 0, 0, 0, 0, 0]), cabi.ST_BAD_PAGES),
                              ("page_ids", torch.tensor([0, -10 ** 6, 0, 0, 0, 0, 0, 0]), cabi.ST_BAD_PAGES),
                              ("seq_offset", torch.tensor([0, 70, 0, 0]), cabi.ST_BAD_OFFSETS | cabi.ST_BAD_PAGES),
                              ("page_offsets", torch.tensor([0, 10 ** 6, 0, 0]), cabi.ST_BAD_PAGES)):
        t = table(args | {name: args[name] + change})
        st = cabi.hstu_cache_append(**t, return_status=True)
        assert st & bit and not st & ~(bit | cabi.ST_BAD_PAGES | cabi.ST_BAD_OFFSETS), name
        if name == "last_page_len":                  # the other users' rows are written all the same
            got = t["kv_cache"].cpu().view(torch.uint8)
            others = [p for p in range(got.shape[0]) if p not in first]
            assert torch.equal(got[others], clean[0].view(torch.uint8)[others])
            assert torch.equal(got[first], args["kv_cache"].view(torch.uint8)[first])
    t = table(args | dict(num_target=torch.tensor([11, 0, 0])))
    assert cabi.hstu_cache_append(**t, return_status=True) & cabi.ST_BAD_CTX_TARGET
    check_append(args)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,held", [(BF16, E4M3), (FP16, INT8), (BF16, INT8), (FP16, E4M3), (FP32, E4M3), (FP32, INT8)])
@pytest.mark.parametrize("d,page,block", [(64, 32, 16), (128, 128, 32), (128, 64, 8), (96, 64, 64), (32, 256, 128), (16, 24, 3), (256, 16, 16)])
@pytest.mark.parametrize("window,sink", [(0, 0), (50, 0), (100, 70)])
def test_paged_types_and_layouts(dtype, held, d, page, block, window, sink):
    args = make([1, 130, 75, 300, 513, 64], [1, 1, 20, 3, 1, 64], [3, 0, 9, 80, 0, 1], 4, 2, d, dtype, held, page, block, seed=d + block)
    check_paged(args, window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (8, 1), (16, 2), (6, 3)])
@pytest.mark.parametrize("new", [1, 2, 5, 17, 70])
def test_paged_heads_and_rows(hq, hk, new):
    cached = [new, 90, 200 + new, 640, 71]
    args = make(cached, [new] * 5, None, hq, hk, 128, BF16, E4M3, 64, 32, seed=hq + new)
    check_paged(args)
    check_paged(args, 66, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 1, 63, 64, 65, 1000])
@pytest.mark.parametrize("sink", [0, 1, 64, 65, 700])
def test_paged_borders(window, sink):
    args = make([640, 257, 1, 64, 65, 127], [1, 2, 1, 1, 1, 3], None, 2, 2, 64, seed=window + sink)
    check_paged(args, window, sink if window else 0)
    args = make([640, 257, 1, 64, 65, 127], [1, 2, 1, 1, 1, 3], [2, 70, 1, 0, 5, 40], 2, 2, 64, page=64, seed=window + sink)
    check_paged(args, window, sink if window else 0)


@pytest.mark.gpu
def test_paged_long_few_and_many_short():
    args = make([20000, 13, 8191], [1, 1, 1], None, 4, 4, 128, BF16, E4M3, 128, 64, seed=1)
    check_paged(args)
    check_paged(args, 4096, 16)
    args = make([19000], [1], None, 1, 1, 64, FP16, INT8, 32, 32, seed=2)
    check_paged(args)
    rng = np.random.default_rng(3)
    cached = rng.integers(1, 60, 1500)
    args = make(cached, np.minimum(cached, rng.integers(1, 4, 1500)), rng.integers(0, 9, 1500), 2, 2, 64, seed=4)
    check_paged(args)


@pytest.mark.gpu
def test_paged_empty_users_and_nothing_cached():
    # (no rows at all; targets only; the first event of a user)
    args = make([0, 0, 5, 40, 0], [0, 0, 5, 0, 0], [0, 4, 0, 3, 1], 2, 2, 64, seed=5)
    check_paged(args)
    check_paged(args, 3, 1)
    args = make([0, 0], [0, 0], [2, 1], 2, 2, 128, seed=6)
    check_paged(args)


@pytest.mark.gpu
@pytest.mark.parametrize("new,d", [(1, 128), (40, 64)])
def test_paged_reads_nothing_behind_a_row_or_beside_a_window(new, d):
    """Rows behind a user's last one, pages of nobody and a workspace full of NaN change nothing; nor do keys and values that no
    row of the user sees, where whole tiles of 64 keys lie outside of its window."""
    args = make([200, 77, 640], [new] * 3, None, 2, 2, d, seed=7, page=64, block=32)
    a = check_paged(args)
    w = check_paged(args, 64, 3)
    nan = CO.numbers(torch.tensor(float("nan")), E4M3)
    dirty = args | dict(kv_cache=args["kv_cache"].clone(), kv_scale=args["kv_scale"].clone())
    used = torch.zeros(dirty["kv_cache"].shape[0], 64, dtype=torch.bool)
    for b, n in enumerate((200, 77, 640)):
        for j in range(n):
            used[int(args["page_ids"][int(args["page_offsets"][b]) + j // 64]), j % 64] = True
    raw = dirty["kv_cache"].view(torch.uint8)
    raw.permute(0, 2, 1, 3, 4)[~used] = nan.view(torch.uint8)
    blocks = ~used.unflatten(1, (-1, 32)).any(2)
    dirty["kv_scale"].permute(0, 2, 1, 3)[blocks] = float("nan")
    out = cabi.hstu_paged_8bit_forward(**on_gpu(dirty), workspace_fill=0xFF)
    assert torch.equal(out, a)
    for j in range(64, 640 - new - 192):             # the third user's keys between the sinks and the window
        raw[int(args["page_ids"][int(args["page_offsets"][2]) + j // 64]), :, j % 64] = nan.view(torch.uint8)
    out = cabi.hstu_paged_8bit_forward(**on_gpu(dirty), window=64, num_sink=3, workspace_fill=0xFF)
    assert torch.equal(out, w)


@pytest.mark.gpu
def test_paged_flags_a_bad_table():
    args = make([60, 45, 100], [10, 1, 30], seed=8)
    for name, change in (("last_page_len", torch.tensor([3, 0, 0])), ("page_ids", torch.tensor([0, 10 ** 6, 0, 0, 0, 0, 0, 0])),
                         ("page_ids", torch.tensor([0, 0, 0, 0, 0, 0, -10 ** 6, 0])), ("page_offsets", torch.tensor([0, 1, 1, 1]))):
        for window in (0, 20):
            _, st = cabi.hstu_paged_8bit_forward(**on_gpu(args | {name: args[name] + change}), window=window, return_status=True)
            assert st & cabi.ST_BAD_PAGES, name
    _, st = cabi.hstu_paged_8bit_forward(**on_gpu(args | dict(seq_offset_k=torch.tensor([0, 60, 50, 205]))), return_status=True)
    assert st & cabi.ST_BAD_OFFSETS
    _, st = cabi.hstu_paged_8bit_forward(**on_gpu(args | dict(max_seq_len_k=64)), return_status=True)
    assert st & cabi.ST_LEN_GT_MAX
    check_paged(args)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,held,new,window", [(BF16, E4M3, 1, 0), (FP16, INT8, 3, 100), (BF16, E4M3, 30, 90)])
def test_a_serving_step_of_both_operators(dtype, held, new, window):
    """Append, then attend, through the torch operators: eagerly, on a stream of its own, captured and replayed on new rows; and
    against hstu_paged over the same cache in 16 bits."""
    args = make([150, 33, 400], [new] * 3, [7, 0, 20], 4, 2, 64, dtype, held, 64, 32, seed=9)
    names = ("seq_offset", "seq_offset_k", "page_offsets", "page_ids", "last_page_len", "num_target")

    def step(t):
        append_op(t["k"], t["v"], t["kv_cache"], t["kv_scale"], t["seq_offset"], t["page_offsets"], t["page_ids"],
                  t["last_page_len"], t["num_target"])
        return paged_op(t["q"], t["k"], t["v"], t["kv_cache"], t["kv_scale"], t["max_seq_len"], t["max_seq_len_k"], 0.0,
                        *(t[n] for n in names), 1, t["alpha"], window, 2 if window else 0)

    def want(a):
        cache, scale = CO.append(**table(a, False))
        held_now = a | dict(kv_cache=cache, kv_scale=scale)
        return cache, CO.paged(**on_gpu(held_now), window=window, num_sink=2 if window else 0)

    def same(got, a, t):
        cache, (value, tol) = want(a)
        assert torch.equal(t["kv_cache"].cpu().view(torch.uint8), cache.view(torch.uint8))
        assert ((got.double() - value).abs() <= tol + 1e-7).all()

    t = on_gpu(args)
    same(step(t), args, t)
    side = torch.cuda.Stream()
    t = on_gpu(args)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = step(t)
    torch.cuda.current_stream().wait_stream(side)
    same(out, args, t)
    if not window and held == E4M3:
        value = t["kv_cache"].float().unflatten(2, (-1, 32)) * t["kv_scale"][:, :, :, None, :, None]
        plain = cabi.hstu_paged_forward(t["q"], t["k"], t["v"], value.flatten(2, 3).to(dtype), None, None, 0, t["max_seq_len"],
                                        t["max_seq_len_k"], 0.0, t["seq_offset"], t["seq_offset_k"], None, t["page_offsets"],
                                        t["page_ids"], t["last_page_len"], t["num_target"], 1, t["alpha"])
        tol = CO.paged(**t)[1]
        assert ((plain.double() - out.double()).abs() <= 2 * tol + 1e-7).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(t)
    moved = args | {n: args[n] * -1.5 for n in ("q", "k", "v")}
    moved |= dict(kv_cache=t["kv_cache"].cpu(), kv_scale=t["kv_scale"].cpu())
    for n in ("q", "k", "v"):
        t[n].copy_(moved[n])
    graph.replay()
    same(out, moved, t)


@pytest.mark.gpu
def test_same_bits_every_time():
    for new, targets in ((1, None), (20, [30, 3, 9])):
        args = on_gpu(make([600, 90, 3000], [new] * 3, targets, 4, 4, 128, page=64, block=32, seed=10))
        a = cabi.hstu_paged_8bit_forward(**args)
        assert all(torch.equal(a, cabi.hstu_paged_8bit_forward(**args)) for _ in range(3))


@pytest.mark.gpu
def test_tensors_that_start_anywhere():
    """Inputs cut out of larger tensors, so that they start where no vector load may."""
    args = make([130, 75], [1, 20], [3, 9], 4, 2, 64, seed=11)
    shifted = {}
    for n in ("q", "k", "v", "kv_cache"):
        flat = torch.empty(args[n].numel() + 1, dtype=args[n].dtype, device="cuda")
        flat[1:].view(torch.uint8 if n == "kv_cache" else args[n].dtype).copy_(
            args[n].flatten().view(torch.uint8 if n == "kv_cache" else args[n].dtype))
        shifted[n] = flat[1:].view(args[n].shape)
    want, tol = CO.paged(**on_gpu(args))
    out = cabi.hstu_paged_8bit_forward(**(on_gpu(args) | shifted))
    assert ((out.double() - want).abs() <= tol + 1e-9).all()
    cache, scale = CO.append(**table(args, False))
    t = table(args) | {n: shifted[n] for n in ("k", "v", "kv_cache")}
    assert cabi.hstu_cache_append(**t, return_status=True) == 0
    assert torch.equal(t["kv_cache"].cpu().view(torch.uint8), cache.view(torch.uint8)) and torch.equal(t["kv_scale"].cpu(), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("size", [1.0, 1e-3, 300.0])
def test_paged_small_numbers_and_uneven_scales(dtype, new, size):
    """Numbers below e4m3's normal range only, and scales that differ by 2^20 from block to block."""
    args = make([200, 77, 640], [new] * 3, None, 2, 2, 64, dtype, page=64, block=16, seed=12)
    raw = args["kv_cache"].view(torch.uint8)
    raw[:, 0] = (raw[:, 0] & 0x87)                   # keys: at most 7 * 2^-9
    raw[::2, 1] &= 0x87
    args["kv_scale"][:, 0] *= 64
    args["kv_scale"][:, 1] *= torch.exp2(torch.randint(-10, 11, args["kv_scale"][:, 1].shape, generator=torch.Generator().manual_seed(1)).float())
    args["q"] = args["q"] * size
    check_paged(args)
    check_paged(args, 100, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new", [1, 30])
def test_paged_keeps_what_is_not_finite(dtype, new):
    args = make([200, 77], [new] * 2, None, 2, 2, 64, dtype, page=64, block=32, seed=13)
    want, tol = CO.paged(**on_gpu(args))
    page = int(args["page_ids"][0])
    args["kv_cache"].view(torch.uint8)[page, 1, 3, 0, 5] = 0x7f      # a value: its column of head 0 of the first user
    args["kv_cache"].view(torch.uint8)[page, 0, 4, 1, 6] = 0xff      # a key: everything of head 1
    out = cabi.hstu_paged_8bit_forward(**on_gpu(args))
    assert out[:new, 0, 5].isnan().all() and out[:new, 1].isnan().all()
    out[:new, 0, 5], out[:new, 1] = 0, 0
    want[:new, 0, 5], want[:new, 1] = 0, 0
    assert ((out.double() - want).abs() <= tol + 1e-9).all()


MANY = 140        # users of 4 heads and more than 32 rows: their pages are unpacked for the kernel that many rows share


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,held", [(BF16, E4M3), (FP16, INT8), (BF16, INT8), (FP16, E4M3)])
@pytest.mark.parametrize("d,page,block", [(64, 64, 16), (64, 128, 128), (128, 64, 64)])
@pytest.mark.parametrize("window,sink", [(0, 0), (70, 5)])
def test_paged_many_users_of_many_rows(dtype, held, d, page, block, window, sink):
    rng = np.random.default_rng(21)
    cached = rng.integers(1, 400, MANY)
    cached[:4] = 1, 64, 65, 128
    new = np.minimum(cached, rng.integers(0, 50, MANY))
    new[5], cached[5] = 49, 399
    check_paged(make(cached, new, None, 4, 4, d, dtype, held, page, block, seed=22), window, sink)
    check_paged(make(cached, new, rng.integers(0, 40, MANY), 8, 4, d, dtype, held, page, block, seed=23, index=torch.int32), window, sink)


@pytest.mark.gpu
def test_paged_many_users_reads_nothing_behind_a_row_and_flags_bad_pages():
    rng = np.random.default_rng(24)
    cached = rng.integers(60, 300, MANY)
    args = make(cached, np.full(MANY, 40), rng.integers(0, 9, MANY), 4, 4, 64, page=64, block=32, seed=25)
    a, w = check_paged(args), check_paged(args, 50, 3)
    nan = CO.numbers(torch.tensor(float("nan")), E4M3).view(torch.uint8)
    dirty = args | dict(kv_cache=args["kv_cache"].clone(), kv_scale=args["kv_scale"].clone())
    raw, used = dirty["kv_cache"].view(torch.uint8), torch.zeros(dirty["kv_cache"].shape[0], 64, dtype=torch.bool)
    for b, n in enumerate(cached):
        for j in range(0, int(n), 64):
            used[int(args["page_ids"][int(args["page_offsets"][b]) + j // 64]), :int(n) - j] = True
    raw.permute(0, 2, 1, 3, 4)[~used] = nan
    dirty["kv_scale"].permute(0, 2, 1, 3)[~used.unflatten(1, (-1, 32)).any(2)] = float("nan")
    assert torch.equal(cabi.hstu_paged_8bit_forward(**on_gpu(dirty), workspace_fill=0xFF), a)
    assert torch.equal(cabi.hstu_paged_8bit_forward(**on_gpu(dirty), window=50, num_sink=3, workspace_fill=0xFF), w)
    # a page that is not there: flagged, and every other user's rows as they were
    for bad in (10 ** 6, -1, -2 ** 40):
        ids = args["page_ids"].clone()
        ids[int(args["page_offsets"][7])] = bad
        for window, good in ((0, a), (50, w)):
            out, st = cabi.hstu_paged_8bit_forward(**on_gpu(args | dict(page_ids=ids)), window=window, num_sink=3 if window else 0, return_status=True)
            assert st & cabi.ST_BAD_PAGES
            here = torch.ones(out.shape[0], dtype=torch.bool, device="cuda")
            here[int(args["seq_offset"][7]):int(args["seq_offset"][8])] = False
            assert torch.equal(out[here], good[here])
    for name, change in (("last_page_len", 70), ("page_offsets", 1)):
        wrong = args[name].clone()
        wrong[3] += change
        _, st = cabi.hstu_paged_8bit_forward(**on_gpu(args | {name: wrong}), return_status=True)
        assert st & cabi.ST_BAD_PAGES, name


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 16])
@pytest.mark.parametrize("d,hq,hk", [(64, 4, 2), (128, 2, 2), (96, 3, 3)])
def test_paged_groups_of_targets(group, d, hq, hk):
    args = make([700, 77, 0, 1300], [20, 1, 0, 0], [30, 7, 5, 64], hq, hk, d, page=64, block=32, seed=26) | dict(target_group_size=group)
    check_paged(args)
    check_paged(args, 100, 17)
    rng = np.random.default_rng(27)
    cached = rng.integers(1, 200, MANY)
    args = make(cached, np.minimum(cached, 30), rng.integers(1, 40, MANY), 4, 4, d, FP16, INT8, 64, 32, seed=28) | dict(target_group_size=group)
    check_paged(args)
    check_paged(args, 33, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sink", [(0, 0), (5000, 64), (1, 0)])
def test_paged_long_histories_of_few_users_with_targets(window, sink):
    """Split over the keys, and over the rows."""
    check_paged(make([15000, 130], [200, 3], [150, 9], 2, 1, 128, BF16, E4M3, 128, 64, seed=29), window, sink)
    check_paged(make([15000], [0], [300], 1, 1, 64, FP16, INT8, 32, 16, seed=30), window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("users,new", [(3, 1), (3, 20), (MANY, 40)])
def test_paged_on_two_streams_and_captured(users, new):
    """Two calls at once on streams of their own; a captured step of both operators, replayed with other contents."""
    rng = np.random.default_rng(31)
    cached = rng.integers(new, 500, users)
    args = on_gpu(make(cached, np.full(users, new), None, 4, 4, 64, page=64, block=32, seed=32))
    other = on_gpu(make(cached + 1, np.full(users, new), None, 4, 4, 64, page=64, block=32, seed=33))
    names = ["q", "k", "v", "kv_cache", "kv_scale", "max_seq_len", "max_seq_len_k", "seq_offset", "seq_offset_k", "page_offsets", "page_ids",
             "last_page_len", "alpha"]
    call = lambda a: paged_op(**{n: a[n] for n in names}, window=99, num_sink=4)   # noqa: E731
    want, want_other = call(args), call(other)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            got.append((call(args), want))
        with torch.cuda.stream(s2):
            got.append((call(other), want_other))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append_op(**{n: args[n] for n in TABLE})
        out = call(args)
    args["k"].mul_(1.5), args["q"].mul_(0.5)
    twin = args | {n: args[n].clone() for n in ("kv_cache", "kv_scale")}
    append_op(**{n: twin[n] for n in TABLE})
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(args["kv_cache"].view(torch.uint8), twin["kv_cache"].view(torch.uint8)) and torch.equal(out, call(twin))


@pytest.mark.gpu
@pytest.mark.parametrize("users,new,targets", [(3, 1, None), (300, 1, None), (3, 20, None), (300, 5, 9)])
def test_paged_a_loose_bound_of_the_lengths(users, new, targets):
    rng = np.random.default_rng(34)
    cached = rng.integers(new, 150, users)
    args = make(cached, np.full(users, new), None if targets is None else np.full(users, targets), 2, 1, 64, seed=35)
    check_paged(args | dict(max_seq_len_k=20480))
    check_paged(args | dict(max_seq_len_k=20480), 20, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,held", [(BF16, E4M3), (FP16, INT8), (FP16, E4M3)])
@pytest.mark.parametrize("hk,d,page,block", [(4, 64, 64, 32), (5, 64, 32, 32), (1, 256, 24, 8), (16, 16, 10, 5), (3, 128, 16, 1), (4, 64, 64, 64)])
def test_append_histories(dtype, held, hk, d, page, block):
    """Rows that fill a warp's columns, blocks that are mostly full: with infinities, NaN and blocks that grow."""
    args = make([300, 33, 1, 129, 64], [300, 20, 1, 100, 0], [7, 0, 2, 0, 3], hk=hk, hq=hk, d=d, dtype=dtype, held=held, page=page, block=block, seed=50 + d)
    check_append(args)
    args["k"], args["v"] = args["k"] * 37, args["v"] * 0.01
    args["k"][3, 0, 5], args["v"][40, hk - 1, 7], args["v"][6, 0, 1], args["v"][70] = float("inf"), float("-inf"), float("nan"), float("nan")
    check_append(args)
    wide = {n: torch.zeros(args[n].shape[0], 2 * hk, d, dtype=dtype) for n in ("k", "v")}     # heads of a larger tensor
    for n in wide:
        wide[n][:, ::2] = args[n]
    cache, scale = CO.append(**table(args, False))
    t = table(args) | {n: x.cuda()[:, ::2] for n, x in wide.items()}
    append_op(**t)
    assert torch.equal(t["kv_cache"].cpu().view(torch.uint8), cache.view(torch.uint8)) and torch.equal(t["kv_scale"].cpu(), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("users,new,d", [(3, 1, 64), (3, 30, 64), (MANY, 40, 64), (3, 5, 320)])
def test_offsets_beyond_32_bits(users, new, d):
    """The same pages at the end of a cache of more than 4 GB: the same bits, from the attention and of the append."""
    rng = np.random.default_rng(51)
    cached = rng.integers(new, 300, users)
    args = on_gpu(make(cached, np.full(users, new), None, 4, 4, d, page=64, block=32, seed=52))
    small, shift = args["kv_cache"], (5 << 30) // (2 * 64 * 4 * d)
    far = args | dict(page_ids=args["page_ids"] + shift)
    far["kv_cache"] = torch.empty(shift + small.shape[0], *small.shape[1:], dtype=small.dtype, device="cuda")
    far["kv_scale"] = torch.empty(shift + small.shape[0], *args["kv_scale"].shape[1:], device="cuda")
    for n in ("kv_cache", "kv_scale"):
        far[n][shift:] = args[n]
    for window in (0, 70):
        assert torch.equal(cabi.hstu_paged_8bit_forward(**far, window=window), cabi.hstu_paged_8bit_forward(**args, window=window))
    for a in (args, far):
        assert cabi.hstu_cache_append(**{n: a[n] for n in TABLE}, return_status=True) == 0
    assert torch.equal(far["kv_cache"][shift:].view(torch.uint8), small.view(torch.uint8)) and torch.equal(far["kv_scale"][shift:], args["kv_scale"])


@pytest.mark.gpu
@pytest.mark.parametrize("held", [E4M3, INT8])
@pytest.mark.parametrize("new,d,targets", [(1, 64, None), (1, 128, None), (20, 64, None), (9, 128, [3, 8, 5, 1])])
def test_half_precision_loses_nothing_but_its_own_rounding(held, new, d, targets):
    """fp16 in place: P is held in two halves, 2^-22 of it off, so what the output is off is its own rounding - a tenth on top for
    SiLU's 2^-20 and for sums of 32 bits."""
    args = on_gpu(make([200, 77, 640, 31], [new] * 4, targets, 4, 2, d, FP16, held, 64, 16, seed=53))
    want, _ = CO.paged(**args)
    out = cabi.hstu_paged_8bit_forward(**args)
    off, least = ((x.double() - want).square().mean().sqrt().item() for x in (out, want.half()))
    assert off <= 1.1 * least, off / least
