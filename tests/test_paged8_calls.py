"""hstu_paged_8bit and hstu_cache_append: calls that the tests of values (tests/test_paged8.py) do not make."""
import ctypes as C

import numpy as np
import pytest
import torch

import ops_rec_b200 as ops_rec
from oracle import hstu_window_oracle as WO
from ops_rec_b200 import cabi
from tests.test_paged8 import BF16, E4M3, FP16, FP32, INT8, MANY, TABLE, make, meta, on_gpu

append_op = ops_rec.ascendc.attention.hstu_cache_append
paged_op = ops_rec.ascendc.attention.hstu_paged_8bit


def products(args, window, sink):
    """(outputs in 64 bits, the sum of the squares of the products P v behind each)."""
    off, off_k, po = (args[n].tolist() for n in ("seq_offset", "seq_offset_k", "page_offsets"))
    out, square = (torch.zeros(args["q"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    ratio = args["q"].shape[1] // args["k"].shape[1]
    value = args["kv_cache"].double().unflatten(2, (args["kv_scale"].shape[2], -1)) * args["kv_scale"].double()[:, :, :, None, :, None]
    value = value.flatten(2, 3)
    for b in range(len(off) - 1):
        t = int(args["num_target"][b]) if "num_target" in args else 0
        n, rows = off_k[b + 1] - off_k[b], slice(off[b], off[b + 1])
        mine = value[args["page_ids"][po[b]:po[b + 1]]].transpose(0, 1).flatten(1, 2)[:, :n - t]
        k, v = (torch.cat((mine[w], args[x][off[b + 1] - t:off[b + 1]].double())).transpose(0, 1).repeat_interleave(ratio, 0)
                for w, x in ((0, "k"), (1, "v")))
        see = WO.window_mask(off[b + 1] - off[b], n, t, args.get("target_group_size", 0), window, sink, "cuda")
        x = args["alpha"] * args["q"][rows].double().transpose(0, 1) @ k.transpose(1, 2)
        p = torch.where(see, x * torch.sigmoid(x) * args["silu_scale"], 0.0)
        out[rows], square[rows] = (p @ v).transpose(0, 1), (p ** 2 @ v ** 2).transpose(0, 1)
    return out, square


@pytest.mark.gpu
@pytest.mark.parametrize("users,new,targets,group,d,page", [
    (4, 1, None, 1, 64, 64), (4, 20, 5, 1, 128, 64), (MANY, 40, None, 1, 64, 64),          # in place; unpacked
    (4, 20, 5, 1, 64, 24), (4, 20, 9, 5, 128, 32), (4, 300, None, 1, 64, 32), (4, 7, 3, 1, 320, 16), (4, 9, 5, 2, 48, 20),   # staged
])
@pytest.mark.parametrize("window,sink", [(0, 0), (70, 4)])
def test_half_precision_keeps_its_bits_under_a_small_scale(users, new, targets, group, d, page, window, sink):
    """fp16 with a scale of 1 / 4096, whichever kernel a call goes to: P of the usual sizes times it would be below the type's normal
    range.  A value rounded once is u x / sqrt(3) off at most in the mean square (u: half a step), so an output y = sum(P v) of
    rounded P that is rounded itself u / sqrt(3) sqrt(sum((P v)^2) + y^2), and 2^-25 / sqrt(3) where it is subnormal; a tenth on top
    for the sample and for what 32 bits add.  (The cache's values are numbers of 8 bits times powers of two: exact in fp16.)"""
    rng = np.random.default_rng(61)
    cached = rng.integers(new, 500, users) if users > 4 else np.array([new + 200, new, 640, new + 31])
    args = make(cached, np.full(users, new), None if targets is None else np.full(users, targets), 4, 2, d, FP16, INT8, page, 4, seed=62)
    args = on_gpu(args | dict(silu_scale=1 / 4096, v=args["v"] * 8, kv_scale=args["kv_scale"] * 8))
    args["kv_scale"][:, 0] /= 8
    if targets is not None:
        args["target_group_size"] = group
    out, st = cabi.hstu_paged_8bit_forward(**args, window=window, num_sink=sink, return_status=True)
    want, square = products(args, window, sink)
    off = (out.double() - want).square().mean().sqrt()
    most = 1.1 * ((2.0 ** -22 * (square + want ** 2).mean() + 2.0 ** -50) / 3).sqrt()
    assert st == 0 and off <= most, (off / most).item()


def test_tolerance_follows_the_form_of_silu():
    """CPU: the 2^-12 |x| of tanh.approx is allowed where a kernel takes that form - bf16, heads of 64 and 128 - and nowhere else."""
    from oracle import hstu_cache_oracle as CO
    for dtype, d, tanh in ((BF16, 64, True), (BF16, 128, True), (BF16, 96, False), (BF16, 256, False), (FP16, 64, False), (FP32, 64, False)):
        args = make([40], [3], [2], 2, 1, d, dtype, E4M3, 32, 16, seed=63)
        tight, loose = (CO.paged(**args, tanh=form)[1] for form in (False, True))
        got = CO.paged(**args)[1]
        assert (tight < loose).any() and torch.equal(got, loose if tanh else tight), (dtype, d)


def workspace_size(batch, rows, hq, hk, d, max_seq_len_k, pages, page=32, window=0, dtype=0):
    """What a call of `rows` query rows of each user asks for (addresses that are not read)."""
    lib, at, n = cabi.load(), 0x7F0000000000, C.c_uint64()
    base = cabi.HstuJaggedArgs()
    base.struct_bytes, base.dtype, base.q, base.k, base.v, base.out = C.sizeof(base), dtype, at, at, at, at
    base.seq_offset_q, base.seq_offset_k, base.index_bytes, base.batch = at, at, 8, batch
    base.total_q = base.total_k = batch * rows
    base.heads_q, base.heads_k, base.dim_qk, base.dim_v = hq, hk, d, d
    base.max_seq_len_q, base.max_seq_len_k, base.alpha = rows, max_seq_len_k, 1.0
    p = cabi.HstuPagedArgs(C.sizeof(cabi.HstuPagedArgs), page, base, at, at, at, at, None, pages, pages)
    a = cabi.HstuPaged8Args(C.sizeof(cabi.HstuPaged8Args), 0, 16, window, 0, 0, at, p)
    cabi.check(lib.hstu_paged_8bit_fwd_get_workspace_size(C.byref(a), C.byref(n)))
    return n.value


@pytest.mark.parametrize("rows", [1, 8, 9, 80, 200])
@pytest.mark.parametrize("users,pages", [(4096, 16), (2048, 16), (300, 200), (4700, 2), (65535, 1), (1, 640), (40, 10)])
@pytest.mark.parametrize("max_seq_len_k", [512, 2128, 20480])
@pytest.mark.parametrize("window", [0, 1000])
def test_workspace_follows_what_can_be_split(rows, users, pages, max_seq_len_k, window):
    """Partial sums are of some 1200 CTAs' shares of the pages (8 of each of 148 SMs), twice that at most, and one share more per
    head - whatever the bound of the lengths: of 64 rows of 128 numbers in 32 bits, 32 KB each; and a counter per problem."""
    size = workspace_size(users, rows, 8, 8, 128, max_seq_len_k, users * pages, window=window)
    blocks = (rows + 63) // 64
    assert size <= (2 * 8 * 148 + 2 * 8 * blocks) * 64 * 128 * 4 + 4 * users * 8 * blocks + 4096


@pytest.mark.gpu
@pytest.mark.parametrize("new,targets,hq", [(1, None, 16), (9, None, 16), (3, 4, 16)])
@pytest.mark.parametrize("dtype,held", [(BF16, E4M3), (FP16, INT8)])
@pytest.mark.parametrize("window,sink", [(0, 0), (9000, 70)])
def test_a_few_long_histories_among_many(new, targets, hq, dtype, held, window, sink):
    """CTAs of more than 200 tiles, several for some of the users, whose partial sums lie in slots that go by their pages."""
    rng = np.random.default_rng(64)
    cached = np.maximum(rng.integers(1, 100, 600), new)
    cached[[0, 77, 300, 301, 599]] = 20000, 15001, 8192, 20001, 12345
    args = make(cached, np.full(600, new), None if targets is None else np.full(600, targets), hq, hq, 32, dtype, held, 64, 32, seed=65)
    from tests.test_paged8 import check_paged
    a = check_paged(args, window, sink)
    cu = on_gpu(args | dict(max_seq_len_k=20480))
    for _ in range(3):
        out = cabi.hstu_paged_8bit_forward(**cu, window=window, num_sink=sink, workspace_fill=0xFF)
        assert torch.equal(out, cabi.hstu_paged_8bit_forward(**cu, window=window, num_sink=sink))
    assert (out.double() - a.double()).abs().max() <= 2.0 ** -7 * a.double().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 9])
def test_pages_that_do_not_hold_a_long_history_are_flagged(new):
    """A table with fewer pages than the lengths say, where CTAs share a history and their slots go by the pages."""
    cached = np.full(600, 40)
    cached[[3, 500]] = 20000, 16000
    args = make(cached, np.full(600, new), None, 16, 16, 32, page=64, block=32, seed=66)
    good, st = cabi.hstu_paged_8bit_forward(**on_gpu(args), return_status=True)
    assert st == 0
    po = args["page_offsets"].clone()
    po[501:] -= 200                                  # user 500 lacks 200 pages; the users behind it read what is not theirs
    out, st = cabi.hstu_paged_8bit_forward(**on_gpu(args | dict(page_offsets=po)), return_status=True)
    assert st & cabi.ST_BAD_PAGES and torch.equal(out[:500 * new], good[:500 * new])
    po = args["page_offsets"].clone()
    po[4:] = torch.where(po[4:] > po[3] + 2, po[3] + 2, po[4:])
    out, st = cabi.hstu_paged_8bit_forward(**on_gpu(args | dict(page_offsets=po)), return_status=True)
    assert st & cabi.ST_BAD_PAGES and torch.equal(out[:3 * new], good[:3 * new])


def _meta_call(**grads):
    i = lambda n: meta(n, dtype=torch.int64)   # noqa: E731
    t = dict(q=meta(10, 4, 64), k=meta(10, 2, 64), v=meta(10, 2, 64), kv_cache=meta(6, 2, 32, 2, 64, dtype=E4M3), kv_scale=meta(6, 2, 2, 2, dtype=FP32))
    for n in grads:
        t[n].requires_grad_()
    return t, paged_op(**t, max_seq_len=8, max_seq_len_k=32, seq_offset=i(3), seq_offset_k=i(3), page_offsets=i(3), page_ids=i(6),
                       last_page_len=i(2))


@pytest.mark.parametrize("name", ["q", "k", "v", "kv_scale"])
def test_paged_refuses_a_backward_pass(name):
    """The output of queries that require gradients can be had; gradients through it cannot, and are not left out in silence."""
    t, out = _meta_call(**{name: True})
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="hstu_paged_8bit has no gradients"):
        out.sum().backward()
    with torch.no_grad():
        assert not _meta_call(**{name: True})[1].requires_grad
    assert not _meta_call()[1].requires_grad


@pytest.mark.gpu
def test_paged_of_queries_that_require_gradients():
    args = on_gpu(make([60, 45], [1, 3], None, seed=67))
    want = paged_op(**{n: args[n] for n in ("q", *TABLE)}, **{n: args[n] for n in ("max_seq_len", "max_seq_len_k", "seq_offset_k", "alpha")})
    args["q"].requires_grad_()
    out = paged_op(**{n: args[n] for n in ("q", *TABLE)}, **{n: args[n] for n in ("max_seq_len", "max_seq_len_k", "seq_offset_k", "alpha")})
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="has no gradients"):
        (out.float().sum() + args["q"].float().sum()).backward()


def _meta_append(**change):
    i = lambda n: meta(n, dtype=torch.int64)   # noqa: E731
    t = dict(k=meta(10, 2, 64), v=meta(10, 2, 64), kv_cache=meta(6, 2, 32, 2, 64, dtype=E4M3), kv_scale=meta(6, 2, 2, 2, dtype=FP32),
             seq_offset=i(3), page_offsets=i(3), page_ids=i(6), last_page_len=i(2)) | change
    append_op(**t)
    return t


def test_append_counts_up_the_versions_of_what_it_writes():
    t = _meta_append()
    assert [t[n]._version for n in ("kv_cache", "kv_scale", "k", "v", "page_ids")] == [1, 1, 0, 0, 0]
    with torch.no_grad():
        append_op(**t)
    assert t["kv_cache"]._version == 2 and t["kv_scale"]._version == 2
    # a graph that saved the scales finds out
    leaf = meta(6, 2, 2, 2, dtype=FP32).requires_grad_()
    product = leaf * t["kv_scale"]
    append_op(**t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        t = _meta_append()
    _meta_append(kv_cache=t["kv_cache"], kv_scale=t["kv_scale"])   # (tensors of inference mode have no version)
    with pytest.raises(RuntimeError, match="no gradients"):
        _meta_append(kv_scale=meta(6, 2, 2, 2, dtype=FP32).requires_grad_())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("users,new", [(4, 1), (4, 20), (MANY, 40)])
@pytest.mark.parametrize("window,sink", [(60, 3), (1000, 0)])
def test_a_model_is_served_with_the_scale_it_was_trained_with(dtype, users, new, window, sink):
    """The last rows of hstu_window over whole sequences, with its scale of 1 / max_seq_len, are those of hstu_paged_8bit over the same
    keys and values - what the cache holds, exact in 16 bits - if that scale is passed: 0 would mean 1 / (the longest query here)."""
    from oracle import hstu_cache_oracle as CO
    rng = np.random.default_rng(68)
    cached = rng.integers(new, 500, users)
    args = on_gpu(make(cached, np.full(users, new), None, 4, 2, 64, dtype, INT8, 64, 4, seed=69))
    value = (args["kv_cache"].float().unflatten(2, (-1, 4)) * args["kv_scale"][:, :, :, None, :, None]).flatten(2, 3)
    po = args["page_offsets"].tolist()
    k, v = (torch.cat([value[args["page_ids"][po[b]:po[b + 1]], w].flatten(0, 1)[:n] for b, n in enumerate(cached.tolist())]).to(dtype)
            for w in (0, 1))
    off = args["seq_offset_k"]
    q = torch.randn(int(off[-1]), 4, 64, device="cuda").to(dtype)
    last = torch.cat([torch.arange(int(e) - new, int(e)) for e in off[1:]]).cuda()
    q[last] = args["q"]
    trained = ops_rec.ascendc.attention.hstu_window(q, k, v, window, sink, 512, 0, 0.0, off, None, None, 0, args["alpha"])[last]
    served = paged_op(**{n: t for n, t in args.items()}, silu_scale=1 / 512, window=window, num_sink=sink)
    _, tol = CO.paged(**args, silu_scale=1 / 512, window=window, num_sink=sink)
    assert ((trained.double() - served.double()).abs() <= 2 * tol + 1e-7).all()
    if new > 1:
        other = paged_op(**args, window=window, num_sink=sink)   # (1 / new)
        assert (other.double() - served.double() * 512 / new).abs().max() <= 2.0 ** -6 * other.double().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [3.0, -0.7, 1.0, 2.0 ** -14])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_scales_of_the_call(scale, dtype):
    """Above 1, below 0 and small, on every path and of hstu_window."""
    from tests.test_paged8 import check_paged
    for users, new, targets, d, page in ((3, 1, None, 64, 32), (3, 20, 5, 64, 32), (MANY, 40, 3, 64, 64), (3, 20, 5, 64, 24), (3, 5, None, 160, 16)):
        rng = np.random.default_rng(70)
        cached = rng.integers(new, 200, users)
        args = make(cached, np.full(users, new), None if targets is None else np.full(users, targets), 4, 2, d, dtype, INT8, page, 8, seed=71)
        for window in (0, 50):
            check_paged(args | dict(silu_scale=scale), window, 2, label=(users, new, d, page))
    from tests import test_window as W
    args, grad = W.make([300, 77], 2, 2, 64, dtype=dtype, seed=72)
    W.check(args | dict(silu_scale=scale), grad, 50, 2)
