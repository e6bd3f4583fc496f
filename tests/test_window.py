"""hstu_window: the mask algebra of the kernels against its definition (CPU), refusals (CPU), and the operator and its
gradients against 64 bits with tolerances that count roundings (GPU; oracle/hstu_window_oracle.py derives them)."""
import ctypes as C

import numpy as np
import pytest
import torch

import ops_rec_b200 as ops_rec
from oracle import hstu_window_oracle as WO
from ops_rec_b200 import cabi

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
op = ops_rec.ascendc.attention.hstu_window


# ------------------------------------------------------------------------------------------------------- mask (CPU)
def _mask_cases():
    rng = np.random.default_rng(5)
    cases = [(1, 1, 0, 0, 1, 0), (70, 70, 0, 0, 1, 0), (70, 70, 0, 0, 1, 70), (70, 70, 0, 0, 1 << 30, 0), (300, 300, 0, 0, 40, 3),
             (300, 300, 20, 1, 40, 3), (300, 300, 20, 7, 1, 0), (9, 300, 5, 2, 33, 70), (300, 9, 0, 0, 4, 1), (300, 9, 4, 1, 4, 1),
             (40, 40, 40, 3, 5, 2), (1, 20000, 0, 0, 512, 4), (33, 1, 1, 1, 2, 2)]
    for _ in range(60):
        lk = int(rng.integers(1, 400))
        lq = int(rng.choice([lk, lk, rng.integers(1, 400)]))
        tgt = int(rng.choice([0, rng.integers(0, min(lq, lk) + 1)]))
        cases.append((lq, lk, tgt, int(rng.choice([0, 1, 1, 3])), int(rng.choice([1, 2, 63, 64, 65, rng.integers(1, 300)])),
                      int(rng.choice([0, 1, 4, 64, 65, rng.integers(0, 300)]))))
    return cases


@pytest.mark.parametrize("lq,lk,tgt,group,window,sink", _mask_cases())
def test_mask_algebra(lq, lk, tgt, group, window, sink):
    want = WO.window_mask(lq, lk, tgt, group, window, sink).numpy()
    for rows, bn in ((128, 64), (128, 128), (32, 64), (32, 32), (64, 32), (16, 16)):
        for r0 in {0, (lq - 1) // rows // 2 * rows, (lq - 1) // rows * rows, (lq + rows) // rows * rows}:
            see, visits, full, asked = cabi.debug_window(lq, lk, tgt, group, window, sink, r0, rows, bn)
            assert np.array_equal(see, want)
            mine = want[r0:r0 + rows]
            if mine.size == 0:
                assert not visits.any()
                continue
            assert visits.max(initial=0) <= 1
            seen = mine.any(0)
            assert (visits[seen] == 1).all() and asked[seen].all()
            assert mine[:, full].all()
            # what is visited in vain: the ends of two or three tiles, the corner of the q-tile, other groups of targets
            wasted = visits.sum() - seen.sum()
            assert wasted <= 2 * bn + rows + (bn if sink else 0) + tgt


def test_window_of_everything_is_the_causal_mask():
    for args in ((50, 50, 0, 0), (50, 50, 9, 1), (20, 50, 9, 4)):
        see = cabi.debug_window(*args, 1 << 30, 0, 0, 128, 64)[0]
        assert np.array_equal(see, cabi.debug_mask(args[0], args[1], 0, args[2], args[3]))


# ------------------------------------------------------------------------------------------------------- refusals (CPU)
def meta(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def _block(**kw):
    from tests.test_cabi_boundary import _args
    return _args(**kw)


@pytest.mark.parametrize("change,needle", [
    (dict(window=0), "window expect at least 1"), (dict(window=-5), "window expect at least 1"),
    (dict(num_sink=-1), "num_sink expect at least 0"), (dict(struct_bytes=8), "struct_bytes"),
    (dict(mask_type=2), "takes no mask"), (dict(attn_bias=0x7F0000000000), "takes no attn_bias"),
    (dict(num_context=0x7F0000000000), "takes no num_context"), (dict(max_seq_len_q=0), "maxSeqLen expect"),
    (dict(heads_q=17), "head count"), (dict(dim_v=24), "multiple of 16"),
])
def test_c_entry_points_refuse(change, needle):
    lib, n = cabi.load(), C.c_uint64()
    for cls, size, inner in ((cabi.HstuWindowArgs, lib.hstu_window_fwd_get_workspace_size, lambda a: a.fwd),
                             (cabi.HstuWindowBwdArgs, lib.hstu_window_bwd_get_workspace_size, lambda a: a.bwd.fwd)):
        a = cls(C.sizeof(cls), 64, 4, 0)
        if cls is cabi.HstuWindowArgs:
            a.fwd = _block()
        else:
            a.bwd = cabi.HstuJaggedBwdArgs(C.sizeof(cabi.HstuJaggedBwdArgs), 0, _block())
        assert size(C.byref(a), C.byref(n)) == 0 and n.value > 0
        for name, value in change.items():
            setattr(a if hasattr(a, name) else inner(a), name, value)
        assert size(C.byref(a), C.byref(n)) == -2 and needle in lib.hstu_last_error().decode()
    assert lib.hstu_window_fwd(None, None, 0, None) == -1 and lib.hstu_window_bwd(None, None, 0, None) == -1
    a = cabi.HstuWindowArgs(C.sizeof(cabi.HstuWindowArgs), 64, 4, 0, _block())
    assert lib.hstu_window_fwd(C.byref(a), None, 0, None) == -3
    b = cabi.HstuJaggedBwdArgs(C.sizeof(cabi.HstuJaggedBwdArgs), 0, _block())
    b.grad_bias = 0x7F0000000000
    a = cabi.HstuWindowBwdArgs(C.sizeof(cabi.HstuWindowBwdArgs), 64, 4, 0, b)
    assert lib.hstu_window_bwd_get_workspace_size(C.byref(a), C.byref(n)) == -2


def test_operator_on_meta_and_cpu_tensors():
    q, k, v = meta(10, 4, 64), meta(12, 2, 64), meta(12, 2, 32)
    off = torch.empty(3, dtype=torch.int64, device="meta")
    assert op(q, k, v, 5, 1, 16, 16, 0.0, off, off).shape == (10, 4, 32)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = op(*leaves, 5, 1, 16, 16, 0.0, off, off)
    assert [g.shape for g in torch.autograd.grad(out, leaves, torch.empty_like(out))] == [t.shape for t in leaves]
    with torch.no_grad():
        assert not op(*leaves, 5, 1, 16, 16, 0.0, off, off).requires_grad
    c = torch.zeros(4, 1, 64, dtype=BF16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        op(c, c, c, 5, 0, 4, 0, 0.0, torch.tensor([0, 4]))
    with pytest.raises(cabi.HstuError, match="no CPU implementation"):
        cabi.hstu_window_forward(c, c, c, 5, 0, 4, seq_offset=torch.tensor([0, 4]))


# ------------------------------------------------------------------------------------------------------- values (GPU)
def make(lens, hq=2, hk=None, dq=64, dv=None, dtype=BF16, tgt=0, group=1, delta=None, seed=0, index=torch.int64, max_seq_len=None):
    """Inputs of sequences of these lengths (keys); `delta` takes rows off the front of the queries (or adds some)."""
    gen = torch.Generator().manual_seed(seed)
    lens = list(lens)
    lq = [max(0, n - delta) if delta and n else n for n in lens] if delta is not None else lens
    rnd = lambda *s: (torch.randn(*s, generator=gen) * 0.5).to(dtype).cuda()   # noqa: E731
    off = lambda n: torch.tensor([0] + list(np.cumsum(n)), dtype=index).cuda()   # noqa: E731
    hk, dv = hk or hq, dv or dq
    args = dict(q=rnd(sum(lq), hq, dq), k=rnd(sum(lens), hk, dq), v=rnd(sum(lens), hk, dv), seq_offset=off(lq),
                max_seq_len=max_seq_len or max(max(lq), 1), alpha=dq ** -0.5)
    if delta is not None:
        args |= dict(seq_offset_k=off(lens), max_seq_len_k=max(max(lens), 1))
    if tgt:
        t = [min(tgt, a, b) for a, b in zip(lq, lens)]
        args |= dict(num_target=torch.tensor(t, dtype=index).cuda(), target_group_size=group)
    return args, rnd(sum(lq), hq, dv)


def is_tanh(args):
    d = (args["q"].shape[2], args["v"].shape[2])
    return args["q"].dtype == BF16 and d in ((64, 64), (128, 128))


def check(args, grad, window, sink, label="", flags=0):
    want = WO.hstu_window(window=window, sink=sink, grad=grad, tanh=is_tanh(args) and not flags, **args)
    out, st = cabi.hstu_window_forward(window=window, num_sink=sink, flags=flags, return_status=True, **args)
    grads, st2 = cabi.hstu_window_backward(grad, window=window, num_sink=sink, flags=flags, return_status=True, **args)
    assert st == 0 and st2 == 0, label
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        value, tol = want[name]
        assert got.shape == value.shape and torch.isfinite(got.float()).all(), (label, name)
        # (an output below the type's normal range is rounded to a multiple of its smallest step)
        far = (got.double() - value).abs() - tol - torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
        assert (far <= 0).all(), (label, name, far.max().item(), (far > 0).float().mean().item())
    return out, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dq,dv", [(64, 64), (128, 128), (32, 32), (64, 128), (96, 48), (20, 16), (160, 160)])
@pytest.mark.parametrize("window,sink", [(1, 0), (50, 4), (128, 0), (300, 130)])
def test_types_and_widths(dtype, dq, dv, window, sink):
    if dq == 160 and dtype != FP16:
        pytest.skip("one type on the kernels for wide heads")
    args, grad = make([130, 1, 0, 64, 517, 255], 4, 2, dq, dv, dtype, tgt=9, seed=dq + window)
    check(args, grad, window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (FP32, 64)])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 127, 128, 129, 1000])
@pytest.mark.parametrize("sink", [0, 1, 63, 64, 65, 200])
def test_borders_of_window_and_sinks(dtype, d, window, sink):
    args, grad = make([640, 257], 2, 2, d, dtype=dtype, seed=window + sink)
    check(args, grad, window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tgt,group", [(1, 1), (40, 1), (150, 7), (600, 3), (20, 0)])
@pytest.mark.parametrize("window", [1, 30, 300])
def test_targets(dtype, tgt, group, window):
    args, grad = make([600, 300, 33, 1], 4, 1, 64, dtype=dtype, tgt=tgt, group=group, seed=tgt)
    check(args, grad, window, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (FP16, 128), (FP32, 32), (FP32, 20)])
@pytest.mark.parametrize("delta", [599, 300, 1, -200])
def test_rows_other_than_keys(dtype, d, delta):
    """Single-token rows against long keys, and rows in front of the first key, which see nothing."""
    args, grad = make([600, 450, 1], 2, 2, d, 16 if d == 20 else d, dtype, delta=delta, seed=3, index=torch.int32)
    out, (dq, _, _) = check(args, grad, 70, 3)
    if delta < 0:
        assert not out[:200].any() and not dq[:200].any()


@pytest.mark.gpu
def test_long_sequences_and_many():
    args, grad = make([4097, 3000], 2, 1, 128, seed=1)
    check(args, grad, 512, 16)
    lens = np.random.default_rng(0).integers(1, 90, 1500).tolist()
    args, grad = make(lens, 2, 2, 64, seed=2, tgt=4)
    check(args, grad, 20, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_everything_in_the_window_is_the_jagged_operator(dtype):
    args, grad = make([300, 77, 512], 2, 2, 64, dtype=dtype, tgt=8, seed=4)
    w, _ = check(args, grad, 1 << 30, 0)
    j = cabi.hstu_jagged_forward(**args)
    tol = WO.hstu_window(window=0, tanh=is_tanh(args), **args)["out"][1]
    assert ((w.double() - j.double()).abs() <= 2 * tol + 1e-12).all()


@pytest.mark.gpu
def test_same_bits_every_time_and_forced_cuda_cores():
    args, grad = make([900, 31], 2, 2, 64, seed=6)
    a, ga = check(args, grad, 100, 9)
    b, gb = check(args, grad, 100, 9)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(ga, gb))
    check(args, grad, 100, 9, flags=cabi.FLAG_FORCE_GENERIC)


@pytest.mark.gpu
def test_neighbours_do_not_leak_and_rows_behind_the_end_stay():
    """Every second sequence is full of NaN and Inf; the rows behind the last one are left as they were."""
    args, grad = make([200, 77, 300, 50], 2, 2, 64, seed=7)
    off = args["seq_offset"].tolist()
    clean = WO.hstu_window(window=60, sink=3, grad=grad, tanh=True, **args)
    for t in (args["q"], args["k"], args["v"], grad):
        t[off[1]:off[2]] = float("nan")
        t[off[3]:off[4]] = float("inf")
    out = cabi.hstu_window_forward(window=60, num_sink=3, **args)
    got = (out, *cabi.hstu_window_backward(grad, window=60, num_sink=3, **args))
    for name, g in zip(("out", "dq", "dk", "dv"), got):
        for a, b in ((0, 1), (2, 3)):
            value, tol = (t[off[a]:off[b]] for t in clean[name])
            assert ((g[off[a]:off[b]].double() - value).abs() <= tol + 1e-9).all(), name


@pytest.mark.gpu
def test_strides_streams_autograd_and_capture():
    args, grad = make([300, 129], 2, 2, 64, seed=8)
    call = lambda q, k, v: op(q, k, v, 90, 2, args["max_seq_len"], 0, 0.0, args["seq_offset"], None, None, 0, args["alpha"])   # noqa: E731
    want = WO.hstu_window(window=90, sink=2, grad=grad, tanh=True, **args)
    # q, k and v as slices of one projection, as a model has them
    mixed = torch.cat([args[n] for n in "qkv"], 1).requires_grad_()
    out = call(mixed[:, :2], mixed[:, 2:4], mixed[:, 4:])
    g, = torch.autograd.grad(out, mixed, grad)
    for name, got in (("out", out), ("dq", g[:, :2]), ("dk", g[:, 2:4]), ("dv", g[:, 4:])):
        assert ((got.double() - want[name][0]).abs() <= want[name][1] + 1e-12).all(), name
    # a stream of its own, then captured and replayed on new inputs
    leaves = [args[n].clone().requires_grad_() for n in "qkv"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(call(*leaves), leaves, grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(*leaves)
        grads = torch.autograd.grad(held, leaves, grad)
    with torch.no_grad():
        for t in leaves:
            t.mul_(-0.5)
    graph.replay()
    again = {n: t.detach() for n, t in zip("qkv", leaves)}
    want = WO.hstu_window(window=90, sink=2, grad=grad, tanh=True, **(args | again))
    for name, got in zip(("out", "dq", "dk", "dv"), (held, *grads)):
        assert ((got.double() - want[name][0]).abs() <= want[name][1] + 1e-12).all(), name


@pytest.mark.gpu
def test_gradients_against_differences():
    """fp32, the derivative along random directions: a central difference of the 64-bit operator has an error of h^2 times a
    third derivative (of order one here) and 1e-16 / h, both far below the operator's own 1e-5."""
    args, grad = make([60, 25], 2, 1, 32, dtype=FP32, tgt=5, seed=9)
    dq, dk, dv = cabi.hstu_window_backward(grad, window=12, num_sink=2, **args)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for name, g in (("q", dq), ("k", dk), ("v", dv)):
        way = torch.randn(g.shape, generator=gen, device="cuda", dtype=torch.float64)
        h, ends = 1e-4, []
        for sign in (1, -1):
            moved = {n: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for n, t in args.items()}
            moved[name] = moved[name] + sign * h * way
            ends.append((WO.hstu_window(window=12, sink=2, **moved)["out"][0] * grad.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        assert abs((g.double() * way).sum() - slope) <= 1e-5 * (g.double() * way).abs().sum(), name


@pytest.mark.gpu
def test_inconsistent_offsets_are_flagged():
    args, grad = make([100, 50], 2, 2, 64, seed=10)
    bad = args | dict(seq_offset=torch.tensor([0, 120, 100]).cuda())
    _, st = cabi.hstu_window_forward(window=10, return_status=True, **bad)
    assert st & cabi.ST_BAD_OFFSETS
    _, st = cabi.hstu_window_backward(grad, window=10, return_status=True, **(args | dict(max_seq_len=64)))
    assert st & cabi.ST_LEN_GT_MAX
    check(args, grad, 10, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dq,dv", [(64, 64), (128, 128), (96, 96), (20, 16), (17, 32)])
@pytest.mark.parametrize("delta", [None, 30])
def test_half_precision_keeps_its_bits_under_a_small_scale(dq, dv, delta):
    """fp16 with a scale of 1 / 4096: P and dS of the usual sizes times it would be below the type's normal range.  A value x that
    is rounded once is u x / sqrt(3) off at most in the mean square (u: half a step), so a result y = sum(p w) of rounded p that
    is rounded itself u / sqrt(3) sqrt(sum((p w)^2) + y^2), and 2^-25 / sqrt(3) where it is subnormal; a tenth on top for the sample
    and what 32 bits add."""
    args, grad = make([600, 300, 33], 2, 2, dq, dv, FP16, delta=delta, seed=41, max_seq_len=4096)
    args["v"], grad, alpha, scale = args["v"] * 8, grad * 8, args["alpha"], 1 / 4096
    out = cabi.hstu_window_forward(window=20, num_sink=2, **args)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *cabi.hstu_window_backward(grad, window=20, num_sink=2, **args))))
    want = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for n, t in got.items()}
    square = {n: torch.zeros_like(t) for n, t in want.items()}
    offq = args["seq_offset"].tolist()
    offk = args["seq_offset_k"].tolist() if "seq_offset_k" in args else offq
    for b in range(3):
        rows, keys = slice(offq[b], offq[b + 1]), slice(offk[b], offk[b + 1])
        q, g, k, v = (t.double().transpose(0, 1) for t in (args["q"][rows], grad[rows], args["k"][keys], args["v"][keys]))
        see = WO.window_mask(rows.stop - rows.start, keys.stop - keys.start, 0, 0, 20, 2, "cuda")
        x = alpha * q @ k.transpose(1, 2)
        sg = torch.sigmoid(x)
        p = torch.where(see, x * sg * scale, 0.0)
        ds = torch.where(see, g @ v.transpose(1, 2) * scale * alpha * sg * (1 + x * (1 - sg)), 0.0)
        for name, at, a, w in (("out", rows, p, v), ("dq", rows, ds, k), ("dk", keys, ds.transpose(1, 2), q), ("dv", keys, p.transpose(1, 2), g)):
            want[name][at], square[name][at] = (a @ w).transpose(0, 1), (a ** 2 @ w ** 2).transpose(0, 1)
    for name in got:
        off = (got[name].double() - want[name]).square().mean().sqrt()
        most = 1.1 * ((2.0 ** -22 * (square[name] + want[name] ** 2).mean() + 2.0 ** -50) / 3).sqrt()
        assert off <= most, (name, (off / most).item())
