"""hstu_window and hstu_paged_8bit in fp16 where a score, or dS of large gradients, lies beyond the type although what the scale
makes of it does not: against 64 bits, with the tolerances of oracle/hstu_window_oracle.py."""
import numpy as np
import pytest
import torch

import ops_rec_b200 as ops_rec
from oracle import hstu_cache_oracle as CO
from oracle import hstu_window_oracle as WO
from ops_rec_b200 import cabi
from tests import test_paged8 as P8
from tests.test_window import FP16, make

NAMES = ("out", "dq", "dk", "dv")


def reference(args, grad, window, sink):
    """{name: (value, tolerance)}; P and dS may be rounded with or without the scale, so half a smallest step is one of the scaled
    numbers here (2^-25 of each that a sum has)."""
    offq = args["seq_offset"].tolist()
    offk = args["seq_offset_k"].tolist() if "seq_offset_k" in args else offq
    tgt = args["num_target"].tolist() if "num_target" in args else [0] * (len(offq) - 1)
    got = {n: [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for _ in range(2)]
           for n, t in zip(NAMES, (grad, args["q"], args["k"], args["v"]))}
    for b, t in enumerate(tgt):
        rows, keys = slice(offq[b], offq[b + 1]), slice(offk[b], offk[b + 1])
        see = WO.window_mask(rows.stop - rows.start, keys.stop - keys.start, t, args.get("target_group_size", 0), window, sink, "cuda")
        one = WO.attention(args["q"][rows], args["k"][keys], args["v"][keys], see, args["alpha"], 1 / args["max_seq_len"], FP16, grad[rows])
        for n in NAMES:
            for full, part in zip(got[n], one[n]):
                full[rows if n in ("out", "dq") else keys] = part
    return got


def run(args, grad, window, sink):
    out, st = cabi.hstu_window_forward(window=window, num_sink=sink, return_status=True, **args)
    grads, st2 = cabi.hstu_window_backward(grad, window=window, num_sink=sink, return_status=True, **args)
    assert st == 0 and st2 == 0
    return dict(zip(NAMES, (out, *grads)))


def close(got, want):
    for n, (value, tol) in want.items():
        assert value.abs().max() < 65504, n   # (what is asked for is in range)
        assert torch.isfinite(got[n].float()).all(), (n, (~torch.isfinite(got[n].float())).float().mean().item())
        far = (got[n].double() - value).abs() - tol - 2.0 ** -24
        assert (far <= 0).all(), (n, far.max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dq,dv", [(64, 64), (128, 128), (96, 48), (20, 16), (17, 32), (160, 160)])
@pytest.mark.parametrize("window,sink,targets", [(1 << 30, 0, 0), (40, 3, 9)])
def test_gradients_of_a_large_loss_scale(dq, dv, window, sink, targets):
    """|dO.V| alpha reaches 10^6; times the scale of 1 / 4096 it is in the hundreds."""
    args, grad = make([517, 1, 130, 300], 4, 2, dq, dv, FP16, tgt=targets, seed=60 + dq, max_seq_len=4096)
    args["v"] = args["v"] * 8
    grad = grad.sign() * 6e4
    got = run(args, grad, window, sink)
    close(got, reference(args, grad, window, sink))
    if window == 1 << 30:   # finite where the jagged operator's are
        for n, g in zip(NAMES[1:], cabi.hstu_jagged_backward(grad, **args)):
            assert torch.isfinite(got[n].float())[torch.isfinite(g.float())].all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("dq,dv", [(64, 64), (128, 128), (96, 48), (20, 16), (17, 32), (160, 160)])
@pytest.mark.parametrize("delta", [None, 250])
def test_scores_beyond_the_type(dq, dv, delta):
    """Some rows' scores reach 10^5 to 10^6; their outputs, and the gradients, are in the thousands."""
    args, grad = make([517, 1, 130, 300], 4, 2, dq, dv, FP16, delta=delta, seed=70 + dq, max_seq_len=4096)
    args["alpha"] = 1.0
    args["q"] = args["q"] * 60
    args["q"][::3] = args["q"][::3] / 60    # (and others' are of the usual size)
    args["k"] = args["k"] * 600
    args["v"], grad = args["v"] / 8, grad / 8
    own = (args["q"][-300:, 0].float() * args["k"][-300:, 0].float()).sum(1) if delta is None else args["q"][-50:, 0].float() @ args["k"][-25:, 0].float().T
    assert own.abs().max() > 65504
    close(run(args, grad, 30, 2), reference(args, grad, 30, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_other_rows_keep_their_bits(d):
    """What one sequence holds - numbers beyond the type, infinities, NaN - leaves the bits of the others as they are."""
    args, grad = make([200, 77, 300, 50], 2, 2, d, dtype=FP16, seed=80, max_seq_len=4096)
    clean = run(args, grad, 60, 3)
    off = args["seq_offset"].tolist()
    for what in (3e4, float("inf"), float("nan")):
        other, g = {n: t.clone() if torch.is_tensor(t) else t for n, t in args.items()}, grad.clone()
        other["v"][off[1]:off[2]], g[off[1]:off[2]] = what, what
        other["q"][off[3]:off[4]] = what
        got = run(other, g, 60, 3)
        for n in NAMES:
            for a, b in ((0, 1), (2, 3)):
                assert torch.equal(got[n][off[a]:off[b]], clean[n][off[a]:off[b]]), (what, n)
            if what != 3e4:
                assert not torch.isfinite(got[n][off[1]:off[2]].float()).all(), (what, n)


@pytest.mark.gpu
def test_captured_with_usual_numbers_and_replayed_with_large_ones():
    args, grad = make([300, 129], 2, 2, 64, dtype=FP16, seed=81, max_seq_len=4096)
    op = ops_rec.ascendc.attention.hstu_window
    leaves = [args[n].clone().requires_grad_() for n in "qkv"]
    g = grad.clone()

    def step():
        out = op(*leaves, 90, 2, 4096, 0, 0.0, args["seq_offset"], None, None, 0, args["alpha"])
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        usual = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, usual))
    g.copy_(grad.sign() * 6e4)
    with torch.no_grad():
        leaves[2].mul_(8)
    graph.replay()
    large = args | dict(v=leaves[2].detach())
    close(dict(zip(NAMES, held)), reference(large, g, 90, 2))
    assert all(torch.equal(a, b) for a, b in zip(held, step()))
    g.copy_(grad)
    with torch.no_grad():
        leaves[2].copy_(args["v"])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, usual))


@pytest.mark.gpu
@pytest.mark.parametrize("users,new,d,page,targets,group", [
    (P8.MANY, 40, 64, 64, None, 1), (P8.MANY, 40, 128, 128, 9, 1),   # unpacked
    (3, 1, 64, 64, None, 1), (3, 20, 64, 64, 5, 1),                  # in place
    (3, 30, 64, 24, 5, 1), (3, 30, 128, 32, 20, 5), (3, 9, 320, 16, None, 1),   # staged
])
@pytest.mark.parametrize("window,sink", [(0, 0), (50, 3)])
def test_scores_beyond_the_type_over_a_cache(users, new, d, page, targets, group, window, sink):
    rng = np.random.default_rng(82)
    cached = rng.integers(new, 300, users)
    args = P8.make(cached, np.full(users, new), None if targets is None else np.full(users, targets), 4, 2, d, FP16, P8.INT8, page, 8, seed=83)
    args |= dict(alpha=1.0, silu_scale=1 / 4096, q=args["q"] * 60, k=args["k"] * 60)
    args["q"][1::3] = args["q"][1::3] / 60
    args["kv_scale"][:, 0] *= 2048
    args["kv_scale"][:, 1] /= 4
    if targets is not None:
        args["target_group_size"] = group
    cu = P8.on_gpu(args)
    mine = cu["page_ids"][:int(args["page_offsets"][1])]     # the first user's scores: its last new row, with the last head
    keys = cu["kv_cache"][mine, 0, :, -1].float().flatten(0, 1) * cu["kv_scale"][mine, 0, :, -1].repeat_interleave(8, 1).flatten()[:, None]
    assert keys[:int(cached[0])].abs().max() < 65504 < (cu["q"][:new, -1].float() @ keys[:int(cached[0])].T).abs().max()
    assert CO.paged(**cu, window=window, num_sink=sink)[0].abs().max() < 65504
    P8.check_paged(args, window, sink)
