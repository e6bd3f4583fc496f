"""The ctypes entry points of hstu_window, hstu_cache_append and hstu_paged_8bit: arguments that a kernel would read past."""
import pytest
import torch

from ops_rec_b200 import cabi
from tests.test_paged8 import BF16, E4M3, FP32, make, on_gpu, table

OFF = torch.tensor([0, 4, 10])


def rows(heads, dim=64, n=10, dtype=BF16):
    return torch.zeros(n, heads, dim, dtype=dtype)


@pytest.mark.parametrize("change,needle", [
    (dict(k=rows(2, dtype=FP32)), "same dtype"), (dict(v=rows(2, dtype=FP32)), "same dtype"), (dict(v=rows(2, n=9)), "agree in tokens"),
    (dict(k=rows(2, 32)), "agree in tokens"), (dict(seq_offset_k=OFF[:2]), "seq_offset_k must have 3"),
    (dict(num_target=OFF[:1]), "num_target must have 2"), (dict(seq_offset=OFF.float()), "int32 or int64"),
    (dict(grad=rows(4, 32)), "grad must be"), (dict(grad=rows(4, dtype=FP32)), "grad must be"),
])
def test_window_refuses(change, needle):
    args = dict(q=rows(4), k=rows(2), v=rows(2), seq_offset=OFF, max_seq_len=8, window=3) | change
    grad = args.pop("grad", rows(4))
    if "grad" not in change:
        with pytest.raises(cabi.HstuError, match=needle):
            cabi.hstu_window_forward(**args)
    with pytest.raises(cabi.HstuError, match=needle):
        cabi.hstu_window_backward(grad, **args)


@pytest.mark.parametrize("change,needle", [
    (dict(v=rows(2, dtype=FP32)), "same dtype"), (dict(page_offsets=OFF[:2]), "page_offsets must have 3"),
    (dict(page_offsets=torch.tensor([0, 1, 2, 2])), "page_offsets must have 3"), (dict(last_page_len=OFF[:1]), "last_page_len must have 2"),
    (dict(num_target=OFF[:1]), "num_target must have 2"), (dict(seq_offset=OFF.float()), "int32 or int64"),
])
def test_cache_calls_refuse(change, needle):
    cache, scale = torch.zeros(3, 2, 32, 2, 64).to(E4M3), torch.zeros(3, 2, 2, 2)
    args = dict(k=rows(2), v=rows(2), kv_cache=cache, kv_scale=scale, seq_offset=OFF, page_offsets=torch.tensor([0, 1, 2]),
                page_ids=torch.tensor([0, 1]), last_page_len=torch.tensor([4, 6]), num_target=None) | change
    with pytest.raises(cabi.HstuError, match=needle):
        cabi.hstu_cache_append(**args)
    with pytest.raises(cabi.HstuError, match=needle):
        cabi.hstu_paged_8bit_forward(rows(4), **args, seq_offset_k=OFF, max_seq_len=8)
    if "v" in change:
        with pytest.raises(cabi.HstuError, match="same tokens as q"):
            cabi.hstu_paged_8bit_forward(rows(4, n=12), **(args | dict(v=rows(2))), seq_offset_k=OFF, max_seq_len=8)
        with pytest.raises(cabi.HstuError, match="seq_offset_k must have 3"):
            cabi.hstu_paged_8bit_forward(rows(4), **(args | dict(v=rows(2))), seq_offset_k=OFF[:2], max_seq_len=8)


def strided(t):
    """The same numbers, every second of a larger tensor."""
    return torch.stack((t, t + 1000), 1).flatten()[::2]


@pytest.mark.gpu
def test_index_tensors_of_other_types_and_strides():
    args = make([60, 45, 100], [10, 5, 30], [3, 0, 7], seed=74)
    cu = on_gpu(args)
    names = [n for n, t in cu.items() if torch.is_tensor(t) and not t.is_floating_point()]
    want = cabi.hstu_paged_8bit_forward(**cu)
    t = table(args)
    cabi.hstu_cache_append(**t)
    for n in names:
        other = cu | {n: strided(cu[n])}
        assert torch.equal(cabi.hstu_paged_8bit_forward(**other), want), n
        other = cu | {m: cu[m].int() for m in names if m != n}
        assert torch.equal(cabi.hstu_paged_8bit_forward(**other), want), n
        if n in t:
            again = table(args)
            again[n] = strided(again[n])
            cabi.hstu_cache_append(**again)
            assert torch.equal(again["kv_cache"].view(torch.uint8), t["kv_cache"].view(torch.uint8)), n
    w = dict(q=cu["q"], k=cu["k"], v=cu["v"], seq_offset=cu["seq_offset"], seq_offset_k=cu["seq_offset"], num_target=cu["num_target"],
             target_group_size=1, max_seq_len=64, window=7)
    want = cabi.hstu_window_forward(**w), *cabi.hstu_window_backward(cu["q"], **w)
    for n in ("seq_offset", "seq_offset_k", "num_target"):
        for change in (strided(w[n]), w[n].int()):
            got = cabi.hstu_window_forward(**(w | {n: change})), *cabi.hstu_window_backward(cu["q"], **(w | {n: change}))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), n
    wide = w | dict(window=1 << 40, num_sink=1 << 40)
    assert torch.equal(cabi.hstu_window_forward(**wide), cabi.hstu_window_forward(**(w | dict(window=1 << 30))))
