"""CPU checks behind tests/test_gpu_norm_edges.py: which layouts the group norm reads in place (nothing here reaches a kernel)."""
import pytest
import torch

from sfm_amd import norm


def grad_of(f, *shape):
    """the gradient that autograd hands to y of `shape` from f(y), with the strides it has"""
    y = torch.randn(*shape, requires_grad=True)
    seen = []
    y.register_hook(seen.append)
    f(y).backward()
    return seen[0]


def _filled(t):
    """t's strides over a storage of different numbers"""
    n = t.untyped_storage().nbytes() // t.element_size()
    return torch.arange(n, dtype=torch.float32).as_strided(t.shape, t.stride(), t.storage_offset())


wide = torch.zeros(3, 5, 7, 50)
LAYOUTS = {  # name -> (tensor, whether it has to be read in place)
    # broadcast gradients: a stride of 0 in some row dimension
    "sum over H, W": (grad_of(lambda y: (y.sum(dim=(1, 2)) * torch.randn(4, 32)).sum(), 4, 8, 8, 32), False),
    "sum over N": (grad_of(lambda y: (y.sum(1) * torch.randn(2, 24)).sum(), 2, 64, 24), False),
    "sum over W": (grad_of(lambda y: (y.sum(dim=2) * torch.randn(4, 8, 32)).sum(), 4, 8, 8, 32), False),
    "sum over B": (grad_of(lambda y: (y.sum(0) * torch.randn(8, 32)).sum(), 4, 8, 32), False),
    "sum over all rows": (grad_of(lambda y: (y.sum(dim=(0, 1, 2)) * torch.randn(32)).sum(), 4, 8, 8, 32), False),
    "sum over B of [B, C]": (grad_of(lambda y: (y.sum(0) * torch.randn(8)).sum(), 6, 8), False),
    "sum of one channel": (grad_of(lambda y: y.sum(), 2, 64, 1), False),
    "sum of everything": (grad_of(lambda y: y.sum(), 2, 9, 24), False),
    "expanded rows": (torch.zeros(1, 1, 24).expand(4, 10, 24), False),
    "expanded items": (torch.zeros(1, 10, 24).expand(4, 10, 24), False),
    "expanded inside": (torch.zeros(4, 10, 1, 24).expand(4, 10, 3, 24), False),
    "expanded slice": (wide[:, :1, :, 4:28].expand(3, 5, 7, 24), False),
    # rows that overlap, have gaps of two kinds, or stand in another order
    "overlapping rows": (torch.zeros(100).as_strided((5, 24), (8, 1)), False),
    "every second column": (wide[:, :, ::2, 1:25], False),
    "some rows": (wide[:, 1:4, :, :24], False),
    "permuted": (wide.permute(0, 2, 1, 3)[..., :24], False),
    "every second channel": (wide[..., ::2][..., :24], False),
    # what is read in place
    "dense": (torch.zeros(3, 5, 24), True),
    "channel slice": (wide[..., 3:27], True),
    "one item's slice": (wide[1:2, ..., 3:27], True),
    "one row": (wide[1:2, 2:3, 3:4, 1:25], True),
    "one column of one channel": (wide[..., 7:8], True),
    "no rows": (wide[:0, ..., 1:25], True),
    "no rows inside": (wide[:, :0, :, 1:25], True),
}


@pytest.mark.parametrize("name", LAYOUTS)
def test_rows_are_where_the_kernels_look_for_them(name):
    """the address, the row stride and the reach that the kernels are given lie in the storage and hold the tensor's values"""
    t, in_place = LAYOUTS[name]
    x = _filled(t)
    rows, ld = norm._nodes().rows_of(x)
    C = x.shape[-1]
    assert ld >= C
    n = x.numel() // C
    if n:
        have = rows.untyped_storage().nbytes() // rows.element_size()
        assert rows.storage_offset() + (n - 1) * ld + C <= have, "read past the storage"
        assert torch.equal(rows.as_strided((n, C), (ld, 1), rows.storage_offset()), x.reshape(n, C))
    assert (rows is x) == in_place


@pytest.mark.parametrize("dtype,ld,in_place", [(torch.float32, 2 ** 29 - 1, True), (torch.float32, 2 ** 29, False), (torch.bfloat16, 2 ** 30 - 1, True),
                                               (torch.bfloat16, 2 ** 30, False)])
def test_rows_farther_apart_than_the_kernels_reach_are_copied(dtype, ld, in_place):
    x = torch.empty(2, 3, ld, dtype=dtype, device="meta")[..., :24]
    rows, got = norm._nodes().rows_of(x)
    assert (rows is x) == in_place and got == (ld if in_place else 24)


@pytest.mark.parametrize("item0,rc", [(2 ** 32 - 1, -2), (2 ** 32 - 2, -1)])
def test_items_that_the_counter_holds(item0, rc):
    """two items behind item0: refused where the second would be item 2^32; else the call goes on to the next refusal, its missing tensors"""
    import ctypes
    from sfm_amd import _lib
    lib, f = _lib.load(), 0x10000  # (stands for a device address: nothing is read before the refusal)
    mask = (None, 0, 0, 0, item0, 9, 0)
    src, ld = (ctypes.c_void_p * 1)(None if rc == -1 else f), (ctypes.c_longlong * 1)(8)
    assert lib.sfm_group_norm_act_bwd(f, 8, 0, src, ld, 1, f, f, f, f, 2, 3, 8, 4, 1, *mask, f, f, f, f, None) == rc


def _node_calls():
    n, g = norm._nodes(), torch.ones(8)
    none = (None, 0, 0, 0, 0, 0, False)
    return {"group_norm_act": lambda x: n.group_norm_act(x, g, g, 2, 1e-5, 1, *none), "dropout": lambda x: n.dropout(x, None, 1, 2, 0, 0, 9, False),
            "group_norm_act (buckets)": lambda x: n.refuse_tracing("group_norm_act") or x * 1}


@pytest.mark.parametrize("name", _node_calls())
def test_tracing_is_refused(name):
    """a tracer would record the allocation of the result and nothing of what fills it (refused before a tensor's memory is looked at)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = _node_calls()[name], torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, (x,))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(f)(x)
    if "buckets" in name:
        f(x)


def test_the_bounds_see_a_difference_of_large_sums():
    """what tests/test_gpu_norm_edges.py allows where the mean is far from the deviation is not enough for a variance that is E[x^2] - mean^2 in
    fp32, and is enough for one from deviations"""
    import numpy as np
    from oracle import norm_ref as R
    from test_gpu_norm import U, f64, inputs
    x, _, gamma, beta = inputs((2, 5000, 32), torch.float32, 213, "cpu")
    x = x + 1000.0
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), 8, 1e-5, "elu")
    v = x.reshape(2, 5000, 8, 4)
    mean = v.mean(dim=(1, 3), keepdim=True)
    share = []
    for var in ((v * v).mean(dim=(1, 3), keepdim=True) - mean * mean, ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True)):
        y = torch.nn.functional.elu(((v - mean) / (var + 1e-5).sqrt()).reshape(x.shape) * gamma + beta)
        off = np.abs(f64(y) - want["y"]) / (40 * U * want["z_size"] + U * np.abs(want["y"]))
        share.append(off[np.isfinite(off)].max() if np.isfinite(off).any() else np.inf)
    assert share[0] > 10 and share[1] < 1, share
