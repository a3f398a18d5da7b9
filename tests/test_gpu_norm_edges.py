"""Group norm and dropout at the edges of what their documentation allows."""
import pytest
import torch

import sfm_amd
from test_gpu_norm import inputs

pytestmark = pytest.mark.gpu


# ---- layouts
SUMS = [((4, 8, 8, 32), (1, 2)), ((2, 64, 24), (1,)), ((4, 8, 8, 32), (2,)), ((4, 8, 32), (0,)), ((4, 8, 8, 32), (0, 1, 2)), ((6, 8), (0,)),
        ((2, 64, 1), (0, 1, 2)), ((2, 9, 24), (0, 1, 2)), ((3, 700, 32), (1,)), ((2, 31, 17, 45), (1, 2))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,over", SUMS, ids=[f"{'x'.join(map(str, s))}over{''.join(map(str, o))}" for s, o in SUMS])
def test_gradients_of_sums(dev, shape, over, dtype):
    """dL/dy is an expanded tensor, whose row strides are 0 where y was summed: the gradients of its dense copy, bit by bit"""
    x, _, gamma, beta = inputs(shape, dtype, 201, dev)
    groups = 1 if shape[-1] == 1 else shape[-1] // 8 if shape[-1] % 8 == 0 else 5
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, groups)
    seen = []
    y.register_hook(lambda g: seen.append(g))
    s = y.sum(dim=over)
    w = torch.randn(s.shape, generator=torch.Generator().manual_seed(202)).to(dtype).to(dev)
    got = torch.autograd.grad(s, leaves, w)
    assert len(seen) == 1 and 0 in seen[0].stride()
    want = torch.autograd.grad(sfm_amd.group_norm_act(*leaves, groups), leaves, seen[0].contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("shape,of", [((4, 10, 24), (24,)), ((4, 10, 24), (10, 24)), ((4, 10, 3, 24), (4, 10, 1, 24)), ((5, 24), (1, 24)),
                                      ((3, 7, 1), (1, 7, 1))], ids=str)
def test_expanded_input(dev, shape, of):
    v, gy, gamma, beta = inputs(of if len(of) > 1 else (1, *of), torch.float32, 203, dev)
    x = v.reshape(of).expand(shape)
    assert 0 in x.stride()
    gy = torch.randn(shape, generator=torch.Generator().manual_seed(204)).to(dev)
    runs = []
    for t in (x, x.contiguous()):
        leaves = [u.detach().requires_grad_(True) for u in (t, gamma, beta)]
        y = sfm_amd.group_norm_act(*leaves, max(1, shape[-1] // 6))
        runs.append((y, *torch.autograd.grad(y, leaves, gy)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
