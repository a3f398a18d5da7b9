"""GPU parity of group norm with an activation and of dropout (csrc/group_norm.hip, csrc/dropout.hip) against the definitions in
float64 (oracle/norm_ref.py).

Tolerances, with u = 2^-24 (half a step of fp32, relative) and h = eps(type) / 2:
  y     every value passes at most 32 roundings of fp32 on values no larger than z_size = 1 + |gamma| (|x| + |x - mean|) / std (the
        mean's own error counts against |x|), |act'| <= 1.1: |y - y64| <= 40 u z_size s + h |y64|, s the mask's factor
  gx    the same counts on r |gamma dz| (1 + |xhat|)^2, the largest of the (item, group), c1 and c2 being averages of such terms
        with at most 64 sequential additions: 160 u gx_size + h |gx64|; act' is moved by z's error, under the same bound
  sums  a sum of terms passes at most 256 sequential fp32 additions here (rows of a thread, then row lanes; chunks are joined
        in fp64), each term 32 roundings: 300 u sum|terms|.  Two errors of a term are not relative to it, however small it is:
        xhat = (x - mean) r is off by d = 40 u z_size (as y above: the mean's own rounding), and act'(z), near a zero of it, by
        |act''| d <= d.  So gbeta = sum dz, dz = s gy act'(z): + d sum|s gy|; ggamma = sum dz xhat: + d (sum|dz| + max|xhat| sum|s gy|)
A 16-bit type's smallest step near zero (fp16: 2^-25 absolute) is added for values in its subnormal range."""
import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import sfm_amd
from oracle import norm_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def inputs(shape, dtype, seed, dev, offset=1.0):
    """activations with means and scales of their own per channel, and dL/dy"""
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = torch.randn(*shape, generator=g) * (0.5 + torch.rand(C, generator=g)) + offset * torch.randn(C, generator=g)
    gy = torch.randn(*shape, generator=g)
    gamma, beta = 1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)
    return x.to(dtype).to(dev), gy.to(dtype).to(dev), gamma.to(dev), beta.to(dev)


def f64(t):
    return t.detach().double().cpu().numpy()


def within(got, want, bound, what):
    got = f64(got)
    assert np.isfinite(got).all(), f"{what}: not finite"
    off = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(off), off.shape)
    assert off[at] <= 0, f"{what}: {got[at]} for {want[at]} at {at}: off {abs(got[at] - want[at]):.3e}, allowed {np.broadcast_to(bound, off.shape)[at]:.3e}"


def compare(y, grads, want, dtype, scale=1.0, loose=None):
    """loose: what relu's jump adds to the bounds of (gx, ggamma, gbeta)"""
    h, tiny = HALF[dtype], TINY[dtype]
    lx, lg, lb = loose if loose is not None else (0.0, 0.0, 0.0)
    within(y, want["y"], 40 * U * want["z_size"] * scale + h * np.abs(want["y"]) * (1 + 2 * h) + tiny, "y")
    if grads is not None:
        gx, gg, gb = grads
        d = 40 * U * want["z_size"].max()
        assert gg.dtype == gb.dtype == torch.float32
        within(gx, want["gx"], 160 * U * want["gx_size"] + h * np.abs(want["gx"]) * (1 + 2 * h) + tiny + lx, "gx")
        within(gg, want["ggamma"], 300 * U * want["abs_ggamma"] + d * (want["abs_gbeta"] + want["xhat_max"] * want["abs_gy"]) + tiny + lg, "ggamma")
        within(gb, want["gbeta"], 300 * U * want["abs_gbeta"] + d * want["abs_gy"] + tiny + lb, "gbeta")


SHAPES = [  # shape, groups: every vector width, whole and split groups, ragged slabs and chunks
    ((1, 1, 1, 8), 2), ((1, 1, 8), 8), ((2, 1, 1, 32), 4),          # one row; one value per group (the variance is 0)
    ((2, 2, 16), 4), ((3, 3, 5, 12), 4), ((2, 63, 6), 3),           # cpg 3 and 2: a vector crosses groups
    ((2, 7, 9, 45), 5), ((1, 64, 1), 1), ((2, 65, 7), 7), ((2, 65, 7), 1),  # odd channel counts
    ((3, 37, 53, 90), 6), ((2, 31, 17, 1000), 2), ((2, 31, 17, 1000), 250),
    ((1, 4, 13, 2048), 32), ((4, 8, 26, 512), 32), ((2, 16, 52, 256), 16), ((1, 64, 208, 64), 16), ((1, 128, 416, 32), 8),
    ((2, 19, 4096), 1), ((2, 19, 1028), 1), ((1, 9, 2500), 2), ((1, 11, 4100), 2),  # groups wider than a workgroup
    ((1000, 1, 24), 3), ((300, 5, 8), 1), ((70, 3, 3, 40), 40),     # many small items; one channel per group
    ((1, 5000, 8), 2), ((1, 4099, 20), 5), ((1, 257, 2048), 2048),
    ((2, 300, 64), 64), ((2, 511, 32), 8), ((2, 512, 32), 8), ((2, 513, 32), 8), ((3, 130, 96), 2), ((1, 128, 1024), 1),  # about what a workgroup holds
    # workgroups with several tiles of rows, the last tile short: the last pass starts with it (few rows, and one row lane's worth)
    ((300, 1801, 32), 8), ((300, 1825, 32), 32), ((600, 700, 9), 3), ((500, 613, 36), 4),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=[f"{'x'.join(map(str, s))}g{g}" for s, g in SHAPES])
def test_group_norm_forward_and_gradients(dev, shape, groups, dtype):
    k = SHAPES.index((shape, groups))
    act = ("elu", "silu", "none")[k % 3]
    x, gy, gamma, beta = inputs(shape, dtype, 100 + k, dev)
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), groups, 1e-5, act, f64(gy))
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, groups, activation=act)
    assert y.dtype == dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, leaves, gy)
    compare(y, grads, want, dtype)
    with torch.no_grad():  # the serving form gives the same bits
        assert torch.equal(sfm_amd.group_norm_act(*leaves, groups, activation=act), y)


@pytest.mark.parametrize("act", ["elu", "relu", "silu", None])
@pytest.mark.parametrize("p,per_channel", [(0.0, False), (0.3, False), (0.3, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,groups", [((3, 9, 11, 48), 6), ((2, 50, 30), 5), ((2, 21, 9), 3), ((1, 3, 1028), 1)],
                         ids=["c48", "c30", "c9", "wide"])
def test_activations_and_masks(dev, shape, groups, dtype, p, per_channel, act):
    x, gy, gamma, beta = inputs(shape, dtype, 7, dev)
    mask, keep, t = None, None, 0
    if p:
        mask = sfm_amd.DropoutMask(p, (2 ** 45 + 17, 12), layer=5, per_channel=per_channel, first_item=2)
        t = mask.threshold
        keep = R.keep_mask(shape, t, 2 ** 45 + 17, 12, 5, per_channel, 2)
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), groups, 1e-5, act, f64(gy), keep, t)
    loose = None
    if act == "relu":
        # where z is nearer to 0 than its own error, relu' may be 0 or 1: such a value's dz, at most g = s |gy|, is then there or not.  That
        # moves gx at its place by at most r |gamma| g (1 + |xhat|)^2 and, through c1 and c2, its group by the m-th part of that
        # each; ggamma of its channel by |xhat| g and gbeta by g.  (Few values: the bound for all others hardly moves.)
        near = np.abs(want["z"]) <= 40 * U * want["z_size"]
        assert near.mean() <= 1e-3
        xhat = (f64(x).reshape(shape[0], -1, groups, shape[-1] // groups) - want["mean"][:, None, :, None]) * want["rstd"][:, None, :, None]
        g = 65536 / (65536 - t) * np.abs(f64(gy))
        most = want["rstd"].max() * np.abs(f64(gamma)).max() * g.max() * (1 + np.abs(xhat).max()) ** 2
        m = x.numel() // (shape[0] * groups)
        over = tuple(range(len(shape) - 1))
        loose = (near * most + near.sum() * most / m, (near * g * np.abs(xhat).max()).sum(axis=over), (near * g).sum(axis=over))
    leaves = [v.requires_grad_(True) for v in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, groups, activation=act, dropout=mask)
    grads = torch.autograd.grad(y, leaves, gy)
    compare(y, grads, want, dtype, 65536 / (65536 - t), loose)
    if p:
        assert np.array_equal(f64(y) == 0, ~np.asarray(keep) | (want["y"] == 0))


@pytest.mark.parametrize("per_channel", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,groups", SHAPES[-4:], ids=["c32g8", "c32g32", "c9", "c36"])
def test_masks_where_workgroups_take_several_tiles(dev, shape, groups, dtype, per_channel):
    x, gy, gamma, beta = inputs(shape, dtype, 9, dev)
    mask = sfm_amd.DropoutMask(0.4, (77, 3), layer=1, per_channel=per_channel, first_item=1)
    keep = R.keep_mask(shape, mask.threshold, 77, 3, 1, per_channel, 1)
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), groups, 1e-5, "elu", f64(gy), keep, mask.threshold)
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, groups, activation="elu", dropout=mask)
    compare(y, torch.autograd.grad(y, leaves, gy), want, dtype, 65536 / (65536 - mask.threshold))


@pytest.mark.parametrize("per_channel", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,groups", [((2, 5, 2072), 2), ((3, 9, 2080), 2), ((2, 4, 6216), 6), ((2, 7, 1, 5140), 4)],
                         ids=["parts520of1036", "parts520of1040", "parts520of1036x6", "parts of 1285"])
def test_masks_where_a_group_has_parts(dev, shape, groups, dtype, per_channel):
    """a part of a group may start in the middle of the mask's blocks of eight"""
    x, gy, gamma, beta = inputs(shape, dtype, 13, dev)
    mask = sfm_amd.DropoutMask(0.5, (91, 4), layer=2, per_channel=per_channel)
    keep = R.keep_mask(shape, mask.threshold, 91, 4, 2, per_channel, 0)
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), groups, 1e-5, "silu", f64(gy), keep, mask.threshold)
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, groups, activation="silu", dropout=mask)
    compare(y, torch.autograd.grad(y, leaves, gy), want, dtype, 65536 / (65536 - mask.threshold))


def test_gradient_against_differences(dev):
    """directional differences of the fp32 kernel itself, at a step where the difference's own rounding (2 u |f| / step) and its
    curvature (step^2) are both under 1e-3 of the derivative"""
    x, gy, gamma, beta = inputs((2, 30, 24), torch.float32, 21, dev)
    mask = sfm_amd.DropoutMask(0.2, (5, 6))
    f = lambda *a: float((sfm_amd.group_norm_act(*a, 4, activation="silu", dropout=mask).double() * gy.double()).sum())  # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in (x, gamma, beta)]
    grads = torch.autograd.grad(sfm_amd.group_norm_act(*leaves, 4, activation="silu", dropout=mask), leaves, gy)
    g = torch.Generator().manual_seed(1)
    for k, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g).to(dev)
        v = v * torch.sign(v * grad)       # every term of <grad, v> is positive: the derivative is large
        step = 2.0 ** -9
        up, down = [x, gamma, beta], [x, gamma, beta]
        up[k], down[k] = up[k] + step * v, down[k] - step * v
        want = float((grad.double() * v.double()).sum())
        assert abs((f(*up) - f(*down)) / (2 * step) - want) <= 3e-3 * want


def test_mean_far_from_the_deviation(dev):
    """statistics are not differences of large sums: mean 1000 (and a first row far off), deviation 1; error bound as ever, z_size holds |x| / std"""
    x, gy, gamma, beta = inputs((2, 700, 32), torch.float32, 31, dev)
    x = x + 1000.0
    x[:, 0] = -3.0e4
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), 4, 1e-5, "elu", f64(gy))
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, 4)
    compare(y, None, want, torch.float32)


def test_constant_groups(dev):
    """variance 0: y = act(beta) exactly"""
    x = torch.full((2, 50, 24), 7.25, device=dev)
    beta = torch.linspace(-1, 1, 24, device=dev)
    y = sfm_amd.group_norm_act(x, torch.ones(24, device=dev), beta, 3, activation=None)
    assert torch.equal(y, beta.expand_as(y))


def test_what_is_not_finite_stays_in_its_group(dev):
    x, gy, gamma, beta = inputs((3, 40, 24), torch.float32, 41, dev)
    clean = sfm_amd.group_norm_act(x, gamma, beta, 4)
    bad = x.clone()
    bad[1, 7, 8] = float("nan")
    bad[2, 3, 23] = float("inf")
    y = sfm_amd.group_norm_act(bad, gamma, beta, 4)
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, :, 6:12] = True
    hit[2, :, 18:24] = True
    assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])
    y = sfm_amd.group_norm_act(bad, gamma, beta, 4, activation="relu")
    assert torch.isnan(y[hit]).all()


def test_strides(dev):
    """channel slices are read in place, whatever their alignment; other orders are copied; gradients that are expanded or transposed"""
    wide = torch.randn(3, 5, 7, 50, generator=torch.Generator().manual_seed(51)).to(dev)
    _, _, gamma, beta = inputs((1, 1, 24), torch.float32, 52, dev)
    for dtype in (torch.float32, torch.float16):
        w = wide.to(dtype)
        for x in (w[..., 3:27], w[:, :, :, 26:], w[:, 1:4, :, :24], w[:, :, ::2, 1:25], w[..., ::2][..., :24], w[1:2, 2:3, 3:4, 1:25],
                  w.permute(0, 2, 1, 3)[..., :24]):
            want = sfm_amd.group_norm_act(x.contiguous(), gamma, beta, 4)
            assert torch.equal(sfm_amd.group_norm_act(x, gamma, beta, 4), want)
            a, b = x.detach().requires_grad_(True), x.contiguous().detach().requires_grad_(True)
            gy = torch.randn(x.shape, device=dev).to(dtype).transpose(1, 2).contiguous().transpose(1, 2)
            (ga,) = torch.autograd.grad(sfm_amd.group_norm_act(a, gamma, beta, 4), a, gy)
            (gb,) = torch.autograd.grad(sfm_amd.group_norm_act(b, gamma, beta, 4), b, gy.contiguous())
            assert torch.equal(ga, gb)
    x = torch.randn(2, 9, 24, device=dev, requires_grad=True)
    one = torch.ones_like(x)
    (g1,) = torch.autograd.grad(sfm_amd.group_norm_act(x, gamma, beta, 4).sum(), x)     # dL/dy is one expanded number
    (g2,) = torch.autograd.grad(sfm_amd.group_norm_act(x, gamma, beta, 4), x, one)
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,C,groups", [(37, 24, 4), (700, 32, 8), (5000, 20, 5), (65, 7, 7), (9, 2500, 2)])
def test_slices_of_buffers(dev, N, C, groups, dtype):
    """the C ABI as a level without concats calls it: x and y slices of wider buffers, nothing beside the slices written, dL/dy the
    sum of three slices with strides of their own"""
    import ctypes
    from sfm_amd import _lib
    from sfm_amd._lib import ptr, stream_of
    B, act = 2, 1
    x, gy, gamma, beta = inputs((B, N, C), dtype, 55, dev)
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), groups, 1e-5, "elu", f64(gy))
    wx, wy = torch.full((B, N, C + 11), 7.0, device=dev, dtype=dtype), torch.full((B, N, C + 5), 7.0, device=dev, dtype=dtype)
    wx[..., 3:3 + C] = x
    parts = [torch.full((B, N, C + k), 5.0, device=dev, dtype=dtype) for k in (1, 4, 0)]
    halves = [(gy.float() * f).to(dtype) for f in (0.5, 0.25)]
    for p, v in zip(parts, (*halves, (gy.float() - halves[0].float() - halves[1].float()).to(dtype))):
        p[..., p.shape[-1] - C:] = v                      # powers of two and an exact rest: the sum is gy again
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    lib, es = _lib.load(), x.element_size()
    mean, rstd = (torch.empty(B, groups, device=dev) for _ in range(2))
    ws = torch.empty(lib.sfm_group_norm_workspace_floats(B, N, C, groups, code, 1) + 2, device=dev)
    no_mask = (None, 0, 0, 0, 0, 0, 0)
    at = ctypes.c_void_p
    rc = lib.sfm_group_norm_act_fwd(at(wx.data_ptr() + 3 * es), C + 11, code, ptr(gamma), ptr(beta), B, N, C, groups, 1e-5, act, *no_mask,
                                    at(wy.data_ptr() + 2 * es), C + 5, ptr(mean), ptr(rstd), ptr(ws), stream_of(x))
    assert rc == 0
    assert (wy[..., :2] == 7).all() and (wy[..., 2 + C:] == 7).all()
    gx, gg, gb = torch.empty_like(x), torch.empty(C, device=dev), torch.empty(C, device=dev)
    srcs = (ctypes.c_void_p * 3)(*[p.data_ptr() + (p.shape[-1] - C) * es for p in parts])
    lds = (ctypes.c_longlong * 3)(*[p.shape[-1] for p in parts])
    rc = lib.sfm_group_norm_act_bwd(at(wx.data_ptr() + 3 * es), C + 11, code, srcs, lds, 3, ptr(gamma), ptr(beta), ptr(mean), ptr(rstd), B, N,
                                    C, groups, act, *no_mask, ptr(gx), ptr(gg), ptr(gb), ptr(ws), stream_of(x))
    assert rc == 0
    compare(wy[..., 2:2 + C], (gx, gg, gb), want, dtype)


def test_sizes_of_zero(dev):
    g = torch.ones(8, device=dev, requires_grad=True)
    for shape in ((0, 3, 8), (2, 0, 8), (0, 8)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        y = sfm_amd.group_norm_act(x, g, g, 2)
        assert y.shape == x.shape
        gx, gg = torch.autograd.grad(y, (x, g), torch.zeros_like(y))
        assert gx.shape == x.shape and float(gg.abs().sum()) == 0
        assert sfm_amd.dropout(x, sfm_amd.DropoutMask(0.5, (1, 2))).shape == x.shape


def test_only_the_gradients_that_are_asked_for(dev):
    x, gy, gamma, beta = inputs((2, 33, 24), torch.float32, 61, dev)
    leaves = [t.clone().requires_grad_(True) for t in (x, gamma, beta)]
    full = torch.autograd.grad(sfm_amd.group_norm_act(*leaves, 4), leaves, gy)
    for k in range(3):
        some = [t.clone() for t in (x, gamma, beta)]
        some[k].requires_grad_(True)
        (g,) = torch.autograd.grad(sfm_amd.group_norm_act(*some, 4), some[k], gy)
        assert torch.equal(g, full[k])


# ---- dropout alone
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("per_channel", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (3, 1, 1), (1, 7), (2, 8), (5, 3, 3), (4, 5, 9), (2, 63, 65), (1, 100, 24), (3, 37, 53, 90), (1000, 1, 3),
                                   (8, 8, 26, 512), (3, 11000)], ids=lambda s: "x".join(map(str, s)))
def test_dropout(dev, shape, per_channel, dtype):
    g = torch.Generator().manual_seed(71)
    x, gy = (torch.randn(*shape, generator=g).to(dtype).to(dev) for _ in range(2))
    mask = sfm_amd.DropoutMask(0.25, (99, 2 ** 33 + 3), layer=2 ** 32 - 1, per_channel=per_channel, first_item=2 ** 31)
    keep = torch.from_numpy(R.keep_mask(shape, mask.threshold, 99, 3, 2 ** 32 - 1, per_channel, 2 ** 31).copy()).to(dev)
    x.requires_grad_(True)
    y = sfm_amd.dropout(x, mask)
    (gx,) = torch.autograd.grad(y, x, gy)
    scale = torch.tensor(65536 / (65536 - mask.threshold), dtype=torch.float32, device=dev)
    for out, src in ((y, x), (gx, gy)):  # one product in fp32 and one rounding: the same bits
        assert torch.equal(out, torch.where(keep, (src.detach().float() * scale).to(dtype), torch.zeros_like(src)))
    assert not y.isnan().any()


def test_dropout_of_many_blocks(dev):
    """more workgroups than one dimension of a grid holds, and offsets past 32 bits: an item's result is that of the item by itself"""
    x = torch.ones(2050, 2 ** 22, dtype=torch.bfloat16, device=dev)
    mask = lambda first: sfm_amd.DropoutMask(0.5, (3, 4), first_item=first)  # noqa: E731
    y = sfm_amd.dropout(x, mask(0))
    for first, last in ((0, 2), (1023, 1025), (2046, 2050)):
        want = sfm_amd.dropout(x[first:last], mask(first))
        assert torch.equal(y[first:last], want) and 0.4 < float(want.float().mean()) / 2 < 0.6
    del y
    x = torch.ones(3, 2 ** 29 + 1, 3, dtype=torch.float16, device=dev)  # items that start and end in the middle of a block
    y = sfm_amd.dropout(x, mask(0))
    assert torch.equal(y[2:], sfm_amd.dropout(x[2:], mask(2)))


def test_group_norm_of_many_elements(dev):
    """offsets past 32 bits: an item's result is that of the item by itself, but for the order of its sums.  Each of the two is off by at most
    what `compare` allows: together two half steps of bf16 and twice the fp32 part, with the largest factors of the tensor"""
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(3, 1500001, 512, dtype=torch.bfloat16, device=dev, generator=g)
    gy = torch.randn(x.shape, dtype=torch.bfloat16, device=dev, generator=g)
    gamma, beta = torch.ones(512, device=dev), torch.zeros(512, device=dev)
    mask = lambda first: sfm_amd.DropoutMask(0.25, (3, 4), first_item=first)  # noqa: E731

    def run(x, gy, first):
        x.requires_grad_(True)
        y = sfm_amd.group_norm_act(x, gamma, beta, 4, dropout=mask(first))
        return y.detach(), torch.autograd.grad(y, x, gy)[0]

    y, gx = run(x, gy, 0)
    scale, most, steep = 4 / 3, float(x.detach().abs().max()), float(gy.abs().max())
    assert 0.99 < float(x.detach()[2].float().var()) < 1.01
    for k in (0, 2):
        want_y, want_gx = run(x.detach()[k:k + 1], gy[k:k + 1], k)
        for at in range(0, x.shape[1], 300001):  # (in pieces: the comparison is in fp32)
            a, b = y[k, at:at + 300001].float(), want_y[0, at:at + 300001].float()
            assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() * (1 + 2.0 ** -6) + 80 * U * scale * (2 + 3 * most)).all())
            a, b = gx[k, at:at + 300001].float(), want_gx[0, at:at + 300001].float()
            assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() * (1 + 2.0 ** -6) + 320 * U * scale * 1.01 * steep * (1 + 1.01 * most) ** 2).all())


def test_dropout_of_what_is_not_finite(dev):
    x = torch.full((4, 64, 8), float("inf"), device=dev)
    x[2:] = float("nan")
    y = sfm_amd.dropout(x, sfm_amd.DropoutMask(0.5, (3, 1)))
    keep = torch.from_numpy(R.keep_mask((4, 64, 8), 32768, 3, 1).copy()).to(dev)
    assert (y[~keep] == 0).all() and torch.isinf(y[:2][keep[:2]]).all() and torch.isnan(y[2:][keep[2:]]).all()


def test_probability_zero_changes_nothing(dev):
    x, gy, gamma, beta = inputs((2, 33, 24), torch.float32, 81, dev)
    mask = sfm_amd.DropoutMask(0.0, (3, 1))
    assert torch.equal(sfm_amd.dropout(x, mask), x)
    assert torch.equal(sfm_amd.group_norm_act(x, gamma, beta, 4, dropout=mask), sfm_amd.group_norm_act(x, gamma, beta, 4))


def test_shards_draw_what_the_whole_batch_draws(dev):
    x, gy, gamma, beta = inputs((6, 20, 40), torch.bfloat16, 91, dev)
    mask = lambda first: sfm_amd.DropoutMask(0.4, (11, 4), layer=1, first_item=first)  # noqa: E731
    whole = sfm_amd.group_norm_act(x, gamma, beta, 5, dropout=mask(0))
    parts = torch.cat([sfm_amd.group_norm_act(x[a:b], gamma, beta, 5, dropout=mask(a)) for a, b in ((0, 1), (1, 4), (4, 6))])
    assert torch.equal(whole, parts)
    assert torch.equal(sfm_amd.dropout(x, mask(0))[4:], sfm_amd.dropout(x[4:], mask(4)))


def test_fused_mask_is_the_mask_alone(dev):
    x, gy, gamma, beta = inputs((3, 21, 40), torch.float32, 95, dev)
    for per_channel in (False, True):
        mask = sfm_amd.DropoutMask(0.3, (8, 1), per_channel=per_channel)
        assert torch.equal(sfm_amd.group_norm_act(x, gamma, beta, 5, dropout=mask),
                           sfm_amd.dropout(sfm_amd.group_norm_act(x, gamma, beta, 5), mask))


def test_seed_and_step_on_the_device(dev):
    """the kernels read the tensor when they run; a backward that finds it changed raises"""
    x, gy, gamma, beta = inputs((2, 30, 24), torch.float32, 97, dev)
    x.requires_grad_(True)
    rng = torch.tensor([-5, 2 ** 32 + 8], dtype=torch.int64, device=dev)
    on_device, on_host = sfm_amd.DropoutMask(0.3, rng), sfm_amd.DropoutMask(0.3, (2 ** 64 - 5, 8))
    for f in (lambda m: sfm_amd.dropout(x, m), lambda m: sfm_amd.group_norm_act(x, gamma, beta, 4, dropout=m)):
        a, b = f(on_device), f(on_host)
        assert torch.equal(a, b)
        assert torch.equal(*(torch.autograd.grad(v, x, gy)[0] for v in (a, b)))
        late = f(on_device)
        rng[1] += 1
        assert not torch.equal(f(on_device), late)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(late, x, gy)
        rng[1] -= 1


# ---- how it is used
def test_saved_tensors_elsewhere(dev):
    """what is saved may come back as other tensors (here through the host), and a graph may be run twice"""
    x, gy, gamma, beta = inputs((3, 200, 40), torch.float32, 99, dev)
    mask = sfm_amd.DropoutMask(0.2, torch.tensor([4, 4], device=dev))
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, 5, dropout=mask)
    want = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, gy), want))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, gy)
    with torch.autograd.graph.save_on_cpu():
        y = sfm_amd.group_norm_act(*leaves, 5, dropout=mask)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, gy), want))
    y = torch.utils.checkpoint.checkpoint(lambda *a: sfm_amd.group_norm_act(*a, 5, dropout=mask), *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, gy), want))


def test_threads(dev):
    """two Python threads, each on a stream of its own, forward and backward"""
    import threading
    x, gy, gamma, beta = inputs((4, 900, 48), torch.bfloat16, 102, dev)
    mask = sfm_amd.DropoutMask(0.1, (1, 1))

    def step():
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, gamma, beta)]
        y = sfm_amd.group_norm_act(*leaves, 6, dropout=mask)
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))
    want, got = step(), [None, None]
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[k] = [step() for _ in range(10)]
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for runs in got for r in runs for a, b in zip(r, want))


def test_reproducible(dev):
    x, gy, gamma, beta = inputs((4, 500, 48), torch.float32, 101, dev)
    mask = sfm_amd.DropoutMask(0.1, (1, 1))
    runs = []
    for _ in range(3):
        leaves = [t.clone().requires_grad_(True) for t in (x, gamma, beta)]
        y = sfm_amd.group_norm_act(*leaves, 6, dropout=mask)
        runs.append((y.detach(), *torch.autograd.grad(y, leaves, gy)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_two_streams_at_once(dev):
    x, gy, gamma, beta = inputs((4, 3000, 64), torch.float32, 103, dev)
    want = [sfm_amd.group_norm_act(x * k, gamma, beta, 8) for k in (1.0, 2.0)]
    ins = [x * k for k in (1.0, 2.0)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[k].append(sfm_amd.group_norm_act(ins[k], gamma, beta, 8))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in outs[k])


def test_captured_step(dev):
    """a captured forward and backward follow the step on the device; every replay against the eager result, with eager work between"""
    x, gy, gamma, beta = inputs((4, 600, 48), torch.bfloat16, 105, dev)
    rng = torch.tensor([77, 0], dtype=torch.int64, device=dev)
    mask = sfm_amd.DropoutMask(0.2, rng)

    def step(x):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, gamma, beta)]
        y = sfm_amd.group_norm_act(*leaves, 6, dropout=mask)
        z = sfm_amd.dropout(y, mask.for_layer(1))
        return (z.detach(), *torch.autograd.grad(z, leaves, gy))

    static = x.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    seen = []
    for k in range(4):
        rng.copy_(torch.tensor([77, k], dtype=torch.int64))
        static.copy_(x * (1 + k))
        graph.replay()
        got = [o.clone() for o in out]
        want = step(x * (1 + k))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {k}"
        seen.append(got[0])
    assert not torch.equal(seen[0] == 0, seen[1] == 0)


def test_capture_refuses_leaves_that_an_eager_graph_holds(dev):
    x, _, gamma, beta = inputs((2, 40, 32), torch.float32, 109, dev)
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    mask = sfm_amd.DropoutMask(0.2, (1, 2))
    alive = sfm_amd.group_norm_act(*leaves, 4)
    for call in (lambda: sfm_amd.group_norm_act(*leaves, 4), lambda: sfm_amd.group_norm_act(x.detach(), gamma, beta.detach(), 4),
                 lambda: sfm_amd.dropout(x, mask)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = x.detach() + 1  # (a capture of nothing is warned of)
            with pytest.raises(RuntimeError, match="stream capture"):
                call()
            with torch.no_grad():  # no backward: nothing is in the way
                y = sfm_amd.group_norm_act(*leaves, 4)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, alive) and torch.equal(kept, x.detach() + 1)
    buckets = sfm_amd.GradBuckets([beta, gamma])  # (the node in Python)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = x.detach() + 1
            with pytest.raises(RuntimeError, match="stream capture"):
                sfm_amd.group_norm_act(*leaves, 4)
    finally:
        buckets.release()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(sfm_amd.group_norm_act(*leaves, 4).square().mean(), leaves)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    want = torch.autograd.grad(sfm_amd.group_norm_act(*leaves, 4).square().mean(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_are_born_in_the_buckets(dev):
    x, gy, gamma, beta = inputs((2, 40, 32), torch.float32, 107, dev)
    g, b = gamma.clone().requires_grad_(True), beta.clone().requires_grad_(True)
    want = torch.autograd.grad(sfm_amd.group_norm_act(x, g, b, 4), (g, b), gy)
    buckets = sfm_amd.GradBuckets([b, g])
    try:
        sfm_amd.group_norm_act(x, g, b, 4).backward(gy)
        assert torch.equal(buckets.grad(g), want[0]) and torch.equal(buckets.grad(b), want[1])
        assert g.grad.data_ptr() == buckets.grad(g).data_ptr()
    finally:
        buckets.release()


def test_refusals_with_device_tensors(dev):
    x, g = torch.zeros(2, 3, 8, device=dev), torch.ones(8, device=dev)
    for kw, err in ((dict(groups=3), ValueError), (dict(groups=0), ValueError), (dict(groups=16), ValueError), (dict(groups=2.0), TypeError),
                    (dict(groups=2, epsilon=0.0), ValueError), (dict(groups=2, epsilon=float("nan")), ValueError),
                    (dict(groups=2, epsilon=1e-50), ValueError), (dict(groups=2, epsilon=1e39), ValueError),
                    (dict(groups=2, activation="gelu"), ValueError), (dict(groups=2, activation=True), ValueError),
                    (dict(groups=2, dropout=0.5), TypeError),
                    (dict(groups=2, dropout=sfm_amd.DropoutMask(0.1, (1, 2), first_item=2 ** 32 - 1)), ValueError)):
        with pytest.raises(err):
            sfm_amd.group_norm_act(x, g, g, **kw)
    with pytest.raises(ValueError):
        sfm_amd.group_norm_act(x, g[:4], g, 2)
    with pytest.raises(TypeError):
        sfm_amd.group_norm_act(x, g.half(), g, 2)
    with pytest.raises(TypeError):
        sfm_amd.group_norm_act(x, g.cpu(), g, 2)
    with pytest.raises(ValueError):
        sfm_amd.group_norm_act(g, g, g, 2)
    with pytest.raises(ValueError, match="channels"):
        sfm_amd.dropout(g[:1].expand(1, 2 ** 31), sfm_amd.DropoutMask(0.1, (1, 2)))
    with pytest.raises(TypeError):
        sfm_amd.dropout(x, 0.5)
    with pytest.raises(ValueError):
        sfm_amd.DropoutMask(0.1, torch.zeros(4, dtype=torch.int64, device=dev)[::2])
    x.requires_grad_(True)
    for y in (sfm_amd.group_norm_act(x, g, g, 2), sfm_amd.dropout(x, sfm_amd.DropoutMask(0.1, (1, 2)))):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), x, create_graph=True)
