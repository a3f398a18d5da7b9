"""Group norm and dropout at the edges of what their documentation allows."""
import numpy as np
import pytest
import torch

import sfm_amd
from oracle import norm_ref as R
from test_gpu_norm import HALF, TINY, U, compare, f64, inputs, within
from test_gpu_norm_decoder import block, level_inputs, on

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


# ---- values
# one launch forward; several chunks of rows; groups wider than a workgroup; an odd channel count
FORMS = [((2, 100, 32), 4), ((2, 5000, 32), 8), ((2, 19, 4096), 1), ((3, 37, 53, 45), 5)]
FORM_IDS = ["held", "chunks", "parts", "odd"]


@pytest.mark.parametrize("scale", [1e-2, 1e-4, 1e-7])
@pytest.mark.parametrize("shift", [0.0, 1.0], ids=["beta0", "beta"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape,groups", FORMS, ids=FORM_IDS)
def test_elu_of_small_values(dev, shape, groups, dtype, shift, scale):
    """with small gamma and beta z is small and as exact, relative to them, as ever; so is elu(z).  z is off by at most 32 roundings of terms
    no larger than |gamma| (|x| + |x - mean|) / std + |beta| (40 u of that), elu adds 2^-20 of itself in fp32, 2^-16 before a 16-bit rounding"""
    x, _, gamma, beta = inputs(shape, dtype, 211, dev)
    gamma, beta = gamma * scale, beta * (scale * shift)
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), groups, 1e-5, "elu")
    size, h = want["z_size"] - 1 + np.abs(f64(beta)), HALF[dtype]
    bound = 40 * U * size + ((2.0 ** -20 if dtype == torch.float32 else 2.0 ** -16) + h * (1 + 2 * h)) * np.abs(want["y"]) + TINY[dtype]
    within(sfm_amd.group_norm_act(x, gamma, beta, groups), want["y"], bound, "y")


# ---- what is kept and who writes it
def _saved(f):
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        return f(), kept


@pytest.mark.parametrize("buckets", [False, True])
def test_a_backward_writes_nothing_that_is_kept(dev, buckets):
    """a graph may be run several times, and its passes captured into graphs of their own that replay side by side: what the node keeps is only
    read, and each pass has a workspace to itself"""
    x, gy, gamma, beta = inputs((4, 900, 48), torch.float32, 221, dev)
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    sink = sfm_amd.GradBuckets([beta, gamma]) if buckets else None
    try:
        y, kept = _saved(lambda: sfm_amd.group_norm_act(*leaves, 6))
        before = [t.detach().clone() for t in kept]
        assert len(kept) == 4
        first = [g.clone() for g in torch.autograd.grad(y, leaves, gy, retain_graph=True)]
        assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(kept, before))
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, gy)))
    finally:
        if sink:
            sink.release()


@pytest.mark.parametrize("per_channel", [False, True])
def test_last_item_of_the_counter(dev, per_channel):
    """first_item plus the batch size may be 2^32"""
    x, gy, gamma, beta = inputs((2, 30, 24), torch.float32, 219, dev)
    mask = sfm_amd.DropoutMask(0.3, (8, 9), per_channel=per_channel, first_item=2 ** 32 - 2)
    keep = torch.from_numpy(R.keep_mask((2, 30, 24), mask.threshold, 8, 9, 0, per_channel, 2 ** 32 - 2).copy()).to(dev)
    plain = sfm_amd.group_norm_act(x, gamma, beta, 4)
    x.requires_grad_(True)
    for y, of in ((sfm_amd.dropout(x, mask), x.detach()), (sfm_amd.group_norm_act(x, gamma, beta, 4, dropout=mask), plain)):
        assert torch.equal(y == 0, ~keep | (of == 0))
        torch.autograd.grad(y, x, gy)


def test_slices_are_read_in_place_with_buckets(dev):
    """a training step under data parallelism (gradients born in buckets) copies no channel slice, of x or of dL/dy"""
    wide = torch.randn(3, 40, 7, 50, device=dev, generator=torch.Generator(device=dev).manual_seed(223))
    _, _, gamma, beta = inputs((1, 1, 24), torch.float32, 224, dev)
    x, gy = wide[..., 3:27].detach().requires_grad_(True), wide[..., 20:44]
    leaves = [x, gamma.requires_grad_(True), beta.requires_grad_(True)]
    want = torch.autograd.grad(sfm_amd.group_norm_act(*leaves, 4), leaves, gy)
    sink = sfm_amd.GradBuckets([beta, gamma])
    try:
        y, kept = _saved(lambda: sfm_amd.group_norm_act(*leaves, 4))
        assert x.data_ptr() in [t.data_ptr() for t in kept]
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        base = torch.cuda.memory_allocated()
        got = torch.autograd.grad(y, leaves, gy)
        # gx, and a workspace and sums that are small beside it
        assert torch.cuda.max_memory_allocated() - base < 1.9 * x.numel() * 4
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # rows that are no slice are copied
        z = torch.randn(3, 24, device=dev).unsqueeze(1).expand(3, 40, 24)
        a, b = (torch.autograd.grad(sfm_amd.group_norm_act(*leaves, 4).sum(dim=(1, 2)), leaves, wide[:, 0, 0, :24]) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        sink.release()
        c = torch.autograd.grad(sfm_amd.group_norm_act(*leaves, 4).sum(dim=(1, 2)), leaves, wide[:, 0, 0, :24])
        assert all(torch.equal(p, q) for p, q in zip(a, c))
        assert torch.equal(sfm_amd.group_norm_act(z, gamma, beta, 4), sfm_amd.group_norm_act(z.contiguous(), gamma, beta, 4))
    finally:
        sink.release()


# ---- in the decoder
def _level(dev):
    g = torch.Generator().manual_seed(225)
    params, ins = block(g, 64, 32, True, True), level_inputs(g, 64, True, True)
    return on(params, lambda t: t.to(dev).requires_grad_(True)), on(ins, lambda t: t.to(dev))


def test_serving_keeps_nothing_for_a_backward(dev, monkeypatch):
    """statistics are saved where a backward may come, and there alone"""
    from sfm_amd import norm
    saved = []

    def spy(name, *args):
        if name == "sfm_group_norm_act_fwd":
            saved.append((args[20] is not None, args[21] is not None))
        return call(name, *args)
    call = norm.call
    monkeypatch.setattr(norm, "call", spy)
    params, ins = _level(dev)
    run = lambda **kw: sfm_amd.disp_bottleneck_dense(params, ins["concat"], ins["skip_feat"], (2, 4), True, True, ins["skip2"], groups=8, **kw)  # noqa: E731

    def how(**kw):
        saved.clear()
        y, up = run(**kw)
        return y.detach(), set(saved), len(saved)
    trained, kept, n = how()
    assert kept == {(True, True)} and n == 8
    served, kept, n = how(is_training=False)
    assert kept == {(False, False)} and n == 8 and torch.equal(served, trained)
    with torch.no_grad():
        assert how()[1] == {(False, False)}
    for q in params.values():
        for t in q.values():
            t.requires_grad_(False)
    assert how()[1] == {(False, False)}       # no leaf wants a gradient
    ins["skip2"].requires_grad_(True)
    assert how()[1] == {(True, True)}


def test_level_draws_under_inference_mode(dev):
    """a tensor made under inference_mode has no version to check, and no backward that would need it"""
    params, ins = _level(dev)
    run = lambda rng: sfm_amd.disp_bottleneck_dense(params, ins["concat"], ins["skip_feat"], (2, 4), True, True, ins["skip2"], groups=8,  # noqa: E731
                                                    dropout=sfm_amd.DropoutMask(0.2, rng))[0]
    want = run((5, 6)).detach()
    with torch.inference_mode():
        assert torch.equal(run(torch.tensor([5, 6], device=dev)), want)


@pytest.mark.parametrize("first_row", [None, -3.0e4], ids=["no outlier", "outlier"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,groups", FORMS, ids=FORM_IDS)
def test_gradients_where_the_mean_is_far_from_the_deviation(dev, shape, groups, dtype, first_row):
    """mean 1000, deviation about 1 (in fp32 a sum of squares less the squared mean leaves nothing of it), or with a first row far off.
    y as in `compare`.  d bounds what z and xhat are off by, the mean's rounding being most of it; then act' is off by d, c1 by d and c2 by
    d (1 + |xhat|) of their largest term, so gx is off by 2 d r s |gamma gy| (1 + |xhat|)^2 beside `compare`'s bound"""
    x, gy, gamma, beta = inputs(shape, torch.float32, 213, dev)
    x = x + 1000.0
    if first_row is not None:
        x[:, 0] = first_row
    x, gy = x.to(dtype), gy.to(dtype)
    want = R.group_norm_act(f64(x), f64(gamma), f64(beta), groups, 1e-5, "elu", f64(gy))
    d = 40 * U * (1 + want["z_size"].max())
    extra = 2 * d * want["rstd"].max() * np.abs(f64(gamma)).max() * np.abs(f64(gy)).max() * (1 + want["xhat_max"]) ** 2
    leaves = [t.requires_grad_(True) for t in (x, gamma, beta)]
    y = sfm_amd.group_norm_act(*leaves, groups)
    compare(y, torch.autograd.grad(y, leaves, gy), want, dtype, loose=(extra, 0.0, 0.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,groups", [((300, 1801, 32), 8), ((300, 1825, 32), 16), ((600, 700, 10), 5), ((500, 613, 36), 9), ((2, 100, 32), 4),
                                          ((2, 19, 4096), 1), ((3, 37, 53, 90), 5), ((1, 1, 8), 2), ((2, 5000, 32), 4)], ids=str)
def test_no_row_is_lost_or_counted_twice(dev, shape, groups, dtype):
    """whole numbers: gbeta = sum gy exactly.  x = +-1 by turns in every group: mean 0, variance 1, ggamma = r sum x gy.  There x - mean, r, the sums'
    product with it and the result are rounded: 8 u of sum |gy|, which is under half a row's share"""
    g = torch.Generator().manual_seed(215)
    C = shape[-1]
    gy = torch.randint(-1, 2, shape, generator=g).to(dtype).to(dev)
    x = (1.0 - 2.0 * (torch.arange(C) % 2)).expand(shape).contiguous().to(dtype).to(dev)
    gamma, beta = (1 + 0.2 * torch.randn(C, generator=g)).to(dev).requires_grad_(True), torch.zeros(C, device=dev, requires_grad=True)
    gg, gb = torch.autograd.grad(sfm_amd.group_norm_act(x, gamma, beta, groups, activation=None), (gamma, beta), gy)
    flat = f64(gy).reshape(-1, C)
    assert np.array_equal(f64(gb), flat.sum(axis=0))
    bound = 8 * U * np.abs(flat).sum(axis=0)
    assert bound.max() < 0.5
    within(gg, (flat * f64(x).reshape(-1, C)).sum(axis=0) / (1 + 1e-5) ** 0.5, bound, "ggamma")


@pytest.mark.parametrize("act", ["elu", "silu", "relu", None])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N", [40, 3001])
def test_gradients_of_what_is_not_finite_stay_in_their_group(dev, N, dtype, act):
    x, gy, gamma, beta = inputs((3, N, 24), dtype, 217, dev)

    def run(x, gy, mask=None):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, gamma, beta)]
        y = sfm_amd.group_norm_act(*leaves, 4, activation=act, dropout=mask)
        return torch.autograd.grad(y, leaves, gy)
    clean = run(x, gy)
    hit, chan = torch.zeros(x.shape, dtype=torch.bool, device=dev), torch.zeros(24, dtype=torch.bool, device=dev)
    hit[1, :, 6:12] = hit[2, :, 18:24] = chan[6:12] = chan[18:24] = True
    for what in ("x", "gy"):
        bad = {"x": x.clone(), "gy": gy.clone()}
        bad[what][1, N - 3, 8] = float("nan")
        bad[what][2, 3, 23] = float("inf")
        if act == "relu" and what == "gy":  # (relu' = 0 there would make it 0, or a NaN of inf * 0: not asked for)
            continue
        gx, gg, gb = run(bad["x"], bad["gy"])
        # a mean that is none makes all NaN; with an infinite gy c1 and c2 are infinite, and -c1 - xhat c2 is that or a NaN
        assert not torch.isfinite(gx[hit]).any() and (what == "gy" or torch.isnan(gx[hit]).all()) and torch.equal(gx[~hit], clean[0][~hit]), what
        if what == "x":
            assert torch.isnan(gg[chan]).all()
        assert torch.equal(gg[~chan], clean[1][~chan]) and torch.equal(gb[~chan], clean[2][~chan]), what
    # a gradient that the mask drops counts for nothing, whatever it is
    mask = sfm_amd.DropoutMask(0.5, (6, 7))
    keep = torch.from_numpy(R.keep_mask(tuple(x.shape), mask.threshold, 6, 7).copy()).to(dev)
    bad = torch.where(keep, gy, torch.full_like(gy, float("nan")))
    assert all(torch.equal(a, b) for a, b in zip(run(x, bad, mask), run(x, gy, mask)))
