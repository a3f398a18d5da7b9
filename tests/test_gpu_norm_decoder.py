"""Group norm and dropout where the framework uses them: the decoder level as one autograd node and composed, against float64, in
training and in serving, and a captured training step of the decoder into the loss.

Tolerances against float64, relative to the largest value: a convolution adds K <= 1152 products in fp32, at most K u = 7e-5 of the sum
of their sizes, and a level is four convolutions and norms deep: 3e-4 for outputs, ten times that for gradients, which pass the same
depth twice and are sums over pixels with cancellation (what the batch-norm decoder's tests allow at that depth)."""
import copy

import pytest
import torch

import sfm_amd
from oracle import norm_ref as NR
from sfm_amd import aspp as A
from sfm_amd import synth
from helpers import rel_err

pytestmark = pytest.mark.gpu
TOL_OUT, TOL_GRAD = 3e-4, 3e-3

LEVELS = [(64, 32, (2, 4), True, False), (64, 32, (3, 6), True, True), (32, 64, (3, 6), False, True)]
MASKS = [None, dict(p=0.2, per_channel=False), dict(p=0.3, per_channel=True)]


def block(g, cin, cout, use_skip, use_skip2):
    def conv(k, ci, co):
        return dict(w=torch.randn(k, k, ci, co, generator=g) / (k * ci ** 0.5), gamma=1 + 0.1 * torch.randn(co, generator=g),
                    beta=0.1 * torch.randn(co, generator=g))
    p = dict(up=conv(1, cin, cin), sup=conv(1, cin, cout), aspp_up=conv(3, cin, cout), aspp_up2=conv(3, 2 * cout, cout))
    if use_skip:
        p["skip_bn"] = dict(gamma=1 + 0.1 * torch.randn(96, generator=g), beta=0.1 * torch.randn(96, generator=g))
        p["skip"] = conv(1, 96, cout)
    else:
        p["skip"] = conv(3, 2 * cout, cout)
    if use_skip2:
        p["skip2"] = conv(1, cin, cout)
    p["out"] = conv(1, (5 if use_skip2 else 4) * cout, cout)
    return p


def level_inputs(g, cin, use_skip, use_skip2, B=3, h=5, w=9):
    return dict(concat=torch.randn(B, h, w, cin, generator=g), skip_feat=torch.randn(B, 2 * h, 2 * w, 96, generator=g) if use_skip else None,
                skip2=torch.randn(B, h - 1, w - 2, cin, generator=g) if use_skip2 else None)


def leaves_of(params, inputs):
    out = {f"in.{k}": v for k, v in inputs.items() if v is not None}
    out.update({f"{k}.{kk}": vv for k, v in params.items() for kk, vv in v.items()})
    return out


def on(tree, f):
    return {k: on(v, f) if isinstance(v, dict) else None if v is None else f(v) for k, v in tree.items()}


def mask_of(spec, dev, on_device):
    if spec is None:
        return None, None
    seed, step = 77 + 2 ** 40, 5
    m = sfm_amd.DropoutMask(spec["p"], torch.tensor([seed, step], device=dev) if on_device else (seed, step), layer=100,
                            per_channel=spec["per_channel"], first_item=4)
    return m, dict(threshold=m.threshold, seed=seed, step=step, layer=100, per_channel=spec["per_channel"], first_item=4)


@pytest.mark.parametrize("spec", MASKS, ids=["plain", "element", "channel"])
@pytest.mark.parametrize("cin,cout,rates,use_skip,use_skip2", LEVELS)
def test_level(dev, cin, cout, rates, use_skip, use_skip2, spec):
    """one node, composed, and float64: outputs and the gradient of every input and parameter"""
    g = torch.Generator().manual_seed(5)
    params, inputs = block(g, cin, cout, use_skip, use_skip2), level_inputs(g, cin, use_skip, use_skip2)
    B, h, w = inputs["concat"].shape[:3]
    wy, wu = torch.randn(B, 2 * h, 2 * w, cout, generator=g), torch.randn(B, 2 * h, 2 * w, cin, generator=g)
    _, plain = mask_of(spec, dev, False)
    po, io = (on(t, lambda v: v.double().requires_grad_(True)) for t in (params, inputs))
    yo, uo = NR.level(po, io["concat"], io["skip_feat"], rates, use_skip, use_skip2, io["skip2"], 8, plain)
    ((yo * wy).sum() + (uo * wu).sum()).backward()
    want = {k: v.grad for k, v in leaves_of(po, io).items()}
    runs = []
    for fused in (True, False):
        pg, ig = (on(t, lambda v: v.to(dev).requires_grad_(True)) for t in (params, inputs))
        y, u = sfm_amd.disp_bottleneck_dense(pg, ig["concat"], ig["skip_feat"], rates, use_skip, use_skip2, ig["skip2"], fused_level=fused,
                                             groups=8, dropout=mask_of(spec, dev, fused)[0])
        ((y * wy.to(dev)).sum() + (u * wu.to(dev)).sum()).backward()
        assert rel_err(y, yo) <= TOL_OUT and rel_err(u, uo) <= TOL_OUT
        got = {k: v.grad for k, v in leaves_of(pg, ig).items()}
        floor = 1e-3 * max(float(v.abs().max()) for v in want.values())
        bad = {k: rel_err(got[k], want[k], floor) for k in want if rel_err(got[k], want[k], floor) > TOL_GRAD}
        assert not bad, (fused, bad)
        runs.append((y.detach(), u.detach(), got))
    (yf, uf, gf), (yc, uc, gc) = runs
    assert torch.equal(yf, yc) and torch.equal(uf, uc)
    # the node sums the gradients of an activation's readers while loading, autograd in tensors of its own: another order
    assert all(rel_err(gf[k], gc[k], 1e-6 * max(float(v.abs().max()) for v in gc.values())) <= 2e-5 for k in gf)


def test_level_serves_what_it_trains(dev):
    """is_training=False: the same function without the mask, no moving statistics, no graph"""
    g = torch.Generator().manual_seed(6)
    params, inputs = block(g, 64, 32, True, True), level_inputs(g, 64, True, True)
    pg, ig = (on(t, lambda v: v.to(dev).requires_grad_(True)) for t in (params, inputs))
    mask, _ = mask_of(MASKS[1], dev, True)
    args = (pg, ig["concat"], ig["skip_feat"], (3, 6), True, True, ig["skip2"])
    y, u = sfm_amd.disp_bottleneck_dense(*args, is_training=False, groups=8, dropout=mask)
    yt, ut = sfm_amd.disp_bottleneck_dense(*args, groups=8)
    assert torch.equal(y, yt) and torch.equal(u, ut) and not y.requires_grad
    # one item alone gives what it gives in the batch (batch norm's does not)
    one = {k: v[1:2].detach() for k, v in ig.items()}
    y1, _ = sfm_amd.disp_bottleneck_dense(pg, one["concat"], one["skip_feat"], (3, 6), True, True, one["skip2"], is_training=False, groups=8)
    assert rel_err(y1, y[1:2]) <= 1e-5   # (the convolutions cut their sums by the number of rows)


def test_batch_norm_level_with_dropout(dev):
    """behind a batch norm the mask is an operator of its own: the level composed by hand gives the same"""
    g = torch.Generator().manual_seed(7)
    params, inputs = block(g, 64, 32, False, True), level_inputs(g, 64, False, True)
    mask, _ = mask_of(MASKS[1], dev, True)
    p, i = (on(t, lambda v: v.to(dev)) for t in (params, inputs))
    y, _ = sfm_amd.disp_bottleneck_dense(p, i["concat"], None, (3, 6), False, True, i["skip2"], dropout=mask)
    H, W = 2 * i["concat"].shape[1], 2 * i["concat"].shape[2]

    def conv(x, nm, rate=None, draw=None, act=True):
        q = p[nm]
        v = sfm_amd.conv1x1(x, q["w"]) if rate is None else sfm_amd.dilated_conv3x3(x, q["w"], rate)
        v = sfm_amd.batch_norm_elu(v, q["gamma"], q["beta"], activation=act)
        return v if draw is None else sfm_amd.dropout(v, mask.for_layer(100 + draw))
    up = conv(sfm_amd.resize_bilinear(i["concat"], H, W), "up", act=False)
    s, a1 = conv(up, "sup", draw=0), conv(up, "aspp_up", 3, 1)
    a2 = conv(torch.cat([s, a1], 3), "aspp_up2", 6, 2)
    k = conv(torch.cat([a1, a2], 3), "skip", 12, 3)
    k2 = conv(sfm_amd.resize_bilinear(i["skip2"], H, W), "skip2", draw=4)
    assert torch.equal(y, conv(torch.cat([s, a1, a2, k, k2], 3), "out", act=False))
    assert 0.1 < float((s == 0).double().mean()) < 0.3


def test_refusals(dev):
    g = torch.Generator().manual_seed(8)
    params, inputs = block(g, 64, 32, False, True), level_inputs(g, 64, False, True)
    p, i = (on(t, lambda v: v.to(dev)) for t in (params, inputs))
    call = lambda **kw: sfm_amd.disp_bottleneck_dense(p, i["concat"], None, (3, 6), False, True, i["skip2"], **kw)  # noqa: E731
    for kw, err in ((dict(groups=5), ValueError), (dict(groups=0), ValueError), (dict(groups=64), ValueError), (dict(dropout=0.5), TypeError),
                    (dict(groups=8, dropout=sfm_amd.DropoutMask(0.1, (1, 2), layer=2 ** 32 - 2)), ValueError),
                    (dict(groups=8, dropout=sfm_amd.DropoutMask(0.1, (1, 2), first_item=2 ** 32 - 1)), ValueError)):
        for fused in (True, False):
            with pytest.raises(err):
                call(fused_level=fused, **kw)
    with pytest.raises(TypeError):
        sfm_amd.disp_aspp_u_dense_decoder(A.make_end_points(1, 1, 1, dev, width_div=64), A.make_decoder_params(dev, width_div=64), groups=8,
                                          dropout=0.5)
    # a step that has been advanced between a level's forward and its backward
    rng = torch.tensor([1, 2], device=dev)
    x = i["concat"].clone().requires_grad_(True)
    y, _ = sfm_amd.disp_bottleneck_dense(p, x, None, (3, 6), False, True, i["skip2"], groups=8, dropout=sfm_amd.DropoutMask(0.1, rng))
    rng[1] += 1
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()


def _params(params, dev, dtype=torch.float32):
    return on(copy.deepcopy(params), lambda v: v.detach().to(dev, dtype).requires_grad_(True))


def _flat(tree, at=""):
    for k in sorted(tree):
        yield from _flat(tree[k], f"{at}{k}.") if isinstance(tree[k], dict) else [(at + k, tree[k])]


def test_decoder_into_the_loss(dev):
    """decoder with group norm and dropout -> disparities -> loss -> every parameter's gradient, against float64 through the decoder;
    the mask's elements are 30 % of five activations in each of five levels"""
    B, h, w, div = 2, 2, 3, 8
    params, ends = A.make_decoder_params("cpu", 31, div), A.make_end_points(B, h, w, "cpu", 31, div)
    mask, plain = mask_of(dict(p=0.3, per_channel=False), dev, True)
    po, pg = _params(params, "cpu", torch.float64), _params(params, dev)
    do = NR.decoder({k: v.double() for k, v in ends.items()}, po, 8, plain)
    dg = sfm_amd.disp_aspp_u_dense_decoder({k: v.to(dev) for k, v in ends.items()}, pg, groups=8, dropout=mask)
    for a, b in zip(dg, do):
        assert rel_err(a, b) <= 1e-3, rel_err(a, b)     # five levels deep: three times a level's
    g = torch.Generator().manual_seed(32)
    up = [torch.randn(t.shape, generator=g) for t in do]
    sum((a * b).sum() for a, b in zip(do, up)).backward()
    sum((a * b.to(dev)).sum() for a, b in zip(dg, up)).backward()
    floor = 1e-3 * max(float(v.grad.abs().max()) for _, v in _flat(po))
    bad = {n: rel_err(a.grad, b.grad, floor) for (n, a), (_, b) in zip(_flat(pg), _flat(po)) if rel_err(a.grad, b.grad, floor) > 1e-2}
    assert not bad, bad
    # and as it is used: the three maps into the loss, differentiated down to the decoder's first layer
    inp = synth.to_device(synth.make_inputs(B, 32 * h, 32 * w, S=3, N=2, seed=33, full_res=False), dev)
    pg = _params(params, dev)
    disp = sfm_amd.disp_aspp_u_dense_decoder({k: v.to(dev) for k, v in ends.items()}, pg, groups=8, dropout=mask)
    dn, depth = sfm_amd.normalize_disp(disp)
    loss = sfm_amd.multi_scale_loss(inp["tgt"], inp["src"], inp["K"], depth, inp["pose"], inp["trans"], pred_disp=dn, smooth_weight=0.01)
    loss.backward()
    assert torch.isfinite(loss) and all(torch.isfinite(v.grad).all() for _, v in _flat(pg))
    assert float(pg["stem"]["w"].grad.abs().max()) > 0


def test_captured_training_steps(dev):
    """a decoder step captured once and replayed with the step advanced on the device: each replay against the eager step of that number"""
    B, h, w, div = 1, 2, 3, 16
    params, ends = A.make_decoder_params(dev, 41, div), A.make_end_points(B, h, w, dev, 41, div)
    rng = torch.tensor([9, 0], device=dev)
    mask = sfm_amd.DropoutMask(0.25, rng)
    up = [torch.randn(B, 32 * h >> k, 32 * w >> k, 1, device=dev) for k in range(3)]

    def step():
        p = _params(params, dev)
        disp = sfm_amd.disp_aspp_u_dense_decoder(ends, p, groups=8, dropout=mask)
        flat = [v for _, v in _flat(p)]
        return [d.detach() for d in disp], torch.autograd.grad(disp, flat, up)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = step()
    seen = []
    for k in range(4):
        rng.copy_(torch.tensor([9, k]))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out, *grads)]
        eo, eg = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (*eo, *eg))), k
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def test_capture_refuses_a_level_whose_parameters_an_eager_graph_holds(dev):
    g = torch.Generator().manual_seed(43)
    params = on(block(g, 64, 32, True, False), lambda t: t.to(dev).requires_grad_(True))
    x = on(level_inputs(g, 64, True, False), lambda t: t.to(dev))
    run = lambda: sfm_amd.disp_bottleneck_dense(params, x["concat"], x["skip_feat"], use_skip2=False, groups=8)[0]  # noqa: E731
    alive = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = x["concat"] + 1  # (a capture of nothing is warned of)
        with pytest.raises(RuntimeError, match="stream capture"):
            run()
        with torch.no_grad():
            y = run()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alive) and torch.equal(kept, x["concat"] + 1)
