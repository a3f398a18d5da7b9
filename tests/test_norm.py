"""CPU checks of group norm and dropout: the oracle against known answers, against differences and against torch; what the package
and the C ABI refuse (nothing here reaches a kernel)."""
import ctypes

import numpy as np
import pytest
import torch

import sfm_amd
from oracle import norm_ref as R
from sfm_amd import _lib


def test_philox_known_answers():
    """the generator's published test vectors: zero counter and key, all ones, and digits of pi, at seven and at ten rounds"""
    pi = ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0])
    ones = ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2)
    zero = ([0] * 4, [0] * 2)
    want = {(7, "zero"): "5f6fb709 0d893f64 4f121f81 4f730a48", (10, "zero"): "6627e8d5 e169c58d bc57ac4c 9b00dbd8",
            (10, "ones"): "408f276d 41c83b0e a20bc7c6 6d5451fd", (10, "pi"): "d16cfe09 94fdcceb 5001e420 24126ea1"}
    for (rounds, name), words in want.items():
        c, k = {"zero": zero, "ones": ones, "pi": pi}[name]
        got = R.philox(np.array(c, dtype=np.uint64), np.array(k, dtype=np.uint64), rounds)
        assert " ".join("%08x" % int(w) for w in got) == words, (rounds, name)


def test_mask_is_a_function_of_place_and_its_share_is_the_probability():
    t = 16384
    a = R.keep_mask((4, 50, 7, 24), t, seed=2 ** 40 + 5, step=9, layer=2)
    n = a.size
    assert abs(a.mean() - 0.75) <= 5 * (0.75 * 0.25 / n) ** 0.5
    assert np.array_equal(a[2:], R.keep_mask((2, 50, 7, 24), t, seed=2 ** 40 + 5, step=9, layer=2, first_item=2))
    assert np.array_equal(a.reshape(4, 350, 24), R.keep_mask((4, 350, 24), t, seed=2 ** 40 + 5, step=9, layer=2))     # rows are counted, not heights
    for other in ({"seed": 5}, {"step": 10}, {"layer": 3}, {"first_item": 4}):
        b = R.keep_mask(a.shape, t, **{**dict(seed=2 ** 40 + 5, step=9, layer=2), **other})
        assert 0.3 < (a == b).mean() < 0.8                                                        # 0.75^2 + 0.25^2 = 0.625 agree
    c = R.keep_mask(a.shape, t, seed=3, per_channel=True)
    assert (c == c[:, :1, :1]).all() and c[:, 0, 0].any() and not c[:, 0, 0].all()


@pytest.mark.parametrize("kind", ["elu", "silu", "none"])
def test_oracle_gradient_against_differences(kind):
    g = np.random.default_rng(3)
    x, gamma, beta = g.normal(size=(2, 5, 6)), 1 + 0.1 * g.normal(size=6), 0.1 * g.normal(size=6)
    gy = g.normal(size=x.shape)
    keep = R.keep_mask(x.shape, 20000, seed=1)
    kw = dict(groups=3, eps=1e-5, kind=kind, keep=keep, threshold=20000)
    got = R.group_norm_act(x, gamma, beta, gy=gy, **kw)
    f = lambda *a: (R.group_norm_act(*a, **kw)["y"] * gy).sum()  # noqa: E731
    for k, name in enumerate(("gx", "ggamma", "gbeta")):
        args = [x, gamma, beta]
        v = g.normal(size=args[k].shape)
        h = 1e-5
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * v, args[k] - h * v
        assert abs((f(*up) - f(*down)) / (2 * h) - (got[name] * v).sum()) <= 1e-6 * np.abs(got[name] * v).sum(), name


def test_oracle_against_torch():
    x = torch.randn(3, 4, 5, 12, dtype=torch.float64)
    w, b = torch.randn(12, dtype=torch.float64), torch.randn(12, dtype=torch.float64)
    want = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 4, w, b, 1e-5).permute(0, 2, 3, 1)
    for kind, f in (("none", lambda t: t), ("elu", torch.nn.functional.elu), ("relu", torch.relu), ("silu", torch.nn.functional.silu)):
        np.testing.assert_allclose(R.group_norm_act(x, w, b, 4, 1e-5, kind)["y"], f(want).numpy(), rtol=1e-12, atol=1e-12)


def test_autograd_module_is_built():
    from sfm_amd import norm
    assert callable(norm._nodes().group_norm_act) and callable(norm._nodes().dropout)


# ---- refusals
def test_cpu_tensors_are_rejected():
    x, g = torch.zeros(2, 3, 8), torch.ones(8)
    with pytest.raises(TypeError, match="no CPU fallback"):
        sfm_amd.group_norm_act(x, g, g, 4)
    with pytest.raises(TypeError, match="no CPU fallback"):
        sfm_amd.dropout(x, sfm_amd.DropoutMask(0.1, (1, 2)))
    with pytest.raises(TypeError):
        sfm_amd.group_norm_act([1.0], g, g, 4)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        sfm_amd.group_norm_act(x.double(), g, g, 4)


@pytest.mark.parametrize("kw", [dict(p=-0.1), dict(p=1.0), dict(p=float("nan")), dict(p=1 - 2 ** -18), dict(layer=-1), dict(layer=2 ** 32),
                                dict(first_item=-1), dict(first_item=2 ** 32)])
def test_mask_refuses_values(kw):
    with pytest.raises(ValueError):
        sfm_amd.DropoutMask(**{**dict(p=0.1, rng=(1, 2)), **kw})


@pytest.mark.parametrize("kw", [dict(layer=1.0), dict(first_item=0.5), dict(rng=(1.0, 2)), dict(rng=(1, "2"))], ids=str)
def test_mask_refuses_counters_that_are_no_integers(kw):
    with pytest.raises(TypeError):
        sfm_amd.DropoutMask(0.1, **{"rng": (1, 2), **kw})


def test_mask_refuses_types_and_takes_the_nearest_probability():
    with pytest.raises(TypeError):
        sfm_amd.DropoutMask(0.1, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError):
        sfm_amd.DropoutMask(0.1, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError, match="ints"):
        sfm_amd.DropoutMask(0.1, torch.zeros(2, dtype=torch.int64))      # on the CPU
    m = sfm_amd.DropoutMask(0.1, (-1, 2 ** 32 + 7), layer=4, per_channel=True, first_item=9)
    assert m.threshold == 6554 and m.probability == 6554 / 65536 and m.seed == 2 ** 64 - 1 and m.step == 7
    n = m.for_layer(5)
    assert (n.layer, n.threshold, n.seed, n.step, n.per_channel, n.first_item) == (5, m.threshold, m.seed, m.step, True, 9)
    assert sfm_amd.DropoutMask(1e-6, (1, 2)).threshold == 0


F = 0x10000  # stands for a device address: the calls below are refused before anything is read


def _fwd(**kw):
    a = dict(x=F, ld_x=8, dtype=0, gamma=F, beta=F, B=2, N=3, C=8, G=4, eps=1e-5, act=1, rng=None, seed=0, step=0, layer=0, item0=0,
             threshold=0, per_channel=0, y=F, ld_y=8, mean=F, rstd=F, ws=F, stream=None)
    a.update(kw)
    return _lib.load().sfm_group_norm_act_fwd(*a.values())


@pytest.mark.parametrize("kw", [dict(x=None), dict(gamma=None), dict(beta=None), dict(y=None), dict(ws=None), dict(ws=F + 4), dict(B=0),
                                dict(N=0), dict(C=0), dict(G=0), dict(G=3), dict(dtype=3), dict(dtype=-1), dict(ld_x=7), dict(ld_y=7),
                                dict(x=F + 2), dict(dtype=1, x=F + 1), dict(eps=0.0), dict(eps=float("nan")), dict(act=4), dict(act=-1),
                                dict(mean=None), dict(rstd=None), dict(threshold=-1), dict(threshold=65536), dict(rng=F + 4)],
                         ids=lambda kw: ",".join(kw))
def test_forward_refuses(kw):
    assert _fwd(**kw) == -1


@pytest.mark.parametrize("kw", [dict(B=2 ** 31), dict(B=2 ** 22), dict(N=2 ** 40), dict(ld_x=2 ** 29), dict(ld_y=2 ** 29), dict(C=2 ** 22, G=2 ** 20, ld_x=2 ** 22, ld_y=2 ** 22), dict(threshold=9, N=2 ** 33), dict(threshold=9, item0=2 ** 32 - 1)],
                         ids=lambda kw: ",".join(kw))
def test_forward_refuses_what_its_counters_do_not_hold(kw):
    assert _fwd(**kw) == -2


def _bwd(gy=(F,), ld=(8,), n=None, **kw):
    a = dict(x=F, ld_x=8, dtype=0, gy=(ctypes.c_void_p * len(gy))(*gy), ld_gy=(ctypes.c_longlong * len(ld))(*ld),
             n_gy=len(gy) if n is None else n, gamma=F, beta=F, mean=F, rstd=F, B=2, N=3, C=8, G=4, act=1, rng=None, seed=0, step=0,
             layer=0, item0=0, threshold=0, per_channel=0, gx=F, ggamma=F, gbeta=F, ws=F, stream=None)
    a.update(kw)
    return _lib.load().sfm_group_norm_act_bwd(*a.values())


@pytest.mark.parametrize("kw", [dict(x=None), dict(n=0), dict(n=4), dict(gy=(None,)), dict(ld=(7,)), dict(gy=(F, F + 2), ld=(8, 8)),
                                dict(gamma=None), dict(beta=None), dict(mean=None), dict(rstd=None), dict(gx=None, ggamma=None, gbeta=None),
                                dict(gx=F + 2), dict(ggamma=None), dict(gbeta=None), dict(ws=None), dict(ws=F + 4), dict(G=5),
                                dict(act=9), dict(threshold=65536)], ids=lambda kw: ",".join(kw))
def test_backward_refuses(kw):
    assert _bwd(**kw) == -1


def _drop(**kw):
    a = dict(x=F, dtype=0, items=2, elems=24, C=8, rng=None, seed=0, step=0, layer=0, item0=0, threshold=1, per_channel=0, y=F, stream=None)
    a.update(kw)
    return _lib.load().sfm_dropout(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(x=None), -1), (dict(y=None), -1), (dict(dtype=3), -1), (dict(items=0), -1), (dict(elems=0), -1),
                                   (dict(C=0), -1), (dict(C=7), -1), (dict(x=F + 2), -1), (dict(y=F + 1, dtype=1), -1),
                                   (dict(threshold=65536), -1), (dict(threshold=-1), -1), (dict(rng=F + 4), -1),
                                   (dict(items=2 ** 32, item0=1), -2), (dict(elems=2 ** 38), -2),
                                   (dict(items=2 ** 31, elems=16), -2), (dict(items=2 ** 20, elems=2 ** 41), -2)], ids=lambda v: str(v))
def test_dropout_refuses(kw, rc):
    assert _drop(**kw) == rc


def test_workspace():
    f = _lib.load().sfm_group_norm_workspace_floats
    assert f(2, 100, 64, 8, 0, 0) > 0 and f(2, 100, 64, 8, 0, 1) > f(2, 100, 64, 8, 0, 0)
    assert f(0, 100, 64, 8, 0, 0) == -1 and f(2, 100, 64, 7, 0, 0) == -1 and f(2 ** 31, 1, 64, 8, 0, 0) == -2
