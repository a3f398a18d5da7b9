"""Group norm with an activation and counter-based dropout from their definitions, in float64 on the CPU (NumPy): what the kernels
of sfm_amd/csrc/group_norm_fwd.hip, group_norm_bwd.hip and dropout.hip are compared with.  No counterpart in the reference."""
import numpy as np

M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85


def philox(counter, key, rounds=7):
    """Philox 4x32 (Salmon, Moraes, Dror, Shaw, SC 2011).  counter [..., 4], key [..., 2], 32-bit words -> [..., 4]"""
    c = [np.asarray(counter[..., k], dtype=np.uint64) for k in range(4)]
    k0, k1 = (np.asarray(key[..., k], dtype=np.uint64) for k in range(2))
    lo = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(M0), c[2] * np.uint64(M1)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & lo, (a >> np.uint64(32)) ^ c[3] ^ k1, a & lo]
        k0, k1 = (k0 + np.uint64(W0)) & lo, (k1 + np.uint64(W1)) & lo
    return np.stack(c, axis=-1)


def keep_mask(shape, threshold, seed, step=0, layer=0, per_channel=False, first_item=0):
    """truth values of `shape` [B, ..., C]: what is kept"""
    B, C = shape[0], shape[-1]
    n = C if per_channel else int(np.prod(shape[1:]))
    blocks = -(-n // 8)
    ctr = np.zeros((B, blocks, 4), dtype=np.uint64)
    ctr[..., 0] = np.arange(blocks)[None, :]
    ctr[..., 1] = (first_item + np.arange(B))[:, None]
    ctr[..., 2], ctr[..., 3] = step % 2 ** 32, layer
    key = np.array([seed % 2 ** 32, (seed >> 32) % 2 ** 32], dtype=np.uint64)
    w = philox(ctr, np.broadcast_to(key, (B, blocks, 2)))
    u = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], axis=-1).reshape(B, blocks * 8)[:, :n]
    keep = u >= threshold
    return np.broadcast_to(keep.reshape((B,) + (1,) * (len(shape) - 2) + (C,)) if per_channel else keep.reshape(shape), shape)


def act(z, kind):
    if kind == "elu":
        return np.where(z > 0, z, np.expm1(np.minimum(z, 0)))
    if kind == "relu":
        return np.maximum(z, 0)
    if kind == "silu":
        return z / (1 + np.exp(-z))
    return z


def act_grad(z, kind):
    if kind == "elu":
        return np.where(z > 0, 1.0, np.exp(np.minimum(z, 0)))
    if kind == "relu":
        return (z > 0).astype(np.float64)
    if kind == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def group_norm_act(x, gamma, beta, groups, eps, kind, gy=None, keep=None, threshold=0):
    """x [B, ..., C] -> dict of y (and gx, ggamma, gbeta, and the sizes that error bounds are made of)"""
    x, gamma, beta = (np.asarray(a, dtype=np.float64) for a in (x, gamma, beta))
    B, C = x.shape[0], x.shape[-1]
    v = x.reshape(B, -1, groups, C // groups)
    ga, be = gamma.reshape(groups, -1), beta.reshape(groups, -1)
    mean = v.mean(axis=(1, 3), keepdims=True)
    rstd = 1 / np.sqrt(((v - mean) ** 2).mean(axis=(1, 3), keepdims=True) + eps)
    xhat = (v - mean) * rstd
    z = xhat * ga + be
    scale = 1.0 if keep is None else 65536 / (65536 - threshold)
    k = np.ones(v.shape) if keep is None else np.asarray(keep, dtype=np.float64).reshape(v.shape)
    out = {"y": np.where(k > 0, scale * act(z, kind), 0.0).reshape(x.shape), "z": z.reshape(x.shape), "mean": mean.reshape(B, groups),
           "rstd": rstd.reshape(B, groups)}
    if gy is not None:
        dz = np.where(k > 0, scale * np.asarray(gy, dtype=np.float64).reshape(v.shape), 0.0) * act_grad(z, kind)
        dg = dz * ga
        gx = rstd * (dg - dg.mean(axis=(1, 3), keepdims=True) - xhat * (dg * xhat).mean(axis=(1, 3), keepdims=True))
        out.update(gx=gx.reshape(x.shape), ggamma=(dz * xhat).sum(axis=(0, 1)).reshape(C), gbeta=dz.sum(axis=(0, 1)).reshape(C),
                   abs_ggamma=np.abs(dz * xhat).sum(axis=(0, 1)).reshape(C), abs_gbeta=np.abs(dz).sum(axis=(0, 1)).reshape(C),
                   abs_gy=np.where(k > 0, scale * np.abs(np.asarray(gy, dtype=np.float64).reshape(v.shape)), 0.0).sum(axis=(0, 1)).reshape(C),
                   xhat_max=np.abs(xhat).max(),
                   # the largest of each (item, group), broadcast: what an error of gx is measured against
                   gx_size=np.broadcast_to(rstd * np.abs(dg).max(axis=(1, 3), keepdims=True)
                                           * (1 + np.abs(xhat).max(axis=(1, 3), keepdims=True)) ** 2, v.shape).reshape(x.shape))
    out["z_size"] = np.broadcast_to(1 + np.abs(ga).max() * (rstd * np.abs(v).max(axis=(1, 3), keepdims=True)
                                                            + np.abs(xhat).max(axis=(1, 3), keepdims=True)),
                                    v.shape).reshape(x.shape)
    return out


# ---- the decoder with group norm and dropout, in torch float64 on the CPU: ref_graph's wiring with another normaliser
def _torch_norm(x, q, groups, activation, mask, name_index):
    import torch
    B, C = x.shape[0], x.shape[-1]
    v = x.reshape(B, -1, groups, C // groups)
    var, mean = torch.var_mean(v, dim=(1, 3), unbiased=False, keepdim=True)
    z = ((v - mean) / torch.sqrt(var + 1e-5)).reshape(x.shape) * q["gamma"] + q["beta"]
    if not activation:
        return z
    y = torch.where(z > 0, z, torch.expm1(z.clamp(max=0)))
    if mask is not None and name_index is not None:
        t = mask["threshold"]
        keep = keep_mask(tuple(x.shape), t, mask["seed"], mask["step"], mask["layer"] + name_index, mask["per_channel"], mask["first_item"])
        y = y * torch.from_numpy(keep.astype(np.float64)) * (65536 / (65536 - t))
    return y


def level(params, concat, skip_feat=None, rates=(2, 4), use_skip=True, use_skip2=True, skip2=None, groups=8, mask=None):
    """sfm_amd.disp_bottleneck_dense(..., groups=groups, dropout=mask); mask: dict(threshold, seed, step, layer, per_channel, first_item)"""
    import torch
    from . import ref_graph as R
    place = {"sup": 0, "aspp_up": 1, "aspp_up2": 2, "skip": 3, "skip2": 4}

    def sc(x, name, rate=None, activation=True):
        q = params[name]
        y = R.conv1x1(x, q["w"]) if rate is None else R.dilated_conv3x3(x, q["w"], rate)
        return _torch_norm(y, q, groups, activation, mask, place.get(name))
    h, w = concat.shape[1], concat.shape[2]
    upnet = sc(R.resize_bilinear_tf1(concat, 2 * h, 2 * w), "up", activation=False)
    sup = sc(upnet, "sup")
    a1 = sc(upnet, "aspp_up", rate=rates[0])
    a2 = sc(torch.cat([sup, a1], dim=3), "aspp_up2", rate=rates[1])
    if use_skip:
        skip = sc(_torch_norm(skip_feat, params["skip_bn"], groups, True, None, None), "skip")
    else:
        skip = sc(torch.cat([a1, a2], dim=3), "skip", rate=rates[1] * 2)
    parts = [sup, a1, a2, skip]
    if use_skip2:
        parts.append(sc(R.resize_bilinear_tf1(skip2, 2 * h, 2 * w), "skip2"))
    return sc(torch.cat(parts, dim=3), "out", activation=False), upnet


def decoder(end_points, params, groups=8, mask=None):
    """sfm_amd.disp_aspp_u_dense_decoder(..., groups=groups, dropout=mask)"""
    from . import ref_graph as R

    def lvl(k, name, *a, **kw):
        return level(params[name], *a, groups=groups, mask=None if mask is None else {**mask, "layer": mask["layer"] + 8 * k}, **kw)
    x = _torch_norm(end_points["block4"], params["stem_bn"], groups, True, None, None)
    x = _torch_norm(R.conv1x1(x, params["stem"]["w"]), params["stem"], groups, False, None, None)
    x, _ = lvl(0, "concat", x, end_points["block3"], use_skip2=False)
    x, s1 = lvl(1, "concat1", x, end_points["block2"], use_skip2=False)
    x2, s2 = lvl(2, "concat2", x, end_points["block1"], skip2=s1)
    x3, s3 = lvl(3, "concat3", x2, end_points["root_block"], rates=(3, 6), skip2=s2)
    x4, _ = lvl(4, "concat4", x3, None, rates=(3, 6), use_skip=False, skip2=s3)
    return [R.disp_head(x, params[n]["w"], params[n]["b"]) for x, n in ((x4, "disp4"), (x3, "disp3"), (x2, "disp2"))]
