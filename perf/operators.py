"""Group norm with an activation, dropout, and the two fused, at the activation shapes of the depth decoder: the cases that are
measured, their inputs, and each operator in its plain form.

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the calls a user makes of sfm_amd.
A training pass returns the output and every gradient, a serving pass the output."""
import torch

own = False

EPSILON = 1e-5
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _case(name, op, shape, dtype, groups=0, act="none", train=True, p=0.0, per_channel=False):
    b, h, w, c = shape
    return {"name": name, "op": op, "b": b, "h": h, "w": w, "c": c, "dtype": dtype, "groups": groups, "act": act, "train": train,
            "p": p, "per_channel": per_channel}


def listed():
    return [
        # batch norm's place in front of the decoder's stem, one 128 x 416 image served alone: launch latency
        _case("norm stem serve b1", "norm", (1, 4, 13, 2048), "fp32", 32, "elu", train=False),
        # the narrowest level of a 128 x 416 training step at batch 8
        _case("norm concat train b8", "norm", (8, 8, 26, 512), "fp32", 32, "elu"),
        # its full-resolution level: four channels per group
        _case("norm concat4 train b8", "norm", (8, 128, 416, 32), "fp32", 8, "elu"),
        # a cropped image, channels that no 16-byte load divides, half precision
        _case("norm odd train", "norm", (3, 37, 53, 90), "fp16", 6, "silu"),
        # groups wider than a workgroup's slab of channels, odd rows
        _case("norm wide groups train", "norm", (2, 31, 17, 1000), "fp32", 2, "none"),
        # full-resolution activations of eight 1024 x 2048 images, served in bf16
        _case("norm 1024x2048 serve", "norm", (8, 1024, 2048, 32), "bf16", 8, "elu", train=False),
        # the same activations trained at batch 4
        _case("norm 1024x2048 train", "norm", (4, 1024, 2048, 32), "bf16", 8, "silu"),
        # the regularised level before the last, 128 x 416, mixed precision
        _case("norm+drop concat3 train", "norm", (8, 64, 208, 64), "bf16", 16, "elu", p=0.1),
        # half-resolution level of sixteen 384 x 1248 images, whole channels dropped
        _case("norm+drop 192x624 train", "norm", (16, 192, 624, 64), "fp32", 16, "elu", p=0.2, per_channel=True),
        # dropout alone behind a batch norm: the narrowest level, and the full-resolution one in bf16
        _case("drop concat train b8", "drop", (8, 8, 26, 512), "fp32", p=0.1),
        _case("drop concat4 train b8", "drop", (8, 128, 416, 32), "bf16", p=0.25),
        # half-resolution activations of eight 1024 x 2048 images
        _case("drop 512x1024 train", "drop", (8, 512, 1024, 64), "fp32", p=0.5),
    ]


def draw(rng):
    """Any of the above: one to sixteen images, any height and width, 8 to 1024 channels (odd counts among them), up to 2^26 values."""
    while True:
        b = rng.randint(1, 16)
        h, w = (int(round(2 ** rng.uniform(1, 10))) for _ in range(2))
        c = rng.choice([8 * rng.randint(1, 16), 32 * rng.randint(1, 32), rng.randint(8, 200)])
        if 1 << 12 <= b * h * w * c <= 1 << 26:
            break
    op = rng.choice(["norm", "norm", "norm", "drop"])
    train = op == "drop" or rng.random() < 0.75
    p = rng.choice([0.05, 0.1, 0.25, 0.5]) if op == "drop" or (train and rng.random() < 0.5) else 0.0
    # a group holds at least 32 values (fewer, and its gradient is all rounding), and relu is served only (its step is no place to compare gradients)
    groups = rng.choice([g for g in range(1, min(c, 64) + 1) if c % g == 0 and h * w * (c // g) >= 32]) if op == "norm" else 0
    act = rng.choice(["elu", "silu", "none"] if train else ["elu", "silu", "relu", "none"]) if op == "norm" else "none"
    case = _case("", op, (b, h, w, c), rng.choice(["fp32", "bf16", "fp16"]), groups, act, train, p, p > 0 and rng.random() < 0.3)
    del case["name"]
    return case


def work(case):
    n = case["b"] * case["h"] * case["w"] * case["c"]
    tensors = 4 if case["train"] else 2  # x -> y; a training pass also gy -> gx
    params = 4 * case["c"] * (4 if case["train"] else 2) if case["op"] == "norm" else 0
    per = (10 if case["op"] == "norm" else 1) * (3 if case["train"] and case["op"] == "norm" else 2 if case["train"] else 1)
    return {"bytes": n * tensors * BYTES[case["dtype"]] + params, "flops": n * per}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (case["b"], case["h"], case["w"], case["c"])
    c, dt = case["c"], TYPES[case["dtype"]]

    def noise(*s):
        return torch.randn(*s, generator=g, device="cuda")

    # a convolution's output: channels with means and scales of their own
    x = (noise(*shape) * (0.5 + noise(c).abs()) + noise(c)).to(dt)
    state = {"case": case, "x": x.requires_grad_(case["train"])}
    if case["train"]:
        state["gy"] = noise(*shape).to(dt)
    if case["op"] == "norm":
        state["gamma"] = (1.0 + 0.1 * noise(c)).requires_grad_(case["train"])
        state["beta"] = (0.1 * noise(c)).requires_grad_(case["train"])
    if case["p"]:
        # the seed of the run and the training step, on the device, as a program that replays a captured step keeps them
        state["seed"], state["step"], state["layer"] = 1000003 * seed + 12345678901, seed % 1000, 3
        state["rng"] = torch.tensor([state["seed"], state["step"]], dtype=torch.int64, device="cuda")
    return state


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- the framework's calls
def _run_own(s):
    import sfm_amd
    case = s["case"]
    drop = sfm_amd.DropoutMask(case["p"], s["rng"], layer=s["layer"], per_channel=case["per_channel"]) if case["p"] else None
    if case["op"] == "drop":
        y = sfm_amd.dropout(s["x"], drop)
        (gx,) = torch.autograd.grad(y, (s["x"],), s["gy"])
        return {"y": y.detach(), "gx": gx}
    y = sfm_amd.group_norm_act(s["x"], s["gamma"], s["beta"], case["groups"], epsilon=EPSILON, activation=case["act"], dropout=drop)
    if not case["train"]:
        return {"y": y}
    gx, ggamma, gbeta = torch.autograd.grad(y, (s["x"], s["gamma"], s["beta"]), s["gy"])
    return {"y": y.detach(), "gx": gx, "ggamma": ggamma, "gbeta": gbeta}


# ---- the plain forms
MASK32 = 0xFFFFFFFF


def _words(block, item, step, layer, seed):
    """Philox 4x32, seven rounds (Salmon et al. 2011), on int64 tensors that hold 32-bit words: the four words of each block."""
    c0, c1, c2, c3 = block, item, step & MASK32, layer
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products; a product that wraps keeps its bits
        c0, c1, c2, c3 = ((b >> 32) & MASK32) ^ c1 ^ k0, b & MASK32, ((a >> 32) & MASK32) ^ c3 ^ k1, a & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return c0, c1, c2, c3


def _keep(s):
    """The mask as truth values, [B, rows, C] (per channel: [B, 1, C]), and the factor of what is kept."""
    case = s["case"]
    n = case["c"] if case["per_channel"] else case["h"] * case["w"] * case["c"]
    threshold = int(round(case["p"] * 65536))
    block = torch.arange((n + 7) // 8, device="cuda")[None, :]
    item = torch.arange(case["b"], device="cuda")[:, None]
    block, item = block.expand(case["b"], -1), item.expand(-1, block.shape[1])
    step, layer = torch.full_like(block, s["step"]), s["layer"]
    words = _words(block, item, step, layer, s["seed"])
    bits = torch.stack([half for w in words for half in ((w & 0xFFFF) >= threshold, (w >> 16) >= threshold)], dim=2)
    keep = bits.reshape(case["b"], -1)[:, :n].reshape(case["b"], -1, case["c"])
    return keep, 65536.0 / (65536 - threshold)


def _run_plain(s):
    case = s["case"]
    dt, b, c, groups = s["x"].dtype, case["b"], case["c"], case["groups"]
    shape = (b, case["h"] * case["w"], c)
    x = s["x"].detach().float().reshape(shape)
    keep, scale = _keep(s) if case["p"] else (None, 1.0)
    if case["op"] == "drop":
        y = torch.where(keep, x * scale, 0.0)
        gx = torch.where(keep, s["gy"].float().reshape(shape) * scale, 0.0)
        return {"y": y.reshape(s["x"].shape).to(dt), "gx": gx.reshape(s["x"].shape).to(dt)}
    grouped = (b, shape[1], groups, c // groups)
    gamma, beta = s["gamma"].detach().reshape(grouped[2:]), s["beta"].detach().reshape(grouped[2:])
    x = x.reshape(grouped)
    d = x - x.mean(dim=(1, 3), keepdim=True)
    r = torch.rsqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPSILON)
    xhat = d * r
    z = xhat * gamma + beta
    act = case["act"]
    if act == "elu":
        y = torch.where(z > 0, z, torch.expm1(z))
    elif act == "relu":
        y = torch.where(z > 0, z, 0.0)
    elif act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        y = z * sig
    else:
        y = z
    if keep is not None:
        keep = keep.reshape(b, -1, groups, c // groups)
        y = torch.where(keep, y * scale, 0.0)
    y = y.reshape(s["x"].shape).to(dt)
    if not case["train"]:
        return {"y": y}
    dz = s["gy"].float().reshape(grouped)
    if keep is not None:
        dz = torch.where(keep, dz * scale, 0.0)
    if act == "elu":
        dz = dz * torch.where(z > 0, 1.0, torch.exp(z))
    elif act == "relu":
        dz = torch.where(z > 0, dz, 0.0)
    elif act == "silu":
        dz = dz * (sig * (1.0 + z * (1.0 - sig)))
    ggamma, gbeta = (dz * xhat).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    dg = dz * gamma
    gx = r * (dg - dg.mean(dim=(1, 3), keepdim=True) - xhat * (dg * xhat).mean(dim=(1, 3), keepdim=True))
    return {"y": y, "gx": gx.reshape(s["x"].shape).to(dt), "ggamma": ggamma.reshape(c), "gbeta": gbeta.reshape(c)}


# ---- 64 bits, from the definitions
def _high(a, m):
    """The upper word of the product of 32-bit words, from 16-bit halves."""
    a1, a0, m1, m0 = a >> 16, a & 0xFFFF, m >> 16, m & 0xFFFF
    mid = a1 * m0 + ((a0 * m0) >> 16)
    return a1 * m1 + (mid >> 16) + (((mid & 0xFFFF) + a0 * m1) >> 16)


def _low(a, m):
    return ((((a >> 16) * (m & 0xFFFF) + (a & 0xFFFF) * (m >> 16)) & 0xFFFF) << 16) + (a & 0xFFFF) * (m & 0xFFFF) & MASK32


def _uniforms(item, n, s):
    """u16 of the n places of one item."""
    place = torch.arange(n, device="cuda")
    count = (n + 7) // 8
    ctr = [torch.arange(count, device="cuda"), torch.full((count,), item, device="cuda"),
           torch.full((count,), s["step"], device="cuda"), torch.full((count,), s["layer"], device="cuda")]
    for k in range(7):
        key = [(s["seed"] + k * 0x9E3779B9) % 2 ** 32, (s["seed"] // 2 ** 32 + k * 0xBB67AE85) % 2 ** 32]
        ctr = [_high(ctr[2], 0xCD9E8D57) ^ ctr[1] ^ key[0], _low(ctr[2], 0xCD9E8D57),
               _high(ctr[0], 0xD2511F53) ^ ctr[3] ^ key[1], _low(ctr[0], 0xD2511F53)]
    word = torch.stack(ctr)[(place % 8) // 2, place // 8]
    return (word >> (16 * (place % 2))) % 65536


def _factor(s):
    """The mask times its factor in 64 bits, broadcast against [B, H, W, C]."""
    case = s["case"]
    t = int(round(case["p"] * 65536))
    inner = (1, 1, case["c"]) if case["per_channel"] else (case["h"], case["w"], case["c"])
    n = inner[0] * inner[1] * inner[2]
    rows = [(_uniforms(b, n, s) >= t).reshape(inner) for b in range(case["b"])]
    return torch.stack(rows).double() * 65536.0 / (65536 - t)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double().requires_grad_(case["train"])
    leaves = [x]
    if case["op"] == "drop":
        y = x * _factor(s)
    else:
        gamma, beta = (s[k].detach().double().requires_grad_(case["train"]) for k in ("gamma", "beta"))
        leaves += [gamma, beta]
        b, h, w, c = x.shape
        v = x.view(b, h * w, case["groups"], -1).permute(0, 2, 1, 3).reshape(b, case["groups"], -1)
        var, mean = torch.var_mean(v, dim=2, unbiased=False, keepdim=True)
        v = ((v - mean) / torch.sqrt(var + EPSILON)).reshape(b, case["groups"], h * w, -1).permute(0, 2, 1, 3).reshape(b, h, w, c)
        z = v * gamma + beta
        y = {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z),
             "elu": lambda: z.clamp(min=0) + torch.expm1(z.clamp(max=0))}[case["act"]]()
        if case["p"]:
            y = y * _factor(s)
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, leaves, s["gy"].double())
    return {"y": y.detach(), **dict(zip(("gx", "ggamma", "gbeta"), grads))}
