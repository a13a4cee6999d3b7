"""Measured cases of the feature-map operators: group normalisation with an activation
(channels last, optionally followed by dropout) and counter-based dropout.

Each case is one call a feature encoder in front of the correlation makes: inference
(``kind`` "norm" / "dropout") or a training step's forward and backward ("norm_train" /
"dropout_train"). ``run`` computes the operator from elementary torch operations, or, when
``own`` is set, through the public functions of ``localcorr_b200``.

Dropout draws come from Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers:
as easy as 1, 2, 3", 2011): draw e is the 16-bit piece e % 8 (low half of a word first) of the
block with counter (e // 8, offset) and key seed; it drops when it is below
round(65536 p), and what stays is multiplied by 65536 / (65536 - round(65536 p)).
"""

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one pooled token of a streaming (frame by frame) model: latency only
        dict(name="norm_token", kind="norm", dtype="f16", b=1, h=1, w=1, c=256, groups=32,
             act="silu", p=0.0, mode="element"),
        # the small RAFT inference case: one 46 x 62 float32 map of 256 channels
        dict(name="norm_small_f32", kind="norm", dtype="f32", b=1, h=46, w=62, c=256, groups=32,
             act="relu", p=0.0, mode="element"),
        # inference on a batch of 1/8-resolution 1080p maps (the training configuration's maps)
        dict(name="norm_eighth_f16", kind="norm", dtype="f16", b=8, h=135, w=240, c=256,
             groups=32, act="relu", p=0.0, mode="element"),
        # the encoder's first stage at 1/2 resolution: long rows of one group, the largest map
        dict(name="norm_half_f16", kind="norm", dtype="f16", b=8, h=540, w=960, c=64, groups=8,
             act="relu", p=0.0, mode="element"),
        # training step at odd sizes: ragged crops, channels that are no power of two
        dict(name="norm_train_odd_f32", kind="norm_train", dtype="f32", b=3, h=47, w=61, c=96,
             groups=8, act="silu", p=0.0, mode="element"),
        # training step of the 1080p configuration's maps
        dict(name="norm_train_eighth_f16", kind="norm_train", dtype="f16", b=8, h=135, w=240,
             c=256, groups=32, act="relu", p=0.0, mode="element"),
        # instance normalisation (one channel a group) of the high-batch configuration's maps
        dict(name="norm_train_instance_bf16", kind="norm_train", dtype="bf16", b=64, h=64, w=128,
             c=128, groups=128, act="leaky_relu", p=0.0, mode="element"),
        # norm, activation and whole-channel dropout in one call, as an encoder trains them
        dict(name="norm_drop_train_f16", kind="norm_train", dtype="f16", b=8, h=135, w=240,
             c=128, groups=16, act="relu", p=0.1, mode="channel"),
        # dropout of one token's features
        dict(name="dropout_token", kind="dropout", dtype="f16", b=1, h=1, w=1, c=256, p=0.1,
             mode="element", residual=False),
        # elementwise dropout of a projected branch added to its residual, odd sizes
        dict(name="dropout_odd_f32", kind="dropout", dtype="f32", b=3, h=47, w=61, c=99, p=0.5,
             mode="element", residual=True),
        # training step of dropout plus residual on the 1080p configuration's maps
        dict(name="dropout_train_eighth_bf16", kind="dropout_train", dtype="bf16", b=8, h=135,
             w=240, c=256, p=0.1, mode="element", residual=True),
        # whole-channel dropout of an encoder's output, high batch, training
        dict(name="dropout_train_channel_f16", kind="dropout_train", dtype="f16", b=64, h=64,
             w=128, c=128, p=0.2, mode="channel", residual=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "norm_train", "dropout", "dropout_train"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    b, h, w = _log_int(rng, 1, 64), _log_int(rng, 1, 540), _log_int(rng, 1, 960)
    most = 60_000_000
    case = dict(kind=kind, dtype=dtype, b=b, h=h, w=w)
    if kind.startswith("norm"):
        groups = rng.choice([1, 2, 3, 4, 8, 16, 32])
        per = _log_int(rng, 8, 64)
        if rng.random() < 0.2:  # instance normalisation of whole maps
            groups, per = 8 * rng.randint(2, 32), 1
            case["h"], case["w"] = max(h, 9), max(w, 11)
        case.update(c=groups * per, groups=groups,
                    act=rng.choice(["none", "relu", "silu", "leaky_relu"]),
                    p=rng.choice([0.0, 0.0, 0.1, 0.3]), mode=rng.choice(["element", "channel"]))
    else:
        case.update(c=_log_int(rng, 3, 1024), p=rng.choice([0.05, 0.1, 0.2, 0.5]),
                    mode=rng.choice(["element", "channel"]), residual=rng.random() < 0.5)
    while case["b"] > 1 and case["b"] * case["h"] * case["w"] * case["c"] > most:
        case["b"] = (case["b"] + 1) // 2
    while case["h"] * case["w"] * case["c"] > most:
        case["h"] = (case["h"] + 1) // 2
    return case


def _slope(act):
    return 0.1 if act == "leaky_relu" else 0.0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    shape = (case["b"], case["h"], case["w"], case["c"])
    train = case["kind"].endswith("_train")

    def rand(*s):
        return torch.randn(*s, generator=gen, device=dev)

    # a convolution's output: every channel with its own level and spread
    x = rand(*shape).mul_(rand(case["c"]).mul(0.5).exp()).add_(rand(case["c"])).to(dt)
    s = dict(case=case, x=x.requires_grad_(train))
    if case["kind"].startswith("norm"):
        s["weight"] = rand(case["c"]).mul(0.2).add(1.0).requires_grad_(train)
        s["bias"] = rand(case["c"]).mul(0.2).requires_grad_(train)
    elif case["residual"]:
        s["residual"] = rand(*shape).to(dt).requires_grad_(train)
    if train:
        s["grad"] = rand(*shape).to(dt)
    # seed and call number of the draws, on the device as a captured training step keeps them
    s["rng"] = torch.tensor([(seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 62), seed % 1000],
                            dtype=torch.int64, device=dev)
    return s


# ---------------------------------------------------------------------------
# plain form
# ---------------------------------------------------------------------------

_LOW = 0xFFFFFFFF


def _mul_hi_lo(m, c):
    """High and low 32 bits of m * c, both below 2**32, in int64 arithmetic."""
    low, high = m * (c & 0xFFFF), m * (c >> 16)
    return (high + (low >> 16)) >> 16, ((high << 16) + low) & _LOW


def _draws(count, rng):
    """The first ``count`` 16-bit draws of the stream (seed, offset)."""
    block = torch.arange((count + 7) // 8, dtype=torch.int64, device=rng.device)
    c0, c1 = block & _LOW, block >> 32
    c2, c3 = rng[1] & _LOW, (rng[1] >> 32) & _LOW
    k0, k1 = rng[0] & _LOW, (rng[0] >> 32) & _LOW
    for _ in range(10):
        h0, l0 = _mul_hi_lo(0xD2511F53, c0)
        h1, l1 = _mul_hi_lo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), dim=-1)
    return torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(-1)[:count]


def _threshold(p):
    return int(p * 65536.0 + 0.5)


def _kept(case, rng):
    """(which elements stay, as a mask that broadcasts over [B, S, C]; their factor)."""
    b, rows, c = case["b"], case["h"] * case["w"], case["c"]
    t = _threshold(case["p"])
    shape = (b, 1, c) if case["mode"] == "channel" else (b, rows, c)
    return (_draws(shape[0] * shape[1] * shape[2], rng) >= t).view(shape), 65536.0 / (65536 - t)


def _plain_norm(s):
    case = s["case"]
    b, rows, c, g = case["b"], case["h"] * case["w"], case["c"], case["groups"]
    per, n = c // g, rows * (c // g)
    eps, act, slope = 1e-5, case["act"], _slope(case["act"])
    x = s["x"].detach()
    dt = x.dtype
    x = x.view(b, rows, g, per).float()
    weight, bias = s["weight"].detach().view(g, per), s["bias"].detach().view(g, per)
    # statistics: long sums in 64 bits
    mean = x.sum((1, 3), keepdim=True, dtype=torch.float64) / n
    low = mean.float()
    d = x - low
    var = (d * d).sum((1, 3), keepdim=True, dtype=torch.float64) / n - (mean - low) ** 2
    rstd = (var + eps).rsqrt()
    xhat = (d - (mean - low).float()) * rstd.float()
    z = xhat * weight + bias
    if act == "silu":
        sig = 1.0 / (1.0 + (-z).exp())
        y = z * sig
    elif act == "none":
        y = z
    else:
        y = torch.where(z > 0, z, slope * z)
    drop = case["p"] > 0
    if drop:
        kept, factor = _kept(case, s["rng"])
        kept = kept.view(b, -1, g, per)
        y = torch.where(kept, y * factor, 0.0)
    y = y.to(dt).view(s["x"].shape)
    if case["kind"] == "norm":
        return y
    dz = s["grad"].view(b, rows, g, per).float()
    if drop:
        dz = torch.where(kept, dz * factor, 0.0)
    if act == "silu":
        dz = dz * (sig * (1.0 + z * (1.0 - sig)))
    elif act != "none":
        # which side of the corner: in 64 bits, the gradient jumps there
        z64 = (x.double() - mean) * rstd * weight.double() + bias.double()
        dz = torch.where(z64 > 0, dz, slope * dz)
    dxhat = dz * weight
    m1 = (dxhat.sum((1, 3), keepdim=True, dtype=torch.float64) / n).float()
    m2 = ((dxhat * xhat).sum((1, 3), keepdim=True, dtype=torch.float64) / n).float()
    dx = (rstd.float() * (dxhat - m1 - xhat * m2)).to(dt).view(s["x"].shape)
    dw = (dz * xhat).sum((0, 1), dtype=torch.float64).float().view(c)
    db = dz.sum((0, 1), dtype=torch.float64).float().view(c)
    return y, dx, dw, db


def _plain_dropout(s):
    case = s["case"]
    x = s["x"].detach()
    flat = (case["b"], case["h"] * case["w"], case["c"])
    kept, factor = _kept(case, s["rng"])
    y = torch.where(kept, x.view(flat).float() * factor, 0.0)
    if case["residual"]:
        y = s["residual"].detach().view(flat).float() + y
    y = y.to(x.dtype).view(x.shape)
    if case["kind"] == "dropout":
        return y
    grad = s["grad"]
    dx = torch.where(kept, grad.view(flat).float() * factor, 0.0).to(x.dtype).view(x.shape)
    return (y, dx, grad.clone()) if case["residual"] else (y, dx)


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------

def _own_norm(s):
    import localcorr_b200 as lc

    case = s["case"]
    drop = dict(p=case["p"], rng=s["rng"], dropout_mode=case["mode"]) if case["p"] > 0 else {}
    y = lc.group_norm(s["x"], case["groups"], s["weight"], s["bias"], eps=1e-5,
                      activation=case["act"], negative_slope=0.1, **drop)
    if case["kind"] == "norm":
        return y
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
    return y, dx, dw, db


def _own_dropout(s):
    import localcorr_b200 as lc

    case = s["case"]
    y = lc.dropout(s["x"], case["p"], s["rng"], residual=s.get("residual"), mode=case["mode"])
    if case["kind"] == "dropout":
        return y
    leaves = (s["x"], s["residual"]) if case["residual"] else (s["x"],)
    return (y, *torch.autograd.grad(y, leaves, s["grad"]))


def run(state):
    if state["case"]["kind"].startswith("norm"):
        return _own_norm(state) if own else _plain_norm(state)
    return _own_dropout(state) if own else _plain_dropout(state)


def work(case):
    """Each input read once and each output written once; a few operations per element."""
    n = case["b"] * case["h"] * case["w"] * case["c"]
    size = 4 if case["dtype"] == "f32" else 2
    train = case["kind"].endswith("_train")
    if case["kind"].startswith("norm"):
        return {"bytes": n * size * (4 if train else 2) + 4 * case["c"] * (4 if train else 2),
                "flops": n * (20 if train else 8)}
    maps = (4 if train else 2) + int(case["residual"])
    return {"bytes": n * size * maps, "flops": n * (4 if train else 2)}


# ---------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------

def _exact_factors(case, rng):
    """The factor of every element, [B, H, W, C] or [B, 1, 1, C], in 64 bits."""
    seed, offset = (int(v) for v in rng.tolist())
    t = round(case["p"] * 65536)
    shape = (case["b"], case["h"], case["w"], case["c"])
    if case["mode"] == "channel":
        shape = (case["b"], 1, 1, case["c"])
    count = shape[0] * shape[1] * shape[2] * shape[3]
    n = -(-count // 8)
    ctr = [torch.arange(n, device=rng.device)]
    ctr += [torch.full_like(ctr[0], v) for v in (0, offset % 2 ** 32, offset >> 32)]
    for i in range(10):
        # int64 products wrap modulo 2**64, which keeps all 64 bits of the product
        a, b = ctr[0] * 0xD2511F53, ctr[2] * 0xCD9E8D57
        key = ((seed + i * 0x9E3779B9) % 2 ** 32, ((seed >> 32) + i * 0xBB67AE85) % 2 ** 32)
        ctr = [((b >> 32) & _LOW) ^ ctr[1] ^ key[0], b & _LOW,
               ((a >> 32) & _LOW) ^ ctr[3] ^ key[1], a & _LOW]
    pieces = torch.empty(n, 8, dtype=torch.int64, device=rng.device)
    for i in range(4):
        pieces[:, 2 * i], pieces[:, 2 * i + 1] = ctr[i] % 65536, ctr[i] // 65536
    kept = pieces.view(-1)[:count].view(shape) >= t
    return kept.double() * (65536 / (65536 - t))


def exact(case, seed):
    s = prepare(case, seed)
    train = case["kind"].endswith("_train")
    factors = _exact_factors(case, s["rng"]) if case["p"] > 0 else None
    x = s["x"].detach().double().requires_grad_(train)
    if case["kind"].startswith("norm"):
        w = s["weight"].detach().double().requires_grad_(train)
        b = s["bias"].detach().double().requires_grad_(train)
        nb, g, c = case["b"], case["groups"], case["c"]
        by_group = x.reshape(nb, -1, g, c // g).permute(0, 2, 1, 3).reshape(nb, g, -1)
        var, mean = torch.var_mean(by_group, dim=2, correction=0, keepdim=True)
        z = ((by_group - mean) / torch.sqrt(var + 1e-5)).reshape(nb, g, -1, c // g)
        z = z.permute(0, 2, 1, 3).reshape(x.shape) * w + b
        y = {"none": lambda v: v, "silu": lambda v: v * torch.sigmoid(v),
             "relu": lambda v: v.clamp_min(0.0),
             "leaky_relu": lambda v: v.clamp_min(0.0) + 0.1 * v.clamp_max(0.0)}[case["act"]](z)
        leaves = (x, w, b)
    else:
        y = x
        leaves = (x,)
    if factors is not None:
        y = y * factors
    residual = case.get("residual", False)
    if residual:
        r = s["residual"].detach().double().requires_grad_(train)
        y, leaves = y + r, leaves + (r,)
    if not train:
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, leaves, s["grad"].double()))
