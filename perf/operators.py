"""The operators that stand around a convolution layer in a residual block, as cases that can be timed and compared.

Three operators, each through the package's public entry points (`own`) or in plain torch:

  norm     group norm with an activation on [B][C][H][W], channels last or planes: forward, or backward
  linear   rows times a weight matrix, with bias, activation and residual: forward, or backward
  dropout  dropout of a counter-based generator, with a residual: forward, or backward

Parameters (weight, bias of the norm, bias of the products) are float32 whatever the type of the activations, weight
matrices are of the activations' type; outputs, workspaces and saved statistics are allocated once, as a program
that runs the same layer again and again does.
"""
import math

import numpy as np
import torch

own = False  # False: the plain form, in 32 bits; True: the framework's operators

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # serving: one feature map of 64 planes of 27 x 27, channels last; latency counts
        {"name": "norm_one_image", "op": "norm", "dir": "fprop", "type": "bf16", "layout": "last", "act": "silu",
         "b": 1, "c": 64, "h": 27, "w": 27, "g": 8},
        # training, forward: what the 5 x 5 layer on 128 x 64 x 27 x 27 leaves, planes in fp32
        {"name": "norm_layer", "op": "norm", "dir": "fprop", "type": "f32", "layout": "planes", "act": "relu",
         "b": 128, "c": 192, "h": 23, "w": 23, "g": 32},
        # training, backward: the same layer in a 16-bit channels-last net; groups of six channels
        {"name": "norm_layer_grad", "op": "norm", "dir": "bprop", "type": "bf16", "layout": "last", "act": "silu",
         "b": 128, "c": 192, "h": 23, "w": 23, "g": 32},
        # large images: a group of a channels-last image is spread over 4 MiB
        {"name": "norm_large", "op": "norm", "dir": "fprop", "type": "bf16", "layout": "last", "act": "gelu",
         "b": 16, "c": 32, "h": 256, "w": 256, "g": 8},
        # their backward pass
        {"name": "norm_large_grad", "op": "norm", "dir": "bprop", "type": "f16", "layout": "last", "act": "silu",
         "b": 16, "c": 32, "h": 256, "w": 256, "g": 8},
        # serving: one row through one layer, as fast as its weights can be read
        {"name": "linear_one_row", "op": "linear", "dir": "fprop", "type": "bf16", "act": "silu", "residual": False,
         "save": False, "m": 1, "k": 2048, "n": 2048},
        # a batch of 128 vectors of odd length into 1000 classes
        {"name": "linear_classes", "op": "linear", "dir": "fprop", "type": "f32", "act": "none", "residual": False,
         "save": False, "m": 128, "k": 1151, "n": 1000},
        # all pixels of 128 images of 23 x 23, 192 planes into 64: a projection with a residual, in fp32
        {"name": "linear_pixels", "op": "linear", "dir": "fprop", "type": "f32", "act": "gelu", "residual": True,
         "save": True, "m": 67712, "k": 192, "n": 64},
        # a wide layer in training, forward
        {"name": "linear_wide", "op": "linear", "dir": "fprop", "type": "bf16", "act": "gelu", "residual": True,
         "save": True, "m": 8192, "k": 2048, "n": 8192},
        # and backward: all three gradients
        {"name": "linear_wide_grad", "op": "linear", "dir": "bprop", "type": "bf16", "act": "gelu", "m": 4096,
         "k": 1024, "n": 4096},
        # one row of features
        {"name": "dropout_row", "op": "dropout", "dir": "fprop", "type": "f16", "residual": True, "rows": 1,
         "cols": 2000, "pitch": 2000, "p": 0.1},
        # the feature maps of the large images, added to the block's input
        {"name": "dropout_large", "op": "dropout", "dir": "fprop", "type": "bf16", "residual": True, "rows": 1048576,
         "cols": 32, "pitch": 32, "p": 0.2},
    ]


# ---- drawn cases ----

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    op = rng.choice(["norm", "norm", "linear", "linear", "dropout"])
    kind = rng.choice(["f32", "f16", "bf16"])
    direction = rng.choice(["fprop", "bprop"])
    act = rng.choice(["none", "relu", "silu", "gelu"])
    if op == "norm":
        g = rng.choice([1, 4, 8, 16, 32])
        side = _log(rng, 1, 256)
        return {"op": op, "dir": direction, "type": kind, "layout": rng.choice(["last", "last", "planes"]), "act": act,
                "b": _log(rng, 1, 128), "c": g * _log(rng, 1, 24), "h": side, "w": max(1, side + rng.choice([0, 0, -1, 3])),
                "g": g}
    if op == "linear":
        # widths of layers are most often multiples of 16, rows any number
        wide = lambda lo, hi: _log(rng, lo, hi) if rng.random() < 0.4 else 16 * _log(rng, max(1, lo // 16), hi // 16)  # noqa: E731
        c = {"op": op, "dir": direction, "type": kind, "act": act, "m": _log(rng, 1, 65536), "k": wide(16, 4096),
             "n": wide(16, 8192)}
        if direction == "fprop":
            c["residual"], c["save"] = rng.random() < 0.5, rng.random() < 0.5
        return c
    cols = _log(rng, 1, 8192)
    return {"op": op, "dir": direction, "type": kind, "residual": direction == "fprop" and rng.random() < 0.5,
            "rows": _log(rng, 1, max(1, 2 ** 25 // cols)), "cols": cols, "pitch": cols + rng.choice([0, 0, 8, 5]),
            "p": rng.choice([0.1, 0.2, 0.5, 0.013])}


def _cost(c):
    """About what a pass of the plain form takes, in seconds."""
    w = work(c)
    return w["bytes"] / 1e12 * (6 if c["op"] == "dropout" else 3 if c["op"] == "norm" else 1) + w["flops"] / 8e13


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    while True:
        c = _draw_one(rng)
        # (two or three values of a group leave a gradient of rounding errors, a few dropped ones no output)
        if c["op"] == "norm" and c["c"] // c["g"] * c["h"] * c["w"] < 16 or c["op"] == "dropout" and c["rows"] * c["cols"] < 64:
            continue
        if _cost(c) <= most[c["op"]]:
            return c


# ---- state ----

def _normal(gen, shape, kind="f32", std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=gen).to(TYPES[kind])


def _empty(shape, kind="f32"):
    return torch.zeros(shape, dtype=TYPES[kind], device="cuda")


def _images(c, make):
    """[B][C][H][W], in the case's layout; make(shape) gives dense memory."""
    b, ch, h, w = c["b"], c["c"], c["h"], c["w"]
    return make((b, h, w, ch)).permute(0, 3, 1, 2) if c["layout"] == "last" else make((b, ch, h, w))


def _rows(c, make):
    """[rows][cols], rows `pitch` elements apart."""
    return make((c["rows"], c["pitch"]))[:, :c["cols"]]


def prepare(case, seed):
    c, t, gen = case, case["type"], torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "norm":
        # feature maps whose channels have means and deviations of their own
        level, spread = _normal(gen, (1, c["c"], 1, 1), std=0.7), 0.5 + _normal(gen, (1, c["c"], 1, 1)).abs()
        noise = _images(c, lambda shape: _normal(gen, shape))
        s["x"] = noise.mul_(spread).add_(level).to(TYPES[t])
        s["weight"], s["bias"] = _normal(gen, (c["c"],), std=0.3, mean=1.0), _normal(gen, (c["c"],), std=0.3)
        if c["dir"] == "fprop":
            s["y"] = torch.zeros_like(s["x"])
            s["mean"], s["rstd"] = _empty((c["b"], c["g"])), _empty((c["b"], c["g"]))
        else:
            s["dy"] = _images(c, lambda shape: _normal(gen, shape, t, 1e-2))
            # what the forward pass kept
            groups = s["x"].reshape(c["b"], c["g"], -1).double()
            s["mean"] = groups.mean(-1).float()
            s["rstd"] = (groups.var(-1, unbiased=False) + EPS).rsqrt().float()
            s["dx"] = torch.zeros_like(s["x"])
            s["dweight"], s["dbias"] = _empty((c["c"],)), _empty((c["c"],))
    elif c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        s["x"], s["weight"] = _normal(gen, (m, k), t), _normal(gen, (n, k), t, 1 / math.sqrt(k))
        s["bias"] = _normal(gen, (n,), std=0.1)
        if c["dir"] == "fprop":
            s["residual"] = _normal(gen, (m, n), t) if c["residual"] else None
            s["y"] = _empty((m, n), t)
            s["z"] = _empty((m, n), t) if c["save"] else None
        else:
            s["dy"] = _normal(gen, (m, n), t, 1e-2)
            s["z"] = _normal(gen, (m, n), t) if c["act"] != "none" else None  # what the forward pass kept
            s["dx"], s["dweight"], s["dbias"] = _empty((m, k), t), _empty((n, k), t), _empty((n,))
    else:
        s["x"] = _rows(c, lambda shape: _normal(gen, shape, t))
        s["residual"] = _rows(c, lambda shape: _normal(gen, shape, t)) if c["residual"] else None
        s["y"] = _rows(c, lambda shape: _empty(shape, t))
        s["seed"], s["offset"] = seed * 0x9E3779B97F4A7C15 % 2 ** 63, seed * 977 + 5
    return s


# ---- one pass ----

def run(state):
    return _own(state) if own else _plain(state)


def _space(F, s):
    """The workspace of a state's calls, allocated before the first of them."""
    c, back = s["case"], int(s["case"]["dir"] == "bprop")
    if c["op"] == "norm":
        size = F.group_norm_workspace(back, s["x"], c["g"])
    else:
        size = F.linear_workspace(back, c["m"], c["k"], c["n"], s["x"].dtype)
    s["space"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return s["space"]


def _own(s):
    import fbcuda_amd as F
    c = s["case"]
    space = None
    if c["op"] != "dropout":
        space = s["space"] if "space" in s else _space(F, s)
    if c["op"] == "norm":
        if c["dir"] == "fprop":
            code = F.group_norm_fprop(s["x"], s["weight"], s["bias"], s["y"], c["g"], space, activation=c["act"], eps=EPS,
                                      mean=s["mean"], rstd=s["rstd"])
            got = s["y"], s["mean"], s["rstd"]
        else:
            code = F.group_norm_bprop(s["x"], s["weight"], s["bias"], s["mean"], s["rstd"], s["dy"], s["dx"],
                                      s["dweight"], s["dbias"], c["g"], space, activation=c["act"])
            got = s["dx"], s["dweight"], s["dbias"]
    elif c["op"] == "linear":
        if c["dir"] == "fprop":
            code = F.linear_fprop(s["x"], s["weight"], s["bias"], s["y"], space, activation=c["act"],
                                  residual=s["residual"], preactivation=s["z"])
            got = (s["y"], s["z"]) if c["save"] else s["y"]
        else:
            code = F.linear_bprop(s["x"], s["weight"], s["dy"], s["z"], s["dx"], s["dweight"], s["dbias"], space,
                                  activation=c["act"])
            got = s["dx"], s["dweight"], s["dbias"]
    elif c["dir"] == "fprop":
        code = F.dropout_fprop(s["x"], s["y"], c["p"], s["seed"], s["offset"], residual=s["residual"])
        got = s["y"]
    else:
        code = F.dropout_bprop(s["x"], s["y"], c["p"], s["seed"], s["offset"])
        got = s["y"]
    if code != F.Success:
        raise RuntimeError(F.error_string(code))
    return got


def _activate(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, act):
    """The activation's derivative."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        u = 1 / (1 + torch.exp(-z))
        return u * (1 + z * (1 - u))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _halves(blocks, seed, offset, device):
    """[blocks][8] 16-bit numbers: Philox4x32-10 of the counter (block, offset), lower halves first."""
    low = 0xFFFFFFFF
    i = torch.arange(blocks, dtype=torch.int64, device=device)
    a, b = i & low, i >> 32
    c, d = torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        # products of two 32-bit numbers, modulo 2^64: the bits of the unsigned product
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = (q >> 32 & low) ^ b ^ k0, q & low, (p >> 32 & low) ^ d ^ k1, p & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack((a, b, c, d), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(blocks, 8)


def _plain(s):
    c, t = s["case"], TYPES[s["case"]["type"]]
    if c["op"] == "norm":
        b, ch, g = c["b"], c["c"], c["g"]
        x = s["x"].float()
        groups = x.reshape(b, g, -1)
        weight, bias = s["weight"].view(1, ch, 1, 1), s["bias"].view(1, ch, 1, 1)
        each = lambda v: v.repeat_interleave(ch // g, 1).view(b, ch, 1, 1)  # noqa: E731
        if c["dir"] == "fprop":
            mean = groups.mean(-1)
            rstd = torch.rsqrt((groups - mean[..., None]).square().mean(-1) + EPS)
            z = (x - each(mean)) * (each(rstd) * weight) + bias
            return _activate(z, c["act"]).to(t), mean, rstd
        xh = (x - each(s["mean"])) * each(s["rstd"])
        dz = s["dy"].float() * _slope(xh * weight + bias, c["act"])
        dweight, dbias = (dz * xh).sum((0, 2, 3)), dz.sum((0, 2, 3))
        dh = dz * weight
        s1, s2 = (v.reshape(b, g, -1).mean(-1) for v in (dh, dh * xh))
        dx = each(s["rstd"]) * (dh - each(s1) - xh * each(s2))
        return dx.to(t), dweight, dbias
    if c["op"] == "linear":
        x, w = s["x"].float(), s["weight"].float()
        if c["dir"] == "fprop":
            z = x @ w.t() + s["bias"]
            y = _activate(z, c["act"])
            if c["residual"]:
                y = y + s["residual"].float()
            return (y.to(t), z.to(t)) if c["save"] else y.to(t)
        dz = s["dy"].float()
        if c["act"] != "none":
            dz = dz * _slope(s["z"].float(), c["act"])
        return (dz @ w).to(t), (dz.t() @ x).to(t), dz.sum(0)
    x = s["x"].float()
    threshold = int(round(c["p"] * 65536))
    n = c["rows"] * c["cols"]
    u = _halves(-(-n // 8), s["seed"], s["offset"], x.device).reshape(-1)[:n].view(c["rows"], c["cols"])
    y = torch.where(u >= threshold, x * (65536 / (65536 - threshold)), torch.zeros_like(x))
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(t)


# ---- what a pass cannot do without ----

def work(case):
    c, size = case, 4 if case["type"] == "f32" else 2
    back = c["dir"] == "bprop"
    if c["op"] == "norm":
        n = c["b"] * c["c"] * c["h"] * c["w"]
        params = 4 * (2 * c["c"] * (2 if back else 1) + 2 * c["b"] * c["g"])
        return {"bytes": n * size * (3 if back else 2) + params, "flops": n * (12 if back else 8)}
    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        if back:
            outer = m * n * (2 if c["act"] != "none" else 1)
            return {"bytes": size * (2 * (m * k + n * k) + outer) + 4 * n, "flops": 4.0 * m * n * k + 4 * m * n}
        outer = m * n * (1 + int(c["residual"]) + int(c["save"]))
        return {"bytes": size * (m * k + n * k + outer) + 4 * n, "flops": 2.0 * m * n * k + 4 * m * n}
    n = c["rows"] * c["cols"]
    return {"bytes": n * size * (3 if c["residual"] else 2), "flops": 2 * n}


# ---- the same from the definitions, in 64 bits ----

def _philox_numpy(index, seed, offset):
    """The 16-bit number of each element index."""
    mask, word = np.uint64(0xFFFFFFFF), np.uint64(32)
    blocks = np.arange((int(index) + 7) // 8, dtype=np.uint64)
    ctr = [blocks & mask, blocks >> word, np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for r in range(10):
        first, second = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(second >> word) ^ ctr[1] ^ np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), second & mask,
               (first >> word) ^ ctr[3] ^ np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32), first & mask]
    out = np.empty((len(blocks), 8), np.int32)
    for j in range(4):
        out[:, 2 * j], out[:, 2 * j + 1] = ctr[j] & np.uint64(0xFFFF), ctr[j] >> np.uint64(16)
    return out.reshape(-1)[:index]


def _sigmoid64(v):
    return torch.reciprocal(torch.exp(-v) + 1.0)


def _normal_cdf(v):
    return 0.5 * torch.special.erfc(-v / 2.0 ** 0.5)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "norm":
        x, w, bias = s["x"].double(), s["weight"].double()[None, :, None, None], s["bias"].double()[None, :, None, None]
        d = c["c"] // c["g"]
        if c["dir"] == "fprop":
            count = d * c["h"] * c["w"]
            total = x.sum((2, 3)).view(c["b"], c["g"], d).sum(2)
            mean = total / count
            centred = x - mean[:, torch.arange(c["c"], device=x.device) // d, None, None]
            variance = (centred * centred).sum((2, 3)).view(c["b"], c["g"], d).sum(2) / count
            scale = 1.0 / torch.sqrt(variance + EPS)
            z = centred * scale[:, torch.arange(c["c"], device=x.device) // d, None, None] * w + bias
            y = {"none": lambda: z, "relu": lambda: torch.maximum(z, torch.zeros_like(z)),
                 "silu": lambda: z * _sigmoid64(z), "gelu": lambda: z * _normal_cdf(z)}[c["act"]]()
            return y, mean, scale
        owner = torch.arange(c["c"], device=x.device) // d
        scale = s["rstd"].double()[:, owner, None, None]
        normal = (x - s["mean"].double()[:, owner, None, None]) * scale
        up = s["dy"].double() * _derivative64(normal * w + bias, c["act"])
        inner = up * w
        over = d * c["h"] * c["w"]
        first = inner.sum((2, 3)).view(c["b"], c["g"], d).sum(2)[:, owner, None, None] / over
        second = (inner * normal).sum((2, 3)).view(c["b"], c["g"], d).sum(2)[:, owner, None, None] / over
        return scale * (inner - first - normal * second), (up * normal).sum((0, 2, 3)), up.sum((0, 2, 3))
    if c["op"] == "linear":
        x, w = s["x"].double(), s["weight"].double()
        if c["dir"] == "fprop":
            z = torch.addmm(s["bias"].double().expand(c["m"], -1), x, w.t())
            y = {"none": lambda: z, "relu": lambda: torch.maximum(z, torch.zeros_like(z)),
                 "silu": lambda: z * _sigmoid64(z), "gelu": lambda: z * _normal_cdf(z)}[c["act"]]()
            y = y if s["residual"] is None else y + s["residual"].double()
            return (y, z) if c["save"] else y
        up = s["dy"].double()
        up = up if s["z"] is None else up * _derivative64(s["z"].double(), c["act"])
        return torch.mm(up, w), torch.mm(up.t(), x), up.sum(0)
    cut = int(math.floor(c["p"] * 65536 + 0.5))
    u = _philox_numpy(c["rows"] * c["cols"], s["seed"], s["offset"])
    keep = torch.from_numpy(u >= cut).to(s["x"].device).view(c["rows"], c["cols"])
    y = s["x"].double().masked_fill(~keep, 0.0) / (1.0 - cut / 65536)
    return y if s["residual"] is None else y + s["residual"].double()


def _derivative64(v, act):
    if act == "relu":
        return torch.heaviside(v, torch.zeros((), dtype=v.dtype, device=v.device))
    if act == "silu":
        return _sigmoid64(v) + v * _sigmoid64(v) * _sigmoid64(-v)
    if act == "gelu":
        return _normal_cdf(v) + v * torch.exp(-v * v / 2.0) / (2.0 * math.pi) ** 0.5
    return torch.ones_like(v)
