"""Measured cases of the training operators around a transformer block's residual joins.

  layer_norm              y = (x - mean) * rstd * weight + bias over the last dimension, and its gradients
  dropout                 y = keep ? x / (1 - p) : 0 with the mask regenerated from (seed, offset), and its gradient
  dropout_add_layer_norm  y = layer_norm(residual + dropout(x)), and its gradients

The mask: element e (row-major index in the tensor) sits in block e // 8, slot e % 8.  Philox4x32-10 (Salmon et al., SC'11) of the 128-bit
counter (2 * block + part, offset) under the 64-bit key `seed` gives four words = eight 16-bit numbers; part 0 holds the upper and part 1
the lower half of the element's 32-bit number, which keeps the element where it is at least round(p * 2^32).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases

def _case(name, op, direction, rows, cols, x="f32", res=None, params="f32", affine="both", p=0.1, of=0):
    c = {"op": op, "direction": direction, "rows": rows, "cols": cols, "x": x, "p": p if op != "layer_norm" else 0.0}
    if op != "dropout":
        c.update(params=params, affine=affine)
    if op == "dropout_add_layer_norm":
        c["res"] = res or x
    if of:
        c["of"] = of           # x is the first `cols` columns of rows of this many
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one frame's normalisation of a handful of clicked points: a launch's latency is all there is
        _case("ln fwd 8x256 f32", "layer_norm", "fwd", 8, 256),
        # the points of a frame (1024 tracked points, 256 channels), a training step
        _case("ln train 1024x256 f32", "layer_norm", "train", 1024, 256),
        # 64 streams x 1024 points: the query columns of a merged projection, normalised where they lie
        _case("ln fwd 65536x256of1024 f16", "layer_norm", "fwd", 65536, 256, x="f16", of=1024),
        # a pyramid's tokens (16320) with one channel appended: rows that start at odd addresses
        _case("ln train 16320x257 bf16", "layer_norm", "train", 16320, 257, x="bf16", params="x"),
        # generic: a wide model's tokens
        _case("ln train 8192x8192 bf16", "layer_norm", "train", 8192, 8192, x="bf16"),
        # hidden activations of the feed-forward (4 x 256) at a frame's points
        _case("drop fwd 1024x1024 f32", "dropout", "fwd", 1024, 1024),
        # generic odd sizes, half precision: a total that is no multiple of any vector
        _case("drop train 9217x1021 f16", "dropout", "train", 9217, 1021, x="f16", p=0.25),
        # hidden activations of 64 streams x 1024 points
        _case("drop train 65536x1024 bf16", "dropout", "train", 65536, 1024, x="bf16"),
        # a block's residual join at a few points
        _case("join train 64x256 f32", "dropout_add_layer_norm", "train", 64, 256),
        # lattice tokens (1024 points x 9 neighbours) under half-precision autocast: products f16, residual stream f32
        _case("join train 9216x256 f16+f32", "dropout_add_layer_norm", "train", 9216, 256, x="f16", res="f32"),
        # the first pass of a checkpointed block (no gradient taken), odd sizes
        _case("join fwd 4099x1537 bf16", "dropout_add_layer_norm", "fwd", 4099, 1537, x="bf16", params="x"),
        # lattice tokens of 64 streams x 1024 points x 9 neighbours
        _case("join train 589824x256 bf16", "dropout_add_layer_norm", "train", 589824, 256, x="bf16"),
    ]


def draw(rng):
    while True:
        op = rng.choice(["layer_norm", "dropout", "dropout_add_layer_norm"])
        direction = rng.choice(["fwd", "train", "train"])
        x = rng.choice(["f32", "f16", "bf16"])
        cols = int(math.exp(rng.uniform(math.log(32), math.log(16384))))
        if rng.random() < 0.5:
            cols = max(32, cols // 8 * 8)          # the rest as it falls: odd ones among them
        total = math.exp(rng.uniform(math.log(2048), math.log(589824 * 256)))
        rows = max(1, min(589824, int(total / cols)))
        res = rng.choice([x, "f32"])
        of = cols + 8 * rng.randint(1, 64) if op == "layer_norm" and rng.random() < 0.25 else 0
        c = _case(None, op, direction, rows, cols, x=x, res=res, params=rng.choice(["f32", "x"]), affine=rng.choice(["both", "both", "weight", "none"]),
                  p=round(rng.uniform(0.01, 0.6), 4), of=of)
        if work(c)["bytes"] <= 6 * 589824 * 256 * 2 and rows * (of or cols) * TYPES[x].itemsize <= 2 * 2 ** 30:
            return c


def _dtypes(case):
    x = TYPES[case["x"]]
    res = TYPES[case.get("res", case["x"])]
    return x, res, (torch.float32 if case.get("params") == "f32" else x)


def work(case):
    n, d = case["rows"] * case["cols"], case["cols"]
    tx, tr, tw = (t.itemsize for t in _dtypes(case))
    train = case["direction"] == "train"
    if case["op"] == "dropout":
        return {"bytes": n * tx * (4 if train else 2), "flops": n * (6 if train else 3)}
    par = {"both": 2, "weight": 1, "none": 0}[case["affine"]] * d * tw
    if case["op"] == "layer_norm":
        return {"bytes": n * tx * (4 if train else 2) + par * (2 if train else 1), "flops": n * (20 if train else 8)}
    # x, residual -> y; and dy -> dx, dresidual
    return {"bytes": n * ((2 * tx + 4 * tr) if train else (tx + 2 * tr)) + par * (2 if train else 1), "flops": n * (26 if train else 12)}


# ---------------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tx, tr, tw = _dtypes(case)
    rows, cols, train = case["rows"], case["cols"], case["direction"] == "train"

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    # activations: rows of different scales and offsets
    x = (normal(rows, case.get("of") or cols).mul_(normal(rows, 1).mul_(0.5).exp_()).add_(normal(rows, 1).mul_(0.3))).to(tx)
    s = {"case": case, "x": x[:, :cols]}
    if case["op"] != "layer_norm":
        s["seed"] = int(torch.randint(0, 2 ** 62, (1,), generator=torch.Generator().manual_seed(seed)))
        s["offset"] = seed % 1000 + 3
    if case["op"] != "dropout":
        s["weight"] = (1 + 0.1 * normal(cols)).to(tw) if case["affine"] != "none" else None
        s["bias"] = (0.1 * normal(cols)).to(tw) if case["affine"] == "both" else None
    if case["op"] == "dropout_add_layer_norm":
        s["residual"] = normal(rows, cols).to(tr)
    if train:
        s["dy"] = normal(rows, cols).to(tr if case["op"] == "dropout_add_layer_norm" else tx)
        s["wanted"] = [k for k in ("x", "residual", "weight", "bias") if s.get(k) is not None]
        for k in s["wanted"]:
            s[k].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------- one pass through an operator

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from lbm_amd import dropout, dropout_add_layer_norm, layer_norm
    case = s["case"]
    if case["op"] == "layer_norm":
        y = layer_norm(s["x"], s["weight"], s["bias"])
    elif case["op"] == "dropout":
        y = dropout(s["x"], case["p"], s["seed"], s["offset"])
    else:
        y = dropout_add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], p=case["p"], seed=s["seed"], offset=s["offset"])
    if case["direction"] == "fwd":
        return {"y": y}
    grads = torch.autograd.grad(y, [s[k] for k in s["wanted"]], s["dy"])
    return {"y": y.detach(), **{"d" + k: t for k, t in zip(s["wanted"], grads)}}


def _philox(counter, offset, seed):
    """Philox4x32-10 over an int64 tensor of 64-bit counters; 32-bit words in int64 (products wrap, their bits stay right)."""
    m = 0xFFFFFFFF
    c = [counter & m, (counter >> 32) & m, torch.full_like(counter, offset & m), torch.full_like(counter, (offset >> 32) & m)]
    k0, k1 = seed & m, (seed >> 32) & m
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & m) ^ c[1] ^ k0, b & m, ((a >> 32) & m) ^ c[3] ^ k1, a & m]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return c


def _plain_keep(s, shape):
    n = shape[0] * shape[1]
    block = torch.arange((n + 7) // 8, device="cuda")
    high, low = _philox(2 * block, s["offset"], s["seed"]), _philox(2 * block + 1, s["offset"], s["seed"])
    number = torch.stack([((high[j >> 1] >> 16 * (j & 1) & 0xFFFF) << 16) | (low[j >> 1] >> 16 * (j & 1) & 0xFFFF) for j in range(8)], 1)
    return (number.reshape(-1)[:n] >= round(s["case"]["p"] * 2 ** 32)).view(shape)


@torch.no_grad()
def _plain(s):
    case, train = s["case"], s["case"]["direction"] == "train"
    x = s["x"].float()
    if case["op"] != "layer_norm":
        keep, scale = _plain_keep(s, x.shape), 1 / (1 - case["p"])
        x = torch.where(keep, x * scale, 0.0)
    if case["op"] == "dropout":
        out = {"y": x.to(s["x"].dtype)}
        if train:
            out["dx"] = torch.where(keep, s["dy"].float() * scale, 0.0).to(s["x"].dtype)
        return out
    kind = s["x"].dtype
    if case["op"] == "dropout_add_layer_norm":
        x = s["residual"].float() + x
        kind = s["residual"].dtype
    x = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-5)
    xhat = x * rstd
    y = xhat
    if s["weight"] is not None:
        y = y * s["weight"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    out = {"y": y.to(kind)}
    if train:
        dy = s["dy"].float()
        g = dy if s["weight"] is None else dy * s["weight"].float()
        dz = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * rstd
        if case["op"] == "dropout_add_layer_norm":
            out["dx"] = torch.where(keep, dz * scale, 0.0).to(s["x"].dtype)
            out["dresidual"] = dz.to(kind)
        else:
            out["dx"] = dz.to(kind)
        if s["weight"] is not None:
            out["dweight"] = (dy * xhat).sum(0).to(s["weight"].dtype)
        if s["bias"] is not None:
            out["dbias"] = dy.sum(0).to(s["bias"].dtype)
    return out


# ------------------------------------------------------------------------------------------------- the definition in 64 bits

def _exact_numbers(first, count, seed, offset, part):
    """The eight 16-bit halves of `count` blocks from block `first`, by 16-bit limbs: (count, 8)."""
    def times(v, mul):                                    # 32 x 32 -> (high, low), no product over 48 bits
        upper, lower = v * (mul >> 16), v * (mul & 0xFFFF)
        rest = (upper & 0xFFFF) * 65536 + lower
        return (upper >> 16) + (rest >> 32), rest % 4294967296

    n = (torch.arange(count, device="cuda") + first) * 2 + part
    w = torch.stack([n % 4294967296, n // 4294967296, torch.full_like(n, offset % 4294967296), torch.full_like(n, offset // 4294967296)])
    for r in range(10):
        key = [(seed % 4294967296 + r * 0x9E3779B9) % 4294967296, (seed // 4294967296 + r * 0xBB67AE85) % 4294967296]
        h0, l0 = times(w[0], 0xD2511F53)
        h1, l1 = times(w[2], 0xCD9E8D57)
        w = torch.stack([torch.bitwise_xor(torch.bitwise_xor(h1, w[1]), key[0]), l1, torch.bitwise_xor(torch.bitwise_xor(h0, w[3]), key[1]), l0])
    return torch.stack([w % 65536, w // 65536], 1).permute(2, 0, 1).reshape(count, 8)


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        rows, cols = case["rows"], case["cols"]
        z = s["x"].double()
        if case["op"] != "layer_norm":
            factor = torch.empty(rows * cols, device="cuda", dtype=torch.float64)
            per = 1 << 22
            for b in range(0, (rows * cols + 7) // 8, per):
                k = min(per, (rows * cols + 7) // 8 - b)
                u = _exact_numbers(b, k, s["seed"], s["offset"], 0) * 65536 + _exact_numbers(b, k, s["seed"], s["offset"], 1)
                part = factor[8 * b:8 * (b + k)]
                part.copy_((u >= round(case["p"] * 2 ** 32)).double().div_(1 - case["p"]).reshape(-1)[:part.numel()])
            factor = factor.view(rows, cols)
            z = z * factor
        if case["op"] == "dropout":
            out = {"y": z}
            if case["direction"] == "train":
                out["dx"] = s["dy"].double() * factor
            return out
        if case["op"] == "dropout_add_layer_norm":
            z += s["residual"].double()
        var, mean = torch.var_mean(z, 1, correction=0, keepdim=True)
        sd = (var + 1e-5).sqrt()
        z = z.sub_(mean).div_(sd)                         # the normalised rows
        w = torch.ones(cols, device="cuda", dtype=torch.float64) if s["weight"] is None else s["weight"].double()
        b = torch.zeros(cols, device="cuda", dtype=torch.float64) if s["bias"] is None else s["bias"].double()
        out = {"y": torch.addcmul(b, z, w)}
        if case["direction"] == "train":
            dy = s["dy"].double()
            if s["weight"] is not None:
                dw = torch.einsum("ij,ij->j", dy, z)
            if s["bias"] is not None:
                db = torch.einsum("ij->j", dy)
            dy = dy.mul_(w)
            slope, level = torch.einsum("ij,ij->i", dy, z)[:, None] / cols, torch.einsum("ij->i", dy)[:, None] / cols
            dz = dy.sub_(level).sub_(z.mul_(slope)).div_(sd)
            if case["op"] == "dropout_add_layer_norm":
                out["dx"], out["dresidual"] = dz * factor, dz
            else:
                out["dx"] = dz
            if s["weight"] is not None:
                out["dweight"] = dw
            if s["bias"] is not None:
                out["dbias"] = db
        return out
