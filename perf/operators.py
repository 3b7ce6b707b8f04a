"""What the operators of a feature-map decoder cost: matrix product with bias, activation and residual in its epilogue
(``linear``), layer norm (``layer_norm``) and dropout from a counter-based generator (``dropout``).

The rasterizer's index map hands every pixel a 64-wide feature row; the networks that turn such rows into colours are
stacks of these three operators, run over whole images when training and rendering and over single rows when a point is
queried.  This file lists cases of that work, makes their inputs, and computes them in a plain form (elementary torch
operations) or, where ``own`` is true, through ``neuralgaussiansplatting_amd.decoder_ops``.

A case is a dict of plain values:

    op        "linear", "norm" or "dropout"
    rows      number of rows (pixels, points or tokens)
    k         width of a row: what a product sums over, what a norm is taken of
    n         linear: width of its output
    dtype     "float32", "bfloat16" or "float16"
    act       linear: "none", "relu", "gelu" (x Phi(x)), "silu" or "sigmoid"
    residual  linear, dropout: whether a residual of the output's shape is added last
    first     columns in front of the row inside the wider tensor that it is a slice of
    pitch     width of that tensor (k when the rows are contiguous)
    p         dropout: the probability
    train     whether the pass goes back as well, with a given gradient of the output
"""
import math

import torch

own = False

FULL_HD = 1920 * 1080
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


def _case(name, op, rows, k, dtype, n=0, act="none", residual=False, first=0, pitch=0, p=0.0, train=False):
    return dict(name=name, op=op, rows=rows, k=k, n=n, dtype=dtype, act=act, residual=residual, first=first,
                pitch=pitch or k, p=p, train=train)


def listed():
    return [
        # one point is asked for its value by a wide network: nothing but the weights' way through the memory counts
        _case("linear_one_row", "linear", 1, 1024, "bfloat16", n=4096, act="gelu"),
        # the first layer over a full-HD feature map in the rasterizer's own type, while rendering
        _case("linear_image_f32", "linear", FULL_HD, 64, "float32", n=128, act="relu"),
        # the second half of a residual block over an 800 x 800 training view, there and back
        _case("linear_block_train", "linear", 800 * 800, 128, "bfloat16", n=128, act="gelu", residual=True, train=True),
        # colours straight from the copied features (columns 25..63 of a feature row), there and back: odd and unaligned
        _case("linear_rgb_train", "linear", 800 * 800, 39, "float32", n=3, act="sigmoid", first=25, pitch=64, train=True),
        # the products of a wide network's training step: bound by the matrix units
        _case("linear_wide_train", "linear", 8192, 4096, "bfloat16", n=4096, act="silu", train=True),
        # the same kind of work at sizes that divide by nothing
        _case("linear_odd", "linear", 4099, 1001, "float16", n=2003, residual=True),
        # the norm in front of a block over a full-HD feature map, there and back
        _case("norm_image_train", "norm", FULL_HD, 64, "float32", train=True),
        # one row
        _case("norm_one_row", "norm", 1, 4096, "bfloat16"),
        # wide rows of an odd width and number, there and back
        _case("norm_wide_train", "norm", 8191, 5001, "float16", train=True),
        # a 64 x 64 tile of features
        _case("dropout_tile", "dropout", 64 * 64, 64, "float32", p=0.1),
        # dropout in front of the sum of a residual block over a full-HD map, there and back
        _case("dropout_image_train", "dropout", FULL_HD, 64, "bfloat16", residual=True, p=0.1, train=True),
        # the copied features alone, as a slice of the feature map
        _case("dropout_slice", "dropout", 400 * 400, 39, "float16", first=25, pitch=64, p=0.5),
    ]


def _between(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]; every other time a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 16:
        v = v // 8 * 8
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "dropout"])
    dtype = rng.choice(sorted(DTYPES))
    c = _case("", op, 1, 1, dtype, train=rng.random() < 0.5)
    if op == "linear":
        kind = rng.choice(["rows", "image", "wide"])
        if kind == "rows":  # a few queries of a wide network
            c["rows"], c["k"], c["n"], c["train"] = _between(rng, 1, 48), _between(rng, 64, 8192), _between(rng, 64, 8192), False
        elif kind == "image":  # a narrow layer over many pixels
            c["rows"], c["k"], c["n"] = _between(rng, 4096, FULL_HD), _between(rng, 3, 256), _between(rng, 3, 256)
        else:
            c["rows"], c["k"], c["n"] = _between(rng, 64, 16384), _between(rng, 256, 8192), _between(rng, 256, 8192)
        # (the gradient of relu at a product that is zero but for rounding is either of two values: forward only)
        c["act"] = rng.choice(["none", "gelu", "silu", "sigmoid"] + ([] if c["train"] else ["relu"]))
        c["residual"] = rng.random() < 0.5
    else:
        c["rows"], c["k"] = _between(rng, 1, FULL_HD), _between(rng, 2, 16384)
        if op == "dropout":
            c["p"], c["residual"] = rng.choice([0.05, 0.1, 0.25, 0.5]), rng.random() < 0.5
    c["first"] = rng.choice([0, 0, 0, 25])
    c["pitch"] = c["first"] + c["k"] + rng.choice([0, 0, 8]) if c["first"] else c["k"]
    most = [work(x) for x in listed()]
    while c["rows"] > 1 and any(work(c)[key] > max(m[key] for m in most) for key in ("bytes", "flops")):
        c["rows"] = c["rows"] * 3 // 4
    while any(work(c)[key] > max(m[key] for m in most) for key in ("bytes", "flops")):
        c["k"], c["n"] = max(c["k"] * 3 // 4, 1), max(c["n"] * 3 // 4, 1)
        c["pitch"] = c["first"] + c["k"]
    del c["name"]
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, k = DTYPES[case["dtype"]], case["rows"], case["k"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)

    def leaf(t):
        return t.detach().requires_grad_(case["train"])

    x = normal(rows, case["pitch"])
    if case["op"] == "norm":  # channels of a residual stream have scales and offsets of their own
        x = (x.float() * (0.5 + torch.rand(case["pitch"], generator=g, device="cuda")) + normal(case["pitch"], scale=0.5)).to(dtype)
    s = {"case": case, "x": leaf(x[:, case["first"]:case["first"] + k])}
    if case["op"] == "linear":
        s["weight"] = leaf(normal(case["n"], k, scale=k ** -0.5))
        s["bias"] = leaf(normal(case["n"], scale=0.1))
    elif case["op"] == "norm":
        s["weight"] = leaf(normal(k, scale=0.1) + 1)
        s["bias"] = leaf(normal(k, scale=0.1))
    else:
        s["seed"], s["offset"] = seed * 7919 + 12345, seed % 97
    out = case["n"] if case["op"] == "linear" else k
    if case["residual"]:
        s["residual"] = leaf(normal(rows, out))
    if case["train"]:
        s["dy"] = normal(rows, out, scale=0.02)
    return s


def run(state):
    case = state["case"]
    if own:
        from neuralgaussiansplatting_amd import decoder_ops
        if case["op"] == "linear":
            y = decoder_ops.linear(state["x"], state["weight"], state["bias"], activation=case["act"],
                                   residual=state.get("residual"))
        elif case["op"] == "norm":
            y = decoder_ops.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS)
        else:
            y = decoder_ops.dropout(state["x"], case["p"], state["seed"], offset=state["offset"],
                                    residual=state.get("residual"))
        return _with_gradients(state, y)
    with torch.no_grad():
        return {"linear": _linear, "norm": _norm, "dropout": _dropout}[case["op"]](state)


def _with_gradients(state, y):
    if not state["case"]["train"]:
        return {"y": y}
    names = [n for n in ("x", "weight", "bias", "residual") if n in state]
    grads = torch.autograd.grad(y, [state[n] for n in names], state["dy"])
    return {"y": y.detach(), **{"d" + n: d for n, d in zip(names, grads)}}


# ---- the plain forms: 32 bits throughout, one rounding at the end ----


def _linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t() + s["bias"].float()
    y, slope = _activation(z, case["act"], case["train"])
    if "residual" in s:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dz = s["dy"].float()
        if slope is not None:
            dz = dz * slope
        out["dx"] = (dz @ w).to(dtype)
        out["dweight"] = (dz.t() @ x).to(dtype)
        out["dbias"] = dz.sum(0).to(dtype)
        if "residual" in s:
            out["dresidual"] = s["dy"]
    return out


def _activation(z, act, train):
    """The activation of z and, for training, its derivative (None: one everywhere)."""
    if act == "relu":
        return torch.where(z < 0, 0.0, z), (z > 0).float() if train else None
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5 if train else None
    if act in ("silu", "sigmoid"):
        s = 1.0 / (1.0 + torch.exp(-z))
        if act == "sigmoid":
            return s, s * (1.0 - s) if train else None
        return z * s, s * (1.0 + z * (1.0 - s)) if train else None
    return z, None


def _norm(s):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xhat = centred * rstd
    out = {"y": (xhat * w + s["bias"].float()).to(dtype)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy * w
        out["dx"] = (rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))).to(dtype)
        out["dweight"] = (dy * xhat).sum(0).to(dtype)
        out["dbias"] = dy.sum(0).to(dtype)
    return out


LOW = 0xFFFFFFFF


def _times(a, b):
    """High and low word of the product of a 32-bit constant and 32-bit words, held in 64-bit integers: the constant
    goes in two halves, since the whole product would not fit below the sign."""
    low = (a & 0xFFFF) * b
    high = (a >> 16) * b + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _kept(numel, p, seed, offset, device):
    """Element i takes 16 bits from block i // 8 of Philox 4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw: Parallel
    Random Numbers: As Easy as 1, 2, 3, 2011): key = the seed's two words, counter = (block, offset), two words each.
    Kept are the elements whose bits are at least p 2^16."""
    block = torch.arange((numel + 7) // 8, device=device)
    c = [block & LOW, block >> 32, torch.full_like(block, offset & LOW), torch.full_like(block, (offset >> 32) & LOW)]
    key = [seed & LOW, (seed >> 32) & LOW]
    for _ in range(7):
        h0, l0 = _times(0xD2511F53, c[0])
        h1, l1 = _times(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & LOW, (key[1] + 0xBB67AE85) & LOW]
    words = torch.stack(c, 1)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:numel]
    return bits >= _threshold(p)


def _threshold(p):
    return int(math.floor(p * 65536.0 + 0.5))


def _dropout(s):
    case, dtype = s["case"], s["x"].dtype
    rows, k = s["x"].shape
    keep = _kept(rows * k, case["p"], s["seed"], s["offset"], s["x"].device).view(rows, k)
    scale = 65536.0 / (65536 - _threshold(case["p"]))
    y = torch.where(keep, s["x"].float() * scale, 0.0)
    if "residual" in s:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        out["dx"] = torch.where(keep, s["dy"].float() * scale, 0.0).to(dtype)
        if "residual" in s:
            out["dresidual"] = s["dy"]
    return out


# ---- the definitions in 64 bits, written apart from the plain forms ----


def exact(case, seed):
    s = {n: t.detach().double() if torch.is_tensor(t) else t for n, t in prepare(case, seed).items()}
    return {"linear": _exact_linear, "norm": _exact_norm, "dropout": _exact_dropout}[case["op"]](case, s)


def _exact_linear(case, s):
    z = torch.addmm(s["bias"], s["x"], s["weight"].t().contiguous())
    value = {"none": lambda: z.clone(), "relu": lambda: z.clamp(min=0), "gelu": lambda: z * torch.special.ndtr(z),
             "silu": lambda: z * torch.sigmoid(z), "sigmoid": lambda: torch.sigmoid(z)}[case["act"]]()
    out = {"y": value + s["residual"] if "residual" in s else value}
    if case["train"]:
        if case["act"] == "none":
            slope = torch.ones_like(z)
        elif case["act"] == "relu":
            slope = torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
        elif case["act"] == "gelu":
            slope = torch.special.ndtr(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        else:
            up, down = torch.sigmoid(z), torch.sigmoid(-z)
            slope = up * down if case["act"] == "sigmoid" else up + z * up * down
        dz = s["dy"] * slope
        out["dx"] = torch.mm(dz, s["weight"])
        out["dweight"] = torch.mm(dz.t().contiguous(), s["x"])
        out["dbias"] = dz.sum(0)
        if "residual" in s:
            out["dresidual"] = s["dy"]
    return out


def _exact_norm(case, s):
    x = s["x"]
    spread, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    root = (spread + EPS).sqrt()
    unit = (x - mean) / root
    out = {"y": torch.addcmul(s["bias"], unit, s["weight"])}
    if case["train"]:
        # the gradient of w.unit is projected off the constant row and off the row itself
        up = s["dy"] * s["weight"]
        along = (up * unit).sum(1, keepdim=True) / case["k"]
        out["dx"] = (up - up.sum(1, keepdim=True) / case["k"] - along * unit) / root
        out["dweight"] = (s["dy"] * unit).sum(0)
        out["dbias"] = s["dy"].sum(0)
    return out


def _exact_dropout(case, s):
    import numpy as np
    numel = case["rows"] * case["k"]
    # counters and key as unsigned 64-bit numbers: the product of two words fits
    word, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    block = np.arange((numel + 7) // 8, dtype=np.uint64)
    a, b = block & word, block >> half
    c, d = np.full_like(block, s["offset"] & 0xFFFFFFFF), np.full_like(block, (s["offset"] >> 32) & 0xFFFFFFFF)
    for r in range(7):
        k0 = np.uint64(((s["seed"] & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = np.uint64((((s["seed"] >> 32) & 0xFFFFFFFF) + r * 0xBB67AE85) & 0xFFFFFFFF)
        left, right = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (right >> half) ^ b ^ k0, right & word, (left >> half) ^ d ^ k1, left & word
    bits = np.ascontiguousarray(np.stack((a, b, c, d), 1).astype("<u4")).view("<u2").reshape(-1)[:numel]
    drop = round(case["p"] * 65536)
    keep = torch.from_numpy(bits.astype(np.int32) >= drop).to(s["x"].device).view(case["rows"], case["k"])
    factor = keep.double() * (65536 / (65536 - drop))
    out = {"y": s["x"] * factor + (s["residual"] if "residual" in s else 0)}
    if case["train"]:
        out["dx"] = s["dy"] * factor
        if "residual" in s:
            out["dresidual"] = s["dy"]
    return out


def work(case):
    """Each input read once, each output written once; a residual's gradient is the output's and costs nothing."""
    size = 4 if case["dtype"] == "float32" else 2
    rows, k, n = case["rows"], case["k"], case["n"]
    if case["op"] == "linear":
        params, out = n * k + n, rows * n
        elements = rows * k + params + out * (2 if case["residual"] else 1)
        if case["train"]:
            elements += out + rows * k + params
        return {"bytes": elements * size, "flops": (6 if case["train"] else 2) * rows * n * k}
    if case["op"] == "norm":
        elements = 2 * rows * k + 2 * k
        if case["train"]:
            elements += 2 * rows * k + 2 * k
        return {"bytes": elements * size, "flops": (20 if case["train"] else 8) * rows * k}
    elements = rows * k * (3 if case["residual"] else 2)
    if case["train"]:
        elements += 2 * rows * k
    return {"bytes": elements * size, "flops": (4 if case["train"] else 2) * rows * k}
