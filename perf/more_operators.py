"""The calls that the encoder-layer operators are measured on.

``op`` names the call and the rest its sizes, types and options:

dropout    prims.dropout, with or without a residual
norm       prims.group_norm: group norm, channels last, with an activation
norm_train prims.group_norm with dropout, then prims.group_norm_grad
fp8        prims.linear_fp8: a layer in 8-bit floating point, weights laid out
           beforehand
fp8_train  prims.fp8_weight, prims.linear_fp8, then prims.linear_fp8_grad

With ``own`` false the same is computed from elementary torch operations in
float32, rounded once at the end.

What both sides compute.  Random bits: element i takes 16 bits of Philox 4x32
(7 rounds; Salmon et al., SC 2011) with the key `seed` and the counter (i / 8,
`offset`): the low half of word (i % 8) / 2 where i is even, else the high one.
It is kept where they are at least t = round(65536 p).  8-bit floating point:
e4m3 codes (largest 448, no infinities); a block's scale is the least power of
two with which no magnitude passes 448 (1 for a block of zeros).  A block is 128
consecutive elements of a contraction axis, of weights a 128 x 128 tile.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SEED, OFFSET, EPS = 0x5EED12345678, 41, 1e-5


def listed():
    return [
        # A small training batch of an encoder's hidden layer: latency.
        dict(name="dropout_small_f32", op="dropout", dtype="f32", n=256, d=512, p=0.1, residual=False),
        # The end of a residual block at a training batch.
        dict(name="dropout_residual", op="dropout", dtype="bf16", n=16384, d=4096, p=0.1, residual=True),
        # One row through a hidden layer's norm, as an online encoder answers a
        # single request.
        dict(name="norm_one_row", op="norm", dtype="bf16", n=1, s=1, c=1024, groups=8, act="silu"),
        # Feature maps of 64 x 64 positions, channels last, evaluated.
        dict(name="norm_map", op="norm", dtype="f16", n=16, s=4096, c=320, groups=32, act="silu"),
        # A training step through a hidden layer's norm, rows only.
        dict(name="norm_train_rows", op="norm_train", dtype="bf16", n=16384, s=1, c=2048, groups=16, act="gelu", p=0.1),
        # A training step on small feature maps, no size a multiple of a vector.
        dict(name="norm_train_ragged_f32", op="norm_train", dtype="f32", n=37, s=49, c=250, groups=10, act="relu",
             p=0.25),
        # A training step on middle feature maps.
        dict(name="norm_train_map", op="norm_train", dtype="bf16", n=16, s=1024, c=640, groups=32, act="silu", p=0.0),
        # One row through a wide layer: the weights' bytes are all there is.
        dict(name="fp8_one_row", op="fp8", dtype="bf16", n=1, k=4096, m=8192, act="none", bias=True, residual=False),
        # The benchmark's small query batch through a layer of odd sizes.
        dict(name="fp8_ragged_f16", op="fp8", dtype="f16", n=1001, k=1000, m=2050, act="gelu_tanh", bias=True,
             residual=True),
        # A large batch through a square layer with everything its epilogue can do.
        dict(name="fp8_batch", op="fp8", dtype="bf16", n=16384, k=4096, m=4096, act="gelu", bias=True, residual=True),
        # A training step of a single-precision layer, odd counts everywhere.
        dict(name="fp8_train_ragged_f32", op="fp8_train", dtype="f32", n=3001, k=1000, m=2050, act="relu"),
        # A training step of a wide layer: the largest call.
        dict(name="fp8_train_batch", op="fp8_train", dtype="bf16", n=8192, k=4096, m=8192, act="gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo + 1, hi))))))


def draw(rng):
    """One more call of the ranges the listed ones stand for."""
    op = rng.choice(["dropout", "norm", "norm_train", "norm_train", "fp8", "fp8", "fp8_train", "fp8_train"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    if op == "dropout":
        d = _log(rng, 1, 8192)
        n = _log(rng, 1, 6e7 / d)
        return dict(op=op, dtype=dtype, n=n, d=d, p=round(rng.uniform(0.0, 0.9), 3), residual=rng.random() < 0.5)
    if op in ("norm", "norm_train"):
        groups = _log(rng, 1, 64)
        s = 1 if rng.random() < 0.4 else _log(rng, 4, 4096)
        c = groups * _log(rng, 8 if s == 1 else 2, 8192 / groups)
        n = _log(rng, 1, min(32768, max(2, 3e7 / (c * s))))
        case = dict(op=op, dtype=dtype, n=n, s=s, c=c, groups=groups, act=act)
        if op == "norm_train":
            case["p"] = round(rng.uniform(0.0, 0.5), 3) if rng.random() < 0.6 else 0.0
        return case
    k, m = _log(rng, 16, 8192), _log(rng, 16, 8192)
    if rng.random() < 0.5:
        k, m = (-(-t // 64) * 64 for t in (k, m))
    most = 2.7e11 if op == "fp8" or dtype != "f32" else 1.3e11
    n = _log(rng, 1 if op == "fp8" else 16, min(32768, most / (k * m)))
    if op == "fp8":
        return dict(op=op, dtype=dtype, n=n, k=k, m=m, act=act, bias=rng.random() < 0.7, residual=rng.random() < 0.5)
    return dict(op=op, dtype=dtype, n=n, k=k, m=m, act=act)


def _normal(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    t = torch.empty(shape, dtype=torch.float32, device="cuda")
    t.normal_(mean, std, generator=g)
    return t.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6271 + 5)
    dt = _DT[case["dtype"]]
    s = dict(case=case, seed=SEED + int(seed))
    if case["op"] == "dropout":
        n, d = case["n"], case["d"]
        s["x"] = _normal(g, n, d, dtype=dt)
        s["res"] = _normal(g, n, d, dtype=dt) if case["residual"] else None
        return s
    if case["op"] in ("norm", "norm_train"):
        n, p, c = case["n"], case["s"], case["c"]
        # what a layer puts out: its own mean and size in every channel
        scale = torch.empty(c, device="cuda").uniform_(0.5, 2.0, generator=g)
        shift = _normal(g, c, std=0.5)
        s["x"] = (_normal(g, n, p, c) * scale + shift).to(dt)
        s["w"] = _normal(g, c, dtype=dt, std=0.2, mean=1.0)
        s["b"] = _normal(g, c, dtype=dt, std=0.2)
        if case["op"] == "norm_train":
            s["dy"] = _normal(g, n, p, c, dtype=dt)
        return s
    n, k, m = case["n"], case["k"], case["m"]
    x = _normal(g, n, k)
    x *= torch.where(torch.rand(k, generator=g, device="cuda") < 0.02, 8.0, 1.0)  # a few strong features
    s["x"] = x.to(dt)
    s["w"] = _normal(g, m, k, dtype=dt, std=k ** -0.5)
    s["b"] = _normal(g, m, dtype=dt, std=0.1) if case.get("bias", True) else None
    if case["op"] == "fp8_train":
        s["dy"] = _normal(g, n, m, dtype=dt, std=0.02)
        return s
    s["res"] = _normal(g, n, m, dtype=dt) if case["residual"] else None
    # the weights as the layer keeps them: codes of whole blocks, and a byte (the
    # exponent + 127) for each tile, a row of tiles in whole words
    value, exponent = _tiles(s.pop("w").float())
    codes = torch.zeros(m, -(-k // 128) * 128, device="cuda")
    codes[:, :k] = value / _spread(exponent, m, k)
    s["codes"] = codes.to(torch.float8_e4m3fn)
    s["scales"] = torch.full((exponent.shape[0], -(-k // 512) * 4), 127, dtype=torch.uint8, device="cuda")
    s["scales"][:, :exponent.shape[1]] = (exponent + 127).to(torch.uint8)
    return s


# ---- the plain forms: float32 throughout, rounded once at the end ----

def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-z))
        return sg * (1.0 + z * (1.0 - sg))
    return torch.ones_like(z)


def _threshold(p):
    return min(65535, int(math.floor(p * 65536 + 0.5)))


def _factor(shape, p, seed, device):
    """What dropout multiplies by, float32: 0, or 1 / (1 - t / 65536)."""
    t = _threshold(p)
    count = math.prod(shape)
    block = torch.arange(-(-count // 8), device=device)
    low = 0xFFFFFFFF
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, OFFSET & low), torch.full_like(block, OFFSET >> 32)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).view(-1)[:count]
    return torch.where(halves >= t, torch.full((), 65536.0 / (65536 - t), device=device), 0.0).view(shape)


def _plain_dropout(s):
    x = s["x"]
    y = x.float() * _factor(x.shape, s["case"]["p"], s["seed"], x.device)
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(x.dtype)


def _plain_norm(s):
    case = s["case"]
    x, dt = s["x"], s["x"].dtype
    n, p, c = x.shape
    g = case["groups"]
    count = p * (c // g)
    v = x.float().view(n, p, g, c // g)
    mean = v.sum((1, 3)) / count
    v = v - mean.view(n, 1, g, 1)
    rstd = 1.0 / torch.sqrt((v * v).sum((1, 3)) / count + EPS)
    v = (v * rstd.view(n, 1, g, 1)).view(n, p, c)  # the normalised x
    w = s["w"].float()
    z = v * w + s["b"].float()
    y = _act(z, case["act"])
    if case["op"] == "norm":
        return y.to(dt)
    dz = s["dy"].float()
    if case["p"]:
        by = _factor(x.shape, case["p"], s["seed"], x.device)
        y = y * by
        dz = dz * by
        del by
    dz = dz * _act_slope(z, case["act"])
    out = [y.to(dt), mean, rstd]
    del y, z
    db, dw = dz.sum((0, 1)), (dz * v).sum((0, 1))
    dv = (dz * w).view(n, p, g, c // g)
    v = v.view(n, p, g, c // g)
    s1, s2 = dv.sum((1, 3)) / count, (dv * v).sum((1, 3)) / count
    dx = rstd.view(n, 1, g, 1) * (dv - s1.view(n, 1, g, 1) - v * s2.view(n, 1, g, 1))
    return out + [dx.view(n, p, c).to(dt), dw.to(dt), db.to(dt)]


def _exponent(top):
    """The least e with top <= 448 * 2^e, 0 for no magnitude at all."""
    bits = top.view(torch.int32)
    e = ((bits >> 23) & 255) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)
    return torch.where(top > 0, e, 0).clamp_(-127, 127)


def _power(e):
    """2^e, -127 <= e <= 127, from its bits."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _e4m3(v):
    """v (at most 448 in magnitude) rounded to three bits of fraction, half to even."""
    bits = v.view(torch.int32)
    big = ((bits + 0x7FFFF + ((bits >> 20) & 1)) & ~0xFFFFF).view(torch.float32)
    return torch.where(v.abs() < 2.0 ** -6, torch.round(v * 512.0) / 512.0, big)


def _rows8(x):
    """The values that 8 bits keep of x, a scale for each 128 of a row."""
    n, k = x.shape
    v = torch.nn.functional.pad(x, (0, -k % 128)).view(n, -1, 128)
    up = _power(_exponent(v.abs().amax(2)))[:, :, None]
    return (_e4m3(v / up) * up).view(n, -1)[:, :k]


def _spread(exponent, m, k):
    """Every element's scale."""
    return _power(exponent).repeat_interleave(128, 0)[:m].repeat_interleave(128, 1)[:, :k]


def _tiles(w):
    """The values that 8 bits keep of w, a scale for each 128 x 128, and the exponents."""
    m, k = w.shape
    v = torch.nn.functional.pad(w, (0, -k % 128, 0, -m % 128))
    top = v.abs().view(v.shape[0] // 128, 128, v.shape[1] // 128, 128).amax((1, 3))
    e = _exponent(top)
    up = _spread(e, m, k)
    return _e4m3(w / up) * up, e


def _plain_fp8(s):
    case, x = s["case"], s["x"]
    dt = x.dtype
    xf = x.float()
    if case["op"] == "fp8":
        k, m = case["k"], case["m"]
        e = (s["scales"].to(torch.int32) - 127)[:, :-(-k // 128)]
        w = s["codes"].float()[:, :k] * _spread(e, m, k)
    else:
        w = _tiles(s["w"].float())[0]
    z = _rows8(xf) @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, case["act"])
    if case["op"] == "fp8":
        if s["res"] is not None:
            y = y + s["res"].float()
        return y.to(dt)
    kept = z.to(dt).float()  # as the layer keeps it for its backward pass
    dz = s["dy"].float() * _act_slope(kept, case["act"])
    dx = _rows8(dz) @ w
    dw = _rows8(dz.t().contiguous()) @ _rows8(xf.t().contiguous()).t()
    return [y.to(dt), dx.to(dt), dw.to(dt), dz.sum(0).to(dt)]


def _own(s):
    from mlrs_amd import prims
    case, x = s["case"], s["x"]
    if case["op"] == "dropout":
        return prims.dropout(x, case["p"], s["seed"], offset=OFFSET, residual=s["res"])
    if case["op"] == "norm":
        return prims.group_norm(x, case["groups"], weight=s["w"], bias=s["b"], eps=EPS, activation=case["act"])
    if case["op"] == "norm_train":
        drop = dict(p=case["p"], seed=s["seed"], offset=OFFSET)
        y, mean, rstd = prims.group_norm(x, case["groups"], weight=s["w"], bias=s["b"], eps=EPS,
                                         activation=case["act"], keep_stats=True, **drop)
        dx, dw, db = prims.group_norm_grad(s["dy"], x, mean, rstd, weight=s["w"], bias=s["b"],
                                           activation=case["act"], **drop)
        return [y, mean, rstd, dx, dw, db]
    if case["op"] == "fp8":
        w8 = prims.Fp8Weight(s["codes"], s["scales"], None, None, case["k"])
        return prims.linear_fp8(x, w8, bias=s["b"], activation=case["act"], residual=s["res"])
    w8 = prims.fp8_weight(s["w"], backward=True)
    y, z = prims.linear_fp8(x, w8, bias=s["b"], activation=case["act"], keep_preact=True)
    return [y] + list(prims.linear_fp8_grad(s["dy"], x, w8, preact=z, activation=case["act"]))


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_dropout(state) if op == "dropout" else (_plain_norm if op.startswith("norm") else _plain_fp8)(state)


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "dropout":
        count = case["n"] * case["d"]
        return {"bytes": e * count * (2 + case["residual"]), "flops": 2.0 * count}
    if case["op"] in ("norm", "norm_train"):
        n, c = case["n"], case["c"]
        count = n * case["s"] * c
        if case["op"] == "norm":
            return {"bytes": e * (2 * count + 2 * c), "flops": 10.0 * count}
        return {"bytes": e * (4 * count + 4 * c) + 8 * n * case["groups"], "flops": 30.0 * count}
    n, k, m = case["n"], case["k"], case["m"]
    if case["op"] == "fp8":
        b = e * (n * k + n * m * (1 + case["residual"]) + m * case["bias"]) + m * k
        return {"bytes": b, "flops": 2.0 * n * m * k}
    # x, w, dy, the bias; y, dx, dw, dbias
    return {"bytes": e * (2 * n * k + 2 * m * k + 2 * n * m + 2 * m), "flops": 6.0 * n * m * k}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].to(torch.float64)
    if case["op"] == "dropout":
        y = x * _exact_factor(tuple(x.shape), case["p"], s["seed"])
        return y if s["res"] is None else y + s["res"].to(torch.float64)
    if case["op"] in ("norm", "norm_train"):
        n, p, c = x.shape
        g = case["groups"]
        train = case["op"] == "norm_train"
        x, w, b = (t.to(torch.float64).requires_grad_(train) for t in (x, s["w"], s["b"]))
        rows = x.view(n, p, g, c // g).transpose(1, 2).reshape(n, g, -1)
        mean = rows.mean(2)
        rstd = (rows.var(2, unbiased=False) + EPS).rsqrt()
        rows = (rows - mean[:, :, None]) * rstd[:, :, None]
        z = rows.view(n, g, p, c // g).transpose(1, 2).reshape(n, p, c) * w + b
        y = _exact_act(z, case["act"])
        if not train:
            return y
        if case["p"]:
            y = y * _exact_factor(tuple(x.shape), case["p"], s["seed"])
        dx, dw, db = torch.autograd.grad(y, [x, w, b], s["dy"].to(torch.float64))
        return [y.detach(), mean.detach(), rstd.detach(), dx, dw, db]
    k, m = case["k"], case["m"]
    if case["op"] == "fp8":
        tile = _exact_power(s["scales"].to(torch.int64) - 127)
        w = s["codes"].to(torch.float64)
        for i in range(tile.shape[0]):
            for j in range(w.shape[1] // 128):
                w[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= tile[i, j]
        w = w[:, :k].contiguous()
    else:
        w = _exact_blocks(s["w"].to(torch.float64), 128)
    z = torch.mm(_exact_blocks(x, 1), w.t().contiguous())
    if s["b"] is not None:
        z += s["b"].to(torch.float64)
    if case["op"] == "fp8":
        y = _exact_act(z, case["act"])
        return y if s["res"] is None else y + s["res"].to(torch.float64)
    y = _exact_act(z, case["act"])
    kept = z.to(s["x"].dtype).to(torch.float64).requires_grad_(True)
    dz, = torch.autograd.grad(_exact_act(kept, case["act"]), kept, s["dy"].to(torch.float64))
    dx = torch.mm(_exact_blocks(dz, 1), w)
    dw = torch.mm(_exact_blocks(dz.t().contiguous(), 1), _exact_blocks(x.t().contiguous(), 1).t().contiguous())
    return [y, dx, dw, dz.sum(dim=0)]


def _exact_act(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":  # (1 + tanh u) / 2 is the logistic function of 2u
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z * 1.0


def _exact_factor(shape, p, seed):
    """The generator on the host, in unsigned 64-bit integers."""
    count = int(np.prod(shape))
    t = _threshold(p)
    i = np.arange((count + 7) // 8, dtype=np.uint64)
    word, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    state = [i & word, i >> half, np.full_like(i, OFFSET), np.zeros_like(i)]
    keys = [seed & 0xFFFFFFFF, seed >> 32]
    for r in range(7):
        first, second = state[0] * np.uint64(0xD2511F53), state[2] * np.uint64(0xCD9E8D57)
        ka, kb = ((k + r * step) & 0xFFFFFFFF for k, step in zip(keys, (0x9E3779B9, 0xBB67AE85)))
        state = [(second >> half) ^ state[1] ^ np.uint64(ka), second & word,
                 (first >> half) ^ state[3] ^ np.uint64(kb), first & word]
    bits = np.stack([w.astype(np.uint32) for w in state], 1).view(np.uint16).reshape(-1)[:count]
    kept = torch.from_numpy((bits >= t).reshape(shape)).to("cuda")
    return kept.to(torch.float64) / (1.0 - t / 65536.0)


def _exact_power(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_blocks(v, rows):
    """What 8 bits keep of v in blocks of `rows` x 128."""
    n, k = v.shape
    room = torch.nn.functional.pad(v, (0, (128 - k % 128) % 128, 0, (rows - n % rows) % rows))
    room = room.view(room.shape[0] // rows, rows, room.shape[1] // 128, 128)
    top = room.abs().amax(dim=(1, 3), keepdim=True)
    # top / 448 = f * 2^e with f in [1/2, 1): the least power of two not below it
    f, e = torch.frexp(top / 448.0)
    scale = _exact_power(torch.where(f == 0.5, e - 1, e).clamp(-127, 127))
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    q = room / scale
    _, e = torch.frexp(q)
    step = _exact_power((e - 1).clamp(min=-6) - 3)
    q = torch.round(q / step) * step * scale
    return q.view(q.shape[0] * rows, q.shape[2] * 128)[:n, :k].contiguous()
