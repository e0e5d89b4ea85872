"""The calls that the embedding-training operators are measured on.

``op`` names the call and the rest its sizes, types and options:

linear    prims.linear: a layer with bias, activation and residual
grad      prims.linear_grad: its backward pass from the kept pre-activations
eval      prims.softmax_xent: the loss of every row, nothing else
train     prims.softmax_xent, then prims.softmax_xent_grad
adamw     prims.adamw_step over a model's tensors (``clip``: prims.clip_scale
          before it), states in 32 or in 8 bits

With ``own`` false the same is computed from elementary torch operations in
float32, rounded once at the end.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
IGNORE = -100
LR, BETAS, EPS, DECAY, STEP, SEED = 3e-4, (0.9, 0.999), 1e-8, 0.1, 10, 20240
BLOCK = 256  # elements that share a scale of an 8-bit state
PAD = 256  # a tensor's start in the flat buffers is a multiple of this


def listed():
    return [
        # One row through a wide layer, as an online encoder answers a single
        # request: the weights are read once and nothing else matters.
        dict(name="linear_one_row", op="linear", dtype="bf16", n=1, k=1024, m=4096, act="silu", bias=True,
             residual=False, keep=False),
        # The benchmark's small query batch through a single-precision layer
        # whose sizes are no multiples of a vector or a tile.
        dict(name="linear_ragged_f32", op="linear", dtype="f32", n=1001, k=257, m=1030, act="relu", bias=True,
             residual=True, keep=True),
        # A training batch through a square layer with everything that its
        # epilogue can do.
        dict(name="linear_batch", op="linear", dtype="bf16", n=16384, k=4096, m=4096, act="gelu", bias=True,
             residual=True, keep=True),
        # Backward of a half-precision layer, odd counts everywhere.
        dict(name="grad_ragged_f16", op="grad", dtype="f16", n=4099, k=1000, m=2050, act="silu", bias=True),
        # Backward of a wide layer at a training batch.
        dict(name="grad_batch", op="grad", dtype="bf16", n=8192, k=2048, m=8192, act="gelu_tanh", bias=True),
        # A classification head of the benchmark's row width, in single
        # precision, on a small batch.
        dict(name="train_small_f32", op="train", dtype="f32", n=64, v=1000, k=128, bias=True),
        # Loss of a validation batch over a mid vocabulary.
        dict(name="eval_mid", op="eval", dtype="bf16", n=2048, v=32000, k=1024, bias=False),
        # A single-precision training step against the benchmark's thousand
        # centres' worth of classes many times over, ragged.
        dict(name="train_ragged_f32", op="train", dtype="f32", n=3001, v=10007, k=250, bias=True),
        # A training step over a large vocabulary: the largest call.
        dict(name="train_large", op="train", dtype="bf16", n=8192, v=128000, k=2048, bias=False),
        # The optimizer step of a two-layer head: launches are all there is.
        dict(name="adamw_small", op="adamw", dtype="f32", bits=32, layers=2, width=64, vocab=100, clip=True),
        # A half-precision model with single-precision master weights, the
        # gradients clipped to a norm first.
        dict(name="adamw_master", op="adamw", dtype="bf16", bits=32, layers=12, width=1024, vocab=50021, clip=True),
        # A single-precision model whose two moments are kept in 8 bits.
        dict(name="adamw_8bit", op="adamw", dtype="f32", bits=8, layers=12, width=1000, vocab=20011, clip=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo + 1, hi))))))


def draw(rng):
    """One more call of the ranges the listed ones stand for."""
    op = rng.choice(["linear", "linear", "grad", "eval", "train", "train", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    most = 6e11 if dtype == "f32" else 3e12  # of multiply-adds
    if op in ("linear", "grad"):
        k, m = _log(rng, 16, 8192), _log(rng, 16, 8192)
        if rng.random() < 0.5:
            k, m = (-(-t // 64) * 64 for t in (k, m))
        k, m = (t + 64 if t == 3072 else t for t in (k, m))
        n = _log(rng, 1 if op == "linear" else 64, min(65536, most / 3 / (k * m)))
        c = dict(op=op, dtype=dtype, n=n, k=k, m=m, act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                 bias=rng.random() < 0.7)
        if op == "linear":
            c.update(residual=rng.random() < 0.5, keep=rng.random() < 0.5)
        return c
    if op in ("eval", "train"):
        k = _log(rng, 32, 4096)
        if rng.random() < 0.5:
            k = -(-k // 64) * 64
        k += 64 if k == 3072 else 0
        v = _log(rng, 100, 128000)
        n = _log(rng, 16, min(16384, most / 4 / (k * v), 1e9 / v))
        return dict(op=op, dtype=dtype, n=n, v=v, k=k, bias=rng.random() < 0.5)
    bits = rng.choice([32, 8])
    width = _log(rng, 24, 1500)
    width += 1 if width == 768 else 0
    layers = _log(rng, 1, min(24, max(2, 1.5e8 / (12 * width * width))))
    return dict(op=op, dtype=dtype, bits=bits, layers=layers, width=width, vocab=_log(rng, 10, 30000),
                clip=bits == 32 and rng.random() < 0.6)


def _sizes(case):
    """Element counts of the model's tensors, and which of them decay."""
    w = case["width"]
    sizes, decays = [case["vocab"] * w], [True]
    for _ in range(case["layers"]):
        sizes += [w * w] * 4 + [4 * w * w] * 2 + [w, w, 4 * w, 1]
        decays += [True] * 6 + [False] * 4
    return sizes, decays


def _offsets(sizes):
    at, offs = 0, []
    for s in sizes:
        offs.append(at)
        at += -(-s // PAD) * PAD
    return offs, at


def _normal(g, *shape, dtype=torch.float32, std=1.0):
    t = torch.empty(shape, dtype=torch.float32, device="cuda")
    t.normal_(0.0, std, generator=g)
    return t.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    dt = _DT[case["dtype"]]
    s = dict(case=case)
    if case["op"] in ("linear", "grad"):
        n, k, m = case["n"], case["k"], case["m"]
        s["x"] = _normal(g, n, k, dtype=dt)
        s["w"] = _normal(g, m, k, dtype=dt, std=k ** -0.5)
        if case["op"] == "linear":
            s["b"] = _normal(g, m, dtype=dt, std=0.1) if case["bias"] else None
            s["res"] = _normal(g, n, m, dtype=dt) if case["residual"] else None
        else:
            s["dy"] = _normal(g, n, m, dtype=dt, std=0.02)
            s["z"] = _normal(g, n, m, dtype=dt) if case["act"] != "none" else None
        return s
    if case["op"] in ("eval", "train"):
        n, v, k = case["n"], case["v"], case["k"]
        s["h"] = _normal(g, n, k, dtype=dt)
        s["w"] = _normal(g, v, k, dtype=dt, std=1.5 * k ** -0.5)
        s["b"] = _normal(g, v, dtype=dt, std=0.5) if case["bias"] else None
        t = torch.randint(0, v, (n,), generator=g, device="cuda")
        t[torch.rand(n, generator=g, device="cuda") < 0.05] = IGNORE  # padding between documents
        s["t"] = t
        # the mean over the batch; half precision comes with a loss scale
        s["g"] = torch.full((n,), (1024.0 if case["dtype"] == "f16" else 1.0) / n, device="cuda")
        return s
    sizes, decays = _sizes(case)
    offs, total = _offsets(sizes)
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for o, z in zip(offs, sizes):
        live[o:o + z] = True

    def flat(t):
        return torch.where(live, t, torch.zeros((), dtype=t.dtype, device="cuda"))

    master = flat(_normal(g, total, std=0.02))
    s["p"] = master.to(dt)
    s["master"] = master if dt != torch.float32 else None
    s["grad"] = flat(_normal(g, total, std=0.01)).to(dt)
    if case["bits"] == 32:
        s["m"] = flat(_normal(g, total, std=0.003))
        s["v"] = flat(_normal(g, total, std=0.01).square_())
    else:
        s["m"] = flat(torch.randint(0, 256, (total,), generator=g, device="cuda", dtype=torch.uint8))
        s["v"] = flat(torch.randint(100, 256, (total,), generator=g, device="cuda", dtype=torch.uint8))
        s["ms"] = 0.002 + 0.002 * torch.rand(total // BLOCK, generator=g, device="cuda")
        s["vs"] = 0.01 + 0.01 * torch.rand(total // BLOCK, generator=g, device="cuda")
        s["scale"] = torch.full((1,), 0.75, device="cuda")

    def views(t, div=1):
        return None if t is None else [t[o // div:o // div + -(-z // div)] for o, z in zip(offs, sizes)]

    s["lists"] = dict(params=views(s["p"]), grads=views(s["grad"]), exp_avg=views(s["m"]), exp_avg_sq=views(s["v"]),
                      masters=views(s["master"]))
    if case["bits"] == 8:
        s["lists"].update(avg_scales=views(s["ms"], BLOCK), avg_sq_scales=views(s["vs"], BLOCK))
    s["decays"] = [DECAY if d else 0.0 for d in decays]
    s["plan"] = dict(offs=offs, total=total)
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
    sg = 1.0 / (1.0 + torch.exp(-z))
    return sg * (1.0 + z * (1.0 - sg))


def _plain_linear(s):
    dt = s["x"].dtype
    z = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["case"]["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    return (y.to(dt), z.to(dt)) if s["case"]["keep"] else y.to(dt)


def _plain_grad(s):
    dt = s["x"].dtype
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_slope(s["z"].float(), s["case"]["act"])
    out = [(dz @ s["w"].float()).to(dt), (dz.t() @ s["x"].float()).to(dt)]
    if s["case"]["bias"]:
        out.append(dz.sum(0).to(dt))
    return out


def _plain_xent(s):
    h, w, t = s["h"].float(), s["w"].float(), s["t"]
    dt = s["h"].dtype
    z = h @ w.t()
    if s["b"] is not None:
        z += s["b"].float()
    top = z.amax(1)
    p = torch.exp(z - top[:, None])
    total = p.sum(1)
    lse = top + torch.log(total)
    kept = t != IGNORE
    at = torch.where(kept, t, 0)[:, None]
    loss = torch.where(kept, lse - z.gather(1, at)[:, 0], 0.0)
    if s["case"]["op"] == "eval":
        return loss, lse
    del z
    p /= total[:, None]
    p.scatter_add_(1, at, torch.full_like(lse, -1.0)[:, None])
    p *= torch.where(kept, s["g"], 0.0)[:, None]
    out = [loss, lse, (p @ w).to(dt), (p.t() @ h).to(dt)]
    if s["b"] is not None:
        out.append(p.sum(0).to(dt))
    return out


def _mix(x):
    """A 32-bit integer hash, on int64 tensors that hold 32-bit values."""
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _pack(y, r16, mant):
    """Codes of magnitudes y with a 4-bit exponent (15 is 2^0) and `mant` bits,
    rounded up where the fraction left over is above 1 - r16 / 65536."""
    bits = y.view(torch.int32).to(torch.int64)
    big = ((bits + (r16 << (7 - mant))) >> (23 - mant)) - (112 << mant)
    small = torch.floor(y * 2.0 ** (14 + mant) + r16.to(torch.float32) * 2.0 ** -16).to(torch.int64)
    return torch.where(y < 2.0 ** -14, small, big).clamp_(max=(16 << mant) - 1)


def _unpack(code, mant):
    e, f = code >> mant, code & ((1 << mant) - 1)
    return torch.where(e > 0, ((code + (112 << mant)) << (23 - mant)).view(torch.float32), f * 2.0 ** (-14 - mant))


def _avg_values(code, scale):
    c = code.to(torch.int32)
    v = _unpack(c & 127, 3)
    return torch.where(c > 127, -v, v) * scale.repeat_interleave(BLOCK)


def _root_values(code, scale):
    return _unpack(code.to(torch.int32), 4) * scale.repeat_interleave(BLOCK)


def _plain_adamw(s):
    case, plan = s["case"], s["plan"]
    dev = s["p"].device
    b1, b2 = BETAS
    step, rc2 = LR / (1.0 - b1 ** STEP), 1.0 / math.sqrt(1.0 - b2 ** STEP)
    starts = torch.tensor(plan["offs"] + [plan["total"]], device=dev)
    spans = starts[1:] - starts[:-1]
    decay = (1.0 - LR * torch.tensor(s["decays"], dtype=torch.float64)).float().to(dev).repeat_interleave(spans)
    g = s["grad"].float()
    norm = None
    if case["clip"]:
        norm = torch.sqrt((g * g).sum())
        scale = torch.where(norm > 1.0, 1.0 / norm, 1.0)
        g = g * scale
    if case["bits"] == 8:
        g = g * s["scale"]
        m, r = _avg_values(s["m"], s["ms"]), _root_values(s["v"], s["vs"])
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * (1.0 - b2)) * g
    r = torch.sqrt(v)
    p = s["master"] if s["master"] is not None else s["p"]
    new = p * decay - (m / (r * rc2 + EPS)) * step
    if s["master"] is not None:
        s["master"].copy_(new)
    s["p"].copy_(new)
    out = dict(p=s["p"])
    if s["master"] is not None:
        out["master"] = s["master"]
    if norm is not None:
        out["norm"] = norm.reshape(1)
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        out.update(m=s["m"], v=s["v"])
        return out
    del g, v, new, decay
    ordinal = torch.arange(len(spans), device=dev)
    key = _mix((SEED + ordinal * 0x9E3779B1) & 0xFFFFFFFF).repeat_interleave(spans)
    index = torch.arange(plan["total"], device=dev) - starts[:-1].repeat_interleave(spans)
    u = _mix(index ^ key)
    del key, index
    s["ms"].copy_(m.abs().view(-1, BLOCK).amax(1) / torch.full((), 1.875, device=dev))
    s["vs"].copy_(r.view(-1, BLOCK).amax(1) / torch.full((), 1.9375, device=dev))
    ms, vs = s["ms"].repeat_interleave(BLOCK), s["vs"].repeat_interleave(BLOCK)
    code = _pack(torch.where(ms > 0, m.abs() / ms, 0.0), u & 0xFFFF, 3)
    s["m"].copy_(torch.where(m < 0, code + 128, code))
    code = _pack(torch.where(vs > 0, r / vs, 0.0), u >> 16, 4)
    s["v"].copy_(torch.where((r > 0) & (code == 0), 1, code))
    out.update(ms=s["ms"], vs=s["vs"], m=_avg_values(s["m"], s["ms"]), v=_root_values(s["v"], s["vs"]))
    return out


def _own(s):
    from mlrs_amd import prims
    case = s["case"]
    op = case["op"]
    if op == "linear":
        return prims.linear(s["x"], s["w"], bias=s["b"], activation=case["act"], residual=s["res"],
                            keep_preact=case["keep"])
    if op == "grad":
        dx, dw, db = prims.linear_grad(s["dy"], s["x"], s["w"], preact=s["z"], activation=case["act"],
                                       bias=case["bias"])
        return [dx, dw, db] if case["bias"] else [dx, dw]
    if op in ("eval", "train"):
        loss, lse = prims.softmax_xent(s["h"], s["w"], s["t"], bias=s["b"], ignore_index=IGNORE)
        if op == "eval":
            return loss, lse
        dh, dw, db = prims.softmax_xent_grad(s["h"], s["w"], s["t"], lse, s["g"], bias=s["b"], ignore_index=IGNORE)
        return [loss, lse, dh, dw] + ([db] if s["b"] is not None else [])
    norm, scale = None, s.get("scale")
    if case["clip"]:
        norm, scale = prims.clip_scale(s["lists"]["grads"], 1.0)
    prims.adamw_step(step=STEP, lr=LR, betas=BETAS, eps=EPS, weight_decay=s["decays"], scale=scale, seed=SEED,
                     **s["lists"])
    out = dict(p=s["p"])
    if s["master"] is not None:
        out["master"] = s["master"]
    if norm is not None:
        out["norm"] = norm
    if case["bits"] == 32:
        out.update(m=s["m"], v=s["v"])
    else:
        out.update(ms=s["ms"], vs=s["vs"], m=prims.adamw_state_values(s["m"], s["ms"], "exp_avg"),
                   v=prims.adamw_state_values(s["v"], s["vs"], "exp_avg_sq"))
    return out


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "grad": _plain_grad, "eval": _plain_xent, "train": _plain_xent,
            "adamw": _plain_adamw}[state["case"]["op"]](state)


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "linear":
        n, k, m = case["n"], case["k"], case["m"]
        b = n * k + m * k + n * m + m * case["bias"] + n * m * (case["residual"] + case["keep"])
        return {"bytes": e * b, "flops": 2.0 * n * m * k}
    if case["op"] == "grad":
        n, k, m = case["n"], case["k"], case["m"]
        b = 2 * n * k + 2 * m * k + n * m * (1 + (case["act"] != "none")) + m * case["bias"]
        return {"bytes": e * b, "flops": 4.0 * n * m * k}
    if case["op"] in ("eval", "train"):
        n, v, k = case["n"], case["v"], case["k"]
        b = e * (n * k + v * k + v * case["bias"]) + 16 * n
        if case["op"] == "eval":
            return {"bytes": b, "flops": 2.0 * n * v * k}
        return {"bytes": b + e * (n * k + v * k + v * case["bias"]) + 4 * n, "flops": 6.0 * n * v * k}
    total = sum(_sizes(case)[0])
    per = e + (8 if e == 2 else 4) + e  # gradient in; the master or the parameter in, out; a half parameter out
    if case["bits"] == 32:
        return {"bytes": total * (per + 16), "flops": 16.0 * total}
    # both codes in and out, and their values out
    return {"bytes": total * (per + 4 + 8) + 16 * (total // BLOCK), "flops": 40.0 * total}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)

    def wide(name):
        return None if s[name] is None else s[name].to(torch.float64)

    if case["op"] == "linear":
        z = torch.mm(wide("x"), wide("w").t().contiguous())
        if s["b"] is not None:
            z += wide("b")[None, :]
        y = _exact_act(z, case["act"])[0]
        if s["res"] is not None:
            y = y + wide("res")
        return (y, z) if case["keep"] else y
    if case["op"] == "grad":
        dz = wide("dy")
        if s["z"] is not None:
            dz = dz * _exact_act(wide("z"), case["act"])[1]
        out = [torch.mm(dz, wide("w")), torch.mm(dz.t().contiguous(), wide("x"))]
        return out + ([dz.sum(dim=0)] if case["bias"] else [])
    if case["op"] in ("eval", "train"):
        n, v, k = case["n"], case["v"], case["k"]
        h, w, t = wide("h"), wide("w"), s["t"]
        loss = torch.zeros(n, dtype=torch.float64, device="cuda")
        lse = torch.zeros_like(loss)
        dh = torch.zeros_like(h)
        dw = torch.zeros_like(w)
        db = torch.zeros(v, dtype=torch.float64, device="cuda")
        rows = max(1, min(n, int(1e9 // v)))
        for a in range(0, n, rows):
            z = torch.mm(h[a:a + rows], w.t().contiguous())
            if s["b"] is not None:
                z = z + wide("b")
            lse[a:a + rows] = torch.logsumexp(z, dim=1)
            tt = t[a:a + rows]
            pick = (tt != IGNORE).nonzero()[:, 0]
            loss[a + pick] = lse[a + pick] - z[pick, tt[pick]]
            if case["op"] == "eval":
                continue
            d = torch.exp(z - lse[a:a + rows, None])
            d[pick, tt[pick]] -= 1.0
            gate = torch.zeros(len(tt), dtype=torch.float64, device="cuda")
            gate[pick] = s["g"][a + pick].to(torch.float64)
            d *= gate[:, None]
            dh[a:a + rows] = torch.mm(d, w)
            dw += torch.mm(d.t().contiguous(), h[a:a + rows])
            db += d.sum(dim=0)
        if case["op"] == "eval":
            return loss, lse
        return [loss, lse, dh, dw] + ([db] if s["b"] is not None else [])
    b1, b2 = BETAS
    lists = s["lists"]
    outs = dict(p=[], m=[], v=[], ms=[], vs=[])
    square = sum(float(t.to(torch.float64).square().sum()) for t in lists["grads"])
    factor = min(1.0, 1.0 / math.sqrt(square)) if case["clip"] else float(s["scale"]) if "scale" in s else 1.0
    for i, p in enumerate(lists["masters"] or lists["params"]):
        size = p.numel()
        g = lists["grads"][i].to(torch.float64) * factor
        if case["bits"] == 32:
            m, v = lists["exp_avg"][i].to(torch.float64), lists["exp_avg_sq"][i].to(torch.float64)
        else:
            code = lists["exp_avg"][i].to(torch.float64)
            m = _exact_code(code % 128, 8) * torch.where(code >= 128, -1.0, 1.0).to(torch.float64)
            m = m * lists["avg_scales"][i].to(torch.float64).repeat_interleave(BLOCK)[:size]
            v = _exact_code(lists["exp_avg_sq"][i].to(torch.float64), 16)
            v = (v * lists["avg_sq_scales"][i].to(torch.float64).repeat_interleave(BLOCK)[:size]) ** 2
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        q = p.to(torch.float64) * (1 - LR * s["decays"][i])
        q = q - LR * (m / (1 - b1 ** STEP)) / ((v / (1 - b2 ** STEP)).sqrt() + EPS)
        room = -(-size // PAD) * PAD - size
        for name, t in (("p", q), ("m", m), ("v", v)):
            outs[name].append(torch.nn.functional.pad(t, (0, room)))
        outs["ms"].append(outs["m"][-1].abs().view(-1, BLOCK).amax(1) / 1.875)
        outs["vs"].append(outs["v"][-1].sqrt().view(-1, BLOCK).amax(1) / 1.9375)
    out = dict(p=torch.cat(outs["p"]))
    if s["master"] is not None:
        out["master"] = out["p"]
    if case["clip"]:
        out["norm"] = torch.full((1,), math.sqrt(square), dtype=torch.float64)
    if case["bits"] == 32:
        out.update(m=torch.cat(outs["m"]), v=torch.cat(outs["v"]))
    else:  # which code a rounding takes is chance: the codes have no exact value
        out.update(ms=torch.cat(outs["ms"]), vs=torch.cat(outs["vs"]), m=None, v=None)
    return out


def _exact_act(z, act):
    """An activation and its slope."""
    one = torch.ones_like(z)
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":  # (1 + tanh u) / 2 is the logistic function of 2u
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        half = torch.sigmoid(2 * u)
        return z * half, half + z * 2 * half * (1 - half) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    if act == "silu":
        half = torch.sigmoid(z)
        return z * half, half + z * half * (1 - half)
    return z, one


def _exact_code(code, steps):
    """The value of a code: `steps` of them to a power of two, 15 the highest power, 2^0."""
    e = torch.floor(code / steps)
    f = (code - e * steps) / steps
    return torch.where(e > 0, (1 + f) * torch.exp2(e - 15), f * 2.0 ** -14)
