"""The measured cases of the operators for dense layers and their training step (popvae_amd.ops).

Four operators: a dense layer with bias, activation and residual in one pass (``dense``), its gradients (``dense_bwd``),
clipping by the global norm over all tensors of a model (``clip``), and the Adam update with that clipping folded in (``adam``).

Shapes come from this repository's configurations (hidden layers of width 128 and 512, 32-row batches, 2504 samples, models
of 3887, 100 000 and 1 000 000 SNPs at depth 6) and, for 16-bit types, from generic square and ragged blocks.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTIVATIONS = ("linear", "relu", "elu", "sigmoid", "tanh", "silu", "gelu")


def _dense(name, op, m, k, n, dtype, act, residual, pre=False, w_t=False, bias=True):
    c = {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "w_t": w_t, "bias": bias}
    if op == "dense":
        c.update(residual=residual, pre=pre)
    if name:
        c["name"] = name
    return c


def _model(name, op, snps, width, depth, latent, dtype, clip):
    c = {"op": op, "snps": snps, "width": width, "depth": depth, "latent": latent, "dtype": dtype, "clip": clip}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one hidden layer of the default network on one batch, in training (z is kept for the backward): latency
        _dense("hidden 32x128", "dense", 32, 128, 128, "f32", "elu", True, pre=True),
        # the output layer answering for one latent point: the weights are read once
        _dense("one point to 100k", "dense", 1, 128, 100_000, "f32", "sigmoid", False),
        # the output layer answering for a whole sample set: bound by the products and by what is written
        _dense("2504 points to 100k", "dense", 2504, 128, 100_000, "f32", "sigmoid", False),
        # a ragged block in half precision: no size divides a tile, rows are not aligned
        _dense("ragged block f16", "dense", 1543, 1021, 2027, "f16", "gelu", True),
        # a large block in training: bound by the matrix pipe
        _dense("block 4096 bf16", "dense", 4096, 4096, 4096, "bf16", "silu", True, pre=True),
        # the gradients of the first case
        _dense("hidden 32x128 backward", "dense_bwd", 32, 128, 128, "f32", "elu", True),
        # a hidden layer of the widest network, all 2504 samples in one batch
        _dense("hidden 2504x512 backward", "dense_bwd", 2504, 512, 512, "f32", "elu", True),
        # a large block's gradients
        _dense("block 4096 bf16 backward", "dense_bwd", 4096, 2048, 4096, "bf16", "gelu", True),
        # the gradients of the smallest model's 30 tensors: latency over many tensors
        _model("clip 3887 SNPs", "clip", 3887, 128, 6, 2, "f32", 0.5),
        # 100 000 SNPs with 16-bit gradients
        _model("clip 100k SNPs bf16", "clip", 100_000, 128, 6, 2, "bf16", 0.5),
        # one update of the smallest model
        _model("adam 3887 SNPs", "adam", 3887, 128, 6, 2, "f32", 0.5),
        # one update of the 1 000 000 SNP model: 257 million parameters, bound by memory
        _model("adam 1M SNPs", "adam", 1_000_000, 128, 6, 2, "f32", 0.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("dense", "dense", "dense_bwd", "dense_bwd", "clip", "adam"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op in ("dense", "dense_bwd"):
        while True:
            m, k, n = _log(rng, 1, 4096), _log(rng, 1, 4096), _log(rng, 1, 20_000)
            if m * k * n <= 1 << 35:
                break
        return _dense(None, op, m, k, n, dtype, rng.choice(ACTIVATIONS), rng.random() < 0.5, pre=rng.random() < 0.5,
                      w_t=rng.random() < 0.3, bias=rng.random() < 0.8)
    return _model(None, op, _log(rng, 31, 200_000), rng.choice((32, 100, 128, 256, 512)), rng.choice((1, 3, 6, 10)),
                  rng.choice((2, 3, 8)), dtype, rng.choice((0.25, 0.5, 2.0)))


def _shapes(c):
    """The tensors of a model, in the order of its weights."""
    s, w, d, k = c["snps"], c["width"], c["depth"], c["latent"]
    out = [(s, w), (w,)] + [(w, w), (w,)] * (d - 1) + [(w, k), (k,)] * 2 + [(k, w), (w,)] + [(w, w), (w,)] * (d - 1)
    return out + [(w, s), (s,)]


def _dense_inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, m, k, n = DTYPES[c["dtype"]], c["m"], c["k"], c["n"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    limit = math.sqrt(6.0 / (k + n))  # glorot_uniform, widened so that z spans the activation's bend for every ratio k / n
    limit *= max(1.0, math.sqrt(3.0 / k) / limit)
    w = (torch.rand((n, k) if c["w_t"] else (k, n), generator=gen, device="cuda") * 2 - 1) * limit
    i = {"x": normal(m, k).to(t), "w": w.to(t), "bias": (normal(n) * 0.1).to(t) if c["bias"] else None}
    if c["w_t"]:
        i["w"] = i["w"].t()
    if c["op"] == "dense":
        i["residual"] = normal(m, n).to(t) if c["residual"] else None
    else:
        i["dy"] = normal(m, n).to(t)
        z = i["x"].double() @ i["w"].double().contiguous()  # what the forward left behind
        i["pre"] = (z if i["bias"] is None else z + i["bias"].double()).float()
    return i


def _slots(shapes):
    """Where each tensor begins in one flat buffer (256-byte steps), and the buffer's length."""
    at, n = [], 0
    for shape in shapes:
        at.append(n)
        n += (math.prod(shape) + 63) // 64 * 64
    return at, n


def _flat(tensors, dtype):
    """The tensors in one flat buffer, as a training program keeps its moments: (buffer, views)."""
    at, n = _slots([t.shape for t in tensors])
    buf = torch.zeros(n, dtype=dtype, device="cuda")
    views = [buf[a:a + t.numel()].view(t.shape) for a, t in zip(at, tensors)]
    for v, t in zip(views, tensors):
        v.copy_(t)
    return buf, views


def _model_inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(c)
    rms = 1.0 / math.sqrt(sum(math.prod(s) for s in shapes))

    def each():
        return [torch.randn(s, generator=gen, device="cuda") for s in shapes]

    # gradients whose global norm is near 1, tensors differing in scale as layers do
    i = {"grads": [(g * ((0.5 + (j % 3) * 0.5) * rms)).to(DTYPES[c["dtype"]]) for j, g in enumerate(each())]}
    if c["op"] == "adam":
        i["params"] = [p * 0.05 for p in each()]
        i["m"] = [p * (0.3 * rms) for p in each()]
        i["v"] = [p.square() * (0.3 * rms * rms) for p in each()]
    return i


def prepare(case, seed):
    if case["op"] in ("dense", "dense_bwd"):
        return {"case": case, **_dense_inputs(case, seed)}
    s = {"case": case, **_model_inputs(case, seed), "step": 10}
    if case["op"] == "clip":
        s["out"] = [torch.empty_like(g) for g in s["grads"]]
    else:
        s["m_all"], s["m"] = _flat(s["m"], torch.float32)
        s["v_all"], s["v"] = _flat(s["v"], torch.float32)
    if own:  # the handles on its tensors that a training program makes once
        from popvae_amd import ops
        s["sets"] = {k: ops.TensorSet(s[k]) for k in ("grads", "out", "params", "m", "v") if k in s}
    return s


def _act(z, name):
    if name == "linear":
        return z
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "elu":
        return torch.where(z > 0, z, torch.expm1(z))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if name == "tanh":
        return torch.tanh(z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _act_grad(z, name):
    if name == "linear":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "elu":
        return torch.where(z > 0, torch.ones_like(z), torch.exp(z))
    if name == "tanh":
        return 1 - torch.tanh(z).square()
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 - s) if name == "sigmoid" else s * (1 + z * (1 - s))


def _plain_scale(grads, clip):
    """min(1, clip / norm); the sum of squares in 64 bits."""
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    return norm.float(), torch.clamp(clip / norm, max=1.0).float()


def run(state):
    c = state["case"]
    if own:
        from popvae_amd import ops
        if c["op"] == "dense":
            pre = torch.empty((c["m"], c["n"]), dtype=torch.float32, device="cuda") if c["pre"] else None
            y = ops.dense(state["x"], state["w"], state["bias"], c["act"], residual=state["residual"], pre=pre)
            return {"y": y, "pre": pre}
        if c["op"] == "dense_bwd":
            dx, dw, db = ops.dense_backward(state["dy"], state["x"], state["w"], state["pre"], c["act"], need_bias=c["bias"])
            return {"dx": dx, "dw": dw, "db": db}
        s = state["sets"]
        if c["op"] == "clip":
            norm = ops.clip_by_global_norm(s["grads"], c["clip"], out=s["out"])
            return {"out": state["out"], "norm": norm}
        norm = ops.adam_step(s["params"], s["grads"], s["m"], s["v"], state["step"], clip_norm=c["clip"])
        return {"params": state["params"], "m": state["m_all"], "v": state["v_all"], "norm": norm}
    if c["op"] == "dense":
        z = state["x"].float() @ state["w"].float()
        if state["bias"] is not None:
            z = z + state["bias"].float()
        y = _act(z, c["act"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return {"y": y.to(state["x"].dtype), "pre": z if c["pre"] else None}
    if c["op"] == "dense_bwd":
        t = state["x"].dtype
        g = state["dy"].float() * _act_grad(state["pre"], c["act"])
        dx = g @ state["w"].float().t()
        dw = state["x"].float().t() @ g
        return {"dx": dx.to(t), "dw": dw.to(t), "db": g.sum(0).to(t) if c["bias"] else None}
    norm, scale = _plain_scale(state["grads"], c["clip"])
    if c["op"] == "clip":
        for o, g in zip(state["out"], state["grads"]):
            o.copy_((g.float() * scale).to(g.dtype))
        return {"out": state["out"], "norm": norm}
    t, lr, b1, b2, eps = state["step"], 1e-3, 0.9, 0.999, 1e-7
    alpha = lr * math.sqrt(1 - b2 ** t) / (1 - b1 ** t)
    for p, g, m, v in zip(state["params"], state["grads"], state["m"], state["v"]):
        g = g.float() * scale
        m.add_((g - m) * (1 - b1))
        v.add_((g * g - v) * (1 - b2))
        p.sub_(alpha * m / (torch.sqrt(v) + eps))
    return {"params": state["params"], "m": state["m_all"], "v": state["v_all"], "norm": norm}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("dense", "dense_bwd"):
        m, k, n = case["m"], case["k"], case["n"]
        b = n if case["bias"] else 0
        if case["op"] == "dense":
            moved = (m * k + k * n + b + m * n * (2 if case["residual"] else 1)) * size + (4 * m * n if case["pre"] else 0)
            return {"bytes": moved, "flops": 2 * m * n * k}
        return {"bytes": (m * n + 2 * m * k + 2 * k * n + b) * size + 4 * m * n, "flops": 4 * m * n * k}
    total = sum(math.prod(s) for s in _shapes(case))
    if case["op"] == "clip":
        return {"bytes": 2 * total * size, "flops": 3 * total}
    return {"bytes": total * (24 + size), "flops": 16 * total}


def exact(case, seed):
    """The same in 64 bits, from the definitions."""
    c = case
    if c["op"] in ("dense", "dense_bwd"):
        i = {k: v if v is None else v.to(torch.float64).contiguous() for k, v in _dense_inputs(c, seed).items()}

        def sig(a):
            return torch.sigmoid(a)

        def phi(a):
            return torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)

        def big_phi(a):
            return torch.erfc(-a / math.sqrt(2.0)) / 2

        f = {"linear": lambda a: a, "relu": lambda a: a.clamp(min=0), "elu": lambda a: a.clamp(min=0) + torch.expm1(a.clamp(max=0)),
             "sigmoid": sig, "tanh": torch.tanh, "silu": lambda a: a * sig(a), "gelu": lambda a: a * big_phi(a)}[c["act"]]
        df = {"linear": lambda a: torch.ones_like(a), "relu": lambda a: torch.heaviside(a, torch.zeros_like(a)),
              "elu": lambda a: torch.exp(a.clamp(max=0)), "sigmoid": lambda a: sig(a) * sig(-a),
              "tanh": lambda a: 1 / torch.cosh(a).square(), "silu": lambda a: sig(a) + a * sig(a) * sig(-a),
              "gelu": lambda a: big_phi(a) + a * phi(a)}[c["act"]]
        if c["op"] == "dense":
            z = torch.mm(i["x"], i["w"])
            if i["bias"] is not None:
                z += i["bias"]
            y = f(z)
            if i["residual"] is not None:
                y += i["residual"]
            return {"y": y, "pre": z if c["pre"] else None}
        g = i["dy"] * df(i["pre"])
        return {"dx": torch.mm(g, i["w"].t().contiguous()), "dw": torch.mm(i["x"].t().contiguous(), g),
                "db": g.sum(dim=0) if c["bias"] else None}
    i = _model_inputs(c, seed)
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.reshape(-1), dtype=torch.float64)) ** 2 for g in i["grads"]))
    scale = 1.0 if norm <= c["clip"] else c["clip"] / norm
    if c["op"] == "clip":
        return {"out": [g.double() * scale for g in i["grads"]], "norm": norm}
    params, ms, vs = [], [], []
    b1, b2, t = 0.9, 0.999, 10
    for p, g, m, v in zip(i["params"], i["grads"], i["m"], i["v"]):
        g = g.double() * scale
        m = b1 * m.double() + (1 - b1) * g
        v = b2 * v.double() + (1 - b2) * g ** 2
        params.append(p.double() - 1e-3 * (math.sqrt(1 - b2 ** t) / (1 - b1 ** t)) * m / (v.sqrt() + 1e-7))
        ms.append(m)
        vs.append(v)
    return {"params": params, "m": _flat(ms, torch.float64)[0], "v": _flat(vs, torch.float64)[0], "norm": norm}
