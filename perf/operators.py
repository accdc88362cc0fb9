"""The operators of a residual feed-forward block and of the loss it is trained on, as measurable cases.

  norm     root-mean-square norm with the residual's addition, alone or with its backward pass
  linear   matrix product with bias, activation and residual in its epilogue, alone or with its backward pass
  int8     the norm (or a plain row quantiser) writing Int8 rows with a scale each, and the Int8 product that reads them
  distill  divergence of a student's logits from a teacher's top logits: loss, loss of each row and gradient

`own` chooses between elementary torch operations (False) and this repository's operators (True).  `exact` states the
same results in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


def listed():
    return [
        # one token of a decoder between two layers: nothing but latency
        dict(name="norm, one token", op="norm", rows=1, n=4096, dtype="bf16", residual=True, train=False),
        # a prompt of 16384 tokens on its way through a layer
        dict(name="norm, prompt", op="norm", rows=16384, n=4096, dtype="bf16", residual=True, train=False),
        # a training step's activations, forward and backward, with the gradient that arrives over the residual
        dict(name="norm, training", op="norm", rows=8192, n=8192, dtype="bf16", residual=True, train=True),
        # an odd width in full precision, without a residual, as at the head of a small network
        dict(name="norm, odd width", op="norm", rows=1003, n=1999, dtype="f32", residual=False, train=True),
        # a few sequences that decode together: the weights are read once for 16 rows
        dict(name="linear, few rows", op="linear", m=16, k=8192, n=8192, dtype="bf16", act="silu", bias=True, residual=True,
             train=False),
        # a small ragged training batch whose rows are not whole 16-byte pieces
        dict(name="linear, ragged", op="linear", m=333, k=1001, n=1030, dtype="f16", act="gelu_tanh", bias=True, residual=True,
             train=True),
        # the first layer of the 4096 -> 16384 -> 4096 perceptron at its batch of 8192, forward and backward
        dict(name="linear, training", op="linear", m=8192, k=4096, n=16384, dtype="bf16", act="gelu", bias=True, residual=False,
             train=True),
        # full precision, a middle-sized batch
        dict(name="linear, full precision", op="linear", m=512, k=1024, n=4096, dtype="f32", act="silu", bias=True, residual=True,
             train=False),
        # eight tokens decoding through an 8-bit layer: norm and product
        dict(name="int8, few rows", op="int8", m=8, k=8192, n=8192, dtype="bf16", act="none", bias=False, residual=True,
             norm=True),
        # a prompt through the first 8-bit layer of a feed-forward block
        dict(name="int8, prompt", op="int8", m=8192, k=4096, n=16384, dtype="bf16", act="gelu_tanh", bias=True, residual=False,
             norm=True),
        # a short batch against a middle-sized vocabulary
        dict(name="distill, short", op="distill", rows=127, vocab=32001, top=8, dtype="f32", temperature=1.0),
        # a training step's logits over a large vocabulary
        dict(name="distill, large vocabulary", op="distill", rows=4096, vocab=131072, top=64, dtype="bf16", temperature=2.0),
    ]


def _between(rng, lo, hi):
    """A whole number, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Mostly multiples of 64, one in four of any size."""
    v = _between(rng, lo, hi)
    return v if rng.random() < 0.25 else max(64, v // 64 * 64)


def draw(rng):
    op = rng.choice(["norm", "linear", "int8", "distill"])
    if op == "norm":
        n = _width(rng, 64, 16384)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return dict(op=op, rows=_between(rng, 1, min(16384, (1 << (25 if dtype == "f32" else 26)) // n)), n=n, dtype=dtype,
                    residual=rng.random() < 0.7, train=rng.random() < 0.5)
    if op == "distill":
        vocab = _width(rng, 1000, 131072)
        return dict(op=op, rows=_between(rng, 1, min(4096, (1 << 28) // vocab)), vocab=vocab, top=_between(rng, 1, 128),
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), temperature=rng.choice([0.7, 1.0, 2.0, 4.0]))
    k, n = _width(rng, 256, 8192), _width(rng, 256, 16384)
    m = _between(rng, 1, min(8192, (1 << 39) // (k * n)))
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    bias, residual = rng.random() < 0.7, rng.random() < 0.5
    if op == "int8":
        return dict(op=op, m=m, k=k, n=n, dtype=rng.choice(["bf16", "bf16", "f16"]), act=act, bias=bias, residual=residual,
                    norm=rng.random() < 0.6)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if dtype == "f32":
        m, k, n = min(m, 2048), min(k, 2048), min(n, 4096)
    return dict(op=op, m=m, k=k, n=n, dtype=dtype, act=act, bias=bias, residual=residual, train=rng.random() < 0.5)


def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _stream(gen, rows, n, dtype):
    """A residual stream: some channels are far larger than the others, and a few rows are small."""
    v = torch.randn(rows, n, generator=gen, device="cuda") * 2.0
    v *= 1.0 + 15.0 * (torch.rand(n, generator=gen, device="cuda") < 0.01).float()
    v *= torch.exp(torch.randn(rows, 1, generator=gen, device="cuda") * 0.5)
    return v.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s, t = dict(case), _TYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        s["x"] = _normal(gen, rows, n, dtype=t) if case["residual"] else _stream(gen, rows, n, t)
        s["r"] = _stream(gen, rows, n, t) if case["residual"] else None
        s["w"] = (1.0 + _normal(gen, n, scale=0.2)).to(t)
        if case["train"]:
            s["gy"] = _normal(gen, rows, n, dtype=t)
            s["gh"] = _normal(gen, rows, n, dtype=t) if case["residual"] else None
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = _normal(gen, m, k, dtype=t)
        s["w"] = _normal(gen, k, n, scale=1.5 / math.sqrt(k), dtype=t)      # [in, out], as the layers hold it
        s["b"] = _normal(gen, n, scale=0.5, dtype=t) if case["bias"] else None
        s["r"] = _normal(gen, m, n, dtype=t) if case["residual"] else None
        s["gy"] = _normal(gen, m, n, dtype=t) if case["train"] else None
    elif case["op"] == "int8":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = _normal(gen, m, k, dtype=t)
        s["xr"] = _stream(gen, m, k, t) if case["norm"] else None            # the residual stream before the norm
        s["nw"] = (1.0 + _normal(gen, k, scale=0.2)).to(t) if case["norm"] else None
        w = _normal(gen, n, k, scale=1.5 / math.sqrt(k))                     # quantised once, a scale for each output
        s["ws"] = w.abs().amax(dim=1) / 127.0
        s["w"] = torch.clamp(torch.round(w / s["ws"][:, None]), -127, 127).to(torch.int8)   # [out, in]
        s["b"] = _normal(gen, n, scale=0.5, dtype=t) if case["bias"] else None
        s["r"] = _normal(gen, m, n, dtype=t) if case["residual"] else None
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        s["s"] = _normal(gen, rows, vocab, scale=2.0, dtype=t)
        # the teacher's largest logits, falling, at distinct places; some rows have fewer, a few none at all
        first = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        step = 1 + torch.randint(0, max(1, vocab // top - 1), (rows, 1), generator=gen, device="cuda")
        s["i"] = ((first + step * torch.arange(top, device="cuda")) % vocab).to(torch.int32)
        fall = torch.cumsum(torch.rand(rows, top, generator=gen, device="cuda"), dim=1)
        s["t"] = (12.0 - fall).to(t)
        kept = torch.randint(0, 2 * top + 1, (rows, 1), generator=gen, device="cuda")
        s["i"][torch.arange(top, device="cuda")[None, :] >= kept] = -1
        # each row's share of the loss: a mean over the batch without its padding (Float16 trains with a loss scale)
        live = (torch.rand(rows, generator=gen, device="cuda") < 0.9).float()
        live[0] = 1.0
        s["rw"] = live / live.sum() * (16384.0 if case["dtype"] == "f16" else 1.0)
    return s


# ---- plain forms: elementary operations in 32 bits, one rounding at the end ---------------------------------------

def _act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), torch.ones_like(z))
    if act == "gelu":
        return 0.5 * torch.special.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if act == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    return torch.ones_like(z)


def _plain_norm(s):
    t = s["x"].dtype
    h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
    w = s["w"].float()
    rstd = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + _EPS)
    y = (h * rstd * w).to(t)
    out = {"y": y}
    if s["r"] is not None:
        out["h"] = h.to(t)
    if s["train"]:
        gy = s["gy"].float()
        xhat = h * rstd
        g = gy * w
        gx = rstd * (g - xhat * (g * xhat).mean(dim=1, keepdim=True))
        if s["gh"] is not None:
            gx = gx + s["gh"].float()
        out["gx"], out["gw"] = gx.to(t), (gy * xhat).sum(dim=0).to(t)
    return out


def _plain_linear(s):
    t = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(t)}
    if s["train"]:
        gz = s["gy"].float() * _act_slope(z, s["act"])
        out["gx"], out["gw"] = (gz @ w.t()).to(t), (x.t() @ gz).to(t)
        if s["b"] is not None:
            out["gb"] = gz.sum(dim=0).to(t)
    return out


def _plain_int8(s):
    t = s["x"].dtype
    out = {}
    u = s["x"].float()
    rstd = 1.0
    if s["norm"]:
        h = u + s["xr"].float()
        out["h"] = h.to(t)
        rstd = 1.0 / torch.sqrt((h * h).mean(dim=1) + _EPS)
        u = h * s["nw"].float()
    # the rounded value does not depend on the row's norm, only its scale does
    top = u.abs().amax(dim=1)
    q = torch.clamp(torch.round(u * torch.div(torch.full_like(top, 127.0), top)[:, None]), -127, 127)
    out["scale"] = top * rstd / 127.0
    z = (q @ s["w"].float().t()) * out["scale"][:, None] * s["ws"]
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out["y"] = y.to(t)
    return out


def _plain_distill(s):
    x = s["s"].float() * (1.0 / s["temperature"])
    top = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(dim=1, keepdim=True)
    there = s["i"] >= 0
    at = torch.where(there, s["i"], torch.zeros_like(s["i"])).long()
    t = torch.where(there, s["t"].float() * (1.0 / s["temperature"]), torch.full_like(s["t"], -math.inf, dtype=torch.float32))
    some = there.any(dim=1, keepdim=True)
    p = torch.exp(t - torch.where(some, t.amax(dim=1, keepdim=True), torch.zeros_like(total)))
    p = p / torch.where(some, p.sum(dim=1, keepdim=True), torch.ones_like(total))
    logq = x.gather(1, at) - top - torch.log(total)
    terms = torch.where(p > 0, p * (torch.log(p) - logq), torch.zeros_like(p))
    tt = s["temperature"] * s["temperature"]
    row = tt * terms.sum(dim=1)
    g = (e / total) * some
    g.scatter_add_(1, at, -p)
    grad = (g * (s["temperature"] * s["rw"])[:, None]).to(s["s"].dtype)
    row = torch.where(s["rw"] != 0, row, torch.zeros_like(row))
    return {"loss": (s["rw"] * row).sum(), "row": row, "grad": grad}


def _own(s):
    from neurotensor_b200 import api
    if s["op"] == "norm":
        y, h, rstd = api.rms_norm(s["x"], s["w"], eps=_EPS, residual=s["r"])
        out = {"y": y}
        if s["r"] is not None:
            out["h"] = h
        if s["train"]:
            out["gx"], out["gw"] = api.rms_norm_backward(h, s["w"], rstd, s["gy"], grad_h=s["gh"])
        return out
    if s["op"] == "linear":
        if not s["train"]:
            return {"y": api.linear_act(s["x"], s["w"], s["b"], s["act"], residual=s["r"])}
        y, pre = api.linear_act(s["x"], s["w"], s["b"], s["act"], residual=s["r"], want_pre=True)
        gx, gw, gb = api.linear_act_backward(s["x"], s["w"], pre, s["gy"], s["act"], want_bias=s["b"] is not None)
        out = {"y": y, "gx": gx, "gw": gw}
        if gb is not None:
            out["gb"] = gb
        return out
    if s["op"] == "int8":
        out = {}
        if s["norm"]:
            q, out["scale"], out["h"] = api.rms_norm_int8(s["x"], s["nw"], eps=_EPS, residual=s["xr"])
        else:
            q, out["scale"] = api.quantize_rows(s["x"])
        out["y"] = api.linear_int8(q, out["scale"], s["w"], s["ws"], s["b"], s["act"], residual=s["r"], transpose_w=True,
                                   dtype=s["x"].dtype)
        return out
    loss, row, grad = api.distill_topk(s["s"], s["t"], s["i"], temperature=s["temperature"], row_weight=s["rw"])
    return {"loss": loss, "row": row, "grad": grad}


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "linear": _plain_linear, "int8": _plain_int8, "distill": _plain_distill}[state["op"]](state)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        e = case["rows"] * case["n"]
        tensors = (4 if case["residual"] else 2) + (case["train"] and (3 if case["residual"] else 2))
        return {"bytes": e * es * tensors + case["n"] * es * (2 if case["train"] else 1), "flops": e * (14 if case["train"] else 5)}
    if case["op"] == "distill":
        e = case["rows"] * case["vocab"]
        return {"bytes": 2 * e * es + case["rows"] * (case["top"] * (4 + es) + 8), "flops": 6 * e}
    m, k, n = case["m"], case["k"], case["n"]
    flops = 2 * m * k * n
    if case["op"] == "int8":
        stream = m * k * es * (3 if case["norm"] else 1)
        return {"bytes": stream + n * k + 4 * (m + n) + m * n * es * (2 if case["residual"] else 1), "flops": flops}
    size = m * k + k * n + (n if case["bias"] else 0) + m * n * (2 if case["residual"] else 1)
    if case["train"]:
        size += m * n + m * k + k * n + (n if case["bias"] else 0)
        flops *= 3
    return {"bytes": size * es, "flops": flops}


# ---- the same results from the definitions, in 64 bits --------------------------------------------------------------

def _phi(z):
    return 0.5 * (1.0 + torch.erf(z / math.sqrt(2.0)))


def _exact_act(z, act):
    """(value, slope) of an activation."""
    if act == "relu":
        return z.clamp(min=0.0), (z >= 0).double()
    if act == "gelu":
        return z * _phi(z), _phi(z) + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":      # z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3)
        c = 2.0 * math.sqrt(2.0 / math.pi)
        g = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return z * g, g + z * g * (1 - g) * c * (1 + 0.134145 * z ** 2)
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    return z, torch.ones_like(z)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: (v.double() if isinstance(v, torch.Tensor) and v.dtype != torch.int32 else v) for k, v in s.items()}
    if case["op"] == "norm":
        h = d["x"] if d["r"] is None else d["x"] + d["r"]
        inv = (h.pow(2).sum(1, keepdim=True) / case["n"] + _EPS).rsqrt()
        out = {"y": h * inv * d["w"]}
        if d["r"] is not None:
            out["h"] = h
        if case["train"]:
            a = d["gy"] * d["w"]
            out["gx"] = a * inv - h * inv.pow(3) * (a * h).sum(1, keepdim=True) / case["n"]
            if d["gh"] is not None:
                out["gx"] = out["gx"] + d["gh"]
            out["gw"] = torch.einsum("rn,rn->n", d["gy"], h * inv)
        return out
    if case["op"] == "linear":
        z = torch.matmul(d["x"], d["w"])
        if d["b"] is not None:
            z += d["b"]
        value, slope = _exact_act(z, case["act"])
        out = {"y": value if d["r"] is None else value + d["r"]}
        if case["train"]:
            gz = d["gy"] * slope
            out["gx"], out["gw"] = torch.matmul(gz, d["w"].T), torch.matmul(d["x"].T, gz)
            if d["b"] is not None:
                out["gb"] = gz.sum(0)
        return out
    if case["op"] == "int8":
        out = {}
        v = d["x"]
        if case["norm"]:
            out["h"] = d["x"] + d["xr"]
            v = out["h"] / (out["h"].pow(2).sum(1, keepdim=True) / case["k"] + _EPS).sqrt() * d["nw"]
        out["scale"] = v.abs().max(1).values / 127
        q = (v / out["scale"].unsqueeze(1)).round()
        z = torch.matmul(q * out["scale"].unsqueeze(1), (d["w"] * d["ws"].unsqueeze(1)).T)
        if d["b"] is not None:
            z += d["b"]
        value, _ = _exact_act(z, case["act"])
        out["y"] = value if d["r"] is None else value + d["r"]
        return out
    # a block of rows at a time: 64-bit copies of the logits are large
    temp, rows = case["temperature"], case["rows"]
    loss_rows, grads = [], []
    for r0 in range(0, rows, 512):
        logits, i, t, rw = (d[k][r0:r0 + 512] for k in ("s", "i", "t", "rw"))
        logq = torch.log_softmax(logits / temp, dim=1)
        row = torch.zeros(logits.shape[0], dtype=torch.float64, device="cuda")
        grad = torch.zeros_like(logits)
        there = i >= 0
        live = (there.any(1) & (rw != 0)).nonzero().flatten()
        if live.numel():
            pt = torch.softmax((t / temp).masked_fill(~there, -math.inf)[live], dim=1)
            at = i[live].clamp(min=0).long()
            full = torch.zeros(live.numel(), logits.shape[1], dtype=torch.float64, device="cuda").scatter_add_(1, at, pt)
            row[live] = temp ** 2 * (torch.xlogy(pt, pt) - pt * logq[live].gather(1, at)).sum(1)
            grad[live] = temp * rw[live].unsqueeze(1) * (logq[live].exp() - full)
        loss_rows.append(row)
        grads.append(grad.float() if case["dtype"] != "f32" else grad)     # 32 bits are far finer than the 16 it is held against
    row = torch.cat(loss_rows)
    return {"loss": (row * d["rw"]).sum(), "row": row, "grad": torch.cat(grads)}
