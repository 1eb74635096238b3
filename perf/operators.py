"""What the distillation operators are measured on: the linear layer in 8-bit floating point (serving and training), the selection of a
teacher's top logits, and the loss that a student takes from them, with its gradient.

`own` false: the plain forms (elementary torch operations in 32 bits); `own` true: the same calls through cnmnet_amd.  `exact` computes
the definitions in 64 bits.  The 8-bit format is e4m3 with one power-of-two scale (an 8-bit exponent) per block: 1 x 128 along the reduced
axis for activations and gradients, 128 x 128 for weights; the reduced axis is padded with zeros to a multiple of 128.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # linear: y = x w^T, w in 8 bits and in hand, x quantised by the call
        {"name": "linear 1x4096x4096", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16"},                 # serving: one token, latency counts
        {"name": "linear 37x5003x2057", "op": "linear", "m": 37, "n": 5003, "k": 2057, "dtype": "f16"},                # a ragged batch of tokens, odd in all three sizes
        {"name": "linear 49152x64x512", "op": "linear", "m": 49152, "n": 64, "k": 512, "dtype": "f32"},                # 64 plane logits for every pixel of a 192 x 256 frame from 512 channels
        {"name": "linear 8192x8192x8192", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16"},           # a large prompt batch through a wide layer
        # linear_train: y, dx, dw of one training step of such a layer, weight quantised in the step as its packing is
        {"name": "train 1001x776x520", "op": "linear_train", "m": 1001, "n": 776, "k": 520, "dtype": "f32"},           # a small head, odd number of rows
        {"name": "train 8192x4096x4096", "op": "linear_train", "m": 8192, "n": 4096, "k": 4096, "dtype": "bf16"},      # an ordinary training batch
        # top: a teacher's k largest logits per row, their classes, and the row's log-sum-exp
        {"name": "top 1x131072", "op": "top", "outer": 1, "classes": 131072, "inner": 1, "k": 64, "dtype": "bf16", "t": 1.0},        # one token of a served teacher
        {"name": "top 4x64x192x256", "op": "top", "outer": 4, "classes": 64, "inner": 49152, "k": 8, "dtype": "f32", "t": 1.0},      # plane volumes of a training batch, classes in dim 1
        {"name": "top 4096x32768", "op": "top", "outer": 4096, "classes": 32768, "inner": 1, "k": 32, "dtype": "bf16", "t": 2.0},    # a batch of tokens for a teacher's cache
        # distill: the loss against stored top logits and the gradient of the student's logits
        {"name": "distill 7x50021", "op": "distill", "outer": 7, "classes": 50021, "inner": 1, "k": 16, "dtype": "f32", "t": 2.0,
         "tail": True, "weight": False, "short": True, "grad": True},                                                              # few rows, odd length, rows with fewer or no entries
        {"name": "distill 4x64x192x256", "op": "distill", "outer": 4, "classes": 64, "inner": 49152, "k": 8, "dtype": "f32", "t": 1.0,
         "tail": True, "weight": True, "short": False, "grad": True},                                                              # a student's plane volumes with the frame's valid mask
        {"name": "distill 4096x32768", "op": "distill", "outer": 4096, "classes": 32768, "inner": 1, "k": 32, "dtype": "bf16", "t": 2.0,
         "tail": False, "weight": True, "short": True, "grad": True},                                                              # a batch of tokens, entries renormalised, padded rows
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear_train", "top", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "linear":
        while True:
            c = {"op": op, "m": _log_int(rng, 1, 49152), "n": _log_int(rng, 16, 8192), "k": _log_int(rng, 32, 8192), "dtype": dtype}
            if c["m"] * c["n"] * c["k"] <= 2 ** 37 and c["m"] * max(c["n"], c["k"]) <= 2 ** 26:
                return c
    if op == "linear_train":
        while True:
            c = {"op": op, "m": _log_int(rng, 1, 16384), "n": _log_int(rng, 16, 4096), "k": _log_int(rng, 32, 4096), "dtype": dtype}
            if c["m"] * c["n"] * c["k"] <= 2 ** 36 and c["m"] * max(c["n"], c["k"]) <= 2 ** 25:
                return c
    strided = rng.random() < 0.4
    while True:
        if strided:                                                      # class planes of images: [outer, classes, inner]
            classes, outer, inner = _log_int(rng, 16, 256), rng.randint(1, 8), _log_int(rng, 100, 307200)
        else:
            classes, outer, inner = _log_int(rng, 16, 131072), _log_int(rng, 1, 16384), 1
        if outer * classes * inner <= 2 ** 26:
            break
    c = {"op": op, "outer": outer, "classes": classes, "inner": inner, "k": _log_int(rng, 1, min(128, classes // 2)), "dtype": dtype, "t": rng.choice([1.0, 2.0, 4.0, 0.5])}
    if strided:
        c["k"] = min(c["k"], 16)
    if op == "distill":
        many = outer * inner >= 16                                       # a mask and missing entries are a matter of many rows
        c.update(tail=rng.random() < 0.6, weight=many and rng.random() < 0.5, short=many and rng.random() < 0.5, grad=rng.random() < 0.7)
    return c


# --------------------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(0x5EED0 + seed)
    return g


def _data(case, seed):
    """The case's inputs as a user's program holds them, from the seed alone."""
    g, dt = _gen(seed), DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] in ("linear", "linear_train"):
        m, n, k = case["m"], case["n"], case["k"]
        x = (randn(m, k) * torch.exp(0.5 * randn(m, 1)) * torch.exp(0.5 * randn(1, k))).to(dt)      # rows and channels of different sizes
        w = (randn(n, k) / math.sqrt(k)).to(dt)
        if case["op"] == "linear":
            q, s = _pack_weight(w)
            return {"x": x, "q": q, "s": s}
        return {"x": x, "w": w, "dy": (randn(m, n) * torch.exp(randn(m, 1)) / m).to(dt)}
    outer, classes, inner, k, t = case["outer"], case["classes"], case["inner"], case["k"], case["t"]
    shape = (outer, classes) if inner == 1 else (outer, classes, inner)
    z = (3.0 * randn(*shape)).to(dt)
    if case["op"] == "top":
        return {"z": z}
    teacher = 0.8 * z.float() + 1.5 * randn(*shape)
    val, idx = torch.topk(teacher, k, dim=1)
    lse = torch.logsumexp(teacher / t, 1) if case["tail"] else None
    idx = idx.to(torch.int32)
    if case["short"]:                                                    # rows with fewer entries than k, some with none: index -1
        n_have = torch.randint(0, k + 1, (outer, 1) + shape[2:], device="cuda", generator=g)
        pos = torch.arange(k, device="cuda").view((1, k) + (1,) * (len(shape) - 2))
        idx = torch.where(pos < n_have, idx, torch.full_like(idx, -1))
    w = None
    if case["weight"]:                                                   # a valid mask with weights: a fifth of the rows count for nothing
        u = torch.rand((outer,) + shape[2:], device="cuda", generator=g)
        w = torch.where(u < 0.2, torch.zeros_like(u), u + 0.5)
    return {"z": z, "idx": idx, "val": val.to(dt), "lse": lse, "w": w}


def _blocks(x, rows):
    """x [R, C] as [ceil(R / rows), rows, ceil(C / 128), 128], padded with zeros."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // 128, 128)


def _scale_exponent(amax):
    """The exponent e of the smallest power of two with amax <= 448 * 2^e, from -127 on; amax >= 0 in 32 or 64 bits."""
    mant, ex = torch.frexp(amax)                                         # amax = mant * 2^ex, 0.5 <= mant < 1;  448 = 0.875 * 2^9
    e = ex - 9 + (mant > 0.875).to(ex.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(min=-127)


def _pow2(e):
    """2^e in 32 bits, exactly, e from -149 to 127 (exponents as integers: a power function may be an ulp off, and ties would round the other way)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64).float()


def _pack_weight(w):
    """A weight [N, K] in the layer's 8-bit format: values [N, K padded to 128] and one exponent per 128 x 128 block."""
    n, k = w.shape
    b = _blocks(w.float(), 128)
    e = _scale_exponent(b.abs().amax((1, 3), keepdim=True))
    q = (b * _pow2(-e)).reshape(b.shape[0] * 128, -1)[:n].contiguous().to(torch.float8_e4m3fn)
    return q, (e.view(b.shape[0], b.shape[2]) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    state = dict(_data(case, seed), case=case)
    if case["op"] == "linear_train":
        state["x"].requires_grad_()
        state["w"].requires_grad_()
    elif case["op"] == "distill" and case["grad"]:
        state["z"].requires_grad_()
    if own and case["op"] == "distill":
        from cnmnet_amd.depthnet.losses import TopLogitsDistillLoss
        state["loss"] = TopLogitsDistillLoss(temperature=case["t"], dim=1, reduction="mean" if case["grad"] else "none")
    return state


# ------------------------------------------------------------------------------------------------------------ plain forms

def _rounded(x, rows):
    """x [R, C] -> the values its 8-bit form stands for, 32 bits, [R, C padded to 128]."""
    b = _blocks(x.float(), rows)
    e = _scale_exponent(b.abs().amax((1, 3), keepdim=True))
    q = (b * _pow2(-e)).to(torch.float8_e4m3fn).float()
    return (q * _pow2(e)).reshape(b.shape[0] * rows, -1)[: x.shape[0]]


def _plain_linear(s):
    n, kp = s["q"].shape
    w = s["q"].float() * s["s"].float().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    return (_rounded(s["x"].detach(), 1) @ w.t()).to(s["x"].dtype)


def _plain_linear_train(s):
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
    n, k = w.shape
    w8 = _rounded(w, 128)[:, :k]
    y = _rounded(x, 1)[:, :k] @ w8.t()
    dx = _rounded(dy, 1)[:, :n] @ w8
    dw = _rounded(dy.t(), 1) @ _rounded(x.t(), 1).t()                    # the reduced axis is the rows: both blocked along it
    return y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype)


def _plain_top(s):
    z, c = s["z"], s["case"]
    idx = torch.sort(z, dim=1, descending=True, stable=True)[1].narrow(1, 0, c["k"])
    a = z.float() / c["t"]
    m = a.amax(1, keepdim=True)
    lse = (m + (a - m).exp().sum(1, keepdim=True).log()).squeeze(1)
    return z.gather(1, idx), idx.to(torch.int32), lse


def _plain_distill(s):
    c, z, idx = s["case"], s["z"].detach(), s["idx"].long()
    t = c["t"]
    a = z.float() / t
    have = idx >= 0
    at = idx.clamp(min=0)
    # the row's few numbers in 64 bits: a small loss is the difference of logarithms that nearly cancel
    none = torch.full((), -math.inf, device=z.device, dtype=torch.float64)
    zero = torch.zeros((), device=z.device, dtype=torch.float64)
    b = torch.where(have, s["val"].double() / t, none)
    if c["tail"]:
        lp = b - s["lse"].double().unsqueeze(1)
    else:
        m = b.amax(1, keepdim=True)
        m = torch.where(m > none, m, zero)
        lp = b - (m + (b - m).exp().sum(1, keepdim=True).log())
    p = torch.where(have, lp.exp(), zero)
    m = a.amax(1, keepdim=True)
    ex = (a - m).exp()
    total = ex.sum(1, keepdim=True, dtype=torch.float64)
    lq = a.gather(1, at).double() - m.double() - total.log()
    loss = torch.where(p > 0, p * (lp - lq), zero).sum(1)
    some = have.any(1)
    q = ex * (1 / total).float()
    grad = q - torch.zeros_like(a).scatter_add_(1, at, p.float())
    if c["tail"]:
        listed_ = torch.zeros_like(a).scatter_add_(1, at, have.float()) > 0
        pr = (1 - p.sum(1)).clamp(min=0)
        qr = torch.where(listed_, torch.zeros_like(ex), ex).sum(1, dtype=torch.float64) / total.squeeze(1)
        loss = loss + torch.where(some & (pr > 0), pr * (pr.log() - qr.log()), zero)
        grad = torch.where(listed_, grad, q * (1 - pr / qr).float().unsqueeze(1))
    loss = loss * (t * t)
    if not c["grad"]:
        return loss.float()
    w = s["w"].double() if s["w"] is not None else torch.ones_like(loss)
    grad = grad * (some * w / w.sum() * t).float().unsqueeze(1)
    return ((loss * w).sum() / w.sum()).float(), grad.to(z.dtype)


def run(state):
    c = state["case"]
    if not own:
        return {"linear": _plain_linear, "linear_train": _plain_linear_train, "top": _plain_top, "distill": _plain_distill}[c["op"]](state)
    from cnmnet_amd import autograd, ops
    if c["op"] == "linear":
        return ops.linear_fp8(state["x"], state["q"], state["s"])
    if c["op"] == "linear_train":
        y = autograd.linear_fp8(state["x"], state["w"])
        return (y.detach(),) + torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
    if c["op"] == "top":
        return ops.top_logits(state["z"], c["k"], dim=1, temperature=c["t"])
    loss = state["loss"](state["z"], state["idx"], state["val"], state["lse"], state["w"] if c["grad"] else None)      # rows' losses by themselves: unweighted
    if not c["grad"]:
        return loss
    return loss.detach(), torch.autograd.grad(loss, state["z"])[0]


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": b * (m * k + m * n) + n * k, "flops": 2 * m * n * k}
    if case["op"] == "linear_train":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": b * 2 * (m * k + m * n + n * k), "flops": 6 * m * n * k}
    rows, classes, k = case["outer"] * case["inner"], case["classes"], case["k"]
    if case["op"] == "top":
        return {"bytes": rows * (classes * b + k * (b + 4) + 4), "flops": 4 * rows * classes}
    grad = 2 if case["grad"] else 1
    entries = rows * (k * (b + 4) + 4 * (bool(case["tail"]) + bool(case["weight"])))
    return {"bytes": grad * rows * classes * b + entries + (4 if case["grad"] else 4 * rows), "flops": (8 if case["grad"] else 4) * rows * classes}


# ----------------------------------------------------------------------------------------------------------------- 64 bits

def _stands_for(x, rows):
    """The values of x's 8-bit form from its definition: e4m3 has 3 fraction bits, exponents from -6 on, ties to even."""
    x = x.double()
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    power = torch.tensor([2.0 ** i for i in range(-200, 200)], dtype=torch.float64, device=x.device)
    for r0 in range(0, x.shape[0], max(rows, 4096)):
        part = x[r0:r0 + max(rows, 4096)]
        r, c = part.shape
        grid = torch.zeros(-(-r // rows) * rows, -(-c // 128) * 128, dtype=torch.float64, device=x.device)
        grid[:r, :c] = part
        grid = grid.view(-1, rows, grid.shape[1] // 128, 128)
        amax = grid.abs().amax(3, keepdim=True).amax(1, keepdim=True)
        e = torch.ceil(torch.log2(amax / 448.0)).clamp(min=-127).long()
        e = torch.where(448.0 * power[e - 1 + 200] >= amax, e - 1, e)    # log2 may round across a power of two
        e = torch.where(448.0 * power[e + 200] < amax, e + 1, e).clamp(min=-127)
        v = grid / power[e + 200]
        step = power[torch.frexp(v)[1].clamp(min=-5).long() - 4 + 200]
        out[r0:r0 + r] = (torch.round(v / step) * step * power[e + 200]).view(-1, grid.shape[2] * 128)[:r, :c]
    return out


def exact(case, seed):
    d = _data(case, seed)
    if case["op"] == "linear":
        n, kp = d["q"].shape
        scale = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=torch.float64, device="cuda")[d["s"].view(torch.uint8).long()]
        rows, cols = torch.arange(n, device="cuda") // 128, torch.arange(kp, device="cuda") // 128
        w = d["q"].double() * scale[rows][:, cols]
        return torch.matmul(_stands_for(d["x"], 1), w[:, : case["k"]].t().contiguous())
    if case["op"] == "linear_train":
        w8 = _stands_for(d["w"], 128)
        y = torch.matmul(_stands_for(d["x"], 1), w8.t().contiguous())
        dx = torch.matmul(_stands_for(d["dy"], 1), w8)
        dw = torch.matmul(_stands_for(d["dy"].t().contiguous(), 1), _stands_for(d["x"].t().contiguous(), 1).t().contiguous())
        return y, dx, dw
    classes_last = d["z"] if case["inner"] == 1 else d["z"].transpose(1, 2).reshape(-1, case["classes"])
    rows = classes_last.shape[0]
    step = max(1, 2 ** 25 // case["classes"])

    def last(x):
        return x if x is None or x.dim() == 2 else x.transpose(1, 2).reshape(rows, -1)

    if case["op"] == "top":
        lse = torch.cat([torch.logsumexp(classes_last[r:r + step].double() / case["t"], 1) for r in range(0, rows, step)])
        val = torch.cat([torch.topk(classes_last[r:r + step].double(), case["k"], dim=1)[0] for r in range(0, rows, step)])
        if case["inner"] > 1:
            val, lse = val.view(case["outer"], case["inner"], -1).transpose(1, 2), lse.view(case["outer"], case["inner"])
        return val.contiguous(), None, lse
    t, idx, val = case["t"], last(d["idx"]).long(), last(d["val"]).double()
    t_lse = None if d["lse"] is None else d["lse"].reshape(-1).double()
    weight = torch.ones(rows, dtype=torch.float64, device="cuda") if d["w"] is None else d["w"].reshape(-1).double()
    losses, grads = [], []
    for r in range(0, rows, step):
        logq = torch.log_softmax(classes_last[r:r + step].double() / t, 1)
        have = idx[r:r + step] >= 0
        at = torch.where(have, idx[r:r + step], 0)
        raw = torch.where(have, val[r:r + step] / t, -math.inf)
        logp = raw - t_lse[r:r + step, None] if t_lse is not None else torch.log_softmax(raw, 1)
        p = torch.where(have, logp.exp(), 0.0)
        kl = torch.where(p > 0, p * (logp - torch.gather(logq, 1, at)), 0.0).sum(1)
        q = logq.exp()
        part = q - torch.zeros_like(q).scatter_add_(1, at, p)
        if t_lse is not None:
            inside = torch.zeros_like(q, dtype=torch.int32).scatter_add_(1, at, have.int()) > 0
            rest_p = (1.0 - p.sum(1)).clamp(min=0.0)
            rest_q = torch.where(inside, 0.0, q).sum(1)
            kl = kl + torch.where(have.any(1) & (rest_p > 0), rest_p * (rest_p.log() - rest_q.log()), 0.0)
            part = torch.where(inside, part, q * (1.0 - rest_p / rest_q)[:, None])
        losses.append(t * t * kl)
        if case["grad"]:
            grads.append(part * (t * weight[r:r + step] / weight.sum() * have.any(1))[:, None])
    loss = torch.cat(losses)
    if not case["grad"]:
        return loss if case["inner"] == 1 else loss.view(case["outer"], case["inner"])
    grad = torch.cat(grads)
    if case["inner"] > 1:
        grad = grad.view(case["outer"], case["inner"], case["classes"]).transpose(1, 2).contiguous()
    return (loss * weight).sum() / weight.sum(), grad
