"""The block-scaled FP8 operators as timed cases: the Linear with one scale for every 128 values, the experts' Linears over
rows sorted by expert, and the residual RMS norm that hands its result on in 8 bits.

Every quantized block is 128 values long: along a row for an activation (rows x columns / 128 scales), along the tokens of one
expert for the two operands of a weight gradient, 128 x 128 for a weight. A scale that the operators make is the smallest power
of two with max|block| <= 448 scale; weights that come quantized (a checkpoint) have any fp32 scale.

A case is {"kind": ...} and:
  linear_serve   tokens, cin, cout                 y of a quantized weight
  linear_train   tokens, cin, cout, weight         y, dx, dw; the weight in fp32 or bf16
  experts_serve  rows, tail, experts, cin, cout    y of quantized weights; `tail` of the rows belong to no expert
  experts_train  rows, tail, experts, cin, cout, weight
  norm_linear    tokens, cin, cout, add, gain      the residual's addition, norm, and the Linear that reads its 8 bits
  norm_train     tokens, cin, add, gain            norm forward and backward: res, n, its 8 bits, dx, dgain; the scales of
                                                   the 8 bits show in norm_linear (a last bit of rstd may double one)
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
BLOCK = 128


def listed():
    return [
        # one token through a d24 attention-output projection: decoding
        {"name": "serve_1", "kind": "linear_serve", "tokens": 1, "cin": 1536, "cout": 1536},
        # a decoding batch through the d24 MLP's first projection
        {"name": "serve_48", "kind": "linear_serve", "tokens": 48, "cin": 1536, "cout": 6144},
        # a prompt of odd length through the d26 MLP's first projection
        {"name": "serve_prompt_odd", "kind": "linear_serve", "tokens": 3001, "cin": 1664, "cout": 6656},
        # a training step's micro-batch through the d24 MLP's second projection: the largest call
        {"name": "train_d24", "kind": "linear_train", "tokens": 16384, "cin": 6144, "cout": 1536, "weight": "fp32"},
        # a short odd batch through a layer whose sides are no multiples of 128, weight kept in bf16
        {"name": "train_odd", "kind": "linear_train", "tokens": 1111, "cin": 1040, "cout": 2000, "weight": "bf16"},
        # 24 decoded tokens at two experts each: most experts have no row or one
        {"name": "experts_decode", "kind": "experts_serve", "rows": 48, "tail": 0, "experts": 64, "cin": 1536, "cout": 2048},
        # a prompt's tokens over 32 experts, the batch padded at its end
        {"name": "experts_prompt", "kind": "experts_serve", "rows": 8192, "tail": 100, "experts": 32, "cin": 1536, "cout": 2048},
        # a training step over 16 experts, forward and backward
        {"name": "experts_train", "kind": "experts_train", "rows": 16384, "tail": 0, "experts": 16, "cin": 1536, "cout": 2048, "weight": "fp32"},
        # one decoded token: the block's entry and its merged q/k/v projection
        {"name": "norm_linear_1", "kind": "norm_linear", "tokens": 1, "cin": 1536, "cout": 4608, "add": True, "gain": True},
        # a prompt through the same of a d20 model without gains
        {"name": "norm_linear_prompt", "kind": "norm_linear", "tokens": 2500, "cin": 1280, "cout": 3840, "add": True, "gain": False},
        # the norm of a d24 training micro-batch, forward and backward
        {"name": "norm_train_d24", "kind": "norm_train", "tokens": 16384, "cin": 1536, "add": True, "gain": True},
        # a wide norm over few rows, its width no multiple of 128
        {"name": "norm_train_odd", "kind": "norm_train", "tokens": 509, "cin": 5040, "add": False, "gain": True},
    ]


def _log(rng, low, high, step=1):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v // step * step if v >= step else step))


def draw(rng):
    kind = rng.choice(["linear_serve", "linear_train", "experts_serve", "experts_train", "norm_linear", "norm_train"])
    cin, cout = _log(rng, 256, 6144, 16), _log(rng, 256, 6144, 16)
    if kind == "linear_serve":
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "cin": cin, "cout": cout}
    if kind == "linear_train":
        return {"kind": kind, "tokens": _log(rng, 16, 8192), "cin": cin, "cout": cout, "weight": rng.choice(["fp32", "bf16"])}
    if kind == "norm_linear":
        return {"kind": kind, "tokens": _log(rng, 1, 4096), "cin": cin, "cout": cout, "add": rng.random() < 0.7, "gain": rng.random() < 0.7}
    if kind == "norm_train":
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "cin": _log(rng, 128, 4096, 16), "add": rng.random() < 0.7, "gain": rng.random() < 0.7}
    experts, cin, cout = _log(rng, 2, 128), _log(rng, 256, 2048, 16), _log(rng, 256, 2048, 16)
    if kind == "experts_serve":
        rows = _log(rng, 1, 16384)
        return {"kind": kind, "rows": rows, "tail": rng.choice([0, rng.randint(0, rows // 8)]), "experts": experts, "cin": cin, "cout": cout}
    rows = _log(rng, 128, 16384)
    return {"kind": kind, "rows": rows, "tail": rng.choice([0, rng.randint(0, rows // 8)]), "experts": experts, "cin": cin, "cout": cout,
            "weight": rng.choice(["fp32", "bf16"])}


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, cin, cout = case["kind"], case["cin"], case.get("cout")
    rows = case["tokens"] if "tokens" in case else case["rows"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    # activations: unit variance, some columns several times larger than others
    x = (normal(rows, cin) * torch.exp(0.5 * normal(cin))).to(torch.bfloat16)
    s = {"case": dict(case), "x": x}
    if kind.startswith("norm"):
        s["r"] = normal(rows, cin).to(torch.bfloat16) if case["add"] else None
        s["gain"] = 1.0 + 0.1 * normal(cin) if case["gain"] else None
    if kind.startswith("experts"):
        # a router's choice: some experts are asked for more often than others, some by nobody
        liked = torch.softmax(normal(case["experts"]), 0)
        if case["experts"] > 2:
            liked[case["experts"] // 3] = 0
        chosen = torch.multinomial(liked, rows - case["tail"], replacement=True, generator=g)
        counts = torch.bincount(chosen, minlength=case["experts"])
        s["ends"] = torch.cumsum(counts, 0).to(torch.int32)
        s["most"] = int(counts.max())
    if cout is not None:
        lead = (case["experts"],) if kind.startswith("experts") else ()
        w = normal(*lead, cout, cin) / math.sqrt(cin)
        if kind.endswith("train"):
            s["w"] = w.to(torch.bfloat16 if case["weight"] == "bf16" else torch.float32)
        else:  # a quantized checkpoint: one fp32 scale for 128 x 128 values
            a = torch.zeros(*lead, _up(cout) * BLOCK, _up(cin) * BLOCK, device="cuda")
            a[..., :cout, :cin] = w
            a = a.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))  # (..., nb, 128, kb, 128)
            scale = a.abs().amax(dim=(-3, -1)) / 448
            a = a / scale[..., :, None, :, None]
            s["w_data"] = a.flatten(-2).flatten(-3, -2)[..., :cout, :cin].to(torch.float8_e4m3fn).contiguous()
            s["w_scale"] = scale
    if kind.endswith("train"):
        s["grad"] = normal(rows, cout if cout is not None else cin).to(torch.bfloat16) * 0.01
        if kind == "norm_train":
            s["grad_res"] = normal(rows, cin).to(torch.bfloat16) * 0.01
    return s


def _up(n):
    return -(-n // BLOCK)


# ---------------------------------------------------------------------------------------------------- the plain forms

def _power(amax):
    """The smallest power of two p >= 2^-126 with amax <= 448 p (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    return ((torch.clamp(e - 9 + (m > 0.875), min=-126) + 127) << 23).to(torch.int32).view(torch.float32)


def _values(x, dim):
    """What x stands for after quantization in blocks of 128 along dim."""
    x = x.movedim(dim, -1)
    n = x.size(-1)
    p = torch.nn.functional.pad(x, (0, _up(n) * BLOCK - n)).unflatten(-1, (-1, BLOCK))
    s = _power(p.abs().amax(-1, keepdim=True))
    return ((p / s).to(torch.float8_e4m3fn).float() * s).flatten(-2)[..., :n].movedim(-1, dim)


def _weight_values(w):
    """The same for a weight in blocks of 128 x 128."""
    n, k = w.shape[-2:]
    p = torch.nn.functional.pad(w, (0, _up(k) * BLOCK - k, 0, _up(n) * BLOCK - n)).unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))
    s = _power(p.abs().amax(dim=(-3, -1), keepdim=True))
    return ((p / s).to(torch.float8_e4m3fn).float() * s).flatten(-2).flatten(-3, -2)[..., :n, :k]


def _given_values(data, scale):
    n, k = data.shape[-2:]
    return data.float() * scale.repeat_interleave(BLOCK, -1)[..., :k].repeat_interleave(BLOCK, -2)[..., :n, :]


def _plain_linear(s, w):
    return (_values(s["x"].float(), -1) @ w.transpose(-1, -2)).to(torch.bfloat16)


def _places(s):
    """Where each row stands when every expert's rows are padded to one length: (expert, place), and which rows have an expert."""
    row = torch.arange(s["x"].size(0), device="cuda")
    e = torch.searchsorted(s["ends"].long(), row, right=True)
    kept = e < s["ends"].numel()
    e = torch.where(kept, e, 0)
    start = torch.nn.functional.pad(s["ends"][:-1].long(), (1, 0))
    return e, row - start[e], kept, max(1, s["most"])


def _spread(t, where, experts):
    e, p, kept, most = where
    out = torch.zeros(experts, _up(most) * BLOCK, t.size(-1), device="cuda")
    out[e[kept], p[kept]] = t[kept]
    return out


def _gathered(t, where):
    e, p, kept, most = where
    return torch.where(kept[:, None], t[e, torch.where(kept, p, 0)], 0.0)


def _plain_experts(s, w):
    where = _places(s)
    xs = _spread(_values(s["x"].float(), -1), where, w.size(0))
    return _gathered(torch.bmm(xs, w.transpose(-1, -2)), where).to(torch.bfloat16)


def _plain_norm(s):
    res = (s["x"].float() + s["r"].float()).to(torch.bfloat16) if s["r"] is not None else s["x"]
    v = res.float()
    rstd = torch.rsqrt(v.square().mean(-1) + EPS)
    n = v * rstd[:, None]
    if s["gain"] is not None:
        n = n * s["gain"]
    return res, rstd, n.to(torch.bfloat16)


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "linear_serve":
        return _plain_linear(s, _given_values(s["w_data"], s["w_scale"]))
    if kind == "experts_serve":
        return _plain_experts(s, _given_values(s["w_data"], s["w_scale"]))
    if kind == "linear_train":
        x, g, w = s["x"].float(), s["grad"].float(), _weight_values(s["w"].float())
        y = _plain_linear(s, w)
        dx = (_values(g, -1) @ w).to(torch.bfloat16)
        dw = _values(g, 0).t() @ _values(x, 0)
        return y, dx, dw.to(s["w"].dtype)
    if kind == "experts_train":
        w, where = _weight_values(s["w"].float()), _places(s)
        y = _plain_experts(s, w)
        dx = _gathered(torch.bmm(_spread(_values(s["grad"].float(), -1), where, w.size(0)), w), where).to(torch.bfloat16)
        gs, xs = _spread(s["grad"].float(), where, w.size(0)), _spread(s["x"].float(), where, w.size(0))
        dw = torch.bmm(_values(gs, 1).transpose(1, 2), _values(xs, 1))
        return y, dx, dw.to(s["w"].dtype)
    res, rstd, n = _plain_norm(s)
    if kind == "norm_linear":
        return res, (_values(n.float(), -1) @ _given_values(s["w_data"], s["w_scale"]).t()).to(torch.bfloat16)
    v = res.float()
    p = torch.nn.functional.pad(n.float(), (0, _up(n.size(1)) * BLOCK - n.size(1))).unflatten(-1, (-1, BLOCK))
    data = (p / _power(p.abs().amax(-1, keepdim=True))).flatten(-2)[:, :n.size(1)].to(torch.float8_e4m3fn)
    hat, g = v * rstd[:, None], s["grad"].float()
    d = g * s["gain"] if s["gain"] is not None else g
    dx = rstd[:, None] * (d - hat * (d * hat).mean(-1, keepdim=True)) + s["grad_res"].float()
    out = {"res": res, "n": n, "data": data, "rstd": rstd, "dx": dx.to(torch.bfloat16)}
    if s["gain"] is not None:
        out["dgain"] = (g * hat).sum(0)
    return out


# ---------------------------------------------------------------------------------------------------- the framework's calls

def _own(s):
    import nanochat_cpp_b200 as nc
    kind = s["case"]["kind"]
    if kind == "linear_serve":
        return nc.fp8_block_matmul(s["x"], nc.BlockTensor(s["w_data"], s["w_scale"]))
    if kind == "experts_serve":
        return nc.fp8_block_experts(s["x"], nc.BlockTensor(s["w_data"], s["w_scale"]), s["ends"])
    if kind == "norm_linear":
        res, _, q, _ = nc.residual_norm_block(s["x"], s["r"], s["gain"], eps=EPS, with_n=False)
        return res, nc.fp8_block_matmul(None, nc.BlockTensor(s["w_data"], s["w_scale"]), x_block=q)
    x = s["x"].detach().requires_grad_()
    if kind == "norm_train":
        gain = s["gain"].detach().requires_grad_() if s["gain"] is not None else None
        res, n, q, rstd = nc.residual_norm_block(x, s["r"], gain, eps=EPS)
        grads = torch.autograd.grad((res, n), (x,) if gain is None else (x, gain), (s["grad_res"], s["grad"]))
        out = {"res": res, "n": n, "data": q.data, "rstd": rstd, "dx": grads[0]}
        if gain is not None:
            out["dgain"] = grads[1]
        return out
    w = s["w"].detach().requires_grad_()
    y = nc.fp8_block_matmul(x, w) if kind == "linear_train" else nc.fp8_block_experts(x, w, s["ends"])
    dx, dw = torch.autograd.grad(y, (x, w), s["grad"])
    return y.detach(), dx, dw


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------------------------------------------- work

def work(case):
    """Each input read once, each output written once, and the products; 8-bit intermediates count nothing."""
    kind, cin, cout = case["kind"], case["cin"], case.get("cout", 0)
    rows = case["tokens"] if "tokens" in case else case["rows"]
    experts = case.get("experts", 1)
    if kind == "norm_train":
        # x, with r its sum, n and its 8 bits; the two incoming gradients, dx; scales, rstd; gain, dgain
        b = rows * cin * (2 + 4 * case["add"] + 2 + 1 + 2 + 2 + 2) + 4 * rows * (_up(cin) + 1) + 8 * cin * case["gain"]
        return {"bytes": b, "flops": rows * cin * 16}
    routed = rows - case.get("tail", 0)
    if kind.endswith("serve") or kind == "norm_linear":
        used = experts if experts == 1 else min(experts, routed)
        b = 2 * rows * (cin + cout) + used * cin * cout
        if kind == "norm_linear":
            b += 4 * rows * cin * case["add"] + 4 * cin * case["gain"]
        return {"bytes": b, "flops": 2 * routed * cin * cout}
    size = 4 if case["weight"] == "fp32" else 2
    b = 2 * rows * (2 * cin + 2 * cout) + experts * cin * cout * 2 * size
    return {"bytes": b, "flops": 6 * routed * cin * cout}


# ---------------------------------------------------------------------------------------------------- 64 bits

def _e4m3(v):
    """v (64 bits, |v| <= 448) at the nearest value of 4 exponent and 3 mantissa bits, ties to even, steps of 2^-9 below 2^-6."""
    step = _two_to(torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(v / step) * step


def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _block_scale(a):
    p = _two_to(torch.frexp(torch.clamp(a / 448, min=2.0 ** -126))[1] - 2)
    for _ in range(3):  # upwards from a power that is at most the wanted one
        p = torch.where(448 * p < a, 2 * p, p)
    return torch.clamp(p, min=2.0 ** -126)


def _held(v, rows, cols):
    """A matrix (64 bits) as it is held in blocks of rows x cols, block row by block row."""
    out = torch.empty_like(v)
    for k in range(0, v.size(1), cols):
        c = v[:, k:k + cols]
        for n in range(0, v.size(0), max(rows, 1 << 14)):
            part = c[n:n + max(rows, 1 << 14)]
            if rows == 1:
                s = _block_scale(part.abs().amax(1, keepdim=True))
            else:
                s = _block_scale(torch.stack([q.abs().amax() if cols > 1 else q.abs().amax(0) for q in part.split(rows)]))
                s = s.reshape(len(s), -1).repeat_interleave(rows, 0)[:part.size(0)]
            out[n:n + max(rows, 1 << 14), k:k + cols] = _e4m3(part / s) * s
    return out


def _columns(v):
    """Blocks of 128 rows and one column."""
    return torch.cat([_held_column(part) for part in v.split(BLOCK)]) if v.size(0) else v


def _held_column(part):
    s = _block_scale(part.abs().amax(0, keepdim=True))
    return _e4m3(part / s) * s


def _stored(data, scale):
    out = data.double()
    for i in range(scale.size(0)):
        for j in range(scale.size(1)):
            out[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[i, j].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    x = s["x"].double()
    if kind.startswith("norm"):
        res = (x + s["r"].double()).to(torch.bfloat16) if s["r"] is not None else s["x"]
        v = res.double()
        rstd = 1 / torch.sqrt((v * v).sum(1) / v.size(1) + EPS)
        hat = v * rstd[:, None]
        n = hat * s["gain"].double() if s["gain"] is not None else hat
        held = n.to(torch.bfloat16).double()
        if kind == "norm_linear":
            return res.double(), _held(held, 1, BLOCK) @ _stored(s["w_data"], s["w_scale"]).t()
        data = torch.cat([_e4m3(c / _block_scale(c.abs().amax(1, keepdim=True))) for c in held.split(BLOCK, 1)], 1)
        g = s["grad"].double()
        d = g * s["gain"].double() if s["gain"] is not None else g
        dx = rstd[:, None] * (d - hat * ((d * hat).sum(1, keepdim=True) / v.size(1))) + s["grad_res"].double()
        out = {"res": res.double(), "n": n, "data": data, "rstd": rstd, "dx": dx}
        if s["gain"] is not None:
            out["dgain"] = (g * hat).sum(0)
        return out
    held = _held(x, 1, BLOCK)
    train = kind.endswith("train")
    if kind.startswith("linear"):
        w = _held(s["w"].double(), BLOCK, BLOCK) if train else _stored(s["w_data"], s["w_scale"])
        y = held @ w.t()
        if not train:
            return y
        g = s["grad"].double()
        return y, _held(g, 1, BLOCK) @ w, _columns(g).t() @ _columns(x)
    y = torch.zeros(x.size(0), case["cout"], device="cuda", dtype=torch.float64)
    if train:
        g = s["grad"].double()
        g_held, dx = _held(g, 1, BLOCK), torch.zeros_like(x)
        dw = torch.zeros(s["w"].shape, device="cuda", dtype=torch.float64)
    first = 0
    for e, last in enumerate(np.asarray(s["ends"].cpu()).tolist()):
        if last > first:
            w = _held(s["w"][e].double(), BLOCK, BLOCK) if train else _stored(s["w_data"][e], s["w_scale"][e])
            y[first:last] = held[first:last] @ w.t()
            if train:
                dx[first:last] = g_held[first:last] @ w
                dw[e] = _columns(g[first:last]).t() @ _columns(x[first:last])
        first = last
    return (y, dx, dw) if train else y
