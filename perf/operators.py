"""The operators of the 8-bit integer path of a decoder block, as cases that can be timed and compared: the per-token
cast, the matrix product with scales per token and channel, its gated form for a gate_up projection, and the norms
before and after a block with its gate and residual scale, with their gradients.

With ``own`` false, `run` computes them from elementary torch operations in 32 bits; with ``own`` true it calls
this package.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
LARGEST = 4096 * 28672 * 8192  # multiply-adds of the largest listed product
ROWS = 8192 * 8192              # elements of the largest drawn row-wise case
EPS = 1e-6


def listed():
    return [
        # One decode token through an attention output projection: the smallest product, nearly all latency.
        _product("matmul_m1_4096", 1, 4096, 4096, "float16"),
        # A ragged batch whose sizes fill no tile evenly.
        _product("matmul_m100_11008x4224", 100, 11008, 4224, "bfloat16"),
        # Prompt processing with one row more than whole tiles, with biases.
        _product("matmul_m4097_12288_bias", 4097, 12288, 4096, "bfloat16", bias=True),
        # gate_up of a decode batch of 8.
        _product("gate_up_m8_28672", 8, 28672, 4096, "float16", gated=True),
        # The largest: prefill through a 70B-class gate_up projection, clamped as the cast behind gate_up may be.
        _product("gate_up_m4096_28672x8192", 4096, 28672, 8192, "bfloat16", gated=True, clamp=6.0),
        # The activations of one decode token, cast: the smallest call of all.
        dict(name="cast_t1_4096", op="cast", t=1, d=4096, act="float16"),
        # The activations in front of a down projection at prefill.
        dict(name="cast_t4097_14336", op="cast", t=4097, d=14336, act="bfloat16"),
        # The feed-forward block of a decode step of 64 sequences: norm and cast, gate_up, cast, down.
        _norm("ffn_t64_4096x14336", "ffn", 64, 4096, "bfloat16", post=True, n=14336),
        # Between two blocks of a decode step of 8 sequences, in front of an attention block: norm and cast, then QKV.
        _norm("norm_matmul_t8_4096x6144", "norm_matmul", 8, 4096, "float16", post=True, gates=1, n=6144),
        # Between two blocks at prefill, with a gate per channel, and the residual stream in 32 bits.
        _norm("norm_t4097_8192_f32", "norm", 4097, 8192, "bfloat16", residual="float32", gates=1, scale=0.7),
        # Training on one short sequence.
        _norm("norm_backward_t511_4096", "backward", 511, 4096, "bfloat16", post=True, gates=1),
        # Training on a batch of eight sequences, each with a gate of its own.
        _norm("norm_backward_t8192_5120", "backward", 8192, 5120, "bfloat16", residual="float32", post=True, gates=8,
              scale=0.9),
    ]


def _product(name, m, n, k, act, bias=False, gated=False, clamp=None):
    return dict(name=name, op="gate_up" if gated else "matmul", m=m, n=n, k=k, act=act, bias=bias, clamp=clamp)


def _norm(name, op, t, d, act, residual=None, post=False, gates=0, scale=1.0, n=0):
    """`n`: outputs of the projection behind the norm ("norm_matmul"), or channels of the feed-forward block ("ffn")."""
    return dict(name=name, op=op, t=t, d=d, act=act, residual=residual or act, post=post, gates=gates, scale=scale, n=n)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matmul", "matmul", "gate_up", "cast", "norm", "norm_matmul", "ffn", "backward", "backward"])
    act = rng.choice(["float16", "bfloat16"])
    if op in ("matmul", "gate_up"):
        step = 32 if op == "gate_up" else 16
        m = _log_int(rng, 1, 8192)
        n = step * max(1, _log_int(rng, 256, 28672) // step)
        k = 16 * (_log_int(rng, 256, 14336) // 16)
        m = min(m, max(1, LARGEST // (n * k)))
        case = _product("", m, n, k, act, bias=op == "matmul" and rng.random() < 0.5, gated=op == "gate_up",
                        clamp=6.0 if op == "gate_up" and rng.random() < 0.5 else None)
    else:
        d = 8 * (_log_int(rng, 256, 16384) // 8)
        t = min(_log_int(rng, 1, 16384), ROWS // d)
        if op == "cast":
            return dict(op="cast", t=t, d=d, act=act)
        n = 0
        if op in ("norm_matmul", "ffn"):
            d = 16 * (_log_int(rng, 256, 8192) // 16)
            n = 16 * (_log_int(rng, 256, 16384) // 16)
            t = min(_log_int(rng, 1, 4096), max(1, LARGEST // (3 * n * d)))
        gates = rng.choice([0, 1, 1, rng.randint(2, 8)])
        if gates > 1:
            t = gates * max(1, t // gates)
        case = _norm("", op, t, d, act, residual=rng.choice([act, "float32"]), post=rng.random() < 0.6, gates=gates,
                     scale=rng.choice([1.0, round(rng.uniform(0.5, 1.0), 3)]), n=n)
    case.pop("name")
    return case


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _weights(gen, n, k):
    """8-bit weights and the scales of their channels: outputs near one for activations near one."""
    codes = torch.randint(-127, 128, (n, k), generator=gen, device=DEVICE, dtype=torch.int8)
    return codes, (0.5 + torch.rand(n, generator=gen, device=DEVICE)) / (73.0 * math.sqrt(k))


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["act"]]
    if case["op"] in ("matmul", "gate_up"):
        m, n, k = case["m"], case["n"], case["k"]
        # codes of normally distributed values, cast by their largest magnitude (about four deviations)
        a = (_normal(gen, m, k) * 31.0).round_().clamp_(-127, 127).to(torch.int8)
        a_sf = (1.0 + 0.5 * torch.rand(m, generator=gen, device=DEVICE)) / 31.0
        b, b_sf = _weights(gen, n, k)
        bias = _normal(gen, n).to(dtype) if case["bias"] else None
        return dict(case=case, dtype=dtype, a=a, b=b, a_sf=a_sf, b_sf=b_sf, bias=bias)
    t, d = case["t"], case["d"]
    block = _normal(gen, t, d)
    block[:, :: max(1, d // 16)] *= 8.0  # a few channels far larger than the others, as activations have them
    block = block.to(dtype)
    if case["op"] == "cast":
        return dict(case=case, dtype=dtype, x=block)
    s = dict(case=case, dtype=dtype, block=block, residual=(_normal(gen, t, d) * 3.0).to(DTYPES[case["residual"]]),
             weight=(1.0 + 0.2 * _normal(gen, d)).to(dtype),
             post=(1.0 + 0.2 * _normal(gen, d)).to(dtype) if case["post"] else None, gate=None)
    if case["gates"]:
        shape = (d,) if case["gates"] == 1 else (case["gates"], d)
        s["gate"] = (0.5 + 0.3 * _normal(gen, *shape)).to(dtype)
    if case["op"] == "backward":
        s["grad_x"] = _normal(gen, t, d).to(dtype)
        s["grad_residual"] = _normal(gen, t, d).to(DTYPES[case["residual"]])
    if case["op"] == "norm_matmul":
        s["w"], s["w_sf"] = _weights(gen, case["n"], d)
    if case["op"] == "ffn":
        s["w"], s["w_sf"] = _weights(gen, 2 * case["n"], d)
        s["down"], s["down_sf"] = _weights(gen, d, case["n"])
    return s


# ---- the operators from elementary operations ---------------------------------------------------------
def _cast(x):
    """Codes (as 32-bit floats) and scales: quotients and products rounded once each, codes to the nearest even."""
    x = x.float()
    top = x.abs().amax(1)
    top127 = torch.full_like(top, 127.0)  # (a tensor: a division by a number would multiply by its reciprocal)
    return (x * (top127 / top)[:, None]).round(), top / top127


def _product_of(a, b, a_sf, b_sf):
    return (a.float() @ b.float().t()) * a_sf[:, None] * b_sf


def _silu_product(c, clamp):
    h = c.shape[1] // 2
    g, u = c[:, :h], c[:, h:]
    if clamp is not None:
        g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
    return g / (1.0 + torch.exp(-g)) * u


def _block_norm(s):
    """x and the new residual, in 32 bits."""
    case = s["case"]
    n = s["block"].float()
    t, d = n.shape
    if s["post"] is not None:
        n = n * torch.rsqrt(n.square().mean(1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        n = (n.view(case["gates"], -1, d) * s["gate"].float().view(-1, 1, d)).view(t, d)
    r = case["scale"] * s["residual"].float() + n
    return r * torch.rsqrt(r.square().mean(1, keepdim=True) + EPS) * s["weight"].float(), r


def _block_norm_backward(s):
    case = s["case"]
    block, dx = s["block"].float(), s["grad_x"].float()
    t, d = block.shape
    groups = max(1, case["gates"])
    gate = s["gate"].float().view(-1, 1, d) if s["gate"] is not None else torch.ones(1, 1, d, device=block.device)
    hat, post = block, None
    if s["post"] is not None:
        inverse = torch.rsqrt(block.square().mean(1, keepdim=True) + EPS)
        hat, post = block * inverse, s["post"].float()
    n = hat if post is None else hat * post
    r = case["scale"] * s["residual"].float() + (n.view(groups, -1, d) * gate).view(t, d)
    inverse2 = torch.rsqrt(r.square().mean(1, keepdim=True) + EPS)
    xhat = r * inverse2
    e = dx * s["weight"].float()
    dr = s["grad_residual"].float() + inverse2 * (e - xhat * (e * xhat).mean(1, keepdim=True))
    dn = (dr.view(groups, -1, d) * gate).view(t, d)
    out = {"weight": (dx * xhat).sum(0), "residual": (case["scale"] * dr).to(s["residual"].dtype)}
    if s["gate"] is not None:
        out["gate"] = (dr * n).view(groups, -1, d).sum(1).view(s["gate"].shape)
    if post is not None:
        out["post"] = (dn * hat).sum(0)
        f = dn * post
        dn = inverse * (f - hat * (f * hat).mean(1, keepdim=True))
    out["block"] = dn.to(s["dtype"])
    return out


def run(state):
    if own:
        return _run_own(state)
    s, op, dtype = state, state["case"]["op"], state["dtype"]
    if op == "matmul":
        c = _product_of(s["a"], s["b"], s["a_sf"], s["b_sf"])
        return (c + s["bias"].float() if s["bias"] is not None else c).to(dtype)
    if op == "gate_up":
        return _silu_product(_product_of(s["a"], s["b"], s["a_sf"], s["b_sf"]), s["case"]["clamp"]).to(dtype)
    if op == "cast":
        codes, sf = _cast(s["x"])
        return {"codes": codes.to(torch.int8), "sf": sf}
    if op == "backward":
        return _block_norm_backward(s)
    x, r = _block_norm(s)
    x, r = x.to(dtype), r.to(s["residual"].dtype)
    if op == "norm":
        return {"x": x, "residual": r}
    x, sf = _cast(x)
    c = _product_of(x, s["w"], sf, s["w_sf"])
    if op == "ffn":
        h, h_sf = _cast(_silu_product(c, None).to(dtype))
        c = _product_of(h, s["down"], h_sf, s["down_sf"])
    return {"c": c.to(dtype), "residual": r}


def _run_own(s):
    from tilus_b200 import ops

    case, dtype = s["case"], s["dtype"]
    op = case["op"]
    if op == "matmul":
        return ops.int8_matmul(s["a"], s["b"], s["a_sf"], s["b_sf"], bias=s["bias"], out_dtype=dtype)
    if op == "gate_up":
        return ops.int8_gate_up(s["a"], s["b"], s["a_sf"], s["b_sf"], out_dtype=dtype, swiglu_clamp_value=case["clamp"])
    if op == "cast":
        codes, sf = ops.per_token_cast_int8(s["x"])
        return {"codes": codes, "sf": sf}
    args = dict(post_weight=s["post"], gate=s["gate"], residual_scale=case["scale"], eps=EPS)
    if op == "backward":
        got = ops.block_norm_backward(s["grad_x"], s["grad_residual"], s["block"], s["residual"], s["weight"], **args)
        return {k: v for k, v in zip(("block", "residual", "weight", "post", "gate"), got) if v is not None}
    if op == "norm":
        x, r = ops.block_norm(s["block"], s["residual"], s["weight"], **args)
        return {"x": x, "residual": r}
    x, sf, r = ops.block_norm_cast_int8(s["block"], s["residual"], s["weight"], **args)
    if op == "ffn":
        h, h_sf = ops.per_token_cast_int8(ops.int8_gate_up(x, s["w"], sf, s["w_sf"], out_dtype=dtype))
        return {"c": ops.int8_matmul(h, s["down"], h_sf, s["down_sf"], out_dtype=dtype), "residual": r}
    return {"c": ops.int8_matmul(x, s["w"], sf, s["w_sf"], out_dtype=dtype), "residual": r}


# ---- what a pass cannot do without ---------------------------------------------------------------------
def _product_work(m, n, k, outputs, in_bytes=None):
    """`in_bytes`: of the activations, where they are not an 8-bit matrix with its scales that the pass is given."""
    return {"bytes": n * k + 4 * n + (m * k + 4 * m if in_bytes is None else in_bytes) + 2 * m * outputs, "flops": 2 * m * n * k}


def work(case):
    op = case["op"]
    if op in ("matmul", "gate_up"):
        m, n, k = case["m"], case["n"], case["k"]
        w = _product_work(m, n, k, n // 2 if op == "gate_up" else n)
        w["bytes"] += 2 * n if case["bias"] else 0
        return w
    t, d, n = case["t"], case["d"], case["n"] if "n" in case else 0
    if op == "cast":
        return {"bytes": 3 * t * d + 4 * t, "flops": 3 * t * d}
    rb = 4 if case["residual"] == "float32" else 2
    channels = 2 * d * (1 + case["post"] + case["gates"])
    if op == "backward":
        return {"bytes": t * d * (2 + 2 + rb + rb + 2 + rb) + 3 * channels, "flops": 40 * t * d}
    w = {"bytes": t * d * (2 + 2 * rb + (2 if op == "norm" else 0)) + channels, "flops": 15 * t * d}
    if op == "norm":
        return w
    products = [_product_work(t, n, d, n, 0)] if op == "norm_matmul" else [_product_work(t, 2 * n, d, 0, 0), _product_work(t, d, n, d, 0)]
    return {k: w[k] + sum(p[k] for p in products) for k in w}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64

    def quantized(x):
        # x holds 16-bit values.  The scale and its inverse are 32-bit numbers by definition, and so is the product that is rounded.
        x = x.to(f64)
        m = x.abs().max(dim=1, keepdim=True).values
        sf = torch.div(m, 127.0).to(torch.float32).to(f64)
        inverse = torch.div(127.0, m).to(torch.float32).to(f64)
        return torch.round(torch.mul(x, inverse).to(torch.float32).to(f64)), sf

    def dot(q, q_sf, w, w_sf):
        return torch.mm(q.to(f64), w.to(f64).T) * (q_sf.to(f64).reshape(-1, 1) * w_sf.to(f64).reshape(1, -1))

    def swiglu(c, limit):
        left, right = torch.chunk(c, 2, dim=1)
        if limit is not None:
            left = torch.minimum(left, torch.full_like(left, limit))
            right = torch.maximum(torch.minimum(right, torch.full_like(right, limit)), torch.full_like(right, -limit))
        return left * torch.sigmoid(left) * right

    op = case["op"]
    if op in ("matmul", "gate_up"):
        c = dot(s["a"], s["a_sf"], s["b"], s["b_sf"])
        if op == "gate_up":
            return swiglu(c, case["clamp"])
        return c if s["bias"] is None else c + s["bias"].to(f64)
    if op == "cast":
        codes, sf = quantized(s["x"])
        return {"codes": codes.to(torch.int8), "sf": sf[:, 0]}
    names = ["block", "residual", "weight"] + [k for k in ("post", "gate") if s[k] is not None]
    v = {k: s[k].to(f64).requires_grad_(op == "backward") for k in names}

    def norm(y, w):
        return w * y / torch.sqrt((y * y).sum(dim=1, keepdim=True) / y.shape[1] + EPS)

    branch = norm(v["block"], v["post"]) if "post" in v else v["block"]
    if "gate" in v:
        rows = v["gate"].reshape(-1, case["d"])
        branch = branch * rows.repeat_interleave(case["t"] // rows.shape[0], dim=0)
    new = v["residual"] * case["scale"] + branch
    x = norm(new, v["weight"])
    if op == "backward":
        grads = torch.autograd.grad([x, new], [v[k] for k in names], [s["grad_x"].to(f64), s["grad_residual"].to(f64)])
        return dict(zip(names, grads))
    if op == "norm":
        return {"x": x, "residual": new}
    codes, sf = quantized(x.to(s["dtype"]))
    c = dot(codes, sf, s["w"], s["w_sf"])
    if op == "ffn":
        codes, sf = quantized(swiglu(c, None).to(s["dtype"]))
        c = dot(codes, sf, s["down"], s["down_sf"])
    return {"c": c, "residual": new}
