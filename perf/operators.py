"""What the operators of a transformer's feed-forward block cost: cases, their plain forms and the calls into ascb200.

  norm         residual addition, root-mean-square norm and an 8-bit output with scales (ascb200_rms_norm)
  norm_grad    its gradients (ascb200_rms_norm_grad)
  linear       matrix product with bias, activation and residual in the epilogue (ascb200_linear)
  linear_grad  its gradients (ascb200_linear_grad)
  route        softmax over experts, top-k, counts per expert and the balance loss (ascb200_route)
  route_grad   its gradients (ascb200_route_grad)
"""
import math
import os
import sys

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "s8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "s8": 1}
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a decode step: latency
        {"name": "norm one token", "op": "norm", "m": 1, "k": 4096, "dtype": "bf16", "q": "fp8", "residual": True, "pad": 0},
        # a prefill batch in front of an int8 matmul of K = 7168, one row short of a round number
        {"name": "norm to int8", "op": "norm", "m": 16383, "k": 7168, "dtype": "bf16", "q": "int8", "residual": True, "pad": 0},
        # ragged rows of a small fp32 model
        {"name": "norm grad ragged", "op": "norm_grad", "m": 1000, "k": 1111, "dtype": "f32", "dh": False, "pad": 1},
        # a training batch
        {"name": "norm grad", "op": "norm_grad", "m": 8192, "k": 4096, "dtype": "bf16", "dh": True, "pad": 0},
        # one token of a decode step through an up projection
        {"name": "linear one token", "op": "linear", "m": 1, "n": 11008, "k": 4096, "dtype": "bf16", "act": "silu", "bias": True, "residual": False, "z": False},
        # the int8 down projection of a prefill batch with its residual
        {"name": "linear int8", "op": "linear", "m": 4096, "n": 4096, "k": 11008, "dtype": "s8", "act": "none", "bias": True, "residual": True, "z": False},
        # a ragged training batch of a narrow layer
        {"name": "linear grad ragged", "op": "linear_grad", "m": 777, "n": 1000, "k": 515, "dtype": "f16", "act": "gelu", "bias": True},
        # a training batch of an up projection
        {"name": "linear grad", "op": "linear_grad", "m": 4096, "n": 11008, "k": 4096, "dtype": "bf16", "act": "silu", "bias": True},
        # one token of a decode step
        {"name": "route one token", "op": "route", "tokens": 1, "experts": 60, "top_k": 4, "dtype": "bf16", "renorm": True, "padding": False},
        # a long prefill over many experts, part of it padding
        {"name": "route", "op": "route", "tokens": 32768, "experts": 256, "top_k": 8, "dtype": "f32", "renorm": True, "padding": True},
        {"name": "route grad ragged", "op": "route_grad", "tokens": 1003, "experts": 72, "top_k": 6, "dtype": "f16", "renorm": False, "padding": True},
        {"name": "route grad", "op": "route_grad", "tokens": 32768, "experts": 256, "top_k": 8, "dtype": "f32", "renorm": True, "padding": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _even(rng, v, step):
    """Half of the sizes are multiples of `step`, as layers mostly are; the others stay as they fell."""
    return max(step, v // step * step) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "linear", "linear_grad", "route", "route_grad"])
    if op in ("norm", "norm_grad"):
        k = _even(rng, _log(rng, 64, 16384), 64)
        m = _log(rng, 1, min(32768, 117_000_000 // k))
        c = {"op": op, "m": m, "k": k, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "pad": rng.choice([0, 0, 8])}
        if op == "norm":
            return c | {"q": rng.choice(["none", "fp8", "int8", "fp8 group", "mx"]), "residual": rng.random() < 0.7}
        return c | {"dh": rng.random() < 0.5}
    if op in ("linear", "linear_grad"):
        n, k = _even(rng, _log(rng, 64, 11008), 64), _even(rng, _log(rng, 64, 11008), 64)
        c = {"op": op, "m": _log(rng, 1, min(4096, 184_000_000_000 // (n * k))), "n": n, "k": k, "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.7}
        if op == "linear_grad":
            return c | {"dtype": rng.choice(["bf16", "f16"])}
        dtype = rng.choice(["bf16", "f16", "s8"])
        return c | {"dtype": dtype, "residual": rng.random() < 0.5, "z": dtype != "s8" and rng.random() < 0.3}
    experts = _log(rng, 8, 512)
    c = {"op": op, "tokens": _log(rng, 1, 8_388_608 // max(256, experts)), "experts": experts, "top_k": rng.randint(1, 8)}
    return c | {"dtype": rng.choice(["f32", "bf16", "f16"]), "renorm": rng.random() < 0.5, "padding": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _rows(rows, cols, dtype, align, gen, scale=1.0):
    """[rows, cols] of normal values; rows start `align` elements apart (0: packed, 1: on 16 bytes)."""
    step = 16 // SIZE[dtype] if align == 1 else align
    ld = -(-cols // step) * step if step else cols
    if dtype == "s8":
        full = torch.randint(-127, 128, (rows, ld), generator=gen, device="cuda", dtype=torch.int8)
    else:
        full = (torch.randn((rows, ld), generator=gen, device="cuda") * scale).to(DTYPE[dtype])
    return full[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    op, dt = case["op"], case["dtype"]
    if op in ("norm", "norm_grad"):
        m, k, pad = case["m"], case["k"], case["pad"]
        s["gamma"] = (1 + 0.1 * randn(k)).to(DTYPE[dt])
        if op == "norm":
            s["x"] = _rows(m, k, dt, pad, gen)
            s["residual"] = _rows(m, k, dt, pad, gen, 2.0) if case["residual"] else None
        else:
            s["h"], s["dy"] = _rows(m, k, dt, pad, gen, 2.0), _rows(m, k, dt, pad, gen)
            s["dh"] = _rows(m, k, dt, pad, gen) if case["dh"] else None
            s["rstd"] = (s["h"].float().square().mean(1) + EPS).rsqrt()  # what the forward pass has left
    elif op in ("linear", "linear_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        out = "bf16" if dt == "s8" else dt
        s["x"], s["w"] = _rows(m, k, dt, 1, gen), _rows(n, k, dt, 1, gen, k**-0.5)
        s["bias"] = randn(n) if case["bias"] else None
        if op == "linear":
            if dt == "s8":
                s["tok"] = torch.rand(m, generator=gen, device="cuda") * 0.02 + 0.01
                s["ch"] = (torch.rand(n, generator=gen, device="cuda") + 0.5) * (k**-0.5 / 100)
            s["residual"] = _rows(m, n, out, 1, gen) if case["residual"] else None
        else:
            s["dy"], s["z"] = _rows(m, n, dt, 1, gen), _rows(m, n, dt, 1, gen)
    else:
        t, e, top = case["tokens"], case["experts"], case["top_k"]
        s["logits"] = (randn(t, e) * 1.5 + randn(e)).to(DTYPE[dt])  # some experts are liked better than others
        s["valid"] = None
        if case["padding"]:
            s["valid"] = (torch.rand(t, generator=gen, device="cuda") < 0.8).to(torch.uint8)
        if op == "route_grad":
            s["idx"], s["weights"], s["counts"], s["num"], _, _ = _route_plain(s["logits"], s["valid"], top, case["renorm"])
            s["dloss"], s["dweights"] = randn(1), randn(t, top)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if act == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608028654 * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        g = 1 / (1 + torch.exp(-z))
        return g * (1 + z * (1 - g))
    return torch.ones_like(z)


def _quantise(y, q, dtype):
    """The 8-bit form of y and its scales. int8 comes back as the values it stands for, in the type of the activations."""
    if q == "mx":
        m, k = y.shape
        blocks = torch.nn.functional.pad(y, (0, -k % 32)).view(m, -1, 32)
        _, e = torch.frexp(blocks.abs().amax(2))
        byte = torch.where(blocks.abs().amax(2) > 0, e - 1 - 8 + 127, torch.zeros_like(e)).clamp(0, 254)
        v = torch.ldexp(blocks, (127 - byte)[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(m, -1)[:, :k]
        return v, byte.to(torch.uint8).view(torch.float8_e8m0fnu)
    top = 127.0 if q == "int8" else 448.0
    if q == "fp8 group":
        m, k = y.shape
        blocks = torch.nn.functional.pad(y, (0, -k % 128)).view(m, -1, 128)
        scale = blocks.abs().amax(2) / top
        v = torch.where(scale[:, :, None] > 0, blocks / scale[:, :, None], torch.zeros_like(blocks))
        return v.clamp(-top, top).to(torch.float8_e4m3fn).view(m, -1)[:, :k], scale
    scale = y.abs().amax(1) / top
    v = torch.where(scale[:, None] > 0, y / scale[:, None], torch.zeros_like(y))
    if q == "int8":
        return (torch.round(v).clamp(-128, 127) * scale[:, None]).to(dtype), scale
    return v.clamp(-top, top).to(torch.float8_e4m3fn), scale


def _norm_plain(s):
    c, dtype = s["case"], s["x"].dtype
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    rstd = torch.rsqrt((h * h).mean(1) + EPS)
    y = h * rstd[:, None] * s["gamma"].float()
    out = {"rstd": rstd}
    if s["residual"] is not None:
        out["sum"] = h.to(dtype)
    if c["q"] == "none":
        out["y"] = y.to(dtype)
    else:
        out["q"], out["scale"] = _quantise(y, c["q"], torch.bfloat16 if dtype == torch.float32 else dtype)
    return out


def _norm_grad_plain(s):
    h, dy, rstd = s["h"].float(), s["dy"].float(), s["rstd"][:, None]
    hat, g = h * rstd, dy * s["gamma"].float()
    dx = rstd * (g - hat * (g * hat).mean(1, keepdim=True))
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return {"dx": dx.to(s["h"].dtype), "dgamma": (dy * hat).sum(0)}


def _linear_plain(s):
    c, x = s["case"], s["x"]
    z = x.float() @ s["w"].float().t()
    if x.dtype == torch.int8:
        z = z * s["ch"] * s["tok"][:, None]
    if s["bias"] is not None:
        z = z + s["bias"]
    y = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = torch.bfloat16 if x.dtype == torch.int8 else x.dtype
    return {"y": y.to(out), "z": z.to(out)} if c["z"] else {"y": y.to(out)}


def _linear_grad_plain(s):
    c, dtype = s["case"], s["x"].dtype
    dz = s["dy"].float() * _act_slope(s["z"].float(), c["act"])
    out = {"dx": (dz @ s["w"].float()).to(dtype), "dw": (dz.t() @ s["x"].float()).to(dtype)}
    if c["bias"]:
        out["dbias"] = dz.sum(0)
    return out


def _route_plain(logits, valid, top_k, renorm):
    x = logits.float()
    t, e = x.shape
    top_k = min(top_k, e)
    open_ = x > -math.inf
    if valid is not None:
        open_ = open_ & (valid != 0)[:, None]
    alive = open_.any(1, keepdim=True)
    x = torch.where(open_, x, torch.full_like(x, -math.inf))
    p = torch.exp(x - torch.where(alive, x.amax(1, keepdim=True), torch.zeros_like(x[:, :1])))
    p = p / torch.where(alive, p.sum(1, keepdim=True), torch.ones_like(p[:, :1]))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_k]
    chosen = torch.gather(open_, 1, order)
    weights = torch.gather(p, 1, order) * chosen
    if renorm:
        weights = weights / torch.where(alive, weights.sum(1, keepdim=True), torch.ones_like(weights[:, :1]))
    counts = torch.zeros(e + 1, dtype=torch.int64, device=x.device)
    counts.scatter_add_(0, torch.where(chosen, order, e).view(-1), torch.ones(t * top_k, dtype=torch.int64, device=x.device))
    num = alive.sum(0)
    n = num.clamp(min=1).float()
    mean = p.sum(0) / n
    loss = (counts[:e] * mean).sum(0, keepdim=True) * (e / (n * top_k))
    return torch.where(chosen, order, -1).to(torch.int32), weights, counts[:e], num, mean, loss


def _route_grad_plain(s):
    x, idx = s["logits"].float(), s["idx"].long()
    t, e = x.shape
    chosen = idx >= 0
    alive = chosen.any(1, keepdim=True)
    p = torch.exp(x - x.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    gw = torch.where(chosen, s["dweights"], torch.zeros_like(s["dweights"]))
    if s["case"]["renorm"]:
        total = (torch.gather(p, 1, idx.clamp(min=0)) * chosen).sum(1, keepdim=True)
        w = torch.gather(p, 1, idx.clamp(min=0)) * chosen / total
        gw = (gw - (gw * w).sum(1, keepdim=True)) / total * chosen
    n = s["num"].clamp(min=1).float()
    dp = (s["dloss"] * e * s["counts"] / (n * n * idx.shape[1])).expand(t, e).clone()
    dp.scatter_add_(1, idx.clamp(min=0), gw)
    d = p * (dp - (p * dp).sum(1, keepdim=True))
    return {"dlogits": torch.where(alive, d, torch.zeros_like(d)).to(s["logits"].dtype)}


def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    if op == "norm":
        return _norm_plain(s)
    if op == "norm_grad":
        return _norm_grad_plain(s)
    if op == "linear":
        return _linear_plain(s)
    if op == "linear_grad":
        return _linear_grad_plain(s)
    if op == "route":
        c = s["case"]
        idx, weights, counts, num, mean, loss = _route_plain(s["logits"], s["valid"], c["top_k"], c["renorm"])
        return {"idx": idx, "weights": weights, "counts": counts, "num": num, "mean": mean, "loss": loss}
    return _route_grad_plain(s)


# ---- the framework's calls -------------------------------------------------------------------------------------------------------
# A program keeps a descriptor for the buffers that it owns, and gives it to the library with a stream, as here: `plan` holds the
# descriptor, the outputs and the workspace, and is made in the first pass over a state.
def _ascb200():
    if "ascb200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "asc-devkit_clone_b200"))
        import ascb200

        ascb200.init(torch.cuda.current_device())
    return sys.modules["ascb200"]


def _dt(ab, tensor):
    return {torch.float32: ab.F32, torch.float16: ab.F16, torch.bfloat16: ab.BF16, torch.int8: ab.S8}[tensor.dtype]


def _ptr(tensor):
    return None if tensor is None else tensor.data_ptr()


def _ld(tensor):
    return 0 if tensor is None else tensor.stride(0)


def _norm_own(s):
    ab, c, x, r = _ascb200(), s["case"], s["x"], s["residual"]
    if "plan" not in s:
        m, k, q = c["m"], c["k"], c["q"]
        out = {"rstd": torch.empty(m, device="cuda")}
        if r is not None:
            out["sum"] = torch.empty(m, k, device="cuda", dtype=x.dtype)
        if q == "none":
            out["y"] = torch.empty(m, k, device="cuda", dtype=x.dtype)
            codes = None
        else:
            codes = torch.empty(m, k, device="cuda", dtype=torch.int8 if q == "int8" else torch.float8_e4m3fn)
            groups = {"fp8 group": (m, -(-k // 128)), "mx": (m, -(-k // 32))}.get(q, (m,))
            out["scale"] = torch.empty(groups, device="cuda", dtype=torch.float8_e8m0fnu if q == "mx" else torch.float32)
            out["q"] = codes if q != "int8" else torch.empty(m, k, device="cuda", dtype=torch.bfloat16 if x.dtype == torch.float32 else x.dtype)
        d = ab.RmsNormDesc(m=m, k=k, dtype=_dt(ab, x), x_dev=_ptr(x), ldx=_ld(x), residual_dev=_ptr(r), ld_residual=_ld(r), gamma_dev=_ptr(s["gamma"]),
                           gamma_dtype=_dt(ab, s["gamma"]), eps=EPS, sum_dev=_ptr(out.get("sum")), y_dev=_ptr(out.get("y")), rstd_dev=_ptr(out["rstd"]))
        if codes is not None:
            d.q_dev, d.scale_dev, d.q_dtype = _ptr(codes), _ptr(out["scale"]), ab.S8 if q == "int8" else ab.FP8_E4M3
            d.scale_mode = {"fp8 group": ab.SCALE_PER_GROUP, "mx": ab.SCALE_MX}.get(q, ab.SCALE_PER_TOKEN)
            d.group_size = 128 if q == "fp8 group" else 0
        s["plan"] = (d, out, codes)
    d, out, codes = s["plan"]
    ab.check(ab.rms_norm(d, torch.cuda.current_stream().cuda_stream))
    if c["q"] == "int8":  # the values that the int8 codes stand for
        torch.mul(codes, out["scale"][:, None], out=out["q"])
    return out


def _norm_grad_own(s):
    ab, c, h = _ascb200(), s["case"], s["h"]
    if "plan" not in s:
        m, k = c["m"], c["k"]
        out = {"dx": torch.empty(m, k, device="cuda", dtype=h.dtype), "dgamma": torch.empty(k, device="cuda")}
        room = torch.empty(ab.rms_norm_grad_workspace_bytes(m, k), device="cuda", dtype=torch.uint8)
        d = ab.RmsNormGradDesc(m=m, k=k, dtype=_dt(ab, h), dy_dev=_ptr(s["dy"]), ld_dy=_ld(s["dy"]), h_dev=_ptr(h), ldh=_ld(h), rstd_dev=_ptr(s["rstd"]),
                               gamma_dev=_ptr(s["gamma"]), gamma_dtype=_dt(ab, s["gamma"]), dh_dev=_ptr(s["dh"]), ld_dh=_ld(s["dh"]),
                               dx_dev=_ptr(out["dx"]), dgamma_dev=_ptr(out["dgamma"]), dgamma_dtype=ab.F32, workspace_dev=_ptr(room),
                               workspace_bytes=room.numel())
        s["plan"] = (d, out, room)
    d, out, _ = s["plan"]
    ab.check(ab.rms_norm_grad(d, torch.cuda.current_stream().cuda_stream))
    return out


def _kind(ab, tensor):
    return {torch.float16: ab.KIND_F16, torch.bfloat16: ab.KIND_BF16, torch.int8: ab.KIND_S8}[tensor.dtype]


def _act_code(ab, act):
    return {"none": ab.ACT_NONE, "relu": ab.ACT_RELU, "gelu": ab.ACT_GELU, "gelu_tanh": ab.ACT_GELU_TANH, "silu": ab.ACT_SILU}[act]


def _linear_own(s):
    ab, c, x, w, r = _ascb200(), s["case"], s["x"], s["w"], s["residual"]
    if "plan" not in s:
        m, n = c["m"], c["n"]
        dtype = torch.bfloat16 if x.dtype == torch.int8 else x.dtype
        out = {"y": torch.empty(m, n, device="cuda", dtype=dtype)}
        if c["z"]:
            out["z"] = torch.empty(m, n, device="cuda", dtype=dtype)
        d = ab.LinearDesc(kind=_kind(ab, x), m=m, n=n, k=c["k"], x_dev=_ptr(x), ldx=_ld(x), w_dev=_ptr(w), ldw=_ld(w), trans_w=1, tok_scale_dev=_ptr(s.get("tok")),
                          ch_scale_dev=_ptr(s.get("ch")), bias_dev=_ptr(s["bias"]), bias_dtype=ab.F32, act=_act_code(ab, c["act"]), residual_dev=_ptr(r),
                          ld_residual=_ld(r), y_dev=_ptr(out["y"]), y_dtype=_dt(ab, out["y"]), z_dev=_ptr(out.get("z")))
        s["plan"] = (d, out)
    d, out = s["plan"]
    ab.check(ab.linear(d, torch.cuda.current_stream().cuda_stream))
    return out


def _linear_grad_own(s):
    ab, c, x, w = _ascb200(), s["case"], s["x"], s["w"]
    if "plan" not in s:
        m, n, k = c["m"], c["n"], c["k"]
        out = {"dx": torch.empty(m, k, device="cuda", dtype=x.dtype), "dw": torch.empty(n, k, device="cuda", dtype=x.dtype)}
        if c["bias"]:
            out["dbias"] = torch.empty(n, device="cuda")
        room = torch.empty(ab.linear_grad_workspace_bytes(m, n), device="cuda", dtype=torch.uint8)
        d = ab.LinearGradDesc(kind=_kind(ab, x), m=m, n=n, k=k, act=_act_code(ab, c["act"]), dy_dev=_ptr(s["dy"]), ld_dy=_ld(s["dy"]), z_dev=_ptr(s["z"]),
                              ldz=_ld(s["z"]), x_dev=_ptr(x), ldx=_ld(x), w_dev=_ptr(w), ldw=_ld(w), trans_w=1, dx_dev=_ptr(out["dx"]), dw_dev=_ptr(out["dw"]),
                              dw_dtype=_dt(ab, out["dw"]), dbias_dev=_ptr(out.get("dbias")), workspace_dev=_ptr(room), workspace_bytes=room.numel())
        s["plan"] = (d, out, room)
    d, out, _ = s["plan"]
    ab.check(ab.linear_grad(d, torch.cuda.current_stream().cuda_stream))
    return out


def _route_own(s):
    ab, c, x = _ascb200(), s["case"], s["logits"]
    if "plan" not in s:
        t, e, top = c["tokens"], c["experts"], min(c["top_k"], c["experts"])
        out = {"idx": torch.empty(t, top, device="cuda", dtype=torch.int32), "weights": torch.empty(t, top, device="cuda"),
               "counts": torch.empty(e, device="cuda", dtype=torch.int64), "num": torch.empty(1, device="cuda", dtype=torch.int64),
               "mean": torch.empty(e, device="cuda"), "loss": torch.empty(1, device="cuda")}
        room = torch.empty(ab.route_workspace_bytes(t, e), device="cuda", dtype=torch.uint8)
        d = ab.RouteDesc(tokens=t, experts=e, top_k=top, dtype=_dt(ab, x), renorm=c["renorm"], logits_dev=_ptr(x), ld_logits=_ld(x), valid_dev=_ptr(s["valid"]),
                         idx_dev=_ptr(out["idx"]), weights_dev=_ptr(out["weights"]), counts_dev=_ptr(out["counts"]), num_tokens_dev=_ptr(out["num"]),
                         prob_mean_dev=_ptr(out["mean"]), loss_dev=_ptr(out["loss"]), workspace_dev=_ptr(room), workspace_bytes=room.numel())
        s["plan"] = (d, out, room)
    d, out, _ = s["plan"]
    ab.check(ab.route(d, torch.cuda.current_stream().cuda_stream))
    return out


def _route_grad_own(s):
    ab, c, x = _ascb200(), s["case"], s["logits"]
    if "plan" not in s:
        out = {"dlogits": torch.empty(x.shape, device="cuda", dtype=x.dtype)}
        d = ab.RouteGradDesc(tokens=c["tokens"], experts=c["experts"], top_k=s["idx"].shape[1], dtype=_dt(ab, x), renorm=c["renorm"], logits_dev=_ptr(x),
                             ld_logits=_ld(x), idx_dev=_ptr(s["idx"]), counts_dev=_ptr(s["counts"]), num_tokens_dev=_ptr(s["num"]), dloss_dev=_ptr(s["dloss"]),
                             dweights_dev=_ptr(s["dweights"]), dlogits_dev=_ptr(out["dlogits"]))
        s["plan"] = (d, out)
    d, out = s["plan"]
    ab.check(ab.route_grad(d, torch.cuda.current_stream().cuda_stream))
    return out


_OWN = {"norm": _norm_own, "norm_grad": _norm_grad_own, "linear": _linear_own, "linear_grad": _linear_grad_own, "route": _route_own, "route_grad": _route_grad_own}


# ---- the work that a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    op, b = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        m, k, q = case["m"], case["k"], case["q"]
        scales = {"none": 0, "fp8 group": 4 * -(-k // 128), "mx": -(-k // 32)}.get(q, 4)
        return {"bytes": m * (k * (b * (3 if case["residual"] else 1) + (b if q == "none" else 1)) + scales + 4) + k * b, "flops": 6 * m * k}
    if op == "norm_grad":
        m, k = case["m"], case["k"]
        return {"bytes": m * (k * b * (4 if case["dh"] else 3) + 4) + k * (b + 4), "flops": 10 * m * k}
    if op == "linear":
        m, n, k, o = case["m"], case["n"], case["k"], 2
        outs = 1 + (1 if case["residual"] else 0) + (1 if case["z"] else 0)
        return {"bytes": (m + n) * k * b + m * n * o * outs + (4 * n if case["bias"] else 0) + (4 * (m + n) if case["dtype"] == "s8" else 0), "flops": 2 * m * n * k}
    if op == "linear_grad":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * b * (m + n) * k + 2 * b * m * n + (4 * n if case["bias"] else 0), "flops": 4 * m * n * k}
    t, e, top = case["tokens"], case["experts"], min(case["top_k"], case["experts"])
    if op == "route":
        return {"bytes": t * (e * b + top * 8 + (1 if case["padding"] else 0)) + 12 * e + 12, "flops": 8 * t * e}
    return {"bytes": t * (2 * e * b + top * 8) + 8 * e, "flops": 10 * t * e}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.dtype != torch.uint8 else v for k, v in s.items()}
    return _EXACT[case["op"]](case, d)


def _norm_exact(c, d):
    h = d["x"] if d["residual"] is None else d["x"] + d["residual"]
    root = torch.sqrt(h.pow(2).sum(1) / c["k"] + EPS)
    y = h / root.unsqueeze(1) * d["gamma"]
    out = {"rstd": root.reciprocal(), "sum": None if d["residual"] is None else h}
    if d["residual"] is None:
        del out["sum"]
    if c["q"] == "none":
        return out | {"y": y}
    width = {"fp8 group": 128, "mx": 32}.get(c["q"], c["k"])
    count = -(-c["k"] // width)
    wide = torch.zeros(c["m"], count * width, dtype=torch.float64, device=y.device)
    wide[:, : c["k"]] = y
    wide = wide.reshape(c["m"], count, width)
    largest = wide.abs().max(2).values
    if c["q"] == "mx":
        scale = torch.exp2(torch.floor(torch.log2(largest.clamp(min=1e-300))) - 8).clamp(min=2.0**-127)
    else:
        scale = largest / (127 if c["q"] == "int8" else 448)
    v = wide / scale.clamp(min=1e-300).unsqueeze(2)
    if c["q"] == "int8":
        v = v.round().clamp(-128, 127) * scale.unsqueeze(2)
    else:  # e4m3: four significant bits, the smallest step 2^-9
        _, e = torch.frexp(v)
        step = torch.exp2((e - 4).clamp(min=-9).double())
        v = (torch.round(v / step) * step).clamp(-448, 448)
    v = v.reshape(c["m"], -1)[:, : c["k"]]
    return out | {"q": v, "scale": scale if c["q"] in ("fp8 group", "mx") else scale[:, 0]}


def _norm_grad_exact(c, d):
    # x -> y = x / sqrt(mean x^2 + eps) * gamma, differentiated: d y_i / d x_j = gamma_i (delta_ij r - x_i x_j r^3 / k), r the saved 1 / root
    r = d["rstd"].unsqueeze(1)
    u = d["dy"] * d["gamma"]
    dx = u * r - d["h"] * (u * d["h"]).sum(1, keepdim=True) * r**3 / c["k"]
    return {"dx": dx if d["dh"] is None else dx + d["dh"], "dgamma": torch.einsum("mk,mk->k", d["dy"] * r, d["h"])}


def _act_exact(z, act):
    """(value, slope) of the activation."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, g + z * g * (1 - g)
    if act == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    g = torch.sigmoid(2 * c * (z + 0.044715 * z**3))
    return z * g, g + z * g * (1 - g) * 2 * c * (1 + 0.134145 * z**2)


def _linear_exact(c, d):
    z = torch.matmul(d["x"], d["w"].transpose(0, 1))
    if c["dtype"] == "s8":
        z = z * torch.outer(d["tok"], d["ch"])
    if d["bias"] is not None:
        z = z + d["bias"]
    y = _act_exact(z, c["act"])[0]
    if d["residual"] is not None:
        y = y + d["residual"]
    return {"y": y, "z": z} if c["z"] else {"y": y}


def _linear_grad_exact(c, d):
    dz = d["dy"] * _act_exact(d["z"], c["act"])[1]
    out = {"dx": torch.matmul(dz, d["w"]), "dw": torch.matmul(dz.transpose(0, 1), d["x"])}
    return out | {"dbias": dz.sum(0)} if c["bias"] else out


def _softmax_exact(x, alive):
    return torch.where(alive, torch.softmax(torch.where(alive, x, torch.zeros_like(x)), 1), torch.zeros_like(x))


def _route_exact(c, d):
    x = d["logits"]
    top = min(c["top_k"], c["experts"])
    alive = torch.ones_like(x[:, :1], dtype=torch.bool) if d["valid"] is None else d["valid"].bool().unsqueeze(1)
    p = _softmax_exact(x, alive)
    # the k-th choice: the largest left, and of equal ones the first
    left, idx, w = x.clone(), [], []
    for _ in range(top):
        first = (left == left.max(1, keepdim=True).values).int().argmax(1, keepdim=True)
        idx.append(first)
        w.append(p.gather(1, first))
        left.scatter_(1, first, -math.inf)
    idx, w = torch.cat(idx, 1), torch.cat(w, 1)
    if c["renorm"]:
        w = torch.where(alive, w / w.sum(1, keepdim=True).clamp(min=1e-300), torch.zeros_like(w))
    n = int(alive.sum())
    counts = torch.bincount(idx[alive.expand_as(idx)], minlength=c["experts"])
    mean = p.sum(0) / max(n, 1)
    loss = (counts * mean).sum().reshape(1) * c["experts"] / (max(n, 1) * top)
    return {"idx": torch.where(alive, idx, -1).int(), "weights": w, "counts": counts, "num": torch.tensor([n]), "mean": mean, "loss": loss}


def _route_grad_exact(c, d):
    x, idx = d["logits"], d["idx"].long()
    alive = idx[:, :1] >= 0
    p = _softmax_exact(x, alive)
    n = max(float(d["num"]), 1.0)
    seen = torch.zeros_like(x).scatter_(1, idx.clamp(min=0), 1.0) * alive
    given = torch.zeros_like(x).scatter_(1, idx.clamp(min=0), d["dweights"]) * alive
    if c["renorm"]:
        total = torch.where(alive, (p * seen).sum(1, keepdim=True), torch.ones_like(p[:, :1]))
        given = seen * (given / total - (given * p).sum(1, keepdim=True) / total**2)
    dp = given + d["dloss"] * c["experts"] / (n * n * idx.shape[1]) * d["counts"]
    return {"dlogits": p * dp - p * (p * dp).sum(1, keepdim=True)}


_EXACT = {"norm": _norm_exact, "norm_grad": _norm_grad_exact, "linear": _linear_exact, "linear_grad": _linear_grad_exact, "route": _route_exact,
          "route_grad": _route_grad_exact}
