"""The feed-forward operators together, as a model's layers use them."""
import ctypes as C

import pytest
import torch

import ascb200 as ab
from test_gpu_linear import act
from torch_util import CODE, HALF_STEP, Out, dev, near, ptr, stream

pytestmark = pytest.mark.gpu
EPS = 1e-6


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rel(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm())


def room_for(size):
    return torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("m", [1, 7, 300])
def test_int8_block(m):
    """residual + norm -> int8 up projection with GELU -> norm -> int8 down projection with bias and the residual added, one graph."""
    dev()
    k, n = 512, 1360
    g = gen(m)
    x, r = torch.randn(m, k, generator=g, device="cuda").bfloat16(), torch.randn(m, k, generator=g, device="cuda").bfloat16()
    g1, g2 = (1 + 0.1 * torch.randn(c, generator=g, device="cuda") for c in (k, n))
    w1, w2 = (torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8) for s in ((n, k), (k, n)))
    c1, c2 = (torch.rand(c, generator=g, device="cuda") * 0.001 + 0.0005 for c in (n, k))
    bias = torch.randn(k, generator=g, device="cuda")
    h, q1, s1 = torch.empty_like(x), torch.empty(m, k, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    u, q2, s2, y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda"), torch.empty(m, n, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda"), torch.empty_like(x)
    side = C.c_void_p()
    ab.check(ab.lib().ascb200_stream_create(C.byref(side)))
    calls = [
        (ab.rms_norm, ab.RmsNormDesc(m=m, k=k, dtype=ab.BF16, x_dev=ptr(x), residual_dev=ptr(r), gamma_dev=ptr(g1), gamma_dtype=ab.F32, sum_dev=ptr(h), q_dev=ptr(q1), q_dtype=ab.S8,
                                     scale_dev=ptr(s1), eps=EPS)),
        (ab.linear, ab.LinearDesc(kind=ab.KIND_S8, m=m, n=n, k=k, x_dev=ptr(q1), w_dev=ptr(w1), trans_w=1, tok_scale_dev=ptr(s1), ch_scale_dev=ptr(c1), act=ab.ACT_GELU, y_dev=ptr(u),
                                  y_dtype=ab.BF16)),
        (ab.rms_norm, ab.RmsNormDesc(m=m, k=n, dtype=ab.BF16, x_dev=ptr(u), gamma_dev=ptr(g2), gamma_dtype=ab.F32, q_dev=ptr(q2), q_dtype=ab.S8, scale_dev=ptr(s2), eps=EPS)),
        (ab.linear, ab.LinearDesc(kind=ab.KIND_S8, m=m, n=k, k=n, x_dev=ptr(q2), w_dev=ptr(w2), trans_w=1, tok_scale_dev=ptr(s2), ch_scale_dev=ptr(c2), bias_dev=ptr(bias), residual_dev=ptr(h),
                                  y_dev=ptr(y), y_dtype=ab.BF16)),
    ]
    torch.cuda.synchronize()
    graph = ab.Graph(side, lambda: [ab.check(f(d, side)) for f, d in calls])
    for _ in range(2):
        graph.launch()
    torch.cuda.synchronize()
    # in 64 bits without any rounding between: an int8 value is off by half a step of max / 127, about 1.3 % of a row's rms with normal
    # values (max about 4 rms, rms of the error 1 / sqrt(12) steps); two such roundings and four of bf16 (0.2 % rms each)
    hd = x.double() + r.double()
    n1 = hd / torch.sqrt((hd * hd).mean(1, keepdim=True) + EPS) * g1.double()
    ud = act(n1 @ (w1.double() * c1.double()[:, None]).t(), "gelu")[0]
    n2 = ud / torch.sqrt((ud * ud).mean(1, keepdim=True) + EPS) * g2.double()
    yd = n2 @ (w2.double() * c2.double()[:, None]).t() + bias.double() + hd
    assert rel(h, hd) < 2.0**-8
    assert rel(u, ud) < 0.03 and rel(y, yd) < 0.05
    # and stage by stage from what the stages before it have left: one bf16 rounding each
    zu = (q1.double() @ w1.double().t()) * c1.double() * s1.double()[:, None]
    assert rel(u, act(zu, "gelu")[0]) < 2.0**-8
    assert rel(y, (q2.double() @ w2.double().t()) * c2.double() * s2.double()[:, None] + bias.double() + h.double()) < 2.0**-8
    graph.destroy()
    ab.lib().ascb200_stream_destroy(side)


def test_norm_into_mxfp8_matmul():
    """The MX form of the norm's output is the A operand of ascb200_gemm's MXFP8 kind as it stands."""
    dev()
    m, k, n = 130, 1024, 192
    g = gen(1)
    x, w = torch.randn(m, k, generator=g, device="cuda").half(), torch.randn(n, k, generator=g, device="cuda")
    wq, ws = torch.empty(n, k, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(n, k // 32, dtype=torch.uint8, device="cuda")
    q, s, y = torch.empty(m, k, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(m, k // 32, dtype=torch.uint8, device="cuda"), torch.empty(m, n, device="cuda")
    blocks = w.view(n, k // 32, 32)
    e = torch.floor(torch.log2(blocks.abs().amax(2))) - 8
    wq.copy_((blocks * torch.exp2(-e)[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(n, k))
    ws.copy_((e + 127).to(torch.uint8))
    ab.check(ab.rms_norm(ab.RmsNormDesc(m=m, k=k, dtype=ab.F16, x_dev=ptr(x), q_dev=ptr(q), q_dtype=ab.FP8_E4M3, scale_dev=ptr(s), scale_mode=ab.SCALE_MX, eps=EPS), stream()))
    ab.check(ab.gemm(ab.KIND_MXFP8_E4M3, m, n, k, ptr(q), ptr(wq), ptr(y), ab.F32, trans_b=True, scale_a=ptr(s), scale_b=ptr(ws), stream=stream()))
    torch.cuda.synchronize()

    def value(c, b):
        return (c.double().view(c.shape[0], -1, 32) * torch.exp2(b.double() - 127)[:, :, None]).view(c.shape)

    want = value(q, s) @ value(wq, ws).t()
    assert rel(y, want) < 1e-5
    exact = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + EPS) @ w.double().t()
    # e4m3 has four significant bits: a step of 1/16 to 1/8 of the value, rms 1/12^0.5 of that: 2.6 % on either side
    assert rel(y, exact) < 0.06


@pytest.mark.parametrize("tokens", [5, 200, 1500])
def test_int8_experts(tokens):
    """norm -> router logits -> routing -> grouped int8 matmul over the rows in expert order, whose counts are the routing's own."""
    dev()
    k, n, experts, top = 256, 384, 12, 3
    g = gen(tokens)
    x, wr = torch.randn(tokens, k, generator=g, device="cuda").bfloat16(), torch.randn(experts, k, generator=g, device="cuda").bfloat16() * 0.1
    w = torch.randint(-127, 128, (experts, n, k), generator=g, device="cuda", dtype=torch.int8)
    ch = torch.rand(experts, n, generator=g, device="cuda") * 0.001 + 0.0005
    valid = (torch.rand(tokens, generator=g, device="cuda") < 0.9).to(torch.uint8)
    y, q, s = torch.empty_like(x), torch.empty(tokens, k, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda")
    logits = torch.empty(tokens, experts, device="cuda")
    idx, weights = torch.empty(tokens, top, dtype=torch.int32, device="cuda"), torch.empty(tokens, top, device="cuda")
    counts, num, loss = torch.empty(experts, dtype=torch.int64, device="cuda"), torch.empty(1, dtype=torch.int64, device="cuda"), torch.empty(1, device="cuda")
    room = room_for(ab.route_workspace_bytes(tokens, experts))
    ab.check(ab.rms_norm(ab.RmsNormDesc(m=tokens, k=k, dtype=ab.BF16, x_dev=ptr(x), y_dev=ptr(y), q_dev=ptr(q), q_dtype=ab.S8, scale_dev=ptr(s), eps=EPS), stream()))
    ab.check(ab.linear(ab.LinearDesc(kind=ab.KIND_BF16, m=tokens, n=experts, k=k, x_dev=ptr(y), w_dev=ptr(wr), trans_w=1, y_dev=ptr(logits), y_dtype=ab.F32), stream()))
    ab.check(ab.route(ab.RouteDesc(tokens=tokens, experts=experts, top_k=top, dtype=ab.F32, logits_dev=ptr(logits), valid_dev=ptr(valid), idx_dev=ptr(idx), weights_dev=ptr(weights),
                                   counts_dev=ptr(counts), num_tokens_dev=ptr(num), loss_dev=ptr(loss), workspace_dev=ptr(room), workspace_bytes=room.numel(), renorm=1), stream()))
    flat = idx.flatten().long()
    order = torch.argsort(torch.where(flat < 0, experts, flat), stable=True)[: int(counts.sum())]
    rows = torch.div(order, top, rounding_mode="floor")
    a, tok, out = q[rows].contiguous(), s[rows].contiguous(), torch.empty(len(rows), n, dtype=torch.bfloat16, device="cuda")
    ab.check(ab.gemm(ab.KIND_S8, len(rows), n, k, ptr(a), ptr(w), ptr(out), ab.BF16, epilogue=ab.EPI_DEQUANT_TOKEN_CHANNEL, trans_b=True, tok=ptr(tok), ch=ptr(ch), group_counts=ptr(counts),
                     groups=experts, stream=stream()))
    torch.cuda.synchronize()
    want = torch.zeros(tokens, n, dtype=torch.float64, device="cuda")
    got = torch.zeros_like(want).index_add_(0, rows, out.double() * weights.flatten()[order].double()[:, None])
    for t in range(tokens):
        for j in range(top):
            e = int(idx[t, j])
            assert (e < 0) == (int(valid[t]) == 0)
            if e >= 0:
                want[t] += float(weights[t, j]) * (w[e].double() @ q[t].double()) * ch[e].double() * float(s[t])
    assert rel(got, want) < 2.0**-8
    assert int(num) == int(valid.sum()) and int(counts.sum()) == top * int(num)


def test_training_step():
    """Forward and backward of residual + norm -> linear (SiLU) -> linear + residual, with a routed balance loss beside it; every gradient against
    autograd of the same network in 64 bits.  Its tensors are rounded to bf16 eleven times on the longest way (0.2 % rms each)."""
    dev()
    m, k, n, experts, top = 260, 320, 448, 16, 2
    g = gen(9)
    bf = torch.bfloat16

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(bf)

    x, r, w1, w2, wr = randn(m, k), randn(m, k), randn(n, k, scale=k**-0.5), randn(k, n, scale=n**-0.5), randn(experts, k, scale=k**-0.5)
    gamma, b1, gy = 1 + 0.1 * torch.randn(k, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda"), randn(m, k)
    e = lambda *s, t=bf: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
    f32 = torch.float32
    h, y, rstd, u, z, out, logits = e(m, k), e(m, k), e(m, t=f32), e(m, n), e(m, n), e(m, k), e(m, experts)
    idx, wts, counts, num, loss = e(m, top, t=torch.int32), e(m, top, t=f32), e(experts, t=torch.int64), e(1, t=torch.int64), e(1, t=f32)
    room = room_for(max(ab.route_workspace_bytes(m, experts), ab.linear_grad_workspace_bytes(m, n), ab.linear_grad_workspace_bytes(m, k), ab.rms_norm_grad_workspace_bytes(m, k)))
    S = dict(workspace_dev=ptr(room), workspace_bytes=room.numel())
    bfk = dict(kind=ab.KIND_BF16, trans_w=1)
    ab.check(ab.rms_norm(ab.RmsNormDesc(m=m, k=k, dtype=ab.BF16, x_dev=ptr(x), residual_dev=ptr(r), gamma_dev=ptr(gamma), gamma_dtype=ab.F32, sum_dev=ptr(h), y_dev=ptr(y), rstd_dev=ptr(rstd),
                                        eps=EPS), stream()))
    ab.check(ab.linear(ab.LinearDesc(m=m, n=experts, k=k, x_dev=ptr(y), w_dev=ptr(wr), y_dev=ptr(logits), y_dtype=ab.BF16, **bfk), stream()))
    ab.check(ab.route(ab.RouteDesc(tokens=m, experts=experts, top_k=top, dtype=ab.BF16, logits_dev=ptr(logits), idx_dev=ptr(idx), weights_dev=ptr(wts), counts_dev=ptr(counts),
                                   num_tokens_dev=ptr(num), loss_dev=ptr(loss), renorm=1, **S), stream()))
    ab.check(ab.linear(ab.LinearDesc(m=m, n=n, k=k, x_dev=ptr(y), w_dev=ptr(w1), bias_dev=ptr(b1), act=ab.ACT_SILU, y_dev=ptr(u), y_dtype=ab.BF16, z_dev=ptr(z), **bfk), stream()))
    ab.check(ab.linear(ab.LinearDesc(m=m, n=k, k=n, x_dev=ptr(u), w_dev=ptr(w2), residual_dev=ptr(h), y_dev=ptr(out), y_dtype=ab.BF16, **bfk), stream()))
    # backward: out's gradient gy, the loss's 10
    du, dw2, dy1, dw1, db1, dl, dyr, dwr, dx, dgamma = e(m, n), e(k, n), e(m, k), e(n, k), e(n, t=f32), e(m, experts), e(m, k), e(experts, k), e(m, k), e(k, t=f32)
    ten = torch.full((1,), 10.0, device="cuda")
    ab.check(ab.linear_grad(ab.LinearGradDesc(m=m, n=k, k=n, dy_dev=ptr(gy), x_dev=ptr(u), w_dev=ptr(w2), dx_dev=ptr(du), dw_dev=ptr(dw2), dw_dtype=ab.BF16, **bfk), stream()))
    ab.check(ab.linear_grad(ab.LinearGradDesc(m=m, n=n, k=k, act=ab.ACT_SILU, dy_dev=ptr(du), z_dev=ptr(z), x_dev=ptr(y), w_dev=ptr(w1), dx_dev=ptr(dy1), dw_dev=ptr(dw1), dw_dtype=ab.BF16,
                                              dbias_dev=ptr(db1), **bfk, **S), stream()))
    ab.check(ab.route_grad(ab.RouteGradDesc(tokens=m, experts=experts, top_k=top, dtype=ab.BF16, logits_dev=ptr(logits), idx_dev=ptr(idx), counts_dev=ptr(counts), num_tokens_dev=ptr(num),
                                            dloss_dev=ptr(ten), dlogits_dev=ptr(dl), renorm=1), stream()))
    ab.check(ab.linear_grad(ab.LinearGradDesc(m=m, n=experts, k=k, dy_dev=ptr(dl), x_dev=ptr(y), w_dev=ptr(wr), dx_dev=ptr(dyr), dw_dev=ptr(dwr), dw_dtype=ab.BF16, **bfk, **S), stream()))
    dy = (dy1.float() + dyr.float()).to(bf)
    ab.check(ab.rms_norm_grad(ab.RmsNormGradDesc(m=m, k=k, dtype=ab.BF16, dy_dev=ptr(dy), h_dev=ptr(h), rstd_dev=ptr(rstd), gamma_dev=ptr(gamma), gamma_dtype=ab.F32, dh_dev=ptr(gy), dx_dev=ptr(dx),
                                                 dgamma_dev=ptr(dgamma), dgamma_dtype=ab.F32, **S), stream()))
    torch.cuda.synchronize()
    leaves = [t.double().requires_grad_() for t in (x, w1, w2, wr, gamma, b1)]
    xd, w1d, w2d, wrd, gd, bd = leaves
    hd = xd + r.double()
    yd = hd / torch.sqrt((hd * hd).mean(1, keepdim=True) + EPS) * gd
    zd = yd @ w1d.t() + bd
    od = (zd * torch.sigmoid(zd)) @ w2d.t() + hd
    p = torch.softmax(yd @ wrd.t(), 1)
    ld = experts / (m * m * top) * (counts.double() * p.sum(0)).sum()
    ((od * gy.double()).sum() + 10 * ld).backward()
    assert rel(out, od) < 0.01 and abs(float(loss) - float(ld)) < 0.01 * float(ld)
    for name, got, leaf in (("x", dx, xd), ("w1", dw1, w1d), ("w2", dw2, w2d), ("router", dwr, wrd), ("gamma", dgamma, gd), ("bias", db1, bd)):
        assert rel(got, leaf.grad) < 11 * 2.0**-8, name


@pytest.mark.parametrize("policy,group", [(ab.DEQUANT_PER_TOKEN, 0), (ab.DEQUANT_PER_GROUP, 32), (ab.DEQUANT_PER_GROUP, 64)])
@pytest.mark.parametrize("dst,scale_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 7), (5, 8), (4, 96), (33, 1000), (7, 1001), (300, 4096), (2, 40960)])
def test_values_of_int8_codes(m, n, dst, scale_dtype, policy, group):
    """dst = cast(code * scale): one product, one rounding, so within half a step of it and equal for fp32."""
    dev()
    g = torch.Generator().manual_seed(m + n)
    codes = torch.randint(-128, 128, (m, n), generator=g).to(torch.int8)
    scale = (torch.rand(m, 1 if group == 0 else -(-n // group), generator=g) * 0.1 + 1e-3).to(scale_dtype)
    cs, ss, out = codes.cuda(), scale.cuda(), Out(m, n, dst)
    ab.check(ab.dequant_policy(ptr(cs), out.ptr(), m, n, ab.S8, CODE[scale_dtype], CODE[dst], policy, ptr(ss), k_dim=1, group_size=group, stream=stream()))
    torch.cuda.synchronize()
    out.check()
    wide = scale.double().repeat_interleave(group or n, 1)[:, :n]
    want = codes.double() * wide
    near(out.t, want, HALF_STEP[dst] * (1 + 2.0**-10) * want.abs() + 2.0**-24 * want.abs(), "values")
