"""ascb200_linear / ascb200_linear_grad against their formulas in 64 bits.

Tolerances.  Products of 16-bit values are exact in fp32.  Their sum is made in fp32 by the tensor cores, 16 terms at a time, with at most a unit in
the last place (2^-23) of the running magnitude lost per step and per term of a step: (k / 16 + 32) 2^-23 of the sum of absolute products.
int8 sums are exact.  z then takes at most four more roundings.  An activation's slope is at most 1.13; its own evaluation (one ex2, one rcp, a
rounded argument a) is off by |value| (|a| 2^-21 + 2^-20), GELU's by |z| (1.5e-7 + 2^-21); a slope's by 2^-18 + |z| 2^-22.  Outputs are rounded once.
"""
import ctypes as C
import math

import pytest
import torch

import ascb200 as ab
from torch_util import CODE, HALF_STEP, TINY, Out, dev, near, ptr, rows_in, stream

pytestmark = pytest.mark.gpu
F = 2.0**-24
ACTS = {"none": ab.ACT_NONE, "faster_gelu": ab.ACT_FASTER_GELU, "relu": ab.ACT_RELU, "gelu": ab.ACT_GELU, "gelu_tanh": ab.ACT_GELU_TANH, "silu": ab.ACT_SILU}
KIND = {torch.float16: ab.KIND_F16, torch.bfloat16: ab.KIND_BF16, torch.int8: ab.KIND_S8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def act(z, name):
    """(value, slope, bound of |a|) in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z), torch.zeros_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), torch.zeros_like(z)
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), torch.zeros_like(z)
    if name == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        a, da = c * (z + 0.044715 * z**3), c * (1 + 3 * 0.044715 * z**2)
    else:
        scale = 1.702 if name == "faster_gelu" else 1.0
        a, da = scale * z, torch.full_like(z, scale)
    g = torch.sigmoid(a)
    return z * g, g + z * g * (1 - g) * da, 1.45 * a.abs()


def operands(m, n, k, dtype, trans_w, pad, seed=0):
    g = gen(seed + 31 * m + 7 * n + k)
    if dtype == torch.int8:
        x, w = torch.randint(-127, 128, (m, k), generator=g).to(dtype), torch.randint(-127, 128, (n, k), generator=g).to(dtype)
    else:
        x, w = torch.randn(m, k, generator=g).to(dtype), (torch.randn(n, k, generator=g) * 2 / math.sqrt(k)).to(dtype)
    step = 16 if dtype == torch.int8 else 8
    up = lambda c: -c % step + (step if pad else 0)  # noqa: E731  rows start on 16 bytes; what lies behind them is NaN (int8: 77)
    ws = w if trans_w else w.t().contiguous()
    return x, w, rows_in(x, dtype, up(k)), rows_in(ws, dtype, up(ws.shape[1]))


def forward(m, n, k, dtype, name="none", bias="f32", residual=True, z=False, trans_w=1, out=None, pad=0, y_pad=0, offset=0, in_place=False, tok=True):
    dev()
    out = out or (torch.bfloat16 if dtype == torch.int8 else dtype)
    x, w, xs, ws = operands(m, n, k, dtype, trans_w, pad)
    g = gen(m + n + k)
    b = None if bias is None else torch.randn(n, generator=g).to(torch.float32 if bias == "f32" else out)
    r = torch.randn(m, n, generator=g).to(out) if residual else None
    y = Out(m, n, out, y_pad, offset)
    rs = None
    if r is not None:
        rs = rows_in(r, out, y_pad, offset)
        if in_place:
            y.t.copy_(r)
            rs = y.t
    d = ab.LinearDesc(kind=KIND[dtype], m=m, n=n, k=k, x_dev=ptr(xs), ldx=xs.stride(0), w_dev=ptr(ws), ldw=ws.stride(0), trans_w=trans_w, act=ACTS[name], y_dev=y.ptr(), ldy=y.ld,
                      y_dtype=CODE[out], residual_dev=ptr(rs), ld_residual=y.ld if rs is not None else 0)
    bs = None if b is None else b.cuda()
    if b is not None:
        d.bias_dev, d.bias_dtype = ptr(bs), CODE[b.dtype]
    # (the products in 64 bits on the device: exact enough by 2^29)
    xd, wd = x.cuda().double(), w.cuda().double()
    acc, mass = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if dtype == torch.int8:
        ch, ts = (torch.rand(n, generator=g) + 0.5) * 0.01 / math.sqrt(k), torch.rand(m, generator=g) * 0.01 + 0.005 if tok else None
        chs, tss = ch.cuda(), None if ts is None else ts.cuda()
        d.ch_scale_dev, d.tok_scale_dev = ptr(chs), ptr(tss)
        acc = acc * chs.double() * (1 if ts is None else tss.double()[:, None])
        err = 4 * F * acc.abs()
    else:
        err = (k / 16 + 32) * 2 * F * mass
    zs = Out(m, n, out, y_pad, offset) if z else None
    if z:
        d.z_dev, d.ldz = zs.ptr(), zs.ld
    ab.check(ab.linear(d, stream()))
    torch.cuda.synchronize()
    y.check()
    ref = acc if b is None else acc + bs.double()
    err = err + 2 * F * ref.abs()
    if z:
        zs.check()
        near(zs.t, ref, err + HALF_STEP[out] * ref.abs() + TINY[out], "z")
    v, _, a = act(ref, name)
    err = 1.13 * err + v.abs() * (a * 2.0**-21 + 2.0**-20) + (ref.abs() * (1.5e-7 + 2.0**-21) if name == "gelu" else 0)
    if r is not None:
        v = v + r.cuda().double()
    near(y.t, v, err + (HALF_STEP[out] + F) * v.abs() + TINY[out], "y")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 17, 33), (2, 16, 64), (7, 100, 1000), (8, 130, 257), (9, 64, 512), (16, 255, 515), (1, 1000, 4099), (17, 33, 65), (33, 64, 64), (64, 200, 130),
                                   (65, 257, 1030), (130, 96, 77), (256, 512, 256), (300, 1000, 2050), (129, 8, 4096), (1000, 130, 72)])
def test_sizes(m, n, k, dtype):
    forward(m, n, k, dtype, "silu", z=dtype != torch.int8)


@pytest.mark.parametrize("m,n,k", [(17, 40, 70), (31, 512, 500), (100, 77, 1030), (128, 1024, 512), (200, 16, 2100), (256, 100, 300), (257, 100, 300)])
def test_blocks_of_tokens(m, n, k):
    """Several blocks of tokens over the weights' rows, up to where the GEMM kernels take over."""
    forward(m, n, k, torch.bfloat16, "gelu_tanh", z=True, bias="out")
    forward(m, n, k, torch.int8, "silu")


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
@pytest.mark.parametrize("m", [5, 200])
def test_activations(m, dtype, name):
    for out in (None, torch.float32):
        forward(m, 300, 200, dtype, name, out=out, bias="f32")


@pytest.mark.parametrize("bias,residual,z,trans_w,y_pad,offset", [(None, False, False, 1, 0, 0), ("out", True, True, 1, 3, 1), ("f32", False, True, 0, 8, 8), ("out", True, False, 0, 0, 0),
                                                                  (None, True, True, 1, 1, 0), ("f32", True, False, 0, 5, 3)])
@pytest.mark.parametrize("m,n,k", [(3, 40, 96), (13, 129, 300), (40, 77, 260), (260, 513, 384)])
def test_forms_and_strides(m, n, k, bias, residual, z, trans_w, y_pad, offset):
    for dtype, out in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)):
        forward(m, n, k, dtype, "gelu_tanh", bias=bias, residual=residual, z=z, trans_w=trans_w, pad=1, y_pad=y_pad, offset=offset, out=out)


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,trans_w,tok", [(4, 1, True), (12, 1, False), (48, 1, False), (300, 1, True), (70, 0, True)])
def test_int8_outputs(m, trans_w, tok, out):
    forward(m, 272, 528, torch.int8, "gelu", bias="out", out=out, trans_w=trans_w, pad=1, tok=tok)


@pytest.mark.parametrize("m,n,k", [(6, 50, 64), (100, 300, 128), (513, 768, 256)])
def test_residual_in_place(m, n, k):
    for dtype in (torch.bfloat16, torch.int8):
        forward(m, n, k, dtype, "relu", in_place=True)
    forward(m, n, k, torch.float16, "none", in_place=True, out=torch.float32)


@pytest.mark.parametrize("m,n,k", [(64, 128, 4096), (20, 256, 8192), (256, 256, 2048)])
def test_split_k(m, n, k):
    """Few tiles and a long K: the library's own choice is a cluster per tile."""
    forward(m, n, k, torch.bfloat16, "gelu", z=True)
    forward(m, n, k, torch.int8, "silu")


@pytest.mark.parametrize("m,n,k", [(40, 1100, 4100), (64, 2100, 2100), (65, 1101, 4100), (130, 3001, 1000), (200, 4096, 264), (300, 515, 1000), (1025, 65, 300)])
def test_gemm_kernels(m, n, k):
    """Sizes that the GEMM kernels take: tiles of 64 rows and less, ragged ones, odd widths through the staging buffer, every output type."""
    for dtype in (torch.bfloat16, torch.float16):
        forward(m, n, k, dtype, "gelu", z=True, bias="out")
        forward(m, n, k, dtype, "silu", z=True, out=torch.float32, y_pad=3, offset=1)
        forward(m, n, k, dtype, "relu", residual=True, z=True, y_pad=-n % 8 + 8, offset=8, pad=1)
        forward(m, n, k, dtype, "none", in_place=True, trans_w=0)
    for out in (torch.bfloat16, torch.float32):
        forward(m, n, k, torch.int8, "gelu_tanh", out=out, pad=1, tok=out == torch.float32)
        forward(m, n, k, torch.int8, "faster_gelu", out=out, residual=False, bias=None, y_pad=5)


@pytest.mark.parametrize("m,n,k", [(64, 512, 16384), (300, 256, 4096), (20, 300, 20000), (60, 128, 18000)])
def test_gemm_kernels_split_k(m, n, k):
    forward(m, n, k, torch.bfloat16, "gelu", z=True)
    forward(m, n + 1, k, torch.float16, "silu", z=True, out=torch.float32)
    forward(m, n, k, torch.int8, "silu")


def test_unaligned_residual_beside_aligned_output():
    """y's rows on 16 bytes, the residual's not, and the other way round."""
    dev()
    m, n, k = 300, 515, 1000
    x, w, xs, ws = operands(m, n, k, torch.bfloat16, 1, 0)
    r = torch.randn(m, n, generator=gen(21)).bfloat16()
    want = (x.cuda().double() @ w.cuda().double().t()) + r.cuda().double()
    tol = (k / 16 + 32) * 2 * F * (x.cuda().double().abs() @ w.cuda().double().abs().t()) + (2.0**-8 + 4 * F) * want.abs() + TINY[torch.bfloat16]
    for y_pad, r_pad in ((5, 0), (0, 5), (5, 13)):
        y, rs = Out(m, n, torch.bfloat16, y_pad), rows_in(r, torch.bfloat16, r_pad)
        ab.check(ab.linear(ab.LinearDesc(kind=ab.KIND_BF16, m=m, n=n, k=k, x_dev=ptr(xs), ldx=xs.stride(0), w_dev=ptr(ws), ldw=ws.stride(0), trans_w=1, residual_dev=ptr(rs), ld_residual=n + r_pad,
                                         y_dev=y.ptr(), ldy=y.ld, y_dtype=ab.BF16), stream()))
        torch.cuda.synchronize()
        y.check()
        near(y.t, want, tol, "y")


@pytest.mark.parametrize("width", [64, 112, 160, 256])
def test_pair_tiles(width, monkeypatch):
    monkeypatch.setenv("ASCB200_PAIR_N", str(width))
    for m, n, k in ((300, 700, 320), (512, 515, 64)):
        forward(m, n, k, torch.bfloat16, "silu", z=True)
        forward(m, n, k, torch.int8, "gelu")


def test_infinite_and_nan_inputs_stay_in_their_rows():
    dev()
    for m in (6, 150):
        x, w = torch.randn(m, 64, generator=gen(1)).half(), torch.randn(40, 64, generator=gen(2)).half()
        x[1, 3], x[2, 5] = math.nan, math.inf
        y = torch.empty(m, 40, device="cuda", dtype=torch.float16)
        xs, ws = x.cuda(), w.cuda()
        ab.check(ab.linear(ab.LinearDesc(kind=ab.KIND_F16, m=m, n=40, k=64, x_dev=ptr(xs), w_dev=ptr(ws), trans_w=1, act=ab.ACT_RELU, y_dev=ptr(y), y_dtype=ab.F16), stream()))
        torch.cuda.synchronize()
        assert torch.isnan(y[1]).all()
        # F16 outputs saturate: the infinity shows as the largest value, or as 0 behind relu
        assert ((y[2] == 65504) | (y[2] == 0)).all()
        rows = [0, 3, 4, 5]
        assert torch.isfinite(y[rows]).all()


@pytest.mark.parametrize("name", ACTS)
def test_activations_at_the_ends_of_the_range(name):
    """z comes from the bias alone.  From |z| = 200 on every activation is z or 0 and every slope 1 or 0 to the last bit; the infinities as in
    the formula (NaN where it has an infinity times 0)."""
    dev()
    z = torch.tensor([200.0, 1e10, 2.5e38, 3.3e38, -200.0, -1e10, -2.5e38, -3.3e38, math.inf] + ([] if name == "relu" else [math.nan]))
    n = len(z)
    code = ACTS[name] if isinstance(ACTS, dict) else getattr(ab, "ACT_" + name.upper())
    want, slope, _ = act(z.bfloat16().double(), name)
    for m in (2, 300):
        x, w = torch.zeros(m, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, 16, dtype=torch.bfloat16, device="cuda")
        bias, y = z.bfloat16().float().cuda(), torch.empty(m, n, device="cuda")
        ab.check(ab.linear(ab.LinearDesc(kind=ab.KIND_BF16, m=m, n=n, k=16, x_dev=ptr(x), w_dev=ptr(w), trans_w=1, act=code, bias_dev=ptr(bias), bias_dtype=ab.F32, y_dev=ptr(y),
                                         y_dtype=ab.F32), stream()))
        torch.cuda.synchronize()
        near(y, want.expand(m, n), 1e-37, "y")
    # the slope of finite z: dbias of one row with dy = 1
    z, slope = z[:8].bfloat16(), slope[:8]
    zs, dy, dbias = z[None].cuda(), torch.ones(1, 8, dtype=torch.bfloat16, device="cuda"), torch.empty(8, device="cuda")
    work = torch.empty(ab.linear_grad_workspace_bytes(1, 8), dtype=torch.uint8, device="cuda")
    ab.check(ab.linear_grad(ab.LinearGradDesc(kind=ab.KIND_BF16, m=1, n=8, k=16, act=code, trans_w=1, dy_dev=ptr(dy), z_dev=ptr(zs), dbias_dev=ptr(dbias), dbias_dtype=ab.F32,
                                              workspace_dev=ptr(work), workspace_bytes=work.numel()), stream()))
    torch.cuda.synchronize()
    near(dbias, slope, 1e-37, "slope")


# ---- gradients -----------------------------------------------------------------------------------------------------------------
def backward(m, n, k, dtype, name="silu", trans_w=1, pad=0, dx=True, dw=True, dbias=True, dw_dtype=None, dbias_dtype=torch.float32, dy_pad=None, offset=0, out_pads=(3, 5)):
    dev()
    x, w, xs, ws = operands(m, n, k, dtype, trans_w, pad)
    g = gen(m * n + k)
    dy, z = torch.randn(m, n, generator=g).to(dtype), (torch.randn(m, n, generator=g) * 2).to(dtype)
    dy_pad = -n % 8 if dy_pad is None else dy_pad
    ds, zs = rows_in(dy, dtype, dy_pad, offset), rows_in(z, dtype, dy_pad, offset)
    size = ab.linear_grad_workspace_bytes(m, n)
    room = torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    d = ab.LinearGradDesc(kind=KIND[dtype], m=m, n=n, k=k, act=ACTS[name], trans_w=trans_w, dy_dev=ptr(ds), ld_dy=n + dy_pad, z_dev=ptr(zs), ldz=n + dy_pad, x_dev=ptr(xs), ldx=xs.stride(0),
                          w_dev=ptr(ws), ldw=ws.stride(0), workspace_dev=ptr(room), workspace_bytes=size)
    dw_dtype = dw_dtype or dtype
    gx, gw, gb = Out(m, k, dtype, out_pads[0]), Out(n if trans_w else k, k if trans_w else n, dw_dtype, out_pads[1]), Out(1, n, dbias_dtype)
    if dx:
        d.dx_dev, d.ld_dx = gx.ptr(), gx.ld
    if dw:
        d.dw_dev, d.ld_dw, d.dw_dtype = gw.ptr(), gw.ld, CODE[dw_dtype]
    if dbias:
        d.dbias_dev, d.dbias_dtype = gb.ptr(), CODE[dbias_dtype]
    ab.check(ab.linear_grad(d, stream()))
    torch.cuda.synchronize()
    assert (room[size:] == 0xFF).all()
    x, w, dy, z = (t.cuda().double() for t in (x, w, dy, z))
    slope = act(z, name)[1]
    dz = dy * slope
    exact = name in ("none", "relu")
    err32 = torch.zeros_like(dz) if exact else dy.abs() * (2.0**-18 + z.abs() * 2.0**-22) + F * dz.abs()
    # up to 16 rows: two numbers of the type, the second of which holds the first one's rounding and is rounded itself
    half = HALF_STEP[dtype] ** 2 if m <= 16 and trans_w else HALF_STEP[dtype]
    err16 = err32 + (0 if exact else (half * (dz.abs() + err32) + 2 * TINY[dtype]))
    if dx:
        gx.check()
        want = dz @ w
        near(gx.t, want, err16 @ w.abs() + (n / 16 + 32) * 2 * F * (dz.abs() @ w.abs()) * 1.01 + HALF_STEP[dtype] * want.abs() + TINY[dtype], "dx")
    if dw:
        gw.check()
        want = dz.t() @ x
        tol = err16.t() @ x.abs() + (m / 16 + 32) * 2 * F * (dz.abs().t() @ x.abs()) * 1.01 + HALF_STEP[dw_dtype] * want.abs() + TINY[dw_dtype]
        near(gw.t, want if trans_w else want.t(), tol if trans_w else tol.t(), "dw")
    if dbias:
        gb.check()
        want = dz.sum(0)
        near(gb.t[0], want, err32.sum(0) + (m / 8 + 64) * F * dz.abs().sum(0) + HALF_STEP[dbias_dtype] * want.abs() + TINY[dbias_dtype], "dbias")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 64), (3, 17, 33), (16, 100, 40), (65, 257, 130), (130, 1000, 72), (300, 130, 515), (1000, 64, 264), (2049, 300, 96)])
def test_gradient_sizes(m, n, k, dtype):
    backward(m, n, k, dtype)


@pytest.mark.parametrize("out_pads", [(0, 0), (8, 8), (1, 4)])
@pytest.mark.parametrize("dtype,dw_dtype", [(torch.float16, None), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (2, 15, 64), (1, 4000, 64), (5, 2050, 515), (16, 1000, 1000), (9, 257, 72), (15, 5312, 1200), (2, 300, 2048), (16, 64, 4096), (8, 16, 20000), (7, 3001, 129)])
def test_gradient_of_few_rows(m, n, k, dtype, dw_dtype, out_pads):
    backward(m, n, k, dtype, dw_dtype=dw_dtype, out_pads=out_pads)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("kw", [dict(dx=False), dict(dw=False), dict(dbias=False), dict(dx=False, dbias=False), dict(dbias_dtype=torch.float16, dy_pad=3, offset=1), dict(dy_pad=0),
                                dict(dy_pad=16, offset=8, dw=False, dbias=False)])
def test_gradient_forms_of_few_rows(name, kw):
    backward(13, 1030, 200, torch.float16, name, pad=1, **kw)


@pytest.mark.parametrize("name", ACTS)
def test_gradient_activations(name):
    backward(150, 210, 90, torch.float16, name)
    backward(150, 210, 90, torch.bfloat16, name, trans_w=0, pad=1)


@pytest.mark.parametrize("kw", [dict(dx=False), dict(dw=False), dict(dbias=False), dict(dx=False, dw=False), dict(dw_dtype=torch.float32), dict(dbias_dtype=torch.float16), dict(dy_pad=3, offset=1),
                                dict(dy_pad=0), dict(dy_pad=16, offset=8, dbias=False)])
@pytest.mark.parametrize("name", ["none", "gelu"])
@pytest.mark.parametrize("trans_w", [0, 1])
def test_gradient_forms(trans_w, name, kw):
    backward(77, 131, 200, torch.float16, name, trans_w=trans_w, pad=1, **kw)


@pytest.mark.parametrize("name", ACTS)
def test_gradient_against_differences(name):
    """sum(gy * y) of the forward call itself, moved along x, w and the bias."""
    dev()
    m, n, k, step = 3, 16, 8, 2.0**-5
    g = gen(9)
    # multiples of 2^-6, so that the moved operands are still exact halves; z stays clear of relu's corner
    x, w = torch.randint(-64, 65, (m, k), generator=g) / 64, torch.randint(-32, 33, (n, k), generator=g) / 64
    b = torch.randint(-64, 65, (n,), generator=g) / 64 + 1 / 128
    gy = torch.randn(m, n, generator=g).half().float()

    def value(x, w, b):
        xs, ws, bs, y, z = x.half().cuda(), w.half().cuda(), b.cuda(), torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
        ab.check(ab.linear(ab.LinearDesc(kind=ab.KIND_F16, m=m, n=n, k=k, x_dev=ptr(xs), w_dev=ptr(ws), trans_w=1, act=ACTS[name], bias_dev=ptr(bs), y_dev=ptr(y), y_dtype=ab.F32,
                                         z_dev=ptr(z)), stream()))
        torch.cuda.synchronize()
        return float((y.cpu().double() * gy.double()).sum()), z.cpu().double()

    _, z = value(x, w, b)
    zh = z.half()  # what a training step keeps: a rounding of 2^-11 of z, which moves a slope by at most 1.2 of that
    xs, ws, ds, zs = x.half().cuda(), w.half().cuda(), gy.half().cuda(), zh.cuda()
    dx, dw, db = torch.empty(m, k, device="cuda", dtype=torch.float16), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    room = torch.empty(ab.linear_grad_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")
    ab.check(ab.linear_grad(ab.LinearGradDesc(kind=ab.KIND_F16, m=m, n=n, k=k, act=ACTS[name], trans_w=1, dy_dev=ptr(ds), z_dev=ptr(zs), x_dev=ptr(xs), w_dev=ptr(ws), dx_dev=ptr(dx),
                                              dw_dev=ptr(dw), dw_dtype=ab.F32, dbias_dev=ptr(db), workspace_dev=ptr(room), workspace_bytes=room.numel()), stream()))
    torch.cuda.synchronize()
    corner = (z.abs() < step * 1.01) if name == "relu" else torch.zeros_like(z, dtype=torch.bool)  # there the difference sees both sides
    slack = lambda i, j: gy.double()[i, j].abs() * (0.3 * step**2 + 2.0**-10 + 1.3 * 2.0**-11 * z[i, j].abs() + corner[i, j])  # noqa: E731
    noise = 2.0**-19 * float(gy.abs().sum()) / step
    every = torch.tensor([[float(slack(i, j)) for j in range(n)] for i in range(m)])
    for i in range(m):
        for c in range(k):
            d = torch.zeros(m, k)
            d[i, c] = step
            diff = (value(x + d, w, b)[0] - value(x - d, w, b)[0]) / (2 * step)
            assert abs(diff - float(dx[i, c])) <= float((every[i] * w[:, c].abs()).sum()) + 2.0**-11 * abs(diff) + noise, ("dx", i, c)
    for j in range(n):
        for c in range(k):
            d = torch.zeros(n, k)
            d[j, c] = step
            diff = (value(x, w + d, b)[0] - value(x, w - d, b)[0]) / (2 * step)
            assert abs(diff - float(dw[j, c])) <= float((every[:, j] * x[:, c].abs()).sum()) + noise, ("dw", j, c)
        d = torch.zeros(n)
        d[j] = step
        diff = (value(x, w, b + d)[0] - value(x, w, b - d)[0]) / (2 * step)
        assert abs(diff - float(db[j])) <= float(every[:, j].sum()) + noise, ("dbias", j)


def test_no_rows():
    dev()
    dw, db = torch.ones(5, 12, device="cuda"), torch.ones(5, device="cuda")
    ab.check(ab.linear_grad(ab.LinearGradDesc(kind=ab.KIND_F16, m=0, n=5, k=8, trans_w=1, dw_dev=ptr(dw), ld_dw=12, dw_dtype=ab.F32, dbias_dev=ptr(db)), stream()))
    ab.check(ab.linear(ab.LinearDesc(kind=ab.KIND_F16, m=0, n=5, k=8, trans_w=1, y_dtype=ab.F16), stream()))
    torch.cuda.synchronize()
    assert (dw[:, :8] == 0).all() and (dw[:, 8:] == 1).all() and (db == 0).all()


# ---- calls ---------------------------------------------------------------------------------------------------------------------
def test_refusals():
    dev()
    x, w, y, f = (torch.zeros(64, 64, device="cuda", dtype=torch.float16) for _ in range(4))
    s = torch.zeros(64, device="cuda")

    def rc(**kw):
        v = dict(kind=ab.KIND_F16, m=32, n=64, k=64, x_dev=ptr(x), w_dev=ptr(w), trans_w=1, y_dev=ptr(y), y_dtype=ab.F16) | kw
        return ab.linear(ab.LinearDesc(**v), stream())

    assert rc() == 0
    for bad in (dict(m=-1), dict(n=-1), dict(k=0), dict(x_dev=None), dict(w_dev=None), dict(y_dev=None), dict(ldx=56), dict(ldw=56), dict(ldy=63), dict(ldz=63), dict(ld_residual=63), dict(act=6),
                dict(act=-1), dict(trans_w=2), dict(reserved=1), dict(tok_scale_dev=ptr(s)), dict(z_dev=ptr(y)), dict(residual_dev=ptr(y), ld_residual=72), dict(residual_dev=ptr(f), z_dev=ptr(f)), dict(kind=ab.KIND_S8, y_dtype=ab.BF16)):
        assert rc(**bad) == ab.EINVAL, bad
    for bad in (dict(kind=ab.KIND_MXFP4), dict(kind=9), dict(y_dtype=ab.BF16), dict(y_dtype=ab.S8), dict(bias_dev=ptr(s), bias_dtype=ab.BF16),
                dict(kind=ab.KIND_S8, y_dtype=ab.BF16, ch_scale_dev=ptr(s), z_dev=ptr(f))):
        assert rc(**bad) == ab.EUNSUPPORTED, bad
    for m in (4, 32):  # both kernels
        for bad in (dict(x_dev=ptr(x) + 2), dict(w_dev=ptr(w) + 8), dict(k=60, ldx=60), dict(k=60, ldw=60), dict(y_dev=ptr(y) + 1), dict(residual_dev=ptr(f) + 1), dict(bias_dev=ptr(s) + 2)):
            assert rc(m=m, **bad) == ab.EALIGN, bad
    assert ab.lib().ascb200_linear(None, None) == ab.EINVAL

    room = torch.zeros(ab.linear_grad_workspace_bytes(32, 64), device="cuda", dtype=torch.uint8)

    def grad(**kw):
        v = dict(kind=ab.KIND_F16, m=32, n=64, k=64, act=ab.ACT_SILU, trans_w=1, dy_dev=ptr(y), z_dev=ptr(f), x_dev=ptr(x), w_dev=ptr(w), dx_dev=ptr(x), dw_dev=ptr(w), dw_dtype=ab.F16,
                 workspace_dev=ptr(room), workspace_bytes=room.numel()) | kw
        return ab.linear_grad(ab.LinearGradDesc(**v), stream())

    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(dy_dev=None), dict(z_dev=None), dict(x_dev=None), dict(w_dev=None), dict(workspace_dev=None), dict(workspace_bytes=room.numel() - 1),
                dict(act=6), dict(trans_w=-1), dict(ld_dy=63), dict(ldz=63), dict(ldx=63), dict(ldw=63), dict(ld_dx=63), dict(ld_dw=63)):
        assert grad(**bad) == ab.EINVAL, bad
    for bad in (dict(kind=ab.KIND_S8), dict(dw_dtype=ab.BF16), dict(dbias_dev=ptr(s), dbias_dtype=ab.BF16)):
        assert grad(**bad) == ab.EUNSUPPORTED, bad
    for bad in (dict(x_dev=ptr(x) + 2), dict(w_dev=ptr(w) + 8), dict(workspace_dev=ptr(room) + 8), dict(dy_dev=ptr(y) + 1), dict(dbias_dev=ptr(s) + 1)):
        assert grad(**bad) == ab.EALIGN, bad
    assert ab.linear_grad_workspace_bytes(0, 4) == 0 and ab.linear_grad_workspace_bytes(-1, 4) == 0
    assert ab.lib().ascb200_linear_grad(None, None) == ab.EINVAL
    torch.cuda.synchronize()


def test_captured_and_replayed():
    dev()
    m, n, k = 120, 96, 160
    t = {c: torch.zeros(a, b, device="cuda", dtype=torch.bfloat16) for c, a, b in (("x", m, k), ("w", n, k), ("y", m, n), ("z", m, n), ("dy", m, n), ("dx", m, k), ("dw", n, k))}
    room, db = torch.zeros(ab.linear_grad_workspace_bytes(m, n), device="cuda", dtype=torch.uint8), torch.zeros(n, device="cuda")
    f = ab.LinearDesc(kind=ab.KIND_BF16, m=m, n=n, k=k, x_dev=ptr(t["x"]), w_dev=ptr(t["w"]), trans_w=1, act=ab.ACT_GELU, y_dev=ptr(t["y"]), y_dtype=ab.BF16, z_dev=ptr(t["z"]))
    b = ab.LinearGradDesc(kind=ab.KIND_BF16, m=m, n=n, k=k, act=ab.ACT_GELU, trans_w=1, dy_dev=ptr(t["dy"]), z_dev=ptr(t["z"]), x_dev=ptr(t["x"]), w_dev=ptr(t["w"]), dx_dev=ptr(t["dx"]),
                          dw_dev=ptr(t["dw"]), dw_dtype=ab.BF16, dbias_dev=ptr(db), workspace_dev=ptr(room), workspace_bytes=room.numel())
    side = C.c_void_p()
    ab.check(ab.lib().ascb200_stream_create(C.byref(side)))
    torch.cuda.synchronize()
    graph = ab.Graph(side, lambda: (ab.check(ab.linear(f, side)), ab.check(ab.linear_grad(b, side))))
    for seed in (3, 4):
        for c in ("x", "w", "dy"):
            t[c].copy_(torch.randn(t[c].shape, generator=gen(seed + ord(c[0]))) * (0.2 if c == "w" else 1))
        torch.cuda.synchronize()
        graph.launch()
        torch.cuda.synchronize()
        x, w, dy, zz = (t[c].double() for c in ("x", "w", "dy", "z"))
        z = x @ w.t()
        near(t["z"], z, 2.0**-8 * z.abs() + 64 * F * (x.abs() @ w.abs().t()), "z")
        dz = dy * act(zz, "gelu")[1]
        err = dy.abs() * 2.0**-17 + 2.0**-8 * 1.01 * dz.abs()
        near(t["dx"], dz @ w, err @ w.abs() + 2.0**-8 * (dz @ w).abs() + 128 * F * (dz.abs() @ w.abs()), "dx")
        near(t["dw"], dz.t() @ x, err.t() @ x.abs() + 2.0**-8 * (dz.t() @ x).abs() + 128 * F * (dz.abs().t() @ x.abs()), "dw")
        near(db, dz.sum(0), (dy.abs() * 2.0**-17 + 128 * F * dz.abs()).sum(0), "dbias")
    graph.destroy()
    ab.lib().ascb200_stream_destroy(side)


@pytest.mark.parametrize("act", ["none", "silu"])
def test_side_by_side_products_in_a_row(act):
    """Gradients back to back on one stream, each reading what the call before wrote: dx of one is dy of the next, and a workspace is shared."""
    dev()
    m, n, k, calls = 200, 136, 136, 12
    g = gen(5)
    w = (torch.randn(n, k, generator=g) / math.sqrt(k)).half().cuda()
    x, z = torch.randn(m, k, generator=g).half().cuda(), torch.randn(m, n, generator=g).half().cuda()
    d = [torch.randn(m, n, generator=g).half().cuda()] + [torch.empty(m, k, device="cuda", dtype=torch.float16) for _ in range(calls)]
    dw, db = torch.empty(calls, n, k, device="cuda", dtype=torch.float16), torch.empty(calls, n, device="cuda")
    room = torch.empty(ab.linear_grad_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for i in range(calls):
        ab.check(ab.linear_grad(ab.LinearGradDesc(kind=ab.KIND_F16, m=m, n=n, k=k, act=ACTS[act], trans_w=1, dy_dev=ptr(d[i]), z_dev=ptr(z), x_dev=ptr(x), w_dev=ptr(w),
                                                  dx_dev=ptr(d[i + 1]), dw_dev=ptr(dw[i]), dw_dtype=ab.F16, dbias_dev=ptr(db[i]), workspace_dev=ptr(room),
                                                  workspace_bytes=room.numel()), stream()))
    torch.cuda.synchronize()
    for i in range(calls):
        # each call against its own input as it was written
        dy = d[i].double()
        dz, wd, xd = dy * globals()["act"](z.double(), act)[1], w.double(), x.double()
        err = 0 if act == "none" else dy.abs() * (2.0**-18 + z.double().abs() * 2.0**-22) + 2.0**-11 * 1.01 * dz.abs() + 2.0**-24
        err = err if torch.is_tensor(err) else torch.zeros_like(dz)
        near(d[i + 1], dz @ wd, err @ wd.abs() + 2.0**-11 * (dz @ wd).abs() + 100 * F * (dz.abs() @ wd.abs()) + TINY[torch.float16], f"dx {i}")
        near(dw[i], dz.t() @ xd, err.t() @ xd.abs() + 2.0**-11 * (dz.t() @ xd).abs() + 100 * F * (dz.abs().t() @ xd.abs()) + TINY[torch.float16], f"dw {i}")
        near(db[i], dz.sum(0), err.sum(0) + 120 * F * dz.abs().sum(0) + 2.0**-149, f"dbias {i}")


@pytest.mark.parametrize("r_pad,z_pad", [(3, None), (0, 1), (None, 5), (7, 3)])
@pytest.mark.parametrize("m,n,trans_w", [(700, 6272, 0), (513, 7488, 1), (1560, 5504, 1)])
def test_last_rows_behind_a_full_tile(m, n, trans_w, r_pad, z_pad):
    """About two tiles per SM, of which the second may be the matrix' last block of at most 64 rows: its residual and z, off 16 bytes, pass
    through shared memory from which the first tile's y may still be on its way."""
    dev()
    for dtype, k in ((torch.bfloat16, 64), (torch.float16, 200), (torch.int8, 64)):
        if dtype == torch.int8 and z_pad is not None:
            continue
        out = torch.bfloat16 if dtype == torch.int8 else dtype
        x, w, xs, ws = operands(m, n, k, dtype, trans_w, 0)
        g = gen(m + n)
        r = None if r_pad is None else torch.randn(m, n, generator=g).to(out)
        rs = None if r is None else rows_in(r, out, r_pad)
        y, z = Out(m, n, out), None if z_pad is None else Out(m, n, out, z_pad)
        d = ab.LinearDesc(kind=KIND[dtype], m=m, n=n, k=k, x_dev=ptr(xs), ldx=xs.stride(0), w_dev=ptr(ws), ldw=ws.stride(0), trans_w=trans_w, y_dev=y.ptr(), ldy=y.ld, y_dtype=CODE[out])
        if r is not None:
            d.residual_dev, d.ld_residual = ptr(rs), n + r_pad
        if z is not None:
            d.z_dev, d.ldz = z.ptr(), z.ld
        xd, wd = x.cuda().double(), w.cuda().double()
        want, mass = xd @ wd.t(), xd.abs() @ wd.abs().t()
        tol = (k / 16 + 32) * 2 * F * mass
        if dtype == torch.int8:
            ch = (torch.rand(n, generator=g) + 0.5).cuda() * 0.001
            d.ch_scale_dev = ptr(ch)
            want = want * ch.double()
            tol = 4 * F * want.abs()
        ab.check(ab.linear(d, stream()))
        torch.cuda.synchronize()
        y.check()
        if z is not None:
            z.check()
            near(z.t, want, tol + (HALF_STEP[out] + 4 * F) * want.abs() + TINY[out], "z")
        if r is not None:
            want = want + r.cuda().double()
        near(y.t, want, tol + (HALF_STEP[out] + 4 * F) * want.abs() + TINY[out], "y")


@pytest.mark.parametrize("name", [a for a in ACTS if a not in ("none", "relu")])  # (the slopes of these are 1, and 1 or 0 by a comparison)
@pytest.mark.parametrize("m", [1, 5, 60])
def test_the_slope_of_nan_is_nan(m, name):
    dev()
    n, k = 24, 16
    z, dy = torch.randn(m, n, generator=gen(m)), torch.randn(m, n, generator=gen(m + 1))
    z[m // 2, 7] = math.nan
    x, w = torch.randn(m, k, generator=gen(m + 2)), torch.randn(n, k, generator=gen(m + 3))
    x, w, dy, z = (t.bfloat16().cuda() for t in (x, w, dy, z))
    dx, dw, db = torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    dx = dx.bfloat16()
    room = torch.empty(ab.linear_grad_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")
    ab.check(ab.linear_grad(ab.LinearGradDesc(kind=ab.KIND_BF16, m=m, n=n, k=k, act=ACTS[name], trans_w=1, dy_dev=ptr(dy), z_dev=ptr(z), x_dev=ptr(x), w_dev=ptr(w), dx_dev=ptr(dx),
                                              dw_dev=ptr(dw), dw_dtype=ab.F32, dbias_dev=ptr(db), dbias_dtype=ab.F32, workspace_dev=ptr(room), workspace_bytes=room.numel()), stream()))
    torch.cuda.synchronize()
    rows, cols = torch.arange(m) == m // 2, torch.arange(n) == 7
    assert torch.equal(torch.isnan(dx).cpu(), rows[:, None].expand(m, k)) and torch.equal(torch.isnan(dw).cpu(), cols[:, None].expand(n, k)) and torch.equal(torch.isnan(db).cpu(), cols)


def normal(z):
    """(upper tail at |z|, density at z) in 64 bits."""
    return 0.5 * torch.erfc(z.abs() / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


# Relative errors of the tail: the exponent's rounding, up to 2.5 * 2^-24 of z^2 / 2 and so 1.25 z^2 2^-24; ex2 2^-22, the fit 1.7e-8, rcp and the polynomial's nine steps, whose
# terms add up to at most three times the result, together under 2^-20; below the normal numbers (from |z| = 13 on) a tail is 0.
def tail_error(z):
    return 2.0**-20 + z * z * 2.0**-23


@pytest.mark.parametrize("m", [2, 300])
def test_gelu_of_far_negative_values(m):
    """GELU is right relative to itself, not to z: its fp32 output shows it."""
    dev()
    z = torch.cat([torch.linspace(-13, 13, 417), torch.tensor([-1e-3, 1e-3, -1e-30, 0.0, -14.0, -40.0, 14.0, 40.0])])
    n = len(z)
    x, w = torch.zeros(m, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, 16, dtype=torch.bfloat16, device="cuda")
    bias, y = z.cuda(), torch.empty(m, n, device="cuda")
    ab.check(ab.linear(ab.LinearDesc(kind=ab.KIND_BF16, m=m, n=n, k=16, x_dev=ptr(x), w_dev=ptr(w), trans_w=1, act=ab.ACT_GELU, bias_dev=ptr(bias), bias_dtype=ab.F32, y_dev=ptr(y),
                                     y_dtype=ab.F32), stream()))
    torch.cuda.synchronize()
    z = z.double()
    tail, _ = normal(z)
    want = torch.where(z > 0, z - z * tail, z * tail)
    tol = (z * tail).abs() * (tail_error(z) + F) + F * want.abs() + 2.0**-122
    near(y, want.expand(m, n), tol.expand(m, n), "y")


@pytest.mark.parametrize("m", [1, 40])
def test_gelu_slope_of_far_negative_values(m):
    dev()
    z = torch.linspace(-13, 13, 417).half()
    n = len(z)
    zs, dy, db = torch.zeros(m, n, dtype=torch.float16, device="cuda"), torch.zeros(m, n, dtype=torch.float16, device="cuda"), torch.empty(n, device="cuda")
    zs[0], dy[0] = z.cuda(), 1.0
    room = torch.empty(ab.linear_grad_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")
    ab.check(ab.linear_grad(ab.LinearGradDesc(kind=ab.KIND_F16, m=m, n=n, k=16, act=ab.ACT_GELU, trans_w=1, dy_dev=ptr(dy), z_dev=ptr(zs), dbias_dev=ptr(db), dbias_dtype=ab.F32,
                                              workspace_dev=ptr(room), workspace_bytes=room.numel()), stream()))
    torch.cuda.synchronize()
    z = z.double()
    tail, phi = normal(z)
    want = torch.where(z > 0, 1 - tail, tail) + z * phi
    near(db, want, (tail + (z * phi).abs()) * (tail_error(z) + 3 * F) + 2 * F * want.abs() + 2.0**-120, "slope")


@pytest.mark.parametrize("name", ["silu", "gelu", "none"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 5, 16, 17, 40])
def test_gradient_with_infinities_in_the_operands(m, dtype, name):
    """An infinity in w or x makes the products that it enters infinite with their sign (two of opposite signs, or one times 0, NaN), on both sides of
    16 rows; the columns beside them are what they are without it."""
    dev()
    n, k = 72, 520
    g = gen(m + 5)
    x, w, dy, z = (torch.randn(a, b, generator=g).to(dtype) for a, b in ((m, k), (n, k), (m, n), (m, n)))
    w[5, 7], w[33, 300], w[5, 301], w[6, 301], w[60, 519] = math.inf, -math.inf, math.inf, math.inf, math.nan
    x[m // 2, 9], x[0, 256], x[m - 1, 511] = -math.inf, math.inf, math.nan
    xs, ws, ds, zs = x.cuda(), w.cuda(), dy.cuda(), z.cuda()
    dx, dw = Out(m, k, dtype), Out(n, k, torch.float32)
    room = torch.empty(ab.linear_grad_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")
    ab.check(ab.linear_grad(ab.LinearGradDesc(kind=KIND[dtype], m=m, n=n, k=k, act=ACTS[name], trans_w=1, dy_dev=ptr(ds), z_dev=ptr(zs), x_dev=ptr(xs), w_dev=ptr(ws), dx_dev=dx.ptr(),
                                              dw_dev=dw.ptr(), dw_dtype=ab.F32, workspace_dev=ptr(room), workspace_bytes=room.numel()), stream()))
    torch.cuda.synchronize()
    dx.check()
    dw.check()
    x, w, dy, z = x.double(), w.double(), dy.double(), z.double()
    dz = dy * act(z, name)[1]
    xf, wf = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)).abs() for t in (x, w))  # what the tolerances count
    err = torch.zeros_like(dz) if name == "none" else dy.abs() * (2.0**-18 + z.abs() * 2.0**-22) + F * dz.abs()
    half = HALF_STEP[dtype] ** 2 if m <= 16 else HALF_STEP[dtype]
    err = err + (0 if name == "none" else half * (dz.abs() + err) + 2 * TINY[dtype])
    want = dz @ w
    top = 65504.0 if dtype == torch.float16 else math.inf  # F16 outputs saturate
    finite = torch.where(torch.isfinite(want), want, torch.zeros_like(want)).abs()
    near(dx.t, want.clamp(-top, top), err @ wf + (n / 16 + 32) * 2 * F * (dz.abs() @ wf) * 1.01 + HALF_STEP[dtype] * finite + TINY[dtype], "dx")
    want = dz.t() @ x
    finite = torch.where(torch.isfinite(want), want, torch.zeros_like(want)).abs()
    near(dw.t, want, err.t() @ xf + (m / 16 + 32) * 2 * F * (dz.abs().t() @ xf) * 1.01 + F * finite + 2.0**-149, "dw")
