"""ascb200_rms_norm / ascb200_rms_norm_grad against their formulas in 64 bits.

Tolerances.  Everything is computed in fp32 and rounded once to the output type.  A row's sum of squares of k terms is at most 32
additions per thread and ten more across threads: relative error under 64 * 2^-24, half of it in rstd; with the three products of y
fewer than 48 * 2^-24 of |y|.  On top comes half a step of the output type.
"""
import ctypes as C
import math

import pytest
import torch

import ascb200 as ab
from torch_util import CODE, HALF_STEP, TINY, TORCH, Out, dev, near, ptr, rows_in, stream

pytestmark = pytest.mark.gpu
F = 2.0**-24
EPS = 1e-6


def gen(seed):
    return torch.Generator().manual_seed(seed)


def reference(x, r, gamma, eps=EPS):
    h = x.double() if r is None else x.double() + r.double()
    rstd = 1 / torch.sqrt((h * h).mean(1) + eps)
    y = h * rstd[:, None]
    return h, rstd, y if gamma is None else y * gamma.double()


def forward(m, k, dtype, residual=True, gamma="same", pad=0, offset=0, q=None, mode=ab.SCALE_PER_TOKEN, group=0, y=True, seed=0, x=None, r=None, scale=1.0):
    dev()
    g = gen(seed + 1000 * m + k)
    x = (torch.randn(m, k, generator=g) * scale).to(dtype) if x is None else x
    r = (torch.randn(m, k, generator=g) * 2 * scale).to(dtype) if residual and r is None else r
    w = None if gamma is None else (1 + 0.3 * torch.randn(k, generator=g)).to(dtype if gamma == "same" else torch.float32)
    xs, rs = rows_in(x, dtype, pad, offset), None if r is None else rows_in(r, dtype, pad, offset)
    ws = None if w is None else w.cuda()
    out = {"sum": Out(m, k, dtype, pad, offset), "rstd": torch.full((m + 1,), 5.5, device="cuda")}
    d = ab.RmsNormDesc(m=m, k=k, dtype=CODE[dtype], gamma_dtype=0 if w is None else CODE[w.dtype], x_dev=ptr(xs), ldx=k + pad, residual_dev=ptr(rs), ld_residual=k + pad,
                       gamma_dev=ptr(ws), sum_dev=out["sum"].ptr(), ld_sum=k + pad, rstd_dev=ptr(out["rstd"]), eps=EPS)
    if y:
        out["y"] = Out(m, k, dtype, pad, offset)
        d.y_dev, d.ldy = out["y"].ptr(), k + pad
    if q is not None:
        out["q"] = Out(m, k, q, pad, offset)
        groups = 1 if mode == ab.SCALE_PER_TOKEN else -(-k // (group or 32))
        out["scale"] = torch.full((m + 1, groups), 99, device="cuda", dtype=torch.uint8 if mode == ab.SCALE_MX else torch.float32)
        d.q_dev, d.ldq, d.scale_dev, d.q_dtype, d.scale_mode, d.group_size = out["q"].ptr(), k + pad, ptr(out["scale"]), CODE[q], mode, group
    ab.check(ab.rms_norm(d, stream()))
    torch.cuda.synchronize()
    for o in out.values():
        if isinstance(o, Out):
            o.check()
    assert float(out["rstd"][m]) == 5.5
    return x, r, w, out


def check_floats(x, r, w, out, dtype):
    h, rstd, y = reference(x, r, w)
    near(out["sum"].t, h, (HALF_STEP[dtype] + F) * h.abs() + TINY[dtype], "sum")
    near(out["rstd"][: len(rstd)], rstd, 40 * F * rstd, "rstd")
    if "y" in out:
        near(out["y"].t, y, (HALF_STEP[dtype] + 48 * F) * y.abs() + TINY[dtype], "y")
    return y


def check_codes(y, out, q, mode, group):
    m, k = y.shape
    width = {ab.SCALE_PER_TOKEN: k, ab.SCALE_MX: 32}.get(mode, group)
    groups = -(-k // width)
    blocks = torch.nn.functional.pad(y, (0, groups * width - k)).view(m, groups, width)
    top = blocks.abs().amax(2)
    codes = torch.nn.functional.pad(out["q"].t.cpu().double(), (0, groups * width - k)).view(m, groups, width)
    if mode == ab.SCALE_MX:
        byte = out["scale"][:m].cpu().long()
        want = (torch.floor(torch.log2(top.clamp(min=2.0**-140))).long() - 8 + 127).clamp(min=0)
        # a largest value within rounding of a power of two may fall on either side of it
        edge = (top * (1 + 64 * F)).log2().floor() != (top * (1 - 64 * F)).log2().floor()
        assert ((byte == want) | edge | (top == 0)).all()
        scale = torch.exp2(byte.double() - 127)
        v = (blocks / scale[:, :, None]).clamp(-448, 448)
        near(codes, v, (v.abs() * 2.0**-4).clamp(min=2.0**-10) * (1 + 1e-4) + v.abs() * 64 * F, "codes")
        return
    assert (out["scale"][m] == 99).all()
    scale = out["scale"][:m].cpu().double()
    near(scale, top / (127 if q == torch.int8 else 448), 64 * F * top, "scale")
    v = torch.where(scale[:, :, None] > 0, blocks / scale[:, :, None].clamp(min=1e-300), torch.zeros_like(blocks))
    if q == torch.int8:
        near(codes, v, 0.5 + 127 * 64 * F, "codes")
    else:
        near(codes, v.clamp(-448, 448), (v.abs() * 2.0**-4).clamp(min=2.0**-10) * (1 + 1e-4) + v.abs() * 64 * F, "codes")


@pytest.mark.parametrize("dtype", TORCH)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 8), (2, 255), (4, 257), (9, 512), (1, 1024), (3, 1025), (2, 2048), (7, 4096), (1, 4100), (3, 8192), (2, 8200), (2, 16384),
                                 (1, 20001), (1, 32768)])
def test_forward_sizes(m, k, dtype):
    x, r, w, out = forward(m, k, TORCH[dtype])
    check_floats(x, r, w, out, TORCH[dtype])


@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (3, 0), (8, 1), (0, 3)])
@pytest.mark.parametrize("k", [96, 101, 2050])
@pytest.mark.parametrize("dtype", TORCH)
def test_forward_strides_and_alignment(dtype, k, pad, offset):
    x, r, w, out = forward(6, k, TORCH[dtype], pad=pad, offset=offset, q=torch.int8)
    check_codes(check_floats(x, r, w, out, TORCH[dtype]), out, torch.int8, ab.SCALE_PER_TOKEN, 0)


@pytest.mark.parametrize("k", [1, 2, 7, 63, 250, 255, 257, 300, 509, 1022, 2047, 4098, 7167, 16383, 32767])
@pytest.mark.parametrize("pad,offset", [(0, 0), (0, 1), (1, 0), (1, 1), (2, 1), (5, 6)])
def test_forward_in_pairs(k, pad, offset):
    """Rows of every parity, alternating ones among them, with and without codes, whose own rows may lie otherwise."""
    for dtype in (torch.bfloat16, torch.float16):
        x, r, w, out = forward(5, k, dtype, pad=pad, offset=offset, gamma="f32" if k % 2 else "same", q=torch.int8 if k % 3 else torch.float8_e4m3fn)
        check_codes(check_floats(x, r, w, out, dtype), out, torch.int8 if k % 3 else torch.float8_e4m3fn, ab.SCALE_PER_TOKEN, 0)


def test_forward_with_rows_that_lie_differently():
    """x and y on other parities: element by element."""
    dev()
    for ldx, ldy in ((100, 101), (101, 100), (101, 103), (102, 104)):
        x = rows_in(torch.randn(9, 99, generator=gen(ldx)), torch.bfloat16, ldx - 99)
        y = Out(9, 99, torch.bfloat16, ldy - 99)
        ab.check(ab.rms_norm(ab.RmsNormDesc(m=9, k=99, dtype=ab.BF16, x_dev=ptr(x), ldx=ldx, y_dev=y.ptr(), ldy=ldy, eps=EPS), stream()))
        torch.cuda.synchronize()
        y.check()
        want = reference(x.cpu(), None, None)[2]
        near(y.t, want, (2.0**-8 + 48 * F) * want.abs(), "y")


@pytest.mark.parametrize("residual,gamma,y", [(False, "same", True), (True, None, True), (False, "f32", False), (True, "f32", True)])
def test_forward_without_residual_or_gamma(residual, gamma, y):
    for dtype in TORCH.values():
        x, r, w, out = forward(5, 520, dtype, residual=residual, gamma=gamma, y=y, q=torch.float8_e4m3fn)
        check_codes(check_floats(x, r, w, out, dtype), out, torch.float8_e4m3fn, ab.SCALE_PER_TOKEN, 0)


FORMS = [(torch.int8, ab.SCALE_PER_TOKEN, 0), (torch.float8_e4m3fn, ab.SCALE_PER_TOKEN, 0), (torch.int8, ab.SCALE_PER_GROUP, 32), (torch.int8, ab.SCALE_PER_GROUP, 256),
         (torch.float8_e4m3fn, ab.SCALE_PER_GROUP, 64), (torch.float8_e4m3fn, ab.SCALE_PER_GROUP, 128), (torch.float8_e4m3fn, ab.SCALE_MX, 0),
         (torch.float8_e4m3fn, ab.SCALE_MX, 32)]


@pytest.mark.parametrize("q,mode,group", FORMS)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 31), (4, 64), (2, 300), (3, 1000), (2, 2056), (33, 4096), (2, 8191), (1, 16384), (1, 30000)])
def test_codes_and_scales(m, k, q, mode, group):
    dtype = (torch.float32, torch.float16, torch.bfloat16)[(m + k) % 3]
    x, r, w, out = forward(m, k, dtype, q=q, mode=mode, group=group)
    check_codes(check_floats(x, r, w, out, dtype), out, q, mode, group)


@pytest.mark.parametrize("q,mode,group", FORMS)
def test_zero_rows_and_groups(q, mode, group):
    x = torch.randn(4, 600, generator=gen(3))
    x[1] = 0
    x[2, 256:512] = 0
    _, _, _, out = forward(4, 600, torch.float32, residual=False, gamma=None, q=q, mode=mode, group=group, x=x)
    assert (out["q"].t[1].float() == 0).all() and (out["scale"][1] == 0).all() and (out["y"].t[1] == 0).all()
    assert (out["q"].t[2, 256:512].float() == 0).all()
    check_codes(check_floats(x, None, None, out, torch.float32), out, q, mode, group)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_bad_value_shows_in_its_row_only(bad):
    x = torch.randn(3, 1000, generator=gen(4))
    x[1, 17] = bad
    clean = x.clone()
    clean[1] = 0
    for q, mode, group in FORMS:
        _, _, _, out = forward(3, 1000, torch.bfloat16, residual=False, q=q, mode=mode, group=group, x=x.bfloat16(), gamma=None)
        _, _, _, ref = forward(3, 1000, torch.bfloat16, residual=False, q=q, mode=mode, group=group, x=clean.bfloat16(), gamma=None)
        assert torch.isnan(out["y"].t[1, 17])
        assert out["scale"][1, 0] == 255 if mode == ab.SCALE_MX else torch.isnan(out["scale"][1, 0])
        for name in ("y", "q"):
            assert torch.equal(out[name].t[[0, 2]].float(), ref[name].t[[0, 2]].float())
        assert torch.equal(out["scale"][[0, 2]], ref["scale"][[0, 2]])


@pytest.mark.parametrize("k", [1000, 1001])
@pytest.mark.parametrize("mode,group", [(ab.SCALE_PER_TOKEN, 0), (ab.SCALE_PER_GROUP, 64)])
def test_int8_codes_beside_an_infinite_product_are_zero(mode, group, k):
    dev()
    x, w = torch.ones(1, k, dtype=torch.bfloat16, device="cuda"), torch.ones(k, device="cuda")
    w[3] = math.inf
    q, scale = torch.full((1, k), 9, dtype=torch.int8, device="cuda"), torch.zeros(1, -(-k // (group or k)), device="cuda")
    d = ab.RmsNormDesc(m=1, k=k, dtype=ab.BF16, gamma_dtype=ab.F32, x_dev=ptr(x), gamma_dev=ptr(w), q_dev=ptr(q), scale_dev=ptr(scale), q_dtype=ab.S8, scale_mode=mode,
                       group_size=group, eps=EPS)
    ab.check(ab.rms_norm(d, stream()))
    torch.cuda.synchronize()
    assert float(scale[0, 0]) == math.inf
    assert (q[0, : group or k] == 0).all()
    assert group == 0 or (q[0, group:] == 127).all()


def test_extreme_magnitudes():
    # tiny rows under eps, large rows whose squares still fit, halves that saturate
    x = torch.tensor([1e-30, 1e-6, 1.0, 1e15])[:, None] * torch.randn(4, 300, generator=gen(5))
    x, r, w, out = forward(4, 300, torch.float32, residual=False, gamma=None, x=x, q=torch.int8)
    check_codes(check_floats(x, r, w, out, torch.float32), out, torch.int8, ab.SCALE_PER_TOKEN, 0)
    x, r = torch.full((1, 64), 60000.0).half(), torch.full((1, 64), 60000.0).half()
    _, _, _, out = forward(1, 64, torch.float16, gamma=None, x=x, r=r)
    assert (out["sum"].t == 65504).all() and (out["y"].t == 1).all()


@pytest.mark.parametrize("q", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("k", [64, 1001, 4096])
def test_codes_of_tiny_rows(k, q):
    # |y| near 1e-36 from |h| near 1e-2: the codes' factor, rstd / scale, is beyond fp32
    dev()
    x, w = torch.randn(3, k, generator=gen(8)) * 0.01, torch.full((k,), 1e-36)
    _, _, y = reference(x, None, w, 0.0)
    xs, ws, codes, scale = x.cuda(), w.cuda(), torch.empty(3, k, dtype=q, device="cuda"), torch.empty(3, device="cuda")
    ab.check(ab.rms_norm(ab.RmsNormDesc(m=3, k=k, dtype=ab.F32, gamma_dtype=ab.F32, x_dev=ptr(xs), gamma_dev=ptr(ws), q_dev=ptr(codes), scale_dev=ptr(scale), q_dtype=CODE[q],
                                        scale_mode=ab.SCALE_PER_TOKEN), stream()))
    torch.cuda.synchronize()
    top = 127 if q == torch.int8 else 448
    want = y.abs().amax(1) / top
    kept = want > 2.0**-126
    # h * gamma near 1e-38 is below the normal numbers: a step is 2^-149, so its half is up to 2^-24 of the largest of a row and more of its smaller values
    near(scale, torch.where(kept, want, torch.zeros_like(want)), 64 * F * want + 200 * 2.0**-149 / top, "scale")
    v = torch.where(kept[:, None], y / want[:, None], torch.zeros_like(y))
    step = 200 * 2.0**-149 / want.clamp(min=2.0**-126)[:, None]  # rstd is near 100
    near(codes.float(), v, (0.5 if q == torch.int8 else (v.abs() * 2.0**-4).clamp(min=2.0**-10) * (1 + 1e-4)) + v.abs() * 64 * F + step, "codes")


def test_in_place():
    dev()
    x, r = torch.randn(37, 1030, generator=gen(6)).bfloat16().cuda(), torch.randn(37, 1030, generator=gen(7)).bfloat16().cuda()
    h, _, y = reference(x.cpu(), r.cpu(), None)
    d = ab.RmsNormDesc(m=37, k=1030, dtype=ab.BF16, x_dev=ptr(x), residual_dev=ptr(r), sum_dev=ptr(r), y_dev=ptr(x), eps=EPS)
    ab.check(ab.rms_norm(d, stream()))
    torch.cuda.synchronize()
    near(r, h, (2.0**-8 + F) * h.abs(), "sum over the residual")
    near(x, y, (2.0**-8 + 48 * F) * y.abs(), "y over x")


# ---- gradients -----------------------------------------------------------------------------------------------------------------
def grad_reference(dy, h, rstd, gamma, dh):
    """By autograd in 64 bits, with the saved rstd in its place: the formula's own derivative is checked below by differences."""
    dy, h, rstd = dy.double(), h.double(), rstd.double()[:, None]
    g = dy if gamma is None else dy * gamma.double()
    hat = h * rstd
    dx = rstd * (g - hat * (g * hat).mean(1, keepdim=True))
    terms = rstd * (g.abs() + hat.abs() * (g * hat).abs().mean(1, keepdim=True))
    return dx if dh is None else dx + dh.double(), (dy * hat).sum(0), terms + (0 if dh is None else dh.double().abs()), (dy * hat).abs().sum(0)


def backward(m, k, dtype, gamma="same", dh=True, pad=0, offset=0, dgamma=torch.float32, seed=0):
    dev()
    g = gen(seed + 77 * m + k)
    h, dy = (torch.randn(m, k, generator=g) * 2).to(dtype), torch.randn(m, k, generator=g).to(dtype)
    e = torch.randn(m, k, generator=g).to(dtype) if dh else None
    w = None if gamma is None else (1 + 0.3 * torch.randn(k, generator=g)).to(dtype if gamma == "same" else torch.float32)
    rstd = (1 / torch.sqrt(h.double().square().mean(1) + EPS)).float()
    hs, ds, es = rows_in(h, dtype, pad, offset), rows_in(dy, dtype, pad, offset), None if e is None else rows_in(e, dtype, pad, offset)
    ws, rs = None if w is None else w.cuda(), rstd.cuda()
    dx = Out(m, k, dtype, pad, offset)
    size = ab.rms_norm_grad_workspace_bytes(m, k)
    room = torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN: nothing of it may be read before it is written
    dg = None if dgamma is None else Out(1, k, dgamma)
    d = ab.RmsNormGradDesc(m=m, k=k, dtype=CODE[dtype], gamma_dtype=0 if w is None else CODE[w.dtype], dy_dev=ptr(ds), ld_dy=k + pad, h_dev=ptr(hs), ldh=k + pad,
                           rstd_dev=ptr(rs), gamma_dev=ptr(ws), dh_dev=ptr(es), ld_dh=k + pad, dx_dev=dx.ptr(), ld_dx=k + pad, workspace_dev=ptr(room), workspace_bytes=size)
    if dg is not None:
        d.dgamma_dev, d.dgamma_dtype = dg.ptr(), CODE[dgamma]
    ab.check(ab.rms_norm_grad(d, stream()))
    torch.cuda.synchronize()
    dx.check()
    assert (room[size:] == 0xFF).all()
    want, wantg, terms, gterms = grad_reference(dy, h, rstd, w, e)
    # the mean of g * hat: up to 64 roundings of its terms; the rest a handful of products and sums of `terms`
    near(dx.t, want, HALF_STEP[dtype] * want.abs() + 72 * F * terms + TINY[dtype], "dx")
    if dg is not None:
        dg.check()
        # m terms added over at most m / blocks + blocks / 8 + 8 steps, with at least 148 blocks for so many rows
        steps = m / min(m, 148) + 64
        near(dg.t[0], wantg, HALF_STEP[dgamma] * wantg.abs() + steps * F * gterms + TINY[dgamma], "dgamma")


@pytest.mark.parametrize("dtype", TORCH)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (13, 255), (9, 257), (300, 512), (17, 1000), (5, 2048), (700, 2050), (3, 4096), (310, 5000), (2, 8200), (2, 16384), (3, 20001),
                                 (1, 32768)])
def test_gradient_sizes(m, k, dtype):
    backward(m, k, TORCH[dtype])


@pytest.mark.parametrize("gamma,dh,dgamma,pad,offset", [(None, False, torch.float32, 0, 0), ("f32", True, torch.bfloat16, 8, 8), ("same", False, None, 3, 1), ("same", True, torch.bfloat16, 0, 1),
                                                        ("f32", False, torch.float32, 8, 0)])
@pytest.mark.parametrize("k", [104, 1027, 3000])
def test_gradient_forms(k, gamma, dh, dgamma, pad, offset):
    backward(40, k, torch.bfloat16, gamma=gamma, dh=dh, dgamma=dgamma, pad=pad, offset=offset)


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 70, 601])
@pytest.mark.parametrize("k,pad,offset", [(2, 0, 0), (255, 0, 1), (257, 0, 0), (509, 1, 1), (511, 0, 0), (511, 2, 3), (513, 0, 0), (1023, 0, 0), (1026, 1, 0), (3001, 0, 1), (512, 1, 0), (512, 1, 1)])
def test_gradient_in_pairs(m, k, pad, offset):
    backward(m, k, torch.bfloat16, gamma="f32" if m % 2 else "same", pad=pad, offset=offset)
    backward(m, k, torch.float16, dh=False, pad=pad, offset=offset, dgamma=torch.float16)


@pytest.mark.parametrize("dh,pad,offset", [(True, 0, 0), (False, 8, 8), (True, 0, 1)])
@pytest.mark.parametrize("dtype", TORCH)
@pytest.mark.parametrize("m,k", [(20011, 96), (9001, 328), (9001, 519), (5003, 1040), (2500, 2056), (1300, 4104), (900, 8208), (900, 8201), (300, 16400), (4200, 1500), (4200, 3001)])
def test_gradient_of_many_rows(m, k, dtype, dh, pad, offset):
    backward(m, k, TORCH[dtype], dh=dh, pad=pad, offset=offset)


@pytest.mark.parametrize("over", ["dy", "h", "dh"])
@pytest.mark.parametrize("dtype", TORCH)
@pytest.mark.parametrize("m,k", [(3000, 200), (2000, 776), (1700, 1999), (1500, 4096), (700, 8200), (500, 9003), (300, 16392)])
def test_gradient_in_place(m, k, dtype, over):
    dev()
    dtype = TORCH[dtype]
    g = gen(m + k)
    t = {c: torch.randn(m, k, generator=g).to(dtype).cuda() for c in ("dy", "h", "dh")}
    rstd = (1 / torch.sqrt(t["h"].double().square().mean(1) + EPS)).float()
    gamma = (1 + 0.3 * torch.randn(k, generator=g)).cuda()
    want, _, terms, _ = grad_reference(t["dy"], t["h"], rstd, gamma, t["dh"])
    d = ab.RmsNormGradDesc(m=m, k=k, dtype=CODE[dtype], gamma_dtype=ab.F32, dy_dev=ptr(t["dy"]), h_dev=ptr(t["h"]), rstd_dev=ptr(rstd), gamma_dev=ptr(gamma), dh_dev=ptr(t["dh"]),
                           dx_dev=ptr(t[over]))
    ab.check(ab.rms_norm_grad(d, stream()))
    torch.cuda.synchronize()
    near(t[over], want, HALF_STEP[dtype] * want.abs() + 72 * F * terms + TINY[dtype], "dx over " + over)


def test_gradient_against_differences():
    """dx and dgamma of the operators themselves: (f(h + d) - f(h - d)) / 2 over the forward call, in fp32."""
    dev()
    k, step = 48, 2.0**-7
    g = gen(8)
    h, dy, w = torch.randn(1, k, generator=g), torch.randn(1, k, generator=g), 1 + 0.3 * torch.randn(k, generator=g)

    def y(hs, ws):
        """Rows of values through the forward call, one gamma per call."""
        hs, ws = hs.cuda().contiguous(), ws.cuda()
        out, rstd = torch.empty_like(hs), torch.empty(len(hs), device="cuda")
        ab.check(ab.rms_norm(ab.RmsNormDesc(m=len(hs), k=k, x_dev=ptr(hs), gamma_dev=ptr(ws), y_dev=ptr(out), rstd_dev=ptr(rstd), eps=EPS), stream()))
        torch.cuda.synchronize()
        return out.cpu().double(), rstd

    _, rstd = y(h, w)
    dx, dg = torch.empty(1, k, device="cuda"), torch.empty(k, device="cuda")
    room = torch.empty(ab.rms_norm_grad_workspace_bytes(1, k), dtype=torch.uint8, device="cuda")
    hs, ds, ws = h.cuda(), dy.cuda(), w.cuda()
    ab.check(ab.rms_norm_grad(ab.RmsNormGradDesc(m=1, k=k, dy_dev=ptr(ds), h_dev=ptr(hs), rstd_dev=ptr(rstd), gamma_dev=ptr(ws), dx_dev=ptr(dx), dgamma_dev=ptr(dg),
                                                 workspace_dev=ptr(room), workspace_bytes=room.numel()), stream()))
    torch.cuda.synchronize()
    eye = torch.eye(k) * step
    up, down = y(h + eye, w)[0], y(h - eye, w)[0]
    slope = ((up - down) @ dy[0].double()) / (2 * step)
    # the third derivative of y is under 20 in these units: step^2 / 6 * 20 * |dy|; fp32 noise 2^-22 / step of it
    near(dx[0], slope, (step**2 * 4 + 2.0**-21 / step) * float(dy.abs().sum()), "dx by differences")
    both = torch.stack([(y(h, w + eye[i])[0] - y(h, w - eye[i])[0])[0] @ dy[0].double() / (2 * step) for i in range(k)])
    near(dg, both, 2.0**-21 / step * float(dy.abs().sum()), "dgamma by differences")


def test_gradient_of_no_rows_is_zero():
    dev()
    dg = torch.full((40,), 3.0, device="cuda")
    ab.check(ab.rms_norm_grad(ab.RmsNormGradDesc(m=0, k=40, dgamma_dev=ptr(dg)), stream()))
    ab.check(ab.rms_norm(ab.RmsNormDesc(m=0, k=40, eps=EPS), stream()))
    torch.cuda.synchronize()
    assert (dg == 0).all()


# ---- calls ---------------------------------------------------------------------------------------------------------------------
def test_refusals():
    dev()
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    q, s = torch.zeros(4, 64, device="cuda", dtype=torch.int8), torch.zeros(4, device="cuda")

    def rc(**kw):
        f = dict(m=4, k=64, dtype=ab.BF16, x_dev=ptr(x), y_dev=ptr(x), eps=EPS) | kw
        d = ab.RmsNormDesc(**{n: v for n, v in f.items() if n != "reserved"})
        if "reserved" in kw:
            d.reserved[1] = kw["reserved"]
        return ab.rms_norm(d, stream())

    assert rc() == 0
    assert rc(m=-1) == ab.EINVAL and rc(k=0) == ab.EINVAL and rc(x_dev=None) == ab.EINVAL and rc(y_dev=None) == ab.EINVAL and rc(ldx=63) == ab.EINVAL
    assert rc(ldy=72) == ab.EINVAL and rc(residual_dev=ptr(x), sum_dev=ptr(x), y_dev=ptr(q), ld_sum=72) == ab.EINVAL
    assert rc(eps=-1.0) == ab.EINVAL and rc(eps=float("nan")) == ab.EINVAL and rc(reserved=1) == ab.EINVAL and rc(sum_dev=ptr(x)) == ab.EINVAL
    assert rc(dtype=ab.S8) == ab.EUNSUPPORTED and rc(gamma_dev=ptr(x), gamma_dtype=ab.F16) == ab.EUNSUPPORTED
    assert rc(k=32769, ldx=0) == ab.ETOOBIG and rc(x_dev=ptr(x) + 1) == ab.EALIGN and rc(rstd_dev=ptr(s) + 2) == ab.EALIGN
    assert rc(q_dev=ptr(q), q_dtype=ab.S8) == ab.EINVAL                                               # no scale
    assert rc(q_dev=ptr(q), q_dtype=ab.FP8_E5M2, scale_dev=ptr(s)) == ab.EUNSUPPORTED
    assert rc(q_dev=ptr(q), q_dtype=ab.S8, scale_dev=ptr(s), group_size=32) == ab.EINVAL
    assert rc(q_dev=ptr(q), q_dtype=ab.S8, scale_dev=ptr(s), scale_mode=ab.SCALE_PER_GROUP, group_size=48) == ab.EUNSUPPORTED
    assert rc(q_dev=ptr(q), q_dtype=ab.S8, scale_dev=ptr(s), scale_mode=ab.SCALE_MX) == ab.EUNSUPPORTED
    assert rc(q_dev=ptr(q), q_dtype=ab.S8, scale_dev=ptr(s), scale_mode=3) == ab.EINVAL
    assert rc(q_dev=ptr(q), q_dtype=ab.S8, scale_dev=ptr(s) + 1) == ab.EALIGN
    assert ab.lib().ascb200_rms_norm(None, None) == ab.EINVAL

    room = torch.zeros(ab.rms_norm_grad_workspace_bytes(4, 64), device="cuda", dtype=torch.uint8)
    dg = torch.zeros(64, device="cuda")

    def grad(**kw):
        f = dict(m=4, k=64, dtype=ab.BF16, dy_dev=ptr(x), h_dev=ptr(x), rstd_dev=ptr(s), dx_dev=ptr(x), dgamma_dev=ptr(dg), workspace_dev=ptr(room), workspace_bytes=room.numel())
        return ab.rms_norm_grad(ab.RmsNormGradDesc(**(f | kw)), stream())

    assert grad() == 0
    for name in ("dy_dev", "h_dev", "rstd_dev", "dx_dev", "workspace_dev"):
        assert grad(**{name: None}) == ab.EINVAL
    assert grad(ld_dx=72) == ab.EINVAL and grad(workspace_bytes=room.numel() - 1) == ab.EINVAL and grad(workspace_dev=ptr(room) + 4) == ab.EALIGN and grad(ld_dx=63) == ab.EINVAL
    assert grad(k=40000) == ab.ETOOBIG and grad(dgamma_dtype=ab.F16) == ab.EUNSUPPORTED and grad(reserved=1) == ab.EINVAL and grad(dtype=ab.S32) == ab.EUNSUPPORTED
    assert ab.lib().ascb200_rms_norm_grad(None, None) == ab.EINVAL
    torch.cuda.synchronize()


def test_captured_and_replayed():
    """Forward and backward in one graph, replayed on new inputs in the same buffers; two graphs with a workspace each."""
    dev()
    m, k = 300, 1536
    side = C.c_void_p()
    ab.check(ab.lib().ascb200_stream_create(C.byref(side)))
    sets = []
    for i in range(2):
        b = {n: torch.zeros(m, k, device="cuda") for n in ("x", "y", "dy", "dx")}
        b |= {"rstd": torch.zeros(m, device="cuda"), "w": torch.ones(k, device="cuda"), "dg": torch.zeros(k, device="cuda"),
              "room": torch.zeros(ab.rms_norm_grad_workspace_bytes(m, k), device="cuda", dtype=torch.uint8)}
        f = ab.RmsNormDesc(m=m, k=k, x_dev=ptr(b["x"]), gamma_dev=ptr(b["w"]), y_dev=ptr(b["y"]), rstd_dev=ptr(b["rstd"]), eps=EPS)
        g = ab.RmsNormGradDesc(m=m, k=k, dy_dev=ptr(b["dy"]), h_dev=ptr(b["x"]), rstd_dev=ptr(b["rstd"]), gamma_dev=ptr(b["w"]), dx_dev=ptr(b["dx"]), dgamma_dev=ptr(b["dg"]),
                               workspace_dev=ptr(b["room"]), workspace_bytes=b["room"].numel())
        torch.cuda.synchronize()

        def both():
            ab.check(ab.rms_norm(f, side))
            ab.check(ab.rms_norm_grad(g, side))

        sets.append((b, ab.Graph(side, both)))
    for seed in (1, 2):
        for i, (b, graph) in enumerate(sets):
            b["x"].copy_(torch.randn(m, k, generator=gen(seed + 10 * i)))
            b["dy"].copy_(torch.randn(m, k, generator=gen(seed + 10 * i + 5)))
        torch.cuda.synchronize()
        for _, graph in sets:
            graph.launch()
        torch.cuda.synchronize()
        for b, _ in sets:
            x, dy = b["x"].cpu(), b["dy"].cpu()
            _, rstd, y = reference(x, None, None)
            near(b["y"], y, 49 * F * y.abs(), "y")
            want, wantg, terms, gterms = grad_reference(dy, x, rstd, None, None)
            near(b["dx"], want, F * want.abs() + 120 * F * terms, "dx")
            near(b["dg"], wantg, 120 * F * gterms, "dgamma")
    for _, graph in sets:
        graph.destroy()
    ab.lib().ascb200_stream_destroy(side)


def test_same_inputs_give_the_same_bits():
    dev()
    m, k = 5000, 1024
    h, dy = torch.randn(m, k, generator=gen(9)).cuda(), torch.randn(m, k, generator=gen(10)).cuda()
    rstd, w = torch.rand(m, generator=gen(11)).cuda() + 0.5, torch.ones(k, device="cuda")
    first = None
    for _ in range(3):
        dx, dg = torch.empty_like(h), torch.empty(k, device="cuda")
        room = torch.empty(ab.rms_norm_grad_workspace_bytes(m, k), dtype=torch.uint8, device="cuda")
        ab.check(ab.rms_norm_grad(ab.RmsNormGradDesc(m=m, k=k, dy_dev=ptr(dy), h_dev=ptr(h), rstd_dev=ptr(rstd), gamma_dev=ptr(w), dx_dev=ptr(dx), dgamma_dev=ptr(dg),
                                                     workspace_dev=ptr(room), workspace_bytes=room.numel()), stream()))
        torch.cuda.synchronize()
        first = first or (dx, dg)
        assert torch.equal(dx, first[0]) and torch.equal(dg, first[1])


@pytest.mark.parametrize("pad,offset", [(0, 0), (0, 1), (1, 0), (1, 1), (2, 1)])
@pytest.mark.parametrize("m,k", [(1, 8193), (2, 8197), (400, 8201), (301, 12289), (299, 16381)])
def test_gradient_of_long_rows_in_pairs(m, k, pad, offset):
    """Rows of either parity through the ring in shared memory, with threads whose pairs lie behind the row's end."""
    backward(m, k, torch.bfloat16, pad=pad, offset=offset)
    backward(m, k, torch.float16, dh=False, gamma="f32", pad=pad, offset=offset)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (1, 1), (2, 1), (8, 0), (3, 5)])
@pytest.mark.parametrize("k", [32760, 32761, 32766, 32768])
def test_the_longest_rows_at_every_place(k, pad, offset, residual):
    for dtype in (torch.bfloat16, torch.float16):
        x, r, w, out = forward(3, k, dtype, residual=residual, pad=pad, offset=offset, gamma="f32")
        check_floats(x, r, w, out, dtype)
        x, r, w, out = forward(2, k, dtype, residual=residual, pad=pad, offset=offset, q=torch.int8, y=False)
        h, _, y = reference(x, r, w)
        near(out["sum"].t, h, (HALF_STEP[dtype] + F) * h.abs() + TINY[dtype], "sum")
        check_codes(y, out, torch.int8, ab.SCALE_PER_TOKEN, 0)
        backward(3, k, dtype, pad=pad, offset=offset, dh=residual)
