"""ascb200_route / ascb200_route_grad against their formulas in 64 bits.

Tolerances.  Softmax in fp32: the exponent (x - max) log2(e) carries a rounding of 2^-24 of its size, so exp of it a relative error of
2^-24 |x - max| 1.5 and the two units in the last place of ex2; the sum over E experts at most E / 32 + 5 roundings, the quotient two.
"""
import ctypes as C
import math

import pytest
import torch

import ascb200 as ab
from torch_util import CODE, HALF_STEP, TINY, TORCH, Out, dev, near, ptr, rows_in, stream

pytestmark = pytest.mark.gpu
F = 2.0**-24
INF = math.inf


def gen(seed):
    return torch.Generator().manual_seed(seed)


def reference(x, valid, top_k, renorm):
    x = x.double()
    t, e = x.shape
    open_ = x != -INF
    if valid is not None:
        open_ &= (valid != 0)[:, None]
    used = open_.any(1)
    p = torch.zeros_like(x)
    for i in range(t):
        if used[i]:
            v = torch.where(open_[i], x[i], torch.tensor(-INF, dtype=torch.float64))
            p[i] = torch.softmax(v, 0)
    idx, w = torch.full((t, top_k), -1), torch.zeros(t, top_k, dtype=torch.float64)
    for i in range(t):
        rank = lambda k: (1, 0.0, k) if math.isnan(float(x[i, k])) else (0, -float(x[i, k]), k)  # noqa: E731
        order = sorted((k for k in range(e) if open_[i, k]), key=rank)[:top_k]
        idx[i, : len(order)] = torch.tensor(order, dtype=torch.int64)
        if order:
            w[i, : len(order)] = p[i, order]
            if renorm:
                w[i] /= w[i].sum()
    counts = torch.bincount(idx[idx >= 0], minlength=e)
    n = int(used.sum())
    mean = p.sum(0) / max(n, 1)
    return idx, w, counts, n, mean, float((counts * mean).sum()) * e / (max(n, 1) * top_k), p


def forward(x, dtype, top_k, renorm=0, valid=None, pad=0, offset=0, st=None):
    dev()
    t, e = x.shape
    xs = rows_in(x, dtype, pad, offset)
    vs = None if valid is None else valid.cuda()
    size = ab.route_workspace_bytes(t, e)
    out = {"idx": Out(t, top_k, torch.int32), "w": Out(t, top_k, torch.float32), "counts": Out(1, e, torch.int64), "n": Out(1, 1, torch.int64), "mean": Out(1, e, torch.float32),
           "loss": Out(1, 1, torch.float32), "room": torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")}
    d = ab.RouteDesc(tokens=t, experts=e, top_k=top_k, dtype=CODE[dtype], logits_dev=ptr(xs), ld_logits=e + pad, valid_dev=ptr(vs), idx_dev=out["idx"].ptr(),
                     weights_dev=out["w"].ptr(), counts_dev=out["counts"].ptr(), num_tokens_dev=out["n"].ptr(), prob_mean_dev=out["mean"].ptr(), loss_dev=out["loss"].ptr(),
                     workspace_dev=ptr(out["room"]), workspace_bytes=size, renorm=renorm)
    ab.check(ab.route(d, stream()))
    torch.cuda.synchronize()
    for o in out.values():
        if isinstance(o, Out):
            o.check()
    assert (out["room"][size:] == 0xFF).all()
    return xs, out


def check(x, out, valid, top_k, renorm):
    idx, w, counts, n, mean, loss, p = reference(x, valid, top_k, renorm)
    t, e = x.shape
    assert torch.equal(out["idx"].t.cpu().long(), idx), "idx"
    assert torch.equal(out["counts"].t[0].cpu(), counts) and int(out["n"].t) == n
    finite = torch.where(torch.isfinite(x.double()), x.double(), torch.zeros_like(x.double()))
    span = float((finite.amax(1) - finite.amin(1)).max()) if t else 0.0
    rel = (3 * span + e / 32 + 16) * F
    near(out["w"].t, w, 2 * rel * w.abs().nan_to_num() + 2.0**-126, "weights")
    near(out["mean"].t[0], mean, (rel + (t / min(t, 296 * 16) + 64) * F) * mean.abs().nan_to_num() + 2.0**-126, "means")
    near(out["loss"].t[0], torch.tensor([loss]), (rel + (t / min(t, 296 * 16) + 128) * F) * (0 if math.isnan(loss) else abs(loss)), "loss")


@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("t,e,k,dtype", [(1, 1, 1, "f32"), (1, 8, 2, "bf16"), (16, 60, 4, "f32"), (17, 64, 6, "f16"), (3, 33, 32, "f32"), (300, 128, 8, "bf16"), (65, 257, 8, "f32"),
                                         (129, 5, 3, "f32"), (256, 1024, 4, "f16"), (257, 20, 2, "bf16"),
                                         (40, 512, 3, "f16"), (33, 1000, 8, "f32"), (20, 1024, 32, "bf16"), (5000, 16, 2, "f32")])
def test_sizes(t, e, k, dtype, renorm):
    g = gen(t + e)
    x = (torch.randn(t, e, generator=g) * 2 + torch.randn(e, generator=g)).to(TORCH[dtype])
    _, out = forward(x, TORCH[dtype], k, renorm)
    check(x, out, None, k, renorm)


@pytest.mark.parametrize("dtype", TORCH)
def test_ties_go_to_the_first_expert(dtype):
    x = torch.randint(-2, 3, (200, 96), generator=gen(1)).float()
    x[x == 0] = torch.where(torch.rand(int((x == 0).sum()), generator=gen(2)) < 0.5, 0.0, -0.0)  # -0 and 0 are equal
    x = x.to(TORCH[dtype])
    _, out = forward(x, TORCH[dtype], 12, 1)
    check(x, out, None, 12, 1)


def test_padding_and_masks():
    x = torch.randn(400, 40, generator=gen(3)) * 3
    x[torch.rand(400, 40, generator=gen(4)) < 0.5] = -INF
    x[7] = -INF                # nothing left
    x[8, 1:] = -INF            # one left: fewer than top_k
    x[9] = torch.finfo(torch.float32).min   # the type's lowest value masks nothing
    valid = (torch.rand(400, generator=gen(5)) < 0.7).to(torch.uint8) * 255
    valid[[7, 8, 9]] = 1
    for renorm in (0, 1):
        _, out = forward(x, torch.float32, 6, renorm, valid)
        check(x, out, valid, 6, renorm)
        assert (out["idx"].t[7] == -1).all() and (out["w"].t[7] == 0).all()
        assert out["idx"].t[8].tolist() == [0, -1, -1, -1, -1, -1] and out["w"].t[8].tolist() == [1, 0, 0, 0, 0, 0]
        assert out["idx"].t[9].tolist() == [0, 1, 2, 3, 4, 5]
    none = torch.zeros(400, dtype=torch.uint8)
    _, out = forward(x, torch.float32, 6, 1, none)
    assert (out["idx"].t == -1).all() and float(out["loss"].t) == 0 and int(out["n"].t) == 0 and (out["mean"].t == 0).all() and (out["counts"].t == 0).all()


def test_nan_and_infinite_logits():
    x = torch.randn(3, 20, generator=gen(6))
    x[1, 5], x[2, 7] = math.nan, INF
    _, out = forward(x, torch.float32, 20, 0)
    assert out["idx"].t[1].tolist()[-1] == 5 and sorted(out["idx"].t[1].tolist()) == list(range(20)) and out["idx"].t[2].tolist()[0] == 7
    assert torch.isnan(out["w"].t[1]).all() and torch.isnan(out["loss"].t).all()
    idx, w, _, _, _, _, _ = reference(x, None, 20, 0)
    assert torch.equal(out["idx"].t.cpu().long(), idx)
    near(out["w"].t[0], w[0], 64 * F * w[0], "the token beside them")


@pytest.mark.parametrize("pad,offset", [(0, 0), (5, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("dtype", TORCH)
def test_strides(dtype, pad, offset):
    x = torch.randn(50, 72, generator=gen(7)).to(TORCH[dtype])
    xs, out = forward(x, TORCH[dtype], 6, 1, pad=pad, offset=offset)
    check(x, out, None, 6, 1)


# ---- gradients -----------------------------------------------------------------------------------------------------------------
def backward(x, dtype, top_k, renorm, valid=None, pad=0, offset=0, dloss=1.7, dw=True):
    t, e = x.shape
    xs, out = forward(x, dtype, top_k, renorm, valid, pad, offset)
    gw = torch.randn(t, top_k, generator=gen(t + 3))
    gs, ls = gw.cuda(), None if dloss is None else torch.tensor([dloss], device="cuda")
    got = Out(t, e, dtype, pad, offset)
    d = ab.RouteGradDesc(tokens=t, experts=e, top_k=top_k, dtype=CODE[dtype], logits_dev=ptr(xs), ld_logits=e + pad, idx_dev=out["idx"].ptr(), dlogits_dev=got.ptr(),
                         ld_dlogits=e + pad, renorm=renorm)
    if dloss is not None:
        d.dloss_dev, d.counts_dev, d.num_tokens_dev = ptr(ls), out["counts"].ptr(), out["n"].ptr()
    if dw:
        d.dweights_dev = ptr(gs)
    ab.check(ab.route_grad(d, stream()))
    torch.cuda.synchronize()
    got.check()
    # by autograd in 64 bits through softmax, the choice (a constant) and the loss
    leaf = x.double().requires_grad_()
    idx, _, counts, n, _, _, _ = reference(x, valid, top_k, renorm)
    used = idx[:, 0] >= 0
    p = torch.softmax(leaf[used], 1)
    total = torch.zeros((), dtype=torch.float64)
    if dw:
        chosen = idx[used]
        w = torch.where(chosen >= 0, p.gather(1, chosen.clamp(min=0)), torch.zeros(1, dtype=torch.float64))
        if renorm:
            w = w / w.sum(1, keepdim=True)
        total = total + (w * gw[used].double()).sum()
    if dloss is not None:
        total = total + dloss * e / (max(n, 1) ** 2 * top_k) * (counts * p.sum(0)).sum()
    if total.requires_grad:
        total.backward()
    want = leaf.grad if leaf.grad is not None else torch.zeros_like(leaf)
    want = torch.where(used[:, None], want, torch.zeros_like(want))
    # every dlogit is p (dp - sum p dp): its terms are bounded by p (|dp| + sum p |dp|); renormalised weights divide by the chosen sum twice
    full = torch.zeros(t, e, dtype=torch.float64)
    full[used] = p.detach()
    s = torch.where(idx >= 0, full.gather(1, idx.clamp(min=0)), torch.zeros(1, dtype=torch.float64)).sum(1, keepdim=True).clamp(min=1e-9)
    big = (gw.double().abs().max() * (2 / s if renorm else 1) if dw else 0.0) + (abs(dloss) * e * counts.max() / (max(n, 1) ** 2 * top_k) if dloss is not None else 0.0)
    finite = torch.where(torch.isfinite(x.double()), x.double(), torch.zeros(1, dtype=torch.float64))
    rel = (6 * float((finite.amax(1) - finite.amin(1)).max()) + e / 16 + 48) * F
    near(got.t, want.detach(), HALF_STEP[dtype] * want.detach().abs() + TINY[dtype] + rel * full * 2 * big + 2.0**-126, "dlogits")


@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("t,e,k,dtype", [(1, 1, 1, "f32"), (1, 8, 2, "bf16"), (17, 60, 4, "f32"), (3, 33, 32, "f32"), (300, 128, 8, "bf16"), (65, 257, 8, "f16"), (33, 1000, 8, "f32"),
                                         (20, 1024, 32, "f32"), (5000, 16, 2, "f32")])
def test_gradient_sizes(t, e, k, dtype, renorm):
    x = (torch.randn(t, e, generator=gen(t * e)) * 2).to(TORCH[dtype])
    backward(x, TORCH[dtype], k, renorm)


@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("dloss,dw", [(None, True), (0.5, False), (None, False), (-2.0, True)])
def test_gradient_forms(dloss, dw, renorm):
    x = torch.randn(120, 30, generator=gen(12)) * 2
    x[torch.rand(120, 30, generator=gen(13)) < 0.4] = -INF
    x[3] = -INF
    x[4, 1:] = -INF
    valid = (torch.rand(120, generator=gen(14)) < 0.8).to(torch.uint8)
    backward(x, torch.float32, 5, renorm, valid, pad=3, dloss=dloss, dw=dw)


def test_gradient_against_differences():
    """The loss and the weights of the forward call itself, moved along each logit of one token."""
    dev()
    t, e, k, step = 6, 10, 3, 2.0**-8
    x = torch.randn(t, e, generator=gen(15)) * 2
    gw = torch.randn(t, k, generator=gen(16))
    xs, out = forward(x, torch.float32, k, 1)
    got, gs, ls = torch.empty(t, e, device="cuda"), gw.cuda(), torch.tensor([3.0], device="cuda")
    ab.check(ab.route_grad(ab.RouteGradDesc(tokens=t, experts=e, top_k=k, dtype=ab.F32, logits_dev=ptr(xs), idx_dev=out["idx"].ptr(), counts_dev=out["counts"].ptr(),
                                            num_tokens_dev=out["n"].ptr(), dloss_dev=ptr(ls), dweights_dev=ptr(gs), dlogits_dev=ptr(got), renorm=1), stream()))
    torch.cuda.synchronize()

    def value(v):
        _, o = forward(v, torch.float32, k, 1)
        assert torch.equal(o["idx"].t, out["idx"].t), "the step changed a choice"
        return 3.0 * float(o["loss"].t) + float((o["w"].t.cpu().double() * gw.double()).sum())

    for i in range(t):
        for j in range(e):
            d = torch.zeros(t, e)
            d[i, j] = step
            slope = (value(x + d) - value(x - d)) / (2 * step)
            # step^2 / 6 times a third derivative under 6 (|gw| summed + 3), and fp32 noise of the forward call over the step
            assert abs(slope - float(got[i, j])) < step**2 * float(gw.abs().sum() + 3) + 2.0**-19 / step, (i, j)


# ---- calls ---------------------------------------------------------------------------------------------------------------------
def test_no_tokens():
    dev()
    counts, n, mean, loss = torch.ones(5, device="cuda", dtype=torch.int64), torch.ones(1, device="cuda", dtype=torch.int64), torch.ones(5, device="cuda"), torch.ones(1, device="cuda")
    ab.check(ab.route(ab.RouteDesc(tokens=0, experts=5, top_k=2, counts_dev=ptr(counts), num_tokens_dev=ptr(n), prob_mean_dev=ptr(mean), loss_dev=ptr(loss)), stream()))
    ab.check(ab.route_grad(ab.RouteGradDesc(tokens=0, experts=5, top_k=2), stream()))
    torch.cuda.synchronize()
    assert not counts.any() and not n.any() and not mean.any() and not loss.any()


def test_optional_outputs():
    dev()
    x = torch.randn(1000, 24, generator=gen(17)).cuda()
    idx, w = torch.empty(1000, 4, device="cuda", dtype=torch.int32), torch.empty(1000, 4, device="cuda")
    room = torch.empty(ab.route_workspace_bytes(1000, 24), device="cuda", dtype=torch.uint8)
    ab.check(ab.route(ab.RouteDesc(tokens=1000, experts=24, top_k=4, logits_dev=ptr(x), idx_dev=ptr(idx), weights_dev=ptr(w), workspace_dev=ptr(room),
                                   workspace_bytes=room.numel()), stream()))
    torch.cuda.synchronize()
    want = reference(x.cpu(), None, 4, 0)
    assert torch.equal(idx.cpu().long(), want[0])


def test_refusals():
    dev()
    x = torch.zeros(300, 8, device="cuda")
    idx, w, c = torch.zeros(300, 2, device="cuda", dtype=torch.int32), torch.zeros(300, 2, device="cuda"), torch.zeros(8, device="cuda", dtype=torch.int64)
    room = torch.zeros(ab.route_workspace_bytes(300, 8), device="cuda", dtype=torch.uint8)
    assert room.numel() > 0 and ab.route_workspace_bytes(16, 8) == 0 and ab.route_workspace_bytes(0, 8) == 0 and ab.route_workspace_bytes(-1, 8) == 0

    def rc(**kw):
        f = dict(tokens=300, experts=8, top_k=2, logits_dev=ptr(x), idx_dev=ptr(idx), weights_dev=ptr(w), counts_dev=ptr(c), workspace_dev=ptr(room), workspace_bytes=room.numel())
        return ab.route(ab.RouteDesc(**(f | kw)), stream())

    assert rc() == 0
    for bad in (dict(tokens=-1), dict(experts=0), dict(top_k=0), dict(top_k=9), dict(renorm=2), dict(reserved=1), dict(logits_dev=None), dict(idx_dev=None), dict(weights_dev=None),
                dict(workspace_dev=None), dict(workspace_bytes=room.numel() - 1), dict(ld_logits=7)):
        assert rc(**bad) == ab.EINVAL, bad
    assert rc(experts=1025, top_k=2) == ab.ETOOBIG and rc(experts=64, top_k=33) == ab.ETOOBIG and rc(dtype=ab.S8) == ab.EUNSUPPORTED
    assert rc(counts_dev=ptr(c) + 4) == ab.EALIGN and rc(logits_dev=ptr(x) + 2) == ab.EALIGN and rc(workspace_dev=ptr(room) + 4) == ab.EALIGN
    assert ab.lib().ascb200_route(None, None) == ab.EINVAL

    n, l = torch.ones(1, device="cuda", dtype=torch.int64), torch.zeros(1, device="cuda")

    def grad(**kw):
        f = dict(tokens=300, experts=8, top_k=2, logits_dev=ptr(x), idx_dev=ptr(idx), counts_dev=ptr(c), num_tokens_dev=ptr(n), dloss_dev=ptr(l), dlogits_dev=ptr(x))
        return ab.route_grad(ab.RouteGradDesc(**(f | kw)), stream())

    assert grad() == 0
    for bad in (dict(logits_dev=None), dict(idx_dev=None), dict(dlogits_dev=None), dict(counts_dev=None), dict(num_tokens_dev=None), dict(ld_dlogits=7), dict(ld_dlogits=16), dict(reserved=1),
                dict(top_k=9), dict(renorm=-1)):
        assert grad(**bad) == ab.EINVAL, bad
    assert grad(dtype=ab.S32) == ab.EUNSUPPORTED and grad(dloss_dev=ptr(l) + 1) == ab.EALIGN
    assert ab.lib().ascb200_route_grad(None, None) == ab.EINVAL
    torch.cuda.synchronize()


def test_captured_and_replayed():
    dev()
    t, e, k = 700, 64, 4
    x, idx, w = torch.zeros(t, e, device="cuda"), torch.zeros(t, k, device="cuda", dtype=torch.int32), torch.zeros(t, k, device="cuda")
    c, n, m, l = torch.zeros(e, device="cuda", dtype=torch.int64), torch.zeros(1, device="cuda", dtype=torch.int64), torch.zeros(e, device="cuda"), torch.zeros(1, device="cuda")
    room = torch.zeros(ab.route_workspace_bytes(t, e), device="cuda", dtype=torch.uint8)
    d = ab.RouteDesc(tokens=t, experts=e, top_k=k, logits_dev=ptr(x), idx_dev=ptr(idx), weights_dev=ptr(w), counts_dev=ptr(c), num_tokens_dev=ptr(n), prob_mean_dev=ptr(m),
                     loss_dev=ptr(l), workspace_dev=ptr(room), workspace_bytes=room.numel(), renorm=1)
    side = C.c_void_p()
    ab.check(ab.lib().ascb200_stream_create(C.byref(side)))
    torch.cuda.synchronize()
    graph = ab.Graph(side, lambda: ab.check(ab.route(d, side)))
    for seed in (20, 21):
        x.copy_(torch.randn(t, e, generator=gen(seed)))
        torch.cuda.synchronize()
        graph.launch()
        graph.launch()
        torch.cuda.synchronize()
        want = reference(x.cpu(), None, k, 1)
        assert torch.equal(idx.cpu().long(), want[0]) and torch.equal(c.cpu(), want[2]) and int(n) == want[3]
        near(l, torch.tensor([want[5]]), 200 * F * want[5], "loss")
    graph.destroy()
    ab.lib().ascb200_stream_destroy(side)


@pytest.mark.parametrize("e", [8, 60, 256, 1000])
def test_close_and_large_logits(e):
    """fp32 logits that agree in all but their last bits, among few and among many; values whose last bit is large."""
    x = torch.randn(300, e, generator=gen(e))
    near_one = (torch.ones(300, e).view(torch.int32) + torch.randint(0, 40, (300, e), generator=gen(e + 1), dtype=torch.int32)).view(torch.float32)
    pick = torch.rand(300, e, generator=gen(e + 2)) < 0.3
    x[:150] = torch.where(pick[:150], 2 * near_one[:150], x[:150])   # ties and near ties at the top
    x[150:200] = -near_one[150:200]                                  # everywhere, negative
    x[200:250] = 0.25                                                # all equal
    for renorm in (0, 1):
        _, out = forward(x, torch.float32, min(8, e), renorm)
        check(x, out, None, min(8, e), renorm)
    big = torch.randn(64, e, generator=gen(e + 3)) * torch.tensor([1e3, 1e6, 1e12, 1e30]).repeat(16)[:, None]
    _, out = forward(big, torch.float32, min(8, e), 1)
    idx, w, counts, n, _, _, _ = reference(big, None, min(8, e), 1)
    assert torch.equal(out["idx"].t.cpu().long(), idx) and torch.isfinite(out["w"].t).all() and torch.equal(out["counts"].t[0].cpu(), counts)


@pytest.mark.parametrize("e", [1, 8, 32, 72, 256, 300, 1000, 1024])
@pytest.mark.parametrize("dtype", TORCH)
def test_large_negative_logits(dtype, e):
    """Rows whose every open logit is far below zero: exp(x - max) is of their differences, which the row's true maximum alone keeps at or below zero."""
    lowest = float(torch.finfo(TORCH[dtype]).min)
    levels = (-1.5, -60000.0) if dtype == "f16" else (-1.5, -1e7, -1e9, -1e30, lowest)
    x = torch.cat([torch.full((4, e), v) for v in levels])
    steps = 1 - torch.randint(0, 3, x.shape, generator=gen(e)) * 2.0**-7   # of the type; downwards, so that the lowest stays finite
    x[1::4] *= steps[1::4]
    x[2::4, e // 2 + 1 :] = -INF
    x[3::4] = torch.where(torch.arange(e) % 3 == 1, -INF, x[3::4] * steps[3::4])
    x = x.to(TORCH[dtype])
    for renorm in (0, 1):
        k = min(4, e)
        _, out = forward(x, TORCH[dtype], k, renorm)
        idx, w, counts, n, mean, loss, _ = reference(x, None, k, renorm)
        assert torch.equal(out["idx"].t.cpu().long(), idx) and torch.equal(out["counts"].t[0].cpu(), counts) and int(out["n"].t) == n
        # the levels' logits are equal or so far apart that only the largest count, but for those of -1.5, which differ by at most 1/32
        rel = (e / 32 + 24) * F
        near(out["w"].t, w, 2 * rel * w.abs() + 2.0**-126, "weights")
        near(out["mean"].t[0], mean, (rel + 96 * F) * mean.abs() + 2.0**-126, "means")
        near(out["loss"].t[0], torch.tensor([loss]), (rel + 160 * F) * abs(loss), "loss")
