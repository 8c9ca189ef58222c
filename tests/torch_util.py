"""Helpers of the tests that keep their tensors in torch: types, guarded output buffers, descriptors."""
import math

import torch

import ascb200 as ab
from gpu_util import dev  # noqa: F401  (initialises the library once)

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {torch.float32: ab.F32, torch.float16: ab.F16, torch.bfloat16: ab.BF16, torch.int8: ab.S8, torch.float8_e4m3fn: ab.FP8_E4M3}
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}    # of a rounding, relative to the value
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}      # half a step (fp32: one) below the normal numbers
GUARD = 0x5A


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


class Out:
    """A [rows, cols] output with `pad` elements behind every row and a row behind the last, all filled with one byte;
    `t` is the tensor, `check()` tells whether something else than it was written."""

    def __init__(self, rows, cols, dtype, pad=0, offset=0):
        self.rows, self.cols, self.ld, self.offset, self.dtype = rows, cols, cols + pad, offset, dtype
        size = torch.empty(0, dtype=dtype).element_size()
        self.raw = torch.full(((offset + (rows + 1) * self.ld + 32) * size,), GUARD, dtype=torch.uint8, device="cuda")
        self.flat = self.raw.view(dtype)
        self.t = torch.as_strided(self.flat, (rows, cols), (self.ld, 1), offset)

    def ptr(self):
        return self.t.data_ptr()

    def check(self):
        size = self.t.element_size()
        inside = torch.zeros(self.raw.numel() // size, dtype=torch.bool, device="cuda")
        torch.as_strided(inside, (self.rows, self.cols), (self.ld, 1), self.offset).fill_(True)
        outside = (~inside).repeat_interleave(size)
        assert (self.raw[outside] == GUARD).all(), "written outside the output"


def rows_in(values, dtype, pad=0, offset=0, fill=math.nan):
    """[m, k] values in a buffer whose rows are `pad` elements apart and start `offset` elements in; the rest holds `fill`."""
    m, k = values.shape
    flat = torch.full((offset + m * (k + pad) + 32,), fill, dtype=torch.float32).to(dtype).cuda() if dtype != torch.int8 else torch.full(
        (offset + m * (k + pad) + 32,), 77, dtype=dtype, device="cuda")
    t = torch.as_strided(flat, (m, k), (k + pad, 1), offset)
    t.copy_(values.to(dtype))
    return t


def near(got, want, tol, what=""):
    """|got - want| <= tol elementwise (tol a tensor or number); NaN and infinities in the same places."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    fine = ~torch.isnan(want)
    d = torch.where(fine & (got != want), (got - want).abs(), torch.zeros_like(want))
    over = d - (tol.cpu() if isinstance(tol, torch.Tensor) else tol)
    over = torch.where(fine, over, -torch.ones_like(over))
    assert over.numel() == 0 or over.max() <= 0, f"{what}: off by {float(d.flatten()[over.argmax()])} at {int(over.argmax())}, {float(over.max())} over the tolerance"
