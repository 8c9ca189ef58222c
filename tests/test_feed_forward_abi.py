"""The descriptors of the feed-forward operators on a machine without a GPU: the ctypes binding lays them out as a C compiler does, the
workspace sizes are plain host functions, and without a device nothing is computed."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

import ascb200 as ab

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DESCS = {"ascb200_gemm_desc": ab.GemmDesc, "ascb200_rms_norm_desc": ab.RmsNormDesc, "ascb200_rms_norm_grad_desc": ab.RmsNormGradDesc, "ascb200_linear_desc": ab.LinearDesc,
         "ascb200_linear_grad_desc": ab.LinearGradDesc, "ascb200_route_desc": ab.RouteDesc, "ascb200_route_grad_desc": ab.RouteGradDesc}


@pytest.mark.parametrize("name", DESCS)
def test_layout_matches_the_header(name, tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    fields = [f[0] for f in DESCS[name]._fields_]
    text = open(os.path.join(ROOT, "include", "ascb200.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1), flags=re.S)
    declared = [re.sub(r"\[.*", "", v).split()[-1].lstrip("*") for line in body.split(";") if line.strip() for v in line.split(",")]
    assert declared == fields
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ascb200.h"\nint main(void) { printf("%%zu", sizeof(%s));\n%s\nreturn 0; }\n' % (
        name, "\n".join('printf(" %%zu", offsetof(%s, %s));' % (name, f) for f in fields)))
    subprocess.check_call(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "layout")]).split()]
    assert got == [C.sizeof(DESCS[name])] + [getattr(DESCS[name], f).offset for f in fields]


def test_workspace_sizes():
    assert ab.rms_norm_grad_workspace_bytes(0, 64) == 0 and ab.rms_norm_grad_workspace_bytes(-3, 64) == 0 and ab.rms_norm_grad_workspace_bytes(4, -1) == 0
    many = ab.rms_norm_grad_workspace_bytes(1 << 30, 32768)  # whole rows of partial sums, a bounded number of them
    assert ab.rms_norm_grad_workspace_bytes(1, 64) == 256 and many % (32768 * 4) == 0 and 0 < many <= 1024 * 32768 * 4
    assert ab.route_workspace_bytes(1, 1024) == 0 and ab.route_workspace_bytes(0, 8) == 0 and ab.route_workspace_bytes(2**31 - 1, 1024) > 0
    assert ab.linear_grad_workspace_bytes(0, 8) == 0 and ab.linear_grad_workspace_bytes(100, 9) >= 100 * 16 * 2
    big = ab.linear_grad_workspace_bytes(1 << 20, 1 << 15)   # past 32 bits
    assert big > (1 << 36)


def test_no_cpu_fallback_without_device():
    lib = ab.lib()
    if lib.ascb200_init(0) == 0:  # running on a GPU box: nothing to check here
        return
    for f, d in ((ab.rms_norm, ab.RmsNormDesc()), (ab.rms_norm_grad, ab.RmsNormGradDesc()), (ab.linear, ab.LinearDesc()), (ab.linear_grad, ab.LinearGradDesc()),
                 (ab.route, ab.RouteDesc()), (ab.route_grad, ab.RouteGradDesc())):
        assert f(d) == ab.ENODEV
