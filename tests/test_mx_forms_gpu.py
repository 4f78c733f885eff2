"""mx_linear at sizes on both sides of the rules that choose between its tile forms."""
import pytest
import torch

from support import run_op
from test_mx_cpu import DTYPES, some
from test_mx_gpu import TINY, UNIT, c_linear
from test_mx_stream_gpu import coded, values

pytestmark = pytest.mark.gpu


def check(form, out_dtype, m, n, k):
    w, ws, w64 = coded(n, k, "fp4", 7)
    x, xs, x64 = coded(m, k, form, m)
    t = DTYPES[out_dtype]
    inputs = {"x": x, "xs": xs, "w": w, "ws": ws, "b": some((n,), t, 3).cuda(),
              "r": some((m, n), t, 4).cuda()}
    out = run_op("mx_linear", inputs, ("out",), {"out_dtype": out_dtype, "residual": True})["out"]
    ref = x64 @ w64.t() + inputs["b"].double() + inputs["r"].double()
    terms = x64.abs() @ w64.abs().t() + inputs["b"].double().abs() + inputs["r"].double().abs()
    # as in test_mx_stream_gpu.py
    bound = UNIT[out_dtype] * ref.abs() + (k // 8 + 3) * 2.0 ** -23 * terms + TINY[out_dtype]
    if form == "fp8" and out_dtype != "float32":
        bound = bound + 2.0 ** -10 * terms
    good = ref.abs() < torch.finfo(t).max
    err = (out.double() - ref).abs()
    assert (err <= bound)[good].all()
    rel = (err[good].norm() / ref[good].norm()).item()
    assert rel < {"bfloat16": 2.5e-3, "float16": 4e-4, "float32": 1e-6}[out_dtype], rel
    return inputs, out


FORMS = [("fp8", "float32"), ("fp4", "float32"), ("fp8", "bfloat16"), ("fp4", "float16")]


@pytest.mark.parametrize("form,out_dtype", FORMS)
@pytest.mark.parametrize("m,n,k", [(64, 33000, 4224), (17, 40001, 8192), (50, 65536, 4608),
                                   (33, 32776, 18944), (64, 65537, 2176), (64, 33000, 4256)])
def test_runs_of_columns(form, out_dtype, m, n, k):
    check(form, out_dtype, m, n, k)


@pytest.mark.parametrize("form,out_dtype", FORMS)
@pytest.mark.parametrize("m,n,k", [
    (3001, 4104, 1824), (1537, 8193, 1952), (4100, 8200, 2592), (8191, 9721, 992),  # 256 x 256, past every end
    (257, 24577, 896), (513, 16385, 1056), (2049, 9729, 640), (1025, 9857, 2560)])  # 128 x 128
def test_large_and_smaller_tiles(form, out_dtype, m, n, k):
    check(form, out_dtype, m, n, k)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("m,n,k", [(300, 11520, 4224), (700, 5633, 4480), (64, 70001, 4224)])
def test_tiles_without_a_workspace(form, m, n, k):
    """Without room for laid-out scales the same tiles read them as they are: the same sums, bit for
    bit. Products that a graph captures on a stream of its own run so."""
    inputs, out = check(form, "float32", m, n, k)
    assert torch.equal(c_linear(form, inputs, m, n, k), out)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("m,n,k", [(70, 896, 18944), (64, 3584, 8192), (300, 11520, 4256), (484, 3584, 8192),
                                   (300, 20000, 4224), (3001, 4104, 4224)])
def test_no_workspace(form, m, n, k):
    """The stream, tiles that walk all of K, and large products in smaller tiles."""
    inputs, out = check(form, "float32", m, n, k)
    # both within half the bound of check: two orders of the same fp32 sums
    terms = (values(inputs["x"], inputs["xs"]).abs() @ values(inputs["w"], inputs["ws"]).abs().t()
             + inputs["b"].double().abs() + inputs["r"].double().abs())
    got = c_linear(form, inputs, m, n, k)
    assert ((got.double() - out.double()).abs() <= (k // 8 + 4) * 2.0 ** -22 * terms).all()
