"""mx_linear at sizes on both sides of the rules that choose between its tile forms."""
import pytest
import torch

from support import run_op
from test_mx_cpu import DTYPES, some
from test_mx_gpu import TINY, UNIT
from test_mx_stream_gpu import coded

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
