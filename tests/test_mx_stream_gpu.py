"""mx_linear's weight stream at the sizes that decode steps run it with: every split of K over waves,
rings that go round, runs of more than 16 units of 256 columns per wave, a last unit in part."""
import pytest
import torch

import mx_oracle as mx
from support import run_op
from test_mx_cpu import DTYPES, some
from test_mx_gpu import TINY, UNIT

pytestmark = pytest.mark.gpu


def values(codes, scales):
    """What finite codes and scales on the GPU stand for, in float64."""
    if codes.shape[1] == scales.shape[1] * 32:
        e = torch.from_numpy(mx.E4M3).cuda()[(codes % 128).int()]
        e = e * torch.where(codes >= 128, -1.0, 1.0)
    else:
        both = torch.stack([codes % 16, codes // 16], -1).flatten(1)
        e = torch.from_numpy(mx.E2M1).cuda()[(both % 8).int()] * torch.where(both >= 8, -1.0, 1.0)
    s = torch.exp2(scales.double() - 127)
    return (e.view(*scales.shape, 32) * s.unsqueeze(-1)).flatten(1)


def coded(rows, k, form, seed):
    """A microscaled tensor of random finite codes and scales 2^-4 .. 2^4, and its values."""
    g = torch.Generator().manual_seed(seed)
    scales = torch.randint(123, 132, (rows, k // 32), generator=g, dtype=torch.uint8).cuda()
    codes = torch.randint(0, 254 if form == "fp8" else 256, (rows, k if form == "fp8" else k // 2),
                          generator=g, dtype=torch.uint8).cuda()
    if form == "fp8":
        codes = codes + (codes >= 127).to(torch.uint8)  # 127 and 255 are NaN
    return codes, scales, values(codes, scales)


# the waves that share K, and units of 256 columns per wave: K in whole words of scales, then not
SHAPES = [(896, 4864), (896, 4896),      # 8 waves, 2 or 3
          (100, 18944), (100, 18976),    # 8, 9 or 10
          (40, 36864), (40, 36896),      # 8, 18 or 19
          (8200, 17408), (8200, 17440),  # 4, 17 or 18
          (20000, 8448), (20000, 9248),  # 2, 16 to 19
          (33000, 3584), (33000, 3616),  # 1, 14 or 15
          (33000, 4224), (33000, 4640)]  # 1, 17 or 19


@pytest.mark.parametrize("form,out_dtype", [("fp8", "float32"), ("fp4", "float32"),
                                            ("fp8", "bfloat16"), ("fp4", "float16")])
@pytest.mark.parametrize("n,k", SHAPES)
def test_stream(form, out_dtype, n, k):
    w, ws, w64 = coded(n, k, "fp4", 7)
    t = DTYPES[out_dtype]
    bias = some((n,), t, 3).cuda()
    for m in (1, 3, 16):
        x, xs, x64 = coded(m, k, form, m)
        residual = some((m, n), t, 4).cuda()
        out = run_op("mx_linear", {"x": x, "xs": xs, "w": w, "ws": ws, "b": bias, "r": residual},
                     ("out",), {"out_dtype": out_dtype, "residual": True})["out"]
        ref = x64 @ w64.t() + bias.double() + residual.double()
        terms = x64.abs() @ w64.abs().t() + bias.double().abs() + residual.double().abs()
        # the output's rounding; fp32 sums of at most k / 8 + 3 terms; with e4m3 rows and a 16-bit
        # result 7 of 8 neighbouring products lose up to 2^-13 of the largest
        bound = UNIT[out_dtype] * ref.abs() + (k // 8 + 3) * 2.0 ** -23 * terms + TINY[out_dtype]
        if form == "fp8" and out_dtype != "float32":
            bound = bound + 2.0 ** -10 * terms
        good = ref.abs() < torch.finfo(t).max  # (past it the result is infinite)
        err = (out.double() - ref).abs()
        assert (err <= bound)[good].all(), m
        # what goes missing on average is far less: a unit or a scale in the wrong place shows
        rel = (err[good].norm() / ref[good].norm()).item()
        assert rel < {"bfloat16": 2.5e-3, "float16": 4e-4, "float32": 1e-6}[out_dtype], (m, rel)
