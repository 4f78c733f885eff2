"""Microscaled operators on host tensors (the ATen CPU plugin) against float64, the entry points'
argument checks, and uint8 tensors in the weights format. No GPU."""
import ctypes

import numpy as np
import pytest
import torch

import dli
import mx_oracle as mx
from dli import hip
from dli.weights import save_weights
from support import run_op

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_ENGINE = []


def aten(op, inputs, outputs, attrs=None):
    if not _ENGINE:
        _ENGINE.append(dli.Engine().load_aten_plugin())
    from support import one_node_graph
    return _ENGINE[0].run(one_node_graph(op, inputs, outputs, attrs), inputs)


def some(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def special_rows():
    """Rows of 64: ties and ends of both element types, zeros, the smallest and largest floats,
    infinities and NaN in one block of two."""
    r = torch.zeros(8, 64)
    r[0, :32] = torch.tensor([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.9, -.25, -5, -7]
                             + [4.0] * 18)
    r[0, 32:] = torch.linspace(-500, 500, 32)
    r[1, 3] = 2.0 ** -126
    r[1, 40] = 2.0 ** -149
    r[2, :32] = 3.0e38
    r[2, 32:] = torch.arange(32) * 2.0 ** -130
    r[3, 5] = float("inf")
    r[4, 50] = float("nan")
    r[5, 1], r[5, 2] = float("nan"), float("-inf")
    r[5, 32:] = -1.0
    r[6] = -0.0
    r[7, :32] = torch.tensor([1.0 - 2.0 ** -24, 1.0] * 16)
    r[7, 32:] = 448.0 + torch.arange(32)
    return r


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_quantize_and_back(form, dtype):
    for x in (special_rows().to(DTYPES[dtype]), some((3, 5, 96), DTYPES[dtype], 1),
              some((1, 32), DTYPES[dtype], 2, 1e-3), torch.zeros(0, 64, dtype=DTYPES[dtype])):
        out = aten("mx_quantize", {"x": x}, ("codes", "scales"), {"format": form})
        codes, scales = out["codes"], out["scales"]
        if x.numel():
            c, s = mx.quantize(x.double().numpy(), form)
            assert np.array_equal(scales.numpy(), s)
            assert np.array_equal(codes.numpy(), c)
        back = aten("mx_dequantize", {"c": codes, "s": scales}, ("out",), {"dtype": "float32"})
        if x.numel():
            want = torch.from_numpy(mx.values(codes.numpy(), scales.numpy())).float()
            assert torch.equal(back["out"].nan_to_num(-1), want.nan_to_num(-1))
            assert torch.equal(back["out"].isnan(), want.isnan())


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_norm_and_gate(form, dtype):
    t = DTYPES[dtype]
    x, res, w = some((5, 160), t, 3), some((5, 160), t, 4), some((160,), t, 5)
    x[2] = 0
    res[2] = 0
    out = aten("rms_norm_mx", {"x": x, "w": w, "r": res}, ("codes", "scales", "h"),
               {"format": form, "eps": 1e-6})
    h = (x.float() + res.float()).to(t)
    assert torch.equal(out["h"], h)
    c, s = mx.quantize(mx.rms_norm32(h.float().numpy(), w.float().numpy(), 1e-6), form)
    assert np.array_equal(out["codes"].numpy(), c) and np.array_equal(out["scales"].numpy(), s)
    one = aten("rms_norm_mx", {"x": h, "w": w}, ("codes", "scales"), {"format": form})
    assert torch.equal(one["codes"], out["codes"]) and torch.equal(one["scales"], out["scales"])
    two = aten("silu_mul_mx", {"g": x, "u": res}, ("codes", "scales"), {"format": form})
    both = aten("silu_mul_mx", {"gu": torch.cat([x, res], -1)}, ("codes", "scales"),
                {"format": form})
    assert torch.equal(two["codes"], both["codes"]) and torch.equal(two["scales"], both["scales"])
    g = x.double()
    y = (g / (1 + torch.exp(-g)) * res.double()).numpy()
    got = mx.values(two["codes"].numpy(), two["scales"].numpy())
    # half a step of the element type at the block's largest magnitude, saturation included (an
    # eighth of it for e4m3, a quarter for e2m1)
    top = np.abs(y).reshape(-1, 32).max(1)[:, None]
    assert (np.abs(got - y).reshape(-1, 32) <= top * (0.25 if form == "fp4" else 0.125)).all()


@pytest.mark.parametrize("form", ["fp8", "fp4"])
def test_linear(form):
    x, w, b, r = (some(s, torch.float32, i) for i, s in
                  enumerate([(2, 3, 96), (7, 96), (7,), (2, 3, 7)]))
    q = [torch.from_numpy(a) for a in mx.quantize(x.double().numpy(), form)]
    p = [torch.from_numpy(a) for a in mx.quantize(w.double().numpy(), "fp4")]
    ref = mx.values(*(a.numpy() for a in q)) @ mx.values(*(a.numpy() for a in p)).T
    base = {"x": q[0], "xs": q[1], "w": p[0], "ws": p[1]}
    for more, attrs, want in (({}, {}, ref), ({"b": b}, {}, ref + b.double().numpy()),
                              ({"r": r}, {"residual": True}, ref + r.double().numpy()),
                              ({"b": b, "r": r}, {"residual": True},
                               ref + b.double().numpy() + r.double().numpy())):
        out = aten("mx_linear", {**base, **more}, ("out",), {**attrs, "out_dtype": "float32"})
        # sums of 98 fp32 terms of magnitude at most about 10
        np.testing.assert_allclose(out["out"].double().numpy(), want, atol=98 * 10 * 2.0 ** -23)


def test_operators_refuse_what_is_not_microscaled():
    x = torch.randn(2, 64)
    c, s = (torch.from_numpy(a) for a in mx.quantize(x.double().numpy(), "fp4"))
    refused = [
        ("mx_quantize", {"x": torch.randn(2, 40)}, ("a", "b"), {}, "multiple of 32"),
        ("mx_quantize", {"x": x}, ("a", "b"), {"format": "fp6"}, "format must be"),
        ("mx_quantize", {"x": c}, ("a", "b"), {}, "float32, bfloat16 or float16"),
        ("mx_dequantize", {"c": c, "s": s[:1]}, ("a",), {}, "not a microscaled"),
        ("mx_dequantize", {"c": c[:, :20], "s": s}, ("a",), {}, "not a microscaled"),
        ("mx_dequantize", {"c": c, "s": s}, ("a",), {"dtype": "int64"}, "floating type"),
        ("rms_norm_mx", {"x": x, "w": torch.ones(32)}, ("a", "b"), {}, "weight size"),
        ("rms_norm_mx", {"x": x, "w": torch.ones(64), "r": x[:1]}, ("a", "b", "c"), {},
         "shape of x"),
        ("silu_mul_mx", {"g": x, "u": x[:, :32]}, ("a", "b"), {}, "one shape"),
        ("silu_mul_mx", {"g": torch.randn(2, 33)}, ("a", "b"), {}, "even"),
        ("mx_linear", {"x": c, "xs": s, "w": c, "ws": s, "b": torch.ones(2)}, ("a",), {},
         "out_dtype"),
        ("mx_linear", {"x": c, "xs": s, "w": c[:, :16].contiguous(), "ws": s[:, :1].contiguous()},
         ("a",), {}, "does not match"),
    ]
    q = [torch.from_numpy(a) for a in mx.quantize(x.double().numpy(), "fp8")]
    refused.append(("mx_linear", {"x": c, "xs": s, "w": q[0], "ws": q[1]}, ("a",), {},
                    "must be fp4"))
    for op, inputs, outputs, attrs, text in refused:
        with pytest.raises(ValueError, match=text):
            aten(op, inputs, outputs, attrs)


def test_operators_refuse_scalars():
    one, byte = torch.tensor(1.0), torch.tensor(1, dtype=torch.uint8)
    c, s = (torch.from_numpy(a) for a in mx.quantize(np.ones((2, 64)), "fp4"))
    for op, inputs, n, text in (
            ("mx_quantize", {"x": one}, 2, "multiple of 32"),
            ("mx_dequantize", {"c": byte, "s": byte}, 1, "not a microscaled"),
            ("rms_norm_mx", {"x": one, "w": one}, 2, "multiple of 32"),
            ("silu_mul_mx", {"g": one}, 2, "even"),
            ("silu_mul_mx", {"g": one, "u": one}, 2, "multiple of 32"),
            ("mx_linear", {"x": byte, "xs": byte, "w": c, "ws": s}, 1, "not a microscaled")):
        with pytest.raises(ValueError, match=text):
            aten(op, inputs, tuple(f"o{i}" for i in range(n)))


def test_gpu_operators_refuse_host_tensors():
    x = torch.randn(2, 64)
    for op, inputs, n in (("mx_quantize", {"x": x}, 2), ("rms_norm_mx", {"x": x, "w": x[0]}, 2),
                          ("silu_mul_mx", {"g": x}, 2),
                          ("mx_dequantize", {"c": x, "s": x}, 1),
                          ("mx_linear", {"x": x, "xs": x, "w": x, "ws": x}, 1)):
        engine = dli.Engine().load_plugin()
        from support import one_node_graph
        with pytest.raises(ValueError, match="CUDA"):
            engine.run(one_node_graph(op, inputs, [f"o{i}" for i in range(n)]), inputs)


def test_entry_points_check_their_arguments():
    lib, fake = hip.load(), ctypes.c_void_p(256)  # never dereferenced: refused before a launch

    def says(rc, text):
        assert rc == -1 and text in lib.dli_hip_last_error(), lib.dli_hip_last_error()

    q = lib.dli_hip_mx_quantize
    assert q(hip.BF16, hip.MX_FP8, None, None, None, 0, 64, None) == 0
    assert q(hip.BF16, hip.MX_FP8, None, None, None, 5, 0, None) == 0
    says(q(hip.I64, hip.MX_FP8, fake, fake, fake, 1, 32, None), b"unsupported dtype")
    says(q(hip.U8, hip.MX_FP8, fake, fake, fake, 1, 32, None), b"unsupported dtype")
    says(q(hip.F32, 2, fake, fake, fake, 1, 32, None), b"unsupported format")
    says(q(hip.F32, 0, fake, fake, fake, 1, 48, None), b"multiple of 32")
    says(q(hip.F32, 0, fake, fake, fake, -1, 32, None), b"negative")
    says(q(hip.F32, 0, fake, fake, fake, 1 << 60, 1 << 20, None), b"too large")
    says(q(hip.F32, 0, fake, None, fake, 1, 32, None), b"NULL")
    d = lib.dli_hip_mx_dequantize
    says(d(hip.F32, 0, fake, fake, None, 1, 32, None), b"NULL")
    says(d(hip.F32, 0, fake, fake, fake, 1, 33, None), b"multiple of 32")
    r = lib.dli_hip_rms_norm_mx
    says(r(hip.F32, 0, fake, None, None, None, fake, fake, 1, 32, 1e-6, None), b"NULL")
    says(r(hip.F32, 0, fake, None, fake, None, fake, fake, 1, 0, 1e-6, None), b"positive")
    s = lib.dli_hip_silu_mul_mx
    says(s(hip.F32, 0, fake, fake, 16, fake, fake, 1, 32, None), b"stride")
    says(s(hip.F32, 0, fake, fake, 1 << 60, fake, fake, 1 << 20, 32, None), b"too large")
    m = lib.dli_hip_mx_linear

    def linear(x=fake, xf=0, out=hip.BF16, w=fake, m_=4, n=8, k=64):
        return m(xf, out, x, fake, w, fake, None, None, fake, m_, n, k, None, 0, None)

    assert linear(m_=0) == 0 and linear(n=0) == 0
    says(linear(xf=7), b"unsupported format")
    says(linear(out=hip.I32), b"unsupported dtype")
    says(linear(k=0), b"positive")
    says(linear(k=16), b"multiple of 32")
    says(linear(x=ctypes.c_void_p(264)), b"16-byte aligned")
    says(linear(w=None), b"NULL")
    says(linear(m_=1 << 40, n=1 << 40), b"too large")
    says(linear(n=(1 << 29) + 1), b"n at most 2^29")
    says(linear(m_=(1 << 20) - 15), b"m must be at most 1048560")
    says(linear(k=(1 << 28) + 32), b"k must be at most 2^28")
    assert lib.dli_hip_mx_linear_workspace(0, 0, 8, 64) == 0
    assert lib.dli_hip_mx_linear_workspace(0, 4, 8, 33) == 0


def test_uint8_tensors_in_the_weights_format(tmp_path):
    t = {"codes": torch.randint(0, 256, (5, 48), dtype=torch.uint8),
         "empty": torch.zeros(0, 3, dtype=torch.uint8)}
    back = dli.load_weights(str(save_weights(tmp_path, "mx", t)))
    for name in t:
        assert back[name].dtype == torch.uint8 and torch.equal(back[name], t[name])
