"""Microscaled operators on the GPU against float64: every element type, data type and route, odd
sizes, unaligned data, special values, streams and captured graphs."""
import numpy as np
import pytest
import torch

import dli
import mx_oracle as mx
from dli import hip
from support import one_node_graph, plugin_engine, run_op
from test_mx_cpu import DTYPES, some, special_rows

pytestmark = pytest.mark.gpu
UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}  # half a step, at most
# the smallest spacing of the type (subnormals of float16 come into reach)
TINY = {"bfloat16": 2.0 ** -133, "float16": 2.0 ** -24, "float32": 2.0 ** -149}


def host(t):
    return t.cpu().numpy()


def unaligned(t):
    """A copy of t one element past a 16-byte boundary."""
    flat = torch.empty(t.numel() + 17, dtype=t.dtype, device="cuda")
    skip = next(i for i in range(17) if (flat.data_ptr() + i * t.element_size()) % 16
                == t.element_size() % 16)
    view = flat[skip:skip + t.numel()].view(t.shape)
    view.copy_(t)
    assert view.data_ptr() % 16 != 0
    return view


def quantized(x, form):
    return [torch.from_numpy(a).cuda() for a in mx.quantize(x.double().cpu().numpy(), form)]


# ---- quantisation ------------------------------------------------------------------------------


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(1, 32), (1, 896), (3, 5, 96), (333, 928), (70, 4864), (0, 64)])
def test_quantize_and_back(form, dtype, shape):
    x = some(shape, DTYPES[dtype], 1).cuda()
    for t in (x, unaligned(x)) if x.numel() else (x,):
        out = run_op("mx_quantize", {"x": t}, ("codes", "scales"), {"format": form})
        assert out["codes"].shape == shape[:-1] + (shape[-1] // (1 if form == "fp8" else 2),)
        assert out["scales"].shape == shape[:-1] + (shape[-1] // 32,)
        if not x.numel():
            continue
        c, s = mx.quantize(x.double().cpu().numpy(), form)
        assert np.array_equal(host(out["scales"]), s)
        assert np.array_equal(host(out["codes"]), c)
        for name in DTYPES:
            codes = out["codes"] if t is x else unaligned(out["codes"])
            back = run_op("mx_dequantize", {"c": codes, "s": out["scales"]}, ("out",),
                          {"dtype": name})["out"]
            assert torch.equal(back.cpu(), torch.from_numpy(mx.values(c, s)).to(DTYPES[name]))


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_special_values(form, dtype):
    x = special_rows().to(DTYPES[dtype])
    out = run_op("mx_quantize", {"x": x.cuda()}, ("codes", "scales"), {"format": form})
    c, s = mx.quantize(x.double().numpy(), form)
    assert np.array_equal(host(out["scales"]), s) and np.array_equal(host(out["codes"]), c)


def test_every_code_stands_for_its_value():
    for scale in (0, 1, 127, 200, 252, 255):
        s = torch.full((1, 8), scale, dtype=torch.uint8)
        c = torch.arange(256, dtype=torch.uint8).view(1, 256)
        got = run_op("mx_dequantize", {"c": c.cuda(), "s": s.cuda()}, ("out",),
                     {"dtype": "float32"})["out"].cpu()
        want = torch.from_numpy(mx.values(c.numpy(), s.numpy())).float()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(7), want.nan_to_num(7)), scale
        c = torch.arange(256, dtype=torch.uint8).view(2, 128)
        s = torch.full((2, 8), scale, dtype=torch.uint8)
        got = run_op("mx_dequantize", {"c": c.cuda(), "s": s.cuda()}, ("out",),
                     {"dtype": "float32"})["out"].cpu()
        want = torch.from_numpy(mx.values(c.numpy(), s.numpy())).float()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(7), want.nan_to_num(7)), scale


# ---- norm and gate -----------------------------------------------------------------------------


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,hidden", [(1, 32), (1, 896), (5, 1024), (333, 160), (7, 1056),
                                         (64, 3584), (3, 4864), (2, 8224), (3, 18944), (2, 33024)])
def test_norm(form, dtype, rows, hidden):
    t = DTYPES[dtype]
    x, res, w = (some(s, t, i).cuda() for i, s in enumerate([(rows, hidden), (rows, hidden),
                                                             (hidden,)]))
    x[rows // 2] *= 100
    if rows > 2:
        x[2], res[2] = 0, 0
    h = (x.float() + res.float()).to(t)
    for name in ("residual", "plain", "unaligned"):
        if name == "plain":
            out = run_op("rms_norm_mx", {"x": h, "w": w}, ("codes", "scales"), {"format": form})
        else:
            a = (x, res, w) if name == "residual" else tuple(unaligned(v) for v in (x, res, w))
            out = run_op("rms_norm_mx", {"x": a[0], "w": a[1 + 1], "r": a[1]},
                         ("codes", "scales", "h"), {"format": form, "eps": 1e-6})
            assert torch.equal(out["h"], h)
        c, s = mx.quantize(mx.rms_norm32(h.float().cpu().numpy(), w.float().cpu().numpy(), 1e-6),
                           form)
        assert np.array_equal(host(out["scales"]), s)
        assert np.array_equal(host(out["codes"]), c)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
def test_norm_of_special_rows(form):
    """A NaN or an infinity spoils its own row: every block of it becomes NaN (an infinite mean makes
    the other values 0, the infinity itself NaN)."""
    x, w = some((6, 96), torch.float32, 1), torch.ones(96)
    clean = run_op("rms_norm_mx", {"x": x.cuda(), "w": w.cuda()}, ("codes", "scales"),
                   {"format": form})
    x[1, 4], x[3, 40] = float("nan"), float("inf")
    x[5] *= 1e30  # squares past the range of 32 bits
    out = run_op("rms_norm_mx", {"x": x.cuda(), "w": w.cuda()}, ("codes", "scales"),
                 {"format": form})
    assert (out["scales"][1] == 255).all() and (out["codes"][1] == 0).all()
    assert out["scales"][3].tolist() == [0, 255, 0] and (out["codes"][3] & 119 == 0).all()
    keep = [0, 2, 4]
    assert torch.equal(out["codes"][keep], clean["codes"][keep])
    c, s = mx.quantize(mx.rms_norm32(x[5:].numpy(), w.numpy(), 1e-6), form)
    assert np.array_equal(host(out["codes"][5:]), c) and np.array_equal(host(out["scales"][5:]), s)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,ffn", [(1, 32), (1, 4864), (5, 96), (70, 928), (333, 4864)])
def test_gate(form, dtype, rows, ffn):
    t = DTYPES[dtype]
    g, u = some((rows, ffn), t, 1, 3.0), some((rows, ffn), t, 2)
    g[0, :8] = torch.tensor([0, -0.0, 60, -60, 88, -88, 100, -100])
    y = (g.double() / (1 + torch.exp(-g.double())) * u.double()).numpy()
    top = np.abs(y).reshape(-1, 32).max(1)[:, None]
    g, u = g.cuda(), u.cuda()
    outs = [run_op("silu_mul_mx", i, ("codes", "scales"), {"format": form}) for i in
            ({"g": g, "u": u}, {"g": torch.cat([g, u], -1)},
             {"g": unaligned(g), "u": unaligned(u)}, {"g": unaligned(torch.cat([g, u], -1))})]
    for out in outs[1:]:
        assert torch.equal(out["codes"], outs[0]["codes"])
        assert torch.equal(out["scales"], outs[0]["scales"])
    got = mx.values(host(outs[0]["codes"]), host(outs[0]["scales"]))
    # Where 32-bit arithmetic puts a value across a rounding border the code differs, so the values
    # are compared: half a step at the block's top, saturation included (test_mx_cpu.py), the
    # errors of exp, quotient and products (at most 2^-20) added.
    limit = 0.25 if form == "fp4" else 0.125
    assert (np.abs(got - y).reshape(-1, 32) <= top * (limit + 2.0 ** -20) + 2.0 ** -136).all()
    # and nearly every code is that of the 64-bit value
    c, s = mx.quantize(y, form)
    assert (host(outs[0]["codes"]) != c).mean() < 1e-3


# ---- the product -------------------------------------------------------------------------------


def check_linear(form, out_dtype, m, n, k, seed=0, bias=True, residual=True):
    x, w = some((m, k), torch.float32, seed), some((n, k), torch.float32, seed + 1, 0.05)
    x[:, ::37] *= 16
    q, p = quantized(x, form), quantized(w, "fp4")
    t = DTYPES[out_dtype]
    x64 = torch.from_numpy(mx.values(host(q[0]), host(q[1]))).cuda()
    w64 = torch.from_numpy(mx.values(host(p[0]), host(p[1]))).cuda()
    ref, terms = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    inputs, attrs = {"x": q[0], "xs": q[1], "w": p[0], "ws": p[1]}, {"out_dtype": out_dtype}
    if bias:
        inputs["b"] = some((n,), t, seed + 2).cuda()
        ref, terms = ref + inputs["b"].double(), terms + inputs["b"].double().abs()
    if residual:
        inputs["r"] = some((m, n), t, seed + 3).cuda()
        attrs["residual"] = True
        ref, terms = ref + inputs["r"].double(), terms + inputs["r"].double().abs()
    out = run_op("mx_linear", inputs, ("out",), attrs)["out"]
    assert out.dtype == t and out.shape == (m, n)
    # the output's rounding; fp32 sums of at most k / 8 + 3 terms (the unit sums 8 products at once);
    # e4m3 products of a 16-bit result lose what lies 2^-13 below the largest of 8 neighbours
    bound = UNIT[out_dtype] * ref.abs() + (k // 8 + 3) * 2.0 ** -23 * terms + TINY[out_dtype]
    if form == "fp8" and out_dtype != "float32":
        bound = bound + 2.0 ** -13 * terms
    err = (out.double() - ref).abs()
    assert (err <= bound).all(), (err - bound).max()
    # what goes missing on average is far less than the worst case allows
    rel = (err.norm() / ref.norm()).item()
    assert rel < {"bfloat16": 2.5e-3, "float16": 4e-4, "float32": 1e-6}[out_dtype], rel
    return inputs, attrs, out


SHAPES = [(1, 1, 32), (1, 1152, 896), (3, 50, 64), (16, 17, 96), (17, 896, 4864), (32, 100, 928),
          (33, 70, 128), (64, 4608, 3584), (65, 33, 160), (100, 1003, 1056), (128, 256, 256),
          (129, 257, 288), (333, 1003, 928), (300, 3584, 4864), (1000, 640, 896)]


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("out_dtype", list(DTYPES))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(form, out_dtype, m, n, k):
    check_linear(form, out_dtype, m, n, k)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("m", [2, 40, 200])
def test_linear_with_and_without_its_epilogue(form, m):
    for bias in (False, True):
        for residual in (False, True):
            check_linear(form, "bfloat16", m, 200, 512, 7, bias, residual)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("m,k", [(1, 256), (20, 928), (150, 896)])
def test_linear_rows_do_not_touch(form, m, k):
    """A NaN scale spoils its activation row or its weight's column, and nothing else; scales from
    one end of the range to the other multiply exactly."""
    inputs, attrs, clean = check_linear(form, "float32", m, 90, k, 11)
    q = {name: t.clone() for name, t in inputs.items()}
    q["xs"][m - 1, k // 32 - 1] = 255
    q["ws"][7, 0] = 255
    out = run_op("mx_linear", q, ("out",), attrs)["out"]
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[m - 1], bad[:, 7] = True, True
    assert out[bad].isnan().all() and torch.equal(out[~bad], clean[~bad])
    del q["b"], q["r"]
    plain = run_op("mx_linear", {**q, "xs": inputs["xs"], "ws": inputs["ws"]}, ("out",),
                   {"out_dtype": "float32"})["out"]
    for up in (100, -100):  # 2^up * 2^-up = 1
        shifted = run_op("mx_linear", {**q, "xs": (inputs["xs"].int() + up).to(torch.uint8),
                                       "ws": (inputs["ws"].int() - up).to(torch.uint8)}, ("out",),
                         {"out_dtype": "float32"})["out"]
        assert torch.equal(shifted, plain)


def test_linear_of_leading_dimensions_and_slices():
    """Rows behind a slice of a larger batch: views with an offset, as a batch is cut."""
    inputs, _, out = check_linear("fp8", "bfloat16", 12, 48, 96, 3, residual=False)
    cut = {**inputs, "x": inputs["x"].view(3, 4, 96)[1:], "xs": inputs["xs"].view(3, 4, 3)[1:]}
    got = run_op("mx_linear", cut, ("out",), {})["out"]
    assert got.shape == (2, 4, 48) and torch.equal(got.view(8, 48), out[4:])
    tail = {"x": inputs["x"], "xs": inputs["xs"], "w": inputs["w"][3:], "ws": inputs["ws"][3:]}
    got = run_op("mx_linear", tail, ("out",), {})["out"]  # scales at an odd address
    whole = run_op("mx_linear", {n: inputs[n] for n in ("x", "xs", "w", "ws")}, ("out",), {})["out"]
    assert torch.equal(got, whole[:, 3:])


def test_operators_refuse_what_they_cannot_take():
    x = torch.randn(2, 64).cuda()
    c, s = quantized(x, "fp4")
    for op, inputs, outputs, attrs, text in [
            ("mx_quantize", {"x": torch.randn(2, 40).cuda()}, ("a", "b"), {}, "multiple of 32"),
            ("mx_quantize", {"x": x}, ("a", "b"), {"format": "fp6"}, "format must be"),
            ("mx_quantize", {"x": c}, ("a", "b"), {}, "float32, bfloat16 or float16"),
            ("mx_quantize", {"x": x}, ("a",), {}, "arity"),
            ("mx_dequantize", {"c": c, "s": s[:1]}, ("a",), {}, "different rows"),
            ("mx_dequantize", {"c": c[:, :20].contiguous(), "s": s}, ("a",), {}, "not a micro"),
            ("mx_dequantize", {"c": c, "s": s}, ("a",), {"dtype": "int64"}, "floating type"),
            ("rms_norm_mx", {"x": x, "w": torch.ones(32).cuda()}, ("a", "b"), {}, "weight size"),
            ("rms_norm_mx", {"x": x, "w": torch.ones(64).cuda().half()}, ("a", "b"), {}, "dtype"),
            ("silu_mul_mx", {"g": x, "u": x.half()}, ("a", "b"), {}, "dtype"),
            ("silu_mul_mx", {"g": x[:, :33].contiguous()}, ("a", "b"), {}, "even"),
            ("mx_linear", {"x": c, "xs": s, "w": c, "ws": s, "b": x}, ("a",), {}, "bias"),
            ("mx_linear", {"x": c, "xs": s, "w": c, "ws": s, "r": x}, ("a",), {"residual": True},
             "residual"),
            ("mx_linear", {"x": c, "xs": s, "w": c, "ws": s.int()}, ("a",), {}, "uint8")]:
        with pytest.raises(ValueError, match=text):
            run_op(op, inputs, outputs, attrs)
    wide = torch.zeros(49, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="16-byte aligned"):
        run_op("mx_linear", {"x": wide[1:33].view(1, 32), "xs": s[:1, :1].contiguous(),
                             "w": c[:, :16].contiguous(), "ws": s[:, :1].contiguous()}, ("a",), {})


# ---- a run of them together --------------------------------------------------------------------


def mlp_graph(form):
    import json

    def node(op, i, o, **attrs):
        return {"name": o[0], "op": op, "inputs": i, "outputs": o, "attrs": attrs}

    nodes = [node("rms_norm_mx", ["x", "norm", "r"], ["a", "as", "h"], format=form),
             node("mx_linear", ["a", "as", "gu", "gus"], ["y"]),
             node("silu_mul_mx", ["y"], ["m", "ms"], format=form),
             node("mx_linear", ["m", "ms", "down", "downs", "h"], ["out"], residual=True)]
    inputs = ["x", "r", "norm", "gu", "gus", "down", "downs"]
    return dli.Graph.from_json(json.dumps({"format": "dli.graph.v1", "model_type": "mlp",
                                           "inputs": inputs, "outputs": ["h", "out"],
                                           "nodes": nodes}))


def mlp_inputs(rows, hidden=256, ffn=608):
    x, r, norm = (some(s, torch.bfloat16, i).cuda() for i, s in
                  enumerate([(rows, hidden), (rows, hidden), (hidden,)]))
    gu = quantized(some((2 * ffn, hidden), torch.float32, 5, 0.05), "fp4")
    down = quantized(some((hidden, ffn), torch.float32, 6, 0.05), "fp4")
    return {"x": x, "r": r, "norm": norm, "gu": gu[0], "gus": gu[1], "down": down[0],
            "downs": down[1]}


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("rows", [1, 33, 200])
def test_an_mlp(form, rows):
    """Norm, product, gate and product as one graph, each step against the same step in 64 bits on
    what the graph's step before it gave (the operators themselves, one at a time)."""
    t = mlp_inputs(rows)
    out = plugin_engine().run(mlp_graph(form), t)
    a = run_op("rms_norm_mx", {"x": t["x"], "w": t["norm"], "r": t["r"]}, ("a", "s", "h"),
               {"format": form})
    assert torch.equal(out["h"], a["h"])
    v = mx.values(host(a["a"]), host(a["s"])) @ mx.values(host(t["gu"]), host(t["gus"])).T
    y = torch.from_numpy(v).bfloat16().double().numpy()
    f = y.shape[1] // 2
    m = mx.values(*mx.quantize(y[:, :f] / (1 + np.exp(-y[:, :f])) * y[:, f:], form))
    want = m @ mx.values(host(t["down"]), host(t["downs"])).T + host(a["h"].double())
    err = host(out["out"].double()) - want
    # a bfloat16 y on the other side of a rounding border moves codes of m by a step, here and there:
    # held to a tenth of what quantising m (2^-4 and 2^-2 relative, at random) does to the sum
    size = np.linalg.norm(m @ mx.values(host(t["down"]), host(t["downs"])).T) / np.sqrt(err.size)
    assert np.sqrt((err ** 2).mean()) <= 2.0 ** -9 * np.sqrt((want ** 2).mean()) + size * (
        0.025 if form == "fp4" else 0.00625)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("rows", [1, 33, 200])
def test_captured_and_replayed(form, rows):
    """Two captured graphs and eager runs between their replays, each replay against the eager run
    on the same inputs."""
    engine, graph = plugin_engine(), mlp_graph(form)
    t = mlp_inputs(rows)
    fresh = [some((rows, 256), torch.bfloat16, 20 + i).cuda() for i in range(3)]
    want = [{k: v.clone() for k, v in engine.run(graph, {**t, "x": x}).items()} for x in fresh]
    captured = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        static = t["x"].clone()
        with torch.cuda.graph(g):
            out = engine.run(graph, {**t, "x": static})
        captured.append((g, static, out))
    for step in range(3):
        for i, (g, static, out) in enumerate(captured):
            static.copy_(fresh[(step + i) % 3])
            g.replay()
            eager = engine.run(graph, {**t, "x": fresh[step]})
            torch.cuda.synchronize()
            for name in ("h", "out"):
                assert torch.equal(out[name], want[(step + i) % 3][name])
                assert torch.equal(eager[name], want[step][name])


def test_on_another_stream_and_two_at_once():
    engine, graph = plugin_engine(), mlp_graph("fp8")
    a, b = mlp_inputs(200), mlp_inputs(40)
    b["x"] = b["x"] * 2
    want_a, want_b = engine.run(graph, a), engine.run(graph, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got_a = engine.run(graph, a, stream=streams[0].cuda_stream)
        with torch.cuda.stream(streams[1]):
            got_b = engine.run(graph, b)
        for s in streams:
            s.synchronize()
        for name in ("h", "out"):
            assert torch.equal(got_a[name], want_a[name])
            assert torch.equal(got_b[name], want_b[name])


def test_offsets_past_32_bits():
    """The last rows of tensors of more than 2^31 bytes (and, in the product's output, elements)."""
    rows, k = 70001, 32768
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-2:] = some((2, k), torch.bfloat16, 1).cuda()
    out = run_op("mx_quantize", {"x": x}, ("codes", "scales"), {"format": "fp8"})
    c, s = mx.quantize(x[-2:].double().cpu().numpy(), "fp8")
    assert np.array_equal(host(out["codes"][-2:]), c)
    assert np.array_equal(host(out["scales"][-2:]), s)
    assert not out["codes"][:-2].any() and not out["scales"][:-2].any()
    back = run_op("mx_dequantize", {"c": out["codes"], "s": out["scales"]}, ("out",),
                  {"dtype": "bfloat16"})["out"]
    assert torch.equal(back[-2:].cpu(), torch.from_numpy(mx.values(c, s)).bfloat16())
    w = quantized(some((40, k), torch.float32, 2, 0.05), "fp4")
    y = run_op("mx_linear", {"x": out["codes"], "xs": out["scales"], "w": w[0], "ws": w[1]},
               ("out",), {})["out"]
    few = run_op("mx_linear", {"x": out["codes"][-2:], "xs": out["scales"][-2:], "w": w[0],
                               "ws": w[1]}, ("out",), {})["out"]
    assert not y[:-2].any()
    ref = mx.values(c, s) @ mx.values(host(w[0]), host(w[1])).T
    for got in (y[-2:], few):
        assert np.linalg.norm(host(got.double()) - ref) <= 2.5e-3 * np.linalg.norm(ref)
    del x, out, back, y
    q = quantized(some((34000, 32), torch.float32, 3), "fp8")
    w = quantized(some((70000, 32), torch.float32, 4), "fp4")
    y = run_op("mx_linear", {"x": q[0], "xs": q[1], "w": w[0], "ws": w[1]}, ("out",), {})["out"]
    assert y.numel() > 2 ** 31
    ref = (mx.values(host(q[0][-3:]), host(q[1][-3:])) @ mx.values(host(w[0]), host(w[1])).T)
    assert np.linalg.norm(host(y[-3:].double()) - ref) <= 2.5e-3 * np.linalg.norm(ref)


@pytest.mark.parametrize("form,out_dtype", [("fp8", "bfloat16"), ("fp4", "float16"),
                                            ("fp8", "float32"), ("fp4", "float32")])
@pytest.mark.parametrize("m,n,k", [
    (3001, 4104, 416), (1537, 8193, 288),   # tiles of 256 x 256, partly past every end
    (4100, 8200, 416), (4200, 8193, 96), (4100, 4104, 768),  # more than one to a CU
    (64, 33000, 2176), (17, 32803, 2048),   # one run of columns per CU
    (50, 9001, 896), (60, 9001, 1056),      # tiles of 64 rows, on scales as they are and laid out
    (60, 4700, 3712), (50, 1300, 8224), (300, 1003, 8288),  # and parts of K
    (2047, 1300, 2336), (90, 520, 8256), (40, 200, 6272)])
def test_linear_of_many_tiles(form, out_dtype, m, n, k):
    check_linear(form, out_dtype, m, n, k)


def c_linear(form, t, m, n, k, workspace=None, ws_bytes=0, out=None):
    """The C entry point on the tensors of check_linear's inputs."""
    out = torch.empty_like(t["r"]) if out is None else out
    hip.call("dli_hip_mx_linear", hip.MX_FP8 if form == "fp8" else hip.MX_FP4, hip.dtype_code(out),
             hip.ptr(t["x"]), hip.ptr(t["xs"]), hip.ptr(t["w"]), hip.ptr(t["ws"]), hip.ptr(t["b"]),
             hip.ptr(t["r"]), hip.ptr(out), m, n, k, workspace, ws_bytes, hip.current_stream())
    return out


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("m,n,k", [(40, 200, 6272), (60, 4700, 3712), (50, 1300, 8224),
                                   (300, 1003, 8288), (700, 1300, 640)])
def test_linear_with_any_workspace(form, m, n, k):
    """Without a workspace, with one that is too small or not aligned, and with one of any content
    inside a larger buffer whose ends stay as they were."""
    inputs, _, out = check_linear(form, "float32", m, n, k)
    size = hip.lib().dli_hip_mx_linear_workspace(hip.MX_FP8 if form == "fp8" else hip.MX_FP4, m, n, k)
    # two orders of the same fp32 sums, each within the bound of check_linear
    x, w = (np.abs(mx.values(host(inputs[a]), host(inputs[b]))) for a, b in (("x", "xs"), ("w", "ws")))
    terms = torch.from_numpy(x @ w.T).cuda() + inputs["b"].abs() + inputs["r"].abs()
    bound = (k // 8 + 4) * 2.0 ** -22 * terms

    def close(got):
        assert ((got.double() - out.double()).abs() <= bound).all()

    close(c_linear(form, inputs, m, n, k))
    buffer = torch.full((size + 512,), 255, dtype=torch.uint8, device="cuda")
    for offset, count in ((256, size), (256, size - 1), (260, size)):
        if count <= 0:
            continue
        buffer.fill_(255)
        got = c_linear(form, inputs, m, n, k, buffer.data_ptr() + offset, count)
        close(got)
        assert (buffer[:256] == 255).all() and (buffer[256 + size:] == 255).all()
    # the residual's own memory as the output
    alias = inputs["r"].clone()
    got = c_linear(form, {**inputs, "r": alias}, m, n, k, buffer.data_ptr() + 256, size, out=alias)
    close(got)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,hidden", [(3, 96), (5, 896), (4, 3584), (2, 8192), (3, 9000 // 32 * 32),
                                         (70000, 32)])
def test_norm_in_place(dtype, rows, hidden):
    """hidden_out as x or as the residual, at every width of the kernel and past 65535 rows."""
    t = DTYPES[dtype]
    x, r, w = (some(s, t, i).cuda() for i, s in enumerate([(rows, hidden), (rows, hidden),
                                                           (hidden,)]))
    want = run_op("rms_norm_mx", {"x": x, "w": w, "r": r}, ("c", "s", "h"), {"format": "fp8"})
    assert torch.equal(want["h"], (x.float() + r.float()).to(t))
    for which in ("x", "r", None):
        a, b = x.clone(), r.clone()
        to = {"x": a, "r": b, None: None}[which]
        c = torch.empty(rows, hidden, dtype=torch.uint8, device="cuda")
        s = torch.empty(rows, hidden // 32, dtype=torch.uint8, device="cuda")
        hip.call("dli_hip_rms_norm_mx", hip.dtype_code(x), hip.MX_FP8, hip.ptr(a), hip.ptr(b),
                 hip.ptr(w), hip.ptr(to), hip.ptr(c), hip.ptr(s), rows, hidden, 1e-6,
                 hip.current_stream())
        assert torch.equal(c, want["c"]) and torch.equal(s, want["s"])
        if to is not None:
            assert torch.equal(to, want["h"])
