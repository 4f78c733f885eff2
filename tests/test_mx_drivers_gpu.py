"""Microscaled graphs under the C++ decode driver, several steps in one captured graph, runs and
captures on a stream that is not torch's current one, and the C++ runner."""
import numpy as np
import pytest
import torch

import dli
from dli import hip
from dli_qwen2 import DecodeSession, build_decode_graph, pack_mx_weights, random_weights, tiny_config
from support import one_node_graph, plugin_engine
from test_mx_stream_gpu import coded

pytestmark = pytest.mark.gpu
CFG = tiny_config(ffn=1216)


def case(batch, seed):
    w = {n: t.cuda() for n, t in random_weights(CFG, seed=seed).items()}
    return w, torch.randint(0, CFG.vocab, (batch, 5), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("capture", [True, False], ids=["replay", "eager"])
@pytest.mark.parametrize("batch", [4, 40])
def test_cpp_driver(form, capture, batch):
    w, prompt = case(batch, 51)
    want = DecodeSession(CFG, w, batch, max_seq_len=64, mx=form).capture().generate(prompt.cuda(), 7).cpu()
    engine = dli.Engine().load_plugin()
    d = dli.GreedyDecoder(engine, build_decode_graph(CFG, batch, mx=form),
                          pack_mx_weights(CFG, w, engine), batch, max_seq_len=64, capture=capture)
    assert torch.equal(d.generate(prompt, 7), want)
    assert torch.equal(d.generate(prompt.cuda(), 7), want)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
def test_several_steps_in_one_graph(form):
    w, prompt = case(4, 52)
    first = prompt[:, 0].cuda()
    one = DecodeSession(CFG, w, 4, max_seq_len=64, mx=form)
    ids, want = first, []
    for t in range(6):
        ids = one.step(ids, torch.full((4,), t, device="cuda"))[1].clone()
        want.append(ids)
    many = DecodeSession(CFG, w, 4, max_seq_len=64, mx=form)
    many.capture(chain_ids=True, steps=3)
    many.ids.copy_(first)
    for turn in range(2):
        for i in range(3):
            many.step_positions[i].fill_(3 * turn + i)
        out = many.replay()
        torch.cuda.synchronize()
        assert torch.equal(out["next_ids"], want[3 * turn + 2])


def product(m, n, k, form="fp8"):
    x, xs, _ = coded(m, k, form, 1)
    w, ws, _ = coded(n, k, "fp4", 2)
    inputs = {"x": x, "xs": xs, "w": w, "ws": ws}
    size = hip.lib().dli_hip_mx_linear_workspace(hip.MX_FP8, m, n, k)
    assert size > 0
    return one_node_graph("mx_linear", list(inputs), ["out"], {"out_dtype": "float32"}), inputs, size


# parts of K, laid out scales, both; large tiles
PRODUCTS = [(64, 3584, 3584), (300, 11520, 4224), (484, 3584, 8192), (3001, 4104, 1824)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_workspace_given_back_waits_for_the_run(m, n, k):
    g, inputs, size = product(m, n, k)
    engine = plugin_engine()
    ref = engine.run(g, inputs)["out"].clone()
    side = torch.cuda.Stream()
    engine.run(g, inputs, stream=side.cuda_stream)
    spare = [torch.full((size // 4,), 7.0, device="cuda") for _ in range(8)]
    del spare
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    out = engine.run(g, inputs, stream=side.cuda_stream)["out"]
    taken = [torch.full((size // 4,), 7.0, device="cuda") for _ in range(4)]
    assert not side.query()
    torch.cuda.synchronize()
    assert torch.equal(out, ref)
    assert all((t == 7.0).all() for t in taken)


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_capture_of_another_stream_takes_no_workspace(m, n, k):
    g, inputs, size = product(m, n, k)
    engine = plugin_engine()
    ref = engine.run(g, inputs)["out"].clone()
    # the form without a workspace, its code objects loaded before the capture
    plain = torch.empty_like(ref)
    hip.call("dli_hip_mx_linear", hip.MX_FP8, hip.F32, *(hip.ptr(inputs[i]) for i in ("x", "xs", "w", "ws")),
             None, None, hip.ptr(plain), m, n, k, None, 0, hip.current_stream())
    torch.cuda.synchronize()
    captured, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    other = torch.cuda.current_stream()
    with torch.cuda.stream(side):
        captured.capture_begin(capture_error_mode="relaxed")
        with torch.cuda.stream(other):
            out = engine.run(g, inputs, stream=side.cuda_stream)["out"]
        captured.capture_end()
    taken = [torch.full((size // 4,), 7.0, device="cuda") for _ in range(4)]
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            captured.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, plain)
        # two orders of the same sums
        assert (out - ref).double().norm() <= 1e-6 * ref.double().norm()
        assert all((t == 7.0).all() for t in taken)


def test_codes_through_the_cpp_runner(tmp_path):
    from test_operator_runner import _NP, run_runner
    import mx_oracle as mx

    x = torch.randn(3, 96, generator=torch.Generator().manual_seed(1))
    _NP.setdefault("uint8", np.uint8)
    nodes = [{"name": "q", "op": "mx_quantize", "inputs": ["x"], "outputs": ["codes", "scales"],
              "attrs": {"format": "fp4"}}]
    for plugin, device in ((dli.aten_plugin_path(), "cpu"), (dli.plugin_path(), "cuda")):
        (tmp_path / device).mkdir()
        rc, err, out = run_runner(tmp_path / device, nodes, {"x": x}, ["codes", "scales"], plugin, device)
        assert rc == 0, err
        codes, scales = mx.quantize(x.double().numpy(), "fp4")
        assert np.array_equal(out["codes"], codes) and np.array_equal(out["scales"], scales)
