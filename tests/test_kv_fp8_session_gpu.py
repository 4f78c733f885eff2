"""Decode sessions, prompts and the C++ driver on an 8-bit KV cache, on the GPU: every append and
attention against the oracle, captured steps against eager ones, two graphs at once, refusals."""
import json
from dataclasses import replace

import numpy as np
import pytest
import torch

import dli
from dli_qwen2 import DecodeSession, build_prefill_graph, random_weights, tiny_config
from dli_qwen2.graph import build_decode_graph, pack_fused_weights
from kv_fp8_oracle import Cache, check_attention
from kv_fp8_session import cache_of, check_nodes, f64
from mx_session import exposed
from support import one_node_graph

pytestmark = pytest.mark.gpu


def normal(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


LARGE = dict(hidden=1152, heads=9, kv_heads=3, head_dim=128, ffn=1280)


@pytest.mark.parametrize("form,cfg,dtype,more", [
    ("fused", {}, torch.bfloat16, {}), ("fused", {}, torch.bfloat16, {"block_size": 16}),
    ("fused", {}, torch.bfloat16, {"block_size": 24}),
    ("large", LARGE, torch.bfloat16, {}), ("unfused", {}, torch.float32, {"fused": False}),
    ("unfused", {}, torch.float16, {"fused": False}),
    ("mx", {"ffn": 1216}, torch.bfloat16, {"mx": "fp8"}), ("mx", {"ffn": 1216}, torch.float16, {"mx": "fp4"})])
def test_decode_steps_node_by_node(form, cfg, dtype, more):
    cfg = tiny_config(**cfg)
    s = DecodeSession(cfg, random_weights(cfg, seed=1, dtype=dtype, device="cuda"), 3, max_seq_len=160,
                      kv="fp8", **more)
    graph, nodes = exposed(s.graph)
    s.step(torch.tensor([5, 900, 2]).cuda(), torch.tensor([0, 0, 0]).cuda())
    ids = torch.tensor([7, 8, 9])
    for past in ([1, 1, 1], [2, 70, 127], [159, 3, 128]):
        before = {f"layer_{i}": cache_of(s.engine, f"layer_{i}") for i in range(2)}
        s.ids.copy_(ids)
        s.positions.copy_(torch.tensor(past))
        out = s.engine.run(graph, s.inputs)
        assert check_nodes(s.engine, nodes, {**s.inputs, **out}, past, before) == {
            "append": 2, "attention": 2}
        ids = out["next_ids"]


@pytest.mark.parametrize("fused,batch,seq", [(True, 2, 90), (False, 1, 7), (True, 1, 1)])
def test_prompt_node_by_node(fused, batch, seq):
    cfg = tiny_config()
    s = DecodeSession(cfg, random_weights(cfg, seed=2, device="cuda"), batch, max_seq_len=128, kv="fp8",
                      prefill=True)
    prompt = torch.randint(0, cfg.vocab, (batch, seq), generator=torch.Generator().manual_seed(3)).cuda()
    s.run_prefill(prompt)
    graph, nodes = exposed(build_prefill_graph(cfg, batch, seq, fused=fused))
    before = {f"layer_{i}": cache_of(s.engine, f"layer_{i}") for i in range(2)}
    s.engine.set_kv_cache_length(0)
    out = s.engine.run(graph, {**s.inputs, "input_ids": prompt})
    assert check_nodes(s.engine, nodes, {**s.inputs, **out}, [0] * batch, before)["attention"] == 2
    assert s.generate(prompt, 4).shape == (batch, 4)


@pytest.mark.parametrize("cfg", [{}, LARGE])
def test_captured_steps(cfg):
    """A captured step, replayed between eager steps of the same session, against an eager session."""
    cfg = tiny_config(**cfg)
    w = random_weights(cfg, seed=4, device="cuda")

    def session():
        return DecodeSession(cfg, w, 5, max_seq_len=192, kv="fp8")

    eager, captured = session(), session().capture()
    eager.run_eager()  # as capture does once: token 0 at position 0 of every sequence
    ids = torch.randint(0, cfg.vocab, (5,), generator=torch.Generator().manual_seed(5)).cuda()
    for step in range(8):
        pos = torch.tensor([step, step + 60, step + 128, 0, 180]).cuda()
        want, next_ids = eager.step(ids, pos)
        got, got_ids = captured.step(ids, pos)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got_ids, next_ids)
        if step % 3 == 1:
            again = captured.run_eager()
            assert torch.equal(again["logits"], want)
        ids = next_ids.clone()
    for i in range(2):
        a, b = (cache_of(s.engine, f"layer_{i}") for s in (eager, captured))
        for pool in ("key", "value", "scales"):
            assert np.array_equal(getattr(a, pool), getattr(b, pool))


def test_two_captured_graphs_at_once():
    """Two sessions on one plugin instance each, their graphs replayed on two streams at the same time:
    nothing is shared."""
    cfg = tiny_config()
    w = random_weights(cfg, seed=4, device="cuda")
    sessions = [DecodeSession(cfg, w, 4, max_seq_len=4096, kv="fp8") for _ in range(2)]
    for i, s in enumerate(sessions):
        s.positions.copy_(torch.tensor([4000, 3000 + i, 4095, 7]))
        s.ids.copy_(torch.tensor([1, 2, 3, 4 + i]))
        s.capture()
    want = []
    for s in sessions:
        s.replay()
        torch.cuda.synchronize()
        want.append({n: t.clone() for n, t in s._out.items()})
    streams = [torch.cuda.Stream() for _ in sessions]
    for _ in range(5):
        for s, stream in zip(sessions, streams):
            with torch.cuda.stream(stream):
                s.replay()
    torch.cuda.synchronize()
    for s, out in zip(sessions, want):
        for n, t in out.items():
            assert torch.equal(s._out[n], t), n


@pytest.mark.parametrize("capture", [True, False])
def test_cpp_driver(capture):
    cfg = tiny_config()
    w = random_weights(cfg, seed=51, device="cuda")
    prompt = torch.randint(0, cfg.vocab, (4, 7), generator=torch.Generator().manual_seed(52))
    want = DecodeSession(cfg, w, 4, max_seq_len=64, kv="fp8").generate(prompt.cuda(), 9).cpu()
    d = dli.GreedyDecoder(dli.Engine().load_plugin(), build_decode_graph(cfg, 4, kv="fp8"),
                          pack_fused_weights(cfg, w, drop_unfused=True), 4, max_seq_len=64,
                          capture=capture, kv_format="fp8")
    assert torch.equal(d.generate(prompt, 9), want)
    assert torch.equal(d.generate(prompt.cuda(), 9), want)


def chunk_graph():
    return dli.Graph.from_json(json.dumps({
        "format": "dli.graph.v1", "model_type": "chunk", "inputs": ["qkv", "cos", "sin", "p"],
        "outputs": ["q", "out"], "nodes": [
            {"name": "r", "op": "rope_append", "inputs": ["qkv", "cos", "sin", "p"], "outputs": ["q"],
             "attrs": {"kv_cache": "c", "q_heads": 14, "kv_heads": 2, "head_dim": 64}},
            {"name": "a", "op": "paged_attention", "inputs": ["q", "p"], "outputs": ["out"],
             "attrs": {"kv_cache": "c"}}]}))


@pytest.mark.parametrize("foreign", [False, True])
def test_a_chunk_of_drafted_tokens(foreign):
    """rope_append of several tokens and paged_attention of them, also on a stream that is not torch's."""
    e = dli.Engine().load_plugin()
    e.configure_kv_cache(block_size=64, max_seq_len=1024, format="fp8")
    angle = torch.arange(1024).double()[:, None] * 1000.0 ** (-torch.arange(32).double() / 32)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    graph, want = chunk_graph(), None
    stream = torch.cuda.Stream()
    for step, past in enumerate(([0, 0], [700, 3], [705, 40])):
        qkv = normal((2, 700 if step == 0 else 5, 18 * 64), step)
        p = torch.tensor(past, device="cuda")
        torch.cuda.synchronize()
        out = e.run(graph, {"qkv": qkv, "cos": cos, "sin": sin, "p": p},
                    stream=stream.cuda_stream if foreign else None)
        torch.cuda.synchronize()
        held = cache_of(e, "c")
        if want is None:
            want = Cache(*(np.zeros_like(x) for x in (held.key, held.value, held.scales)), held.table)
        check_nodes(e, [{"op": "rope_append", "name": "r", "inputs": ["qkv", "cos", "sin"],
                         "outputs": ["q"], "attrs": {"kv_cache": "c", "q_heads": 14, "kv_heads": 2,
                                                     "head_dim": 64}}],
                    {"qkv": qkv, "cos": cos, "sin": sin, "q": out["q"]}, past, {"c": want})
        rows = slice(None) if step else slice(690, 700)
        q = f64(out["q"][:, :, rows])
        check_attention(out["out"][:, :, rows],
                        held.attention(q, [x + (690 if step == 0 else 0) for x in past], True, 0.125),
                        torch.bfloat16, 1024, 64)
    got = e.read_kv_cache("c", 690, 20)
    for x, y in zip(got, want.read([690, 690], 20)):
        assert np.array_equal(x.float().cpu().numpy(), y)


def test_growth():
    """The tracked length past the configured one: blocks move, scales with them."""
    e = dli.Engine().load_plugin()
    e.configure_kv_cache(block_size=16, max_seq_len=32, format="fp8")
    graph = one_node_graph("attention", ["q", "k", "v"], attrs={"causal": True, "kv_cache": "c"})
    ks = []
    for step, seq in enumerate((30, 1, 40, 1)):
        k, v = normal((2, 2, seq, 64), step), normal((2, 2, seq, 64), 9 + step)
        q = normal((2, 4, seq, 64), 30 + step)
        out = e.run(graph, {"q": q, "k": k, "v": v})["output"]
        ks.append(k)
        past = sum(x.shape[2] for x in ks) - seq
        check_attention(out, cache_of(e, "c").attention(f64(q), [past] * 2, True, 0.125), torch.bfloat16,
                        128, 64)
    held = Cache(np.zeros((2, 2, 72, 64), np.uint8), np.zeros((2, 2, 64, 72), np.uint8),
                 np.zeros((2, 2, 2, 72), np.uint8), [[0], [1]])
    held.append(f64(torch.cat(ks, 2)), f64(torch.cat(ks, 2)), [0, 0])
    got = e.read_kv_cache("c", 0, 72, "float32")[0].cpu().double().numpy()
    assert np.array_equal(got, held.read([0, 0], 72)[0])


def test_plain_device_entries_are_read():
    e = dli.Engine().load_plugin()
    e.configure_kv_cache(block_size=16, max_seq_len=64)
    graph = one_node_graph("attention", ["q", "k", "v"], attrs={"causal": True, "kv_cache": "c"})
    k, v = normal((2, 2, 40, 64), 1), normal((2, 2, 40, 64), 2)
    e.run(graph, {"q": normal((2, 4, 40, 64), 3), "k": k, "v": v})
    got = e.read_kv_cache("c", 5, 30)
    assert torch.equal(got[0], k[:, :, 5:35]) and torch.equal(got[1], v[:, :, 5:35])


def test_refusals():
    """Operators that bind 16-bit pools do not take an 8-bit entry, nor the other way round; an entry is
    not made inside a capture."""
    cfg = replace(tiny_config(), layers=1)
    w = random_weights(cfg, seed=1, device="cuda")
    for more in ({}, {"stack": True}):
        s = DecodeSession(cfg, w, 2, max_seq_len=64, **more)
        s.engine.configure_kv_cache(format="fp8")
        with pytest.raises(ValueError, match="8-bit format"):
            s.run_eager()
    with pytest.raises(ValueError, match="stack"):
        DecodeSession(cfg, w, 2, max_seq_len=64, stack=True, kv="fp8")
    angle = torch.zeros((64, 32), device="cuda")
    good = {"qkv": normal((2, 18 * 64), 1), "cos": angle, "sin": angle,
            "p": torch.tensor([0, 0], device="cuda")}
    e = dli.Engine().load_plugin()
    e.configure_kv_cache(max_seq_len=64)
    with pytest.raises(ValueError, match="format fp8"):
        e.run(chunk_graph(), good)
    e = dli.Engine().load_plugin()
    e.configure_kv_cache(max_seq_len=64, format="fp8")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(graph):
            e.run(chunk_graph(), good)
    e.run(chunk_graph(), good)
    for change in ({"qkv": normal((2, 17 * 64), 1)}, {"qkv": normal((3, 18 * 64), 1)},
                   {"p": good["p"][:1]}, {"p": angle[:2, 0]}, {"cos": torch.zeros((64, 33), device="cuda")},
                   {"qkv": normal((2, 18 * 64), 1, torch.float16)}, {"qkv": good["qkv"].cpu()}):
        with pytest.raises(ValueError):
            e.run(chunk_graph(), {**good, **change})
    attend = one_node_graph("paged_attention", ["q", "p"], attrs={"kv_cache": "c"})
    for q in (normal((2, 14, 1, 128), 1), normal((2, 13, 1, 64), 1), normal((3, 14, 1, 64), 1),
              normal((2, 14, 1, 64), 1, torch.float16), normal((2, 14, 64), 1)):
        with pytest.raises(ValueError):
            e.run(attend, {"q": q, "p": good["p"]})
    with pytest.raises(ValueError, match="attention_splits"):
        e.run(one_node_graph("paged_attention", ["q", "p"], attrs={"kv_cache": "c", "attention_splits": 2}),
              {"q": normal((2, 14, 1, 64), 1), "p": good["p"]})
