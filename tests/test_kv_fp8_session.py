"""The 8-bit KV cache through the engine on host tensors (the ATen CPU plugin): entries, sessions,
what is refused. No GPU."""
import numpy as np
import pytest
import torch

import dli
from dli_qwen2 import DecodeSession, build_decode_graph, build_prefill_graph, random_weights, tiny_config
from kv_fp8_oracle import Cache
from kv_fp8_session import cache_of, check_nodes, f64
from mx_session import exposed
from support import one_node_graph


def engine(**more):
    e = dli.Engine().load_aten_plugin()
    if more:
        e.configure_kv_cache(**more)
    return e


def normal(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


ATTENTION = one_node_graph("attention", ["q", "k", "v"], attrs={"causal": True, "kv_cache": "c"})
AT = one_node_graph("attention", ["q", "k", "v", "p"], attrs={"causal": True, "kv_cache": "c"})


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_host_entries(dtype):
    """Appended by the tracked length and by positions, quantised as the oracle has it, read back."""
    e = engine(block_size=16, max_seq_len=48, format="fp8")
    want = None
    for step, (seq, where) in enumerate(((20, None), (1, None), (3, [30, 45]))):
        k, v = normal((2, 2, seq, 24), step, dtype), normal((2, 2, seq, 24), 9 + step, dtype)
        k[0, 0, 0], v[1, 1, seq - 1, 3] = 0, float("nan")
        q = normal((2, 4, seq, 24), 20 + step, dtype)
        inputs = {"q": q, "k": k, "v": v}
        if where is None:
            e.run(ATTENTION, inputs)
        else:
            e.run(AT, {**inputs, "p": torch.tensor(where)})
        if want is None:
            held = cache_of(e, "c")
            want = Cache(*(np.zeros_like(x) for x in (held.key, held.value, held.scales)), held.table)
            first = [0, 0]
        want.append(f64(k), f64(v), where or first)
        first = [x + seq for x in first]
        held = cache_of(e, "c")
        for pool in ("key", "value", "scales"):
            assert np.array_equal(getattr(held, pool), getattr(want, pool))
    assert e.kv_cache_entry("c")["length"] == 21
    for start, length in ((0, 48), (19, 3), (30, 0), (47, 1)):
        got = e.read_kv_cache("c", start, length, "float32")
        for x, y in zip(got, want.read([start] * 2, length)):
            assert np.array_equal(x.double().numpy(), y, equal_nan=True)
    assert e.read_kv_cache("c", 0, 5)[0].dtype == dtype
    for bad in ((-1, 2), (0, 49), (48, 1), (3, -1), (2, 1 << 62)):
        with pytest.raises(IndexError):
            e.read_kv_cache("c", *bad)


def test_plain_entries_are_read_too():
    e = engine(block_size=16, max_seq_len=32)
    k, v = normal((2, 2, 20, 24), 1), normal((2, 2, 20, 24), 2)
    e.run(ATTENTION, {"q": normal((2, 4, 20, 24), 3), "k": k, "v": v})
    got = e.read_kv_cache("c", 3, 17)
    assert torch.equal(got[0], k[:, :, 3:]) and torch.equal(got[1], v[:, :, 3:])
    assert "scales" not in e.kv_cache_entry("c")


def test_refusals():
    e = engine(block_size=16, max_seq_len=32, format="fp8")
    with pytest.raises(ValueError, match="format"):
        e.configure_kv_cache(format="int8")
    with pytest.raises(ValueError, match="unknown entry"):
        e.read_kv_cache("c", 0, 1)
    with pytest.raises(ValueError, match="head_dim"):
        e.run(ATTENTION, {n: normal((1, 1, 2, 257), 1) for n in "qkv"})
    e.run(ATTENTION, {n: normal((1, 1, 2, 8), 1) for n in "qkv"})
    with pytest.raises(ValueError, match="dtype mismatch"):
        e.run(ATTENTION, {n: normal((1, 1, 2, 8), 1).bfloat16() for n in "qkv"})
    with pytest.raises(IndexError):
        e.run(AT, {**{n: normal((1, 1, 2, 8), 1) for n in "qkv"}, "p": torch.tensor([31])})
    with pytest.raises(ValueError):
        e.read_kv_cache("c", 0, 1, "int64")
    cfg = tiny_config(layers=1)
    with pytest.raises(ValueError, match="kv must be"):
        build_decode_graph(cfg, 1, kv="int8")
    with pytest.raises(ValueError, match="stack"):
        build_decode_graph(cfg, 1, stack=True, kv="fp8")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mx", [None, "fp8"])
def test_decode_steps_node_by_node(dtype, mx):
    cfg = tiny_config(ffn=1216)
    s = DecodeSession(cfg, random_weights(cfg, seed=1, dtype=dtype), 2, max_seq_len=32, fused=False,
                      engine=engine(), device="cpu", mx=mx, kv="fp8")
    graph, nodes = exposed(s.graph)
    s.step(torch.tensor([5, 900]), torch.tensor([0, 0]))
    ids = torch.tensor([7, 8])
    for past in ([1, 1], [2, 2], [9, 3]):
        before = {f"layer_{i}": cache_of(s.engine, f"layer_{i}") for i in range(2)}
        s.ids.copy_(ids)
        s.positions.copy_(torch.tensor(past))
        out = s.engine.run(graph, s.inputs)
        assert check_nodes(s.engine, nodes, {**s.inputs, **out}, past, before) == {
            "append": 2, "attention": 2}
        ids = out["next_ids"]


def test_a_prompt_in_one_run_and_by_steps():
    """The prompt's queries see the quantised keys and values, as the steps' do."""
    cfg = tiny_config(ffn=1216)
    w = random_weights(cfg, seed=2, dtype=torch.float32)
    prompt = torch.randint(0, cfg.vocab, (2, 5), generator=torch.Generator().manual_seed(3))

    def session(**more):
        return DecodeSession(cfg, w, 2, max_seq_len=32, fused=False, engine=engine(), device="cpu",
                             kv="fp8", **more)

    s, steps = session(prefill=True), session()
    graph, nodes = exposed(build_prefill_graph(cfg, 2, 5, fused_head=False))
    s.run_prefill(prompt)
    before = {f"layer_{i}": cache_of(s.engine, f"layer_{i}") for i in range(2)}
    s.engine.set_kv_cache_length(0)
    out = s.engine.run(graph, {**s.inputs, "input_ids": prompt})
    assert check_nodes(s.engine, nodes, {**s.inputs, **out}, [0, 0], before)["attention"] == 2
    for t in range(5):
        logits, _ = steps.step(prompt[:, t], torch.full((2,), t))
    # sums in another order (fp32) move an element that lies at a border to its neighbour now and then:
    # 2^-4 of one of 64 or more elements of a row, far below a quarter of that in a row's length
    assert torch.norm(logits - out["logits"]) <= 2.0 ** -6 * torch.norm(logits)
    assert s.generate(prompt, 3).shape == (2, 3)
