"""Decode sessions on microscaled linears, host tensors (the ATen CPU plugin). No GPU."""
import json
from dataclasses import replace

import numpy as np
import pytest
import torch

import dli
import mx_oracle as mx
from dli_qwen2 import (DecodeSession, build_decode_graph, build_prefill_graph, pack_mx_weights,
                       random_weights, tiny_config)
from mx_session import check_nodes, check_step, exposed, raw


def engine():
    return dli.Engine().load_aten_plugin()  # (an engine holds one cache)


def session(cfg, w, batch, mx_format, **more):
    return DecodeSession(cfg, w, batch, max_seq_len=32, fused=False, engine=engine(), device="cpu",
                         mx=mx_format, **more)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_step_node_by_node(form, dtype):
    cfg = tiny_config(ffn=1216)
    s = session(cfg, random_weights(cfg, seed=1, dtype=dtype), 3, form)
    ids = torch.tensor([5, 900, 17])
    for t in range(2):
        out = check_step(s, ids, torch.full((3,), t))
        ids = out["next_ids"]
        assert out["layers_1_output"].dtype == dtype
        assert torch.equal(out["logits"].argmax(-1), ids)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
def test_prompt_node_by_node_and_against_steps(form):
    cfg = tiny_config(ffn=1216)
    w = random_weights(cfg, seed=2, dtype=torch.float32)
    prompt = torch.randint(0, cfg.vocab, (2, 5), generator=torch.Generator().manual_seed(3))
    s = session(cfg, w, 2, form, prefill=True)
    graph, nodes = exposed(build_prefill_graph(cfg, 2, 5, fused_head=False, mx=form,
                                               dtype="float32"))
    s.engine.set_kv_cache_length(0)
    out = s.engine.run(graph, {**s.inputs, "input_ids": prompt})
    assert check_nodes(nodes, {**s.inputs, **out})["mx_linear"] == 12
    logits, ids = s.run_prefill(prompt)
    assert torch.equal(logits, out["logits"])
    steps = session(cfg, w, 2, form)
    for t in range(5):
        stepped, _ = steps.step(prompt[:, t], torch.full((2,), t))
    # attention sums in another order (fp32): now and then an element falls on its neighbour, which
    # moves a row of 896 by 2^-4 / sqrt(896) = 0.2 % (e2m1: 0.8 %) of its length
    assert torch.norm(stepped - logits) <= 2.0 ** (-6 if form == "fp8" else -4) * torch.norm(logits)
    assert s.generate(prompt, 3).shape == (2, 3)


def test_packed_weights():
    cfg = tiny_config(layers=1, ffn=1216)
    w = random_weights(cfg, seed=4)
    packed = pack_mx_weights(cfg, w, engine())
    p = "model.layers.0"
    gate_up = torch.cat([w[f"{p}.mlp.gate_proj.weight"], w[f"{p}.mlp.up_proj.weight"]])
    for name, weight in ((f"{p}.self_attn.k_proj", w[f"{p}.self_attn.k_proj.weight"]),
                         (f"{p}.mlp.gate_up_proj", gate_up)):
        codes, scales = mx.quantize(weight.double().numpy(), "fp4")
        assert np.array_equal(raw(packed[f"{name}.weight.codes"]), codes)
        assert np.array_equal(raw(packed[f"{name}.weight.scales"]), scales)
        assert f"{name}.weight" not in packed
    assert f"{p}.mlp.up_proj.weight" not in packed and f"{p}.mlp.up_proj.weight" in w
    assert packed["lm_head.weight"] is w["lm_head.weight"]


def test_refusals():
    cfg = tiny_config(layers=1, ffn=1216)
    w = random_weights(cfg, seed=4)
    with pytest.raises(ValueError, match="fp8 or fp4"):
        session(cfg, w, 1, "int4")
    with pytest.raises(ValueError, match="no decoder stack"):
        DecodeSession(cfg, w, 1, 32, engine=engine(), device="cpu", mx="fp8", stack=True)
    for odd in (replace(cfg, ffn=1200), replace(cfg, hidden=880), replace(cfg, head_dim=60, heads=15)):
        with pytest.raises(ValueError, match="multiple of 32"):
            build_decode_graph(odd, 1, mx="fp8")
        with pytest.raises(ValueError, match="multiple of 32"):
            build_prefill_graph(odd, 1, 4, mx="fp4")
    # the forms without it are what they were
    plain = json.loads(build_decode_graph(cfg, 1, fused=False).to_json())
    assert not any("mx" in n["op"] for n in plain["nodes"])
