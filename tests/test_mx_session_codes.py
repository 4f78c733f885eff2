"""Decode steps and prompts on microscaled linears, every node's codes against the oracle's."""
import pytest
import torch

import dli
from dli_qwen2 import DecodeSession, build_prefill_graph, random_weights, tiny_config
from mx_codes import check_codes
from mx_session import exposed

CFG = tiny_config(ffn=1216)


def host_session(weights, form):
    return DecodeSession(CFG, weights, 3, max_seq_len=32, fused=False, device="cpu", mx=form,
                         engine=dli.Engine().load_aten_plugin())


def check_a_step(s, ids):
    graph, nodes = exposed(s.graph)
    s.ids.copy_(ids)
    out = s.engine.run(graph, s.inputs)
    assert check_codes(nodes, {**s.inputs, **out}) == 9 * CFG.layers
    return nodes, {**s.inputs, **out}


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_on_the_host(form, dtype):
    s = host_session(random_weights(CFG, seed=1, dtype=dtype), form)
    check_a_step(s, torch.tensor([5, 900, 17]))


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("op", ["rms_norm_mx", "silu_mul_mx"])
def test_the_check_sees_lost_elements(form, op):
    """The smallest element codes of a node set to zero: values within a part of the block's largest,
    which a check of values lets pass."""
    s = host_session(random_weights(CFG, seed=1, dtype=torch.float32), form)
    nodes, tensors = check_a_step(s, torch.tensor([5, 900, 17]))
    name = next(n["outputs"][0] for n in nodes if n["op"] == op)
    codes = tensors[name]
    if form == "fp8":
        bad = torch.where((codes & 127) < 64, codes & 128, codes)
    else:
        bad = torch.where((codes & 7) < 2, codes & 0xF8, codes)
    assert not torch.equal(bad, codes)
    with pytest.raises(AssertionError):
        check_codes([n for n in nodes if name in n["outputs"]], {**tensors, name: bad})


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("batch", [1, 20])
def test_a_step_on_the_gpu(form, dtype, batch):
    w = {n: t.cuda() for n, t in random_weights(CFG, seed=1, dtype=dtype).items()}
    s = DecodeSession(CFG, w, batch, max_seq_len=32, mx=form)
    check_a_step(s, torch.arange(batch, device="cuda") * 7 + 3)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["fp8", "fp4"])
def test_a_prompt_on_the_gpu(form):
    w = {n: t.cuda() for n, t in random_weights(CFG, seed=2).items()}
    prompt = torch.randint(0, CFG.vocab, (2, 90), generator=torch.Generator().manual_seed(3)).cuda()
    s = DecodeSession(CFG, w, 2, max_seq_len=96, mx=form, prefill=True)
    graph, nodes = exposed(build_prefill_graph(CFG, 2, 90, fused=True, mx=form))
    s.engine.set_kv_cache_length(0)
    out = s.engine.run(graph, {**s.inputs, "input_ids": prompt})
    assert check_codes(nodes, {**s.inputs, **out}) == 9 * CFG.layers
