"""Decode sessions on microscaled linears on the GPU: node by node, captured, and against the same
session on host tensors."""
import json
from dataclasses import replace

import pytest
import torch

import dli
from dli_qwen2 import DecodeSession, build_prefill_graph, random_weights, tiny_config
from mx_session import check_nodes, check_step, exposed

pytestmark = pytest.mark.gpu


def on_gpu(w):
    return {k: v.cuda() for k, v in w.items()}


@pytest.mark.parametrize("form", ["fp8", "fp4"])
@pytest.mark.parametrize("batch", [1, 5, 33])
def test_decode_step_node_by_node(form, batch):
    cfg = tiny_config(ffn=1216)
    s = DecodeSession(cfg, on_gpu(random_weights(cfg, seed=1)), batch, max_seq_len=32, mx=form)
    ids = torch.arange(batch, device="cuda") * 7 + 3
    for t in range(2):
        out = check_step(s, ids, torch.full((batch,), t, device="cuda"))
        ids = out["next_ids"]


@pytest.mark.parametrize("form,seq", [("fp8", 70), ("fp4", 130)])
def test_prompt_node_by_node(form, seq):
    """More than 128 rows: the tile kernels; hidden above what the fused head holds: its plain form."""
    cfg = replace(tiny_config(ffn=1216), hidden=1280, tied_embeddings=False)
    w = on_gpu(random_weights(cfg, seed=2))
    prompt = torch.randint(0, cfg.vocab, (2, seq), generator=torch.Generator().manual_seed(3)).cuda()
    s = DecodeSession(cfg, w, 2, max_seq_len=seq + 8, mx=form, prefill=True)
    graph, nodes = exposed(build_prefill_graph(cfg, 2, seq, fused_head=False, fused=True, mx=form))
    s.engine.set_kv_cache_length(0)
    out = s.engine.run(graph, {**s.inputs, "input_ids": prompt})
    assert check_nodes(nodes, {**s.inputs, **out})["mx_linear"] == 12
    logits, ids = s.run_prefill(prompt)
    assert torch.equal(logits, out["logits"]) and torch.equal(ids, out["next_ids"])
    check_step(s, ids, torch.full((2,), seq, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("head_dim,hidden", [(64, 896), (128, 1280)])
def test_prompt_then_steps(dtype, head_dim, hidden):
    """Every type and head size that a prompt may have, then decode steps from its cache."""
    cfg = replace(tiny_config(ffn=1216), hidden=hidden, head_dim=head_dim, heads=8,
                  tied_embeddings=False)
    w = on_gpu(random_weights(cfg, seed=9, dtype=dtype))
    prompt = torch.randint(0, cfg.vocab, (2, 5), generator=torch.Generator().manual_seed(3)).cuda()
    s = DecodeSession(cfg, w, 2, max_seq_len=32, mx="fp8", prefill=True)
    logits, ids = s.run_prefill(prompt)
    assert torch.equal(logits.argmax(-1), ids)
    out = check_step(s, ids, torch.full((2,), 5, device="cuda"))
    assert out["layers_0_output"].dtype == dtype
    assert s.generate(prompt, 3).shape == (2, 3)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
def test_captured_steps_repeat_eager_ones(form):
    cfg = tiny_config(ffn=1216)
    w = on_gpu(random_weights(cfg, seed=5))
    prompt = torch.randint(0, cfg.vocab, (4, 3), generator=torch.Generator().manual_seed(6)).cuda()
    eager = DecodeSession(cfg, w, 4, max_seq_len=64, mx=form)
    want = [eager.step(prompt[:, t], torch.full((4,), t, device="cuda"))[0].clone()
            for t in range(3)]
    tokens = eager.generate(prompt, 6)
    graphed = DecodeSession(cfg, w, 4, max_seq_len=64, mx=form).capture()
    for t in range(3):
        got = graphed.step(prompt[:, t], torch.full((4,), t, device="cuda"))[0]
        torch.cuda.synchronize()
        assert torch.equal(got, want[t])
    assert torch.equal(graphed.generate(prompt, 6), tokens)
    assert torch.equal(eager.generate(prompt, 6), tokens)


@pytest.mark.parametrize("form", ["fp8", "fp4"])
def test_against_host_tensors(form):
    cfg = tiny_config(ffn=1216)
    w = random_weights(cfg, seed=7, dtype=torch.float32)
    host = DecodeSession(cfg, w, 3, max_seq_len=32, fused=False, device="cpu", mx=form,
                         engine=dli.Engine().load_aten_plugin())
    gpu = DecodeSession(cfg, on_gpu(w), 3, max_seq_len=32, fused=False, mx=form)
    ids = torch.tensor([1, 500, 1000])
    for t in range(3):
        a, _ = host.step(ids + t, torch.full((3,), t))
        b, _ = gpu.step((ids + t).cuda(), torch.full((3,), t, device="cuda"))
        # fp32 sums in another order: now and then an element falls on its neighbour, which moves
        # a row of 896 by 2^-4 / sqrt(896) = 0.2 % (e2m1: 0.8 %) of its length
        assert torch.norm(a - b.cpu()) <= 2.0 ** (-6 if form == "fp8" else -4) * torch.norm(a)


def test_graph_as_text_runs_alone():
    """The decode graph and the weights a session packs, run through an engine of their own."""
    cfg = tiny_config(layers=1, ffn=1216)
    s = DecodeSession(cfg, on_gpu(random_weights(cfg, seed=8)), 2, max_seq_len=16, mx="fp8")
    want = s.step(torch.tensor([1, 2], device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"))
    engine = dli.Engine().load_plugin()
    engine.configure_kv_cache(block_size=64, max_seq_len=16)
    graph = dli.Graph.from_json(json.dumps(json.loads(s.graph.to_json())))
    out = engine.run(graph, s.inputs)
    assert torch.equal(out["logits"], want[0]) and torch.equal(out["next_ids"], want[1])
