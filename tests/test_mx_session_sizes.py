"""Microscaled sessions at sizes that the one-node head does not take: more than 64 sequences, hidden
a multiple of 32 but not of 64."""
import json
from dataclasses import replace

import pytest
import torch

from dli_qwen2 import DecodeSession, build_decode_graph, random_weights, tiny_config
from mx_session import check_step


def sized(hidden):
    return replace(tiny_config(layers=1, ffn=608), hidden=hidden, heads=4, kv_heads=2)


def head(cfg, batch, **more):
    return [n["op"] for n in json.loads(build_decode_graph(cfg, batch, mx="fp8", **more).to_json())["nodes"]][-3:]


def test_the_head_of_each_size():
    plain = ["rms_norm", "linear", "argmax"]
    for hidden, batch, more in ((256, 65, {}), (256, 1000, {}), (96, 3, {}), (1056, 3, {}),
                                (256, 3, {"dtype": "float16"}), (256, 3, {"fused": False})):
        assert head(sized(hidden), batch, **more) == plain
    for hidden, batch in ((256, 64), (1024, 1), (64, 3)):
        assert head(sized(hidden), batch)[-1] == "lm_head_argmax"


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,batch", [(256, 65), (256, 130), (96, 3), (160, 70)])
def test_steps_and_prompts_of_each_size(hidden, batch):
    cfg = sized(hidden)
    w = {n: t.cuda() for n, t in random_weights(cfg, seed=3).items()}
    s = DecodeSession(cfg, w, batch, max_seq_len=32, mx="fp8", prefill=True)
    prompt = torch.randint(0, cfg.vocab, (batch, 5), generator=torch.Generator().manual_seed(3)).cuda()
    logits, ids = s.run_prefill(prompt)
    assert torch.equal(logits.argmax(-1), ids)
    out = check_step(s, ids, torch.full((batch,), 5, device="cuda"))
    assert torch.equal(out["logits"].argmax(-1), out["next_ids"])
    assert s.generate(prompt, 3).shape == (batch, 3)
