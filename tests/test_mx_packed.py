"""Sessions built from weights that pack_mx_weights made, stored and loaded."""
import pytest
import torch

import dli
from dli.weights import save_weights
from dli_qwen2 import DecodeSession, pack_mx_weights, random_weights, tiny_config

CFG = tiny_config(layers=2, ffn=1216)


def engine():
    return dli.Engine().load_aten_plugin()


def logits(weights, form="fp8", **more):
    s = DecodeSession(CFG, weights, 2, max_seq_len=16, fused=False, engine=engine(), device="cpu",
                      mx=form, **more)
    if more:
        return s.run_prefill(torch.tensor([[1, 2, 3], [4, 5, 6]]))[0]
    return s.step(torch.tensor([5, 900]), torch.zeros(2, dtype=torch.int64))[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_stored_model_runs(tmp_path, dtype):
    w = random_weights(CFG, seed=4, dtype=dtype)
    packed = pack_mx_weights(CFG, w, engine())
    loaded = dli.load_weights(str(save_weights(tmp_path, "packed", packed)))
    assert not any(n.endswith(("_proj.weight")) for n in loaded)
    for form in ("fp8", "fp4"):
        want = logits(w, form)
        assert torch.equal(logits(packed, form), want) and torch.equal(logits(loaded, form), want)
    assert torch.equal(logits(loaded, prefill=True), logits(w, prefill=True))
    again = pack_mx_weights(CFG, loaded, engine())
    assert again.keys() == packed.keys()
    assert all(again[n] is loaded[n] for n in loaded)


def test_layers_packed_and_not():
    w = random_weights(CFG, seed=4)
    packed = pack_mx_weights(CFG, w, engine())
    mixed = {n: t for n, t in w.items() if "layers.0" not in n}
    mixed.update({n: t for n, t in packed.items() if "layers.0" in n})
    assert torch.equal(logits(mixed), logits(w))
    both = {**w, **packed}  # the packed one counts
    assert pack_mx_weights(CFG, both, engine()).keys() == packed.keys()


def test_refusals():
    packed = pack_mx_weights(CFG, random_weights(CFG, seed=4), engine())
    name = "model.layers.1.mlp.gate_up_proj.weight"
    for change in ({f"{name}.scales": None}, {f"{name}.codes": packed[f"{name}.codes"].int()},
                   {f"{name}.codes": packed[f"{name}.codes"][1:]},
                   {f"{name}.scales": packed[f"{name}.scales"][:, 1:]}):
        bad = {n: t for n, t in {**packed, **change}.items() if t is not None}
        with pytest.raises(ValueError, match="gate_up_proj.weight"):
            pack_mx_weights(CFG, bad, engine())


@pytest.mark.gpu
def test_a_stored_model_runs_on_the_gpu(tmp_path):
    cfg = tiny_config(layers=1, ffn=1216)
    w = {n: t.cuda() for n, t in random_weights(cfg, seed=4).items()}
    gpu = dli.Engine().load_plugin()
    path = save_weights(tmp_path, "packed", {n: t.cpu() for n, t in pack_mx_weights(cfg, w, gpu).items()})
    loaded = {n: t.cuda() for n, t in dli.load_weights(str(path)).items()}
    ids, at = torch.tensor([5, 900], device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    got, want = (DecodeSession(cfg, v, 2, max_seq_len=16, mx="fp8").step(ids, at)[0]
                 for v in (loaded, w))
    assert torch.equal(got, want)
