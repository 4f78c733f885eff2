"""uint8 tensors hold codes and scales: operators that compute with numbers refuse them. No GPU."""
import pytest
import torch

import dli
from support import one_node_graph


def aten(op, inputs, attrs=None, outputs=("out",)):
    return dli.Engine().load_aten_plugin().run(one_node_graph(op, inputs, outputs, attrs), inputs)


def test_linear_refuses_a_uint8_output():
    inputs = {"x": torch.randn(2, 8), "w": torch.randn(3, 8)}
    for name in ("uint8", "u8"):
        with pytest.raises(ValueError, match="out_dtype uint8"):
            aten("linear", inputs, {"out_dtype": name})
    assert aten("linear", inputs, {"out_dtype": "bfloat16"})["out"].dtype == torch.bfloat16


@pytest.mark.parametrize("op,shapes,attrs,outputs", [
    ("add", [(4,), (4,)], {}, ("out",)), ("silu", [(4,)], {}, ("out",)),
    ("softmax", [(2, 4)], {}, ("out",)), ("rms_norm", [(2, 4), (4,)], {}, ("out",)),
    ("matmul", [(2, 4), (4, 2)], {}, ("out",)), ("linear", [(2, 4), (3, 4)], {}, ("out",)),
    ("argmax", [(2, 4)], {}, ("out",)), ("transpose", [(2, 4)], {"perm": [1, 0]}, ("out",)),
    ("attention", [(1, 1, 2, 4)] * 3, {}, ("out",)),
    ("attention", [(1, 1, 2, 4)] * 3, {"kv_cache": "layer_0"}, ("out",)),
    ("rotary_embedding", [(1, 1, 2, 4), (1, 1, 2, 4), (8, 2), (8, 2)], {}, ("q", "k"))])
def test_operators_refuse_uint8_tensors(op, shapes, attrs, outputs):
    inputs = {f"i{n}": torch.ones(s, dtype=torch.uint8) for n, s in enumerate(shapes)}
    with pytest.raises(ValueError, match="expects float32, bfloat16 or float16"):
        aten(op, inputs, attrs, outputs)
    # the first input a float, the others bytes
    if len(shapes) > 1:
        inputs["i0"] = inputs["i0"].float()
        with pytest.raises(ValueError):
            aten(op, inputs, attrs, outputs)


def test_ids_and_positions_refuse_uint8():
    ids = torch.ones(2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="int64 or int32"):
        aten("embedding", {"ids": ids, "table": torch.randn(4, 8)})


def test_caches_refuse_uint8():
    with pytest.raises(ValueError, match="floating"):
        dli.Engine().reserve_kv_cache("layer_0", "uint8", 1, 1, 8, -1)
