"""Checks a run of the microscaled decoder graphs node by node: each microscaled node's outputs
against float64 arithmetic on the tensors it read."""
import json

import numpy as np
import torch

import dli
import mx_oracle as mx

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def exposed(graph):
    """The graph with every tensor that a node writes or reads as an output."""
    g = json.loads(graph.to_json())
    g["outputs"] = list(dict.fromkeys(o for n in g["nodes"] for o in n["outputs"]))
    return dli.Graph.from_json(json.dumps(g)), g["nodes"]


def f64(t):
    return t.detach().cpu().double().numpy()


def raw(t):
    return t.detach().cpu().numpy()


def check_nodes(nodes, tensors):
    """nodes: the graph's; tensors: its inputs, weights and outputs by name. Returns how many nodes
    of each microscaled operator were checked."""
    count = {}
    for n in nodes:
        op, attrs = n["op"], n["attrs"]
        if op not in ("mx_quantize", "rms_norm_mx", "silu_mul_mx", "mx_linear"):
            continue
        count[op] = count.get(op, 0) + 1
        ins, outs = [tensors[i] for i in n["inputs"]], [tensors[o] for o in n["outputs"]]
        if op == "mx_linear":
            x, w = mx.values(raw(ins[0]), raw(ins[1])), mx.values(raw(ins[2]), raw(ins[3]))
            want = x @ w.T
            # the matrix instruction may drop what is below 2^-13 of the largest of 8 neighbouring
            # products: at most 2^-10 of a sum of magnitudes; and one rounding to the output's type
            slack = 2.0 ** -10 * (np.abs(x) @ np.abs(w).T)
            if n["name"].endswith(("q_proj", "k_proj", "v_proj")):
                want = want + f64(ins[4])
            if attrs.get("residual"):
                want = want + f64(ins[-1])
            slack = slack + HALF_STEP[outs[0].dtype] * (np.abs(want) + slack)
            assert (np.abs(f64(outs[0]) - want) <= slack).all(), n["name"]
            continue
        if op == "mx_quantize":
            codes, scales = mx.quantize(f64(ins[0]), attrs["format"])
            assert np.array_equal(raw(outs[0]), codes), n["name"]
            assert np.array_equal(raw(outs[1]), scales), n["name"]
            continue
        if op == "rms_norm_mx":
            h = f64(ins[0])
            y = h / np.sqrt((h ** 2).mean(-1, keepdims=True) + attrs["eps"]) * f64(ins[1])
        else:
            g, u = np.split(f64(ins[0]), 2, -1)
            y = g / (1 + np.exp(-g)) * u
        got = mx.values(raw(outs[0]), raw(outs[1]))
        # half a step of the elements at the block's top, saturation included (an eighth of the
        # largest value for e4m3, a quarter for e2m1), and a few fp32 roundings before it
        top = np.abs(y).reshape(-1, 32).max(1)[:, None]
        part = 0.25 if attrs["format"] == "fp4" else 0.125
        assert (np.abs(got - y).reshape(-1, 32) <= top * (part + 2.0 ** -20)).all(), n["name"]
    return count


def check_step(session, ids, positions):
    """One eager decode step of a session with every node checked; its outputs."""
    graph, nodes = exposed(session.graph)
    session.ids.copy_(ids)
    session.positions.copy_(positions)
    out = session.engine.run(graph, session.inputs)
    layers = session.cfg.layers
    assert check_nodes(nodes, {**session.inputs, **out}) == {
        "rms_norm_mx": 2 * layers, "mx_linear": 6 * layers, "mx_quantize": layers,
        "silu_mul_mx": layers}
    return out
