"""Checks a run of the microscaled decoder graphs code by code, beside mx_session's check of values:
what a node wrote against its own arithmetic, in 32 or 64 bits, on the tensors that it read."""
import numpy as np
import torch

import mx_oracle as mx
from mx_session import HALF_STEP, f64, raw

FEW = 1e-3  # of a node's codes may lie on the other side of a rounding border


def near(got, want, what):
    assert got.shape == want.shape, what
    assert (got != want).mean() <= FEW, (what, (got != want).mean())


def check_codes(nodes, tensors):
    """nodes: the graph's; tensors: its inputs, weights and outputs by name. Returns how many nodes
    were checked."""
    count = 0
    for n in nodes:
        op, attrs, name = n["op"], n["attrs"], n["name"]
        if op not in ("rms_norm_mx", "silu_mul_mx", "mx_linear"):
            continue
        count += 1
        ins, outs = [tensors[i] for i in n["inputs"]], [tensors[o] for o in n["outputs"]]
        if op == "mx_linear":
            x, w = mx.values(raw(ins[0]), raw(ins[1])), mx.values(raw(ins[2]), raw(ins[3]))
            want, terms = x @ w.T, np.abs(x) @ np.abs(w).T
            if name.endswith(("q_proj", "k_proj", "v_proj")):
                want, terms = want + f64(ins[4]), terms + np.abs(f64(ins[4]))
            if attrs.get("residual"):
                want, terms = want + f64(ins[-1]), terms + np.abs(f64(ins[-1]))
            # fp32 sums of k + 2 terms in any order, and the output's rounding; what the matrix unit
            # drops with e4m3 rows only where the result has 16 bits
            k = x.shape[-1]
            slack = (k + 2) * 2.0 ** -24 * terms
            fp8 = ins[0].shape[-1] == k
            if fp8 and outs[0].dtype != torch.float32 and outs[0].is_cuda:
                slack = slack + 2.0 ** -10 * terms
            slack = slack + HALF_STEP[outs[0].dtype] * (np.abs(want) + slack)
            assert (np.abs(f64(outs[0]) - want) <= slack).all(), name
            continue
        if op == "rms_norm_mx":
            y = mx.rms_norm32(ins[0].float().cpu().numpy(), ins[1].float().cpu().numpy(), attrs["eps"])
        else:
            g, u = np.split(f64(ins[0]), 2, -1)
            y = g / (1 + np.exp(-g)) * u
        codes, scales = mx.quantize(y, attrs["format"])
        near(raw(outs[1]), scales, name)
        same = np.repeat(raw(outs[1]) == scales, codes.shape[-1] // scales.shape[-1], -1)
        near(raw(outs[0])[same], codes[same], name)
    return count
