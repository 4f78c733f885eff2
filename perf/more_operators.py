"""The operators of the 8-bit paged KV cache as cases that can be timed and checked.

A cache page holds, per KV head, `block` tokens: keys [block, head_dim] and values [head_dim, block]
as e4m3 elements, and for every token two scales, powers of two: one of its key, one of its value. A
row's scale is the least power of two that brings its largest magnitude to at most 448. The kinds:

  append     kv_append_fp8: new keys and values quantised into the pages
  rope       rope_append_fp8: the same from the joined q|k|v projection, with the rotary embedding of
             q and k in front
  read       kv_read_fp8: tokens of the cache back as 16- or 32-bit keys and values
  attention  paged_attention_fp8: attention of one new token per sequence (decode), or of a chunk of
             them, over the pages

With `own` false every pass runs in elementary torch operations in 32 bits, rounded once at the end;
with `own` true it is one call of the device layer. `exact` is written apart, in 64 bits.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}
LARGEST = 448.0  # of e4m3
# (query heads, KV heads, head_dim): the 0.5B and the 7B shape
HEADS = {"0.5b": (14, 2, 64), "7b": (28, 4, 128)}
THETA = 1_000_000.0


def listed():
    return [
        # the new token of a full decode batch of the larger decoder
        {"name": "append_b64_s1", "kind": "append", "dtype": "bfloat16", "heads": "7b", "batch": 64,
         "seq": 1, "past": 400, "block": 64},
        # four prompts of 2048 tokens of it, each behind what its sequence holds
        {"name": "append_b4_s2048", "kind": "append", "dtype": "bfloat16", "heads": "7b", "batch": 4,
         "seq": 2048, "past": 200, "block": 64},
        # the headline batch's new token, from the projection
        {"name": "rope_b32_s1", "kind": "rope", "dtype": "bfloat16", "heads": "0.5b", "batch": 32,
         "seq": 1, "past": 1000, "block": 64},
        # prompts in chunks of 1000 tokens in float16, small pages
        {"name": "rope_b2_s1000_f16", "kind": "rope", "dtype": "float16", "heads": "7b", "batch": 2,
         "seq": 1000, "past": 333, "block": 16},
        # a short conversation's cache moved elsewhere
        {"name": "read_b1_s300", "kind": "read", "dtype": "bfloat16", "heads": "0.5b", "batch": 1,
         "seq": 300, "past": 300, "block": 64},
        # eight long sequences read back
        {"name": "read_b8_s8192", "kind": "read", "dtype": "bfloat16", "heads": "7b", "batch": 8,
         "seq": 8192, "past": 8192, "block": 64},
        # one user's reply: latency
        {"name": "decode_b1_ctx1000", "kind": "attention", "dtype": "bfloat16", "heads": "0.5b",
         "batch": 1, "seq": 1, "past": 1000, "block": 64, "causal": True},
        # the headline step
        {"name": "decode_b32_ctx4096", "kind": "attention", "dtype": "bfloat16", "heads": "0.5b",
         "batch": 32, "seq": 1, "past": 4095, "block": 64, "causal": True},
        # the larger decoder's long contexts
        {"name": "decode_b64_ctx8192", "kind": "attention", "dtype": "bfloat16", "heads": "7b",
         "batch": 64, "seq": 1, "past": 8191, "block": 64, "causal": True},
        # a conversation's next turn
        {"name": "chunk_b2_s300_ctx3000", "kind": "attention", "dtype": "bfloat16", "heads": "7b",
         "batch": 2, "seq": 300, "past": 3000, "block": 64, "causal": True},
        # a long prompt fed in chunks
        {"name": "chunk_b1_s2048_ctx8192", "kind": "attention", "dtype": "bfloat16", "heads": "7b",
         "batch": 1, "seq": 2048, "past": 8192, "block": 64, "causal": True},
        # a few drafted tokens checked at once, float16, small pages
        {"name": "chunk_b3_s17_f16", "kind": "attention", "dtype": "float16", "heads": "0.5b",
         "batch": 3, "seq": 17, "past": 1500, "block": 16, "causal": True},
    ]


def _log_int(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    high = max(low, high)
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "rope", "read", "attention", "attention", "attention"])
    case = {"kind": kind, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
            "heads": rng.choice(list(HEADS)), "block": rng.choice([16, 32, 64, 64, 128])}
    if kind == "attention":
        case["causal"] = rng.random() < 0.8
        if rng.random() < 0.5:
            batch = _log_int(rng, 1, 64)
            return {**case, "batch": batch, "seq": 1, "past": _log_int(rng, 1, 8191)}
        batch, seq = _log_int(rng, 1, 4), _log_int(rng, 2, 1000)
        return {**case, "batch": batch, "seq": seq,
                "past": rng.choice([0, _log_int(rng, 1, 8192 // batch)])}
    batch = _log_int(rng, 1, 64)
    seq = rng.choice([1, _log_int(rng, 1, 8192 // batch)])
    return {**case, "batch": batch, "seq": seq,
            "past": seq if kind == "read" else rng.randrange(500)}


# ---- inputs, from the seed alone ---------------------------------------------------------------


def _pasts(case):
    """Tokens that each sequence holds before the call; they differ between sequences. read: the
    first token that is read."""
    if case["kind"] == "read":
        return [0] * case["batch"]
    past = case["past"]
    return [past - (37 * b) % (1 + past // 8) for b in range(case["batch"])]


def _pages(case):
    """Pages per sequence."""
    return -(-(case["past"] + (0 if case["kind"] == "read" else case["seq"])) // case["block"])


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _inputs(case, seed):
    """Queries and keys N(0, 1), a few key channels larger, values whose size varies by token. What
    the pages hold beside the sequences' tokens is what an earlier user of them left."""
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 41)
    hq, hkv, d = HEADS[case["heads"]]
    batch, seq, block, pages = case["batch"], case["seq"], case["block"], _pages(case)
    dtype = DTYPES[case["dtype"]]
    count = batch * pages + 3  # some are no sequence's
    key_codes = torch.empty((count, hkv, block, d), dtype=torch.uint8, device="cuda")
    value_codes = torch.empty((count, hkv, d, block), dtype=torch.uint8, device="cuda")
    scales = torch.empty((count, hkv, 2, block), dtype=torch.uint8, device="cuda")
    if case["kind"] in ("read", "attention"):
        step = max(1, (1 << 25) // (hkv * block * d))
        for i in range(0, count, step):
            n = min(step, count - i)
            k = _normal(g, (n, hkv, block, d))
            k[..., ::31] *= 4
            v = _normal(g, (n, hkv, block, d)) * torch.exp(_normal(g, (n, hkv, block, 1), 0.7))
            codes, scales[i:i + n, :, 0] = _quantize(k)
            key_codes[i:i + n] = codes
            codes, scales[i:i + n, :, 1] = _quantize(v)
            value_codes[i:i + n] = codes.transpose(2, 3)
    else:
        for pool in (key_codes, value_codes):
            pool.random_(0, 0x78, generator=g)
        scales.random_(110, 130, generator=g)
    state = {"key_codes": key_codes, "value_codes": value_codes, "scales": scales,
             "table": torch.randperm(count, generator=g, device="cuda")[:batch * pages]
             .to(torch.int32).view(batch, pages),
             "positions": torch.tensor(_pasts(case), device="cuda")}
    if case["kind"] == "attention":
        state["q"] = _normal(g, (batch, hq, seq, d)).to(dtype)
    elif case["kind"] == "append":
        k = _normal(g, (batch, hkv, seq, d))
        k[..., ::31] *= 4
        state["k"], state["v"] = k.to(dtype), _normal(g, (batch, hkv, seq, d), 0.5).to(dtype)
    elif case["kind"] == "rope":
        state["qkv"] = _normal(g, (batch, seq, (hq + 2 * hkv) * d)).to(dtype)
        angles = torch.arange(pages * block, dtype=torch.float64).unsqueeze(1) * THETA ** (
            -torch.arange(0, d, 2, dtype=torch.float64) / d)
        state["cos"], state["sin"] = angles.cos().float().cuda(), angles.sin().float().cuda()
    return state


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own and case["kind"] == "attention":
        hq, hkv, d = HEADS[case["heads"]]
        state["workspace"] = torch.empty(
            _hip().call("dli_hip_paged_attention_fp8_workspace", case["batch"], hq, hkv,
                        case["seq"], d, case["block"], _pages(case)),
            dtype=torch.uint8, device="cuda")
    return state


# ---- one pass ----------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


@functools.lru_cache(maxsize=None)
def _hip():
    path = os.path.join(os.getcwd(), "dl-inference_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from dli import hip

    return hip


def _own(state):
    hip, case = _hip(), state["case"]
    hq, hkv, d = HEADS[case["heads"]]
    batch, seq, dtype = case["batch"], case["seq"], DTYPES[case["dtype"]]
    code = hip._TORCH_CODES[dtype]
    pools = [state[n].data_ptr() for n in ("key_codes", "value_codes", "scales")]
    table = [state["table"].data_ptr(), state["scales"].shape[0]]
    place = [case["block"], state["table"].shape[1], 0, state["positions"].data_ptr(), hip.I64]
    stream = hip.current_stream()
    if case["kind"] == "append":
        hip.call("dli_hip_kv_append_fp8", code, state["k"].data_ptr(), state["v"].data_ptr(), *pools,
                 *table, batch, hkv, seq, d, *place, stream)
        return _pools(state)
    if case["kind"] == "rope":
        q = torch.empty((batch, hq, seq, d), dtype=dtype, device="cuda")
        hip.call("dli_hip_rope_append_fp8", code, state["qkv"].data_ptr(), state["cos"].data_ptr(),
                 state["sin"].data_ptr(), *state["cos"].shape, q.data_ptr(), *pools, *table, batch,
                 seq, hq, hkv, d, *place, stream)
        return {"q": q, **_pools(state)}
    if case["kind"] == "read":
        k = torch.empty((batch, hkv, seq, d), dtype=dtype, device="cuda")
        v = torch.empty_like(k)
        hip.call("dli_hip_kv_read_fp8", code, *pools, *table, k.data_ptr(), v.data_ptr(), batch, hkv,
                 seq, d, *place, stream)
        return k, v
    out = torch.empty_like(state["q"])
    workspace = state["workspace"]
    hip.call("dli_hip_paged_attention_fp8", code, state["q"].data_ptr(), *pools, *table,
             out.data_ptr(), batch, hq, hkv, seq, d, *place, int(case["causal"]), d ** -0.5, 0,
             workspace.data_ptr(), workspace.numel(), stream)
    return out


def _pools(state):
    """The pools as the values that they hold."""
    return {"key_codes": state["key_codes"].view(torch.float8_e4m3fn),
            "value_codes": state["value_codes"].view(torch.float8_e4m3fn),
            "scales": state["scales"].view(torch.float8_e8m0fnu)}


# ---- the plain form ----------------------------------------------------------------------------


def _quantize(x):
    """Codes and scale codes, uint8, of the rows of x in 32 bits."""
    amax = x.abs().amax(-1)
    bits = amax.view(torch.int32)
    code = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp_min(0)
    inverse = ((254 - code) << 23).view(torch.float32)
    codes = (x * inverse.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, code.to(torch.uint8)


def _write(state, k, v):
    """k, v [B, H, S, D] in 32 bits into the pages."""
    batch, _, seq, _ = k.shape
    block = state["case"]["block"]
    at = state["positions"].unsqueeze(1) + torch.arange(seq, device="cuda")  # [B, S]
    page = state["table"].gather(1, at // block).long().flatten()
    slot = (at % block).flatten()
    for row, x, pool in ((0, k, state["key_codes"]), (1, v, state["value_codes"].transpose(2, 3))):
        codes, scale = _quantize(x.transpose(1, 2).flatten(0, 1))  # [B S, H, D], [B S, H]
        pool[page, :, slot] = codes
        state["scales"][page, :, row, slot] = scale


def _held(state, tokens):
    """Keys and values of each sequence's first `tokens` tokens in 32 bits, [B, H, tokens, D]."""
    table = state["table"].long()
    both = []
    for row, pool in ((0, state["key_codes"]), (1, state["value_codes"].transpose(2, 3))):
        codes = pool[table].transpose(1, 2).flatten(2, 3)[:, :, :tokens]
        code = state["scales"][:, :, row][table].transpose(1, 2).flatten(2)[..., :tokens].int()
        scale = torch.where(code == 0, 0x400000, code << 23).view(torch.float32)
        both.append(codes.view(torch.float8_e4m3fn).float() * scale.unsqueeze(-1))
    return both


def _plain(state):
    case = state["case"]
    hq, hkv, d = HEADS[case["heads"]]
    batch, seq, dtype = case["batch"], case["seq"], DTYPES[case["dtype"]]
    if case["kind"] == "append":
        _write(state, state["k"].float(), state["v"].float())
        return _pools(state)
    if case["kind"] == "rope":
        x = state["qkv"].float().view(batch, seq, hq + 2 * hkv, d).transpose(1, 2)
        at = state["positions"].unsqueeze(1) + torch.arange(seq, device="cuda")
        cos, sin = state["cos"][at].unsqueeze(1), state["sin"][at].unsqueeze(1)
        a, b = x[:, :hq + hkv, :, 0::2], x[:, :hq + hkv, :, 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(3).to(dtype)
        _write(state, turned[:, hq:].float(), x[:, hq + hkv:])
        return {"q": turned[:, :hq].contiguous(), **_pools(state)}
    if case["kind"] == "read":
        return tuple(x.to(dtype).contiguous() for x in _held(state, seq))
    longest = max(_pasts(case)) + seq
    k, v = _held(state, longest)
    # a group's query heads share a KV head: rows [group * seq] of each (sequence, KV head)
    q = state["q"].float().reshape(batch * hkv, hq // hkv * seq, d)
    s = torch.bmm(q, k.flatten(0, 1).transpose(1, 2).contiguous()) * d ** -0.5
    s = s.view(batch, hq, seq, longest)
    last = state["positions"].view(-1, 1, 1) + (
        torch.arange(seq, device="cuda").view(1, -1, 1) if case["causal"] else seq - 1)
    seen = (torch.arange(longest, device="cuda") <= last).unsqueeze(1)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(batch * hkv, -1, longest), v.flatten(0, 1)).view(batch, hq, seq, d)
    return (out / total).to(dtype)


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    batch, seq, size = case["batch"], case["seq"], SIZES[case["dtype"]]
    tokens = batch * seq
    held = hkv * (2 * d + 2)  # bytes of one token in the pages
    if case["kind"] == "attention":
        pasts = _pasts(case)
        pairs = sum(seq * p + (seq * (seq + 1) // 2 if case["causal"] else seq * seq) for p in pasts)
        return {"bytes": held * (sum(pasts) + tokens) + 2 * tokens * hq * d * size,
                "flops": 4 * d * hq * pairs}
    moved = tokens * (held + 2 * hkv * d * size)
    if case["kind"] != "rope":
        return {"bytes": moved, "flops": 4 * tokens * hkv * d}
    return {"bytes": moved + 2 * tokens * hq * d * size + 4 * d * tokens,
            "flops": tokens * d * (3 * hq + 7 * hkv)}


# ---- the same in 64 bits -----------------------------------------------------------------------


def _values64(codes):
    """What e4m3 codes stand for: sign, 4 exponent bits (bias 7), 3 of mantissa."""
    c = torch.arange(256, device="cuda")
    e, m = (c >> 3) & 15, (c & 7).double() / 8
    value = torch.where(e > 0, 1 + m, m) * torch.exp2((e.clamp_min(1) - 7).double())
    return (value * (1 - 2 * (c >> 7)).double())[codes.int()]


def _rounded64(x):
    """Nearest elements of the rows of x in 64 bits, and the rows' scales."""
    top = x.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(top).exponent - 9  # top = f 2^(exponent + 9), f in [1/2, 1)
    exponent = torch.where(torch.ldexp(top, -exponent) > LARGEST, exponent + 1, exponent)
    scale = torch.exp2(exponent.clamp_min(-127).double())
    y = x / scale
    gap = torch.exp2((torch.frexp(y.abs()).exponent - 1).clamp_min(-6).double() - 3)
    return torch.round(y / gap) * gap, scale.squeeze(-1)


def exact(case, seed):
    t = _inputs(case, seed)
    hq, hkv, d = HEADS[case["heads"]]
    batch, seq, block = case["batch"], case["seq"], case["block"]
    pasts, dtype = _pasts(case), DTYPES[case["dtype"]]
    if case["kind"] in ("append", "rope"):
        out = {"key_codes": _values64(t["key_codes"]), "value_codes": _values64(t["value_codes"]),
               "scales": torch.exp2(t["scales"].double() - 127)}
        if case["kind"] == "append":
            k, v = t["k"].double(), t["v"].double()
        else:
            x = t["qkv"].double().view(batch, seq, -1, d)
            z = torch.view_as_complex(x[:, :, :hq + hkv].reshape(batch, seq, hq + hkv, d // 2, 2))
            turn = torch.complex(t["cos"].double(), t["sin"].double())
            turn = torch.stack([turn[p:p + seq] for p in pasts]).unsqueeze(2)
            turned = torch.view_as_real(z * turn).flatten(3).transpose(1, 2)
            out["q"] = turned[:, :hq].contiguous()
            # keys are kept in the type of the activations before they are quantised
            k = turned[:, hq:].to(dtype).double()
            v = x[:, :, hq + hkv:].transpose(1, 2)
        (k, k_scale), (v, v_scale) = _rounded64(k), _rounded64(v)
        for b, past in enumerate(pasts):
            at = torch.arange(past, past + seq, device="cuda")
            page, slot = t["table"][b].long()[at // block], at % block
            out["key_codes"][page, :, slot] = k[b].transpose(0, 1)
            out["value_codes"].transpose(2, 3)[page, :, slot] = v[b].transpose(0, 1)
            out["scales"][page, :, 0, slot] = k_scale[b].transpose(0, 1)
            out["scales"][page, :, 1, slot] = v_scale[b].transpose(0, 1)
        return {n: out[n] for n in (("q",) if "q" in out else ()) +
                ("key_codes", "value_codes", "scales")}
    result = []
    for b, past in enumerate(pasts):
        pages = t["table"][b].long()
        scale = torch.exp2(t["scales"][pages].double() - 127)  # [pages, H, 2, block]
        k = (_values64(t["key_codes"][pages]) * scale[:, :, 0].unsqueeze(-1)).transpose(0, 1)
        v = (_values64(t["value_codes"][pages]) * scale[:, :, 1].unsqueeze(2)).permute(1, 0, 3, 2)
        tokens = seq if case["kind"] == "read" else past + seq
        k, v = (x.reshape(hkv, -1, d)[:, :tokens] for x in (k, v))
        if case["kind"] == "read":
            result.append((k, v))
            continue
        q = t["q"][b].double().view(hkv, -1, seq, d)
        heads = []
        for h in range(hkv):
            s = torch.matmul(q[h].flatten(0, 1), k[h].t().contiguous()).view(-1, seq, tokens)
            s = s / math.sqrt(d)
            if case["causal"]:
                s += torch.full((seq, tokens), -math.inf, device="cuda",
                                dtype=torch.float64).triu(past + 1)
            heads.append(torch.matmul(torch.softmax(s, -1).flatten(0, 1), v[h]))
        result.append(torch.stack(heads).view(hq, seq, d))
    if case["kind"] == "read":
        return tuple(torch.stack(x) for x in zip(*result))
    return torch.stack(result)
