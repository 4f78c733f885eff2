"""Checks a run of a decoder graph on an 8-bit KV cache node by node: what each layer's nodes leave in
the cache, and the attention over it, against the oracle on the tensors that they read."""
import torch

from kv_fp8_oracle import Cache, check_attention


def cache_of(engine, name):
    e = engine.kv_cache_entry(name)
    return Cache(*(e[n].cpu().numpy() for n in ("key_pool", "value_pool", "scales", "block_table")))


def f64(t):
    return t.detach().cpu().double().numpy()


def rotated(x, cos, sin, positions):
    """Interleaved RoPE of x [B, H, S, D] in 32 bits at positions[b] + s, rounded to x's type."""
    out = x.float().clone()
    for b, p in enumerate(positions):
        for s in range(x.shape[2]):
            c, n = cos[p + s], sin[p + s]
            e, o = x[b, :, s, 0::2].float(), x[b, :, s, 1::2].float()
            out[b, :, s, 0::2], out[b, :, s, 1::2] = e * c - o * n, e * n + o * c
    return out.to(x.dtype)


def check_nodes(engine, nodes, tensors, past, before):
    """past: tokens that each sequence held; before: layer -> the cache before the run. Returns how
    many appends and attentions were checked."""
    count = {"append": 0, "attention": 0}
    tensors = {n: t.cpu() for n, t in tensors.items()}
    for n in nodes:
        if n["op"] not in ("rope_append", "attention", "paged_attention"):
            continue
        name, ins = n["attrs"]["kv_cache"], [tensors[i] for i in n["inputs"]]
        out, want, held = tensors[n["outputs"][0]], before[name], cache_of(engine, name)
        if n["op"] == "rope_append":
            a = n["attrs"]
            x = ins[0].view(len(past), -1, a["q_heads"] + 2 * a["kv_heads"], a["head_dim"]).transpose(1, 2)
            q, k, v = x.split([a["q_heads"], a["kv_heads"], a["kv_heads"]], 1)
            assert torch.equal(out, rotated(q, ins[1], ins[2], past)), n["name"]
            want.append(f64(rotated(k, ins[1], ins[2], past)), f64(v), past)
            count["append"] += 1
        elif n["op"] == "attention":
            want.append(f64(ins[1]), f64(ins[2]), past)
            count["append"] += 1
        for pool in ("key", "value", "scales"):
            assert (getattr(held, pool) == getattr(want, pool)).all(), (n["name"], pool)
        if n["op"] != "rope_append":
            q = ins[0]
            if n["attrs"].get("output_layout") == "bshd":
                out = out.transpose(1, 2)
            check_attention(out, held.attention(f64(q), past, True, q.shape[3] ** -0.5), q.dtype,
                            max(past) + q.shape[2], q.shape[3])
            count["attention"] += 1
    return count
