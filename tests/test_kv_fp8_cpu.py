"""What the 8-bit KV cache's entry points refuse, and their workspace's size. No GPU: a refused call
launches nothing, and pointers are never read on the host."""
import ctypes

import pytest

from dli import hip

P = 1 << 20  # a pointer that nothing reads
POOLS = dict(key_codes=P, value_codes=P, scales=P, table=P, num_blocks=8)
WHERE = dict(block=64, max_blocks=4, start=0, positions=None, pdtype=hip.I64)


def status(entry, **change):
    a = dict(dtype=hip.BF16, a=P, b=P, batch=2, heads=2, seq=3, dim=64, q_heads=4, max_pos=9, pairs=32,
             out=P, **POOLS, **WHERE)
    a.update(change)
    lib = hip.load()
    pools = (a["key_codes"], a["value_codes"], a["scales"], a["table"], a["num_blocks"])
    where = (a["block"], a["max_blocks"], a["start"], a["positions"], a["pdtype"])
    if entry == "append":
        return lib.dli_hip_kv_append_fp8(a["dtype"], a["a"], a["b"], *pools, a["batch"], a["heads"],
                                         a["seq"], a["dim"], *where, None)
    if entry == "rope":
        return lib.dli_hip_rope_append_fp8(a["dtype"], a["a"], a["b"], a["b"], a["max_pos"], a["pairs"],
                                           a["out"], *pools, a["batch"], a["seq"], a["q_heads"],
                                           a["heads"], a["dim"], *where, None)
    if entry == "read":
        return lib.dli_hip_kv_read_fp8(a["dtype"], *pools, a["a"], a["b"], a["batch"], a["heads"],
                                       a["seq"], a["dim"], *where, None)
    return lib.dli_hip_paged_attention_fp8(a["dtype"], a["a"], *pools, a["out"], a["batch"], a["q_heads"],
                                           a["heads"], a["seq"], a["dim"], *where, 1, 0.125, 0, None, 0,
                                           None)


ENTRIES = ["append", "rope", "read", "attention"]


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("change", [
    dict(dtype=hip.I64), dict(dtype=hip.U8), dict(dtype=77), dict(batch=-1), dict(seq=-1), dict(heads=0),
    dict(dim=0), dict(dim=257), dict(block=0), dict(block=-64), dict(max_blocks=0), dict(num_blocks=0),
    dict(num_blocks=-1), dict(positions=P, pdtype=hip.F32), dict(key_codes=None), dict(value_codes=None),
    dict(scales=None), dict(table=None), dict(a=None), dict(block=1 << 29, max_blocks=2),
    dict(block=1 << 40, max_blocks=1 << 40), dict(batch=1 << 40), dict(seq=1 << 40), dict(heads=1 << 40),
    dict(batch=1 << 21, seq=1 << 20)])
def test_refusals(entry, change):
    assert status(entry, **change) == -1
    name = {"attention": "paged_attention", "rope": "rope_append"}.get(entry, f"kv_{entry}")
    assert hip.load().dli_hip_last_error().decode().startswith(f"{name}_fp8: ")


@pytest.mark.parametrize("entry,change", [
    ("append", dict(b=None)), ("read", dict(b=None)), ("rope", dict(b=None)), ("rope", dict(out=None)),
    ("rope", dict(pairs=33)), ("rope", dict(pairs=0)), ("rope", dict(max_pos=-1)), ("rope", dict(q_heads=0)),
    ("attention", dict(out=None)), ("attention", dict(q_heads=3)), ("attention", dict(q_heads=0)),
    ("attention", dict(batch=1 << 20, seq=1 << 20))])
def test_refusals_of_one(entry, change):
    assert status(entry, **change) == -1


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("change", [dict(batch=0), dict(seq=0)])
def test_nothing_to_do(entry, change):
    """Zero-sized work is a successful no-op, also with null pointers."""
    assert status(entry, **change, key_codes=None, a=None, b=None, out=None) == 0


def size(*args):
    return hip.load().dli_hip_paged_attention_fp8_workspace(*args)


def test_workspace():
    """Parts of a whole number of splits; none for forms that do not split, none of refused sizes."""
    for batch, q_heads, heads, seq, dim in ((1, 14, 2, 1, 64), (32, 14, 2, 1, 64), (2, 28, 4, 300, 128)):
        n = size(batch, q_heads, heads, seq, dim, 64, 64)
        assert n > 0 and n % (batch * q_heads * seq * (dim + 2) * 4) == 0
    assert size(1, 14, 2, 1, 64, 64, 1) == 0        # one page
    assert size(512, 14, 2, 1, 64, 64, 64) == 0     # more pairs than CUs
    assert size(1, 14, 2, 1, 80, 64, 64) == 0 and size(1, 14, 2, 1, 64, 24, 64) == 0  # row by row
    assert size(1, 14, 2, 1, 64, 1 << 25, 8) == 0   # row by row too: a page past 32-bit offsets
    for bad in ((0, 14, 2, 1, 64, 64, 64), (1, 13, 2, 1, 64, 64, 64), (1, 14, 0, 1, 64, 64, 64),
                (1, 14, 2, 0, 64, 64, 64), (1, 14, 2, 1, 64, 0, 64), (1, 14, 2, 1, 64, 64, -1),
                (1, 14, 2, 1, 64, 1 << 40, 1 << 40), (1 << 40, 14, 2, 1, 64, 64, 64),
                (1, 14, 2, 1 << 40, 64, 64, 64)):
        assert size(*bad) == 0


def test_declared():
    for name in ("kv_append", "rope_append", "kv_read", "paged_attention"):
        assert f"dli_hip_{name}_fp8" in hip.declared_symbols()
    image, n = ctypes.c_void_p(), ctypes.c_size_t()
    for module in (b"kv_fp8", b"kv_fp8_attention"):
        assert hip.load().dli_hip_code_object(module, ctypes.byref(image), ctypes.byref(n)) == 0 and n.value
