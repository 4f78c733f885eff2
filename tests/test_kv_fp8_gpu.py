"""The 8-bit paged KV cache's entry points (include/dli_hip.h, section 5) against the float64 oracle:
codes and read-back values exactly, attention within bounds from its roundings."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dli import hip
from kv_fp8_oracle import Cache, check_attention

pytestmark = pytest.mark.gpu
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def rng(seed):
    return torch.Generator().manual_seed(seed)


class Pools:
    """Device pools of random content with a shuffled block table; some pages are no sequence's."""

    def __init__(self, batch, heads, dim, block, max_blocks, seed=0, spare=2, missing=()):
        g = rng(seed)
        self.count = batch * max_blocks + spare
        n = self.count
        finite = torch.tensor([c for c in range(256) if c % 128 != 127], dtype=torch.uint8)

        def codes(*shape):
            return finite[torch.randint(0, len(finite), shape, generator=g)]

        self.key, self.value = codes(n, heads, block, dim), codes(n, heads, dim, block)
        self.scales = torch.randint(110, 121, (n, heads, 2, block), generator=g).to(torch.uint8)
        self.table = torch.randperm(n, generator=g)[:batch * max_blocks].to(torch.int32).view(batch, -1)
        for b, i, page in missing:
            self.table[b, i] = page
        self.block, self.max_blocks, self.heads, self.dim, self.batch = block, max_blocks, heads, dim, batch

    def cuda(self):
        self.key, self.value, self.scales, self.table = (
            t.cuda() for t in (self.key, self.value, self.scales, self.table))
        return self

    def oracle(self):
        return Cache(*(t.cpu().numpy() for t in (self.key, self.value, self.scales, self.table)))

    def pointers(self):
        return (self.key.data_ptr(), self.value.data_ptr(), self.scales.data_ptr(),
                self.table.data_ptr(), self.count)

    def check(self, cache):
        torch.cuda.synchronize()
        assert np.array_equal(self.key.cpu().numpy(), cache.key)
        assert np.array_equal(self.value.cpu().numpy(), cache.value)
        assert np.array_equal(self.scales.cpu().numpy(), cache.scales)


def where(first, index=torch.int64):
    """(start, positions, positions_dtype, what has to stay alive) of a call: a list or a tensor makes
    positions, a number start."""
    if isinstance(first, int):
        return first, None, hip.I64, None
    t = first if isinstance(first, torch.Tensor) else torch.tensor(first, dtype=index, device="cuda")
    return 0, t.data_ptr(), hip.dtype_code(t), t


def append(pools, k, v, first, index=torch.int64, stream=None):
    B, H, S, D = k.shape
    start, ptr, code, keep = where(first, index)
    hip.call("dli_hip_kv_append_fp8", hip.dtype_code(k), k.data_ptr(), v.data_ptr(), *pools.pointers(),
             B, H, S, D, pools.block, pools.max_blocks, start, ptr, code,
             hip.current_stream() if stream is None else stream)


def rope(pools, qkv, cos, sin, q_heads, first, index=torch.int64):
    B, S, _ = qkv.shape
    start, ptr, code, keep = where(first, index)
    q = torch.full((B, q_heads, S, pools.dim), 7.0, dtype=qkv.dtype, device="cuda")
    hip.call("dli_hip_rope_append_fp8", hip.dtype_code(qkv), qkv.data_ptr(), cos.data_ptr(),
             sin.data_ptr(), *cos.shape, q.data_ptr(), *pools.pointers(), B, S, q_heads, pools.heads,
             pools.dim, pools.block, pools.max_blocks, start, ptr, code, hip.current_stream())
    return q


def read(pools, seq, first, dtype, index=torch.int64):
    start, ptr, code, keep = where(first, index)
    k = torch.full((pools.batch, pools.heads, seq, pools.dim), 7.0, dtype=dtype, device="cuda")
    v = k.clone()
    hip.call("dli_hip_kv_read_fp8", hip.dtype_code(k), *pools.pointers(), k.data_ptr(), v.data_ptr(),
             pools.batch, pools.heads, seq, pools.dim, pools.block, pools.max_blocks, start, ptr, code,
             hip.current_stream())
    torch.cuda.synchronize()
    return k, v


def workspace(pools, q):
    B, Hq, S, D = q.shape
    n = hip.call("dli_hip_paged_attention_fp8_workspace", B, Hq, pools.heads, S, D, pools.block,
                 pools.max_blocks)
    return torch.full((n,), 255, dtype=torch.uint8, device="cuda")  # of any content: NaN


def attend(pools, q, first, causal=True, scale=None, bshd=False, ws=None, index=torch.int64, out=None):
    B, Hq, S, D = q.shape
    start, ptr, code, keep = where(first, index)
    if out is None:
        out = torch.full((B, S, Hq, D) if bshd else q.shape, 7.0, dtype=q.dtype, device="cuda")
    hip.call("dli_hip_paged_attention_fp8", hip.dtype_code(q), q.data_ptr(), *pools.pointers(),
             out.data_ptr(), B, Hq, pools.heads, S, D, pools.block, pools.max_blocks, start, ptr, code,
             int(causal), D ** -0.5 if scale is None else scale, int(bshd),
             None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
             hip.current_stream())
    return out


def values(shape, dtype, seed, spread=1.0):
    """Rows of differing size; among them a row of zeros, ones with an infinity and a NaN, the
    largest magnitude at 1.75 times a power of two and just above, subnormals and the largest numbers."""
    g = rng(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn((*shape[:-1], 1), generator=g))
    x = x.to(dtype)
    rows = x.view(-1, shape[-1])
    special = [lambda r: r.zero_(), lambda r: r[0:1].fill_(math.inf), lambda r: r[-1:].fill_(math.nan),
               lambda r: r.copy_(torch.linspace(-1.75, 1.75, len(r))),
               lambda r: r.copy_(torch.linspace(-1, 1, len(r)) * torch.finfo(dtype).max),
               lambda r: r.copy_(torch.linspace(-8, 8, len(r)) * torch.finfo(dtype).smallest_normal
                                 * torch.finfo(dtype).eps),
               lambda r: r.fill_(-0.0),
               lambda r: r.copy_(torch.full_like(r, 1.75) * (1 + torch.finfo(dtype).eps))]
    for i, f in enumerate(special):
        if (i + 1) * 3 < len(rows):
            f(rows[(i + 1) * 3])
    return x


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,dim,block", [(2, 64, 64), (4, 128, 64), (2, 128, 16), (3, 64, 32),
                                             (1, 64, 128), (2, 80, 16), (2, 64, 24), (1, 7, 5),
                                             (1, 256, 64)])
@pytest.mark.parametrize("seq,first", [(1, [0, 65]), (1, [127, -1]), (5, 14), (16, [9, 16]),
                                       (17, [3, 0]), (75, [-10, 70]), (140, [0, 33]), (64, 64)])
def test_append_and_read(dtype, heads, dim, block, seq, first):
    """Written as the oracle writes, everything else left; read back as codes and scales say."""
    t = DTYPES[dtype]
    blocks = -(-128 // block)
    pools = Pools(2, heads, dim, block, blocks, seed=seq, missing=[(1, blocks - 1, -1)]).cuda()
    cache = pools.oracle()
    k, v = values((2, heads, seq, dim), t, 1), values((2, heads, seq, dim), t, 2)
    starts = [first] * 2 if isinstance(first, int) else first
    cache.append(k.double().numpy(), v.double().numpy(), starts)
    append(pools, k.cuda(), v.cuda(), first, torch.int32 if seq % 2 else torch.int64)
    pools.check(cache)
    for got, want in zip(read(pools, seq, first, t), cache.read(starts, seq)):
        want = torch.from_numpy(want).float().to(t)
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=-3.0), torch.nan_to_num(want, nan=-3.0))
        assert torch.equal(got.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("table", [(0, -1), (1, 1 << 30), (1, 99)])
def test_a_missing_page_takes_nothing(table):
    """A page id outside the pool: tokens are dropped there, read as zeros, and passed over."""
    at, page = table
    pools = Pools(1, 2, 64, 64, 3, missing=[(0, at, page)]).cuda()
    cache = pools.oracle()
    k, v = values((1, 2, 150, 64), torch.bfloat16, 1), values((1, 2, 150, 64), torch.bfloat16, 2)
    k, v = k.nan_to_num(0, 1, 1).clamp(-9, 9), v.nan_to_num(0, 1, 1).clamp(-9, 9)
    cache.append(k.double().numpy(), v.double().numpy(), [10])
    append(pools, k.cuda(), v.cuda(), 10)
    pools.check(cache)
    got = read(pools, 192, 0, torch.float32)[0].cpu().double().numpy()
    assert np.array_equal(got, cache.read([0], 192)[0])
    for seq, heads in ((1, 2), (1, 14), (9, 4), (70, 2)):
        q = torch.randn((1, heads, seq, 64), generator=rng(seq)).bfloat16()
        out = attend(pools, q.cuda(), 160 - seq)
        check_attention(out, cache.attention(q.double().numpy(), [160 - seq], True, 0.125),
                        torch.bfloat16, 160, 64)


def tables(dim, length):
    angle = torch.arange(length).double()[:, None] * 10000.0 ** (-torch.arange(dim // 2).double() / 16)
    return angle.cos().float(), angle.sin().float()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q_heads,heads,dim,block,pairs", [(14, 2, 64, 64, 32), (4, 4, 128, 16, 64),
                                                           (3, 1, 64, 24, 32), (2, 1, 96, 16, 48),
                                                           (4, 2, 128, 64, 20)])
@pytest.mark.parametrize("seq,first", [(1, [0, 65]), (7, 14), (16, [-3, 90]), (50, [3, 77])])
def test_rope_append(dtype, q_heads, heads, dim, block, pairs, seq, first):
    """q and the keys are the rotation in 32 bits, products rounded by themselves, rounded to the type;
    positions beyond the tables (100 rows) unrotated."""
    t = DTYPES[dtype]
    pools = Pools(2, heads, dim, block, -(-128 // block), seed=seq).cuda()
    cache = pools.oracle()
    cos, sin = tables(2 * pairs, 100)
    qkv = torch.randn((2, seq, (q_heads + 2 * heads) * dim), generator=rng(seq)).to(t)
    starts = [first] * 2 if isinstance(first, int) else first
    x = qkv.float().view(2, seq, -1, dim).transpose(1, 2).clone()
    for b in range(2):
        for s in range(seq):
            pos = starts[b] + s
            if 0 <= pos < 100:
                row = x[b, :q_heads + heads, s, :2 * pairs]
                e, o, c, n = row[:, 0::2].clone(), row[:, 1::2].clone(), cos[pos], sin[pos]
                row[:, 0::2], row[:, 1::2] = e * c - o * n, e * n + o * c
    x = x.to(t)
    cache.append(x[:, q_heads:q_heads + heads].double().numpy(), x[:, q_heads + heads:].double().numpy(),
                 starts)
    q = rope(pools, qkv.cuda(), cos.cuda(), sin.cuda(), q_heads, first)
    pools.check(cache)
    assert torch.equal(q.cpu(), x[:, :q_heads])


FORMS = [(14, 2, 64, 64), (28, 4, 128, 64), (8, 8, 64, 16), (16, 1, 128, 32), (6, 2, 128, 128),
         (4, 2, 64, 24), (3, 1, 80, 16), (2, 1, 256, 64)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q_heads,heads,dim,block", FORMS)
@pytest.mark.parametrize("seq,past,causal", [(1, [0, 63, 64, 200], True), (1, [-1, 127, 390, 1000], True),
                                             (2, [5, -2, 128, 383], True), (3, [-1, -3, 60, 380], False),
                                             (17, [0, 47, -17, 300], True), (75, [0, 53, -40, 309], True),
                                             (40, [7, 88, 0, 300], False)])
def test_attention(dtype, q_heads, heads, dim, block, seq, past, causal):
    """With and without a workspace; rows that see nothing are zeros; positions past the pages."""
    t = DTYPES[dtype]
    pools = Pools(4, heads, dim, block, -(-384 // block), seed=seq)
    q = torch.randn((4, q_heads, seq, dim), generator=rng(seq + 1)).to(t)
    cache = pools.oracle()
    pools.cuda()
    want = cache.attention(q.double().numpy(), past, causal, dim ** -0.5)
    out = attend(pools, q.cuda(), past, causal)
    check_attention(out, want, t, 384, dim)
    split = attend(pools, q.cuda(), past, causal, ws=workspace(pools, q), index=torch.int32)
    check_attention(split, want, t, 384, dim)
    rows = attend(pools, q.cuda(), past, causal, bshd=True, ws=workspace(pools, q))
    assert torch.equal(rows.transpose(1, 2), split)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("q_heads,heads,dim,block", [(14, 2, 64, 64), (8, 1, 128, 16), (4, 2, 64, 32),
                                                     (3, 1, 128, 192)])
@pytest.mark.parametrize("seq,past", [(1, [2303, 40]), (1, [-1, 1471]), (2, [1100, 2302]),
                                      (19, [2285, 7]), (33, [-40, 1300])])
def test_long_contexts(dtype, q_heads, heads, dim, block, seq, past):
    """Keys split over workgroups: sequences that fill all splits, few of them, none."""
    t = DTYPES[dtype]
    pools = Pools(2, heads, dim, block, 2304 // block, seed=seq)
    q = torch.randn((2, q_heads, seq, dim), generator=rng(seq + 1)).to(t)
    cache = pools.oracle()
    pools.cuda()
    ws = workspace(pools, q)
    assert ws.numel() > 0
    out = attend(pools, q.cuda(), past, ws=ws)
    check_attention(out, cache.attention(q.double().numpy(), past, True, dim ** -0.5), t, 2304, dim)
    # a workspace that holds fewer splits, or none
    for part in (ws[:ws.numel() // 2], ws[:8], ws[1:]):
        other = attend(pools, q.cuda(), past, ws=part)
        check_attention(other, cache.attention(q.double().numpy(), past, True, dim ** -0.5), t, 2304, dim)


@pytest.mark.parametrize("dim,q_heads,seq", [(64, 7, 1), (128, 16, 1), (64, 2, 10), (128, 1, 17)])
def test_many_splits(dim, q_heads, seq):
    """The most splits that a call may have, with a page that holds nothing among them."""
    pools = Pools(1, 1, dim, 64, 300, missing=[(0, 100, -1)])
    q = torch.randn((1, q_heads, seq, dim), generator=rng(1)).bfloat16()
    cache = pools.oracle()
    out = attend(pools.cuda(), q.cuda(), 19000, ws=workspace(pools, q))
    check_attention(out, cache.attention(q.double().numpy(), [19000], True, dim ** -0.5), torch.bfloat16,
                    19200, dim)


@pytest.mark.parametrize("seq,q_heads", [(1, 7), (40, 7)])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.5])
def test_attention_scales(seq, q_heads, scale):
    pools = Pools(2, 1, 64, 64, 3)
    q = torch.randn((2, q_heads, seq, 64), generator=rng(3)).half()
    cache = pools.oracle()
    out = attend(pools.cuda(), q.cuda(), [90, 151], scale=scale)
    check_attention(out, cache.attention(q.double().numpy(), [90, 151], True, scale), torch.float16, 192, 64)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seq,q_heads", [(1, 7), (2, 8), (30, 4)])
def test_attention_of_unaligned_tensors(seq, q_heads, dim):
    pools = Pools(2, 1, dim, 64, 3)
    flat = torch.randn((2 * q_heads * seq * dim + 1,), generator=rng(3)).bfloat16().cuda()
    q = flat[1:].view(2, q_heads, seq, dim)
    cache = pools.oracle()
    out = attend(pools.cuda(), q, [90, 100])
    want = cache.attention(q.cpu().double().numpy(), [90, 100], True, dim ** -0.5)
    check_attention(out, want, torch.bfloat16, 192, dim)


@pytest.mark.parametrize("dim,block", [(64, 64), (128, 16), (64, 24)])
@pytest.mark.parametrize("q_heads,seq", [(7, 1), (4, 4), (7, 40)])
def test_nan_tokens_and_old_content(dim, block, q_heads, seq):
    """Rows that see a token with an infinity or a NaN are NaN, rows that do not are untouched; what
    the pages hold behind the last token (e4m3 NaN among it) does not show."""
    blocks = -(-192 // block)
    pools = Pools(3, 1, dim, block, blocks, spare=0)
    past = [100, 131, 90]
    for b in range(3):
        for pos in range(past[b] + seq, blocks * block):
            page, slot = int(pools.table[b, pos // block]), pos % block
            pools.key[page, :, slot] = 127
            pools.value[page, :, :, slot] = 255
            pools.scales[page, :, :, slot] = 255
    for b, pos, row in ((0, 100 + seq // 2, 0), (1, 131 + seq - 1, 1)):
        page, slot = int(pools.table[b, pos // block]), pos % block
        pools.scales[page, :, row, slot] = 255
    q = torch.randn((3, q_heads, seq, dim), generator=rng(4)).bfloat16()
    cache = pools.oracle()
    pools.cuda()
    for b, pos, row in ((0, 100 + seq // 2, 0), (1, 131 + seq - 1, 1)):
        cache.scales[int(pools.table[b, pos // block]), :, :, pos % block] = 255
    want = cache.attention(q.double().numpy(), past, True, dim ** -0.5)
    for ws in (None, workspace(pools, q)):
        check_attention(attend(pools, q.cuda(), past, ws=ws), want, torch.bfloat16, 192, dim)


@pytest.mark.parametrize("q_heads,seq", [(2, 1), (2, 20)])
def test_infinite_queries(q_heads, seq):
    """As softmax has it: a score of +inf or NaN makes the row NaN, -inf weighs nothing."""
    pools = Pools(1, 1, 64, 64, 3)
    pools.key[..., 0] = 0x38  # 1
    pools.key[int(pools.table[0, 0]), 0, 5, 0] = 0xB8  # -1 at position 5
    q = torch.randn((1, q_heads, seq, 64), generator=rng(4)).float()
    q[0, 0, :, 0] = -math.inf  # every key -inf but position 5, which is +inf
    cache = pools.oracle()
    out = attend(pools.cuda(), q.cuda(), 100)
    assert out[0, 0].isnan().all()
    want = cache.attention(q[:, 1:].double().numpy(), [100], True, 0.125) if q_heads == 1 else None
    if want is None:
        full = cache.attention(np.nan_to_num(q.double().numpy(), neginf=0.0), [100], True, 0.125)
        check_attention(out[:, 1:], tuple(x[:, 1:] for x in full), torch.float32, 192, 64)


def test_scales_far_apart():
    """Values of very different size: the weights' f16 keeps what a token adds, however small the
    values that its neighbours dwarf, as long as it is the one that is attended."""
    pools = Pools(1, 1, 64, 64, 4)
    q = torch.zeros((1, 1, 1, 64))
    q[..., 0] = 80.0
    pools.key[..., 0] = 0
    pools.scales[:, :, 1] = 150
    at = int(pools.table[0, 1])
    pools.key[at, 0, 9, 0] = 0x7E  # 448: all weight on position 73
    pools.scales[:, :, 0] = 120
    pools.scales[at, 0, 1, 9] = 138  # 2^-12 of the others' size
    cache = pools.oracle()
    pools.cuda()
    for t in DTYPES.values():
        for heads in (1, 20):
            x = q.to(t).expand(1, heads, 1, 64).contiguous()
            out = attend(pools, x.cuda(), 255)
            check_attention(out, cache.attention(x.double().numpy(), [255], True, 0.125), t, 256, 64)


def test_offsets_past_32_bits():
    """Pools of more than 2^32 bytes, the sequences' pages at their end."""
    n, heads, dim, block = (1 << 17) + 40, 4, 128, 64
    pools = Pools(2, heads, dim, block, 3)
    small = pools.oracle()
    pools.key = torch.empty((n, heads, block, dim), dtype=torch.uint8, device="cuda")
    pools.value = torch.empty((n, heads, dim, block), dtype=torch.uint8, device="cuda")
    pools.scales = torch.empty((n, heads, 2, block), dtype=torch.uint8, device="cuda")
    base = n - small.key.shape[0]
    for name in ("key", "value", "scales"):
        getattr(pools, name)[base:] = torch.from_numpy(getattr(small, name)).cuda()
    pools.table = (pools.table + base).cuda()
    pools.count = n
    k, v = values((2, heads, 30, dim), torch.bfloat16, 5), values((2, heads, 30, dim), torch.bfloat16, 6)
    k, v = k.nan_to_num(0, 1, 1).clamp(-9, 9), v.nan_to_num(0, 1, 1).clamp(-9, 9)
    small.append(k.double().numpy(), v.double().numpy(), [60, 130])
    append(pools, k.cuda(), v.cuda(), [60, 130])
    torch.cuda.synchronize()
    assert np.array_equal(pools.key[base:].cpu().numpy(), small.key)
    assert np.array_equal(pools.value[base:].cpu().numpy(), small.value)
    got = read(pools, 30, [60, 130], torch.float32)
    for x, want in zip(got, small.read([60, 130], 30)):
        assert np.array_equal(x.cpu().double().numpy(), want)
    for seq in (1, 30):
        q = torch.randn((2, 28, seq, dim), generator=rng(seq)).bfloat16()
        past = [90 - seq, 160 - seq]
        check_attention(attend(pools, q.cuda(), past),
                        small.attention(q.double().numpy(), past, True, dim ** -0.5), torch.bfloat16, 192,
                        dim)


def test_a_captured_run_of_all():
    """rope_append, attention of the chunk, append, decode and read in one graph, replayed with other
    inputs and positions between eager runs, against eager calls."""
    pools = Pools(2, 2, 64, 64, 4).cuda()
    cos, sin = (x.cuda() for x in tables(64, 256))
    qkv = torch.randn((2, 20, 18 * 64), generator=rng(1)).bfloat16().cuda()
    k, v = (torch.randn((2, 2, 1, 64), generator=rng(s)).bfloat16().cuda() for s in (2, 3))
    q1 = torch.randn((2, 14, 1, 64), generator=rng(4)).bfloat16().cuda()
    first = torch.tensor([30, 100], device="cuda")
    after = first + 20
    ws = workspace(pools, torch.empty((2, 14, 20, 64))), workspace(pools, q1)

    def once(p):
        q = rope(p, qkv, cos, sin, 14, first)
        chunk = attend(p, q, first, ws=ws[0])
        append(p, k, v, after)
        one = attend(p, q1, after, ws=ws[1])
        keys = torch.empty((2, 2, 121, 64), dtype=torch.bfloat16, device="cuda")
        vals = torch.empty_like(keys)
        hip.call("dli_hip_kv_read_fp8", hip.BF16, *p.pointers(), keys.data_ptr(), vals.data_ptr(), 2, 2,
                 121, 64, 64, 4, 0, None, hip.I64, hip.current_stream())
        return chunk, one, keys, vals

    once(pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = once(pools)
    for step in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=rng(10 + step)))
        first.copy_(torch.tensor([20 + 7 * step, 90 + 11 * step]))
        after.copy_(first + 20)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in static]
        want = once(pools)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_another_stream():
    pools = Pools(2, 2, 64, 64, 4).cuda()
    cache = pools.oracle()
    side = torch.cuda.Stream()
    k, v = (torch.randn((2, 2, 90, 64), generator=rng(s)).half().cuda() for s in (2, 3))
    q = torch.randn((2, 14, 1, 64), generator=rng(4)).half().cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        append(pools, k, v, 10)
        out = attend(pools, q, 99, ws=workspace(pools, q))
    torch.cuda.current_stream().wait_stream(side)
    cache.append(k.double().cpu().numpy(), v.double().cpu().numpy(), [10, 10])
    pools.check(cache)
    check_attention(out, cache.attention(q.double().cpu().numpy(), [99, 99], True, 0.125),
                    torch.float16, 256, 64)


@pytest.mark.parametrize("dim,block", [(64, 64), (128, 16), (80, 64)])
def test_positions_at_the_ends_of_their_range(dim, block):
    """Tokens before and past the pages: dropped, read as zeros; a query past them sees every key."""
    pools = Pools(2, 2, dim, block, 128 // block)
    cache = pools.oracle()
    pools.cuda()
    ends = [-(1 << 63), (1 << 63) - 1]
    for seq in (1, 20, 70):
        k = torch.randn((2, 2, seq, dim), generator=rng(seq)).bfloat16().cuda()
        append(pools, k, k, ends)
        pools.check(cache)
        for x in read(pools, seq, ends, torch.bfloat16):
            assert (x == 0).all()
        q = torch.randn((2, 4, seq, dim), generator=rng(seq + 1)).bfloat16()
        check_attention(attend(pools, q.cuda(), ends),
                        cache.attention(q.double().numpy(), [-200, 128], True, dim ** -0.5),
                        torch.bfloat16, 128, dim)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("seq", [1, 20])
def test_scores_far_below_zero(dtype, dim, seq):
    """Every score between -2^118 and -2^112: the largest takes all the weight."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, 64, 2)
    pools.key[:] = 0
    pools.key[..., 0] = 0x78  # 256
    pools.scales[:, :, 0] = 127
    best = int(pools.table[0, 1])
    pools.key[best, 0, 3, 0] = 0x48  # 4, at position 67
    q = torch.zeros((1, 2, seq, dim), dtype=t)
    q[..., 0] = -2.0 ** 110
    cache = pools.oracle()
    out = attend(pools.cuda(), q.cuda(), 100, scale=1.0)
    want = torch.from_numpy(cache.rows(0, 67)[1][0]).to(t)
    assert torch.equal(out.cpu(), want.expand(out.shape))


@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("seq", [1, 20])
def test_values_near_the_largest(dim, seq):
    """Sums of values that pass the largest number while their mean does not."""
    pools = Pools(1, 1, dim, 64, 3)
    pools.scales[:, :, 1] = torch.where(torch.arange(64) % 3 == 0, 247, 240).to(torch.uint8)
    pools.value[:] = 0x74  # 192: 2^120 times it is 3/4 of 2^128
    q = torch.randn((1, 3, seq, dim), generator=rng(8))
    cache = pools.oracle()
    for t in (torch.float32, torch.bfloat16):
        x = q.to(t)
        check_attention(attend(pools.cuda(), x.cuda(), 150),
                        cache.attention(x.double().numpy(), [150], True, dim ** -0.5), t, 192, dim)


def test_more_rows_than_workgroups():
    """The row-by-row form goes on from row to row: the same rows in shorter calls, bit for bit."""
    pools = Pools(3, 1, 8, 8, 9).cuda()
    q = torch.randn((3, 2, 13000, 8), generator=rng(9)).bfloat16().cuda()
    past = torch.tensor([0, 40, -6000], device="cuda")
    whole = attend(pools, q, past)
    for at in range(0, 13000, 6500):
        part = attend(pools, q[:, :, at:at + 6500].contiguous(), past + at)
        assert torch.equal(part, whole[:, :, at:at + 6500])


@pytest.mark.parametrize("seq", [1, 20])
def test_a_page_past_32_bit_offsets(seq):
    """A page of 2^33 bytes a head: the dims of the values lie past 32-bit offsets."""
    block, dim = 1 << 26, 128
    small = Pools(1, 1, dim, 64, 2, spare=0)
    small.table[0] = torch.tensor([0, 1])
    cache = small.oracle()
    pools = Pools(1, 1, dim, 8, 1, spare=0)
    pools.block, pools.count = block, 1
    pools.key = torch.empty((1, 1, block, dim), dtype=torch.uint8, device="cuda")
    pools.value = torch.empty((1, 1, dim, block), dtype=torch.uint8, device="cuda")
    pools.scales = torch.empty((1, 1, 2, block), dtype=torch.uint8, device="cuda")
    pools.table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    pools.key[0, 0, :128] = small.key.view(128, dim).cuda()
    for i in range(2):
        pools.value[0, 0, :, 64 * i:64 * i + 64] = small.value[i, 0].cuda()
        pools.scales[0, 0, :, 64 * i:64 * i + 64] = small.scales[i, 0].cuda()
    q = torch.randn((1, 4, seq, dim), generator=rng(seq)).bfloat16()
    out = attend(pools, q.cuda(), 100)
    check_attention(out, cache.attention(q.double().numpy(), [100], True, dim ** -0.5), torch.bfloat16, 128,
                    dim)
    k = torch.randn((1, 1, seq, dim), generator=rng(3)).bfloat16()
    cache.append(k.double().numpy(), k.double().numpy(), [50])
    append(pools, k.cuda(), k.cuda(), 50)
    for x, want in zip(read(pools, 128, 0, torch.float32), cache.read([0], 128)):
        assert np.array_equal(x.cpu().double().numpy(), want)


# bf16, head_dim 128, many workgroups and contexts past 2500 tokens: two splits of 17 rows a pair, rows of
# three workgroups a pair, one split
PHASED = [(16, 8, 8, 17, 64), (16, 32, 2, 40, 128), (32, 8, 8, 33, 64)]


@pytest.mark.parametrize("batch,q_heads,heads,seq,block", PHASED)
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows_over_long_contexts(batch, q_heads, heads, seq, block, causal):
    """Sequences of every length class: none, less than a tile, tile edges, past the pages; pages that hold
    nothing at the start, in the middle and at the end of a sequence."""
    tokens = 2560
    n = tokens // block
    missing = [(1, n - 1, -1), (2, 0, 1 << 30), (3, n // 2, -7), (4, n // 2, -1), (4, n // 2 + 1, -1)]
    missing += [(5, i, -1) for i in range(n)]
    pools = Pools(batch, heads, 128, block, n, seed=seq, missing=missing)
    lengths = [0, 2530, 2400, 1999, 2100, 900, -seq, -9, 2560, 5000, 30, 31, 47, 48, 63, 64]
    past = [x - (seq if 20 < x < 70 else 0) for x in lengths] * (batch // 16)
    q = torch.randn((batch, q_heads, seq, 128), generator=rng(seq + 1)).bfloat16()
    cache = pools.oracle()
    pools.cuda()
    want = cache.attention(q.double().numpy(), past, causal, 128 ** -0.5)
    whole = attend(pools, q.cuda(), past, causal)
    check_attention(whole, want, torch.bfloat16, tokens, 128)
    ws = workspace(pools, q)
    split = attend(pools, q.cuda(), past, causal, ws=ws, index=torch.int32)
    check_attention(split, want, torch.bfloat16, tokens, 128)
    rows = attend(pools, q.cuda(), past, causal, bshd=True, ws=ws)
    assert torch.equal(rows.transpose(1, 2), split)


def test_nan_tokens_and_sizes_over_long_contexts():
    """Rows behind the last token of any content, NaN tokens that some queries see, values from the least to
    the largest, scores far below zero: 17 rows a pair, two splits."""
    pools = Pools(16, 8, 128, 64, 40, seed=3)
    past = [1000 + 64 * b for b in range(16)]
    behind = torch.zeros((16, 2560), dtype=torch.bool)
    for b in range(16):
        behind[b, past[b] + 17:] = True
    cache = pools.oracle()
    for b in range(16):
        for i in range(40):
            page, dead = int(pools.table[b, i]), behind[b, 64 * i:64 * i + 64]
            pools.key[page, :, dead] = 0x7F
            pools.value[page][:, :, dead] = 0xFF
            pools.scales[page][:, :, dead] = 255
            if b == 3:  # one size a tile, from small to large
                size = torch.full((8, 64), 60 + 4 * i, dtype=torch.uint8)
                pools.scales[page, :, 1] = torch.where(dead, pools.scales[page, :, 1], size)
                cache.scales[page, :, 1] = size.numpy()
        if b % 4 == 1:  # in the middle, and where only the last queries see it
            for at in (777, past[b] + 9):
                page = int(pools.table[b, at // 64])
                for p in (pools, cache):
                    p.key[page, :2, at % 64] = 0
                    p.value[page, :2, :, at % 64] = 0
                    p.scales[page, :2, at // 9 % 2, at % 64] = 255
    q = torch.randn((16, 8, 17, 128), generator=rng(5))
    q[7] *= 2.0 ** 100
    q = q.bfloat16()
    want = cache.attention(q.double().numpy(), past, True, 128 ** -0.5)
    ws = workspace(pools, q)
    pools.cuda()
    for space in (None, ws):
        out = attend(pools, q.cuda(), past, ws=space)
        keep = [b for b in range(16) if b != 7]
        check_attention(out[keep], tuple(x[keep] for x in want), torch.bfloat16, 2560, 128)
        # scores of 2^100: the largest takes all the weight
        assert torch.equal(out[7].cpu(), torch.from_numpy(want[0][7]).bfloat16())


def test_long_contexts_captured():
    """A graph of the kernel replayed with other queries and positions, against eager calls."""
    pools = Pools(16, 8, 128, 64, 40, seed=4).cuda()
    q = torch.randn((16, 8, 17, 128), generator=rng(1)).bfloat16().cuda()
    first = torch.randint(0, 2600, (16,), generator=rng(2)).cuda()
    ws = workspace(pools, q)
    attend(pools, q, first, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = attend(pools, q, first, ws=ws)
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=rng(20 + step)))
        first.copy_(torch.randint(0, 2600, (16,), generator=rng(30 + step)))
        graph.replay()
        torch.cuda.synchronize()
        got = static.clone()
        assert torch.equal(got, attend(pools, q, first, ws=ws))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim,q_heads,seq", [(64, 2, 1), (64, 2, 20), (128, 2, 20), (64, 4, 1200), (128, 4, 1200),
                                             (80, 2, 3)])
@pytest.mark.parametrize("size", [26, 60, 100])
def test_scores_past_whole_numbers(dtype, dim, q_heads, seq, size):
    """Scores of about 2^size of either sign: the largest takes all the weight. One key of a row's four
    stands out by a factor of two at least, so sums in fp32 find it."""
    t = DTYPES[dtype]
    pools = Pools(4, 1, dim, 64, 24)
    pools.key[:] = 0
    g = rng(size)
    for b in range(4):
        for i in range(24):
            page = int(pools.table[b, i])
            pools.key[page, 0, :, 0] = torch.randint(0x30, 0x38, (64,), generator=g).to(torch.uint8)
        pools.key[int(pools.table[b, 0]), 0, 3 + b, 0] = 0x48
        pools.key[int(pools.table[b, 0]), 0, 9, 0] = 0xC8
    pools.scales[:, :, 0] = 127
    q = torch.zeros((4, q_heads, seq, dim))
    q[..., 0] = 2.0 ** size * (1 + torch.rand((4, q_heads, seq), generator=g))
    q[:, 1::2] *= -1
    q = q.to(t)
    cache = pools.oracle()
    out = attend(pools.cuda(), q.cuda(), 300, scale=dim ** -0.5 * 0.9).cpu()
    for b in range(4):
        for h in range(2):
            want = torch.from_numpy(cache.rows(b, 9 if h else 3 + b)[1][0]).to(t)
            assert torch.equal(out[b, h::2], want.expand(out[b, h::2].shape))
