"""The 8-bit KV cache's attention at the ends of its numbers' ranges, form by form: large scores, values
and queries. Expected values are exact or float64; inputs are chosen so that fp32 sums are exact."""
from __future__ import annotations

import copy
import math

import pytest
import torch

from dli import hip
from test_kv_fp8_gpu import DTYPES, Pools, attend, rng, workspace

pytestmark = pytest.mark.gpu

# (head_dim, query heads, queries): one token, 16 rows at most, chunks of 64 and 128 rows, row by row
FORMS = [(64, 2, 1), (128, 7, 1), (64, 8, 2), (128, 4, 4), (64, 4, 10), (128, 4, 1200), (64, 4, 1200), (80, 2, 3)]


def code(value):
    """The e4m3 code of an element."""
    return int(torch.tensor(value).to(torch.float8_e4m3fn).view(torch.uint8))


def token(pools, b, pos):
    """(page, slot) of a position."""
    return int(pools.table[b, pos // pools.block]), pos % pools.block


def value_of(pools, b, pos):
    """The value row that a position stands for, float64 [D] of KV head 0."""
    page, slot = token(pools, b, pos)
    elements = pools.value[page, 0, :, slot].cpu().view(torch.float8_e4m3fn).double()
    return elements * 2.0 ** (int(pools.scales[page, 0, 1, slot]) - 127)


def close(got, want, dtype, steps=16):
    """Within the output's rounding (half a step, half of the least subnormal) and `steps` fp32 roundings
    of the largest magnitude among the values."""
    got, want = got.cpu().double(), want.expand(got.shape)
    eps = torch.finfo(dtype).eps
    bound = eps / 2 * want.abs() + steps * 2.0 ** -24 * want.abs().max() + torch.finfo(dtype).smallest_normal * eps
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim,q_heads,seq", FORMS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [20, 22, 23, 24, 25, 26, 27, 28, 29, 31, 60])
def test_weights_of_large_scores(dtype, dim, q_heads, seq, sign, power):
    """Scores (in powers of two) of sign * 1.5 * 2^power at one token and, where fp32 holds it, 4 more at
    another, eight tiles later: weights 1 and 16. Elsewhere scores are lower by 2^power or more."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, 64, 30)
    pools.key[:] = 0
    if sign < 0:
        pools.key[:, :, :, 0] = code(48.0)
    pools.scales[:, :, 0] = 127 + power - 12
    pools.scales[:, :, 1] = 127
    first, second = 70, 70 + 8 * 64
    apart = 4 if power <= 25 else 0
    for pos, more in ((first, 0), (second, apart)):
        page, slot = token(pools, 0, pos)
        pools.key[page, 0, slot, 0] = code(24.0)
        pools.key[page, 0, slot, 1] = code(2.0 ** -5 if more else 0.0)
    q = torch.zeros((1, q_heads, seq, dim))
    q[..., 0] = sign * 2.0 ** 8
    q[..., 1] = 2.0 ** (min(power, 25) * -1 + 12 + 2 + 5)  # times 2^-5 2^(power - 12): 4
    a, b = value_of(pools, 0, first), value_of(pools, 0, second)
    weight = 2.0 ** apart
    want = (a + weight * b) / (1 + weight)
    pools.cuda()
    for ws in (None, workspace(pools, q)):
        out = attend(pools, q.to(t).cuda(), 700, scale=math.log(2), ws=ws)
        # weights are powers of two; the quotient of their sum is rounded, and the output
        close(out, want, t)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim,q_heads,seq", FORMS)
@pytest.mark.parametrize("power", [10, 21, 24, 25, 26, 27, 28, 33, 90])
def test_equal_large_scores(dtype, dim, q_heads, seq, power):
    """Two tokens of one score, eight tiles apart, under a softmax scale that rounds it: equal weights."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, 64, 30, seed=power)
    pools.key[:] = 0
    pools.scales[:, :, 0] = 127 + power - 12
    pools.scales[:, :, 1] = 127
    for pos in (70, 582):
        page, slot = token(pools, 0, pos)
        pools.key[page, 0, slot, 0] = code(26.0)
    q = torch.zeros((1, q_heads, seq, dim))
    q[..., 0] = 2.0 ** 8 * 1.375
    want = (value_of(pools, 0, 70) + value_of(pools, 0, 582)) / 2
    pools.cuda()
    for ws in (None, workspace(pools, q)):
        close(attend(pools, q.to(t).cuda(), 700, scale=0.2718, ws=ws), want, t)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim,q_heads,seq", [(64, 2, 1), (128, 7, 1), (128, 4, 4), (64, 4, 10), (128, 4, 40)])
@pytest.mark.parametrize("exponent", [247, 246, 235, 0])
def test_values_near_the_ends_over_splits(dtype, dim, q_heads, seq, exponent):
    """Every token's values are 448 * 2^(exponent - 127), the weights of a row equal: the join of the splits
    neither overflows nor loses what the output's type holds."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, 64, 30)
    pools.value[:] = code(448.0)
    pools.scales[:, :, 1] = exponent
    q = torch.zeros((1, q_heads, seq, dim), dtype=t)
    pools.cuda()
    ws = workspace(pools, q)
    assert ws.numel() > 0
    want = torch.tensor(448.0 * 2.0 ** (exponent - 127), dtype=torch.float64)
    out = attend(pools, q.cuda(), 1700, ws=ws)
    if exponent == 247:  # 1.75 * 2^128 is past either type
        assert (out == math.inf).all()
    else:
        # some 2000 equal weights: their sum in fp32 is exact, a split's quotient and the join's are rounded
        close(out, want, t)


def bits(word):
    return torch.tensor(word, dtype=torch.int32).view(torch.float32).item()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim,q_heads,seq", FORMS)
def test_queries_that_are_not_finite(dtype, dim, q_heads, seq):
    """As softmax has it, but zeros where every score is -infinity: an infinite query element whose keys'
    elements all have the other sign weighs nothing; one key of its sign, or a NaN, makes the row NaN. Rows
    beside it are those of a call without it, bit for bit."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, 64, 22)
    pools.key[..., 0] = code(1.0)
    pools.key[..., 1] = code(-1.0)
    page, slot = token(pools, 0, 90)
    pools.key[page, 0, slot, 1] = code(0.5)
    pools.cuda()
    q = torch.randn((1, q_heads, seq, dim), generator=rng(1)).to(t).cuda()
    ws = workspace(pools, q)
    past = 1400 - seq
    for space in (None, ws):
        plain = attend(pools, q, past, ws=space)
        assert plain.isfinite().all()
        nans = [math.nan] + ([bits(0x7F800001), bits(-0x7FFFFF)] if dtype == "float32" else [])
        for at, x, want in [(0, -math.inf, 0.0), (1, -math.inf, math.nan), (1, math.inf, math.nan),
                            (0, math.inf, math.nan)] + [(2, n, math.nan) for n in nans]:
            odd = q.clone()
            odd[0, 0, -1, at] = x
            out = attend(pools, odd, past, ws=space)
            row = out[0, 0, -1].clone()
            assert row.isnan().all() if math.isnan(want) else (row == want).all(), (at, x)
            out[0, 0, -1] = plain[0, 0, -1]
            assert torch.equal(out, plain)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim,q_heads,seq", FORMS)
def test_large_queries_over_small_keys(dtype, dim, q_heads, seq):
    """Queries of about 2^120 over keys of 2^-126 times their elements: the scores are those of queries and
    keys that meet in the middle, and so are the results, bit for bit."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, 64, 22)
    pools.key |= 0x48  # elements of 4 and more
    pools.key[pools.key % 128 == 127] = 0x48
    pools.scales[:, :, 0] = 121
    pools.cuda()
    small = torch.randn((1, q_heads, seq, dim), generator=rng(1)).to(t).cuda()
    ws = workspace(pools, small)
    past = 1400 - seq
    want = [attend(pools, small, past, ws=space) for space in (None, ws)]
    assert want[0].isfinite().all()
    pools.scales[:, :, 0] = 1
    large = small * 2.0 ** 120
    for space, x in zip((None, ws), want):
        assert torch.equal(attend(pools, large, past, ws=space), x)
    # one row of a call, the others as they were
    pools.scales[:, :, 0] = 121
    mixed = small.clone()
    mixed[0, 0, -1] *= 2.0 ** 120
    for space, x in zip((None, ws), want):
        out = attend(pools, mixed, past, ws=space)
        out[0, 0, -1] = x[0, 0, -1]
        assert torch.equal(out, x)


def dense(pools, tokens):
    """Keys, value elements and value scales of the one sequence's first tokens, float64: [T, D], [T, D], [T]."""
    pages = pools.table[0].long().cuda()
    key, value, scales = (x.cuda()[pages] for x in (pools.key, pools.value, pools.scales))
    k = key[:, 0].view(torch.float8_e4m3fn).double().flatten(0, 1)[:tokens]
    v = value[:, 0].transpose(1, 2).contiguous().view(torch.float8_e4m3fn).double().flatten(0, 1)[:tokens]
    unit = torch.exp2(scales[:, 0].double() - 127)  # [pages, 2, block]
    return k * unit[:, 0].flatten()[:tokens, None], v, unit[:, 1].flatten()[:tokens]


def check_far_apart(out, pools, q, past, scale, near=0, missing=()):
    """out [1, Hq, S, D] of queries [1, Hq, S, D] (causal), one KV head, against float64; missing: pages of the
    table that hold nothing, though `pools` has them. Off by at most: the
    output's rounding; per weight its rounding (f16 once, or 22 bits) and the shift of its score by fp32's
    sum of D products, scaling and exponent; the sums' roundings; and f16's half least step, 2^-25 with 2^11
    or more at the row's largest weight times value scale, for every token's elements. Chunks count
    from the largest value scale about, which is up to 2^near times that."""
    t, dim = out.dtype, out.shape[3]
    q = q.cuda()
    k, v, unit = dense(pools, past + q.shape[2])
    s = q[0].double() @ k.T * scale
    limit = past + 1 + torch.arange(q.shape[2], device="cuda")
    for page in missing:
        s[..., page * pools.block:(page + 1) * pools.block] = -math.inf
    s = s.masked_fill(torch.arange(len(k), device="cuda") >= limit[:, None], -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    want, mag = (w @ (unit[:, None] * x) / total for x in (v, v.abs()))
    spread = (q[0].double().abs() @ k.abs().T).amax(-1, keepdim=True) * scale
    floor = (w > 0).double() @ v.abs() * ((w * unit).amax(-1, keepdim=True) / total)
    eps, tiny = torch.finfo(t).eps, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    weight = 2.0 ** -12 if t == torch.bfloat16 else 2.0 ** -22
    shift = 2 * (dim + 8) * 2.0 ** -24 * (spread + 30)
    sums = (4 * len(k) / 64 + 96) * 2.0 ** -24
    bound = eps / 2 * want.abs() + (1 + eps) * ((weight + shift + sums) * mag + 2.0 ** (near - 36) * floor) + tiny
    got = out[0].double()
    # infinite where no value within the bound rounds to a finite one; of any such kind where some do (a sum of
    # large terms that cancel)
    over = want.abs() - bound > torch.finfo(t).max * (1 + eps / 2)
    assert (got[over] == want[over].sign() * math.inf).all()
    edge = (want.abs() + bound > torch.finfo(t).max) & ~over
    error = (got - want).abs()[~over & ~edge] / bound[~over & ~edge]
    assert not got[~over].isnan().any()
    assert (error <= 1).all(), error.max()


# value scales against the others': a later token that earlier queries do not see; one seen early on with a
# weight of 2^-300; one that has the largest weight until the others come; one whose small weight its size
# makes up for; every token of another size
APART = ["unseen", "negligible", "at first", "counted", "ladder"]


def apart(kind, dtype, dim, q_heads, seq, octaves, block=64, tokens=1920):
    """(pools, q): q's element 0 is 1 and k's element 0 chooses a score of a few tokens (in powers of two)."""
    pools = Pools(1, 1, dim, block, tokens // block, seed=octaves)
    pools.key[..., 0] = 0
    pools.scales[:, :, 0] = 117
    low = 106 if dtype == "float16" and octaves < 149 else 80  # codes end at 254
    near = torch.randint(0, 3, pools.scales[:, :, 1].shape, generator=rng(3))
    pools.scales[:, :, 1] = (low + near).to(torch.uint8)
    q = torch.randn((1, q_heads, seq, dim), generator=rng(seq))
    q[..., 0] = 1.0

    def place(pos, score, up):
        page, slot = token(pools, 0, pos)
        pools.key[page, 0, slot] = 0
        pools.key[page, 0, slot, 0] = code(math.copysign(1.0, score))
        pools.scales[page, 0, 0, slot] = 127 + int(math.log2(abs(score)))
        pools.scales[page, 0, 1, slot] = low + up

    if kind == "unseen":
        for pos in range(700 + seq - 1, tokens):
            place(pos, 1.0, octaves)
    elif kind == "negligible":
        place(130, -512.0, octaves)
    elif kind == "at first":
        place(1, 64.0, octaves)
        for pos in range(640, 700):
            place(pos, 256.0, 0)
    elif kind == "counted":
        place(300, -float(2 ** int(math.log2(octaves))), octaves)
    else:
        size = torch.randint(0, octaves + 1, pools.scales[:, :, 1].shape, generator=rng(9))
        pools.scales[:, :, 1] = (low + size).to(torch.uint8)
    return pools, q


def far_apart(kind, dtype, dim, q_heads, seq, octaves, near, **more):
    t = DTYPES[dtype]
    pools, q = apart(kind, dtype, dim, q_heads, seq, octaves, **more)
    q = q.to(t)
    pools.cuda()
    for space in (None, workspace(pools, q)):
        out = attend(pools, q.cuda(), [700], scale=math.log(2), ws=space)
        check_far_apart(out, pools, q, 700, math.log(2), near)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim,q_heads,seq", [f for f in FORMS if f[1] * f[2] <= 16 or f[0] == 80])
@pytest.mark.parametrize("kind", APART)
@pytest.mark.parametrize("octaves", [9, 20, 35, 100, 160])
def test_values_far_apart(dtype, dim, q_heads, seq, kind, octaves):
    far_apart(kind, dtype, dim, q_heads, seq, octaves, 0)


# (dtype, head_dim, query heads, queries, tokens of a page): chunks of 64 and of 128 rows
CHUNKS = [("float32", 64, 4, 10, 64), ("float32", 128, 4, 40, 32), ("bfloat16", 64, 4, 40, 64),
          ("bfloat16", 128, 4, 10, 16), ("float16", 64, 4, 10, 32), ("float16", 128, 4, 40, 64),
          ("bfloat16", 64, 14, 1200, 64), ("bfloat16", 128, 14, 1200, 64), ("bfloat16", 64, 14, 1200, 32),
          ("bfloat16", 128, 14, 1200, 16), ("float16", 128, 41, 1200, 64), ("float16", 128, 41, 1200, 32),
          ("float32", 128, 2, 1200, 64)]


@pytest.mark.parametrize("dtype,dim,q_heads,seq,block", CHUNKS)
@pytest.mark.parametrize("kind", APART)
@pytest.mark.parametrize("octaves", [9, 13, 20, 35, 100, 160])
def test_values_far_apart_in_chunks(dtype, dim, q_heads, seq, block, kind, octaves):
    """Scales of up to 2^14 of each other are taken relative to the largest, others by the row."""
    # the others lie within 2^2 of each other
    far_apart(kind, dtype, dim, q_heads, seq, octaves, min(octaves + 2, 14), block=block)


@pytest.mark.parametrize("kind", APART)
@pytest.mark.parametrize("octaves", [9, 13, 20, 35, 100, 160])
@pytest.mark.parametrize("block", [64, 128])
def test_values_far_apart_over_long_contexts(kind, octaves, block):
    """The same where two halves of a workgroup run a phase apart (16800 rows of a pair, up to 2688 tokens)."""
    far_apart(kind, "bfloat16", 128, 14, 1200, octaves, min(octaves + 2, 14), block=block, tokens=2688)


@pytest.mark.parametrize("dim,q_heads,seq", [(64, 14, 1), (128, 14, 1), (64, 14, 20), (128, 14, 20)])
def test_short_sequences_in_long_tables(dim, q_heads, seq):
    """Where the host knows that few tokens are held, keys are not split over workgroups that would find none:
    the workspace is left as it was, and results are those of a short table."""
    pools = Pools(1, 2, dim, 64, 300, seed=1).cuda()
    q = torch.randn((1, q_heads, seq, dim), generator=rng(1)).bfloat16().cuda()
    ws = workspace(pools, q)
    assert ws.numel() > 0
    out = attend(pools, q, 200, ws=ws)
    assert (ws == 255).all()
    pools.max_blocks, pools.table = 4, pools.table[:, :4].contiguous()
    assert torch.equal(attend(pools, q, 200), out)


def without(pools, missing):
    """`pools` with those pages taken out of the table."""
    bare = copy.copy(pools)
    bare.table = pools.table.clone()
    bare.table[0, list(missing)] = -1
    return bare


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim,block,tokens", [(64, 16, 8400), (128, 16, 17000), (64, 32, 17000), (128, 32, 25000),
                                              (64, 64, 33000), (128, 64, 66000)])
def test_single_tokens_over_many_pages(dtype, dim, block, tokens):
    """Keys that are not split: each wave of a workgroup goes through more pages than it has lanes to hold their
    ids, up to two times over. The weight lies on pages at both sides of where it reads more, and some of them
    hold nothing."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, block, -(-tokens // block), seed=block).cuda()
    q = torch.randn((1, 3, 1, dim), generator=rng(1)).to(t)
    per = 64 // block if block < 64 else 1  # pages a tile
    runs = 8 * (64 if block == 64 else 16)  # tiles before ids are read anew
    missing = [p for k in (1, 2) for p in (k * runs * per - 1, k * runs * per + 3, k * runs * per + 9 * per)
               if p < -(-tokens // block)] + [2, 0]
    pools.key[..., 0] = 0
    for page in missing:
        near = pools.table[0, max(page - 1, 0):page + 2].long()
        pools.key[near, :, :, 0] = code(448.0)
        pools.scales[near, :, 0] = 120  # 3.5 in the cache: weights of e^8 and more
    q[..., 0] = 20.0
    out = attend(without(pools, missing), q.cuda(), tokens - 1)
    check_far_apart(out, pools, q, tokens - 1, dim ** -0.5, 0, missing)


@pytest.mark.parametrize("dtype,dim,q_heads,seq", [("bfloat16", 128, 14, 1200), ("float16", 128, 4, 100),
                                                   ("bfloat16", 64, 14, 1200), ("float32", 128, 4, 1),
                                                   ("bfloat16", 128, 8, 2)])
def test_pages_past_32_bits(dtype, dim, q_heads, seq):
    """A sequence whose pages lie behind 2^32 bytes of each pool, in every form that goes by pages."""
    t = DTYPES[dtype]
    n = (1 << 32) // (64 * dim) + 60
    small = Pools(1, 1, dim, 64, 42, seed=5, spare=0)
    pools = copy.copy(small)
    shapes = {"key": (n, 1, 64, dim), "value": (n, 1, dim, 64), "scales": (n, 1, 2, 64)}
    for name, shape in shapes.items():
        pool = torch.empty(shape, dtype=torch.uint8, device="cuda")
        pool[n - 42:] = getattr(small, name).cuda()
        setattr(pools, name, pool)
    pools.table, pools.count = (small.table + n - 42).cuda(), n
    q = torch.randn((1, q_heads, seq, dim), generator=rng(seq)).to(t)
    for ws in (None, workspace(pools, q)):
        out = attend(pools, q.cuda(), [1400], ws=ws)
        check_far_apart(out, small, q, 1400, dim ** -0.5, 14)


# (dtype, head_dim, query heads, queries, tokens of a page, tokens of the table)
MIXED = [("bfloat16", 64, 7, 2, 64, 1920), ("float32", 128, 4, 4, 16, 1920), ("float16", 80, 2, 3, 64, 1920)]
MIXED += [(*c, 1920) for c in CHUNKS if c[3] < 1200 or c[4] == 32]
MIXED += [("bfloat16", 64, 14, 1200, 64, 1920), ("bfloat16", 128, 14, 1200, 128, 2688)]


@pytest.mark.parametrize("dtype,dim,q_heads,seq,block,tokens", MIXED)
@pytest.mark.parametrize("octaves", [8, 110])
@pytest.mark.parametrize("side", [0, 1])
def test_holes_zeros_and_nan_among_values_far_apart(dtype, dim, q_heads, seq, block, tokens, octaves, side):
    """Pages that hold nothing (with scales of any size), rows of zeros, and a token that is not finite and
    that only the last query sees."""
    t = DTYPES[dtype]
    pools, q = apart("ladder", dtype, dim, q_heads, seq, octaves, block, tokens)
    missing = [3, 9, 700 // block - 1]
    for page in missing:
        pools.scales[int(pools.table[0, page])] = torch.tensor([7, 250], dtype=torch.uint8).view(2, 1)
    for pos in (0, 77, 699, 700):
        page, slot = token(pools, 0, pos)
        pools.value[page, 0, :, slot] = 0
        pools.scales[page, 0, 1, slot] = 0
    page, slot = token(pools, 0, 700 + seq - 1)
    pools.key[page, 0, slot] = pools.value[page, 0, :, slot] = 0
    pools.scales[page, 0, side, slot] = 255
    q = q.to(t)
    pools.cuda()
    bare = without(pools, missing)
    for space in (None, workspace(pools, q)):
        out = attend(bare, q.cuda(), [700], scale=math.log(2), ws=space)
        assert out[:, :, -1].isnan().all()
        check_far_apart(out[:, :, :-1], pools, q[:, :, :-1], 700, math.log(2), 14, missing)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim,q_heads,seq", FORMS[:5] + [(128, 4, 40), (80, 2, 3), (128, 14, 300)])
@pytest.mark.parametrize("octaves", [90, 140, 200, 230])
def test_splits_far_apart(dtype, dim, q_heads, seq, octaves):
    """The first 1024 tokens have weights of 2^-octaves and values 2^octaves as large as the others': the
    splits that hold only them count as much as the rest."""
    t = DTYPES[dtype]
    pools = Pools(1, 1, dim, 64, 30, seed=octaves)
    pools.key[:] = 0
    pools.scales[:, :, 0] = 127
    pools.scales[:, :, 1] = 10
    for page in pools.table[0, :16].long():
        pools.key[page, 0, :, 0] = code(-1.0)
        pools.key[page, 0, :, 1] = code(-0.5)
        pools.scales[page, 0, 1] = 10 + octaves
    q = torch.zeros((1, q_heads, seq, dim))
    q[..., 0] = octaves - octaves % 4 - 2
    q[..., 1] = 2 * (octaves % 4 + 2)  # octaves in all, exact in 16 bits
    q = q.to(t)
    pools.cuda()
    for space in (None, workspace(pools, q)):
        out = attend(pools, q.cuda(), [1500], scale=math.log(2), ws=space)
        check_far_apart(out, pools, q, 1500, math.log(2), 0)
