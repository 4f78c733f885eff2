"""What mx_linear's sums lose: nothing for e2m1 rows and for fp32 results, whatever the values; with
e4m3 rows and a 16-bit result at most 7 x 2^-13 of the largest of 8 neighbouring products."""
import numpy as np
import pytest
import torch

import mx_oracle as mx
from support import run_op
from test_mx_cpu import DTYPES
from test_mx_gpu import UNIT

pytestmark = pytest.mark.gpu

# rows, outputs, columns: the stream of 1, 4 and 16 rows, 64-row tiles, runs, tiles of 128 and of 256,
# with scales as they are and laid out
SIZES = [(1, 64, 256), (4, 70, 288), (16, 1200, 4864), (40, 9728, 896), (40, 9729, 928),
         (40, 33000, 2048), (200, 2000, 896), (200, 2000, 4384), (3001, 4104, 1824)]


def codes_of(values, form):
    """Codes of element values that the type holds, one to a column."""
    table = {"fp8": mx.E4M3, "fp4": mx.E2M1}[form]
    e = np.searchsorted(table, np.abs(values))
    assert np.array_equal(table[e], np.abs(values))
    if form == "fp8":
        return (e + 128 * (values < 0)).astype(np.uint8)
    e = (e + 8 * (values < 0)).reshape(*values.shape[:-1], -1, 2)
    return (e[..., 0] + 16 * e[..., 1]).astype(np.uint8)


def product(x, w, form, out_dtype):
    """x [m, k] and w [n, k] of element values, all scales 1."""
    ones = [torch.full((v.shape[0], v.shape[1] // 32), 127, dtype=torch.uint8).cuda() for v in (x, w)]
    return run_op("mx_linear", {"x": torch.from_numpy(codes_of(x, form)).cuda(), "xs": ones[0],
                                "w": torch.from_numpy(codes_of(w, "fp4")).cuda(), "ws": ones[1]},
                  ("out",), {"out_dtype": out_dtype})["out"]


# 8 neighbouring columns of x, each with the weights that make it hardest: the largest product beside
# the smallest that the element type, or one half of its exponents, has
EIGHTS = [([448.0] + [0.05078125] * 7, [6.0] * 8), ([448.0, -448.0] + [0.05078125] * 6, [6.0] * 8),
          ([448.0] + [2.0 ** -9] * 7, [6.0] + [0.5] * 7), ([3.75] + [2.0 ** -9] * 7, [6.0] + [0.5] * 7),
          ([3.75, -3.75] + [2.0 ** -9] * 6, [6.0, 6.0] + [0.5] * 6),
          ([448.0] + [4.5] * 7, [6.0] + [0.5] * 7), ([448.0, -448.0] + [4.5] * 6, [6.0, 6.0] + [0.5] * 6)]


@pytest.mark.parametrize("out_dtype", list(DTYPES))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_one_group_of_eight_columns(out_dtype, m, n, k):
    x, w = np.zeros((m, k)), np.zeros((n, k))
    for i in range(m):  # row i: its eight at some place
        at = 8 * (5 * i % (k // 8))
        x[i, at:at + 8] = np.roll(EIGHTS[i % len(EIGHTS)][0], i)
    for j in range(n):
        eight = EIGHTS[j % len(EIGHTS)][1]
        w[j] = np.tile(np.roll(eight, j // len(EIGHTS)), k // 8)
    got = product(x, w, "fp8", out_dtype).double()
    tx, tw = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
    want = tx @ tw.t()  # (exact: multiples of 2^-10 below 2^15)
    if out_dtype == "float32":
        assert torch.equal(got, want)
        return
    largest = 448.0 * 6
    assert ((got - want).abs() <= UNIT[out_dtype] * (want.abs() + 2) + 7 * 2.0 ** -13 * largest).all()


@pytest.mark.parametrize("low,high", [(0, 72), (72, 127)])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_each_half_of_the_exponents_sums_exactly_into_fp32(m, n, k, low, high):
    """e4m3 codes of exponent fields 0..8 (multiples of 2^-9 up to 3.75) or 9..15 (of 1/2 up to 448) only:
    every partial sum is a multiple of 2^-10 below 2^14, or of 1/4 below 2^22, so fp32 holds it."""
    g = np.random.default_rng(m + n + k + low)
    x = mx.E4M3[g.integers(low, high, (m, k))] * g.choice([-1.0, 1.0], (m, k))
    x[:, 512 if low == 0 else 1536:] = 0  # 512 x 22.5 < 2^14, 1536 x 2688 < 2^22
    w = mx.E2M1[g.integers(0, 8, (n, k))] * g.choice([-1.0, 1.0], (n, k))
    got = product(x, w, "fp8", "float32")
    assert torch.equal(got.double(), torch.from_numpy(x).cuda() @ torch.from_numpy(w).cuda().t())


@pytest.mark.parametrize("m,n,k", SIZES)
def test_fp4_rows_sum_exactly_into_fp32(m, n, k):
    g = np.random.default_rng(m + n + k)
    x = mx.E2M1[g.integers(0, 8, (m, k))] * g.choice([-1.0, 1.0], (m, k))
    w = mx.E2M1[g.integers(0, 8, (n, k))] * g.choice([-1.0, 1.0], (n, k))
    got = product(x, w, "fp4", "float32")  # multiples of 1/4 below 36 x 4864 < 2^18
    assert torch.equal(got.double(), torch.from_numpy(x).cuda() @ torch.from_numpy(w).cuda().t())
