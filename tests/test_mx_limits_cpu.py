"""mx_linear's limits: the workspace's size and the product know the same ones. No GPU."""
import ctypes

import pytest

from dli import hip


def product(m, n, k):
    """The entry point's status for sizes (-1: refused). Called for refused sizes only: nothing runs."""
    fake = ctypes.c_void_p(256)
    return hip.load().dli_hip_mx_linear(hip.MX_FP8, hip.BF16, fake, fake, fake, fake, None, None, fake,
                                        m, n, k, None, 0, None)


@pytest.mark.parametrize("m,n,k", [
    (1 << 50, 1 << 50, 32),              # m n k past 63 bits
    ((1 << 39) + 1, (1 << 39) + 1, 64), (3 << 40, 5 << 41, 1024), ((1 << 35) - 7, 1 << 20, 4096),
    ((1 << 20) - 15, 1024, 4096),        # one row too many
    (1024, (1 << 29) + 1, 4096), (1024, 1024, (1 << 28) + 32), (64, 64, -32), (64, 64, 0),
    (-1, 64, 64), (64, -1, 64)])
def test_no_workspace_for_what_is_refused(m, n, k):
    assert product(m, n, k) == -1
    for form in (hip.MX_FP8, hip.MX_FP4):
        assert hip.load().dli_hip_mx_linear_workspace(form, m, n, k) == 0


def test_workspace_of_the_largest_products():
    """Scales of both operands in words, rows padded to 256; so many tiles take K in one part."""
    size = hip.load().dli_hip_mx_linear_workspace
    for m, n, k in (((1 << 20) - 16, 1024, 32768), (1024, 1 << 29, 4096), (4096, 1 << 20, 8192)):
        rows = (m + 255) // 256 * 256 + (n + 255) // 256 * 256
        assert size(hip.MX_FP8, m, n, k) == (k + 255) // 256 * 8 * rows
    assert size(hip.MX_FP8, 1024, 1024, 1 << 28) == 0  # offsets of a tile past 32 bits: the stream
    assert size(2, 1024, 1024, 4096) == 0              # no such format


@pytest.mark.parametrize("form", [hip.MX_FP8, hip.MX_FP4])
@pytest.mark.parametrize("n", [32769, 49152, 65536])
@pytest.mark.parametrize("k", [2048, 4096, 4224, 8192, 18944, 1 << 20])
def test_runs_of_columns_over_every_long_k(form, n, k):
    """17 to 64 rows of more tiles than CUs, fewer than two each: equal runs of columns, which read the
    scales as they are and sum no parts, so nothing is laid out, however long K is."""
    for m in (17, 64):
        assert hip.load().dli_hip_mx_linear_workspace(form, m, n, k) == 0


@pytest.mark.parametrize("m,n,k,large", [
    (257, 24576, 896, False), (2048, 9728, 896, False), (300, 37888, 3584, False),
    (1024, 18944, 3584, False), (1025, 9856, 3584, True), (768, 18944, 3584, True),
    (8192, 37888, 3584, True), (8192, 37888, 128, True), (4096, 3584, 3584, True), (2000, 3584, 18944, False)])
def test_large_tiles_by_their_rounds(m, n, k, large):
    """Large tiles read scales laid out in words; tiles of 128 read them as they are up to K = 4096."""
    size = hip.load().dli_hip_mx_linear_workspace(hip.MX_FP8, m, n, k)
    assert (size > 0) == (large or k > 4096)
