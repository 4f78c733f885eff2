"""Microscaled tensors in float64 (numpy), written from the format's definition: blocks of 32
values, scale 2^(code - 127) with code the largest magnitude's biased exponent less 8 (e4m3) or 2
(e2m1), elements rounded to the nearest of the type's values, ties to the even code."""
import numpy as np

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
# every finite e4m3 magnitude by code: 4 exponent bits (bias 7), 3 of mantissa, code 127 is NaN
E4M3 = np.array([(c % 8) / 8 * 2.0 ** -6 if c < 8 else (1 + (c % 8) / 8) * 2.0 ** (c // 8 - 7)
                 for c in range(127)])
VALUES = {"fp4": E2M1, "fp8": E4M3}
TOP = {"fp4": 2, "fp8": 8}


def nearest(a, values):
    """Codes of the nearest of the ascending `values` to magnitudes a, ties to the even code."""
    hi = np.clip(np.searchsorted(values, a), 1, len(values) - 1)
    lo = hi - 1
    down, up = a - values[lo], values[hi] - a
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.where(a >= values[-1], len(values) - 1, code)


def quantize(y, form):
    """float64 y [.., K] -> codes and scales as uint8 arrays."""
    y = np.asarray(y, np.float64)
    blocks = y.reshape(-1, 32)
    amax = np.abs(blocks).max(1)
    good = np.isfinite(blocks).all(1)
    safe = np.where(good & (amax > 0), amax, 1.0)
    code = np.floor(np.log2(safe)).astype(int)
    code += (2.0 ** (code + 1.0) <= safe).astype(int) - (2.0 ** code.astype(float) > safe)
    code = np.where(amax > 0, code + 127 - TOP[form], 0).clip(0)
    code = np.where(good, code, 255)
    with np.errstate(invalid="ignore"):
        v = np.where(good[:, None], blocks, 0) / 2.0 ** (np.where(good, code, 127) - 127.0)[:, None]
    e = nearest(np.abs(v), VALUES[form])
    sign = np.signbit(v) & good[:, None]
    if form == "fp8":
        codes = (e + 128 * sign).reshape(y.shape)
    else:
        e = (e + 8 * sign).reshape(-1, 2)
        codes = (e[:, 0] + 16 * e[:, 1]).reshape(y.shape[:-1] + (y.shape[-1] // 2,))
    return codes.astype(np.uint8), code.reshape(y.shape[:-1] + (-1,)).astype(np.uint8)


def values(codes, scales):
    """What codes and scales (uint8 arrays) stand for, in float64."""
    c = codes.astype(int)
    if codes.shape[-1] == scales.shape[-1] * 32:
        e = np.append(E4M3, np.nan)[c % 128] * np.where(c >= 128, -1.0, 1.0)
    else:
        c = np.stack([c % 16, c // 16], -1)
        e = E2M1[c % 8] * np.where(c >= 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(float) - 127))
    return (e.reshape(-1, 32) * s.reshape(-1, 1)).reshape(scales.shape[:-1] + (-1,))


def rms_norm32(h, weight, eps):
    """The operator's own 32-bit steps on h (float32 array of the kept values): the root of the
    mean square in 64 bits, rounded, then two products."""
    inv = (1.0 / np.sqrt((h.astype(np.float64) ** 2).mean(-1, keepdims=True)
                         + np.float64(np.float32(eps)))).astype(np.float32)
    return h * inv * weight.astype(np.float32)
