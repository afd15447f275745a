"""The 4-bit cache format restated in numpy: 4-bit floats (sign, 2 bits of exponent, 1 of mantissa), 32 to a power-of-two
scale. Test infrastructure."""

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def width(d):
    return (d + 31) // 32 * 32


def scales_of(x):
    """The scale byte of each group of x (..., groups, 32) float64: the smallest power of two 2^e with max|x| < 7 2^e, e in
    [-125, 125]; 255 for a group with a NaN, an infinity or a value past fp32's."""
    a = np.abs(x).max(-1)
    bad = ~(a < 2.0 ** 128)
    m, e = np.frexp(np.where(bad, 1.0, a))
    e = np.where(m < 0.875, e - 3, e - 2)
    e = np.where(a == 0, -125, np.clip(e, -125, 125))
    return np.where(bad, 255, e + 127).astype(np.uint8)


def steps(x, scales):
    """x in units of its scale (0 in groups without one)."""
    s = scales.astype(np.int64)[..., None] - 127
    return np.where(s == 128, 0.0, np.ldexp(np.where(np.isfinite(x), x, 0.0), -s))


def codes_of(t):
    """The codes of t, in units of the scale: the nearest level, ties to the even code, the largest beyond it."""
    a = np.abs(t)
    c = ((a > 0.25).astype(np.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return c | (np.signbit(t) << 3).astype(np.uint8)


def pack(codes):
    """(..., d) codes to bytes, element 2 i in the low half."""
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def quantize(x):
    """x (..., d) float64 to (bytes (..., width / 2), scales (..., width / 32)), zeros behind d."""
    d = x.shape[-1]
    x = np.concatenate([x, np.zeros(x.shape[:-1] + (width(d) - d,))], -1)
    g = x.reshape(x.shape[:-1] + (-1, 32))
    s = scales_of(g)
    return pack(codes_of(steps(g, s)).reshape(x.shape)), s


def values(codes, scales, d):
    """The float64 values of bytes and scales (infinities where fp32 has no such number, NaN for 255)."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1,))
    y = np.where(c & 8, -1.0, 1.0) * LEVELS[c & 7]
    s = np.repeat(scales.astype(np.int64), 32, -1) - 127
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.ldexp(y, np.minimum(s, 127))
        x = np.where(np.abs(x) >= 2.0 ** 128, np.sign(x) * np.inf, x)
        x = np.where(s == 128, np.nan, x)
    return x[..., :d]


def random_pool(rng, pages, heads, P, d, lo=-6, hi=6):
    """(k codes, k scales, v codes, v scales): every code as likely, scales 2^lo .. 2^hi; behind d codes of anything."""
    out = []
    for _ in range(2):
        out += [rng.integers(0, 256, (pages, heads, P, width(d) // 2), dtype=np.uint8),
                rng.integers(127 + lo, 128 + hi, (pages, heads, P, width(d) // 32), dtype=np.uint8)]
    return out


def as_bf16(x):
    """float64 values that are bf16 numbers, as bits."""
    f = x.astype(np.float32)
    assert np.array_equal(f.astype(np.float64), x, equal_nan=True)
    b = np.ascontiguousarray(f).view(np.uint32)
    assert not np.any(b[np.isfinite(x)] & 0xFFFF)
    return (b >> 16).astype(np.uint16)
