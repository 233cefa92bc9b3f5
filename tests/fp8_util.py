"""The 8-bit floating point format restated in numpy float64: e4m3 values, the
scale rule, the packed scale layout (include/u15c.h), and bounds for what the
kernels may be off by."""
import numpy as np

# value of every e4m3 code: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7F / 0xFF NaN
_c = np.arange(256)
_e, _m = (_c >> 3) & 15, _c & 7
E4M3 = np.where(_e == 0, _m * 2.0 ** -9, (1 + _m / 8) * 2.0 ** (_e - 7.0)) * np.where(_c > 127, -1, 1)
E4M3[(_c & 127) == 127] = np.nan


def codes(v):
    """Nearest e4m3 code, ties to even, of finite |v| <= 448; NaN -> 0x7F."""
    a = np.abs(np.asarray(v, np.float64))
    nan = np.isnan(a)
    a = np.where(nan, 0, a)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6) - 3)
    r = np.rint(a / step) * step
    c = np.searchsorted(E4M3[:127], r).astype(np.uint8)
    assert np.array_equal(E4M3[c], r)
    return np.where(nan, 0x7F, c | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def scale_byte(amax):
    """Smallest s >= 0 with amax <= 448 * 2^(s - 127)."""
    m, e = np.frexp(np.asarray(amax, np.float64))      # amax = m 2^e; 448 = 0.875 * 2^9
    s = e - 9 + (m > 0.875) + 127
    return np.where(np.asarray(amax) == 0, 0, np.maximum(s, 0)).astype(np.int64)


def block_amax(v, tall=1):
    r, c = v.shape
    p = np.pad(np.abs(v), ((0, -r % tall), (0, -c % 128)))
    a = p.reshape(p.shape[0] // tall, tall, -1, 128).max((1, 3))
    return np.repeat(a, tall, 0)[:r]


def quantise(v, tall=1):
    """(codes [r][c], scale bytes [r][blocks]) of finite float64 v."""
    s = scale_byte(block_amax(v, tall))
    f = np.repeat(2.0 ** (127.0 - s), 128, 1)[:, :v.shape[1]]
    return codes(v * f), s


def places(rows, cols):
    r, b = np.arange(rows)[:, None], np.arange(-(-cols // 128))[None]
    return ((r // 128) * -(-cols // 512) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def scale_bytes(rows, cols):
    return -(-rows // 128) * -(-cols // 512) * 512


def pack(s, cols, fill=0xFF):
    p = np.full(scale_bytes(s.shape[0], cols), fill, np.uint8)
    p[places(s.shape[0], cols)] = s
    return p


def unpack(p, rows, cols):
    return p[places(rows, cols)].astype(np.int64)


def values(q, s):
    f = np.repeat(2.0 ** (s.astype(np.float64) - 127), 128, 1)[:, :q.shape[1]]
    return E4M3[q] * f


def half_step(y, s):
    """Half an e4m3 step at y in a block of scale byte s, per element of y."""
    f = np.repeat(2.0 ** (s.astype(np.float64) - 127), 128, 1)[:, :y.shape[1]]
    return np.maximum(np.abs(y) * 2.0 ** -4, f * 2.0 ** -10)


def product(xq, xs, wq, ws):
    """(y, S): the exact product and the sum of its terms' magnitudes."""
    x, w = values(xq, xs), values(wq, ws)
    return x @ w.T, np.abs(x) @ np.abs(w).T


def sum_error(S, K):
    """An f32 sum over K terms in steps of 32: every step rounds once (2^-23 of
    the magnitudes so far, truncation allowed for), and a step's own 32 terms
    are added at 24 bits."""
    return (K / 32 + 32) * 2.0 ** -23 * S
