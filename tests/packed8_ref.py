"""Plain float64 forms of the 8-bit tensors and of the operators that use them (numpy)."""
import numpy as np


def strides(cols):
    """Bytes of codes and of scales of one packed row."""
    codes = -(-cols // 128) * 128
    return codes, -(-codes // 512) * 4


def nbytes(rows, cols):
    return rows * sum(strides(cols))


def code_values():
    """The value of each of the 256 e4m3 codes."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, np.ldexp(8.0 + m, e - 10), np.ldexp(m.astype(np.float64), -9))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


CODES = code_values()


def round_e4m3(v):
    """Nearest e4m3 value, ties to even, of values up to 448."""
    a = np.abs(v)
    e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0)
    e = np.where(a >= np.exp2(e + 1), e + 1, np.where((a < np.exp2(e)) & (e > -6), e - 1, e))
    step = np.exp2(e - 3)
    return np.rint(v / step) * step


def exponents(x):
    """Exponent of each block of 128 of x's rows [rows, blocks]."""
    rows, cols = x.shape
    blocks = -(-cols // 128)
    pad = np.zeros((rows, blocks * 128))
    pad[:, :cols] = np.where(np.isfinite(x), np.abs(x.astype(np.float64)), 0.0)
    top = pad.reshape(rows, blocks, 128).max(2)
    e = np.full(top.shape, -127)
    pos = top > 0
    f, k = np.frexp(top[pos])  # top = f 2^k, 1/2 <= f < 1; 448 = 0.875 * 2^9
    e[pos] = np.maximum(np.where(f > 0.875, k - 8, k - 9), -127)
    return e


def pack(x):
    """Values (float64, NaN where x is not finite) and exponents."""
    e = exponents(x)
    scale = np.exp2(np.repeat(e, 128, axis=1)[:, :x.shape[1]].astype(np.float64))
    with np.errstate(invalid="ignore"):
        v = np.where(np.isfinite(x), x.astype(np.float64) / scale, 0.0)
    return np.where(np.isfinite(x), round_e4m3(v) * scale, np.nan), e


def value(x):
    return pack(x)[0]


def decode(raw, rows, cols):
    """Values [rows, cols], codes [rows, S] and scale bytes [rows, T] of a packed tensor's bytes."""
    s, t = strides(cols)
    codes = raw[:rows * s].reshape(rows, s)
    scales = raw[rows * s:rows * (s + t)].reshape(rows, t)
    v = CODES[codes] * np.exp2(np.repeat(scales[:, :s // 128].astype(np.float64) - 127.0, 128, axis=1))
    return v[:, :cols], codes, scales


def encode(x):
    """The bytes of x packed."""
    rows, cols = x.shape
    s, t = strides(cols)
    v, e = pack(x)
    with np.errstate(invalid="ignore"):
        u = v / np.exp2(np.repeat(e, 128, axis=1)[:, :cols].astype(np.float64))
    order = {float(CODES[c]): c for c in range(127)}
    codes = np.zeros((rows, s), np.uint8)
    for r in range(rows):
        for c in range(cols):
            codes[r, c] = 0x7F if np.isnan(u[r, c]) else order[abs(float(u[r, c]))] | (128 if np.signbit(x[r, c]) else 0)
    scales = np.zeros((rows, t), np.uint8)
    scales[:, :e.shape[1]] = e + 127
    return np.concatenate([codes.reshape(-1), scales.reshape(-1)])


def _erf(x):
    from math import erf
    return np.vectorize(erf, otypes=[np.float64])(x)


def gelu(x):
    x = x.astype(np.float64)
    return 0.5 * x * (1.0 + _erf(x / np.sqrt(2.0)))


def gelu_slope(x):
    x = x.astype(np.float64)
    return 0.5 * (1.0 + _erf(x / np.sqrt(2.0))) + x * np.exp(-0.5 * x * x) / np.sqrt(2.0 * np.pi)


def layernorm(x, eps):
    """The normalised rows as the library defines them (float32 bits) and 1 / sigma in float32."""
    d = x.astype(np.float64)
    mean = d.mean(1, keepdims=True)
    rstd = (1.0 / np.sqrt(np.square(d - mean).mean(1, keepdims=True) + np.float64(np.float32(eps)))).astype(np.float32)
    return (x - mean.astype(np.float32)) * rstd, rstd


def layernorm_bwd(g, h, gamma, rstd):
    """dx, dgamma, dbeta from the kept rows' values h."""
    g = g.astype(np.float64)
    q = g * gamma.astype(np.float64)
    dx = rstd.astype(np.float64) * (q - q.mean(1, keepdims=True) - h * (q * h).mean(1, keepdims=True))
    return dx, (g * h).sum(0), g.sum(0)
