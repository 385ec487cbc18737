"""The 8-bit operators in 64 bits (numpy), from their definition: the e4m3 grid by enumeration of its
256 codes, a block's scale by the definition of E, the linear layer in float64."""
import numpy as np


def e4m3_table():
    """The value of every code: sign, 4 exponent bits (bias 7), 3 fraction bits; codes 0x7F / 0xFF are NaN."""
    t = np.empty(256)
    for c in range(256):
        s, e, f = c >> 7, (c >> 3) & 15, c & 7
        v = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        t[c] = np.nan if (c & 127) == 127 else (-v if s else v)
    return t


TABLE = e4m3_table()
_POS = TABLE[:127]  # codes 0 .. 126 ascend


def e4m3_code(v):
    """Nearest code, ties to the even code, of finite v with |v| <= 448 (adjacent codes of one sign differ by one)."""
    a = np.abs(v)
    hi = np.searchsorted(_POS, a)  # first code >= a
    hi = np.minimum(hi, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(_POS[hi] == a, hi, c)
    return (c | (np.signbit(v).astype(np.int64) << 7)).astype(np.uint8)


def block_exp(amax):
    """Smallest integer E >= 0 with amax <= 448 * 2^(E - 127)."""
    e = 0
    while amax > 448.0 * 2.0 ** (e - 127):
        e += 1
    return e


def quantize(x, block_rows=1):
    """x [rows, k] float64 -> (codes [rows, k], E [ceil(rows / block_rows), ceil(k / 128)])."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    code = np.zeros((rows, k), np.uint8)
    E = np.zeros((-(-rows // block_rows), -(-k // 128)), np.uint8)
    for i in range(E.shape[0]):
        for b in range(E.shape[1]):
            s = np.s_[i * block_rows:(i + 1) * block_rows, b * 128:(b + 1) * 128]
            blk = x[s]
            fin = np.isfinite(blk)
            E[i, b] = block_exp(np.abs(blk[fin]).max() if fin.any() else 0.0)
            v = np.where(fin, blk, 0.0) * 2.0 ** (127.0 - E[i, b])
            code[s] = np.where(fin, e4m3_code(v), 127)
    return code, E


def dequantize(code, E, block_rows=1):
    s = np.repeat(np.repeat(2.0 ** (E.astype(np.float64) - 127.0), block_rows, 0), 128, 1)
    return TABLE[code] * s[:code.shape[0], :code.shape[1]]


def gelu(v):
    return 0.5 * v * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (v + 0.044715 * v ** 3)))


def linear(x, w, bias=None, act=None, residual=None):
    """(y, S): the result, and the sum of the magnitudes that were added to make each element."""
    with np.errstate(invalid="ignore", over="ignore"):
        y, S = x @ w.T, np.abs(x) @ np.abs(w).T
        if bias is not None:
            y, S = y + bias, S + np.abs(bias)
        if act == "gelu":
            y = gelu(y)
        if residual is not None:
            y, S = y + residual, S + np.abs(residual)
    return y, S
