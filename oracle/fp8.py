"""The 8-bit floating point format, the root-mean-square norm and gradient clipping in float64 numpy, from their definitions (the
oracle of the HIP kernels; no reference implementation exists: parity unpinned)."""
import numpy as np

BLK = 128


def code_values():
    """Value of every e4m3 code: 1 sign, 4 exponent (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN, there are no infinities."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        a = np.nan if e == 15 and m == 7 else (1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6
        v[c] = -a if c & 128 else a
    return v


VALUES = code_values()
_POS = VALUES[:127]  # the codes 0x00 .. 0x7e, ascending


def encode(v):
    """Nearest code of |v| <= 448 (ties to the even code); anything that is not finite: NaN."""
    v = np.asarray(v, np.float64)
    a = np.where(np.isfinite(v), np.abs(v), 0.0)
    hi = np.clip(np.searchsorted(_POS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    c |= np.where(np.signbit(v), 128, 0).astype(np.uint8)
    return np.where(np.isfinite(v), c, np.uint8(0x7f))


def scale_exponent(amax):
    """Smallest e with amax <= 448 * 2^e, at least -126; 0 for amax = 0."""
    if amax == 0:
        return 0
    e = -126
    m, x = np.frexp(amax / 448.0)  # m in [1/2, 1)
    e = int(x) - (1 if m == 0.5 else 0)
    assert amax <= 448.0 * 2.0 ** e and amax > 448.0 * 2.0 ** (e - 1)
    return max(e, -126)


def quantize(x, block_rows=1):
    """-> (codes uint8 (rows, cols), exponents int (row blocks, column blocks))."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    codes = np.zeros((rows, cols), np.uint8)
    exps = np.zeros((-(-rows // block_rows), -(-cols // BLK)), np.int64)
    for i in range(exps.shape[0]):
        for j in range(exps.shape[1]):
            b = x[i * block_rows:(i + 1) * block_rows, j * BLK:(j + 1) * BLK]
            f = np.abs(b[np.isfinite(b)])
            e = scale_exponent(f.max() if f.size else 0.0)
            exps[i, j] = e
            codes[i * block_rows:(i + 1) * block_rows, j * BLK:(j + 1) * BLK] = encode(b / 2.0 ** e)
    return codes, exps


def values(codes, scales, block_rows=1):
    s = np.repeat(np.repeat(np.asarray(scales, np.float64), block_rows, 0)[:codes.shape[0]], BLK, 1)[:, :codes.shape[1]]
    return VALUES[codes] * s


def rms_norm(x, w, eps):
    x = np.asarray(x, np.float64)
    r = 1.0 / np.sqrt((x * x).mean(1, keepdims=True) + eps)
    return x * r * w, r[:, 0]


def rms_norm_grad(dy, h, w, eps, dh=None):
    dy, h = np.asarray(dy, np.float64), np.asarray(h, np.float64)
    _, r = rms_norm(h, w, eps)
    n = h * r[:, None]
    g = dy * w
    dx = r[:, None] * (g - n * (g * n).mean(1, keepdims=True))
    return (dx if dh is None else dx + dh), (dy * n).sum(0)


def grad_norm(gs):
    return np.sqrt(sum((np.asarray(g, np.float64) ** 2).sum() for g in gs))
