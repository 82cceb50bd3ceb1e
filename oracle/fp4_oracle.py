"""The 4-bit cache format in float64 (numpy): quantisation by search over all scales and values, the page layout byte by byte, and
attention over the values a cache stands for."""
import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# byte b stands for the half-precision number with bit pattern b << 7; usable up to 10240
SCALES = (np.arange(256, dtype=np.uint16) << 7).view(np.float16).astype(np.float64)
TOP_BYTE = int(np.argmax(np.where(np.isfinite(SCALES[:248]), SCALES[:248], 0) == 10240.0))


def _nearest(x, grid):
    """Index of the nearest value of the ascending grid; of two equally near the even index."""
    x = np.asarray(x, np.float64)
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    lo = hi - 1
    below, above = np.abs(x - grid[lo]), np.abs(grid[hi] - x)
    pick_hi = (above < below) | ((above == below) & (hi % 2 == 0))
    out = np.where(pick_hi, hi, lo)
    return np.where(x >= grid[-1], len(grid) - 1, out)


def quantise(x):
    """x [..., D] -> (codes [..., D] 0..15, scale bytes [..., D / 16])."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    finite = np.isfinite(b).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1), 0.0)
    byte = _nearest(top / 6.0, SCALES[:TOP_BYTE + 1])
    s = SCALES[byte]
    y = np.where((s > 0) & finite, 1.0, 0.0)[..., None] * np.abs(np.where(np.isfinite(b), b, 0.0)) / np.where(s > 0, s, 1.0)[..., None]
    code = _nearest(np.minimum(y, 6.0), VALUES)
    negative = (b < 0) & ((s > 0) & finite)[..., None]      # a negative zero is a zero
    return (code + 8 * negative).reshape(x.shape).astype(np.uint8), np.where(finite, byte, 255).astype(np.uint8)


def values(codes):
    v = VALUES[codes & 7]
    return np.where(codes & 8, -v, v)


def dequantise(codes, scale_bytes):
    return values(codes) * np.repeat(SCALES[scale_bytes], 16, axis=-1)


def roundtrip(x):
    return dequantise(*quantise(x))


def pack_head(codes, scale_bytes, rows_of_page):
    """Bytes of one head's region of a page with `rows_of_page` rows: codes [rows_of_page, D], scale bytes [rows_of_page, D / 16]."""
    D = codes.shape[1]
    out = []
    for r0 in range(0, rows_of_page, 128):
        n = min(128, rows_of_page - r0)
        padded = n if n == 128 else -(-n // 4) * 4
        c = np.zeros((padded, D), np.uint8)
        s = np.zeros((padded, D // 16), np.uint8)
        c[:n], s[:n] = codes[r0:r0 + n], scale_bytes[r0:r0 + n]
        out += [(c[:, 0::2] | (c[:, 1::2] << 4)).reshape(-1), s.reshape(-1)]
    return np.concatenate(out)


def attention(q, k, v):
    """q [n, H, D], k and v [t, H, D] float64 -> (out [n, H, D], natural log-sum-exp [n, H], sum of weight * |v| [n, H, D])."""
    s = np.einsum("nhd,thd->hnt", q, k) / np.sqrt(q.shape[-1])
    top = s.max(axis=-1, keepdims=True)
    p = np.exp(s - top)
    total = p.sum(axis=-1, keepdims=True)
    p /= total
    lse = (top + np.log(total))[..., 0].T
    return np.einsum("hnt,thd->nhd", p, v), lse, np.einsum("hnt,thd->nhd", p, np.abs(v))
