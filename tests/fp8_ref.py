"""Plain implementations of the 8-bit floating-point operators in 64 bits, on the CPU, from their definitions: e4m3 numbers
from their bits, a block's scale from a search over powers of two, products one block after another."""
import numpy as np
import torch

MOST = 448.0
EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def _table():
    t = np.zeros(256)
    for b in range(256):
        e, f = b >> 3 & 15, b & 7
        v = np.nan if (b & 127) == 127 else (1 + f / 8) * 2.0 ** (e - 7) if e else f / 8 * 2.0 ** -6
        t[b] = -v if b & 128 else v
    return t


TABLE = _table()
POSITIVE = TABLE[:127]  # rising


def values(q):
    """What e4m3 bytes stand for, in f64."""
    return TABLE[q.cpu().view(torch.uint8).numpy()]


def nearest(v):
    """Bytes of the e4m3 numbers next to v (f64, at most 448 in size; NaN: 127), ties to the even byte."""
    size = np.abs(v)
    bad = ~np.isfinite(v)
    size = np.where(bad, 0, size)
    hi = np.clip(np.searchsorted(POSITIVE, size), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = POSITIVE[hi] - size, size - POSITIVE[lo]
    b = np.where((up < down) | ((up == down) & (hi % 2 == 0)) | (lo == hi), hi, lo)
    return np.where(bad, 127, b | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def scale(size):
    """2^e, the least e >= -126 with size <= 448 * 2^e; 1 for 0 (f64 array of largest sizes)."""
    out = np.ones_like(size)
    for at in np.ndindex(size.shape):
        if size[at] > 0:
            e = -126
            while size[at] > MOST * 2.0 ** e:
                e += 1
            out[at] = 2.0 ** e
    return out


def largest(x):
    return np.where(np.isfinite(x), np.abs(x), 0)


def quantize(x):
    """Bytes and scales of rows x (f64)."""
    rows, k = x.shape
    kb = -(-k // 128)
    pad = np.zeros((rows, kb * 128))
    pad[:, :k] = x
    s = scale(largest(pad).reshape(rows, kb, 128).max(2))
    return nearest(x / np.repeat(s, 128, 1)[:, :k]), s


def spread(s, n, k):
    """Scales of blocks of 128 x 128 at each place of [n, k]."""
    return np.repeat(np.repeat(s, 128, 0)[:n], 128, 1)[:, :k]


def product(x, sx, w, sw, dtype, groups8):
    """Rows x (f64 values of e4m3) with scales sx [rows, blocks], weight w [n, k] with scales sw: the product in f64, and how
    far it may be off.  A block's products (exact: 8 bits each) are added in f32 in fewer than 128 steps, each of which
    rounds or cuts at 2^-23 of what is there at most; the scales' product and the step that adds the block round once each,
    the parts of up to 8 waves are added once more; then y is rounded.  groups8: groups of eight products are added with
    each cut at 2^-13 of the largest's power of two.  F16 has steps of 2^-24 below 2^-14, so a y there is up to 2^-25 off."""
    (m, k), n = x.shape, w.shape[0]
    y, size, cut = np.zeros((m, n)), np.zeros((m, n)), np.zeros((m, n))
    for b in range(sx.shape[1]):
        a, c = x[:, 128 * b:128 * b + 128], w[:, 128 * b:128 * b + 128]
        f = sx[:, b:b + 1] * np.repeat(sw[:, b], 128)[:n][None]
        y += a @ c.T * f
        size += np.abs(a) @ np.abs(c).T * np.abs(f)
        if groups8:
            # eight products of at most the block's largest each, sixteen groups
            cut += 16 * 8 * 2.0 ** -13 * np.abs(a).max(1)[:, None] * np.abs(c).max(1)[None] * np.abs(f)
    steps = 128 + sx.shape[1] + 8 + 3
    return y, steps * 2.0 ** -23 * size + cut + EPS[dtype] * np.abs(y) + (2.0 ** -25 if dtype is torch.float16 else 2.0 ** -126)
