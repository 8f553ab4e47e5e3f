"""The microscaled 4-bit format in plain numpy, 64 bits: what the tests hold the kernels to."""
import numpy as np

NUMBERS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])


def quantize(x):
    """float32 [rows, cols] -> (codes uint8 [rows, 32 * blocks], scale bytes uint8 [rows, blocks])"""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    blocks = -(-cols // 32)
    b = np.zeros((rows, blocks * 32), np.float64)
    b[:, :cols] = x
    b = b.reshape(rows, blocks, 32)
    bad = ~np.isfinite(b).all(2)
    top = np.where(bad, 1.0, np.abs(b).max(2, initial=0))
    with np.errstate(divide="ignore"):
        _, e = np.frexp(top)  # top = m * 2^e, 0.5 <= m < 1
    e = np.where(top == 0, -127, np.maximum(e - 3, -127))
    a = np.abs(np.where(bad[:, :, None], 0.0, b)) / np.exp2(e.astype(np.float64))[:, :, None]
    dist = np.abs(a[..., None] - NUMBERS[:8])
    near = dist.min(-1, keepdims=True) == dist
    # of two equally near ones the even code
    code = np.where(near & (np.arange(8) % 2 == 0), np.arange(8), -1).max(-1)
    code = np.where(code < 0, np.where(near, np.arange(8), -1).max(-1), code)
    code = np.where(near.sum(-1) == 1, np.where(near, np.arange(8), 0).sum(-1), code)
    code = code + 8 * np.signbit(b)
    code = np.where(bad[:, :, None], 0, code)
    return code.reshape(rows, -1).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def pack(codes):
    return codes[:, 0::2] | codes[:, 1::2] << 4


def tiles(scale_bytes):
    """scale bytes [rows, blocks] -> uint8 [row tiles, block tiles, 512], byte by byte from the layout's formula"""
    rows, blocks = scale_bytes.shape
    out = np.zeros((-(-rows // 128), -(-blocks // 4), 512), np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = scale_bytes
    return out


def values(codes, scale_bytes):
    """The numbers, float64 [rows, 32 * blocks]."""
    s = np.where(scale_bytes == 255, np.nan, np.exp2(scale_bytes.astype(np.float64) - 127))
    return NUMBERS[codes] * np.repeat(s, 32, axis=1)
