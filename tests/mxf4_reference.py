"""Microscaled 4-bit floating point and rotary positions in numpy, in 64 bits, from their definitions."""
import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """[rows, cols] -> codes [rows, 16 * blocks], scale bytes [rows, blocks]."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32), np.float64)
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    finite = np.isfinite(v).all(-1)
    v = np.where(finite[..., None], v, 0.0)
    largest = np.abs(v).max(-1)
    exponent = np.where(largest > 0, np.frexp(np.where(largest > 0, largest, 1.0))[1] - 1 - 2, -127)
    exponent = np.maximum(exponent, -127)
    scaled = np.ldexp(v, -exponent[..., None])
    # nearest of the eight magnitudes; of two equally near ones the even code
    distance = np.abs(np.abs(scaled)[..., None] - VALUES) * 2 + (np.arange(8) % 2) * 1e-9
    code = distance.argmin(-1).astype(np.uint8)
    code[np.abs(scaled) >= 6] = 7
    code |= np.where(np.signbit(scaled), 8, 0).astype(np.uint8)
    code[~finite] = 0
    code = code.reshape(rows, blocks * 16, 2)
    return code[..., 0] | (code[..., 1] << 4), np.where(finite, exponent + 127, 255).astype(np.uint8)


def tile_scales(scales):
    """[rows, blocks] -> [row tiles, block tiles, 512]."""
    rows, blocks = scales.shape
    out = np.zeros((-(-rows // 128), -(-blocks // 4), 512), np.uint8)
    for r in range(rows):
        for b in range(blocks):
            out[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = scales[r, b]
    return out


def untile_scales(tiles, rows, blocks):
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None]
    return tiles[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4]


def values(codes, tiles):
    """The values that codes and tiled scales stand for, [rows, 32 * blocks]."""
    rows, blocks = codes.shape[0], codes.shape[1] // 16
    nibbles = np.stack((codes & 15, codes >> 4), -1).reshape(rows, blocks, 32)
    scales = untile_scales(tiles, rows, blocks)
    v = np.where(nibbles & 8, -1.0, 1.0) * VALUES[nibbles & 7] * np.ldexp(1.0, scales.astype(int) - 127)[..., None]
    return np.where((scales == 255)[..., None], np.nan, v).reshape(rows, blocks * 32)


def gelu(x):
    from scipy.special import erf
    return 0.5 * x * (1.0 + erf(x / np.sqrt(2.0)))


def rotary(x, positions, frequencies, interleaved=False, backward=False, magnitude=1.0):
    """x [bs, seq, heads, d], positions [bs, seq] or None."""
    x = x.astype(np.float64)
    half = len(frequencies)
    if positions is None:
        positions = np.broadcast_to(np.arange(x.shape[1]), x.shape[:2])
    angle = np.asarray(positions, np.float64)[..., None] * frequencies
    turn = magnitude * np.exp((-1j if backward else 1j) * angle)[:, :, None]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(half), slice(half, 2 * half))
    y = x.copy()
    z = (x[..., first] + 1j * x[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def rotary_tolerance(x, want, frequencies, interleaved, magnitude, eps):
    """An angle is off by at most 2.5e-7 radians (half a step of an fp32 fraction of a turn, and the sine's and the
    cosine's own errors of a step each), each product and the sum by half a step, the result by half a step of its type."""
    half = len(frequencies)
    pair = np.zeros_like(want)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(half), slice(half, 2 * half))
    size = abs(magnitude) * (np.abs(x[..., first].astype(np.float64)) + np.abs(x[..., second].astype(np.float64)))
    pair[..., first] = pair[..., second] = size
    # the smallest fp16 step, 2^-24, where results underflow
    return pair * (2.5e-7 + 4 * 2.0 ** -24) + np.abs(want) * eps / 2 + (2.0 ** -25 if eps > 1e-5 else 0.0)
