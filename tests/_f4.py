"""Plain 64-bit forms of the 4-bit operators, written from the definitions in include/bm_igemm.h."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1])
E8M0, E4M3_FMT = 0, 1
BLOCK = {E8M0: 32, E4M3_FMT: 16}


def nearest(v, grid):
    """Index of the nearest grid point, of two equally near ones the even index; beyond the last: the last."""
    hi = np.clip(np.searchsorted(grid, v), 1, len(grid) - 1)
    down, up = v - grid[hi - 1], grid[hi] - v
    return np.where((down < up) | ((down == up) & (hi % 2 == 1)), hi - 1, hi)


def floor_log2(v):
    return np.frexp(v)[1] - 1


def quantize(x, fmt):
    """(codes 0..15 [R, K padded], scale bytes [R, blocks], row factors or None) of a matrix of any float type."""
    x = np.asarray(x, np.float64)
    R, K = x.shape
    x = np.pad(x, ((0, 0), (0, -K % 32))).reshape(R, -1, BLOCK[fmt])
    good = np.isfinite(x)
    bad = ~good.all(-1)
    a = np.where(good, np.abs(x), 0.0)
    amax = a.max(-1)
    if fmt == E8M0:
        byte = np.where(amax > 0, np.clip(floor_log2(amax) - 2 + 127, 0, 254), 0)
        s, t = np.exp2(byte - 127.0), None
        byte = np.where(bad, 255, byte)
    else:
        top = amax.max(-1)
        t = np.where(top > 0, np.exp2(np.maximum(floor_log2(top) - 10.0, -126.0)), 1.0)
        byte = nearest(amax / (6 * t[:, None]), E4M3)
        s = E4M3[byte] * t[:, None]
        byte = np.where(bad, 127, byte)
    v = np.where(s[..., None] > 0, a / np.where(s > 0, s, 1.0)[..., None], 0.0)
    code = nearest(v, GRID) | np.where(np.signbit(x), 8, 0)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(R, -1).astype(np.uint8), byte.astype(np.uint8), t


def values(code, byte, t, fmt):
    """What codes and scales stand for, in 64 bits."""
    s = np.where(byte == 255, np.nan, np.exp2(byte - 127.0)) if fmt == E8M0 else np.where(byte == 127, np.nan, np.append(E4M3, np.nan)[byte])
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    v = v.reshape(*byte.shape, -1) * s[..., None]
    v = v.reshape(code.shape)
    return v if t is None else v * np.asarray(t, np.float64)[:, None]


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def unpack(q):
    return np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)


def in_rows(byte):
    return np.pad(byte, ((0, 0), (0, -byte.shape[1] % 16)))


def tiled(byte):
    R, G = byte.shape
    tk = -(-G // 4)
    out = np.zeros(-(-R // 128) * tk * 512, np.uint8)
    r, g = np.meshgrid(np.arange(R), np.arange(G), indexing="ij")
    out[((r // 128) * tk + g // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + g % 4] = byte
    return out
