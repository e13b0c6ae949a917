"""Microscaled 4-bit floating point and the row step between two blocks, restated in 64 bits with numpy.

Codes are E2M1, eight per uint32 along K, lowest bits first; block scales are bytes, E8M0 (blocks of 32) or E4M3 (blocks of 16), in
tiles of 128 rows x 4 blocks (include/lux_cuda_quant.h).  Test infrastructure only.
"""
import numpy as np

E8M0, E4M3 = 1, 2
BLOCK = {E8M0: 32, E4M3: 16}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
VALUES = np.concatenate([GRID, -GRID])


def _e4m3_table():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10), m * 2.0 ** -9) * np.where(b & 128, -1.0, 1.0)
    v[(b & 127) == 127] = np.nan
    return v


E4M3_VALUES = _e4m3_table()
E8M0_VALUES = np.where(np.arange(256) == 255, np.nan, 2.0 ** (np.arange(256) - 127.0))


def scale_values(byte, fmt):
    return (E8M0_VALUES if fmt == E8M0 else E4M3_VALUES)[byte]


def _nearest(a, grid):
    """Index of the nearest point of an ascending grid, from halfway the even index."""
    i = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo, hi = a - grid[i - 1], grid[i] - a
    return np.where((lo < hi) | ((lo == hi) & ((i - 1) % 2 == 0)), i - 1, i)


def quantize(w, fmt, pre=1.0):
    """(codes [rows, K], scale bytes [rows, blocks]) of w [rows, K] (float32)."""
    rows, K = w.shape
    with np.errstate(over="ignore", invalid="ignore"):
        u = (w.astype(np.float32) * np.float32(pre)).astype(np.float64).reshape(rows, -1, BLOCK[fmt])
    m = np.abs(u).max(-1)
    nan = np.isnan(m)
    m = np.where(nan, 0, m)
    big = float(np.finfo(np.float32).max)
    if fmt == E8M0:
        e = np.frexp(np.minimum(m, big))[1] - 1  # floor(log2)
        byte = np.where(m > 0, np.maximum(e - 2 + 127, 0), 0)
    else:
        q = (np.minimum(m, big).astype(np.float32) / np.float32(6)).astype(np.float64)
        byte = _nearest(np.minimum(q, 448.0), E4M3_VALUES[:127])
    s = scale_values(byte, fmt)[..., None]
    with np.errstate(invalid="ignore", divide="ignore"):
        a = np.where(s > 0, np.minimum(np.abs(np.nan_to_num(u, nan=0.0, posinf=np.inf, neginf=-np.inf)) / np.where(s > 0, s, 1), 6.0), 0.0)
    code = _nearest(a, GRID) + 8 * (u < 0)
    byte = np.where(nan, 255 if fmt == E8M0 else 127, byte)
    return code.reshape(rows, K).astype(np.uint8), byte.astype(np.uint8)


def values(code, byte, fmt):
    """What codes [rows, K] and scale bytes stand for, in 64 bits."""
    rows, K = code.shape
    return (VALUES[code].reshape(rows, -1, BLOCK[fmt]) * scale_values(byte, fmt)[..., None]).reshape(rows, K)


def pack(code):
    c = code.reshape(code.shape[0], -1, 8).astype(np.uint32)
    return np.bitwise_or.reduce(c << (4 * np.arange(8, dtype=np.uint32)), axis=-1).astype(np.uint32)


def unpack(words):
    return ((words[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(words.shape[0], -1).astype(np.uint8)


def tile_index(rows, blocks):
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    return ((r // 128) * ((blocks + 3) // 4) + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4


def scale_bytes(rows, K, fmt):
    return (rows + 127) // 128 * ((K // BLOCK[fmt] + 3) // 4) * 512


def to_tiles(byte, fill=0):
    """Scale bytes [rows, blocks] in their tiles; `fill` for the rows behind the last (blocks behind the last are zero)."""
    rows, nb = byte.shape
    nt, full = (nb + 3) // 4, (rows + 127) // 128 * 128
    t = np.zeros(full * nt * 4, np.uint8)
    every = np.zeros((full, nt * 4), np.uint8)
    every[rows:] = fill
    every[:rows, :nb] = byte
    t[tile_index(full, nt * 4)] = every
    return t


def from_tiles(tiles, rows, blocks):
    return tiles[tile_index(rows, blocks)]


def random_operand(rng, rows, K, fmt, spread=3):
    """Codes over their whole range, scales over a few binades around one."""
    code = rng.integers(0, 16, (rows, K)).astype(np.uint8)
    nb = K // BLOCK[fmt]
    byte = rng.integers(127 - spread, 128 + spread, (rows, nb)) if fmt == E8M0 else rng.integers(40, 72, (rows, nb))
    return code, byte.astype(np.uint8)


# ---- the row step between two blocks ------------------------------------------------------------------------------------
def norm(v, kind, eps, w=None, b=None):
    """kind 0: as it is, 1: rms, 2: layer; in 64 bits."""
    v = v.astype(np.float64)
    if kind == 0:
        return v
    if kind == 2:
        v = v - v.mean(-1, keepdims=True)
    v = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    v = v if w is None else v * w.astype(np.float64)
    return v if b is None else v + b.astype(np.float64)


def gate(g, act):
    g = g.astype(np.float64)
    return 1 / (1 + np.exp(-g)) if act == 1 else np.tanh(g) if act == 2 else g
