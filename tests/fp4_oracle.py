"""The 4-bit formats in 64 bits, from their definitions, for the tests of the kernels."""

from __future__ import annotations

import numpy as np
import torch

BLOCK = {"mx": 32, "nv": 16}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()


def nearest(grid: np.ndarray, v: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest to v >= 0, ties to the even index, clamped at the top."""
    mid = (grid[1:] + grid[:-1]) / 2
    i = np.searchsorted(mid, v, side="left")  # number of midpoints below v
    tie = (i < len(mid)) & (mid[np.minimum(i, len(mid) - 1)] == v)
    return np.where(tie & (i % 2 == 1), i + 1, i)


def quantize(x: np.ndarray, fmt: str, g: np.ndarray | float = 1.0):
    """Codes [R, K] and scale bytes [R, K/n] of x (float64 holding the inputs exactly); g: the
    factor, a number or one for each row."""
    n = BLOCK[fmt]
    R, K = x.shape
    v = x.reshape(R, K // n, n)
    g = np.broadcast_to(np.asarray(g, dtype=np.float64).reshape(-1, 1), (R, 1))
    with np.errstate(all="ignore"):
        top = np.abs(v).max(-1)
        bad = ~np.isfinite(v).all(-1)
        top = np.where(bad, 0.0, top)
        if fmt == "mx":
            byte = np.where(top > 0, np.clip(np.frexp(top)[1] - 1 - 2 + 127, 0, 254), 0)
            scale = np.ldexp(1.0, byte.astype(int) - 127)
            byte = np.where(bad, 255, byte)
        else:
            byte = nearest(E4M3, top / (6.0 * g))
            scale = E4M3[byte] * g
            byte = np.where(bad, 127, byte)
        a = np.where(scale[..., None] > 0, np.abs(v) / np.where(scale > 0, scale, 1.0)[..., None], 0.0)
        a = np.where(bad[..., None], 0.0, a)
    code = nearest(E2M1, a) | np.where(np.signbit(v), 8, 0)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(R, K).astype(np.uint8), byte.astype(np.uint8)


def values(code: np.ndarray, byte: np.ndarray, fmt: str, g=1.0) -> np.ndarray:
    """float64 values of codes [..., K] and scale bytes [..., K/n]; g broadcasts over the bytes."""
    n = BLOCK[fmt]
    if fmt == "mx":
        s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(int) - 127))
    else:
        s = np.where(byte == 127, np.nan, E4M3[np.minimum(byte, 126)]) * g
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    return (v.reshape(*byte.shape, n) * s[..., None]).reshape(code.shape)


def pack(code: np.ndarray) -> np.ndarray:
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def unpack(q: np.ndarray) -> np.ndarray:
    return np.stack((q & 15, q >> 4), -1).reshape(*q.shape[:-1], 2 * q.shape[-1])


def scale_positions(fmt: str, rows: int, K: int, tile: int):
    """Byte index of every scale [rows, K/n] in the tiled layout."""
    n, cells = BLOCK[fmt], 256 // BLOCK[fmt] // 4
    atoms = max(1, tile // 128)
    per_tile = -(-K // 256) * cells * atoms * 512
    p = np.arange(rows)[:, None]
    j = np.arange(K // n)[None, :]
    r = p % tile
    return ((p // tile) * per_tile + ((j // 4) * atoms + r // 128) * 512 + (r % 32) * 16
            + (r % 128 // 32) * 4 + j % 4)


def layout(topi: np.ndarray, E: int, bn: int, extra: int = 0):
    """Dispatch layout of ids [T, k]: sorted_ids (pads = T*k), expert_ids, padded total;
    `extra` blocks of junk follow, as a buffer of worst-case size has them."""
    flat = topi.reshape(-1)
    R = flat.size
    ids, eids = [], []
    for e in range(E):
        mine = np.flatnonzero(flat == e)
        if mine.size:
            pad = -mine.size % bn
            ids += [mine, np.full(pad, R)]
            eids += [e] * ((mine.size + pad) // bn)
    total = len(eids) * bn
    ids.append(np.full(extra * bn, 7))
    eids += [0] * extra
    return (np.concatenate(ids).astype(np.int32), np.array(eids, dtype=np.int32), total)
