"""Exact host oracles for the tk8s HIP kernels (numpy / hashlib; no GPU).

* :func:`philox4x32_10` / :func:`philox_bytes` — bit-exact model of ``philox_fill``
  (native/src/stream_kernels.hip): Random123 Philox4x32-10, counter = (block index lo, hi, 0, 0),
  key = (seed lo, seed hi).
* :func:`md5_tree` — the chunked, fan-in-4 MD5 tree of ``md5_tree`` (native/src/md5_kernels.hip), built
  from :mod:`hashlib` MD5 so the GPU digest can be checked against an independent implementation.
* :func:`allreduce_expected` — value of the N6 pattern after a sum all-reduce.

Reference anchor: docs/benchmarks.md:11-12 (the /cpu benchmark md5-hashes random numbers).
"""
from __future__ import annotations

import hashlib

import numpy as np

_M0 = np.uint64(0xD2511F53)
_M1 = np.uint64(0xCD9E8D57)
_W0 = 0x9E3779B9
_W1 = 0xBB67AE85
_MASK = np.uint64(0xFFFFFFFF)


def philox4x32_10(ctr: np.ndarray, key: tuple[int, int]) -> np.ndarray:
    """Philox4x32-10 over counters ``ctr`` (shape [n, 4], uint32) with key (k0, k1)."""
    c = ctr.astype(np.uint64)
    c0, c1, c2, c3 = c[:, 0], c[:, 1], c[:, 2], c[:, 3]
    k0, k1 = int(key[0]) & 0xFFFFFFFF, int(key[1]) & 0xFFFFFFFF
    for r in range(10):
        if r:
            k0 = (k0 + _W0) & 0xFFFFFFFF
            k1 = (k1 + _W1) & 0xFFFFFFFF
        p0 = _M0 * c0
        p1 = _M1 * c2
        hi0, lo0 = p0 >> np.uint64(32), p0 & _MASK
        hi1, lo1 = p1 >> np.uint64(32), p1 & _MASK
        c0, c1, c2, c3 = hi1 ^ c1 ^ np.uint64(k0), lo1, hi0 ^ c3 ^ np.uint64(k1), lo0
    return np.stack([c0, c1, c2, c3], axis=1).astype(np.uint32)


def philox_bytes(nbytes: int, seed: int) -> bytes:
    """Bytes written by ``philox_fill(dst, nbytes, seed)`` (nbytes multiple of 16)."""
    if nbytes % 16:
        raise ValueError("nbytes must be a multiple of 16")
    n = nbytes // 16
    idx = np.arange(n, dtype=np.uint64)
    ctr = np.zeros((n, 4), dtype=np.uint32)
    ctr[:, 0] = (idx & _MASK).astype(np.uint32)
    ctr[:, 1] = (idx >> np.uint64(32)).astype(np.uint32)
    out = philox4x32_10(ctr, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    return out.astype("<u4").tobytes()


def md5_tree(data: bytes, chunk_bytes: int = 1024, fan_in: int = 4) -> bytes:
    """MD5 tree: hash each ``chunk_bytes`` chunk (one chunk: its plain MD5), then fold the
    digests ``fan_in`` at a time -- a parent is the MD5 of its children's concatenated digests --
    until one remains."""
    if chunk_bytes <= 0 or chunk_bytes % 64:
        raise ValueError("chunk_bytes must be a positive multiple of 64")
    data = bytes(data)
    if len(data) <= chunk_bytes:
        return hashlib.md5(data).digest()
    level = [hashlib.md5(data[i : i + chunk_bytes]).digest() for i in range(0, len(data), chunk_bytes)]
    while len(level) > 1:
        level = [hashlib.md5(b"".join(level[i : i + fan_in])).digest() for i in range(0, len(level), fan_in)]
    return level[0]


def allreduce_expected(count: int, nranks: int) -> np.ndarray:
    """fp32 reference of the N6 pattern: sum over ranks r of (r + 1) + (i % 7)."""
    i = np.arange(count)
    per_rank = np.stack([(r + 1) + (i % 7) for r in range(nranks)]).astype(np.float32)
    return per_rank.sum(axis=0, dtype=np.float32)


# ---- 8-bit layer (native/src/fp8_kernels.hip, native/src/matmul_kernels.hip), in 64 bits -----------


def e4m3_values() -> np.ndarray:
    """The value of each e4m3 byte: 1 sign, 4 exponent (bias 7) and 3 fraction bits, 0x7f/0xff NaN."""
    code = np.arange(256)
    e, f = (code >> 3) & 15, (code & 7) / 8.0
    v = np.where(e == 0, f * 2.0 ** -6, (1.0 + f) * 2.0 ** (e - 7.0))
    v[code & 0x7F == 0x7F] = np.nan
    return np.where(code & 0x80, -v, v)


def e4m3_bytes(v: np.ndarray) -> np.ndarray:
    """Bytes of the e4m3 values nearest to v (|v| <= 448; ties to the even byte); NaN is 0x7f."""
    table = e4m3_values()[:127]
    m = np.abs(v)
    nan = np.isnan(m)
    above = np.clip(np.searchsorted(table, np.where(nan, 0.0, m)), 1, 126)
    up, down = table[above] - m, m - table[above - 1]
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, above - 1)
    return np.where(nan, 0x7F, code | np.where(np.signbit(v), 0x80, 0)).astype(np.uint8)


def e8m0_bytes(amax: np.ndarray) -> np.ndarray:
    """E8M0 byte of blocks with these largest magnitudes: the least 2^e (e in -127..127) with
    amax <= 448 * 2^e; 1 for zeros, NaN (255) where not finite."""
    out = np.full(amax.shape, 127, dtype=np.int64)
    some = (amax > 0) & np.isfinite(amax)
    mant, expo = np.frexp(amax[some])
    out[some] = np.clip(expo - np.where(mant <= 0.875, 9, 8), -127, 127) + 127
    out[~np.isfinite(amax)] = 255
    return out.astype(np.uint8)


def e8m0_values(byte: np.ndarray) -> np.ndarray:
    return np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))


def fp8_quantize(x: np.ndarray, block_rows: int = 1) -> tuple[np.ndarray, np.ndarray]:
    """(e4m3 bytes, E8M0 bytes) of x with a scale for each block_rows x 128 values."""
    rows, cols = x.shape
    nr, nc = -(-rows // block_rows), -(-cols // 128)
    padded = np.zeros((nr * block_rows, nc * 128))
    padded[:rows, :cols] = x
    blocks = padded.reshape(nr, block_rows, nc, 128)
    scales = e8m0_bytes(np.abs(blocks).max(axis=(1, 3)))
    q = e4m3_bytes(blocks / e8m0_values(scales)[:, None, :, None])
    return q.reshape(nr * block_rows, nc * 128)[:rows, :cols], scales


def fp8_dequantize(q: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """The values of e4m3 bytes q with a scale for each 1 x 128 or 128 x 128 of them."""
    rows, cols = q.shape
    s = e8m0_values(scales)
    if s.shape[0] != rows:
        s = np.repeat(s, 128, axis=0)[:rows]
    return e4m3_values()[q] * np.repeat(s, 128, axis=1)[:, :cols]


def rms_norm(h: np.ndarray, weight: np.ndarray, eps: float) -> tuple[np.ndarray, np.ndarray]:
    """(y, rstd) of an RMS norm over the rows of h."""
    rstd = 1.0 / np.sqrt(np.square(h).mean(axis=1) + eps)
    return h * rstd[:, None] * weight, rstd


def rms_norm_backward(dy: np.ndarray, h: np.ndarray, weight: np.ndarray, rstd: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(dh, dweight) of :func:`rms_norm` for the gradient dy of y."""
    xh = h * rstd[:, None]
    g = dy * weight
    return rstd[:, None] * (g - xh * (g * xh).mean(axis=1, keepdims=True)), (dy * xh).sum(axis=0)
