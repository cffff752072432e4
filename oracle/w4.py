"""MXFP4 weights, FP8 activations and the products on them in numpy -- TEST INFRASTRUCTURE ONLY.

OCP Microscaling: 32 elements of K share an e8m0 scale 2^(byte - 127) (255: NaN); an e2m1 element is
(-1)^s * {0, 0.5, 1, 1.5, 2, 3, 4, 6}; two a byte, the lower index in the low half.
"""

from __future__ import annotations

import numpy as np

from .numerics import E4M3_TABLE, e4m3_encode

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0])
CHUNK_BYTES, CHUNK_K = 4352, 512
#: The FP8 / FP4 MFMA's error on a block of 128 products, relative to the sum of their magnitudes (measured on the
#: instruction by test_gpu_kernels.test_mfma_block_sum_accuracy).
MFMA_REL = 2.5e-4
U32, U16 = 2.0**-24, 2.0**-8  # half a step of fp32 and of bf16, relative


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 [..., K] of codes [..., K / 2] and scales [..., K / 32]."""
    v = np.stack([E2M1[codes & 15], E2M1[codes >> 4]], -1).reshape(*codes.shape[:-1], -1, 32)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int32) - 127))
    return (v * s[..., None]).reshape(*codes.shape[:-1], -1)


def quantize(w: np.ndarray):
    """fp32 [..., K] -> (codes, scales), element by element: the nearest of the eight magnitudes, a tie to the even code."""
    w = np.asarray(w, np.float32)
    g = w.reshape(-1, 32)
    codes, scales = np.zeros(g.shape, np.uint8), np.zeros(g.shape[0], np.uint8)
    for i, row in enumerate(g):
        m = np.abs(row.astype(np.float64)).max()
        if not np.isfinite(m):
            scales[i] = 255
            continue
        ex = max(int(np.floor(np.log2(m))) - 2 + 127, 0) if m > 0 else 0
        if m > 0 and 2.0 ** np.floor(np.log2(m)) > m:  # a logarithm that rounded up
            ex = max(ex - 1, 0)
        scales[i] = ex
        a = np.abs(row.astype(np.float64)) * 2.0 ** (127 - ex)
        dist = np.abs(a[:, None] - E2M1[None, :8])
        best = dist.min(1, keepdims=True)
        near = dist == best
        even = near & (np.arange(8)[None, :] % 2 == 0)
        codes[i] = np.where(even.any(1), even.argmax(1), near.argmax(1)) | (np.signbit(row) * 8).astype(np.uint8)
    codes = codes.reshape(*w.shape)
    return (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8), scales.reshape(*w.shape[:-1], -1)


def pack(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """One matrix [N, K / 2], [N, K / 32] -> uint8 [ceil(N / 16), ceil(K / 512), 4352]: of a K-block of 128, lane
    16 g + i holds row i's elements 32 g .. +32; after a chunk's four K-blocks, per lane their four scales."""
    N, K = codes.shape[0], codes.shape[1] * 2
    nt, kc = -(-N // 16), -(-K // CHUNK_K)
    c = np.zeros((nt * 16, kc * CHUNK_K // 2), np.uint8)
    s = np.full((nt * 16, kc * CHUNK_K // 32), 127, np.uint8)
    c[:N, :K // 2], s[:N, :K // 32] = codes, scales
    c = c.reshape(nt, 16, kc, 4, 4, 16).transpose(0, 2, 3, 4, 1, 5)  # [tile, chunk, K-block, g, row, byte]
    s = s.reshape(nt, 16, kc, 4, 4).transpose(0, 2, 4, 1, 3)         # [tile, chunk, g, row, K-block]
    return np.concatenate([c.reshape(nt, kc, -1), s.reshape(nt, kc, -1)], 2)


def quant_act(x: np.ndarray):
    """fp32 [T, K] -> (e4m3 codes [T, K], scale fp32 [K / 128, T])."""
    T, K = x.shape
    b = np.asarray(x, np.float32).reshape(T, K // 128, 128)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        amax = np.fmax.reduce(np.abs(b), axis=2, initial=0.0)
        scale = np.maximum((amax / np.float32(448.0)).astype(np.float32), np.float32(1e-8)).astype(np.float32)
        q = np.clip((b / scale[:, :, None]).astype(np.float32), np.float32(-448.0), np.float32(448.0))
    return e4m3_encode(q.reshape(T, K)), np.ascontiguousarray(scale.T)


def act_values(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    return E4M3_TABLE[codes] * np.repeat(scale.T.astype(np.float64), 128, axis=1)


def linear(x_codes, x_scale, w: np.ndarray):
    """(y float64 [T, N], bound on the error of a bf16 result): each K-block's sum off by MFMA_REL of its magnitudes,
    one rounding by the scale's product and one by its addition for each of the K / 128 blocks, then bf16."""
    x = act_values(x_codes, x_scale)
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    err = (MFMA_REL + (w.shape[1] // 128 + 2) * U32) * mag
    return y, err + U16 * (np.abs(y) + err)


def _requant(c: np.ndarray, err: np.ndarray):
    """(values of the requantised c [R, I], bound on what an evaluation whose c is off by err differs): the code's
    value is monotone in c and 1 / scale, so the ends of both intervals bound it."""
    R = c.shape[0]
    b, e = c.reshape(R, -1, 128), err.reshape(R, -1, 128)
    amax = np.abs(b).max(2)
    off = e.max(2)

    def value(v, scale):
        q = np.clip(v / scale[:, :, None], -448.0, 448.0).astype(np.float32)
        return E4M3_TABLE[e4m3_encode(q.ravel()).reshape(q.shape)] * scale[:, :, None]

    scale = np.maximum(amax / 448.0, 1e-8)
    lo_s = np.maximum((amax - off) / 448.0 * (1 - 4 * U32), 1e-8)
    hi_s = np.maximum((amax + off) / 448.0 * (1 + 4 * U32), 1e-8)
    mid = value(b, scale)
    far = np.zeros_like(mid)
    for v in (b - e, b, b + e):
        for s in (lo_s, scale, hi_s):
            far = np.maximum(far, np.abs(value(v * (1 + 2 * U32), s) - mid))
            far = np.maximum(far, np.abs(value(v * (1 - 2 * U32), s) - mid))
    return mid.reshape(R, -1), far.reshape(R, -1)


def experts(x_codes, x_scale, w13: np.ndarray, w2: np.ndarray, ids, weights, offset: int):
    """(out float64 [T, hidden], bound on the error of a bf16 result).  w13 [E, 2 I, hidden], w2 [E, hidden, I]."""
    T, k = ids.shape
    E, hidden, inter = w2.shape
    x = act_values(x_codes, x_scale)
    out, err = np.zeros((T, hidden)), np.zeros((T, hidden))
    for e in range(E):
        tok, j = np.nonzero(ids == e + offset)
        if not tok.size:
            continue
        g, mag = x[tok] @ w13[e].T, np.abs(x[tok]) @ np.abs(w13[e]).T
        ge = (MFMA_REL + (hidden // 128 + 2) * U32) * mag
        up, act = g[:, :inter], g[:, inter:]
        with np.errstate(over="ignore"):
            silu = act / (1.0 + np.exp(-act))
        # |silu'| <= 1.1; silu and the product in fp32: under 12 roundings
        ce = np.abs(silu) * ge[:, :inter] + 1.1 * np.abs(up) * ge[:, inter:] + 1.1 * ge[:, :inter] * ge[:, inter:]
        c = up * silu
        c, cd = _requant(c, ce + 12 * U32 * np.abs(c))
        y, ymag = c @ w2[e].T, (np.abs(c) + cd) @ np.abs(w2[e]).T
        ye = cd @ np.abs(w2[e]).T + (MFMA_REL + (inter // 128 + 4) * U32) * ymag
        w = weights[tok, j][:, None].astype(np.float64)
        np.add.at(out, tok, y * w)
        np.add.at(err, tok, (ye + k * U32 * np.abs(y)) * np.abs(w))
    return out, err + U16 * (np.abs(out) + err)
