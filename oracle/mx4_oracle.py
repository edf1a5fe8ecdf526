"""Float64 statement of the 4-bit token cache and of the attention pooling over it (numpy, CPU; test infrastructure only).

The reference has no counterpart; the format is the OCP microscaling MXFP4 layout described in include/ep_hip.h."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """(..., D) -> (codes (..., Dp/2), scales (..., Dp/32)) uint8."""
    x = np.asarray(x, np.float64)
    D = x.shape[-1]
    Dp = -(-D // 128) * 128
    g = np.zeros(x.shape[:-1] + (Dp,))
    g[..., :D] = x
    g = g.reshape(x.shape[:-1] + (Dp // 32, 32))
    with np.errstate(invalid="ignore"):
        amax = np.abs(g).max(-1)
    bad = ~np.isfinite(amax)
    mant, ex = np.frexp(np.where(bad | (amax == 0), 1.0, amax))             # mant in [0.5, 1)
    e = np.clip(ex - 3 + (mant >= 0.875), -125, 125)
    e = np.where(amax == 0, -125, e)
    v = np.where(bad[..., None], 0.0, g) / np.exp2(e.astype(np.float64))[..., None]
    a = np.abs(v)
    dist = np.abs(a[..., None] - GRID)
    best = dist.min(-1, keepdims=True)
    near = dist == best                                                     # one or, at a tie, two neighbours
    code = near.argmax(-1)
    last = 7 - near[..., ::-1].argmax(-1)
    code = np.where(code % 2 == 0, code, last)                              # ties: the even code
    code = np.where((code != 0) & (v < 0), code + 8, code).astype(np.uint8)
    code = code.reshape(x.shape[:-1] + (Dp,))
    return code[..., 0::2] | (code[..., 1::2] << 4), np.where(bad, 255, e + 127).astype(np.uint8)


def dequantize(codes, scales, D):
    nib = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (-1,))
    val = GRID[nib & 7] * np.where(nib >= 8, -1.0, 1.0)
    mult = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (val.reshape(scales.shape + (32,)) * mult[..., None]).reshape(codes.shape[:-1] + (-1,))[..., :D]


def attention(x, lengths, q, scale, dP=None):
    """x (B, N, D), lengths (B,), q (B, Q, D): P, S, A and, with dP, the per-image query gradients and a bound on the size of the
    terms that they are sums of (per component)."""
    B, N, D = x.shape
    Q = q.shape[1]
    P, S, A = np.zeros((B, Q, D)), np.full((B, Q, N), -np.inf), np.zeros((B, Q, N))
    dq, mag = np.zeros((B, Q, D)), np.zeros((B, Q, D))
    for b in range(B):
        n = int(lengths[b])
        if n == 0:
            continue
        xb = x[b, :n]
        s = scale * (q[b] @ xb.T)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        S[b, :, :n], A[b, :, :n], P[b] = s, p, p @ xb
        if dP is not None:
            dA = dP[b] @ xb.T
            delta = (dP[b] * P[b]).sum(-1, keepdims=True)
            dq[b] = scale * ((p * (dA - delta)) @ xb)
            size = np.linalg.norm(dP[b], axis=-1, keepdims=True) * np.linalg.norm(xb, axis=-1)[None, :]
            mag[b] = scale * ((p * size) @ np.abs(xb))
    return P, S, A, dq, mag
