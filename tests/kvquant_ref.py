"""The 8-bit KV cache in 64 bits, in plain numpy: rotation, codes, attention, and how far 32-bit sums and 16-bit weights may be from it."""
import numpy as np


def rotate(x: np.ndarray, cs: np.ndarray, pos: np.ndarray) -> np.ndarray:
    """fp16 rows [rows, heads, hd] turned by the angles cs[pos]: rounded to 32 bits (products of halves are exact there) and to fp16."""
    c, s = (cs[pos][:, None, :, i].astype(np.float64) for i in range(2))
    a, b = x[..., 0::2].astype(np.float64), x[..., 1::2].astype(np.float64)
    out = np.empty(x.shape, np.float32)
    out[..., 0::2], out[..., 1::2] = a * c - b * s, a * s + b * c
    return out.astype(np.float16)


def codes(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """(codes as numbers, scales) of the last axis of finite fp16 values."""
    x = x.astype(np.float64)
    top = np.abs(x).max(-1, keepdims=True)
    if fmt == "int8":
        grain = np.exp2(np.maximum(np.frexp(np.where(top > 0, top / 127, 1))[1] - 4, -24))
        scale = np.ceil(top / 127 / grain) * grain
        code = np.clip(np.rint(np.divide(x, scale, out=np.zeros_like(x), where=scale > 0)), -127, 127)
        code = np.where(np.abs(code) * scale > 65504, code - np.sign(code), code)
        return code, scale
    m, e = np.frexp(np.where(top > 0, top / 448, 1))
    scale = np.where(top > 0, np.exp2(np.maximum(np.where(m == 0.5, e - 1, e), -15)), 0.0)
    y = np.divide(x, scale, out=np.zeros_like(x), where=scale > 0)
    unit = np.exp2(np.maximum(np.frexp(np.where(y != 0, np.abs(y), 1))[1] - 1, -6) - 3.0)
    y = np.rint(y / unit) * unit
    return np.where(np.abs(y) * scale > 65504, np.sign(y) * 240, y), scale


def stored(k: np.ndarray, v: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """What K and V rows [.., hd] are once stored; a row with a NaN or an infinity in either becomes NaN in both."""
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    out = []
    for x in (k, v):
        c, s = codes(np.where(bad[..., None], np.float16(0), x), fmt)
        y = c * s
        assert (y == y.astype(np.float16)).all()  # code x scale is an fp16 number
        y[bad] = np.nan
        out.append(y.astype(np.float16))
    return out[0], out[1]


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, last: int) -> tuple[np.ndarray, np.ndarray]:
    """One row of queries [H, hd] over positions 0 .. last of k, v [T, G, hd]: (result [H * hd], how far off it may be).

    Off by: its rounding to fp16 (2^-11 of it, 2^-25 below 2^-14); for each weight, relative to it, its rounding to fp16 (2^-11), the
    errors of its score and of the exponential (the sum of hd exact products in 32 bits: hd 2^-24 of the sum of their magnitudes, the
    scaled score and its distance to the maximum rounded in the exponent: three more 2^-24 of the score's magnitude each, at a span of twice the
    largest; 2^-22 for the exponential), and those of the 32-bit sums over T positions and of the running maximum's factors
    (T 2^-23); a weight below 2^-14 of the largest may be off by 2^-25 of it instead of a share of itself."""
    H, hd = q.shape
    G = k.shape[1]
    q = q.astype(np.float64).reshape(G, H // G, hd)
    k, v = k[:last + 1].astype(np.float64), v[:last + 1].astype(np.float64)
    s = np.einsum("grd,tgd->grt", q, k) / np.sqrt(hd)
    mag = np.einsum("grd,tgd->grt", np.abs(q), np.abs(k)).max(-1, keepdims=True) / np.sqrt(hd)
    p = np.exp(s - s.max(-1, keepdims=True))
    l = p.sum(-1, keepdims=True)
    o = np.einsum("grt,tgd->grd", p / l, v)
    a = np.einsum("grt,tgd->grd", p / l, np.abs(v))
    small = 2.0 ** -25 * np.abs(v).sum(0)[:, None] / l
    share = 2.0 ** -11 + (hd + 6) * 2.0 ** -24 * mag + 2.0 ** -22 + (last + 1) * 2.0 ** -23
    tol = 2.0 ** -11 * np.abs(o) + 2.0 ** -25 + 2 * share * a + small
    return o.reshape(-1), tol.reshape(-1)
