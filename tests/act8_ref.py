"""Plain 64-bit implementations of the int8 quantizer with its norm, the linear of
int8 rows and 4-bit weights, and the low-rank adapters, by their definitions, with the
bounds that their tests use."""
import numpy as np

U16, U32 = 2.0 ** -11, 2.0 ** -24   # half a step of fp16 and fp32, relative
TINY = 2.0 ** -25                   # half a step of fp16 below its normal numbers


def quant(y, clip=1.0):
    """y [rows, n] in 64 bits -> (codes int8, scales fp32)."""
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.abs(y).max(-1, keepdims=True)
        scale = (top * clip / 127).astype(np.float32)
        bad = ~np.isfinite(top)
        unit = np.where(bad | (scale == 0), 1.0, scale.astype(np.float64))
        q = np.clip(np.rint(np.where(bad, 0.0, y) / unit), -127, 127)
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def norm_quant(x, eps, mean_dim=None, residual=None, weight=None, clip=1.0):
    """(codes, scales, h fp16, y in 64 bits)."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        h = x
        if residual is not None:
            h = (x.astype(np.float32) + residual.astype(np.float32)).astype(np.float16)
        d = h.astype(np.float64)
        y = d if weight is None else d * weight.astype(np.float64)
        y = y * (1.0 / np.sqrt((d * d).sum(-1, keepdims=True) / (mean_dim or x.shape[-1]) + eps))
    return (*quant(y, clip), h, y)


def pack(c):
    u = (c & 15).astype(np.uint8)
    return u[:, 0::2] | (u[:, 1::2] << 4)


def linear(a, sa, c, sb, bias=None, residual=None):
    """(exact, bound): the product is exact; its conversion, two products and two
    additions round to fp32, the result to fp16."""
    acc = a.astype(np.float64) @ c.astype(np.float64).T
    p = acc * sa.astype(np.float64).reshape(-1, 1) * sb.astype(np.float64)[None]
    out, size = p, 3 * np.abs(p)
    for extra in (bias, residual):
        if extra is not None:
            out = out + extra.astype(np.float64)
            size = size + np.abs(out)
    return out, (1 + 2 * U16) * (U16 * np.abs(out) + 1.01 * U32 * size) + TINY


def lora(y, x, la, lb, ids, scaling, widths):
    """(exact, bound).  A sum of k products in fp32 rounds k times at most, by half a
    step of a partial sum that the products' magnitudes bound; the second product reads
    its first operand in 22 bits or more, relative to a token's largest."""
    out = y.astype(np.float64)
    size = np.abs(out)
    r, K = lb.shape[2], x.shape[1]
    extra = np.zeros_like(out)
    for m, i in enumerate(ids):
        if not 0 <= i < la.shape[0]:
            continue
        f = 1.0 if scaling is None else float(scaling[i])
        xa, aa = x[m].astype(np.float64), la[i].astype(np.float64)
        t, at = aa @ xa, 0
        te = (K + 16) * U32 * (np.abs(aa) @ np.abs(xa))       # error of t
        for s, n in enumerate(widths):
            ts, es = t[s * r: (s + 1) * r], te[s * r: (s + 1) * r]
            b = lb[i, at: at + n].astype(np.float64)
            out[m, at: at + n] += f * (b @ ts)
            big = np.abs(ts) + es
            e = es + 2.0 ** -22 * big.max(initial=0)
            extra[m, at: at + n] = abs(f) * (np.abs(b) @ (e + (2 * r + 8) * U32 * big))
            at += n
        size[m] = np.abs(out[m]) + np.abs(y[m].astype(np.float64))
    bound = U16 * np.abs(out) + 1.01 * (extra + 2 * U32 * size)
    return out, (1 + 2 * U16) * bound + TINY
