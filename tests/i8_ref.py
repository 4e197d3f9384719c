"""Plain 64-bit implementations of the q/k norm with RoPE, the int8 cache's append
and its attention, by their definitions, one request, block and row at a time."""
import numpy as np

BLOCK, D = 16, 128


def norm_rope(x, w, cos, sin, eps):
    """x [..., D]; cos / sin broadcast against it.  Returns (out, size), size the
    sum of the magnitudes that were added (for tolerances)."""
    x = x.astype(np.float64)
    y = x
    if eps is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            y = y * w.astype(np.float64)
    h = x.shape[-1] // 2
    turned = np.concatenate((-y[..., h:], y[..., :h]), -1)
    c, s = cos.astype(np.float64), sin.astype(np.float64)
    return y * c + turned * s, np.abs(y * c) + np.abs(turned * s)


def table(lens, page, rng, extra=0, order=None):
    """indptr, indices, last of requests of these lengths on shuffled pages, and
    the number of pages in the pool (`extra` of them unused)."""
    count = [-(-n // page) for n in lens]
    total = sum(count) + extra
    perm = rng.permutation(total).astype(np.int32)
    indptr = np.concatenate(([0], np.cumsum(count))).astype(np.int32)
    last = np.array([(n - 1) % page + 1 if n else 0 for n in lens], np.int32)
    return indptr, perm[: sum(count)].copy(), last, max(1, total)


def lengths(indptr, last, page):
    n = np.diff(indptr)
    return np.where(n > 0, (n - 1) * page + last, 0)


def append(data, scale, indptr, indices, last, layer, k, v, new=None):
    """In place.  new: row index [B + 1] or None."""
    page, heads = data.shape[4], data.shape[3]
    lens = lengths(indptr, last, page)
    for b, ln in enumerate(lens):
        s0, n = (b, 1) if new is None else (int(new[b]), int(new[b + 1] - new[b]))
        old = int(ln) - n
        for j in range(max(old, 0) // BLOCK, -(-int(ln) // BLOCK)):
            if n == 0:
                continue
            pg = indices[indptr[b] + j * BLOCK // page]
            if not 0 <= pg < data.shape[0]:
                continue
            e0 = j * BLOCK % page
            lo, hi = max(old, j * BLOCK), min(int(ln), (j + 1) * BLOCK)
            for kv, src in ((0, k), (1, v)):
                for h in range(heads):
                    x = src[s0 + lo - old: s0 + hi - old, h].astype(np.float64)
                    at = scale[pg, layer, kv, h]
                    was = at[e0 // BLOCK] if lo > j * BLOCK else np.float32(0)
                    rows = data[pg, layer, kv, h, e0: e0 + BLOCK]
                    keep = lo - j * BLOCK
                    if not np.isfinite(x).all() or not np.isfinite(was):
                        rows[: keep] = 0
                        rows[keep: keep + hi - lo] = 0
                        at[e0 // BLOCK] = np.nan
                        continue
                    top = np.float32(np.abs(x).max()) * (np.float32(1) / np.float32(127))
                    now = max(was, top)
                    d = np.float64(now) if now > 0 else 1.0
                    if now != was and keep:
                        rows[: keep] = np.rint(rows[: keep] * np.float64(was) / d)
                    rows[keep: keep + hi - lo] = np.rint(x / d)
                    at[e0 // BLOCK] = now


def attention(q, data, scale, indptr, indices, last, layer, new=None, sm_scale=None, o=None):
    """Returns (out, size): size the sum of weight x |value|; rows of no request
    keep o's values."""
    page, heads = data.shape[4], data.shape[3]
    group = q.shape[1] // heads
    sm = D ** -0.5 if sm_scale is None else sm_scale
    out = np.zeros(q.shape) if o is None else o.astype(np.float64)
    size = np.zeros(q.shape)
    for b, ln in enumerate(lengths(indptr, last, page)):
        s0, n = (b, 1) if new is None else (int(new[b]), int(new[b + 1] - new[b]))
        if n == 0:
            continue
        pages = indices[indptr[b]: indptr[b + 1]]
        here = np.repeat((pages >= 0) & (pages < data.shape[0]), page)[: ln]
        safe = np.where((pages >= 0) & (pages < data.shape[0]), pages, 0)
        codes = data[safe, layer].astype(np.float64)              # [p, 2, H, page, D]
        val = codes * np.repeat(scale[safe, layer].astype(np.float64), BLOCK, -1)[..., None]
        val = val.transpose(1, 2, 0, 3, 4).reshape(2, heads, -1, D)[:, :, : ln]
        for i in range(n):
            seen = here & (np.arange(ln) <= ln - n + i)
            for h in range(q.shape[1]):
                kk, vv = val[0, h // group][seen], val[1, h // group][seen]
                if not len(kk):
                    out[s0 + i, h] = 0
                    continue
                x = kk @ q[s0 + i, h].astype(np.float64) * sm
                p = np.exp(x - x.max())
                p /= p.sum()
                out[s0 + i, h] = p @ vv
                size[s0 + i, h] = p @ np.abs(vv)
    return out, size
