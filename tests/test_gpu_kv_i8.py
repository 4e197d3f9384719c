"""The paged int8 cache: append (codes and scales bit for bit against exact
arithmetic), the fused norm + RoPE + append, and attention over the cache, at the
lengths, pages, layouts and bad values where they can go wrong."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA
from tests import i8_ref
from tests.gpu_util import DEV, assert_bitexact, to_dev, to_np

pytestmark = pytest.mark.gpu
BLOCK, D = 16, 128


def _pool(rng, pages, L, H, page, fill="random"):
    data = rng.integers(-127, 128, (pages, L, 2, H, page, D)).astype(np.int8)
    scale = rng.uniform(0.01, 0.05, (pages, L, 2, H, page // BLOCK)).astype(np.float32)
    return data, scale


def _starts(counts):
    return np.concatenate(([0], np.cumsum(counts))).astype(np.int32)


class Cache:
    """A pool with a table, on the host and on the device."""

    def __init__(self, rng, lens, H=2, page=16, L=2, layer=1, extra=3):
        self.indptr, self.indices, self.last, pages = i8_ref.table(lens, page, rng, extra)
        self.data, self.scale = _pool(rng, pages, L, H, page)
        self.layer, self.lens, self.H, self.page = layer, list(lens), H, page
        self.upload()

    def upload(self):
        self.dev = [to_dev(a) for a in (self.data, self.scale, self.indptr, self.indices,
                                        self.last)]

    def args(self):
        return (*self.dev, self.layer)

    def table(self):
        return self.data, self.scale, self.indptr, self.indices, self.last, self.layer

    def assert_same(self):
        assert_bitexact(to_np(self.dev[0]), self.data, "codes")
        got, want = to_np(self.dev[1]), self.scale
        assert np.array_equal(got, want, equal_nan=True), np.argwhere(got != want)[:5]


def _kv(rng, n, H, mag=1.0):
    return [(mag * rng.standard_normal((n, H, D))).astype(np.float16) for _ in range(2)]


def _append(c, k, v, new=None, hint=None):
    _CUDA.append_kv_i8(*c.args(), to_dev(k), to_dev(v), None if new is None else to_dev(new), hint)
    i8_ref.append(*c.table(), k, v, new)
    torch.cuda.synchronize()
    c.assert_same()


# --------------------------------------------------------------- append

@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("H", [1, 3, 8])
def test_append_one_token_each(page, H):
    """Every place in a block: new blocks, open ones, page ends; large tokens that
    move the scale and small ones that do not.  Codes behind the last token, other
    layers and unused pages stay."""
    rng = np.random.default_rng(page + H)
    c = Cache(rng, [1, 2, 15, 16, 17, 33, page, page + 1, 2 * page - 1], H, page)
    k, v = _kv(rng, len(c.lens), H)
    k[::2] *= 4
    _append(c, k, v)


@pytest.mark.parametrize("page", [16, 64])
def test_append_token_by_token(page):
    """A request grown from nothing over three pages, block scales moving on the
    way."""
    rng = np.random.default_rng(3)
    total = 2 * page + 5
    c = Cache(rng, [total, total], 2, page)
    full = c.indptr.copy(), c.indices.copy()
    pages = [full[1][full[0][b]: full[0][b + 1]] for b in range(2)]
    for t in range(1, total + 1):
        n = -(-t // page)
        c.indptr = np.array([0, n, 2 * n], np.int32)
        c.indices = np.concatenate([p[:n] for p in pages]).astype(np.int32)
        c.last = np.full(2, (t - 1) % page + 1, np.int32)
        c.dev[2:] = [to_dev(a) for a in (c.indptr, c.indices, c.last)]
        k, v = _kv(rng, 2, 2, mag=float(rng.choice([0.1, 1.0, 3.0])))
        _CUDA.append_kv_i8(*c.args(), to_dev(k), to_dev(v))
        i8_ref.append(*c.table(), k, v)
    torch.cuda.synchronize()
    c.assert_same()


@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("hint", [None, 1, 700])
def test_append_ragged(page, hint):
    """Any number of new tokens a request, none among them, more than the table
    holds, and any launch hint; rows behind the last request are not read."""
    rng = np.random.default_rng(page)
    held, new = [0, 5, 16, 31, 100, 40, 0, 20], [1, 11, 1, 300, 0, 17, 47, 33]
    lens = [h + n for h, n in zip(held, new)]
    lens[-1] = 10                      # 33 new tokens, room for 10
    c = Cache(rng, lens, 2, page)
    k, v = _kv(rng, sum(new) + 4, 2)
    k[-4:], v[-4:] = np.nan, np.nan
    _append(c, k, v, _starts(new), hint)


def test_many_uneven_requests_without_a_hint():
    """Launches sized by all the rows for each of 6000 requests are cut down; one of
    them has most of the rows, and any hint is taken."""
    rng = np.random.default_rng(9)
    new = [1] * 6000
    new[17] = 5000
    c = Cache(rng, new, 1, 16, L=1, layer=0)
    k, v = _kv(rng, sum(new), 1)
    q = rng.standard_normal((sum(new), 1, D)).astype(np.float16)
    for hint in (None, 2 ** 62):
        _append(c, k, v, _starts(new), hint)
        c.assert_same()
        got = _attend(c, q, _starts(new), hint)
    first = c.scale[c.indices[c.indptr[:-1]], 0, 1, 0, 0].astype(np.float64)
    rows = c.data[c.indices[c.indptr[:-1]], 0, 1, 0, 0] * first[:, None]
    # one token: its own value, but for its weight's rounding and the result's
    alone = np.array(new) == 1
    at = _starts(new)[:-1]
    assert (np.abs(got[at[alone], 0] - rows[alone])
            <= 2.0 ** -10 * np.abs(rows[alone]) + 2.0 ** -25).all()
    tail = Cache.__new__(Cache)                   # the long one's last 40 rows
    tail.__dict__.update(c.__dict__)
    tail.indptr, tail.last = c.indptr[17:19] - c.indptr[17], c.last[17:18]
    tail.indices = c.indices[c.indptr[17]:c.indptr[18]]
    end = at[17] + 5000
    want, size = i8_ref.attention(q[end - 40:end], *tail.table(), np.array([0, 40]))
    _close(got[end - 40:end], want, size, 5000)


def test_append_values_at_the_ends():
    """Zero blocks, subnormal and largest values, and quotients on ties: x =
    (i + 0.5) s with s a power of two."""
    rng = np.random.default_rng(8)
    c = Cache(rng, [16, 16, 16, 16, 20], 1, 16)
    n = sum(c.lens)
    k, v = _kv(rng, n, 1)
    k[:16] = 0
    k[16:32] = (rng.integers(-3, 4, (16, 1, D)) * 2.0 ** -24).astype(np.float16)
    k[32:48] = np.clip(k[32:48].astype(np.float32) * 30000, -65504, 65504)
    half = (np.arange(D) - 63.5).astype(np.float16)
    k[48:64] = half * np.float16(0.25)
    k[48, 0, 0] = 127 * 0.25                     # scale exactly 0.25
    k[64:84] *= 0
    k[83] = 2.0
    new = _starts(c.lens)
    _append(c, k, v, new)
    assert c.scale[c.indices[3], 1, 0, 0, 0] == 0.25
    # an empty (all-zero) block takes a scale later
    c2 = Cache(rng, [16], 1, 16)
    _append(c2, k[:16], v[:16], _starts([16]))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_nonfinite_poisons_its_block_only(bad):
    rng = np.random.default_rng(9)
    c = Cache(rng, [40, 40], 2, 16)
    k, v = _kv(rng, 70, 2)
    k[20, 1, 3] = bad      # request 0: token 5 + 20 = 25, block 1
    _append(c, k, v, _starts([35, 35]))
    assert np.isnan(c.scale[c.indices[1], 1, 0, 1, 0])
    # the next token of a poisoned block does not heal it, a new block does
    c.last = np.array([8, 9], np.int32)
    c.scale[c.indices[2], 1, 1, 0, 0] = np.nan
    c.upload()
    k, v = _kv(rng, 2, 2)
    _append(c, k, v)
    assert np.isnan(c.scale[c.indices[2], 1, 1, 0, 0])


def test_append_strided_and_bad_tables():
    rng = np.random.default_rng(10)
    H = 2
    c = Cache(rng, [20, 30, 40], H, 16)
    qkv = rng.standard_normal((9, (4 + 2 * H) * D)).astype(np.float16)
    x = to_dev(qkv).view(9, -1, D)
    new = _starts([3, 3, 3])
    c.indices[c.indptr[1] + 1] = -1           # a page that is not there
    c.indices[c.indptr[2] + 2] = 10 ** 6
    c.upload()
    _CUDA.append_kv_i8(*c.args(), x[:, 4: 4 + H], x[:, 4 + H:], to_dev(new), 3)
    h = qkv.reshape(9, -1, D)
    i8_ref.append(*c.table(), h[:, 4: 4 + H], h[:, 4 + H:], new)
    torch.cuda.synchronize()
    c.assert_same()


def test_append_far_pages():
    """Byte offsets past 2^32 in the pool."""
    H, page, pages = 8, 256, 9000
    data = torch.empty((pages, 1, 2, H, page, D), dtype=torch.int8, device=DEV)   # 4.7 GB
    scale = torch.zeros((pages, 1, 2, H, page // BLOCK), device=DEV)
    assert data.numel() > 2 ** 32
    t = [to_dev(np.array(a, np.int32)) for a in ([0, 1, 2], [pages - 1, 8300], [7, 200])]
    rng = np.random.default_rng(11)
    k, v = _kv(rng, 207, H)
    new = _starts([7, 200])
    _CUDA.append_kv_i8(data, scale, *t, 0, to_dev(k), to_dev(v), to_dev(new), 200)
    q = rng.standard_normal((2, 16, D)).astype(np.float16)
    o = torch.zeros(2, 16, D, dtype=torch.float16, device=DEV)
    _CUDA.batch_attention_i8(o, to_dev(q), data, scale, *t, 0)
    small = [np.zeros((2, 1, 2, H, page, D), np.int8),
             np.zeros((2, 1, 2, H, page // 16), np.float32)]
    host = [np.array(a, np.int32) for a in ([0, 1, 2], [0, 1], [7, 200])]
    i8_ref.append(*small, *host, 0, k, v, new)
    for i, pg in enumerate((pages - 1, 8300)):
        n = (7, 200)[i]
        assert_bitexact(to_np(data[pg, 0, :, :, :n]), small[0][i, 0, :, :, :n], "far codes")
        assert np.array_equal(to_np(scale[pg]), small[1][i])
    want, size = i8_ref.attention(q, *small, *host, 0)
    _close(to_np(o), want, size, 200)


# ------------------------------------------------- norm + rope + append

@pytest.mark.parametrize("Hq,H", [(4, 2), (32, 8), (5, 5), (40, 8), (0, 2)])
@pytest.mark.parametrize("norm", [True, False])
def test_fused_append_is_the_two_calls(Hq, H, norm):
    rng = np.random.default_rng(Hq + H)
    held, new = [0, 7, 30, 3], [1, 20, 2, 70]
    a = Cache(rng, [h + n for h, n in zip(held, new)], H, 16)
    rows = sum(new)
    qkv = rng.standard_normal((rows, (Hq + 2 * H) * D)).astype(np.float16)
    ang = rng.uniform(0, 6.3, (rows, D))
    cos, sin = (to_dev(f(ang).astype(np.float16)) for f in (np.cos, np.sin))
    w = [to_dev(rng.uniform(0.5, 1.5, D).astype(np.float16)) for _ in range(2)] if norm \
        else [None, None]
    eps = 1e-6 if norm else None
    idx = to_dev(_starts(new))
    x = to_dev(qkv)
    heads = x.view(1, rows, Hq + 2 * H, D)
    q, k = _CUDA.qk_norm_rope(heads[:, :, :Hq], heads[:, :, Hq: Hq + H], cos[None], sin[None], *w,
                              eps)
    other = [t.clone() for t in a.dev[:2]]
    _CUDA.append_kv_i8(*other, *a.dev[2:], a.layer, k[0], heads[0, :, Hq + H:], idx, 70)
    got = _CUDA.qkv_norm_rope_append_i8(*a.args(), x, cos, sin, Hq, *w, eps, idx, 70)
    torch.cuda.synchronize()
    assert torch.equal(got, q[0])
    assert torch.equal(a.dev[0], other[0]) and torch.equal(a.dev[1], other[1])


def test_fused_append_decode_with_one_table():
    """One row per request, one cos / sin row for all, a strided projection output."""
    rng = np.random.default_rng(21)
    a = Cache(rng, [1, 16, 17, 90], 2, 16)
    wide = to_dev(rng.standard_normal((4, 8 * D + 64)).astype(np.float16))
    x = wide[:, : 8 * D]
    cos, sin = (to_dev(f(rng.uniform(0, 6.3, (1, D))).astype(np.float16)) for f in (np.cos, np.sin))
    other = [t.clone() for t in a.dev[:2]]
    got = _CUDA.qkv_norm_rope_append_i8(*a.args(), x, cos, sin, 4)
    heads = x.contiguous().view(4, 1, 8, D)
    q, k = _CUDA.qk_norm_rope(heads[:, :, :4], heads[:, :, 4:6], cos[None], sin[None])
    _CUDA.append_kv_i8(*other, *a.dev[2:], a.layer, k[:, 0], heads[:, 0, 6:])
    assert torch.equal(got, q[:, 0])
    assert torch.equal(a.dev[0], other[0]) and torch.equal(a.dev[1], other[1])


# ------------------------------------------------------------ attention

def _close(got, want, size, n):
    """Weights are rounded to fp16 for the second product (2^-11 of each, or 2^-25
    beside the largest, which is at least 1: n 2^-25 of the largest value, at most
    127 times the mean block scale times the spread of the scales, here under 2^3
    of the values' mean size), scores carry under 2^-14 of relative error into the
    weights, and the result is rounded once (2^-11, or 2^-25)."""
    tol = (2.0 ** -11 * np.abs(want) + (2.0 ** -11 + 2.0 ** -14) * size
           + n * 2.0 ** -25 * 8 * size.max() + 2.0 ** -25)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (err / tol).max()


def _attend(c, q, new=None, hint=None, kv=None, sm=None, o=None):
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV) if o is None else o
    _CUDA.batch_attention_i8(out, to_dev(q), *c.args(), None if new is None else to_dev(new), hint,
                             kv, sm)
    torch.cuda.synchronize()
    return to_np(out)


def _check(c, q, new=None, hint=None, kv=None, sm=None):
    base = np.full(q.shape, 7.0)
    got = _attend(c, q, new, hint, kv, sm)
    want, size = i8_ref.attention(q, *c.table(), new, sm, base)
    _close(got, want, size, max(c.lens))
    return got


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("Hq,H", [(4, 1), (8, 8), (32, 8), (40, 8), (16, 1), (34, 2), (9, 3)])
def test_decode_lengths(Hq, H, page):
    rng = np.random.default_rng(Hq * page + H)
    c = Cache(rng, [1, 0, 2, 15, 16, 17, 31, 32, 33, 64, 65, 255, 256, 257, 700], H, page)
    q = (2 * rng.standard_normal((len(c.lens), Hq, D))).astype(np.float16)
    got = _check(c, q)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("Hq,H", [(64, 1), (130, 1), (66, 2)])
def test_large_groups(Hq, H):
    rng = np.random.default_rng(Hq)
    c = Cache(rng, [1, 40, 0, 333], H, 16)
    q = (2 * rng.standard_normal((4, Hq, D))).astype(np.float16)
    _check(c, q)


@pytest.mark.parametrize("kv", [1, 300, 5000, 10 ** 6])
@pytest.mark.parametrize("lens", [[5000], [1, 3000], [2500, 0, 17]])
def test_decode_split(lens, kv):
    """Chunk counts from one to far more than there are tiles."""
    rng = np.random.default_rng(kv + len(lens))
    c = Cache(rng, lens, 2, 64)
    q = (2 * rng.standard_normal((len(lens), 8, D))).astype(np.float16)
    _check(c, q, kv=kv)


@pytest.mark.parametrize("new", [[2, 0, 3, 1], [4, 4, 4, 4], [9, 1, 70, 33], [130, 0, 5, 257]])
@pytest.mark.parametrize("Hq,H", [(4, 1), (8, 8), (32, 8), (40, 8), (18, 2)])
def test_many_query_tokens(new, Hq, H):
    rng = np.random.default_rng(sum(new) + Hq)
    held = [0, 5, 300, 63]
    c = Cache(rng, [h + n for h, n in zip(held, new)], H, 16)
    q = (2 * rng.standard_normal((sum(new) + 3, Hq, D))).astype(np.float16)   # 3 rows of no one
    idx = _starts(new)
    got = _check(c, q, idx, max(new))
    assert (got[-3:] == 7).all()
    # any hint
    again = _attend(c, q, idx, 1)
    want, size = i8_ref.attention(q, *c.table(), idx, None, np.full(q.shape, 7.0))
    _close(again, want, size, max(c.lens))


def test_more_queries_than_tokens():
    """Rows before the first token see nothing and are 0."""
    rng = np.random.default_rng(31)
    c = Cache(rng, [3, 0, 20], 2, 16)
    q = rng.standard_normal((5 + 2 + 4, 4, D)).astype(np.float16)
    got = _check(c, q, _starts([5, 2, 4]), 5)
    assert (got[:2] == 0).all() and (got[5:7] == 0).all() and (got[2] != 0).any()


@pytest.mark.parametrize("sm", [1.0, -0.2, 0.0, 1e-3])
def test_softmax_scales(sm):
    rng = np.random.default_rng(33)
    c = Cache(rng, [50, 200], 2, 16)
    q = (0.5 * rng.standard_normal((2, 8, D))).astype(np.float16)
    _check(c, q, sm=sm)


def test_scales_far_apart_and_zero():
    """Blocks whose V scales differ by many powers of two, zero scales (blocks of
    zeros), and keys so large that one token takes all the weight."""
    rng = np.random.default_rng(34)
    c = Cache(rng, [96, 96, 64], 1, 16)
    for b in range(2):
        for j in range(6):
            pg = c.indices[c.indptr[b] + j]
            c.scale[pg, 1, 1, 0, 0] = np.float32(2.0 ** (4 * j - 20 if b else -4 * j))
    pg = c.indices[c.indptr[2]]
    c.scale[pg, 1] = 0
    c.data[pg, 1] = 0
    c.scale[c.indices[c.indptr[2] + 1], 1, 0] = 3.0
    c.upload()
    q = rng.standard_normal((3, 4, D)).astype(np.float16)
    got = _attend(c, q)
    want, size = i8_ref.attention(q, *c.table())
    for b in range(3):   # each request has its own magnitudes
        _close(got[b], want[b], size[b], 96)


@pytest.mark.parametrize("new", [[257, 130, 65, 20], [9, 40, 33, 1]])
def test_blocks_of_zero_keys(new):
    """Key blocks that hold only zeros (scale 0), among them those that a causal row
    sees in part: their scores are 0, and what is behind the row stays out."""
    rng = np.random.default_rng(sum(new))
    held = [0, 5, 30, 63]
    c = Cache(rng, [h + n for h, n in zip(held, new)], 8, 16)
    for pg in c.indices[::2]:
        c.scale[pg, 1, 0] = 0
        c.data[pg, 1, 0] = 0
    c.upload()
    q = (2 * rng.standard_normal((sum(new), 32, D))).astype(np.float16)
    _check(c, q, _starts(new), max(new))


@pytest.mark.parametrize("new", [None, [9, 40, 33, 1], [257, 130, 65, 20]])
def test_small_values_beside_a_block_of_zeros(new):
    """A block whose values are all 0 (scale 0) takes most of the weight; what the
    others, of scale 2^-15, add keeps its precision."""
    rng = np.random.default_rng(36)
    count = [1] * 4 if new is None else new
    c = Cache(rng, [64 + n for n in count], 8, 16)
    q = rng.standard_normal(D).astype(np.float16)
    c.scale[:, 1, 0] = 1e-4
    c.scale[:, 1, 1] = 2.0 ** -15
    for pg in c.indices[c.indptr[:-1]]:          # the first block of each request
        c.scale[pg, 1, 1] = 0
        c.data[pg, 1, 1] = 0
        c.data[pg, 1, 0] = 100 * np.sign(q).astype(np.int8)
        c.scale[pg, 1, 0] = 4 * D ** 0.5 / (100 * np.abs(q.astype(np.float64)).sum())
    c.upload()
    q = np.broadcast_to(q, (sum(count), 32, D)).copy()
    if new is None:
        _check(c, q)
    else:
        _check(c, q, _starts(new), max(new))


@pytest.mark.parametrize("new,room", [([9, 20, 33, 1], [3, 12, 40, 0]),
                                      ([300, 130, 65, 20], [40, 150, 10, 0])])
def test_rows_that_see_nothing_may_hold_anything(new, room):
    """More queries than tokens: the first rows of a request see none.  They are 0
    whatever they hold, and the rows beside them are as without it."""
    rng = np.random.default_rng(37)
    c = Cache(rng, room, 8, 16)
    q = rng.standard_normal((sum(new), 32, D)).astype(np.float16)
    idx = _starts(new)
    want = _check(c, q, idx, max(new))
    for b, (n, r) in enumerate(zip(new, room)):
        q[idx[b]: idx[b] + max(0, n - r)] = [np.nan, np.inf, 3e4, -np.inf][b]
    got = _attend(c, q, idx, max(new))
    assert np.array_equal(got, want)


def test_what_no_row_sees_does_not_matter():
    """Garbage codes behind the last token, NaN scales of blocks behind it, of
    other heads' V and of unused pages; then a poisoned block that only the later
    rows of a request see."""
    rng = np.random.default_rng(35)
    c = Cache(rng, [20, 37, 5], 2, 64)
    q = rng.standard_normal((3, 4, D)).astype(np.float16)
    first = _check(c, q)
    for b, ln in enumerate(c.lens):
        pg = c.indices[c.indptr[b]]
        c.scale[pg, :, :, :, -(-ln // 16):] = np.nan
        c.data[pg, :, :, :, ln:] = -128
    c.scale[:, 0] = np.nan
    c.upload()
    assert np.array_equal(_attend(c, q), first)
    c = Cache(rng, [40], 1, 16)
    q = rng.standard_normal((30, 2, D)).astype(np.float16)
    idx = _starts([30])
    clean = _attend(c, q, idx, 30)
    for kv in (0, 1):
        d = Cache(rng, [40], 1, 16)
        d.data, d.scale = c.data.copy(), c.scale.copy()
        d.indptr, d.indices, d.last = c.indptr, c.indices, c.last
        d.scale[c.indices[2], 1, kv] = np.nan      # tokens 32 .. 39: rows 22 .. 29
        d.upload()
        got = _attend(d, q, idx, 30)
        assert np.array_equal(got[:22], clean[:22]) and np.isnan(got[22:]).all()


def test_bad_pages_are_not_read():
    rng = np.random.default_rng(36)
    c = Cache(rng, [50, 50, 50], 2, 16)
    c.indices[c.indptr[0] + 1] = -3
    c.indices[c.indptr[1]] = c.data.shape[0]
    c.indices[c.indptr[2]: c.indptr[3]] = 2 ** 30      # nothing left: zeros
    c.upload()
    q = rng.standard_normal((3, 4, D)).astype(np.float16)
    got = _check(c, q)
    assert (got[2] == 0).all()
    # a table whose ends lie outside `indices`, and a last page longer than a page
    c = Cache(rng, [50, 50], 2, 16)
    c.dev[2] = to_dev(np.array([-5, 4, 4000], np.int32))
    c.dev[4] = to_dev(np.array([2, 99], np.int32))
    out = _attend(c, q[:2])
    assert np.isfinite(out).all()


def test_shared_pages_and_same_bits_in_any_batch():
    """A prefix that two requests share, and a request alone against the same one
    in a batch with the same split."""
    rng = np.random.default_rng(37)
    c = Cache(rng, [64, 64], 2, 16)
    c.indices[4:7] = c.indices[:3]
    c.upload()
    q = rng.standard_normal((2, 8, D)).astype(np.float16)
    _check(c, q, kv=64)
    two = _attend(c, q, kv=64)
    c.indptr, c.indices, c.last = c.indptr[:2], c.indices[:4], c.last[:1]
    c.upload()
    assert np.array_equal(_attend(c, q[:1], kv=64)[0], two[0])


@pytest.mark.parametrize("new", [None, [1, 40, 3]])
def test_stream_and_graph(new):
    """append then attention on a side stream, and captured in two graphs that are
    replayed in turn with eager work between; every replay gives the eager bits."""
    rng = np.random.default_rng(38)
    lens = [3000, 500, 41]
    rows = 3 if new is None else sum(new)
    idx = None if new is None else to_dev(_starts(new))
    hint = 1 if new is None else max(new)
    caches = [Cache(rng, lens, 2, 16) for _ in range(2)]
    states = []
    for c in caches:
        k, v = _kv(rng, rows, 2)
        q = rng.standard_normal((rows, 8, D)).astype(np.float16)
        states.append([to_dev(t) for t in (k, v, q)])

    def step(c, s, o):
        _CUDA.append_kv_i8(*c.args(), s[0], s[1], idx, hint)
        _CUDA.batch_attention_i8(o, s[2], *c.args(), idx, hint, 3000)

    want, outs, graphs = [], [], []
    for c, s in zip(caches, states):
        o = torch.zeros_like(s[2])
        step(c, s, o)
        want.append((o, [t.clone() for t in c.dev[:2]]))
        c.upload()                     # as before the append
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = torch.zeros_like(states[0][2])
        step(caches[0], states[0], o)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want[0][0])
    caches[0].upload()
    for c, s in zip(caches, states):
        o = torch.zeros_like(s[2])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(c, s, o)
        outs.append(o)
        graphs.append(g)
    for turn in range(3):
        for i in (1, 0):
            outs[i].zero_()
            torch.randn(1000, 1000, device=DEV).sum()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i][0]), (turn, i)
            assert torch.equal(caches[i].dev[0], want[i][1][0])
            assert torch.equal(caches[i].dev[1], want[i][1][1])


# -------------------------------------------------------------- refusals

def test_refusals():
    rng = np.random.default_rng(40)
    c = Cache(rng, [20, 20], 2, 16)
    data, scale, indptr, indices, last = c.dev
    f16 = dict(dtype=torch.float16, device=DEV)
    k, v = torch.zeros(2, 2, D, **f16), torch.zeros(2, 2, D, **f16)
    q, o = torch.zeros(2, 4, D, **f16), torch.zeros(2, 4, D, **f16)
    qkv, cs = torch.zeros(2, 8 * D, **f16), torch.zeros(1, D, **f16)
    new = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)

    def caches():
        ok = [data, scale, indptr, indices, last, 1]
        for i, t in ((0, data.to(torch.uint8)), (0, data[..., :64].contiguous()), (0, data[0]),
                     (0, data[:, :, :, :, :8].contiguous()), (1, scale.half()),
                     (1, scale[:, :, :, :1].contiguous()), (2, indptr.long()), (2, indptr[:2]),
                     (3, indices.cpu()), (3, indices[None]), (4, last[:1]), (5, 2), (5, -1),
                     (0, data.transpose(3, 4).contiguous().transpose(3, 4))):
            yield ok[:i] + [t] + ok[i + 1:]

    for bad in caches():
        with pytest.raises(RuntimeError):
            _CUDA.append_kv_i8(*bad, k, v)
        with pytest.raises(RuntimeError):
            _CUDA.batch_attention_i8(o, q, *bad)
        with pytest.raises(RuntimeError):
            _CUDA.qkv_norm_rope_append_i8(*bad, qkv, cs, cs, 4)
    a = c.args()
    for args in ((k.float(), v), (k, v[:1]), (k[:1], v[:1]), (k[:, :1], v[:, :1]), (k.cpu(), v),
                 (k[..., ::2], v[..., ::2]), (k, v, new.long()), (k, v, new[:2]),
                 (k.transpose(0, 1).contiguous().transpose(0, 1), v),
                 (k[:1].expand(2, 2, D), v)):
        with pytest.raises(RuntimeError):
            _CUDA.append_kv_i8(*a, *args)
    for args in ((o, q.float()), (o[:1], q), (o, q[:, :3].contiguous()), (o[:1], q[:1]),
                 (o[:, :3].contiguous(), q[:, :3].contiguous()), (o.cpu(), q)):
        with pytest.raises(RuntimeError):
            _CUDA.batch_attention_i8(*args, *a)
    for kw in (dict(q_indptr=new.long()), dict(q_indptr=new[:2]), dict(softmax_scale=float("inf"))):
        with pytest.raises(RuntimeError):
            _CUDA.batch_attention_i8(o, q, *a, **kw)
    for args in ((qkv[:, :-1], cs, cs, 4), (qkv.float(), cs, cs, 4), (qkv, cs, cs, 3),
                 (qkv, cs[:, :64], cs[:, :64], 4), (qkv, cs, cs.float(), 4),
                 (qkv, cs, cs, 4, cs, None), (qkv, cs, cs, 4, cs[0], None, None),
                 (qkv[:1], cs, cs, 4), (qkv, cs.expand(3, D).contiguous(),
                                        cs.expand(3, D).contiguous(), 4)):
        with pytest.raises(RuntimeError):
            _CUDA.qkv_norm_rope_append_i8(*a, *args)
    # nothing was written
    c.assert_same()


def test_empty_batch():
    c = Cache(np.random.default_rng(41), [5], 2, 16)
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    t = (c.dev[0], c.dev[1], one, z, z, 0)
    e = torch.zeros(0, 2, D, dtype=torch.float16, device=DEV)
    _CUDA.append_kv_i8(*t, e, e)
    q = torch.zeros(0, 4, D, dtype=torch.float16, device=DEV)
    assert _CUDA.batch_attention_i8(q, q, *t).shape == q.shape
