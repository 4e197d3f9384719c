"""CPU checks of the plain implementations behind the int8 cache's GPU tests, and
of the entry points' refusals, which come before any device call."""
import ctypes

import numpy as np
import pytest
import torch

from tests import i8_ref

P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    from signrot_amd import _native
    return _native.lib()


def test_append_reference_keeps_values_near():
    """What a block reads as stays within one step of what was appended: half a
    step from the last rounding, and half of each smaller step before it."""
    rng = np.random.default_rng(0)
    data = np.zeros((2, 1, 2, 1, 16, 128), np.int8)
    scale = np.zeros((2, 1, 2, 1, 1), np.float32)
    tab = [np.array(a, np.int32) for a in ([0, 2], [1, 0])]
    rows = []
    for t in range(20):
        x = (rng.standard_normal((2, 1, 1, 128)) * (1 + t)).astype(np.float16)
        rows.append(x)
        last = np.array([t % 16 + 1], np.int32)
        tab[0][1] = 1 + t // 16
        i8_ref.append(data, scale, *tab, last, 0, x[0], x[1])
    k = np.concatenate([r[0] for r in rows])[:, 0].astype(np.float64)
    got = np.concatenate([data[1, 0, 0, 0] * np.float64(scale[1, 0, 0, 0, 0]),
                          data[0, 0, 0, 0, :4] * np.float64(scale[0, 0, 0, 0, 0])])
    step = np.repeat([scale[1, 0, 0, 0, 0], scale[0, 0, 0, 0, 0]], [16, 4])[:, None]
    moves = np.arange(20)[:, None] % 16          # at most this many later roundings
    assert (np.abs(got - k) <= step * 0.5 * (1 + 16 - moves) + 1e-12).all()
    assert scale[1, 0, 0, 0, 0] == np.float32(np.abs(k[:16]).max()) * (
        np.float32(1) / np.float32(127))


def test_attention_reference_against_softmax():
    rng = np.random.default_rng(1)
    tab = i8_ref.table([37], 16, rng)
    data = rng.integers(-127, 128, (tab[3], 1, 2, 2, 16, 128)).astype(np.int8)
    scale = rng.uniform(0.01, 0.02, (tab[3], 1, 2, 2, 1)).astype(np.float32)
    q = rng.standard_normal((5, 4, 128)).astype(np.float16)
    out, _ = i8_ref.attention(q, data, scale, *tab[:3], 0, np.array([0, 5]))
    val = torch.from_numpy(data * scale[..., None].astype(np.float64))[tab[1], 0]
    val = val.permute(1, 2, 0, 3, 4).reshape(2, 2, -1, 128)[:, :, :37]
    for h in range(4):
        x = torch.from_numpy(q[:, h].astype(np.float64)) @ val[0, h // 2].T / 128 ** 0.5
        late = torch.arange(37)[None] > torch.arange(32, 37)[:, None]
        w = torch.softmax(x.masked_fill(late, -torch.inf), -1)
        assert np.allclose(out[:, h], (w @ val[1, h // 2]).numpy(), rtol=1e-12, atol=1e-12)


def _cache(batch=2, L=1, layer=0, H=2, page=16, D=128, pages=4, n=4, data=P):
    return [data, P, P, P, P, pages, n, batch, L, layer, H, page, D]


APPEND = [P, P, 256, 256, 2, None, 1, None]
ATTEND = [None, 1, 100, ctypes.c_float(0.1), P, 1 << 20, None]


@pytest.mark.parametrize("kw,msg", [
    (dict(D=64), "head_dim"), (dict(page=24), "multiple of 16"), (dict(page=0), "multiple of 16"),
    (dict(layer=1), "layer_idx"), (dict(layer=-1), "layer_idx"), (dict(batch=70000), "batch"),
    (dict(pages=0), "no pages"), (dict(data=None), "null"), (dict(H=0), "KV heads"),
    (dict(data=ctypes.c_void_p(8)), "aligned"), (dict(n=1 << 30), "2\\^31"),
    (dict(pages=-1), "negative")])
def test_cache_refusals(lib, kw, msg):
    import re
    calls = (lambda c: lib.srq_append_kv_i8(*c, *APPEND),
             lambda c: lib.srq_batch_attention_i8(P, P, 2, 4, *c, *ATTEND),
             lambda c: lib.srq_qkv_norm_rope_append_i8(*c, P, 1024, 2, P, P, 1, 4, None, None,
                                                       ctypes.c_float(1e-6), 1, None, 1, P, None))
    for call in calls:
        assert call(_cache(**kw)) == -1
        assert re.search(msg, lib.srq_last_error().decode())


@pytest.mark.parametrize("args,msg", [
    ([P, P, 256, 256, 3, None, 1, None], "3 rows"), ([None, P, 256, 256, 2, None, 1, None], "null"),
    ([P, P, 128, 256, 2, None, 1, None], "strides"),
    ([P, P, 260, 256, 2, None, 1, None], "strides"),
    ([ctypes.c_void_p(8), P, 256, 256, 2, None, 1, None], "aligned"),
    ([P, P, 256, 256, -1, P, 1, None], "rows")])
def test_append_refusals(lib, args, msg):
    assert lib.srq_append_kv_i8(*_cache(), *args) == -1
    assert msg in lib.srq_last_error().decode()


def test_attention_refusals(lib):
    def call(o=P, q=P, rows=2, hq=4, scale=0.1, idx=None, ws=P, n=1 << 20, kv=100):
        return lib.srq_batch_attention_i8(o, q, rows, hq, *_cache(), idx, 1, kv,
                                          ctypes.c_float(scale), ws, n, None)
    for kw, msg in ((dict(hq=3), "query heads"), (dict(hq=0), "query heads"),
                    (dict(scale=3e38), "finite"),
                    (dict(rows=3), "3 rows"), (dict(scale=float("nan")), "finite"),
                    (dict(o=None), "null"), (dict(q=ctypes.c_void_p(8)), "aligned"),
                    (dict(rows=1 << 30, idx=P), "2^31"), (dict(kv=10000, ws=None), "workspace"),
                    (dict(kv=10000, n=16), "workspace")):
        assert call(**kw) == -1
        assert msg in lib.srq_last_error().decode()
    n = ctypes.c_int64()
    assert lib.srq_batch_attention_i8_workspace(2, 2, 5, 2, 1, 100, ctypes.byref(n)) == -1
    assert lib.srq_batch_attention_i8_workspace(2, 2, 4, 2, 1, 100, None) == -1
    # a hint of one token for a request of 100000 does not split all of its rows
    assert lib.srq_batch_attention_i8_workspace(100000, 1, 32, 8, 1, 100000, ctypes.byref(n)) == 0
    assert n.value == 0


def test_norm_rope_refusals(lib):
    def call(D=128, cb=1, eps=1e-6, norm=1, w=None, tok=512, q=P, seq=2048, B=1, T=4):
        return lib.srq_qk_norm_rope(q, P, P, P, cb, w, None, ctypes.c_float(eps), norm, B, T, 4, 2,
                                    D, tok, seq, tok, seq, P, P, None)
    for kw, msg in ((dict(D=96), "head_dim"), (dict(cb=2), "batch"), (dict(eps=-1.0), "eps"),
                    (dict(eps=float("inf")), "eps"), (dict(norm=0, w=P), "without"),
                    (dict(tok=256), "strides"), (dict(tok=516), "multiples"),
                    (dict(q=ctypes.c_void_p(8)), "aligned"), (dict(q=None), "null"),
                    (dict(B=-1), "shape"), (dict(T=1 << 24), "2^24")):
        assert call(**kw) == -1, kw
        assert msg in lib.srq_last_error().decode(), kw
    assert call(T=0, q=None) == 0


def test_linear_refusals(lib):
    def call(M=1, N=16, K=128, group=64, x=P, w=P, out=P):
        return lib.srq_w4a16_linear(x, w, P, None, None, M, N, K, group, out, None)
    for kw, msg in ((dict(group=48), "multiple of 32"), (dict(K=100), "divides"),
                    (dict(group=0), "multiple"), (dict(M=-1), "negative"), (dict(x=None), "null"),
                    (dict(w=ctypes.c_void_p(8)), "aligned"), (dict(M=1 << 21), "range"),
                    (dict(N=(1 << 26) + 1), "range")):
        assert call(**kw) == -1, kw
        assert msg in lib.srq_last_error().decode(), kw
    assert call(M=0, x=None) == 0 and call(N=0) == 0
