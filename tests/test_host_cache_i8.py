"""MultiLayerPagedKVCache8Bit and the decode layer's use of it on the CPU: what goes
into the pool, what the index tensors say and what is refused, with the plain append
and attention (tests/i8_ref.py) in the place of the two launches."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA
from signrot_amd.transformers import MultiLayerPagedKVCache8Bit
from tests import i8_ref

D = 128


def _np(t):
    return None if t is None else t.numpy()


@pytest.fixture(autouse=True)
def plain_ops(monkeypatch):
    """append_kv_i8, qkv_norm_rope_append_i8 (without a norm or a rotation) and
    batch_attention_i8 on host tensors."""
    def append(kv_data, kv_scale, kv_indptr, kv_indices, last_page_offset, layer_idx, k, v,
               new_indptr=None, max_new=None):
        if k.dtype != torch.float16:
            raise RuntimeError("append_kv_i8: k must be fp16")
        i8_ref.append(_np(kv_data), _np(kv_scale), _np(kv_indptr), _np(kv_indices),
                      _np(last_page_offset), layer_idx, _np(k), _np(v), _np(new_indptr))

    def qkv_append(kv_data, kv_scale, kv_indptr, kv_indices, last_page_offset, layer_idx, qkv, cos,
                   sin, n_q_heads, q_weight=None, k_weight=None, eps=None, new_indptr=None,
                   max_new=None):
        H = kv_data.shape[3]
        if qkv.shape[1] != (n_q_heads + 2 * H) * D:
            raise RuntimeError("qkv_norm_rope_append_i8: columns")
        q, k, v = qkv.view(len(qkv), -1, D).split((n_q_heads, H, H), dim=1)
        append(kv_data, kv_scale, kv_indptr, kv_indices, last_page_offset, layer_idx,
               k.contiguous(), v.contiguous(), new_indptr)
        return q.contiguous()

    def attend(o, q, kv_data, kv_scale, kv_indptr, kv_indices, last_page_offset, layer_idx,
               q_indptr=None, max_q_len=None, max_kv_len=None, softmax_scale=None):
        out, _ = i8_ref.attention(_np(q), _np(kv_data), _np(kv_scale), _np(kv_indptr),
                                  _np(kv_indices), _np(last_page_offset), layer_idx, _np(q_indptr),
                                  softmax_scale, _np(o))
        return o.copy_(torch.from_numpy(out))

    monkeypatch.setattr(_CUDA, "append_kv_i8", append)
    monkeypatch.setattr(_CUDA, "qkv_norm_rope_append_i8", qkv_append)
    monkeypatch.setattr(_CUDA, "batch_attention_i8", attend)


def _cache(B, page=16, most=64, H=2, layers=1):
    return MultiLayerPagedKVCache8Bit(B, page, most, "cpu", layers, H, D)


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).half()


def _held(cache, layer=0):
    """The values of each request [2, H, len, D] and its length, from the index
    tensors as they stand."""
    t = cache.specs()
    ptr, idx, last = (t[n].tolist() for n in ("kv_indptr", "kv_indices", "last_page_offset"))
    out = []
    for b in range(cache.batch_size):
        pg = idx[ptr[b]: ptr[b + 1]]
        n = (len(pg) - 1) * cache.page_size + last[b] if pg else 0
        val = cache.pages[pg, layer].double().unflatten(3, (-1, 16)) * \
            cache.scales[pg, layer].double()[..., None, None]
        out.append(val.flatten(3, 4).permute(1, 2, 0, 3, 4).reshape(2, cache.num_heads, -1, D)
                   [:, :, :n])
    return out


# ------------------------------------------------- masks behind the prefill

@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("masked_prompt", [False, True])
def test_padding_of_a_later_piece_stays_out(T, masked_prompt):
    """An uneven piece behind the prefill: the mask's zeros in its new columns are not
    stored, nothing that was held before is written over, and the piece's queries see
    what the same tokens, appended request by request, let them see."""
    B, H, Hq = 3, 2, 4
    cache = _cache(B)
    mask = torch.ones(B, 8, dtype=torch.int64)
    if masked_prompt:
        mask[2, :3] = 0
    k0, v0 = _rand(1, B, 8, H, D), _rand(2, B, 8, H, D)
    cache.update(k0, v0, 0, {"attention_mask": mask} if masked_prompt else None)
    before = _held(cache)
    new = torch.ones(B, T, dtype=torch.int64)
    new[1, : max(1, T // 2)] = 0
    if T > 1:
        new[2, :1] = 0
    mask = torch.cat([mask, new], 1)
    k, v, q = _rand(3, B, T, H, D), _rand(4, B, T, H, D), _rand(5, B, T, Hq, D)
    bad = [t.clone() for t in (k, v, q)]
    for t in bad:
        t[new == 0] = float("nan")
    got = cache.update(bad[0], bad[1], 0, {"attention_mask": mask})(bad[2])
    held = _held(cache)
    for b in range(B):
        n, live = int(mask[b].sum()), new[b] != 0
        assert held[b].shape[2] == n
        alone = _cache(1)
        first = mask[b, :8] != 0
        alone.update(k0[b: b + 1, first], v0[b: b + 1, first], 0)
        if live.any():
            o = alone.update(k[b: b + 1, live], v[b: b + 1, live], 0)(q[b: b + 1, live])
            assert torch.equal(got[b, live], o[0])
        assert torch.equal(held[b], _held(alone)[0])
        assert (got[b, ~live] == 0).all()
        if not live.any():
            assert torch.equal(held[b], before[b])


def test_masks_that_do_not_fit_are_refused():
    B, H = 2, 2
    cache = _cache(B)
    k = _rand(1, B, 8, H, D)
    one = torch.ones(B, 20, dtype=torch.int64)
    for m in (one[:, :7], one[:, :9], one[:1, :8], one[0, :8]):
        with pytest.raises(ValueError):
            cache.update(k, k, 0, {"attention_mask": m})
    cache.update(k, k, 0, {"attention_mask": one[:, :8]})
    before = _held(cache)
    # of the new tokens alone, or of the held ones alone
    for m in (one[:, :4], one[:, :8], one[:1, :12]):
        with pytest.raises(ValueError):
            cache.update(k[:, :4], k[:, :4], 0, {"attention_mask": m})
    cos = torch.ones(1, 4, D, dtype=torch.float16)
    qkv = _rand(2, B, 4, 8 * D)
    pad = one[:, :12].clone()
    pad[1, 8] = 0
    for m in (one[:, :4], pad):
        with pytest.raises(ValueError):
            cache.update_qkv(qkv, cos, cos, 0, 4, attention_mask=m)
    assert cache.length == 8
    assert all(torch.equal(a, b) for a, b in zip(before, _held(cache)))
    q = cache.update_qkv(qkv, cos, cos, 0, 4, attention_mask=one[:, :12])
    assert q.shape == (B, 4, 4, D) and cache.length == 12


# ------------------------------------------ index tensors and the length agree

def _unchanged(cache, call, error):
    """A refused call leaves length, index tensors and what they show."""
    length, before = cache.length, _held(cache)
    q = _rand(90, cache.batch_size, 1, 4, D)
    want = cache.attend(q, 0)
    with pytest.raises(error):
        call()
    assert cache.length == length
    got = _held(cache)
    assert all(torch.equal(a, b) for a, b in zip(got, before))
    assert torch.equal(cache.attend(q, 0), want)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("masked", [False, True])
def test_a_refused_update_leaves_the_index_tensors(page, masked):
    B, H = 2, 2
    cache = _cache(B, page)
    k = _rand(1, B, 14, H, D)
    mask = torch.ones(B, 14, dtype=torch.int64)
    mask[1, :5] = 0
    cache.update(k, k, 0, {"attention_mask": mask} if masked else None)
    cos = torch.ones(1, 9, D, dtype=torch.float16)
    kw = {}
    if masked:
        mask = torch.cat([mask, torch.ones(B, 9, dtype=torch.int64)], 1)
        kw = {"attention_mask": mask}
    refused = (RuntimeError, ValueError, NotImplementedError)
    f = k[:, :9].float()
    _unchanged(cache, lambda: cache.update(f, f, 0, kw), refused)
    _unchanged(cache, lambda: cache.update_qkv(_rand(2, B, 9, 7 * D), cos, cos, 0, 4, **kw),
               refused)
    # a growth of the pool on the way
    many = k[:, :1].float().expand(B, 300, H, D)
    _unchanged(cache, lambda: cache.update(many, many, 0), refused)
    if page == 16:   # requests that would need unlike numbers of pages
        uneven = torch.ones(B, 23, dtype=torch.int64)
        uneven[1, :20] = 0
        _unchanged(cache, lambda: cache.update(k[:, :9], k[:, :9], 0,
                                               {"attention_mask": uneven}), refused)
    _unchanged(cache, lambda: cache.refresh_specs(10 ** 6), refused)
    out = cache.update(k[:, :9], k[:, :9], 0, kw)
    assert cache.length == 23 and callable(out)


def test_the_index_tensors_follow_every_length():
    """A new cache, one declared full and one reset, asked before their next update."""
    B, q = 2, _rand(3, 2, 1, 4, D)
    cache = _cache(B)
    assert (cache.attend(q, 0) == 0).all()
    k = _rand(4, B, 20, 2, D)
    cache.update(k, k, 0)
    want = cache.attend(q, 0)
    other = _cache(B)
    other.pages.copy_(cache.pages)
    other.scales.copy_(cache.scales)
    other.mark_prefilled(20)
    assert torch.equal(other.attend(q, 0), want)
    copy = cache.clone()
    cache.reset()
    assert (cache.attend(q, 0) == 0).all() and torch.equal(copy.attend(q, 0), want)
    # frozen index tensors are the program's own
    copy.freeze_specs(True)
    copy.reset()
    assert torch.equal(copy.attend(q, 0), want)


def test_a_frozen_step_keeps_the_pool():
    """Passes over frozen index tensors (the warm-up of a captured step) write the same
    slot each time; counted past the pool's end, they neither move nor lose it."""
    B, q = 2, _rand(7, 2, 1, 4, D)
    cache = _cache(B, most=32)
    k = _rand(8, B, 31, 2, D)
    cache.update(k, k, 0)
    cache.refresh_specs(32)
    cache.freeze_specs(True)
    pool, tables = cache.pages, dict(cache.specs())
    k1, v1 = _rand(9, B, 1, 2, D), _rand(10, B, 1, 2, D)
    outs = [cache.update(k1, v1, 0)(q) for _ in range(4)]
    assert all(torch.equal(o, outs[0]) for o in outs)
    assert cache.pages is pool and all(t is cache.specs()[n] for n, t in tables.items())
    # set free, it grows as ever
    cache.freeze_specs(False)
    cache.mark_prefilled(32)
    assert torch.equal(cache.attend(q, 0), outs[0])
    cache.update(k1, v1, 0)
    assert cache.pages.shape[0] > pool.shape[0] and cache.length == 33


@pytest.mark.parametrize("heads,kv", [(6, 2), (3, 2), (128, 2), (2, 4)])
def test_a_refused_decode_step_stores_nothing(heads, kv):
    """Query heads that the attention or the head-axis rotation behind it does not
    take are refused before the token goes into the cache."""
    B = 2
    cache = _cache(B, H=kv)
    k = _rand(1, B, 5, kv, D)
    cache.update(k, k, 0)
    pages, scales, before = cache.pages.clone(), cache.scales.clone(), _held(cache)
    cos = torch.ones(1, 1, D, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="heads"):
        cache.update_qkv_decode_quant(_rand(2, B, (heads + 2 * kv) * D), cos, cos, 0, heads, 1.0)
    assert cache.length == 5 and torch.equal(cache.pages, pages)
    assert torch.equal(cache.scales.view(torch.int32), scales.view(torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(before, _held(cache)))


@pytest.mark.parametrize("sm", [float("nan"), float("inf"), 1e20, 1e-7, -1e-40])
def test_softmax_scales_are_checked_when_the_cache_is_made(sm):
    """And not by the attention, when the token is in the cache already."""
    with pytest.raises(ValueError, match="softmax_scale"):
        MultiLayerPagedKVCache8Bit(1, 16, 16, "cpu", 1, 1, D, softmax_scale=sm)
    for ok in (None, 0.0, 2.0 ** -20, -0.125, 2.0 ** 60):
        MultiLayerPagedKVCache8Bit(1, 16, 16, "cpu", 1, 1, D, softmax_scale=ok)


def test_who_refuses_a_second_prefill():
    """The layer for the caches' own update(), also behind the adapter; an update() that
    a program has put in place is asked itself."""
    from signrot_amd.transformers import HFCacheAdapter
    from signrot_amd.transformers.decode_layer import _refuse_held

    class Rewinds(HFCacheAdapter):
        def update(self, *args):
            self.inner.reset()
            return super().update(*args)

    class Own(MultiLayerPagedKVCache8Bit):
        def update(self, *args):
            return super().update(*args)

    cache, own = _cache(1), Own(1, 16, 64, "cpu", 1, 2, D)
    for c in (cache, HFCacheAdapter(cache), own):
        _refuse_held(c, 0, 4)
    k = _rand(1, 1, 4, 2, D)
    for c in (cache, own):
        c.update(k, k, 0)
    for c in (cache, HFCacheAdapter(cache)):
        with pytest.raises(RuntimeError, match="already holds"):
            _refuse_held(c, 0, 4)
    for c in (own, Rewinds(cache), object()):
        _refuse_held(c, 0, 4)


@pytest.mark.parametrize("pads", [(0, 5), (3, 3)])
def test_padded_requests_go_on_with_their_mask(pads):
    """Without it every request would count as long as the padded prompt, and what lies
    behind the shorter ones is nothing that was stored; a mask of ones may be left out."""
    B = 2
    k, q = _rand(1, B, 14, 2, D), _rand(2, B, 1, 4, D)
    cos = torch.ones(1, 1, D, dtype=torch.float16)
    mask = torch.ones(B, 14, dtype=torch.int64)
    whole = _cache(B, layers=2)
    for layer in range(2):
        whole.update(k, k, layer, {"attention_mask": mask})
    plain = _cache(B, layers=2)
    for layer in range(2):
        plain.update(k, k, layer)
    outs = [c.update(k[:, :1], k[:, :1], 0)(q) for c in (whole, plain)]
    assert torch.equal(*outs)
    for b, n in enumerate(pads):
        mask[b, :n] = 0
    cache = _cache(B, layers=2)
    cache.update(k, k, 0, {"attention_mask": mask})
    refused = (ValueError,)
    _unchanged(cache, lambda: cache.update(k, k, 1), refused)
    cache.update(k, k, 1, {"attention_mask": mask})
    _unchanged(cache, lambda: cache.update(k[:, :1], k[:, :1], 0), refused)
    _unchanged(cache, lambda: cache.update_qkv(_rand(3, B, 1, 8 * D), cos, cos, 0, 4), refused)
    longer = torch.cat([mask, torch.ones(B, 1, dtype=torch.int64)], 1)
    cache.update(k[:, :1], k[:, :1], 0, {"attention_mask": longer})
    assert [h.shape[2] for h in _held(cache)] == [15 - n for n in pads]
    # its own index tensors while frozen, and a fresh start after reset
    cache.freeze_specs(True)
    cache.update(k[:, :1], k[:, :1], 1)
    cache.reset()
    cache.freeze_specs(False)
    cache.update(k, k, 0)
    assert [h.shape[2] for h in _held(cache)] == [14, 14]
