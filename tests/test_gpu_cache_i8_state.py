"""MultiLayerPagedKVCache8Bit on the GPU where its state could go wrong: uneven pieces
behind the prefill, refused calls, frozen index tensors (tests/test_host_cache_i8.py
has the cases; here the launches themselves run)."""
import pytest
import torch

from signrot_amd.functional import kernel
from signrot_amd.transformers import (HFCacheAdapter, MultiLayerPagedKVCache4Bit,
                                      MultiLayerPagedKVCache8Bit)
from signrot_amd.transformers import decode_layer as dl
from tests import i8_ref
from tests.gpu_util import DEV, to_np
from tests.test_gpu_kv_cache_i8 import _cache, _gen, _layer, _rand, _state
from tests.test_gpu_kv_i8 import _close

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("T", [1, 9, 40])
def test_padding_of_a_later_piece_stays_out(T):
    """Codes and scales of an uneven piece are those of the same tokens appended
    request by request; its attention is that of 64 bits over them."""
    B, H, Hq, g = 3, 2, 8, _gen(T)
    cache = MultiLayerPagedKVCache8Bit(B, 64, 64, DEV, 1, H, D)
    mask = torch.ones(B, 20, dtype=torch.int64, device=DEV)
    mask[2, :3] = 0
    k0, v0 = _rand(g, B, 20, H, D), _rand(g, B, 20, H, D)
    cache.update(k0, v0, 0, {"attention_mask": mask})
    new = torch.ones(B, T, dtype=torch.int64, device=DEV)
    new[1, : max(1, T // 2)] = 0
    if T > 1:
        new[2, :1] = 0
    mask = torch.cat([mask, new], 1)
    k, v, q = _rand(g, B, T, H, D), _rand(g, B, T, H, D), _rand(g, B, T, Hq, D)
    for t in (k, v, q):
        t[new == 0] = float("nan")
    got = cache.update(k, v, 0, {"attention_mask": mask})(q)
    st = _state(cache, 0)
    assert i8_ref.lengths(st[2], st[4], 64).tolist() == mask.sum(1).tolist()
    starts = torch.cat([new.new_zeros(1), new.sum(1).cumsum(0)])
    want, size = i8_ref.attention(to_np(q[new != 0]), *st, to_np(starts))
    _close(to_np(got[new != 0]), want, size, 64)
    assert (got[new == 0] == 0).all()
    for b in range(B):
        alone = MultiLayerPagedKVCache8Bit(1, 64, 64, DEV, 1, H, D)
        first, live, n = mask[b, :20] != 0, new[b] != 0, int(mask[b].sum())
        alone.update(k0[b: b + 1, first], v0[b: b + 1, first], 0)
        if live.any():
            alone.update(k[b: b + 1, live], v[b: b + 1, live], 0)
        page = int(st[3][st[2][b]])
        assert torch.equal(cache.pages[page, 0, :, :, :n], alone.pages[0, 0, :, :, :n])
        assert torch.equal(cache.scales[page, 0, :, :, : -(-n // 16)],
                           alone.scales[0, 0, :, :, : -(-n // 16)])


def test_index_tensors_after_refused_calls_and_resets():
    B, H, g = 2, 2, _gen(3)
    cache = MultiLayerPagedKVCache8Bit(B, 16, 32, DEV, 1, H, D)
    k, q = _rand(g, B, 14, H, D), _rand(g, B, 1, 4, D)
    cos = torch.ones(1, 9, D, dtype=torch.float16, device=DEV)
    assert (cache.attend(q, 0) == 0).all()
    cache.update(k, k, 0)
    want, st = cache.attend(q, 0), _state(cache, 0)
    many = torch.zeros(B, 300, H, D, device=DEV)
    for call in (lambda: cache.update(k[:, :9].float(), k[:, :9].float(), 0),
                 lambda: cache.update(many, many, 0),
                 lambda: cache.update_qkv(_rand(g, B, 9, 7 * D), cos, cos, 0, 4),
                 lambda: cache.refresh_specs(10 ** 6)):
        with pytest.raises(RuntimeError):
            call()
        now = _state(cache, 0)
        assert all((a[: len(b)] == b).all() for a, b in zip(now[2:5:2], st[2:5:2]))
        assert torch.equal(cache.attend(q, 0), want)
    copy = cache.clone()
    cache.reset()
    assert (cache.attend(q, 0) == 0).all()
    copy.mark_prefilled(14)
    assert torch.equal(copy.attend(q, 0), want)


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("cls", [MultiLayerPagedKVCache4Bit, MultiLayerPagedKVCache8Bit])
@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("wrap", [False, True])
def test_a_refused_prefill_leaves_the_cache(qk_norm, cls, T, wrap):
    """A prefill of a layer that has its context, fused and op by op: nothing is
    stored or counted, and the next decode step is as without it."""
    layer, B, g = _layer(qk_norm), 2, _gen(4)
    h = _rand(g, B, 20, 1024)
    cos, sin = dl.rope_cos_sin(range(20), D, 10000.0, DEV)
    caches = [_cache(cls, B, 64) for _ in range(2)]
    for c in caches:
        c.pages.zero_()
        layer.prefill(h.clone(), c, cos, sin)
    c = HFCacheAdapter(caches[0]) if wrap else caches[0]
    for trace in (None, {}):
        with pytest.raises((RuntimeError, ValueError)):
            layer.prefill(h[:, :T].clone(), c, cos[:, :T], sin[:, :T], trace=trace)
        assert caches[0].length == 20
    assert torch.equal(caches[0].pages[: B], caches[1].pages[: B])
    cos, sin = dl.rope_cos_sin([20], D, 10000.0, DEV)
    outs = [layer(h[:, :1].clone(), c, cos, sin) for c in caches]
    assert torch.equal(*outs) and caches[0].length == 21


@pytest.mark.parametrize("page", [16, 32, 64])
def test_update_qkv_stores_the_bits_of_the_two_calls(page):
    """Codes of every held token and scales of every block that holds one, in pages of
    one block and of several."""
    B, H, Hq, g = 2, 2, 8, _gen(page)
    caches = [MultiLayerPagedKVCache8Bit(B, page, 100, DEV, 1, H, D) for _ in range(2)]
    w = [(1 + 0.2 * torch.randn(D, device=DEV, generator=g)).half() for _ in range(2)]
    pos = 0
    for T in (40, 1, 17, 1, 30):
        qkv = _rand(g, B, T, (Hq + 2 * H) * D)
        cos, sin = dl.rope_cos_sin(range(pos, pos + T), D, 10000.0, DEV)
        caches[0].update_qkv(qkv, cos, sin, 0, Hq, *w, 1e-6)
        heads = qkv.view(B, T, -1, D)
        _, k = kernel.qk_norm_rope(heads[:, :, :Hq], heads[:, :, Hq: Hq + H], cos, sin, *w, 1e-6)
        caches[1].update(k, heads[:, :, Hq + H:], 0)
        pos += T
        held = []
        for c in caches:
            pg = c.specs()["kv_indices"][: -(-pos // page) * B].view(B, -1).long()
            codes = c.pages[pg, 0].permute(0, 2, 3, 1, 4, 5).reshape(B, 2, H, -1, D)
            scales = c.scales[pg, 0].permute(0, 2, 3, 1, 4).reshape(B, 2, H, -1)
            held.append((codes[:, :, :, :pos], scales[..., : -(-pos // 16)]))
        assert all(torch.equal(a, b) for a, b in zip(*held)), T
