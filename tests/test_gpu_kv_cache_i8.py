"""MultiLayerPagedKVCache8Bit, the decode layer over it and with q/k norms, and an
attention block of grouped 4-bit linears, q/k norms and the int8 cache as a program
runs them: stages against plain 64-bit implementations on the same inputs, fused
forms against the ops they stand for."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA, nn
from signrot_amd.functional import kernel
from signrot_amd.transformers import MultiLayerPagedKVCache4Bit, MultiLayerPagedKVCache8Bit
from signrot_amd.transformers import decode_layer as dl
from tests import i8_ref
from tests.gpu_util import DEV, to_np
from tests.test_gpu_kv_i8 import _close

pytestmark = pytest.mark.gpu
D = 128


def _rand(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g).half()


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _state(cache, layer):
    t = cache.specs()
    return (to_np(cache.pages), to_np(cache.scales), to_np(t["kv_indptr"]), to_np(t["kv_indices"]),
            to_np(t["last_page_offset"]), layer)


def _check_attend(cache, layer, q, got):
    """attention of q [B, T, Hq, D] over what the cache holds now."""
    B, T, Hq, _ = q.shape
    new = np.arange(B + 1) * T
    want, size = i8_ref.attention(to_np(q).reshape(B * T, Hq, D), *_state(cache, layer), new)
    _close(to_np(got).reshape(B * T, Hq, D), want, size, cache.length)


def _follow(ref, cache, layer, k, v):
    """The same append on a host copy of the pool."""
    B, T = k.shape[:2]
    st = _state(cache, layer)
    i8_ref.append(*ref, *st[2:5], layer, to_np(k).reshape(B * T, *k.shape[2:]),
                  to_np(v).reshape(B * T, *k.shape[2:]), np.arange(B + 1) * T)
    for b in range(B):   # only pages of the table are compared
        pg = st[3][st[2][b]: st[2][b + 1]]
        n = cache.length
        codes = [x[pg, layer].transpose(1, 2, 0, 3, 4).reshape(2, -1, len(pg) * cache.page_size, D)
                 for x in (ref[0], st[0])]
        assert np.array_equal(codes[0][:, :, :n], codes[1][:, :, :n])
        sc = [x[pg, layer].transpose(1, 2, 0, 3).reshape(2, k.shape[2], -1)
              for x in (ref[1], st[1])]
        assert np.array_equal(sc[0][:, :, : -(-n // 16)], sc[1][:, :, : -(-n // 16)])


@pytest.mark.parametrize("page", [16, 64])
def test_update_pieces_and_tokens(page):
    """A prompt, two further pieces and single tokens over two layers; the pool
    grows on the way."""
    B, H, Hq, g = 3, 2, 8, _gen(page)
    cache = MultiLayerPagedKVCache8Bit(B, page, 40, DEV, 2, H, D)
    ref = None
    for T in (21, 1, 1, 34, 1, 150, 1):
        for layer in range(2):
            k, v, q = _rand(g, B, T, H, D), _rand(g, B, T, H, D), _rand(g, B, T, Hq, D)
            out = cache.update(k, v, layer)
            if ref is None or ref[0].shape != tuple(cache.pages.shape):
                fresh = [np.zeros(cache.pages.shape, np.int8),
                         np.zeros(cache.scales.shape, np.float32)]
                for new, old in zip(fresh, ref or ()):
                    new[: len(old)] = old
                ref = fresh
            _follow(ref, cache, layer, k, v)
            if T == 21:
                assert out[0] is k and out[1] is v
            else:
                _check_attend(cache, layer, q, out(q))
    assert cache.length == 209 and cache.get_seq_length() == 209 and len(cache) == 2


def test_update_qkv_is_norm_append_and_attend():
    B, H, Hq, g = 2, 2, 8, _gen(1)
    caches = [MultiLayerPagedKVCache8Bit(B, 32, 100, DEV, 1, H, D) for _ in range(2)]
    w = [(1 + 0.2 * torch.randn(D, device=DEV, generator=g)).half() for _ in range(2)]
    pos = 0
    for T, cb in ((40, 1), (1, 1), (17, B), (1, B)):
        qkv = _rand(g, B, T, (Hq + 2 * H) * D)
        cos, sin = dl.rope_cos_sin(range(pos, pos + T), D, 10000.0, DEV)
        cos, sin = cos.expand(cb, T, D), sin.expand(cb, T, D)
        q = caches[0].update_qkv(qkv, cos, sin, 0, Hq, *w, 1e-6)
        heads = qkv.view(B, T, -1, D)
        q2, k2 = kernel.qk_norm_rope(heads[:, :, :Hq], heads[:, :, Hq: Hq + H], cos, sin, *w, 1e-6)
        caches[1].update(k2, heads[:, :, Hq + H:], 0)
        assert torch.equal(q, q2)
        a, b = (_state(c, 0) for c in caches)
        used = a[3][: a[2][-1]]
        assert np.array_equal(a[1][used][..., :1], b[1][used][..., :1])
        _check_attend(caches[0], 0, q, caches[0].attend(q, 0))
        assert torch.equal(caches[0].attend(q, 0), caches[1].attend(q, 0))
        pos += T


def test_clone_and_mark_prefilled():
    g = _gen(11)
    a = MultiLayerPagedKVCache8Bit(2, 16, 64, DEV, 1, 2, D)
    k, q = _rand(g, 2, 20, 2, D), _rand(g, 2, 1, 4, D)
    a.update(k, k, 0)
    b = a.clone()
    c = MultiLayerPagedKVCache8Bit(2, 16, 64, DEV, 1, 2, D)
    c.pages.copy_(a.pages)
    c.scales.copy_(a.scales)
    c.mark_prefilled(20)
    before = a.pages.clone()
    outs = [x.update(k[:, :1], k[:, 1:2], 0)(q) for x in (b, c)]
    assert torch.equal(a.pages, before) and a.length == 20 and b.length == c.length == 21
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(a.update(k[:, :1], k[:, 1:2], 0)(q), outs[0])


def test_left_padded_prefill_then_decode():
    B, T, H, Hq, g = 3, 20, 2, 4, _gen(2)
    cache = MultiLayerPagedKVCache8Bit(B, 32, 40, DEV, 1, H, D)
    mask = torch.ones(B, T, dtype=torch.int64, device=DEV)
    mask[1, :7], mask[2, :3] = 0, 0
    k, v = _rand(g, B, T, H, D), _rand(g, B, T, H, D)
    k[1, :7] = float("nan")          # padding never reaches the cache
    cache.update(k, v, 0, {"attention_mask": mask})
    for _ in range(3):
        mask = torch.cat([mask, torch.ones(B, 1, dtype=torch.int64, device=DEV)], 1)
        k1, v1, q = _rand(g, B, 1, H, D), _rand(g, B, 1, H, D), _rand(g, B, 1, Hq, D)
        attend = cache.update(k1, v1, 0, {"attention_mask": mask})
        st = _state(cache, 0)
        assert i8_ref.lengths(st[2], st[4], 32).tolist() == mask.sum(1).tolist()
        want, size = i8_ref.attention(to_np(q)[:, 0], *st)
        _close(to_np(attend(q))[:, 0], want, size, 30)


def test_refused_updates_leave_the_cache():
    cache = MultiLayerPagedKVCache8Bit(2, 16, 32, DEV, 1, 2, D)
    g = _gen(3)
    k = _rand(g, 2, 5, 2, D)
    cache.update(k, k, 0)
    cos = torch.ones(1, 1, D, dtype=torch.float16, device=DEV)
    for call in (lambda: cache.update(k.float(), k.float(), 0),
                 lambda: cache.update(k[:1], k[:1], 0),
                 lambda: cache.update(k[:, :, :1], k[:, :, :1], 0),
                 lambda: cache.update_qkv(k.reshape(2, 5, 256), cos, cos, 0, 4),
                 lambda: cache.update_qkv(_rand(g, 2, 1, 8 * D), cos[..., :64], cos[..., :64], 0,
                                          4),
                 lambda: cache.update_qkv(_rand(g, 2, 1, 7 * D), cos, cos, 0, 4)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
        assert cache.length == 5
    attend = cache.update(k[:, :1], k[:, :1], 0)
    with pytest.raises(ValueError):
        attend(_rand(g, 2, 2, 4, D))


def test_captured_decode_step():
    """One captured step replayed for growing contexts, specs refreshed outside."""
    B, H, Hq, g = 2, 2, 8, _gen(4)
    qkv, prompt = _rand(g, B, 1, (Hq + 2 * H) * D), _rand(g, B, 700, H, D)
    cos, sin = dl.rope_cos_sin([5], D, 10000.0, DEV)

    def start():
        c = MultiLayerPagedKVCache8Bit(B, 64, 1024, DEV, 1, H, D)
        c.update(prompt, prompt, 0)
        return c

    def step(c):
        return c.attend(c.update_qkv(qkv, cos, sin, 0, Hq, eps=1e-6), 0)

    eager, cap = start(), start()
    want = [step(eager).clone() for _ in range(4)]
    cap.refresh_specs(701)
    cap.freeze_specs(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cap)
    for i in range(4):
        cap.refresh_specs(701 + i)
        graph.replay()
        torch.cuda.synchronize()
        # the split is planned for the longest context: another order of addition
        assert (out.float() - want[i].float()).abs().max() <= 2.0 ** -9 * want[i].abs().max()
        _check_attend_at(cap, 701 + i, out, eager, qkv, cos, sin, Hq, H)
    assert torch.equal(cap.scales[cap._table.indices[:2].long()],
                       eager.scales[eager._table.indices[:2].long()])


def _check_attend_at(cap, length, out, eager, qkv, cos, sin, Hq, H):
    heads = qkv.view(qkv.shape[0], 1, -1, D)
    q, _ = kernel.qk_norm_rope(heads[:, :, :Hq], heads[:, :, Hq: Hq + H], cos, sin, eps=1e-6)
    want, size = i8_ref.attention(to_np(q)[:, 0], *_state(cap, 0))
    _close(to_np(out)[:, 0], want, size, length)


# ------------------------------------------------------- the decode layer

def _layer(qk_norm, seed=0):
    layer = dl.W4A4LlamaDecodeLayer.random(1024, 8, 2, D, 896, seed=seed, qk_norm=qk_norm)
    if qk_norm:
        g = torch.Generator().manual_seed(seed + 1)
        layer.q_norm.copy_(1 + 0.2 * torch.randn(D, generator=g))
        layer.k_norm.copy_(1 + 0.2 * torch.randn(D, generator=g))
    return layer.to(DEV)


def _cache(cls, B, T):
    if cls is MultiLayerPagedKVCache4Bit:
        return cls(B, 32, T, DEV, 1, 2, D, group_size=4)
    return cls(B, 32, T, DEV, 1, 2, D)


@pytest.mark.parametrize("cls", [MultiLayerPagedKVCache4Bit, MultiLayerPagedKVCache8Bit])
@pytest.mark.parametrize("masked", [False, True])
def test_layer_with_qk_norms(cls, masked):
    """Prefill and decode steps, fused and op by op: the same bits."""
    layer, B, T = _layer(True), 3, 21
    mask = None
    if masked:
        mask = torch.ones(B, T, dtype=torch.int64, device=DEV)
        mask[1, :5] = 0
    h = _rand(_gen(5), B, T, 1024)
    outs = []
    for fused in (True, False):
        cache, m = _cache(cls, B, 64), mask
        cos, sin = dl.rope_cos_sin(range(T), D, 10000.0, DEV)
        got = [layer.prefill(h.clone(), cache, cos, sin, m, trace=None if fused else {})]
        for t in range(3):
            if m is not None:
                m = torch.cat([m, torch.ones(B, 1, dtype=torch.int64, device=DEV)], 1)
            cos, sin = dl.rope_cos_sin([T + t], D, 10000.0, DEV)
            got.append(layer(h[:, t: t + 1].clone(), cache, cos, sin, fused=fused,
                             attention_mask=m))
        outs.append(got)
    for a, b in zip(*outs):
        live = slice(None) if mask is None or a.shape[1] == 1 else mask.bool()
        assert torch.equal(a[live], b[live])
    plain = _layer(False)
    cache = _cache(cls, B, 64)
    cos, sin = dl.rope_cos_sin(range(T), D, 10000.0, DEV)
    assert not torch.equal(plain.prefill(h.clone(), cache, cos, sin, mask), outs[0][0])


def test_layer_without_norms_over_the_8bit_cache(monkeypatch):
    """The decode step's q/k/v pass is RoPE in fp32: with that in the op-by-op form's
    place, the same bits."""
    layer, B, T, g = _layer(False, 3), 2, 40, _gen(6)
    h = _rand(g, B, T, 1024)
    outs = []
    for fused in (True, False):
        cache = _cache(MultiLayerPagedKVCache8Bit, B, 64)
        cos, sin = dl.rope_cos_sin(range(T), D, 10000.0, DEV)
        got = [layer.prefill(h.clone(), cache, cos, sin)]
        if not fused:
            monkeypatch.setattr(kernel, "rope_qk", lambda q, k, c, s: kernel.qk_norm_rope(
                q, k, c, s, eps=None))
        for t in range(2):
            cos, sin = dl.rope_cos_sin([T + t], D, 10000.0, DEV)
            got.append(layer(h[:, t: t + 1].clone(), cache, cos, sin, fused=fused))
        outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# ------------------------------------------- grouped linears and the block

@pytest.mark.parametrize("sym", [True, False])
@pytest.mark.parametrize("bias", [True, False])
def test_group_linear(sym, bias):
    g = torch.Generator().manual_seed(7)
    lin = torch.nn.Linear(512, 96, bias=bias, dtype=torch.float16)
    lin.weight.data = (0.05 * torch.randn(96, 512, generator=g)).half()
    mod = nn.GroupLinear4bit.from_float(lin, 64, sym).to(DEV)
    x = torch.randn(100, 512, generator=g).half().to(DEV)
    mod.MAX_ROWS = 64
    w = mod.dequantized().double()
    want = x.double() @ w.t() + (mod.bias.double() if bias else 0)
    size = x.double().abs() @ w.abs().t() + 1
    # the products' fp32 sums, the weight's rounding to fp16 in the long form, and the
    # result's (2^-11 each)
    tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 600 * 2.0 ** -24) * size
    for rows in (1, 64, 65, 100):
        got = mod(x[:rows])
        assert ((got.double() - want[:rows]).abs() <= tol[:rows]).all()
    assert mod(x[:6].view(2, 3, 512)).shape == (2, 3, 96)
    again = nn.GroupLinear4bit(512, 96, 64, sym, bias)
    again.load_state_dict(mod.cpu().state_dict())
    assert torch.equal(again.to(DEV)(x[:3]), mod.to(DEV)(x[:3]))
    y = x[:3].clone().requires_grad_()
    mod(y).sum().backward()
    assert torch.allclose(y.grad.double(), w.sum(0).expand(3, 512), atol=2e-2)


def test_attention_block_as_a_program_runs_it():
    """Grouped linears, q/k norms, the cache and its attention: a prompt in two
    pieces, then tokens.  Each stage is held against 64 bits on the previous one's
    output."""
    B, hidden, Hq, H, g = 2, 256, 4, 2, _gen(8)
    cols = (Hq + 2 * H) * D
    qkv_lin = nn.GroupLinear4bit.from_float(torch.nn.Linear(hidden, cols, bias=False).half(), 32)
    o_lin = nn.GroupLinear4bit.from_float(torch.nn.Linear(Hq * D, hidden, bias=False).half(), 128,
                                          sym=False)
    qkv_lin, o_lin = qkv_lin.to(DEV), o_lin.to(DEV)
    w = [(1 + 0.2 * torch.randn(D, device=DEV, generator=g)).half() for _ in range(2)]
    cache = MultiLayerPagedKVCache8Bit(B, 16, 32, DEV, 1, H, D)
    pos = 0
    for T in (30, 9, 1, 1):
        x = _rand(g, B, T, hidden)
        cos, sin = dl.rope_cos_sin(range(pos, pos + T), D, 10000.0, DEV)
        qkv = qkv_lin(x)
        q = cache.update_qkv(qkv, cos, sin, 0, Hq, *w, 1e-6)
        o = cache.attend(q, 0)
        out = o_lin(o.view(B, T, -1))
        for lin, a, b in ((qkv_lin, x, qkv), (o_lin, o.view(B, T, -1), out)):
            wd = lin.dequantized().double()
            want = a.double() @ wd.t()
            size = a.double().abs() @ wd.abs().t()
            tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 600 * 2.0 ** -24) * size + 2.0 ** -24
            assert ((b.double() - want).abs() <= tol).all()
        heads = to_np(qkv).reshape(B, T, -1, D)
        c, s = to_np(cos)[:, :, None], to_np(sin)[:, :, None]
        want, size = i8_ref.norm_rope(heads[:, :, :Hq], to_np(w[0]), c, s, 1e-6)
        tol = 2.0 ** -11 * np.abs(want) + size * 20 * 2.0 ** -23 + 2.0 ** -25
        assert (np.abs(to_np(q).astype(np.float64) - want) <= tol).all()
        _check_attend(cache, 0, q, o)
        pos += T
    assert cache.length == 41
