"""8-bit activations and low-rank adapters through the modules and the decode layer,
stage by stage: each stage is compared with its definition in 64 bits applied to the
output of the stage before."""
import copy

import numpy as np
import pytest
import torch

from oracle import glue
from oracle import hadamard as oh
from signrot_amd import nn as snn
from signrot_amd.functional import kernel
from signrot_amd.functional.quantization import unpack_i4
from signrot_amd.transformers import MultiLayerPagedKVCache4Bit, MultiLayerPagedKVCache8Bit
from signrot_amd.transformers.decode_layer import W4A4LlamaDecodeLayer, rope_cos_sin
from tests import act8_ref as ref
from tests import layer_check as lc
from tests.gpu_util import DEV, to_dev, to_np

pytestmark = pytest.mark.gpu
D = 128
HIDDEN, HQ, HKV, FFN = 1024, 8, 2, 896
RANK, COUNT = 16, 4


def _layer(seed, **kw):
    return W4A4LlamaDecodeLayer.random(HIDDEN, HQ, HKV, D, FFN, layer_idx=0, seed=seed, **kw)


def _fill(layer, seed, scale=0.05):
    """Adapters of several ranks, some slices without one."""
    rng = np.random.default_rng(seed)
    layer.add_adapters(RANK, COUNT)
    for name, ad in layer.adapters.items():
        for i in range(COUNT):
            r = (4, 8, 16, 13)[i]
            a, b = [], []
            for j, n in enumerate(ad.widths):
                skip = name == "qkv" and i == 1 and j == 1
                a.append(None if skip else torch.from_numpy(
                    rng.standard_normal((r, ad.in_features)).astype(np.float16)
                    / np.float16(ad.in_features ** 0.5)))
                b.append(None if skip else torch.from_numpy(
                    (scale * rng.standard_normal((n, r))).astype(np.float16)))
            ad.load(i, a, b, 0.5 + i)
    return layer


def _cache(kind, B, T, seed, heads=HKV):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if kind == 4:
        cache = MultiLayerPagedKVCache4Bit(B, 32, T + 8, DEV, 1, heads, D, group_size=HQ // heads)
    else:
        cache = MultiLayerPagedKVCache8Bit(B, 32, T + 8, DEV, 1, heads, D)
    kv = torch.randn((2, B, T, heads, D), device=DEV, generator=g).half()
    cache.update(kv[0], kv[1], 0, {})
    return cache


def _close(got, want, tol, what):
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), f"{what}: {(err / tol).max()}"


def _weights(layer, name):
    return to_np(unpack_i4(getattr(layer, f"w_{name}"))), to_np(getattr(layer, f"s_{name}"))


def _projection(layer, name, q, s, x, ids, residual=None):
    """(exact, bound) of a projection with its adapters: fp16 in between."""
    want, tol = ref.linear(q, s, *_weights(layer, name), None, residual)
    if ids is None:
        return want, tol
    ad = layer.adapters[name]
    want, more = ref.lora(want, x, to_np(ad.lora_a), to_np(ad.lora_b), ids, to_np(ad.scaling),
                          ad.widths)
    return want, tol * (1 + 2 * ref.U16) + more


def _check_rows(layer, tr, h, out, ids):
    R = h.shape[0]
    q, s, _, y = ref.norm_quant(h, layer.eps)
    assert np.array_equal(tr["q1"], q) and np.array_equal(tr["s1"], s)
    _close(tr["norm1"], y, (ref.U16 + 4 * ref.U32) * np.abs(y) + ref.TINY, "norm1")
    _close(tr["qkv"], *_projection(layer, "qkv", q, s, tr["norm1"], ids), "qkv")
    attn = tr["attn"].reshape(R, HQ, D)
    rot = oh.rotate(np.ascontiguousarray(attn.transpose(0, 2, 1)).reshape(-1, HQ)
                    ).reshape(R, D, HQ).transpose(0, 2, 1).reshape(R, HIDDEN)
    lc.ulps(tr["attn_rot"], rot, "head-axis Hadamard")
    q, s = ref.quant(tr["attn_rot"].astype(np.float64))
    assert np.array_equal(tr["oq"], q) and np.array_equal(tr["os"], s)
    _close(tr["o"], *_projection(layer, "o", q, s, attn.reshape(R, HIDDEN), ids), "o")
    q, s, x, y = ref.norm_quant(tr["o"], layer.eps, residual=h)
    assert np.array_equal(tr["resid1"], x)
    assert np.array_equal(tr["q2"], q) and np.array_equal(tr["s2"], s)
    _close(tr["norm2"], y, (ref.U16 + 4 * ref.U32) * np.abs(y) + ref.TINY, "norm2")
    _close(tr["gu"], *_projection(layer, "gu", q, s, tr["norm2"], ids), "gu")
    sw = glue.swiglu(tr["gu"][:, :FFN], tr["gu"][:, FFN:])
    assert (tr["act"].view(np.uint16) != sw.view(np.uint16)).mean() < 1e-3
    np.testing.assert_allclose(tr["act_rot"].astype(np.float32),
                               oh.online_hadamard(tr["act"], to_np(layer.down_sign))
                               .astype(np.float32), rtol=1e-2, atol=1e-2)
    q, s = ref.quant(tr["act_rot"].astype(np.float64))
    assert np.array_equal(tr["down_q"], q) and np.array_equal(tr["down_s"], s)
    _close(out, *_projection(layer, "down", q, s, tr["act"], ids, tr["resid1"]), "down")


@pytest.mark.parametrize("kind", [4, 8])
@pytest.mark.parametrize("B,adapters,qk_norm", [(1, False, False), (3, True, False),
                                                (5, True, True), (40, True, False)])
def test_decode_step_stagewise(kind, B, adapters, qk_norm):
    layer = _layer(B, act_bits=8, qk_norm=qk_norm)
    ids = None
    if adapters:
        _fill(layer, B)
        ids = (np.arange(B) % (COUNT + 1) - 1).astype(np.int32)
    T = 50
    cache = _cache(kind, B, T, B)
    again = cache.clone()
    h = (np.random.default_rng(B).standard_normal((B, HIDDEN)) * 0.5).astype(np.float16)
    cos, sin = rope_cos_sin([T], D, 500000.0, DEV)
    tr = {}
    out = layer(to_dev(h).view(B, 1, HIDDEN), cache, cos, sin, trace=tr,
                adapter_ids=None if ids is None else to_dev(ids))
    # the attention saw the adapted q, k and v: the cache's own update() of them
    heads = tr["qkv"].view(B, 1, -1, D)
    q, k, v = (t.clone() for t in heads.split((HQ, HKV, HKV), 2))
    q, k = layer._rope(q, k, cos, sin)
    attn = again.update(k, v, 0, {})(q)
    assert (attn.float() - tr["attn"].view_as(attn).float()).abs().max() < 4e-3
    _check_rows(layer, {k: to_np(v) for k, v in tr.items()}, h, to_np(out).reshape(B, HIDDEN), ids)


@pytest.mark.parametrize("kind", [4, 8])
@pytest.mark.parametrize("B,T", [(2, 9), (3, 70)])
def test_prefill_stagewise_then_decode(kind, B, T):
    layer = _fill(_layer(T, act_bits=8), T)
    ids = np.array([2, -1, 3][:B], np.int32)
    cache = MultiLayerPagedKVCache4Bit(B, 32, T + 8, DEV, 1, HKV, D, group_size=HQ // HKV) \
        if kind == 4 else MultiLayerPagedKVCache8Bit(B, 32, T + 8, DEV, 1, HKV, D)
    h = (np.random.default_rng(T).standard_normal((B, T, HIDDEN)) * 0.5).astype(np.float16)
    cos, sin = rope_cos_sin(list(range(T + 1)), D, 500000.0, DEV)
    tr = {}
    out = layer.prefill(to_dev(h), cache, cos[:, :T], sin[:, :T], trace=tr,
                        adapter_ids=to_dev(ids))
    heads = tr["qkv"].view(B, T, -1, D)
    q, k, v = (t.clone() for t in heads.split((HQ, HKV, HKV), 2))
    q, k = kernel.rope_qk(q, k, cos[:, :T], sin[:, :T])
    from signrot_amd import _CUDA
    attn = _CUDA.prefill_attention(q, k, v, None, causal=True)
    assert (attn.float() - tr["attn"].view_as(attn).float()).abs().max() < 4e-3
    rows = np.repeat(ids, T)
    _check_rows(layer, {k: to_np(v) for k, v in tr.items()}, h.reshape(B * T, HIDDEN),
                to_np(out).reshape(B * T, HIDDEN), rows)
    new = (np.random.default_rng(1).standard_normal((B, HIDDEN)) * 0.5).astype(np.float16)
    tr = {}
    out = layer(to_dev(new).view(B, 1, HIDDEN), cache, cos[:, T:], sin[:, T:], trace=tr,
                adapter_ids=to_dev(ids))
    _check_rows(layer, {k: to_np(v) for k, v in tr.items()}, new, to_np(out).reshape(B, HIDDEN),
                ids)
    assert cache.get_seq_length() == T + 1


@pytest.mark.parametrize("kind", [4, 8])
def test_requests_without_an_adapter_are_the_layer_itself(kind):
    """4-bit activations: rows without an adapter are bit for bit the layer's fused
    step and prefill."""
    layer = _fill(_layer(11), 11)
    for T in (1, 40):
        ids = torch.tensor([-1, 2, -1], dtype=torch.int32, device=DEV)
        g = torch.Generator(device=DEV).manual_seed(T)
        cos, sin = rope_cos_sin(list(range(60, 60 + T)), D, 500000.0, DEV)
        h = torch.randn(3, T, HIDDEN, device=DEV, generator=g).half()
        if T == 1:
            one, two = _cache(kind, 3, 60, 5), _cache(kind, 3, 60, 5)
            want = layer(h.clone(), one, cos, sin)
            got = layer(h.clone(), two, cos, sin, adapter_ids=ids)
        else:
            one, two = (MultiLayerPagedKVCache4Bit(3, 32, 64, DEV, 1, HKV, D, group_size=HQ // HKV)
                        if kind == 4 else MultiLayerPagedKVCache8Bit(3, 32, 64, DEV, 1, HKV, D)
                        for _ in range(2))
            want = layer.prefill(h.clone(), one, cos, sin)
            got = layer.prefill(h.clone(), two, cos, sin, adapter_ids=ids)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
        assert not torch.equal(got[1], want[1])


def test_captured_step_follows_its_inputs():
    """A decode step with adapters in a graph, replayed on other rows, adapters and
    lengths, with eager work between."""
    B, T = 4, 33
    layer = _fill(_layer(21, act_bits=8), 21)
    cache = _cache(8, B, T, 21)
    h = torch.zeros(B, 1, HIDDEN, dtype=torch.float16, device=DEV)
    ids = torch.full((B,), -1, dtype=torch.int32, device=DEV)
    cos, sin = rope_cos_sin([T], D, 500000.0, DEV)
    eager = cache.clone()
    start = cache.clone()
    cache.freeze_specs(True)
    cache.refresh_specs(T + 1)
    layer(h.clone(), start, cos, sin, adapter_ids=ids)   # first calls outside the capture
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer(h, cache, cos, sin, adapter_ids=ids)
    for step in range(3):
        gen = torch.Generator(device=DEV).manual_seed(step)
        h.copy_(torch.randn(B, 1, HIDDEN, device=DEV, generator=gen).half() * 0.5)
        ids.copy_(torch.randint(-1, COUNT, (B,), device=DEV, generator=gen))
        c, s = rope_cos_sin([T + step], D, 500000.0, DEV)
        cos.copy_(c)
        sin.copy_(s)
        cache.refresh_specs(T + 1 + step)
        g.replay()
        want = layer(h.clone(), eager, cos, sin, adapter_ids=ids)
        torch.cuda.synchronize()
        assert (out.float() - want.float()).abs().max() < 2e-2 * want.float().abs().max()


@pytest.mark.parametrize("rows,bias", [(1, True), (37, False), (300, True)])
def test_modules(rows, bias):
    """Quantizer8bit -> Linear4bit, and LoraAdapters beside it."""
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, 512)).astype(np.float16)
    lin = torch.nn.Linear(512, 200, bias=bias).half()
    scales = lin.weight.detach().abs().amax(1, keepdim=True) / 7
    m = snn.Linear4bit.from_float(lin, scales).to(DEV)
    seq = torch.nn.Sequential(snn.Quantizer8bit(), m)
    got = seq(to_dev(x).view(rows, 1, 512))
    assert got.shape == (rows, 1, 200)
    q, s = ref.quant(x.astype(np.float64))
    c = to_np(unpack_i4(m.weight))
    want, tol = ref.linear(q, s, c, to_np(m.weight_scales.half()).reshape(-1),
                           to_np(m.bias) if bias else None)
    _close(to_np(got).reshape(rows, 200), want, tol, "linear")
    ad = snn.LoraAdapters(512, 200, 8, 3).to(DEV)
    a = torch.randn(5, 512, generator=torch.Generator().manual_seed(1)) * 0.05
    b = torch.randn(200, 5, generator=torch.Generator().manual_seed(2))
    ad.load(1, a, b, 2.0)
    ids = torch.tensor(rng.integers(-1, 3, rows), dtype=torch.int32, device=DEV)
    out = to_np(ad(got.view(rows, 200), to_dev(x), ids))
    want, tol = ref.lora(to_np(got).reshape(rows, 200), x, to_np(ad.lora_a), to_np(ad.lora_b),
                         to_np(ids), to_np(ad.scaling), ad.widths)
    _close(out, want, tol, "adapters")
    ad.clear(1)
    assert np.array_equal(to_np(ad(got.view(rows, 200), to_dev(x), ids)),
                          to_np(got).reshape(rows, 200))


def test_copies_and_refusals():
    layer = _fill(_layer(3, act_bits=8), 3)
    twin = copy.deepcopy(layer)
    assert torch.equal(twin.adapters["gu"].lora_b, layer.adapters["gu"].lora_b)
    cos, sin = rope_cos_sin([9], D, 500000.0, DEV)
    h = torch.randn(2, 1, HIDDEN, device=DEV).half()
    ids = torch.zeros(2, dtype=torch.int32, device=DEV)
    plain = _layer(3)
    with pytest.raises(ValueError, match="add_adapters"):
        plain(h, _cache(4, 2, 9, 1), cos, sin, adapter_ids=ids)
    with pytest.raises(ValueError, match="one a request"):
        layer(h, _cache(4, 2, 9, 1), cos, sin, adapter_ids=ids[:1])
    m = snn.Linear4bit(64, 16).to(DEV)
    q, s = kernel.sym_quant_dynamic_i8(torch.ones(2, 64, dtype=torch.float16, device=DEV))
    with pytest.raises(RuntimeError, match="zero points"):
        m(kernel.PackedQuantizedTensor(q, s, torch.zeros(2, 1, dtype=torch.int8, device=DEV)))
    empty = MultiLayerPagedKVCache8Bit(2, 32, 32, DEV, 1, HKV, D)
    with pytest.raises(RuntimeError, match="no prefill"):
        layer(h, empty, cos, sin)
    assert empty.get_seq_length() == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_another_norm_is_called(bits):
    """A norm module with a weight in the norm's place is called, not replaced."""
    class Weighted(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.calls = 0

        def forward(self, x):
            self.calls += 1
            f = x.float()
            return (2 * f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5)).half()

    layer = _fill(_layer(6, act_bits=bits), 6)
    norm = layer.post_attention_layernorm = Weighted()
    h = torch.randn(2, 1, HIDDEN, device=DEV).half()
    ids = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    cos, sin = rope_cos_sin([9], D, 500000.0, DEV)
    tr = {}
    layer(h, _cache(4, 2, 9, 1), cos, sin, trace=tr, adapter_ids=ids)
    assert norm.calls == 1
    assert torch.equal(tr["norm2"], norm(tr["resid1"]))
