"""Refusals of the 8-bit-activation and adapter entry points, before a device is
touched, and the reference forms against each other."""
import ctypes

import numpy as np
import pytest

from tests import act8_ref as ref

P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    from signrot_amd import _native
    return _native.lib()


def _refused(lib, rc, msg):
    assert rc == -1 and msg in lib.srq_last_error().decode(), lib.srq_last_error()


@pytest.mark.parametrize("change,msg", [
    (dict(rows=-1), "negative"), (dict(rows=1 << 31), "rows"), (dict(n=0), "empty rows"),
    (dict(mean=0), "mean_dim"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(clip=0.0), "clip_ratio"), (dict(clip=1.01), "clip_ratio"),
    (dict(clip=float("nan")), "clip_ratio"), (dict(x=None), "null"), (dict(q=None), "null"),
    (dict(scale=None), "null"), (dict(sum=P), "without a residual"), (dict(xs=63), "row stride"),
    (dict(res=P, rs=8), "row stride")])
def test_norm_quant(lib, change, msg):
    a = dict(x=P, xs=64, res=None, rs=0, w=None, rows=4, n=64, eps=1e-5, mean=64, clip=1.0,
             sum=None, norm=None, q=P, scale=P, st=None)
    assert set(change) <= set(a)
    a.update(change)
    _refused(lib, lib.srq_rmsnorm_quant_i8(*a.values()), msg)
    if set(change) <= {"x", "xs", "rows", "n", "clip", "q", "scale"}:
        _refused(lib, lib.srq_sym_quant_dynamic_i8(*(a[k] for k in "x xs rows n clip q scale st"
                                                     .split())), msg)


@pytest.mark.parametrize("change,msg", [
    (dict(M=-1), "negative"), (dict(K=48), "multiple of 32"), (dict(K=0), "multiple of 32"),
    (dict(K=131072), "131072"), (dict(M=1 << 40), "range"), (dict(M=1 << 30, N=1 << 30), "range"),
    (dict(a=None), "null"), (dict(out=None), "null"), (dict(sa=None), "null"),
    (dict(a=ctypes.c_void_p(264)), "aligned"), (dict(w=ctypes.c_void_p(264)), "aligned"),
    (dict(M=48, K=8192), "workspace"),
    (dict(M=48, K=8192, ws=P, wb=4 * 48 * 64), "workspace"),
    (dict(M=48, K=8192, ws=ctypes.c_void_p(260), wb=1 << 40), "workspace")])
def test_w4a8(lib, change, msg):
    a = dict(a=P, sa=P, w=P, sw=P, bias=None, res=None, M=4, N=64, K=64, out=P, ws=None, wb=0,
             st=None)
    assert set(change) <= set(a)
    a.update(change)
    _refused(lib, lib.srq_w4a8_linear(*a.values()), msg)


@pytest.mark.parametrize("change,msg", [
    (dict(M=-1), "negative"), (dict(L=-1), "negative"), (dict(r=4), "rank"), (dict(r=264), "rank"),
    (dict(r=0), "rank"), (dict(S=0), "slices"), (dict(S=9), "slices"), (dict(cols=None), "slices"),
    (dict(K=60), "K=60"), (dict(K=0), "K=0"), (dict(K=(1 << 20) + 8), "K="),
    (dict(widths=(0,)), "slice of"), (dict(widths=(-8,)), "slice of"), (dict(M=1 << 40), "range"),
    (dict(x=None), "null"), (dict(ids=None), "null"), (dict(la=None), "null"), (dict(out=P), "not x"),
    (dict(x=ctypes.c_void_p(264)), "aligned"), (dict(lb=ctypes.c_void_p(258)), "aligned"),
    (dict(xs=65), "aligned"), (dict(xs=56), "row stride"), (dict(ys=39), "row stride"),
    (dict(os=39), "row stride"), (dict(xs=1 << 25), "row stride"), (dict(ws=None), "workspace"),
    (dict(wb=4 * 3 * 8 - 1), "workspace"), (dict(ws=ctypes.c_void_p(8)), "workspace")])
def test_lora(lib, change, msg):
    a = dict(y=P, ys=40, x=P, xs=64, la=P, lb=P, ids=P, sc=None, M=3, K=64, L=2, r=8, S=1, cols=0,
             out=ctypes.c_void_p(512), os=40, ws=P, wb=4 * 3 * 8, st=None)
    widths = change.get("widths", (40,))
    a["cols"] = (ctypes.c_int64 * 9)(*widths)
    change = {k: v for k, v in change.items() if k != "widths"}
    assert set(change) <= set(a)
    a.update(change)
    _refused(lib, lib.srq_lora_add(*a.values()), msg)


def test_empty_inputs_are_noops(lib):
    assert lib.srq_rmsnorm_quant_i8(None, 0, None, 0, None, 0, 64, 1e-5, 64, 1.0, None, None, None,
                                    None, None) == 0
    assert lib.srq_sym_quant_dynamic_i8(None, 0, 0, 64, 1.0, None, None, None) == 0
    assert lib.srq_w4a8_linear(*[None] * 6, 0, 64, 64, None, None, 0, None) == 0
    assert lib.srq_w4a8_linear(*[None] * 6, 8, 0, 64, None, None, 0, None) == 0
    cols = (ctypes.c_int64 * 1)(8)
    assert lib.srq_lora_add(None, 0, None, 0, None, None, None, None, 0, 64, 2, 8, 1, cols, None, 0,
                            None, 0, None) == 0


def test_reference_quantizer_rounds_as_rational_numbers():
    """Codes and scales by fractions: the scale is the fp32 number next to top / 127,
    a code the whole number next to x / scale, ties to the even one."""
    from fractions import Fraction
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 40)).astype(np.float16).astype(np.float64)
    x[2, :3] = 127, 0.5, 2.5
    q, s = ref.quant(x)
    for row, codes, scale in zip(x, q, s):
        top = max(abs(Fraction(v)) for v in row)
        near = [np.nextafter(scale[0], np.float32(d)) for d in (-np.inf, np.inf)]
        assert all(abs(Fraction(float(scale[0])) - top / 127) <= abs(Fraction(float(v)) - top / 127)
                   for v in near)
        for v, c in zip(row, codes):
            assert round(Fraction(v) / Fraction(float(scale[0]))) == c


def test_lora_adapters_hold_what_is_loaded():
    import torch
    from signrot_amd.nn import LoraAdapters
    ad = LoraAdapters(16, (24, 8), 8, 3)
    a, b = torch.randn(4, 16), torch.randn(8, 4)
    ad.load(2, (None, a), (None, b), 0.5)
    assert torch.equal(ad.lora_a[2, 8:12], a.half()) and torch.equal(ad.lora_b[2, 24:, :4], b.half())
    assert not ad.lora_a[2, :8].any() and not ad.lora_a[2, 12:].any() and not ad.lora_a[:2].any()
    assert not ad.lora_b[2, :24].any() and not ad.lora_b[2, 24:, 4:].any()
    assert ad.scaling.tolist() == [1, 1, 0.5]
    # a smaller one in its place leaves nothing of it
    ad.load(2, (torch.ones(1, 16), None), (torch.ones(24, 1), None))
    assert ad.lora_a[2].sum() == 16 and ad.lora_b[2].sum() == 24 and ad.scaling[2] == 1
    ad.clear(2)
    assert not ad.lora_a.any() and not ad.lora_b.any()
    one = LoraAdapters(16, 24, 8, 1)
    one.load(0, torch.ones(8, 16), torch.ones(24, 8))
    with pytest.raises(ValueError, match="outside"):
        one.load(1, torch.ones(8, 16), torch.ones(24, 8))
    before = one.lora_a.clone()
    for x, y in [(torch.ones(9, 16), torch.ones(24, 9)), (torch.ones(8, 15), torch.ones(24, 8)),
                 (torch.ones(8, 16), torch.ones(23, 8)), (torch.ones(8, 16), torch.ones(24, 7)),
                 (torch.ones(16), torch.ones(24, 1)), (torch.ones(8, 16), None)]:
        with pytest.raises(ValueError):
            one.load(0, x, y)
    with pytest.raises(ValueError, match="slices"):
        ad.load(0, (a,), (b,))
    assert torch.equal(one.lora_a, before)
    for bad in [dict(rank=4), dict(rank=0), dict(rank=264), dict(in_features=12),
                dict(out_features=()), dict(out_features=(8,) * 9), dict(out_features=(8, 0))]:
        with pytest.raises(ValueError):
            LoraAdapters(**{**dict(in_features=16, out_features=24, rank=8, adapters=1), **bad})


def test_decode_layer_refuses_other_widths():
    from signrot_amd.transformers.decode_layer import W4A4LlamaDecodeLayer
    with pytest.raises(ValueError, match="act_bits"):
        W4A4LlamaDecodeLayer(256, 2, 1, 128, 384, act_bits=6)
    layer = W4A4LlamaDecodeLayer(256, 2, 1, 128, 384)
    with pytest.raises(ValueError, match="adapters of"):
        layer.add_adapters(8, 1, ("q",))
    with pytest.raises(ValueError, match="rank"):
        layer.add_adapters(12, 1)
    assert set(layer.add_adapters(8, 2, ("o", "down"))) == {"o", "down"}
    assert layer.adapters["down"].in_features == 384
