"""Scales and zero points of grouped 4-bit weights: what GPTQ by groups gives reaches
the linear, and what does not fit the groups is refused."""
import pytest
import torch

from signrot_amd import nn, offline
from signrot_amd.functional.quantization import rtn_group_pack, unpack_i4, unpack_ui4


@pytest.mark.parametrize("sym", [True, False])
def test_given_scales_have_one_for_each_group(sym):
    """Scales and zeros of another shape, which would broadcast, zeros that a byte does
    not hold and zeros without their scales are refused."""
    lin = torch.nn.Linear(128, 6, dtype=torch.float16)
    s, z = torch.full((6, 4), 0.01).half(), None if sym else torch.full((6, 4), 8.0)
    ok = nn.GroupLinear4bit.from_float(lin, 32, sym, s, z)
    assert ok.weight_scales.shape == (6, 4)
    bad = [(s[:, :1], z), (s[:1], z), (s[:, :2], z), (s.flatten(), z), (s[:5], z),
           (s.float() * 1e-7, z), (s.float() * 1e8, z), (s * float("nan"), z)]
    if sym:
        with_zeros = nn.GroupLinear4bit.from_float(lin, 32, sym, s, torch.zeros(6, 4))
        assert torch.equal(with_zeros.weight, ok.weight) and with_zeros.weight_zeros is None
        bad += [(s, torch.ones(6, 4)), (None, torch.zeros(6, 4))]
    else:
        bad += [(s, z[:, :1]), (s, z - 9), (s, z + 248), (s, z + 0.5), (None, z),
                (s, torch.full((6, 4), float("nan")))]
    for scales, zeros in bad:
        with pytest.raises(ValueError):
            nn.GroupLinear4bit.from_float(lin, 32, sym, scales, zeros)
    with pytest.raises(ValueError):
        rtn_group_pack(lin.weight.data, 48)


def _calibrated(sym, groupsize, seed=0, **kw):
    """GPTQ by groups of a 24 x 256 linear whose halves differ 20-fold."""
    g = torch.Generator().manual_seed(seed)
    lin = torch.nn.Linear(256, 24, bias=True, dtype=torch.float16)
    w = torch.randn(24, 256, generator=g) * 0.05
    w[:, :128] *= 20
    lin.weight.data = w.half()
    x = torch.randn(4, 300, 256, generator=g) @ torch.randn(256, 256, generator=g)
    work = offline.GPTQ(lin, offline.WeightQuantizer(4, sym=sym, mse=kw.pop("mse", False)))
    work.add_batch(x)
    return lin, work.fasterquant(groupsize=groupsize, **kw)


@pytest.mark.parametrize("sym", [True, False])
@pytest.mark.parametrize("groupsize", [32, 64, 256])
@pytest.mark.parametrize("kw", [dict(), dict(mse=True), dict(static_groups=True),
                                dict(static_groups=True, actorder=True), dict(blocksize=48)])
def test_the_module_holds_what_gptq_by_groups_gives(sym, groupsize, kw):
    """The codes are GPTQ's own: its weight c s, rounded to fp16, read on the grid of
    fp16(s), is off by at most 15 (2^-11 + 2^-11) steps, far from a half; so what the
    module stands for is off by the scale's rounding and the fp16 weights' (2^-11
    each)."""
    lin, q = _calibrated(sym, groupsize, **dict(kw))
    assert q.group_scale.shape == q.group_zero.shape == (24, 256 // groupsize)
    mod = nn.GroupLinear4bit.from_float(lin, groupsize, sym, q.group_scale, q.group_zero)
    w, back = lin.weight.data.double(), mod.dequantized().double()
    assert ((back - w).abs() <= 3 * 2.0 ** -11 * w.abs() + 2.0 ** -24).all()
    c = unpack_i4(mod.weight) if sym else unpack_ui4(mod.weight)
    step = q.group_scale.double().repeat_interleave(groupsize, 1)
    want = torch.round(w / step) + (0 if sym else q.group_zero.repeat_interleave(groupsize, 1))
    assert torch.equal(c.double(), want.double())
    assert torch.equal(mod.bias, lin.bias.data)


def test_gptq_without_groups_of_neighbours_has_no_group_scales():
    for kw in (dict(groupsize=-1), dict(groupsize=64, actorder=True)):
        _, q = _calibrated(True, **kw)
        assert q.group_scale is None and q.group_zero is None and q.scale.shape == (24, 1)
    # the last group's scale alone is refused
    lin, q = _calibrated(True, 64)
    with pytest.raises(ValueError):
        nn.GroupLinear4bit.from_float(lin, 64, scales=q.scale)
