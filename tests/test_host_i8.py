"""CPU checks of what surrounds the int8 cache and the grouped linears: constructor
refusals, the group quantizer, the linear's dequantized form."""
import pytest
import torch
from transformers.cache_utils import Cache

from signrot_amd import _native, nn
from signrot_amd.functional.quantization import rtn_group_pack, unpack_i4, unpack_ui4
from signrot_amd.transformers import MultiLayerPagedKVCache8Bit


def test_cache_is_a_transformers_cache():
    c = MultiLayerPagedKVCache8Bit(2, 32, 100, "cpu", 3, 4, 128)
    assert isinstance(c, Cache) and len(c) == 3 and c.batch_size == 2
    assert c.pages.shape == (8, 3, 2, 4, 32, 128) and c.pages.dtype == torch.int8
    assert c.scales.shape == (8, 3, 2, 4, 2) and c.get_max_length() is None
    for bad in (dict(head_dim=64), dict(page_size=24), dict(page_size=0)):
        args = dict(batch_size=1, page_size=16, max_seq_len=10, device="cpu", n_layers=1,
                    num_heads=1, head_dim=128)
        with pytest.raises(ValueError):
            MultiLayerPagedKVCache8Bit(**{**args, **bad})


@pytest.mark.parametrize("sym", [True, False])
def test_group_quantizer(sym):
    g = torch.Generator().manual_seed(0)
    w = (torch.randn(6, 192, generator=g) * torch.rand(6, 1, generator=g)).half()
    w[2, 64:128] = 0
    q, s, z = rtn_group_pack(w, 64, sym)
    c = (unpack_i4(q) if sym else unpack_ui4(q)).float().view(6, 3, 64)
    c = c if sym else c - z.float()[..., None]
    back = (c * s.float()[..., None]).view(6, 192)
    step = s.float().repeat_interleave(64, 1)
    # half a step, and the fp16 rounding of the scale over at most 15 steps
    assert ((back - w.float()).abs() <= step * (0.5 + 15 * 2.0 ** -11) + 1e-7).all()
    assert (back[2, 64:128] == 0).all()
    again = rtn_group_pack(back.half(), 64, sym, s, z)
    assert torch.equal(again[0], q) and torch.equal(again[1], s)


def test_given_scales_come_with_their_zeros():
    w = torch.randn(4, 64).half()
    with pytest.raises(ValueError):
        rtn_group_pack(w, 32, False, torch.ones(4, 2).half())


def test_group_linear_on_the_host():
    lin = torch.nn.Linear(64, 8, dtype=torch.float16)
    mod = nn.GroupLinear4bit.from_float(lin, 32)
    x = torch.randn(3, 64).half()
    want = torch.nn.functional.linear(x, mod.dequantized(), lin.bias)
    assert torch.equal(mod(x), want)
    for args in ((64, 8, 24), (64, 8, 128), (96, 8, 64), (64, 8, 0)):
        with pytest.raises(ValueError):
            nn.GroupLinear4bit(*args)


@pytest.mark.parametrize("sm", [float("nan"), float("inf"), -3e38, 1e20, 1e-7, -1e-40])
def test_softmax_scales_that_leave_the_range_are_refused(sm):
    """The entry point's own check, before any launch: the pointers are only
    aligned numbers here."""
    rc = _native.lib().srq_batch_attention_i8(
        64, 64, 1, 1, 64, 64, 64, 64, 64, 1, 1, 1, 1, 0, 1, 16, 128, None, 1, 16, sm, None, 0, None)
    assert rc != 0 and b"sm_scale" in _native.lib().srq_last_error()
