"""GroupLinear4bit on the GPU beside tests/test_gpu_kv_cache_i8.py: derivatives in
forward mode, and the form it takes at and behind MAX_ROWS."""
import pytest
import torch

from signrot_amd import _CUDA, nn
from tests.gpu_util import DEV

pytestmark = pytest.mark.gpu


def _module(seed=0):
    g = torch.Generator().manual_seed(seed)
    lin = torch.nn.Linear(256, 48, dtype=torch.float16)
    lin.weight.data = (0.05 * torch.randn(48, 256, generator=g)).half()
    return nn.GroupLinear4bit.from_float(lin, 64).to(DEV), g


def test_forward_mode_tangents_are_kept():
    """A dual input's tangent goes through the product: W t, each a rounding to fp16 of
    the weight and of the result behind fp32 sums."""
    mod, g = _module()
    x, t = (torch.randn(3, 256, generator=g).half().to(DEV) for _ in range(2))
    w = mod.dequantized().double()
    want, size = t.double() @ w.t(), t.double().abs() @ w.abs().t()
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        out = fw.unpack_dual(mod(fw.make_dual(x, t)))
        assert out.tangent is not None
        assert ((out.tangent.double() - want).abs()
                <= 2.0 ** -11 * want.abs() + 256 * 2.0 ** -24 * size + 2.0 ** -24).all()
        # an input without one, at the same level, has none to lose
        assert torch.equal(mod(x), mod(x.clone()))
    assert fw.unpack_dual(mod(x)).tangent is None


def test_a_linear_without_columns_is_refused_by_name():
    f16 = dict(dtype=torch.float16, device=DEV)
    w = torch.zeros(16, 0, dtype=torch.uint8, device=DEV)
    for groups in (0, 2):
        with pytest.raises(RuntimeError, match="w4a16_linear"):
            _CUDA.w4a16_linear(torch.zeros(2, 0, **f16), w, torch.ones(16, groups, **f16))
