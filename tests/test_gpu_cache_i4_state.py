"""MultiLayerPagedKVCache4Bit: a refused update() leaves its count of tokens."""
import pytest
import torch

from signrot_amd.transformers import MultiLayerPagedKVCache4Bit
from tests.gpu_util import DEV

pytestmark = pytest.mark.gpu


def test_a_refused_update_is_not_counted():
    g = torch.Generator(DEV).manual_seed(0)
    caches = [MultiLayerPagedKVCache4Bit(2, 16, 64, DEV, 1, 2, 128, group_size=2) for _ in range(2)]
    k = torch.randn(2, 9, 2, 128, device=DEV, generator=g).half()
    q = torch.randn(2, 1, 4, 128, device=DEV, generator=g).half()
    for c in caches:
        c.update(k, k, 0)
    for T in (2, 9):
        with pytest.raises(ValueError, match="one token"):
            caches[0].update(k[:, :T], k[:, :T], 0)
        assert caches[0].length == 9
    outs = [c.update(k[:, :1], k[:, 1:2], 0)(q) for c in caches]
    assert torch.equal(*outs) and caches[0].length == 10
