"""Checkpoints of decode layers with query / key norms: their weights are written,
read, and missed or refused where layer and checkpoint differ."""
import pytest
import torch

from signrot_amd import checkpoint as ck
from signrot_amd.transformers.decode_layer import W4A4LlamaDecodeLayer

P = "model.layers.2."


def _layer(qk_norm, seed=3):
    layer = W4A4LlamaDecodeLayer.random(256, 4, 2, 64, 512, seed=seed, device="cpu",
                                        qk_norm=qk_norm)
    if qk_norm:
        g = torch.Generator().manual_seed(seed)
        layer.q_norm.copy_(1 + 0.2 * torch.randn(64, generator=g))
        layer.k_norm.copy_(1 + 0.2 * torch.randn(64, generator=g))
    return layer


def _saved(path, tensors):
    ck.save_packed_checkpoint(str(path), tensors, {"format": "packed_int4"})
    return ck.PackedCheckpoint(str(path))


@pytest.mark.parametrize("qk_norm", [True, False])
def test_round_trip(tmp_path, qk_norm):
    src = _layer(qk_norm)
    t = ck.decode_layer_tensors(src, P)
    assert (P + "self_attn.q_norm.weight" in t) == qk_norm
    dst = W4A4LlamaDecodeLayer(256, 4, 2, 64, 512, qk_norm=qk_norm)
    ck.load_decode_layer(dst, _saved(tmp_path, t), P)
    want = dict(src.named_buffers())
    for name, b in dst.named_buffers():
        assert torch.equal(b, want[name]), name


def test_layer_and_checkpoint_that_differ_are_refused(tmp_path):
    full = ck.decode_layer_tensors(_layer(True), P)
    half = {k: v for k, v in full.items() if "k_norm" not in k}
    none = {k: v for k, v in full.items() if "_norm" not in k}
    short = dict(full)
    short[P + "self_attn.q_norm.weight"] = torch.ones(1).half()   # would broadcast
    for i, (t, qk_norm) in enumerate(((none, True), (half, True), (full, False), (half, False),
                                      (short, True))):
        layer = W4A4LlamaDecodeLayer(256, 4, 2, 64, 512, qk_norm=qk_norm)
        with pytest.raises(ValueError, match="norm"):
            ck.load_decode_layer(layer, _saved(tmp_path / str(i), t), P)
        assert (layer.w_qkv == 0).all()
