"""qk_norm_rope against the formula in 64 bits: head dims, layouts, weights,
no norm, values at the ends of fp16, and its refusals."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA
from tests import i8_ref
from tests.gpu_util import DEV, to_np

pytestmark = pytest.mark.gpu


def _close(got, want, size, D):
    """One rounding to fp16 (2^-11 of the value, half the subnormal step 2^-25)
    behind fp32 arithmetic: the sum of D squares, a square root, a division and
    four products, each off by at most 2^-23 relative, the sum of squares by D / 8
    + 6 additions (halved by the square root)."""
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + size * (D / 16 + 12) * 2.0 ** -23
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (err / tol).max()


def _case(B, T, Hq, Hk, D, seed=0, scale=1.0, cos_batch=1):
    g = torch.Generator().manual_seed(seed)
    qkv = (scale * torch.randn(B, T, Hq + 2 * Hk, D, generator=g)).half()
    ang = torch.rand(cos_batch, T, D, generator=g) * 6.3
    w = [(1 + 0.3 * torch.randn(D, generator=g)).half() for _ in range(2)]
    return qkv, ang.cos().half(), ang.sin().half(), w


def _run(qkv, Hq, Hk, cos, sin, w, eps):
    x = qkv.to(DEV)
    q, k = x[:, :, :Hq], x[:, :, Hq: Hq + Hk]
    qw, kw = (None if t is None else t.to(DEV) for t in w)
    out = _CUDA.qk_norm_rope(q, k, cos.to(DEV), sin.to(DEV), qw, kw, eps)
    torch.cuda.synchronize()
    return out


def _check(qkv, Hq, Hk, cos, sin, w, eps):
    qo, ko = _run(qkv, Hq, Hk, cos, sin, w, eps)
    D = qkv.shape[-1]
    c, s = cos.numpy()[:, :, None], sin.numpy()[:, :, None]
    for got, x, wt in ((qo, qkv[:, :, :Hq], w[0]), (ko, qkv[:, :, Hq: Hq + Hk], w[1])):
        assert got.is_contiguous() and got.shape == x.shape
        want, size = i8_ref.norm_rope(x.numpy(), None if wt is None else wt.numpy(), c, s, eps)
        _close(to_np(got), want, size, D)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,T,Hq,Hk", [(1, 1, 1, 1), (5, 1, 32, 8), (2, 33, 40, 8), (1, 1100, 7, 3),
                                       (3, 17, 4, 0), (2, 3, 65, 1)])
def test_matches_formula(B, T, Hq, Hk, D):
    _check(*_slots(_case(B, T, Hq, Hk, D, seed=B * 100 + T), Hq, Hk), 1e-6)


def _slots(case, Hq, Hk):
    qkv, cos, sin, w = case
    return qkv, Hq, Hk, cos, sin, w


def test_batched_tables():
    _check(*_slots(_case(4, 9, 8, 2, 128, seed=3, cos_batch=4), 8, 2), 1e-5)


@pytest.mark.parametrize("T", [512, 513])
def test_tokens_with_many_heads(T):
    """A block for every group of heads, and one for all of a token's."""
    _check(*_slots(_case(1, T, 33, 8, 128, seed=T), 33, 8), 1e-6)


@pytest.mark.parametrize("use", [(False, False), (True, False), (False, True)])
def test_optional_weights(use):
    qkv, cos, sin, w = _case(2, 7, 8, 2, 128, seed=4)
    _check(qkv, 8, 2, cos, sin, [t if u else None for t, u in zip(w, use)], 1e-6)


def test_without_norm():
    qkv, cos, sin, _ = _case(2, 7, 8, 2, 128, seed=5)
    _check(qkv, 8, 2, cos, sin, (None, None), None)


@pytest.mark.parametrize("scale", [1e-4, 1e3, 15000.0])
def test_far_magnitudes(scale):
    """Subnormal inputs, and squares that only fp32 holds."""
    _check(*_slots(_case(2, 5, 8, 2, 256, seed=6, scale=scale), 8, 2), 1e-6)


def test_zero_rows_and_nonfinite_values():
    qkv, cos, sin, w = _case(1, 4, 4, 1, 128, seed=7)
    qkv[0, 0] = 0
    qkv[0, 1, 0, 5] = float("nan")
    qkv[0, 2, 1, 100] = float("inf")
    qo, ko = _run(qkv, 4, 1, cos, sin, w, 1e-6)
    assert (qo[0, 0] == 0).all() and (ko[0, 0] == 0).all()
    assert torch.isnan(qo[0, 1, 0]).all()            # the row's mean is NaN
    bad = torch.isnan(qo[0, 2, 1]) | (qo[0, 2, 1] == 0)
    assert bad.all() and torch.isnan(qo[0, 2, 1, 100])   # inf / inf, finite / inf
    clean = [(0, 1, 1), (0, 1, 2), (0, 1, 3), (0, 2, 0), (0, 2, 2), (0, 3, 0)]
    assert all(torch.isfinite(qo[i]).all() for i in clean) and torch.isfinite(ko).all()


def test_inputs_are_kept_and_empty_calls():
    qkv, cos, sin, w = _case(2, 3, 4, 2, 128, seed=8)
    x = qkv.to(DEV)
    before = x.clone()
    _CUDA.qk_norm_rope(x[:, :, :4], x[:, :, 4:6], cos.to(DEV), sin.to(DEV))
    assert torch.equal(x, before)
    q, k = _CUDA.qk_norm_rope(x[:0, :, :4], x[:0, :, 4:6], cos.to(DEV), sin.to(DEV))
    assert q.shape == (0, 3, 4, 128) and k.shape == (0, 3, 2, 128)


def test_refusals():
    qkv, cos, sin, w = _case(2, 3, 4, 2, 128, seed=9)
    x, c, s = qkv.to(DEV), cos.to(DEV), sin.to(DEV)
    q, k = x[:, :, :4], x[:, :, 4:6]
    w = [t.to(DEV) for t in w]
    bad = [
        (q.float(), k, c, s), (q, k.bfloat16(), c, s), (q.cpu(), k, c, s),
        (q[:, :2], k, c, s), (q, k[..., :64], c, s), (q[..., ::2], k[..., ::2], c, s),
        (q.transpose(1, 2), k.transpose(1, 2), c, s), (q, k, c[:, :2], s[:, :2]),
        (q, k, c, s[..., :64]), (q[0], k[0], c, s), (q, k, c.float(), s),
        (q, k, c, s, w[0][:64]), (q, k, c, s, None, w[1][None]), (q, k, c, s, w[0], None, None),
        (q, k, c, s, None, None, -1.0), (q, k, c, s, None, None, float("nan")),
        (q[..., 1:97], k[..., 1:97], c[..., :96].contiguous(), s[..., :96].contiguous()),
        (x.view(2, 3, -1)[:, :, 4: 4 + 512].view(2, 3, 4, 128), k, c, s),   # 8-byte aligned
        (q[:, :1].expand(2, 3, 4, 128), k, c, s),                            # token stride 0
    ]
    for args in bad:
        with pytest.raises(RuntimeError):
            _CUDA.qk_norm_rope(*args)
