"""w4a16_linear: 4-bit weights with group scales against the product in 64 bits."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA
from tests.gpu_util import DEV, to_np

pytestmark = pytest.mark.gpu


def _pack(c):
    u = (c & 15).astype(np.uint8)
    return u[:, 0::2] | (u[:, 1::2] << 4)


def _weights(rng, N, K, group, asym):
    c = rng.integers(0, 16, (N, K)) if asym else rng.integers(-8, 8, (N, K))
    z = rng.integers(0, 16, (N, K // group)).astype(np.uint8) if asym else None
    return c, z


def _dense(c, z, s, group):
    w = c.astype(np.float64)
    if z is not None:
        w = w - np.repeat(z.astype(np.float64), group, 1)
    return w * np.repeat(s.astype(np.float64), group, 1)


def _run(x, c, s, z=None, bias=None):
    t = [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
         for a in (x, _pack(c), s, z, bias)]
    return to_np(_CUDA.w4a16_linear(*t))


SHAPES = [(1, 1, 32, 32), (1, 16, 128, 128), (3, 17, 96, 32), (16, 48, 256, 64), (17, 33, 384, 128),
          (2, 1111, 1056, 96), (33, 80, 2048, 256), (5, 64, 11008, 128), (1, 4096, 4096, 128),
          (7, 130, 1024, 1024), (64, 48, 640, 32), (70, 257, 512, 64), (4, 4096, 160, 160),
          # two row tiles a wave
          (5, 8200, 384, 128), (1, 8193, 640, 32), (20, 8192, 1024, 64), (3, 8208, 1056, 96),
          # more groups a wave than it holds in LDS at a time
          (1, 16, 40960, 128), (3, 20, 20480, 64), (2, 16, 12288, 32), (16, 33, 9312, 96)]


@pytest.mark.parametrize("M,N,K,group", SHAPES)
@pytest.mark.parametrize("asym", [False, True])
def test_integer_inputs_are_exact(M, N, K, group, asym):
    """x whole numbers, scales powers of two: every partial sum is a multiple of
    2^-3 below 2^21 (K 3 15 2), which fp32 holds, so only the rounding to fp16 is
    left and the result is the rounded exact product, in any order of addition."""
    rng = np.random.default_rng(M * 7 + N + K)
    c, z = _weights(rng, N, K, group, asym)
    x = rng.integers(-3, 4, (M, K)).astype(np.float16)
    s = (2.0 ** rng.integers(-3, 1, (N, K // group))).astype(np.float16)
    got = _run(x, c, s, z)
    want = x.astype(np.float64) @ _dense(c, z, s, group).T
    assert np.abs(want).max() < 65504
    assert np.array_equal(got, want.astype(np.float16))


@pytest.mark.parametrize("M,N,K,group", SHAPES)
@pytest.mark.parametrize("asym", [False, True])
def test_matches_product(M, N, K, group, asym):
    """fp16 rounding of the result (2^-11) behind fp32 sums of K products, each
    exact in fp32: at most K + groups + 16 roundings of 2^-24 in any order, each of
    a partial sum that the products' magnitudes bound.  (The exact test above is the
    sharper one for the sums.)"""
    rng = np.random.default_rng(M + N * 3 + K)
    c, z = _weights(rng, N, K, group, asym)
    x = rng.standard_normal((M, K)).astype(np.float16)
    s = rng.uniform(0.005, 0.03, (N, K // group)).astype(np.float16)
    bias = rng.standard_normal(N).astype(np.float16)
    got = _run(x, c, s, z, bias)
    w = _dense(c, z, s, group)
    want = x.astype(np.float64) @ w.T + bias.astype(np.float64)
    size = np.abs(x.astype(np.float64)) @ np.abs(w).T + np.abs(bias.astype(np.float64))
    tol = 2.0 ** -11 * np.abs(want) + (K + K // group + 16) * 2.0 ** -24 * size + 2.0 ** -25
    err = np.abs(got - want)
    assert (err <= tol).all(), (err / tol).max()


def test_small_scales_keep_their_precision():
    """Weights far below fp16's smallest normal number: scales stay out of fp16
    products."""
    rng = np.random.default_rng(5)
    c, _ = _weights(rng, 64, 256, 64, False)
    x = (rng.integers(-3, 4, (4, 256)) * 1024).astype(np.float16)
    s = np.full((64, 4), 2.0 ** -20, np.float16)
    want = x.astype(np.float64) @ _dense(c, None, s, 64).T
    assert np.array_equal(_run(x, c, s), want.astype(np.float16))


def test_leading_dims_empty_rows_and_nonfinite():
    rng = np.random.default_rng(6)
    c, _ = _weights(rng, 40, 128, 64, False)
    s = np.ones((40, 2), np.float16)
    w, st = torch.from_numpy(_pack(c)).to(DEV), torch.from_numpy(s).to(DEV)
    x = torch.from_numpy(rng.integers(-3, 4, (2, 3, 128)).astype(np.float16)).to(DEV)
    out = _CUDA.w4a16_linear(x, w, st)
    assert out.shape == (2, 3, 40)
    assert torch.equal(out.view(6, 40), _CUDA.w4a16_linear(x.view(6, 128), w, st))
    assert _CUDA.w4a16_linear(x[:0], w, st).shape == (0, 3, 40)
    bad = x.clone()
    bad[0, 1, 77] = float("nan")    # reaches its own row only
    got = _CUDA.w4a16_linear(bad, w, st)
    assert torch.isnan(got[0, 1]).all()
    keep = torch.ones(2, 3, dtype=torch.bool, device=DEV)
    keep[0, 1] = False
    assert torch.equal(got[keep], out[keep])


def test_refusals():
    f16 = dict(dtype=torch.float16, device=DEV)
    x, w = torch.zeros(2, 128, **f16), torch.zeros(16, 64, dtype=torch.uint8, device=DEV)
    s = torch.ones(16, 2, **f16)
    z = torch.zeros(16, 2, dtype=torch.uint8, device=DEV)
    bad = [(x.float(), w, s), (x, w.to(torch.int8), s), (x, w, s.float()), (x.cpu(), w, s),
           (x[:, :64].contiguous(), w, s), (x, w, s[:8].contiguous()),
           (x, w, torch.ones(16, 3, **f16)), (x, w, torch.ones(16, 8, **f16)),
           (x, w, s, z[:, :1].contiguous()), (x, w, s, z.to(torch.int8)),
           (x, w, s, None, torch.zeros(15, **f16)), (x, w, torch.ones(16, 0, **f16)),
           (torch.zeros(2, 256, **f16)[:, ::2], w, s)]
    for args in bad:
        with pytest.raises(RuntimeError):
            _CUDA.w4a16_linear(*args)
    base = torch.zeros(2 * 128 + 4, **f16)
    with pytest.raises(RuntimeError, match="aligned"):
        _CUDA.w4a16_linear(base[4:].view(2, 128), w, s)


def test_stream_and_graph():
    """A projection and the norms behind it, captured on another stream and replayed
    with new inputs and other work between the replays: every replay is the eager
    result bit for bit."""
    rng = np.random.default_rng(9)
    K, heads, D = 512, 6, 128
    c, z = _weights(rng, heads * D, K, 64, True)
    w, zt = torch.from_numpy(_pack(c)).to(DEV), torch.from_numpy(z).to(DEV)
    s = torch.from_numpy(rng.uniform(0.005, 0.03, (heads * D, K // 64)).astype(np.float16)).to(DEV)
    cos, sin = (torch.rand(1, 3, D, device=DEV).half() for _ in range(2))
    x = torch.zeros(1, 3, K, dtype=torch.float16, device=DEV)

    def run():
        y = _CUDA.w4a16_linear(x, w, s, zt).view(1, 3, heads, D)
        return _CUDA.qk_norm_rope(y[:, :, :4], y[:, :, 4:], cos, sin)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = run()
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        x.copy_(torch.from_numpy(rng.standard_normal((1, 3, K)).astype(np.float16)))
        g.replay()
        out = [t.clone() for t in got]
        (torch.randn(1 << 20, device=DEV) * 2).sum()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn
