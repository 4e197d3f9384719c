"""w4a8_linear against the product in 64 bits."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA
from tests import act8_ref as ref
from tests.gpu_util import DEV, to_dev, to_np

pytestmark = pytest.mark.gpu


def _operands(rng, M, N, K):
    a = rng.integers(-128, 128, (M, K)).astype(np.int8)
    c = rng.integers(-8, 8, (N, K)).astype(np.int8)
    sa = rng.uniform(0.005, 0.05, M).astype(np.float32)
    sb = rng.uniform(0.0005, 0.003, N).astype(np.float16)
    return a, sa, c, sb


def _run(a, sa, c, sb, bias=None, residual=None):
    extra = [None if t is None else to_dev(t) for t in (bias, residual)]
    return to_np(_CUDA.w4a8_linear(to_dev(a), to_dev(sa), to_dev(ref.pack(c)), to_dev(sb), *extra))


# rows and columns on both sides of the tiles' edges, K with and without a tail, few
# tiles (split over K), one row to many
SHAPES = [(1, 1, 32), (1, 16, 128), (2, 17, 96), (7, 33, 160), (8, 48, 4096), (9, 16, 1024),
          (16, 31, 2080), (17, 1111, 416), (31, 100, 4128), (32, 64, 11008), (1, 4128, 4096),
          (5, 8200, 512), (20, 4104, 1056), (33, 65, 128), (33, 64, 4096), (64, 130, 14336),
          (64, 4100, 96), (65, 63, 2048), (100, 1111, 8192), (128, 128, 32), (129, 257, 4064),
          (300, 515, 1024), (200, 8193, 512), (513, 128, 4096), (1000, 515, 2208),
          (257, 12800, 256), (1030, 12801, 288), (515, 17000, 128),
          # a round of large tiles and a rest of half ones
          (1300, 13000, 160), (2049, 8300, 96),
          # each tile, in one part and split over K, with tails of all three sizes
          (100, 14340, 1056), (20, 16400, 2080), (24, 10250, 1056), (128, 28700, 352),
          (129, 14339, 2016), (200, 4111, 9312), (130, 2050, 20512), (512, 2100, 14368),
          (384, 3000, 16416), (256, 2048, 16384), (40, 600, 8224), (33, 1, 32),
          # streams in units of 256 codes, of 128 beside them
          (3, 4100, 32), (16, 8192, 1120), (11, 5000, 2464), (8, 6001, 96), (16, 4500, 5024),
          (16, 8193, 1120), (30, 5000, 2464)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_is_exact(M, N, K):
    """Scales that keep the sums of up to 2^24 exact in fp32 and the result within
    fp16: only its rounding is left, so it is the rounded exact product."""
    rng = np.random.default_rng(M + 3 * N + K)
    a, _, c, _ = _operands(rng, M, N, K)
    sa = np.full(M, 2.0 ** -9, np.float32)
    sb = np.full(N, 2.0 ** -3, np.float16)
    acc = a.astype(np.float64) @ c.astype(np.float64).T
    assert np.abs(acc).max() < 2 ** 24
    assert np.array_equal(_run(a, sa, c, sb), (acc * 2.0 ** -12).astype(np.float16))


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, True)])
def test_matches(M, N, K, bias, residual):
    rng = np.random.default_rng(M * 5 + N + K)
    a, sa, c, sb = _operands(rng, M, N, K)
    b = rng.standard_normal(N).astype(np.float16) if bias else None
    r = (4 * rng.standard_normal((M, N))).astype(np.float16) if residual else None
    want, tol = ref.linear(a, sa, c, sb, b, r)
    err = np.abs(_run(a, sa, c, sb, b, r) - want)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("M,N,K", [(3, 64, 131040), (40, 64, 131040), (300, 96, 65536)])
def test_largest_sums(M, N, K):
    """Every product the largest: sums of up to 2^27, 2^31 inside."""
    a = np.full((M, K), -128, np.int8)
    c = np.full((N, K), -8, np.int8)
    a[1], c[1] = 127, 7
    sa, sb = np.full(M, 2.0 ** -9, np.float32), np.full(N, 2.0 ** -10, np.float16)
    want, tol = ref.linear(a, sa, c, sb)
    assert (np.abs(_run(a, sa, c, sb) - want) <= tol).all()


def test_rows_do_not_meet():
    """A row with NaN scale, and rows of the largest codes, leave the others alone; a
    row's result is the same in any batch of its kernel."""
    rng = np.random.default_rng(1)
    for M in (6, 30, 60, 700):
        a, sa, c, sb = _operands(rng, M, 80, 1024)
        one = _run(a, sa, c, sb)
        sa[2] = np.nan
        a[4] = -128
        two = _run(a, sa, c, sb)
        assert np.isnan(two[2]).all()
        keep = [m for m in range(M) if m not in (2, 4)]
        assert np.array_equal(one[keep], two[keep])


@pytest.mark.parametrize("M", [5, 70, 600])
def test_in_place_residual_and_shapes(M):
    rng = np.random.default_rng(M)
    a, sa, c, sb = _operands(rng, M, 300, 512)
    r = rng.standard_normal((M, 300)).astype(np.float16)
    want = _run(a, sa, c, sb, None, r)
    rd = to_dev(r)
    got = _CUDA.w4a8_linear(to_dev(a).view(M, 1, 512), to_dev(sa).view(M, 1, 1),
                            to_dev(ref.pack(c)), to_dev(sb).view(-1, 1), None, rd.view(M, 1, 300),
                            out=rd.view(M, 1, 300))
    assert got.shape == (M, 1, 300) and np.array_equal(to_np(rd), want)


@pytest.mark.parametrize("M", [1, 48, 130])
def test_stream_and_graph(M):
    """On a stream of its own, and two captured products replayed on new inputs with
    eager work between: their workspaces do not meet."""
    rng = np.random.default_rng(M)
    a, sa, c, sb = _operands(rng, M, 512, 4096)
    t = [to_dev(v) for v in (a, sa, ref.pack(c), sb)]
    want = _run(a, sa, c, sb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _CUDA.w4a8_linear(*t)
    side.synchronize()
    assert np.array_equal(to_np(got), want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, _CUDA.w4a8_linear(*t)))
    for _ in range(3):
        na = rng.integers(-127, 128, a.shape).astype(np.int8)
        t[0].copy_(to_dev(na))
        for g, out in graphs:
            g.replay()
        eager = _CUDA.w4a8_linear(*t)
        torch.cuda.synchronize()
        want = _run(na, sa, c, sb)
        assert np.array_equal(to_np(eager), want)
        for _, out in graphs:
            assert np.array_equal(to_np(out), want)


def test_offsets_past_32_bits():
    """An output of 4.6 GB, and rows of activations beyond 4 GiB."""
    rng = np.random.default_rng(3)
    M, N, K = 40000, 57344, 32
    a, sa, c, sb = _operands(rng, M, N, K)
    out = _CUDA.w4a8_linear(*(to_dev(t) for t in (a, sa, ref.pack(c), sb)))
    rows = np.array([0, 17, 37449, 39999])
    want, tol = ref.linear(a[rows], sa[rows], c, sb)
    assert (np.abs(to_np(out[torch.from_numpy(rows).to(DEV)]) - want) <= tol).all()
    del out
    M, N, K = 70000, 130, 65536
    a = torch.randint(-128, 128, (M, K), dtype=torch.int8, device=DEV)
    c = rng.integers(-8, 8, (N, K)).astype(np.int8)
    sa, sb = rng.uniform(0.001, 0.01, M).astype(np.float32), sb[:N]
    out = _CUDA.w4a8_linear(a, to_dev(sa), to_dev(ref.pack(c)), to_dev(sb))
    rows = np.array([0, 32767, 32768, 65535, 65536, 69999])
    want, tol = ref.linear(to_np(a[torch.from_numpy(rows).to(DEV)]), sa[rows], c, sb)
    assert (np.abs(to_np(out[torch.from_numpy(rows).to(DEV)]) - want) <= tol).all()


def test_two_streams_at_once():
    """Products that are split over K, each with a workspace of its own."""
    rng = np.random.default_rng(4)
    calls = []
    for M in (48, 130):
        a, sa, c, sb = _operands(rng, M, 640, 8192)
        t = [to_dev(v) for v in (a, sa, ref.pack(c), sb)]
        calls.append((t, to_np(_CUDA.w4a8_linear(*t)), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for (t, _, s), o in zip(calls, outs):
            with torch.cuda.stream(s):
                o.append(_CUDA.w4a8_linear(*t))
    torch.cuda.synchronize()
    for (_, want, _), o in zip(calls, outs):
        for got in o:
            assert np.array_equal(to_np(got), want)


def test_refusals():
    a = torch.zeros(4, 64, dtype=torch.int8, device=DEV)
    sa = torch.ones(4, device=DEV)
    w = torch.zeros(16, 32, dtype=torch.uint8, device=DEV)
    sb = torch.ones(16, dtype=torch.float16, device=DEV)
    bad = RuntimeError
    for args, match in [((a.float(), sa, w, sb), "torch.int8"), ((a, sa.half(), w, sb), "float32"),
                        ((a, sa[:3], w, sb), "a value a row"), ((a, sa, w, sb[:8]), "b_scale N"),
                        ((a, sa, w[:, :16].contiguous(), sb), "expected A"),
                        ((a, sa, w, sb, sb[:4]), "bias"),
                        ((a, sa, w, sb, None, torch.zeros(4, 8, dtype=torch.float16, device=DEV)),
                         "residual must be"),
                        ((a[:, :16].contiguous(), sa, w[:, :8].contiguous(), sb), "multiple of 32"),
                        ((a.t(), sa, w, sb), "contiguous"), ((a.cpu(), sa, w, sb), "GPU")]:
        with pytest.raises(bad, match=match):
            _CUDA.w4a8_linear(*args)
    flat = torch.zeros(4 * 64 + 8, dtype=torch.int8, device=DEV)
    with pytest.raises(bad, match="16-byte aligned"):
        _CUDA.w4a8_linear(flat[8:].view(4, 64), sa, w, sb)
    assert _CUDA.w4a8_linear(a[:0], sa[:0], w, sb).shape == (0, 16)
