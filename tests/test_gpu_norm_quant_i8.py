"""rmsnorm_quant_i8 and sym_quant_dynamic_i8 against 64 bits: codes and scales are
equal, since the operators define them by 64-bit arithmetic; the sum is one fp16
addition, and the normalised rows are rounded once."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA
from tests import act8_ref as ref
from tests.gpu_util import DEV, to_dev, to_np

pytestmark = pytest.mark.gpu


def _rows(rng, rows, n, mag=1.0):
    x = rng.standard_normal((rows, n)) * mag
    x[:, rng.permutation(n)[: max(1, n // 1000)]] *= 20
    return x.astype(np.float16)


def _check(x, got, residual=None, weight=None, eps=1e-5, mean_dim=None, clip=1.0, keep=False):
    q, s, h, y = ref.norm_quant(x, eps, mean_dim, residual, weight, clip)
    assert np.array_equal(to_np(got[1]), s, equal_nan=True)
    assert np.array_equal(to_np(got[0]), q)
    if residual is not None:
        assert np.array_equal(to_np(got[2]), h, equal_nan=True)
    if keep:
        out = to_np(got[-1]).astype(np.float64)
        tol = (ref.U16 + 4 * ref.U32) * np.abs(y) + ref.TINY
        assert (np.abs(out - y) <= tol).all()


# every length class: a wave a row (512, 1024), blocks, the long form; odd lengths
SIZES = [(1, 1), (3, 2), (5, 7), (2, 8), (9, 511), (4, 512), (6, 513), (3, 1000), (5, 1025),
         (2, 2047), (1, 2048), (3, 2049), (1, 4096), (7, 4097), (33, 5120), (600, 5120),
         (520, 4096), (513, 8192), (514, 11008), (520, 16000), (2, 8191), (3, 8192),
         (2, 8200), (2, 14336), (3, 16385), (2, 28672), (1, 32768), (3, 32769), (2, 40007)]


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("added,weighted", [(False, False), (True, True), (True, False),
                                            (False, True)])
def test_norm_matches(rows, n, added, weighted):
    rng = np.random.default_rng(rows * 31 + n)
    x = _rows(rng, rows, n)
    r = _rows(rng, rows, n, 4) if added else None
    w = (1 + 0.3 * rng.standard_normal(n)).astype(np.float16) if weighted else None
    got = _CUDA.rmsnorm_quant_i8(to_dev(x), 1e-5, residual=None if r is None else to_dev(r),
                                 weight=None if w is None else to_dev(w), return_norm=True)
    _check(x, got, r, w, keep=True)


@pytest.mark.parametrize("rows,n", SIZES)
def test_quant_matches(rows, n):
    rng = np.random.default_rng(rows + n)
    x = _rows(rng, rows, n)
    got = _CUDA.sym_quant_dynamic_i8(to_dev(x))
    q, s = ref.quant(x.astype(np.float64))
    assert np.array_equal(to_np(got[1]), s) and np.array_equal(to_np(got[0]), q)


@pytest.mark.parametrize("clip", [1.0, 0.9, 0.5, 1e-3])
def test_clip(clip):
    rng = np.random.default_rng(3)
    x = _rows(rng, 6, 4096)
    q, s = ref.quant(x.astype(np.float64), clip)
    got = _CUDA.sym_quant_dynamic_i8(to_dev(x), clip)
    assert np.array_equal(to_np(got[1]), s) and np.array_equal(to_np(got[0]), q)
    got = _CUDA.rmsnorm_quant_i8(to_dev(x), 1e-6, clip_ratio=clip)
    _check(x, got, eps=1e-6, clip=clip)


def test_ties_go_to_even():
    """Scale 1 and values of n + 1/2: quotients are exact ties."""
    x = np.zeros((2, 300), np.float16)
    x[:, :254] = np.arange(-127, 127) + 0.5
    x[:, -1] = 127
    x[1] = -x[1]
    got = _CUDA.sym_quant_dynamic_i8(to_dev(x))
    q, s = ref.quant(x.astype(np.float64))
    assert (s == 1).all()
    assert np.array_equal(to_np(got[0]), q)


@pytest.mark.parametrize("n", [96, 1000, 4096, 40000])
def test_odd_rows(n):
    """Zeros, single values, subnormal ones, the largest, NaN and infinities: one row
    does not reach another."""
    rng = np.random.default_rng(n)
    x = _rows(rng, 10, n)
    x[1] = 0
    x[2] = 0
    x[2, n // 2] = 3
    x[3, n - 1] = np.nan
    x[4, 0] = np.inf
    x[5, 1] = -np.inf
    x[6] = 6e-8
    x[7] = 65504
    x[8, ::2] = -65504
    got = _CUDA.rmsnorm_quant_i8(to_dev(x), 1e-5)
    _check(x, got)
    got = _CUDA.sym_quant_dynamic_i8(to_dev(x))
    q, s = ref.quant(x.astype(np.float64))
    assert np.array_equal(to_np(got[1]), s, equal_nan=True) and np.array_equal(to_np(got[0]), q)
    assert np.isnan(s[3:6]).all() and not np.isnan(np.delete(s, [3, 4, 5])).any()
    # an overflowing sum is an infinity in the residual stream, and is seen
    r = np.zeros_like(x)
    r[0, 0] = x[0, 0] = 60000
    got = _CUDA.rmsnorm_quant_i8(to_dev(x), 1e-5, residual=to_dev(r))
    _check(x, got, r)
    assert np.isnan(to_np(got[1])[0])
    w = np.ones(n, np.float16)
    w[3] = np.nan
    got = _CUDA.rmsnorm_quant_i8(to_dev(x[:2]), 1e-5, weight=to_dev(w))
    assert np.isnan(to_np(got[1])).all() and not to_np(got[0]).any()


def test_eps_zero_and_mean_dim():
    rng = np.random.default_rng(8)
    x = _rows(rng, 3, 640)
    _check(x, _CUDA.rmsnorm_quant_i8(to_dev(x), 0.0, 4096), eps=0.0, mean_dim=4096)
    x[1] = 0   # 0 / 0
    got = to_np(_CUDA.rmsnorm_quant_i8(to_dev(x), 0.0)[1])
    assert np.isnan(got[1]) and not np.isnan(got[[0, 2]]).any()
    _check(x, _CUDA.rmsnorm_quant_i8(to_dev(x), 3, 640), eps=3)


@pytest.mark.parametrize("n", [64, 1001, 4096, 36000])
def test_strided_rows_and_alignment(n):
    """Column slices, transposed leading dims, every alignment of a row."""
    rng = np.random.default_rng(n)
    base = _rows(rng, 12, n + 29)
    x = to_dev(base)
    for lo in (0, 1, 8, 13):
        part = x[:, lo: lo + n]
        _check(base[:, lo: lo + n], _CUDA.rmsnorm_quant_i8(part, 1e-5, residual=part[:, :]),
               base[:, lo: lo + n])
        q, s = _CUDA.sym_quant_dynamic_i8(part[::3])
        rq, rs = ref.quant(base[::3, lo: lo + n].astype(np.float64))
        assert np.array_equal(to_np(q), rq) and np.array_equal(to_np(s), rs)
    q, s = _CUDA.sym_quant_dynamic_i8(x.view(3, 4, -1)[:, :, :n])
    rq, rs = ref.quant(base[:, :n].astype(np.float64))
    assert q.shape == (3, 4, n) and s.shape == (3, 4, 1)
    assert np.array_equal(to_np(q).reshape(12, n), rq)


@pytest.mark.parametrize("n", [700, 4096, 33000])
def test_sum_in_place(n):
    rng = np.random.default_rng(n + 1)
    x, r = _rows(rng, 9, n), _rows(rng, 9, n, 4)
    for alias in range(3):
        xd, rd = to_dev(x), to_dev(r)
        out = (xd, rd, torch.empty_like(xd))[alias]
        got = _CUDA.rmsnorm_quant_i8(xd, 1e-5, residual=rd, out=out)
        assert got[2].data_ptr() == out.data_ptr()
        _check(x, got, r)


def test_many_rows():
    """More rows than one launch dimension of 65535."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((70001, 72)).astype(np.float16)
    got = _CUDA.sym_quant_dynamic_i8(to_dev(x))
    q, s = ref.quant(x.astype(np.float64))
    assert np.array_equal(to_np(got[1]), s) and np.array_equal(to_np(got[0]), q)


def test_more_blocks_than_a_launch_dimension_takes():
    rng = np.random.default_rng(6)
    x = rng.standard_normal(((1 << 22) + 9, 8)).astype(np.float16)
    got = _CUDA.sym_quant_dynamic_i8(to_dev(x))
    q, s = ref.quant(x.astype(np.float64))
    assert np.array_equal(to_np(got[1]), s) and np.array_equal(to_np(got[0]), q)


def test_offsets_past_32_bits():
    """Rows beyond element 2^31 of a strided buffer, sum in place."""
    n, rows = 4099, 530000
    x = torch.zeros(rows, n, dtype=torch.float16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    at = torch.tensor([0, 523776, 524288, rows - 1], device=DEV)
    x[at] = torch.randn(4, n, device=DEV, generator=g).half()
    r = torch.zeros_like(x)
    r[at] = torch.randn(4, n, device=DEV, generator=g).half()
    xs, rs = to_np(x[at]), to_np(r[at])
    got = _CUDA.rmsnorm_quant_i8(x, 1e-5, residual=r, out=r)
    _check(xs, [t[at] for t in got], rs)
    assert not got[1][1:523776].any() and not got[0][1:1000].any()


def test_stream_and_graph():
    """On a stream of its own and replayed on new inputs."""
    rng = np.random.default_rng(4)
    x, r = to_dev(_rows(rng, 17, 4096)), to_dev(_rows(rng, 17, 4096, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _CUDA.rmsnorm_quant_i8(x, 1e-5, residual=r)
    side.synchronize()
    _check(to_np(x), got, to_np(r))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _CUDA.rmsnorm_quant_i8(x, 1e-5, residual=r, return_norm=True)
    for _ in range(3):
        nx, nr = _rows(rng, 17, 4096), _rows(rng, 17, 4096, 4)
        x.copy_(to_dev(nx))
        r.copy_(to_dev(nr))
        g.replay()
        torch.cuda.synchronize()
        _check(nx, got, nr, keep=True)


def test_refusals():
    x = torch.zeros(4, 64, dtype=torch.float16, device=DEV)
    bad = RuntimeError
    with pytest.raises(bad, match="torch.float16"):
        _CUDA.rmsnorm_quant_i8(x.float(), 1e-5)
    with pytest.raises(bad, match="x's shape"):
        _CUDA.rmsnorm_quant_i8(x, 1e-5, residual=x[:2])
    with pytest.raises(bad, match="weight must be"):
        _CUDA.rmsnorm_quant_i8(x, 1e-5, weight=x[0, :32])
    with pytest.raises(bad, match="with a residual"):
        _CUDA.rmsnorm_quant_i8(x, 1e-5, out=x)
    with pytest.raises(bad, match="dense in its last"):
        _CUDA.sym_quant_dynamic_i8(x.t())
    with pytest.raises(bad, match="evenly spaced"):
        _CUDA.sym_quant_dynamic_i8(x.view(2, 2, 64).transpose(0, 1)[:, :, :32])
    with pytest.raises(bad, match="row stride"):
        _CUDA.sym_quant_dynamic_i8(x[:1].expand(3, 64))
    for clip in (0.0, 1.5, float("nan")):
        with pytest.raises(bad, match="clip_ratio"):
            _CUDA.sym_quant_dynamic_i8(x, clip)
    for eps in (-1.0, float("nan")):
        with pytest.raises(bad, match="eps"):
            _CUDA.rmsnorm_quant_i8(x, eps)
    with pytest.raises(bad, match="mean_dim"):
        _CUDA.rmsnorm_quant_i8(x, 1e-5, 0)
    q, s = _CUDA.sym_quant_dynamic_i8(x[:0])
    assert q.shape == (0, 64) and s.shape == (0, 1)
