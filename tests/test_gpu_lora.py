"""lora_add against the adapters in 64 bits."""
import numpy as np
import pytest
import torch

from signrot_amd import _CUDA
from tests import act8_ref as ref
from tests.gpu_util import DEV, to_dev, to_np

pytestmark = pytest.mark.gpu


def _operands(rng, M, K, widths, r, L):
    N = sum(widths)
    x = rng.standard_normal((M, K)).astype(np.float16)
    y = rng.standard_normal((M, N)).astype(np.float16)
    la = (rng.standard_normal((L, len(widths) * r, K)) / np.sqrt(K)).astype(np.float16)
    lb = (0.3 * rng.standard_normal((L, N, r))).astype(np.float16)
    return y, x, la, lb, rng.uniform(0.5, 2, L).astype(np.float32)


def _run(y, x, la, lb, ids, sc=None, widths=None):
    return to_np(_CUDA.lora_add(to_dev(y), to_dev(x), to_dev(la), to_dev(lb), to_dev(ids),
                                None if sc is None else to_dev(sc), widths))


def _ids(rng, M, L, kind):
    if kind == "one":
        ids = np.full(M, L - 1)
    elif kind == "runs":   # requests of uneven lengths, some without an adapter
        ids = np.repeat(rng.integers(-1, L, M), rng.integers(1, 40, M))[:M]
    else:                  # every token another
        ids = rng.integers(-1, L, M)
    return ids.astype(np.int32)


CASES = [(1, 64, (40,), 8, 1), (1, 4096, (4096,), 16, 4), (3, 1000, (111, 7), 8, 5),
         (5, 520, (300,), 24, 3), (32, 4096, (512, 128, 128), 16, 32), (64, 256, (130,), 64, 9),
         (2, 8, (1,), 8, 2), (7, 3144, (64, 3), 256, 2), (33, 128, (9, 8, 7, 6, 5, 4, 3, 2), 8, 4),
         (65, 64, (40,), 8, 1), (70, 1000, (111, 77), 8, 5), (100, 4096, (300,), 16, 3),
         (200, 512, (256, 128, 129), 16, 7), (129, 2056, (1025,), 40, 4), (257, 320, (128,), 64, 64),
         (66, 72, (33, 260), 256, 3), (500, 1096, (65,), 128, 2), (321, 8, (5,), 8, 40),
         (90, 96, (9, 8, 7, 6, 5, 4, 3, 2), 24, 6), (2, 16392, (20,), 8, 2), (3, 64, (2100, 9), 32, 2),
         # tiles of 128 tokens; runs of several column tiles; more rows of A than a block's
         (1100, 264, (700, 60), 16, 3), (1500, 520, (129,), 72, 5), (1300, 128, (20000, 300), 8, 4),
         (1100, 96, (300,) * 8, 24, 6), (1200, 200, (600,), 200, 2),
         # tiles of 64: their adapters' bytes past what is left to single tokens
         (65, 4104, (700, 3), 200, 3), (130, 4096, (1025,), 104, 4), (333, 2056, (128, 129, 1), 40, 7),
         (1000, 264, (4000,), 16, 64), (1024, 3208, (40, 5), 8, 9), (900, 1096, (65,) * 8, 8, 40),
         (701, 6152, (300,), 16, 5), (257, 4096, (20000,), 8, 6),
         # single tokens up to the last
         (1024, 1096, (130,), 8, 40), (1024, 64, (300, 9), 24, 5)]


@pytest.mark.parametrize("M,K,widths,r,L", CASES)
@pytest.mark.parametrize("kind", ["one", "runs", "each"])
def test_matches(M, K, widths, r, L, kind):
    rng = np.random.default_rng(M + K + r)
    y, x, la, lb, sc = _operands(rng, M, K, widths, r, L)
    ids = _ids(rng, M, L, kind)
    got = _run(y, x, la, lb, ids, sc, widths)
    want, tol = ref.lora(y, x, la, lb, ids, sc, widths)
    err = np.abs(got - want)
    assert (err <= tol).all(), (err / tol).max()
    none = ids < 0
    assert np.array_equal(got[none], y[none])


@pytest.mark.parametrize("M,K,widths,r", [(1300, 8192, (300, 40), 96), (17000, 200, (9,), 136),
                                          (20000, 72, (7, 2), 64), (29440, 72, (9,), 136),
                                          (1100, 4160, (33,), 256)])
@pytest.mark.parametrize("lo,hi", [(1, 30), (60, 400), (600, 2000)])
def test_tiles_of_several_requests(M, K, widths, r, lo, hi):
    """Sizes that leave CUs idle, whose blocks take a tile's second adapter: tiles of one
    request, of two and of many, some tokens without an adapter."""
    rng = np.random.default_rng(M + lo)
    L = 6
    y, x, la, lb, sc = _operands(rng, M, K, widths, r, L)
    n = rng.integers(lo, hi, 2 * M // lo + 1)
    ids = np.repeat(rng.integers(-1, L, n.size), n)[:M].astype(np.int32)
    want, tol = ref.lora(y, x, la, lb, ids, sc, widths)
    got = _run(y, x, la, lb, ids, sc, widths)
    assert (np.abs(got - want) <= tol).all()
    assert np.array_equal(got[ids < 0], y[ids < 0])


@pytest.mark.parametrize("M,K", [(40, 512), (300, 512), (900, 2048), (1100, 512)])
def test_integer_inputs_are_exact(M, K):
    """Whole numbers: t below 2^11 and every sum exact in fp32, so the result is the
    rounded exact one, in any order."""
    rng = np.random.default_rng(M)
    widths, r, L = (96, 40), 16, 5
    y = rng.integers(-8, 9, (M, sum(widths))).astype(np.float16)
    x = rng.integers(-1, 2, (M, K)).astype(np.float16)
    la = rng.integers(-2, 3, (L, 2 * r, K)).astype(np.float16)
    lb = rng.integers(-4, 5, (L, sum(widths), r)).astype(np.float16)
    sc = (2.0 ** rng.integers(-2, 2, L)).astype(np.float32)
    ids = _ids(rng, M, L, "runs")
    want, _ = ref.lora(y, x, la, lb, ids, sc, widths)
    assert np.abs(want).max() < 65504
    assert np.array_equal(_run(y, x, la, lb, ids, sc, widths), want.astype(np.float16))


@pytest.mark.parametrize("M,K", [(20, 256), (150, 256), (700, 4096), (1100, 256)])
def test_requests_do_not_meet(M, K):
    """Another request's NaN and infinities, in its tokens or in its adapter, stay with
    it; ids outside the adapters keep y; an unused adapter is not read."""
    rng = np.random.default_rng(M)
    widths, r, L = (128, 33), 16, 6
    y, x, la, lb, sc = _operands(rng, M, K, widths, r, L)
    ids = (np.arange(M) % L).astype(np.int32)
    ids[5], ids[11], ids[13] = -1, L, 2 ** 31 - 1
    want = _run(y, x, la, lb, ids, sc, widths)
    la[1], lb[2, 3], sc[3] = np.inf, np.nan, np.nan
    x[4] = np.nan    # adapter 4's own token
    y[6, 0] = np.inf
    got = _run(y, x, la, lb, ids, sc, widths)
    keep = np.isin(ids, (0, 5)) | (ids < 0) | (ids >= L)
    keep[[4, 6]] = False
    assert np.array_equal(got[keep], want[keep])
    assert np.array_equal(got[[5, 11, 13]], y[[5, 11, 13]])
    assert np.isnan(got[ids == 3]).all() and np.isnan(got[4]).all()
    assert not np.isfinite(got[np.arange(M)[ids == 1]]).any()
    assert np.isinf(got[6, 0]) and np.isfinite(got[6, 1:]).all()


@pytest.mark.parametrize("M,K", [(10, 1024), (100, 1024), (800, 4096), (1100, 1024)])
def test_large_and_small_adapters(M, K):
    """t beyond fp16's range and below its normal numbers: it is held in fp32."""
    rng = np.random.default_rng(M)
    widths, r, L = (96,), 16, 3
    y, x, la, lb, sc = _operands(rng, M, K, widths, r, L)
    ids = _ids(rng, M, L, "each")
    for up in (2.0 ** 13, 2.0 ** -9):
        a = (la.astype(np.float64) * up * 16).astype(np.float16)
        s = (sc / up).astype(np.float32)
        want, tol = ref.lora(y, x, a, lb, ids, s, widths)
        err = np.abs(_run(y, x, a, lb, ids, s, widths) - want)
        assert (err <= tol).all()


@pytest.mark.parametrize("M,K", [(12, 264), (130, 264), (1000, 3272), (1100, 264)])
def test_strides_and_in_place(M, K):
    """Column slices of one projection's output, tokens in two leading dims, out given
    and in place; what lies beside the slice stays."""
    rng = np.random.default_rng(M)
    widths, r, L = (128, 40), 8, 4
    N = sum(widths)
    y, x, la, lb, sc = _operands(rng, M, K, widths, r, L)
    ids = _ids(rng, M, L, "runs")
    want = _run(y, x, la, lb, ids, sc, widths)
    t = [to_dev(v) for v in (la, lb, ids, sc)]
    wide = torch.zeros(M, N + 7, dtype=torch.float16, device=DEV)
    wide[:, 3: 3 + N] = to_dev(y)
    xw = torch.zeros(M, K + 24, dtype=torch.float16, device=DEV)
    xw[:, 8: 8 + K] = to_dev(x)
    part = wide[:, 3: 3 + N]
    got = _CUDA.lora_add(part, xw[:, 8: 8 + K], *t, widths, out=part)
    assert got.data_ptr() == part.data_ptr()
    assert np.array_equal(to_np(part), want)
    assert not wide[:, :3].any() and not wide[:, 3 + N:].any()
    out = torch.zeros(M, 2 * N, dtype=torch.float16, device=DEV)
    _CUDA.lora_add(to_dev(y).view(2, -1, N), to_dev(x).view(2, -1, K), *t, list(widths),
                   out=out.view(2, -1, 2 * N)[..., N:])
    assert np.array_equal(to_np(out[:, N:]), want) and not out[:, :N].any()
    xt = to_dev(np.ascontiguousarray(x))
    assert np.array_equal(to_np(_CUDA.lora_add(to_dev(y), xt, *t[:3], None, widths)),
                          _run(y, x, la, lb, ids, None, widths))


@pytest.mark.parametrize("M", [9, 140, 800, 1100])
def test_stream_and_graph(M):
    rng = np.random.default_rng(M)
    K, widths, r, L = 2048, (256, 64), 16, 8
    y, x, la, lb, sc = _operands(rng, M, K, widths, r, L)
    ids = _ids(rng, M, L, "each")
    t = [to_dev(v) for v in (y, x, la, lb, ids, sc)]
    want = _run(y, x, la, lb, ids, sc, widths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _CUDA.lora_add(*t, widths)
    side.synchronize()
    assert np.array_equal(to_np(got), want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, _CUDA.lora_add(*t, widths)))
    for _ in range(3):   # other tokens and other adapters in the same graph
        nx, nids = rng.standard_normal(x.shape).astype(np.float16), _ids(rng, M, L, "each")
        t[1].copy_(to_dev(nx))
        t[4].copy_(to_dev(nids))
        for g, _ in graphs:
            g.replay()
        eager = _CUDA.lora_add(*t, widths)
        torch.cuda.synchronize()
        want = _run(y, nx, la, lb, nids, sc, widths)
        assert np.array_equal(to_np(eager), want)
        for _, out in graphs:
            assert np.array_equal(to_np(out), want)


@pytest.mark.parametrize("M", [3, 70])
def test_offsets_past_32_bits(M):
    """The last of adapters of 4.4 GB."""
    rng = np.random.default_rng(M)
    K, N, r, L = 64, 28672, 256, 300
    y, x, la, lb, _ = _operands(rng, M, K, (N,), r, 1)
    ad = torch.zeros(L, r, K, dtype=torch.float16, device=DEV)
    bd = torch.zeros(L, N, r, dtype=torch.float16, device=DEV)
    ad[-1], bd[-1] = to_dev(la[0]), to_dev(lb[0])
    ids = np.full(M, L - 1, np.int32)
    ids[1] = 0
    got = to_np(_CUDA.lora_add(to_dev(y), to_dev(x), ad, bd, to_dev(ids)))
    want, tol = ref.lora(y, x, la, lb, np.where(ids == 0, -1, 0), None, (N,))
    assert (np.abs(got - want) <= tol).all()


def test_two_streams_at_once():
    rng = np.random.default_rng(5)
    calls = []
    for M, r in ((300, 16), (1200, 64), (900, 32)):
        y, x, la, lb, sc = _operands(rng, M, 2048, (512, 128), r, 6)
        ids = _ids(rng, M, 6, "runs")
        t = [to_dev(v) for v in (y, x, la, lb, ids, sc)]
        calls.append((t, to_np(_CUDA.lora_add(*t, (512, 128))), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], [], []]
    for _ in range(5):
        for (t, _, s), o in zip(calls, outs):
            with torch.cuda.stream(s):
                o.append(_CUDA.lora_add(*t, (512, 128)))
    torch.cuda.synchronize()
    for (_, want, _), o in zip(calls, outs):
        for got in o:
            assert np.array_equal(to_np(got), want)


def test_refusals():
    f16 = torch.float16

    def z(*s, dt=f16):
        return torch.zeros(*s, dtype=dt, device=DEV)
    y, x, la, lb, ids = z(4, 48), z(4, 64), z(3, 16, 64), z(3, 48, 8), z(4, dt=torch.int32)
    ok = [y, x, la, lb, ids, None, (32, 16)]
    _CUDA.lora_add(*ok)
    bad = RuntimeError

    def refused(match, **kw):
        args = list(ok)
        for k, v in kw.items():
            args["y x la lb ids sc widths".split().index(k)] = v
        with pytest.raises(bad, match=match):
            _CUDA.lora_add(*args)
    refused("do not fit", widths=(32, 8))
    refused("do not fit", widths=None)
    refused("slice of", widths=(48, 0))
    refused("same tokens", x=x[:3])
    refused("one a token", ids=ids[:3])
    refused("torch.int32", ids=ids.long())
    refused("scaling must be", sc=z(2, dt=torch.float32))
    refused("must be", x=z(4, 32))
    refused("expected lora_a", la=la[0])
    refused("16-byte aligned", x=z(4, 68)[:, 4:])
    refused("16-byte aligned", x=z(4, 68)[:, :64])
    refused("rank=4", la=z(3, 8, 64), lb=z(3, 48, 4))
    refused("K=60", la=z(3, 16, 60), x=z(4, 60))
    refused("GPU", y=y.cpu())
    square = z(4, 64)
    with pytest.raises(bad, match="not x"):
        _CUDA.lora_add(z(4, 64), square, z(3, 8, 64), z(3, 64, 8), ids, out=square)
    with pytest.raises(bad, match="out must have"):
        _CUDA.lora_add(*ok, out=z(4, 40))
    assert _CUDA.lora_add(y[:0], x[:0], la, lb, ids[:0], None, (32, 16)).shape == (0, 48)
    # no adapters at all
    assert not _CUDA.lora_add(y, x, la[:0], lb[:0], ids, None, (32, 16)).any()
