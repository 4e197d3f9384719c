"""The C++ host side of the q/k norm, int8 cache and grouped-linear ops against
the Python ops that they stand before: the same results for calls that they take,
None for all others."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv_i8 import Cache, _starts

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


class _NoHost:
    def __getattr__(self, name):
        return lambda *a: None


def _f16(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float16)).to(DEV)


def _setup():
    rng = np.random.default_rng(0)
    t = dict(c=Cache(rng, [40, 7, 300], 2, 16), idx=torch.from_numpy(_starts([3, 1, 20])).to(DEV),
             qkv=_f16(rng, 24, 8 * D), w=_f16(rng, D), cs=_f16(rng, 24, D), sn=_f16(rng, 24, D))
    t["heads"] = t["qkv"].view(24, 8, D)
    t["codes"] = torch.randint(0, 256, (48, 128), dtype=torch.uint8, device=DEV)
    t["s"], t["z"] = _f16(rng, 48, 4), torch.randint(0, 16, (48, 4), dtype=torch.uint8, device=DEV)
    t["x"], t["bias"] = _f16(rng, 2, 3, 256), _f16(rng, 48)
    return t


def _calls(t):
    """(op, arguments, outputs) of each; caches are written in place."""
    c, h = t["c"].args(), t["heads"]
    nr = (h[None, :, :4], h[None, :, 4:6], t["cs"][None], t["sn"][None])
    yield "qk_norm_rope", (*nr, t["w"], None, 1e-6)
    yield "qk_norm_rope", (*nr, None, None, None)
    yield "append_kv_i8", (*c, h[:, 4:6], h[:, 6:], t["idx"], 20)
    yield "append_kv_i8", (*c, h[:3, 4:6], h[:3, 6:], None, None)
    yield "qkv_norm_rope_append_i8", (*c, t["qkv"], t["cs"], t["sn"], 4, t["w"], t["w"], 1e-5,
                                      t["idx"], None)
    yield "qkv_norm_rope_append_i8", (*c, t["qkv"][:3], t["cs"][:1], t["sn"][:1], 4, None, None,
                                      None, None, None)
    q, o = h[:, :4].contiguous(), torch.zeros(24, 4, D, dtype=torch.float16, device=DEV)
    yield "batch_attention_i8", (o, q, *c, t["idx"], 20, None, None)
    yield "batch_attention_i8", (o[:3], q[:3], *c, None, None, 300, 0.25)
    yield "w4a16_linear", (t["x"], t["codes"], t["s"], t["z"], t["bias"])
    yield "w4a16_linear", (t["x"], t["codes"], t["s"], None, None)


def _outputs(t, out):
    out = out if isinstance(out, tuple) else (out,)
    return [x.clone() for x in out if isinstance(x, torch.Tensor)] + \
        [x.clone() for x in t["c"].dev[:2]]


def test_same_results_as_the_python_ops(monkeypatch):
    from signrot_amd import _CUDA
    t = _setup()
    host = _CUDA._host
    for name, args in _calls(t):
        assert getattr(host, name)(*args) is not None, name
    for i in range(10):
        got = []
        for use in (host, _NoHost()):
            t["c"].upload()
            name, args = list(_calls(t))[i]
            monkeypatch.setattr(_CUDA, "_host", use)
            out = getattr(_CUDA, name)(*args)
            got.append(_outputs(t, out))
        for a, b in zip(*got):
            assert torch.equal(a, b), name
        assert len(got[0]) == len(got[1])


def test_other_calls_are_handed_on():
    from signrot_amd import _CUDA
    host, t = _CUDA._host, _setup()
    c, h = t["c"].args(), t["heads"]
    q, k, cs, sn = h[None, :, :4], h[None, :, 4:6], t["cs"][None], t["sn"][None]
    assert host.qk_norm_rope(q, k, cs, sn, None, None, 1e-6) is not None
    for args in ((q.float(), k, cs, sn, None, None, 1e-6), (q, k, cs[:, :2], sn, None, None, 1e-6),
                 (q, k, cs, sn, t["w"][:64], None, 1e-6), (q, k, cs, sn, t["w"], None, None),
                 (q, k, cs, sn, None, None, "x"), (q.cpu(), k, cs, sn, None, None, 1e-6),
                 (q, k[:, :, :0], cs, sn, None, None, 1e-6), (q, k, cs, sn, None, None),
                 (q, k, cs, sn, None, None, -1.0)):
        assert host.qk_norm_rope(*args) is None
    k, v = h[:3, 4:6], h[:3, 6:]
    for args in ((c[0].view(torch.uint8), *c[1:], k, v, None, None), (*c[:5], 2, k, v, None, None),
                 (*c, k[:2], v[:2], None, None), (*c, k, v, t["idx"].long(), None),
                 (*c, k, v, None, 1.0, 2)):
        assert host.append_kv_i8(*args) is None
    o = torch.zeros(3, 4, D, dtype=torch.float16, device=DEV)
    for args in ((o, o[:, :3].contiguous(), *c), (o.float(), o, *c), (o[:2], o[:2], *c)):
        assert host.batch_attention_i8(*args, None, None, None, None) is None
    assert host.batch_attention_i8(o, o, *c, None, None, None, float("nan")) is None
    for args in ((t["x"].float(), t["codes"], t["s"]), (t["x"], t["codes"][:, :64], t["s"]),
                 (t["x"], t["codes"], t["s"][:, :3].contiguous())):
        assert host.w4a16_linear(*args, None, None) is None
