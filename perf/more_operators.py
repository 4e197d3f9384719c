"""Measured cases of the operators that serve 4-bit weights with 8-bit activations
and with many requests' low-rank adapters, each in its plain form (elementary torch
operations) and through the framework's entry points.

Kinds of case, and what each stands for in use:

  norm     what stands before a projection: the residual's addition, the RMSNorm and
           the quantization of its rows to int8 with a scale per token
  quant    the quantization alone, of rows that no norm precedes (the inputs of the
           attention's output projection and of down_proj)
  linear   int8 rows through packed int4 weights with a scale per output channel,
           with a bias or the residual added
  lora     the low-rank adapters of a batch's requests, added beside a projection
           that they share: out = y + s (x A^T) B^T with each token's own A, B and s;
           one call serves a projection that is several in one (q/k/v, gate/up)

Widths (4096, 8192, 11008, 14336, 28672) and head counts (32/8, 64/8) are those of
the benchmark's configurations and of the tests; requests have uneven lengths.
"""
import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5


def listed():
    return [
        # one token of one request: launches count
        dict(name="norm_r1_4096", kind="norm", rows=1, n=4096, residual=True, weight=False,
             keep=False),
        # a decode batch whose normalised rows the adapters read too
        dict(name="norm_r32_8192", kind="norm", rows=32, n=8192, residual=True, weight=True,
             keep=True),
        # four prompts of up to 2048 tokens
        dict(name="norm_r8190_8192", kind="norm", rows=8190, n=8192, residual=True, weight=False,
             keep=False),
        # the input of down_proj: a prompt of 2048 tokens
        dict(name="quant_r2048_14336", kind="quant", rows=2048, n=14336),
        # one token through a projection of 4096 x 4096
        dict(name="linear_m1_4096", kind="linear", m=1, k=4096, n=4096, bias=False,
             residual=False),
        # a decode batch through a down_proj of 28672 columns
        dict(name="linear_m16_28672", kind="linear", m=16, k=28672, n=8192, bias=False,
             residual=True),
        # a short prompt of odd length
        dict(name="linear_m101_4096", kind="linear", m=101, k=4096, n=14336, bias=True,
             residual=False),
        # a prompt of 2048 tokens through gate/up
        dict(name="linear_m2048_28672", kind="linear", m=2048, k=4096, n=28672, bias=False,
             residual=False),
        # one token of one request with an adapter
        dict(name="lora_b1", kind="lora", requests=1, tokens=1, adapters=4, rank=16, k=4096,
             slices="4096"),
        # a decode batch of 32 requests with adapters of their own (some without): q/k/v
        dict(name="lora_b32", kind="lora", requests=32, tokens=1, adapters=32, rank=16, k=4096,
             slices="4096+1024+1024"),
        # short prompts of 12 requests that share 5 adapters: gate/up
        dict(name="lora_b12_t60", kind="lora", requests=12, tokens=60, adapters=5, rank=32, k=4096,
             slices="14336+14336"),
        # four prompts of up to 1500 tokens, adapters of rank 64: q/k/v of 64 / 8 heads
        dict(name="lora_b4_t1500", kind="lora", requests=4, tokens=1500, adapters=4, rank=64,
             k=8192, slices="8192+1024+1024"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quant", "linear", "linear", "linear", "lora", "lora",
                       "lora"])
    if kind in ("norm", "quant"):
        n = rng.choice([4096, 5120, 8192, 8192, 14336, 11008, 1000, 2047, 28672])
        rows = _log_int(rng, 1, 8000 * 8192 // max(n, 4096))
        if kind == "quant":
            return dict(kind=kind, rows=rows, n=n)
        return dict(kind=kind, rows=rows, n=n, residual=rng.random() < 0.7,
                    weight=rng.random() < 0.5, keep=rng.random() < 0.3)
    if kind == "linear":
        k, n = rng.choice([(4096, 4096), (4096, 6144), (4096, 28672), (14336, 4096), (11008, 4096),
                           (8192, 8192), (28672, 8192), (1000 * 32, 1111), (5120, 5125)])
        most = min(2048, 2048 * 4096 * 28672 // (k * n))
        return dict(kind=kind, m=_log_int(rng, 1, most), k=k, n=n, bias=rng.random() < 0.3,
                    residual=rng.random() < 0.4)
    k, slices = rng.choice([(4096, "4096"), (4096, "4096+1024+1024"), (4096, "14336+14336"),
                            (14336, "4096"), (8192, "8192+1024+1024"), (5120, "5125"),
                            (8192, "8192"), (1000, "1111+77")])
    rank = rng.choice([8, 16, 16, 32, 64])
    width = k + 2 * sum(int(v) for v in slices.split("+"))
    most = 4000 * 28000 // max(width, 8000)
    tokens = rng.choice([1, 1, _log_int(rng, 2, most)])
    requests = _log_int(rng, 1, min(64, most // tokens))
    return dict(kind=kind, requests=requests, tokens=tokens, adapters=rng.randint(1, 32),
                rank=rank, k=k, slices=slices)


# ----------------------------------------------------------------- inputs

def _slices(case):
    return [int(v) for v in case["slices"].split("+")]


def _lora_lengths(case):
    """Tokens of each request: uneven, by the case alone."""
    b, n = case["requests"], case["tokens"]
    return [n - n * i // (2 * b) for i in range(b)]


def _lora_place(case, i):
    """Which of the batch's adapters request i has, or -1: every eighth has none."""
    return -1 if i % 8 == 7 else i % case["adapters"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    kind = case["kind"]
    s = dict(kind=kind, case=case)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    def outliers(rows, n):
        """Activations: a few channels are far larger than the others."""
        x = normal(rows, n)
        x[:, torch.randperm(n, device=DEV, generator=g)[:4]] *= 20
        return x.half()

    if kind in ("norm", "quant"):
        rows, n = case["rows"], case["n"]
        s["x"] = outliers(rows, n)
        # what the 8-bit rows stand for, to give them back
        s["values"] = torch.empty(rows, n, dtype=torch.float16, device=DEV)
        if kind == "norm":
            s["residual"] = (4 * normal(rows, n)).half() if case["residual"] else None
            s["weight"] = (1 + 0.2 * normal(n)).half() if case["weight"] else None
        return s
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["a"] = (normal(m, k) * 30).round_().clamp_(-127, 127).to(torch.int8)
        s["sa"] = torch.rand(m, 1, device=DEV, generator=g) * 0.03 + 0.01
        c = (normal(n, k) * 2.2).round_().clamp_(-8, 7).to(torch.int8)
        c = c.view(torch.uint8) & 15
        s["w"] = c[:, 0::2] | (c[:, 1::2] << 4)
        s["sw"] = ((torch.rand(n, device=DEV, generator=g) * 0.4 + 0.8) * (0.02 / 2.2)).half()
        s["bias"] = normal(n).half() if case["bias"] else None
        s["residual"] = (4 * normal(m, n)).half() if case["residual"] else None
        return s
    lens, k, rank, out = _lora_lengths(case), case["k"], case["rank"], _slices(case)
    tokens, count = sum(lens), case["adapters"]
    order = list(range(count))
    random.Random(int(seed)).shuffle(order)
    ids = [-1 if _lora_place(case, i) < 0 else order[_lora_place(case, i)]
           for i in range(len(lens))]
    per_token = [a for a, n in zip(ids, lens) for _ in range(n)]
    s["slices"], s["rank"] = tuple(out), rank
    s["ids"] = torch.tensor(per_token, dtype=torch.int32, device=DEV)
    # the rows of each adapter, as a program without grouped kernels keeps them
    s["rows"] = [(a, torch.tensor([i for i, v in enumerate(per_token) if v == a], device=DEV))
                 for a in sorted(set(per_token)) if a >= 0]
    s["x"] = normal(tokens, k).half()
    s["y"] = normal(tokens, sum(out)).half()
    s["a"] = (normal(count, len(out) * rank, k) / math.sqrt(k)).half()
    s["b"] = (normal(count, sum(out), rank) * 0.2 / math.sqrt(rank)).half()
    s["scaling"] = torch.rand(count, device=DEV, generator=g) + 0.5
    return s


# ------------------------------------------------------------ plain forms

def _quant_plain(y):
    """Codes (as whole numbers in 64 bits) and fp32 scales of the rows y, fp64: the
    codes are decided in 64 bits, since many quotients lie next to a border."""
    scale = (y.abs().amax(-1, keepdim=True) / 127).float()
    unit = torch.where(scale > 0, scale, 1.0).double()
    return (y / unit).round_().clamp_(-127, 127), scale


def _values(codes, scale, out):
    """What codes and scales stand for, as fp16."""
    return torch.mul(codes, scale, out=out)


def _norm_plain(s):
    x = s["x"]
    out = {}
    if s["residual"] is not None:
        x = out["sum"] = (x.float() + s["residual"].float()).half()
    y = x.double()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    if s["weight"] is not None:
        y = y * s["weight"].double()
    if s["case"]["keep"]:
        out["norm"] = y.half()
    codes, scale = _quant_plain(y)
    return dict(out, scale=scale, values=_values(codes.float(), scale, s["values"]))


def _linear_plain(s):
    n, k = s["w"].shape[0], s["w"].shape[1] * 2
    c = torch.stack((s["w"] & 15, s["w"] >> 4), -1).view(n, k).float()
    c = c - 16 * (c >= 8)
    out = torch.matmul(s["a"].float(), c.t()) * s["sa"] * s["sw"].float()
    if s["bias"] is not None:
        out = out + s["bias"].float()
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.half()


def _lora_plain(s):
    out, r = s["y"].float(), s["rank"]
    if s["case"]["tokens"] == 1:   # every token its own adapter: all of them at once
        i = s["ids"].clamp(min=0).long()
        t = torch.matmul(s["a"][i].float(), s["x"].float().unsqueeze(-1))
        t = t * torch.where(s["ids"] < 0, 0.0, s["scaling"][i])[:, None, None]
        at = 0
        for j, n in enumerate(s["slices"]):
            part = t[:, j * r: (j + 1) * r].contiguous()
            out[:, at: at + n] += torch.matmul(s["b"][i, at: at + n].float(), part).squeeze(-1)
            at += n
        return out.half()
    for a, rows in s["rows"]:
        t = torch.matmul(s["x"][rows].float(), s["a"][a].float().t()) * s["scaling"][a]
        at = 0
        for i, n in enumerate(s["slices"]):
            b = s["b"][a, at: at + n].float()
            out[rows, at: at + n] += torch.matmul(t[:, i * r: (i + 1) * r], b.t())
            at += n
    return out.half()


# -------------------------------------------------------------------- run

@torch.no_grad()
def run(s):
    kind = s["kind"]
    if own:
        return _run_own(s)
    if kind == "norm":
        return _norm_plain(s)
    if kind == "quant":
        codes, scale = _quant_plain(s["x"].double())
        return dict(scale=scale, values=_values(codes.float(), scale, s["values"]))
    return _linear_plain(s) if kind == "linear" else _lora_plain(s)


def _run_own(s):
    from signrot_amd import _CUDA
    kind = s["kind"]
    if kind == "norm":
        keep, added = s["case"]["keep"], s["residual"] is not None
        got = _CUDA.rmsnorm_quant_i8(s["x"], EPS, residual=s["residual"], weight=s["weight"],
                                     return_norm=keep)
        out = dict(scale=got[1], values=_values(got[0], got[1], s["values"]))
        if added:
            out["sum"] = got[2]
        if keep:
            out["norm"] = got[-1]
        return out
    if kind == "quant":
        q, scale = _CUDA.sym_quant_dynamic_i8(s["x"])
        return dict(scale=scale, values=_values(q, scale, s["values"]))
    if kind == "linear":
        return _CUDA.w4a8_linear(s["a"], s["sa"], s["w"], s["sw"], s["bias"], s["residual"])
    return _CUDA.lora_add(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scaling"], s["slices"])


# ------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind in ("norm", "quant"):
        n, rows = case["n"], case["rows"]
        # rows in, codes out; codes in and the values that they stand for out
        size = (2 + 1 + 3) * rows * n + 4 * rows
        if kind == "quant":
            return dict(bytes=size, flops=3 * rows * n)
        size += rows * n * (4 * case["residual"] + 2 * case["keep"]) + 2 * n * case["weight"]
        return dict(bytes=size, flops=6 * rows * n)
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return dict(bytes=n * k // 2 + 2 * n + m * k + 4 * m + m * n * (2 + 2 * case["residual"])
                    + 2 * n * case["bias"], flops=2 * m * n * k)
    lens, k, rank, out = _lora_lengths(case), case["k"], case["rank"], _slices(case)
    has = [n for i, n in enumerate(lens) if _lora_place(case, i) >= 0]
    used = {_lora_place(case, i) for i in range(len(lens))} - {-1}
    weights = len(used) * rank * (len(out) * k + sum(out))
    return dict(bytes=2 * weights + 2 * sum(has) * k + 4 * sum(lens) * sum(out) + 4 * sum(lens),
                flops=2 * sum(has) * rank * (len(out) * k + sum(out)))


# ------------------------------------------------------------------ exact

def _quant_exact(y):
    """Scales are fp32 numbers by definition, codes the nearest whole ones."""
    top = y.abs().max(dim=-1, keepdim=True).values
    scale = torch.div(top, 127.0).to(torch.float32).to(torch.float64)
    codes = torch.round(y / scale)
    return torch.where(scale == 0, torch.zeros_like(y), codes) * scale, scale


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quant":
        values, scale = _quant_exact(s["x"].double())
        return dict(scale=scale, values=values)
    if kind == "norm":
        x, out = s["x"].double(), {}
        if s["residual"] is not None:
            out["sum"] = x + s["residual"].double()
            # the norm reads the stream as it is stored
            x = out["sum"].half().double()
        y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
        y = y if s["weight"] is None else y * s["weight"].double()
        if case["keep"]:
            out["norm"] = y
        out["values"], out["scale"] = _quant_exact(y)
        return out
    if kind == "linear":
        n, k = case["n"], case["k"]
        w = torch.empty(n, k, dtype=torch.float64, device=DEV)
        w[:, 0::2] = (s["w"] % 16).double()
        w[:, 1::2] = torch.div(s["w"], 16, rounding_mode="floor").double()
        w = torch.where(w > 7, w - 16, w) * s["sw"].double()[:, None]
        out = (s["a"].double() * s["sa"].double()) @ w.t()
        for extra in (s["bias"], s["residual"]):
            if extra is not None:
                out = out + extra.double()
        return out
    out, ids = s["y"].double(), s["ids"].tolist()
    edges = [0]
    for n in _lora_lengths(case):
        edges.append(edges[-1] + n)
    for lo, hi in zip(edges, edges[1:]):
        a = ids[lo]
        if a < 0:
            continue
        t = s["x"][lo:hi].double() @ s["a"][a].double().t()
        at = 0
        for i, n in enumerate(s["slices"]):
            part = t[:, i * case["rank"]: (i + 1) * case["rank"]]
            out[lo:hi, at: at + n] += s["scaling"][a].double() * (
                part @ s["b"][a, at: at + n].double().t())
            at += n
    return out
