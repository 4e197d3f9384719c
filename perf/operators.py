"""Measured cases of the operators that serve models with query / key norms, an
8-bit KV cache and weights quantized by groups, each in its plain form (elementary
torch operations) and through the framework's entry points.

Kinds of case, and what each stands for in use:

  norm_rope    per-head RMSNorm of queries and keys with the rotary embedding,
               from the strided q/k columns of a fused projection output
  append       new keys and values (fp16) into the paged int8 cache, which holds
               one scale for each block of 16 tokens and head: the open block of a
               request takes the new maximum and its older codes follow
  qkv_append   both in one pass over the projection output, as a layer calls them:
               queries come back, keys and values go into the cache
  attention    attention over that cache: one query token per request (decode), or
               the last n tokens of each request (a prompt's next piece), causal
  linear       a few tokens through a linear of 4-bit weights with a scale (and a
               zero point) for each group of input columns

Head counts (32/8, 64/8, 32/32), hidden and FFN widths (4096, 8192, 14336, 28672,
11008) are those of the benchmark's configurations and of the tests; requests have
uneven lengths.  A pass rewrites the same cache slots, so it can be repeated.
"""
import math

import torch

own = False

DEV = "cuda"
D = 128          # head dim of the cache
BLOCK = 16       # tokens that share a scale
EPS = 1e-6
THETA = 500000.0


def listed():
    return [
        # a decode batch of 32 tokens: the smallest call, launches count
        dict(name="norm_rope_b32", kind="norm_rope", batch=32, tokens=1, heads=32, kv_heads=8,
             dim=128, gamma=True),
        # a prompt of 2048 tokens, 64 / 8 heads
        dict(name="norm_rope_t2048", kind="norm_rope", batch=1, tokens=2048, heads=64, kv_heads=8,
             dim=128, gamma=True),
        # one new token for each of 32 short requests, most blocks open
        dict(name="append_b32", kind="append", batch=32, context=40, new=1, kv_heads=8, page=16),
        # uneven prompts that go on behind a cached prefix which ends inside a block
        dict(name="append_t2000", kind="append", batch=4, context=101, new=2000, kv_heads=8,
             page=256),
        # the layer's step between projection and attention: a decode batch of 16
        dict(name="qkv_append_b16", kind="qkv_append", batch=16, context=45, new=1, heads=32,
             kv_heads=8, page=16),
        # and a prompt of 2048 tokens
        dict(name="qkv_append_t2048", kind="qkv_append", batch=1, context=0, new=2048, heads=32,
             kv_heads=8, page=256),
        # decode of one short request: latency
        dict(name="attention_b1_t300", kind="attention", batch=1, context=299, new=1, heads=32,
             kv_heads=8, page=64),
        # a decode batch with up to 4096 cached tokens each
        dict(name="attention_b32_t4096", kind="attention", batch=32, context=4095, new=1, heads=32,
             kv_heads=8, page=64),
        # two long documents, 64 query heads
        dict(name="attention_b2_t60000", kind="attention", batch=2, context=60000, new=1, heads=64,
             kv_heads=8, page=256),
        # pieces of up to 512 prompt tokens behind up to 5000 cached ones
        dict(name="attention_b4_new512", kind="attention", batch=4, context=5000, new=512, heads=32,
             kv_heads=8, page=64),
        # one token through a projection of 4096 x 4096
        dict(name="linear_m1_4096", kind="linear", m=1, k=4096, n=4096, group=128, asym=False),
        # a decode batch through a down_proj of 28672 columns, with zero points
        dict(name="linear_m16_28672", kind="linear", m=16, k=28672, n=8192, group=128, asym=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "qkv_append", "attention", "attention", "attention",
                       "linear", "linear"])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (32, 32), (40, 8)])
    if kind == "norm_rope":
        dim = rng.choice([64, 128, 128, 256])
        most = 2048 * 72 * 128 // ((heads + kv_heads) * dim)
        tokens = _log_int(rng, 1, most)
        return dict(kind=kind, batch=_log_int(rng, 1, min(64, most // tokens)), tokens=tokens,
                    heads=heads, kv_heads=kv_heads, dim=dim, gamma=rng.random() < 0.8)
    if kind in ("append", "qkv_append"):
        # the cache's values come back, so its pages count as work too
        page, context = rng.choice([16, 64, 256]), rng.randrange(0, 200)
        most = 6000 * 8 // kv_heads if kind == "append" else 2000 * 32 // (heads + 2 * kv_heads)
        new = rng.choice([1, _log_int(rng, 2, most - context - page)])
        case = dict(kind=kind, batch=_log_int(rng, 1, min(64, most // (context + new + page))),
                    context=context, new=new, kv_heads=kv_heads, page=page)
        return case if kind == "append" else dict(case, heads=heads)
    if kind == "attention":
        new = rng.choice([1, 1, 1, _log_int(rng, 2, 8), _log_int(rng, 16, 512)])
        context = _log_int(rng, 1, 5000 if new > 8 else 60000 * 8 // kv_heads)
        most = 100000 * 8 // kv_heads // (context + new)
        if new > 8:
            most = min(most, 4 * 32 // heads)
        return dict(kind=kind, batch=_log_int(rng, 1, max(1, min(48, most))), context=context,
                    new=new, heads=heads, kv_heads=kv_heads, page=rng.choice([16, 64, 256]))
    k, n = rng.choice([(4096, 4096), (4096, 28672), (14336, 4096), (11008, 4096), (8192, 8192),
                       (28672, 8192), (1000 * 32, 1111)])
    return dict(kind=kind, m=_log_int(rng, 1, 16), k=k, n=n, asym=rng.random() < 0.5,
                group=rng.choice([64, 128] if k == 28672 else [32, 64, 128]))


# ----------------------------------------------------------------- inputs

def _lengths(case):
    """(cached tokens, new tokens) of each request: uneven, by the case alone."""
    b, c, n = case["batch"], case["context"], case["new"]
    return [(c - c * i // (2 * b), n - n * i // (2 * b)) for i in range(b)]


def _tables(case, g):
    """The page table of the batch, with every request's new tokens counted in."""
    lens, page = _lengths(case), case["page"]
    pages = [-(-(c + n) // page) for c, n in lens]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    def starts(v):
        return ints([sum(v[:i]) for i in range(len(v) + 1)])

    touched = [(i, j) for i, (c, n) in enumerate(lens)
               for j in range(c // BLOCK, -(-(c + n) // BLOCK))]
    return dict(request=ints([i for i, (_, n) in enumerate(lens) for _ in range(n)]).long(),
                turn=ints([i for _, n in lens for i in range(n)]).long(),
                touched=ints(touched).long(), indptr=starts(pages),
                last=ints([(c + n - 1) % page + 1 for c, n in lens]),
                indices=torch.randperm(sum(pages), device=DEV, generator=g).int(),
                new_indptr=None if case["new"] == 1 else starts([n for _, n in lens]),
                total=sum(pages), tokens=sum(n for _, n in lens),
                longest=max(c + n for c, n in lens))


def _pool(g, pages, kv_heads, page):
    """A cache of one layer whose pages hold the codes of N(0, 1) values with
    scales that differ from block to block."""
    shape = (pages, 1, 2, kv_heads, page, D)
    data = torch.empty(shape, dtype=torch.int8, device=DEV)
    for p in range(0, pages, 256):   # in pieces: the normal values take 4 bytes each
        part = data[p: p + 256]
        x = torch.randn(part.shape, device=DEV, generator=g)
        part.copy_((x * 36).round_().clamp_(-127, 127))
    scale = torch.rand(shape[:4] + (page // BLOCK,), device=DEV, generator=g) * 0.02 + 0.018
    return data, scale


def _rope(positions, dim):
    inv = THETA ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
    ang = positions.double()[:, None] * inv[None, :]
    ang = torch.cat((ang, ang), dim=-1)
    return ang.cos().half(), ang.sin().half()


def _positions(case):
    return torch.cat([torch.arange(c, c + n, device=DEV) for c, n in _lengths(case)])


def _gamma(g, dim):
    return (1 + 0.2 * torch.randn(dim, device=DEV, generator=g)).half()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    kind = case["kind"]
    s = dict(kind=kind, case=case)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if kind == "norm_rope":
        b, t, hq, hk, d = (case[x] for x in ("batch", "tokens", "heads", "kv_heads",
                                               "dim"))
        qkv = (2 * normal(b, t, hq + 2 * hk, d)).half()
        cos, sin = _rope(torch.arange(17, 17 + t, device=DEV), d)
        s.update(q=qkv[:, :, :hq], k=qkv[:, :, hq: hq + hk], cos=cos[None], sin=sin[None],
                 qw=_gamma(g, d) if case["gamma"] else None,
                 kw=_gamma(g, d) if case["gamma"] else None)
        return s
    if kind == "linear":
        m, k, n, grp = case["m"], case["k"], case["n"], case["group"]
        c = (normal(n, k) * 1.75).round_().clamp_(-8, 7).to(torch.int8)
        s["x"] = normal(m, k).half()
        if case["asym"]:
            c = c + 8
            s["zeros"] = torch.randint(6, 11, (n, k // grp), dtype=torch.uint8, device=DEV,
                                       generator=g)
        else:
            s["zeros"] = None
        c = c.view(torch.uint8) & 15
        s["w"] = c[:, 0::2] | (c[:, 1::2] << 4)
        s["scales"] = ((torch.rand(n, k // grp, device=DEV, generator=g) * 0.4 + 0.8)
                       * (0.02 / 1.75)).half()
        return s
    s.update(_tables(case, g))
    s["max_new"] = case["new"]
    s["data"], s["scale"] = _pool(g, s["total"], case["kv_heads"], case["page"])
    n = s["tokens"]
    if kind == "append":
        s["k"], s["v"] = (normal(n, case["kv_heads"], D).half() for _ in range(2))
    elif kind == "qkv_append":
        s["qkv"] = normal(n, (case["heads"] + 2 * case["kv_heads"]) * D).half()
        s["cos"], s["sin"] = _rope(_positions(case), D)
        s["qw"], s["kw"] = _gamma(g, D), _gamma(g, D)
    else:
        s["q"] = (1.5 * normal(n, case["heads"], D)).half()
        s["o"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------------ plain forms

def _norm_rope_plain(x, w, cos, sin):
    """x [..., D] fp16; cos / sin broadcast against it."""
    f = x.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    if w is not None:
        y = y * w.float()
    half = x.shape[-1] // 2
    turned = torch.cat((-y[..., half:], y[..., :half]), dim=-1)
    return (y * cos.float() + turned * sin.float()).half()


def _grid(s):
    """Lengths, first new row and new tokens by request; pages by (request, page)."""
    first = s["indptr"][:-1].long()
    count = s["indptr"][1:].long() - first
    page = s["case"]["page"]
    lens = (count - 1) * page + s["last"].long()
    if s["new_indptr"] is None:
        start = torch.arange(len(lens), device=DEV)
        new = torch.ones_like(start)
    else:
        start = s["new_indptr"][:-1].long()
        new = s["new_indptr"][1:].long() - start
    most = -(-s["longest"] // page)
    at = torch.arange(most, device=DEV)[None, :]
    slot = (first[:, None] + at).clamp(max=len(s["indices"]) - 1)
    pages = s["indices"].long()[slot]
    return lens, start, new, torch.where(at < count[:, None], pages, 0)


def _append_plain(s, k, v):
    """k, v [N, H, D] fp16 into the cache, the touched blocks all at once."""
    page = s["case"]["page"]
    lens, start, new, pages = _grid(s)
    old = lens - new
    b_at, blk = s["touched"].unbind(1)
    tok = blk[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)            # [n, 16]
    held = tok < old[b_at, None]
    fresh = ~held & (tok < lens[b_at, None])
    src = (start[b_at, None] + tok - old[b_at, None]).clamp(0, k.shape[0] - 1)
    pg = pages[b_at, blk * BLOCK // page]
    e0 = blk * BLOCK % page
    rows = e0[:, None] + torch.arange(BLOCK, device=DEV)
    data, scale = s["data"][:, 0], s["scale"][:, 0]                         # [P, 2, H, page, D]
    x = torch.stack((k, v), 1)[src].float()                                 # [n, 16, 2, H, D]
    x = torch.where(fresh[:, :, None, None, None], x, 0.0).permute(0, 2, 3, 1, 4)
    was = torch.where(held[:, :1, None], scale[pg, :, :, e0 // BLOCK], 0.0)  # [n, 2, H]
    now = torch.maximum(was, x.abs().amax((3, 4)) / 127)
    codes = data[pg[:, None], :, :, rows].permute(0, 2, 3, 1, 4)            # [n, 2, H, 16, D]
    div = torch.where(now > 0, now, 1.0).double()[..., None, None]
    moved = (codes.double() * was.double()[..., None, None] / div).round().clamp(-127, 127)
    put = (x.double() / div).round().clamp(-127, 127)
    fresh, held = fresh[:, None, None, :, None], held[:, None, None, :, None]
    out = torch.where(fresh, put.to(torch.int8), torch.where(held, moved.to(torch.int8), codes))
    data[pg[:, None], :, :, rows] = out.permute(0, 3, 1, 2, 4)
    scale[pg, :, :, e0 // BLOCK] = now


def _attention_plain(s):
    case = s["case"]
    hq, hk, page = case["heads"], case["kv_heads"], case["page"]
    lens, start, new, pages = _grid(s)
    b, t = len(lens), s["max_new"]
    kv = s["data"][:, 0][pages].float()                                     # [B, P, 2, H, page, D]
    kv = kv.unflatten(4, (page // BLOCK, BLOCK)) * s["scale"][:, 0][pages][..., None, None]
    kv = kv.flatten(4, 5).permute(2, 0, 3, 1, 4, 5).reshape(2, b, hk, -1, D)
    i = torch.arange(t, device=DEV)[None, :]
    q = s["q"][(start[:, None] + i).clamp(max=s["q"].shape[0] - 1)].float()  # [B, T, Hq, D]
    q = q.view(b, t, hk, hq // hk, D).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, D)
    x = torch.matmul(q, kv[0].transpose(-1, -2).contiguous()) / math.sqrt(D)
    pos = (lens - new)[:, None] + i                                         # [B, T]
    seen = torch.arange(x.shape[-1], device=DEV) <= pos[:, :, None]         # [B, T, L]
    x = x.view(b, hk, hq // hk, t, -1).masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hk, -1, x.shape[-1]), kv[1])
    o = o.view(b, hk, hq // hk, t, D).permute(0, 3, 1, 2, 4).reshape(b, t, hq, D)
    return o[s["request"], s["turn"]].half()


def _linear_plain(s):
    n, k = s["w"].shape[0], s["w"].shape[1] * 2
    c = torch.stack((s["w"] & 15, s["w"] >> 4), -1).view(n, k).float()
    if s["zeros"] is None:
        c = c - 16 * (c >= 8)
    c = c.view(n, -1, s["case"]["group"])
    if s["zeros"] is not None:
        c = c - s["zeros"].float()[..., None]
    w = (c * s["scales"].float()[..., None]).view(n, k)
    return torch.matmul(s["x"].float(), w.t()).half()


# -------------------------------------------------------------------- run

def _values(s):
    """What the cache holds now, as the numbers that the codes stand for."""
    codes = s["data"].unflatten(4, (-1, BLOCK))
    out = torch.empty(codes.shape, dtype=torch.float16, device=codes.device)
    return torch.mul(codes, s["scale"][..., None, None], out=out)


@torch.no_grad()
def run(s):
    kind = s["kind"]
    if own:
        return _run_own(s)
    if kind == "norm_rope":
        cos, sin = s["cos"][:, :, None], s["sin"][:, :, None]
        return (_norm_rope_plain(s["q"], s["qw"], cos, sin),
                _norm_rope_plain(s["k"], s["kw"], cos, sin))
    if kind == "append":
        _append_plain(s, s["k"], s["v"])
        return dict(cache=_values(s), scale=s["scale"])
    if kind == "qkv_append":
        hq, hk = s["case"]["heads"], s["case"]["kv_heads"]
        q, k, v = s["qkv"].view(-1, hq + 2 * hk, D).split((hq, hk, hk), dim=1)
        cos, sin = s["cos"][:, None], s["sin"][:, None]
        q, k = _norm_rope_plain(q, s["qw"], cos, sin), _norm_rope_plain(k, s["kw"], cos, sin)
        _append_plain(s, k, v)
        return dict(q=q, cache=_values(s))
    if kind == "attention":
        return _attention_plain(s)
    return _linear_plain(s)


def _run_own(s):
    from signrot_amd import _CUDA
    kind = s["kind"]
    if kind == "norm_rope":
        return _CUDA.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["qw"], s["kw"], EPS)
    if kind == "linear":
        return _CUDA.w4a16_linear(s["x"], s["w"], s["scales"], s["zeros"])
    cache = (s["data"], s["scale"], s["indptr"], s["indices"], s["last"], 0)
    if kind == "append":
        _CUDA.append_kv_i8(*cache, s["k"], s["v"], s["new_indptr"], s["max_new"])
        return dict(cache=_values(s), scale=s["scale"])
    if kind == "qkv_append":
        q = _CUDA.qkv_norm_rope_append_i8(*cache, s["qkv"], s["cos"], s["sin"], s["case"]["heads"],
                                          s["qw"], s["kw"], EPS, s["new_indptr"], s["max_new"])
        return dict(q=q, cache=_values(s))
    _CUDA.batch_attention_i8(s["o"], s["q"], *cache, s["new_indptr"], s["max_new"], s["longest"])
    return s["o"]


# ------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "norm_rope":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return dict(bytes=4 * n + 4 * case["tokens"] * case["dim"], flops=8 * n)
    if kind == "linear":
        m, k, n, grp = case["m"], case["k"], case["n"], case["group"]
        return dict(bytes=n * k // 2 + n * k // grp * (3 if case["asym"] else 2)
                    + 2 * m * k + 2 * m * n, flops=2 * m * n * k)
    lens, hk, page = _lengths(case), case["kv_heads"], case["page"]
    new = sum(n for _, n in lens)
    if kind == "attention":
        hq = case["heads"]
        cached = sum(c + n for c, n in lens)
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in lens)
        return dict(bytes=cached * hk * 2 * (D + 4 / BLOCK) + 4 * new * hq * D,
                    flops=4 * pairs * hq * D)
    # new keys and values in, codes out, the open blocks' codes in and out, and
    # the values that the pages stand for
    held = sum(-(-(c + n) // page) for c, n in lens) * page * hk * 2 * D
    opened = sum(c % BLOCK for c, _ in lens)
    size = hk * 2 * D * (3 * new + 2 * opened) + 3 * held
    flops = hk * 2 * D * 4 * new
    if kind == "qkv_append":
        size += 4 * new * case["heads"] * D + 4 * new * D
        flops += 8 * new * (case["heads"] + hk) * D
    return dict(bytes=size, flops=flops)


# ------------------------------------------------------------------ exact

def _norm_rope_exact(x, w, cos, sin):
    x, cos, sin = x.double(), cos.double(), sin.double()
    y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    y = y if w is None else y * w.double()
    a, b = y.chunk(2, -1)
    (ca, cb), (sa, sb) = cos.chunk(2, -1), sin.chunk(2, -1)
    return torch.cat((a * ca - b * sa, b * cb + a * sb), -1)


def _requests(s):
    """For each request: its pages, cached and new tokens, and where those start."""
    at, ptr = 0, s["indptr"].tolist()
    for b, (c, n) in enumerate(_lengths(s["case"])):
        yield s["indices"][ptr[b]: ptr[b + 1]].long(), c, n, at
        at += n


def _cache_exact(s, k, v):
    """The cache's values (64 bits) and scales after the append: by the definition,
    a block's scale is the 32-bit quotient of its largest new magnitude and 127, or
    the one that it had where that is larger; codes are rounded to nearest."""
    page, heads = s["case"]["page"], s["case"]["kv_heads"]
    values = _pool_values(s)
    scales = s["scale"].clone()
    for pages, c, n, at in _requests(s):
        seq = values[pages, 0].transpose(0, 2).transpose(0, 1).reshape(2, heads, -1, D)
        sc = scales[pages, 0].transpose(0, 2).transpose(0, 1).reshape(2, heads, -1)
        for j in range(c // BLOCK, -(-(c + n) // BLOCK)):
            lo, hi = max(c, j * BLOCK), min(c + n, (j + 1) * BLOCK)
            rows = torch.stack((k, v))[:, at + lo - c: at + hi - c].double().transpose(1, 2)
            top = (rows.abs().amax((2, 3)).float() / 127).float()
            was = sc[:, :, j] if lo > j * BLOCK else torch.zeros_like(top)
            now = torch.maximum(top, was)
            unit = torch.where(now == 0, torch.ones_like(now), now).double()[:, :, None, None]
            if lo > j * BLOCK:
                kept = seq[:, :, j * BLOCK: lo]
                seq[:, :, j * BLOCK: lo] = torch.round(kept / unit) * unit
            seq[:, :, lo:hi] = torch.round(rows / unit) * unit
            # rows behind the last token keep their codes, and so stand for other numbers
            rest = seq[:, :, hi: (j + 1) * BLOCK]
            old = sc[:, :, j].double()[:, :, None, None]
            seq[:, :, hi: (j + 1) * BLOCK] = torch.round(rest / old) * unit
            sc[:, :, j] = now
        values[pages, 0] = seq.reshape(2, heads, -1, page, D).permute(2, 0, 1, 3, 4)
        scales[pages, 0] = sc.reshape(2, heads, -1, page // BLOCK).permute(2, 0, 1, 3)
    return values.unflatten(4, (-1, BLOCK)), scales.double()


def _pool_values(s):
    scale = s["scale"].double().repeat_interleave(BLOCK, -1)
    return s["data"].double() * scale[..., None]


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm_rope":
        cos, sin = s["cos"].unsqueeze(2), s["sin"].unsqueeze(2)
        return (_norm_rope_exact(s["q"], s["qw"], cos, sin),
                _norm_rope_exact(s["k"], s["kw"], cos, sin))
    if kind == "append":
        values, scales = _cache_exact(s, s["k"], s["v"])
        return dict(cache=values, scale=scales)
    if kind == "qkv_append":
        hq, hk = case["heads"], case["kv_heads"]
        x = s["qkv"].view(-1, hq + 2 * hk, D)
        cos, sin = s["cos"].unsqueeze(1), s["sin"].unsqueeze(1)
        q = _norm_rope_exact(x[:, :hq], s["qw"], cos, sin)
        # keys are fp16 where they reach the cache
        k = _norm_rope_exact(x[:, hq: hq + hk], s["kw"], cos, sin).half()
        return dict(q=q, cache=_cache_exact(s, k, x[:, hq + hk:])[0])
    if kind == "attention":
        hq, hk = case["heads"], case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for pages, c, n, at in _requests(s):
            scale = s["scale"][pages, 0].double().repeat_interleave(BLOCK, -1)
            kv = s["data"][pages, 0].double() * scale[..., None]
            for h in range(hq):
                k, v = (kv[:, i, h // (hq // hk)].reshape(-1, D)[: c + n] for i in (0, 1))
                x = s["q"][at: at + n, h].double() @ k.t() / math.sqrt(D)
                late = torch.arange(c + n, device=DEV)[None] > torch.arange(c, c + n,
                                                                            device=DEV)[:, None]
                out[at: at + n, h] = torch.softmax(x.masked_fill(late, -math.inf), -1) @ v
        return out
    n, k = case["n"], case["k"]
    w = torch.empty(n, k, dtype=torch.float64, device=DEV)
    w[:, 0::2] = (s["w"] % 16).double()
    w[:, 1::2] = torch.div(s["w"], 16, rounding_mode="floor").double()
    if s["zeros"] is None:
        w = torch.where(w > 7, w - 16, w)
    else:
        w = w - s["zeros"].double().repeat_interleave(case["group"], 1)
    w = w * s["scales"].double().repeat_interleave(case["group"], 1)
    return s["x"].double() @ w.t()
