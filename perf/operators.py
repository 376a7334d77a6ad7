"""The serving operators around the quantized GEMMs: cases, plain forms and exact values.

Three operators that share one cache of 4-bit (MXFP4) keys and values in pages:

* ``tables``  block tables and slot maps from request lengths (``Library.block_tables``);
* ``qkv``     norms of queries and keys per head, position rotation and the append to the
              cache (``Library.qkv_append``), the appended rows read back as the values they
              stand for (``Library.kv_read``);
* ``attn``    attention over the cache (``Library.attention``), for single tokens and prompts.

A record of (page, key/value head) holds, for P tokens of hd dims: K codes [P][hd/2], K scales
[P][hd/32], V codes [P][hd/2], V scales [P][hd/32]; dim 2j is the low nibble of byte j, and a
scale byte b stands for 2^(b - 127).
"""
import math
import random

import torch

own = False

E_MIN, E_MAX = -23, 13          # exponents of the cache's block scales
EPS = 1e-6
MAX_POS = 1 << 15               # rows of the rotation table

# ---------------------------------------------------------------------------------------------
# cases


def _tables(name, seqs, fresh, cached, page, mixed):
    """seqs requests; one new token each, or (mixed) a quarter of them prompts of up to `fresh`."""
    return dict(name=name, op="tables", seqs=seqs, fresh=fresh, cached=cached, page=page, mixed=mixed)


def _qkv(name, tokens, heads, kv_heads, hd, page, dtype, norm, rot, axes, interleaved):
    return dict(name=name, op="qkv", tokens=tokens, heads=heads, kv_heads=kv_heads, hd=hd, page=page,
                dtype=dtype, norm=norm, rot=rot, axes=axes, interleaved=interleaved)


def _attn(name, seqs, q, kv, heads, kv_heads, hd, page, causal=True, prefix=0, window=0, cap=0.0,
          bias=False, ragged=False):
    """seqs requests with q new tokens each and kv keys (new ones included); ragged: the first
    has these, the others fewer."""
    return dict(name=name, op="attn", seqs=seqs, q=q, kv=kv, heads=heads, kv_heads=kv_heads, hd=hd,
                page=page, causal=causal, prefix=prefix, window=window, cap=cap, bias=bias,
                ragged=ragged)


def listed():
    return [
        # A few robots served together, one token each: latency alone.
        _tables("tables 8 decoding", 8, 1, 2000, 16, False),
        # A full server's step: decoding requests and prompt chunks in one batch.
        _tables("tables 1024 mixed", 1024, 512, 8000, 16, True),
        # One SmolVLA request's token (15 query heads, 5 key/value heads of 64).
        _qkv("qkv 1 token 15/5x64", 1, 15, 5, 64, 16, "f32", True, 64, 1, False),
        # The SmolVLA prefix of C3: 141 tokens (images, language, state).
        _qkv("qkv 141 tokens 15/5x64", 141, 15, 5, 64, 32, "f32", True, 64, 1, False),
        # A long video prompt: positions in time, height and width, BF16 rows, odd length.
        _qkv("qkv 16387 tokens 32/8x128", 16387, 32, 8, 128, 16, "bf16", True, 128, 3, False),
        # One robot, one token over its short history.
        _attn("decode 1x241 15/5x64", 1, 1, 241, 15, 5, 64, 16),
        # A batch of requests with histories of many lengths, the ordinary decoding step.
        _attn("decode 64x16384 32/8x128", 64, 1, 16384, 32, 8, 128, 16, ragged=True),
        # One very long history: the key axis has to be split.
        _attn("decode 1x131071 32/8x128", 1, 1, 131071, 32, 8, 128, 64),
        # SmolVLA's action expert: 256 requests of 50 action tokens over prefix and actions,
        # every action token sees all of them.
        _attn("expert 256x50 15/5x64", 256, 50, 191, 15, 5, 64, 16, causal=False),
        # SmolVLA prefixes: images and language see each other, the state token only backwards.
        _attn("prefix 32x141 15/5x64", 32, 141, 141, 15, 5, 64, 32, prefix=140),
        # A chunk of a prompt after 8 K cached tokens, scores capped.
        _attn("chunk 512 of 8703 32/8x128", 1, 512, 8703, 32, 8, 128, 16, cap=30.0),
        # A whole long prompt.
        _attn("prompt 8191 32/8x128", 1, 8191, 8191, 32, 8, 128, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(15, 5, 64), (32, 8, 128), (16, 16, 64), (32, 4, 128), (12, 2, 96), (8, 8, 32),
          (28, 4, 128), (16, 1, 64)]


def draw(rng):
    kind = rng.choice(("tables", "qkv", "decode", "prompt"))
    page = rng.choice((16, 32, 64, 128))
    if kind == "tables":
        c = _tables("", _log(rng, 1, 1024), _log(rng, 1, 512), _log(rng, 1, 8000), page,
                    rng.random() < 0.5)
    elif kind == "qkv":
        heads, kv_heads, hd = rng.choice(_HEADS)
        axes = rng.choice((1, 1, 3))
        rot = hd if axes == 3 or rng.random() < 0.7 else hd // 2
        c = _qkv("", _log(rng, 1, 16000 * 6144 // ((heads + 2 * kv_heads) * hd + 6144)), heads,
                 kv_heads, hd, page, rng.choice(("f32", "bf16")), rng.random() < 0.8, rot, axes,
                 rng.random() < 0.3)
    elif kind == "decode":
        heads, kv_heads, hd = rng.choice(_HEADS)
        seqs = _log(rng, 1, 128)
        most = 64 * 16384 * 8 * 136 * 0.6 / (seqs * kv_heads * (hd + hd // 16))
        c = _attn("", seqs, rng.choice((1, 1, 1, 2, 4)), _log(rng, 4, min(most, 100000)), heads,
                  kv_heads, hd, page, cap=rng.choice((0.0, 0.0, 30.0)),
                  window=rng.choice((0, 0, 0, 1024)), bias=rng.random() < 0.2, ragged=True)
    else:
        heads, kv_heads, hd = rng.choice(_HEADS)
        seqs = _log(rng, 1, 16)
        q = _log(rng, 16, 4000 // seqs + 16)
        kv = q + rng.choice((0, _log(rng, 1, 4000)))
        causal = rng.random() < 0.8
        c = _attn("", seqs, q, kv, heads, kv_heads, hd, page, causal=causal,
                  prefix=_log(rng, 1, kv) if causal and rng.random() < 0.3 else 0,
                  window=rng.choice((0, 0, 0, 512)) if causal else 0,
                  cap=rng.choice((0.0, 0.0, 50.0)), bias=rng.random() < 0.2,
                  ragged=rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(case):
    """The new tokens and the cached ones of each request: part of the case, not of its seed."""
    rng = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["seqs"]
    if case["op"] == "tables":
        fresh = [rng.randint(1, case["fresh"]) if case["mixed"] and i % 4 == 0 else 1 for i in range(n)]
        cached = [0 if case["mixed"] and i % 8 == 0 else rng.randint(0, case["cached"]) for i in range(n)]
        return fresh, cached
    q, kv = case["q"], case["kv"]
    if not case["ragged"]:
        return [q] * n, [kv - min(q, kv)] * n
    fresh = [q] + [rng.randint(1, q) for _ in range(n - 1)]
    total = [kv] + [max(f, int(kv * (1 - 0.75 * rng.random()))) for f in fresh[1:]]
    return fresh, [max(0, t - f) for t, f in zip(total, fresh)]


def _pages(tokens, page):
    return -(-tokens // page)


# ---------------------------------------------------------------------------------------------
# the 4-bit format, in elementary operations

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _encode(x):
    """x [..., 32 n] in FP32 -> E2M1 codes (0..15) and scale bytes [..., n]."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = (torch.frexp(top).exponent - 3).clamp(E_MIN, E_MAX)
    e = torch.where(top > 0, e, torch.full_like(e, E_MIN))
    m = torch.ldexp(b.abs(), -e.unsqueeze(-1))
    # Nearest, ties to the even code: the code is the number of ties below |x|.
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5)
            + (m >= 3.5) + (m > 5.0))
    code = torch.where(b < 0, code | 8, code)
    return code.flatten(-2).to(torch.uint8), (e + 127).to(torch.uint8)


def _decode(code, scale):
    """Codes [..., 32 n] and scale bytes [..., n] -> FP32 values."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=code.device)
    v = table[code.long()].unflatten(-1, (-1, 32))
    return torch.ldexp(v, (scale.int() - 127).unsqueeze(-1)).flatten(-2)


def _fill_cache(gen, pages, page, kv_heads, hd):
    """Pages of keys and values as a server's cache holds them: [pages][kv_heads][record]."""
    parts = []
    for spread in (True, False):
        code = torch.empty(pages, kv_heads, page, hd, dtype=torch.uint8, device="cuda")
        scale = torch.empty(pages, kv_heads, page, hd // 32, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // (page * kv_heads * hd))
        for p in range(0, pages, step):
            x = torch.randn(min(step, pages - p), kv_heads, page, hd, device="cuda", generator=gen)
            if spread:  # keys have a few large channels
                x[..., ::16] *= 3.0
            code[p:p + step], scale[p:p + step] = _encode(x)
        parts += [(code[..., 0::2] | (code[..., 1::2] << 4)).flatten(2), scale.flatten(2)]
    return torch.cat(parts, 2).contiguous()


def _split(cache, page, hd):
    """The four parts of the records: K codes, K scales, V codes, V scales."""
    at, parts = 0, []
    for width in (hd // 2, hd // 32, hd // 2, hd // 32):
        parts.append(cache[..., at:at + page * width].unflatten(-1, (page, width)))
        at += page * width
    return parts


# ---------------------------------------------------------------------------------------------
# states


def _rope_table(rot):
    inv = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    angle = torch.arange(MAX_POS, dtype=torch.float64)[:, None] * inv
    return torch.stack((angle.cos(), angle.sin()), -1).float().cuda()


def _sections(rot, axes):
    half = rot // 2
    return (half,) if axes == 1 else (half // 4, (half - half // 4) // 2,
                                      half - half // 4 - (half - half // 4) // 2)


_keep = {}


def _library():
    """The framework's context on torch's stream, one for the process."""
    from hotarubi_b200 import capi
    if "lib" not in _keep:
        _keep["lib"] = capi.Library(torch.cuda.current_device())
    _keep["lib"].set_stream(torch.cuda.current_stream().cuda_stream)
    return capi, _keep["lib"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    s = {"case": case}
    page = case["page"]
    if case["op"] == "tables":
        fresh, cached = _lengths(case)
        ld = max(_pages(f + c, page) for f, c in zip(fresh, cached))
        have = [_pages(c, page) for c in cached]
        pages = sum(_pages(f + c, page) for f, c in zip(fresh, cached)) + 64
        perm = torch.randperm(pages, device=dev, generator=gen).int()
        s["fresh"], s["cached"] = (torch.tensor(v, dtype=torch.int32, device=dev) for v in (fresh, cached))
        table = torch.full((case["seqs"], ld), -1, dtype=torch.int32, device=dev)
        row = torch.tensor([i for i, h in enumerate(have) for _ in range(h)], device=dev, dtype=torch.long)
        col = torch.tensor([n for h in have for n in range(h)], device=dev, dtype=torch.long)
        table[row, col] = perm[:row.numel()]
        s["table"], s["free"], s["tokens"] = table, perm[row.numel():].contiguous(), sum(fresh)
        s["head"] = torch.randint(0, 32, (1,), device=dev, generator=gen, dtype=torch.int32)
        s["slots"] = torch.empty(s["tokens"], dtype=torch.int32, device=dev)
        s["pos"] = torch.empty(s["tokens"], dtype=torch.int32, device=dev)
        s["start"] = torch.empty(case["seqs"] + 1, dtype=torch.int32, device=dev)
        s["kv_len"] = torch.empty(case["seqs"], dtype=torch.int32, device=dev)
        s["head_out"] = torch.empty(1, dtype=torch.int32, device=dev)
        if own:
            capi, _ = _library()
            s["desc"] = capi.blocks_desc(
                case["seqs"], page, cached=s["cached"], fresh=s["fresh"], free_pages=s["free"],
                nfree=s["free"].numel(), head_in=s["head"], head_out=s["head_out"], table=table,
                table_ld=ld, q_start=s["start"], kv_len=s["kv_len"], slots=s["slots"],
                pos=s["pos"], max_tokens=s["tokens"])
        return s
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["hd"]
    if case["op"] == "qkv":
        n = case["tokens"]
        dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        x = torch.randn(n, (heads + 2 * kv_heads) * hd, device=dev, generator=gen)
        s["qkv"] = (x * (0.5 + torch.rand(n, 1, device=dev, generator=gen))).to(dt)
        s["wq"], s["wk"] = (0.5 + torch.rand(hd, device=dev, generator=gen) for _ in range(2))
        s["rope"] = _rope_table(case["rot"])
        s["axis"] = torch.tensor([a for a, count in enumerate(_sections(case["rot"], case["axes"]))
                                  for _ in range(count)], device=dev)   # of each pair
        # A prompt's tokens in order, from a position of its own: frames of 24 x 24 patches where
        # there are three axes. Their pages lie anywhere in the cache.
        t = torch.arange(n, device=dev)
        at = t + torch.randint(0, MAX_POS - n, (1,), device=dev, generator=gen)
        s["pos"] = (at[None] if case["axes"] == 1 else
                    torch.stack((at[0] + t // 576, t // 24 % 24, t % 24))).int().contiguous()
        pages = _pages(n, page) + 3
        perm = torch.randperm(pages, device=dev, generator=gen)
        s["slots"] = (perm[t // page] * page + t % page).int()
        s["cache"] = torch.zeros(pages, kv_heads, page * (hd + hd // 16), dtype=torch.uint8, device=dev)
        s["q"] = torch.empty(n, heads * hd, dtype=torch.bfloat16, device=dev)
        s["k"], s["v"] = (torch.empty(n, kv_heads * hd, dtype=torch.float8_e5m2, device=dev)
                          for _ in range(2))
        if own:
            capi, _ = _library()
            s["e5m2"] = capi.DT_E5M2
            s["kv"] = capi.kv_cache(s["cache"], pages, page, kv_heads, hd)
            s["desc"] = capi.qkv_desc(
                s["kv"], n, heads, dtype=capi.DT_F32 if case["dtype"] == "f32" else capi.DT_BF16,
                q=s["qkv"], k=s["qkv"][:, heads * hd:], v=s["qkv"][:, (heads + kv_heads) * hd:],
                ldq=x.shape[1], ldk=x.shape[1], ldv=x.shape[1],
                q_norm=s["wq"] if case["norm"] else None, k_norm=s["wk"] if case["norm"] else None,
                eps=EPS, rope=s["rope"], max_pos=MAX_POS, rot=case["rot"],
                interleaved=case["interleaved"], pos=s["pos"], axes=case["axes"],
                sections=_sections(case["rot"], case["axes"]), slots=s["slots"], q_out=s["q"])
        return s
    fresh, cached = _lengths(case)
    total = [f + c for f, c in zip(fresh, cached)]
    need = [_pages(t, page) for t in total]
    pages = sum(need) + 5
    perm = torch.randperm(pages, device=dev, generator=gen).int()
    table = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        at += k
    s["cache"] = _fill_cache(gen, pages, page, kv_heads, hd)
    s["table"] = table
    s["kv_len"] = torch.tensor(total, dtype=torch.int32, device=dev)
    start = [0]
    for f in fresh:
        start.append(start[-1] + f)
    s["start"] = torch.tensor(start, dtype=torch.int32, device=dev)
    s["max_q"], s["max_kv"], s["sum_kv"] = max(fresh), max(total), sum(total)
    s["q"] = torch.randn(start[-1], heads * hd, device=dev, generator=gen).to(torch.bfloat16)
    s["prefix"] = s["kv_len"].clamp(max=case["prefix"]).contiguous()
    s["slopes"] = 0.1 * torch.rand(heads, device=dev, generator=gen)
    s["out"] = torch.empty(start[-1], heads * hd, dtype=torch.bfloat16, device=dev)
    if own:
        capi, _ = _library()
        s["desc"] = capi.attn_desc(
            capi.kv_cache(s["cache"], pages, page, kv_heads, hd), case["seqs"], heads, q=s["q"],
            q_start=s["start"], total_q=start[-1], max_q=s["max_q"], kv_len=s["kv_len"],
            max_kv=s["max_kv"], total_kv=s["sum_kv"], table=table, table_ld=table.shape[1],
            scale=hd ** -0.5, causal=case["causal"], softcap=case["cap"], window=case["window"],
            prefix=s["prefix"] if case["prefix"] else None,
            slopes=s["slopes"] if case["bias"] else None, out=s["out"])
    return s


# ---------------------------------------------------------------------------------------------
# one pass


def run(s):
    if own:
        return _run_own(s)
    return {"tables": _plain_tables, "qkv": _plain_qkv, "attn": _plain_attn}[s["case"]["op"]](s)


def _run_own(s):
    lib = _keep["lib"]
    if s["case"]["op"] == "tables":
        lib.block_tables(s["desc"])
        return {k: s[k] for k in ("table", "slots", "pos", "start", "kv_len", "head_out")}
    if s["case"]["op"] == "qkv":
        lib.qkv_append(s["desc"])
        lib.kv_read(s["kv"], s["slots"], s["case"]["tokens"], s["k"], s["v"],
                    dtype=s["e5m2"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    lib.attention(s["desc"])
    return s["out"]


def _plain_tables(s):
    page, cached, fresh = s["case"]["page"], s["cached"], s["fresh"]
    kv_len = cached + fresh
    have = (cached + page - 1) // page
    need = (kv_len + page - 1) // page - have
    base = s["head"] + torch.cumsum(need, 0) - need
    col = torch.arange(s["table"].shape[1], device=cached.device)
    new = (col >= have[:, None]) & (col < (have + need)[:, None])
    page_of = (base[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1).long()
    table = torch.where(new, s["free"][page_of], s["table"])
    start = torch.cat((torch.zeros_like(fresh[:1]), torch.cumsum(fresh, 0)))
    t = torch.arange(s["tokens"], device=cached.device)
    seq = torch.searchsorted(start[1:].long(), t, right=True)
    pos = t - start[seq] + cached[seq]
    slots = table[seq, pos // page] * page + pos % page
    return {"table": table, "slots": slots.int(), "pos": pos.int(), "start": start.int(),
            "kv_len": kv_len, "head_out": (s["head"] + need.sum()).int()}


def _rotate(x, s, case):
    """x [tokens][heads][hd]: pairs of the first `rot` dims turned by their axis' position."""
    rot = case["rot"]
    cs = s["rope"][s["pos"][s["axis"]].long().T, torch.arange(rot // 2, device=x.device)]
    c, d = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = ((x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"]
            else (x[..., :rot // 2], x[..., rot // 2:rot]))
    a, b = a * c - b * d, b * c + a * d
    turned = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_qkv(s):
    case = s["case"]
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["hd"]
    x = s["qkv"].float().unflatten(1, (-1, hd))
    q, k, v = x.split((heads, kv_heads, kv_heads), 1)
    if case["norm"]:
        q = q * (1.0 / torch.sqrt(q.square().mean(-1, keepdim=True) + EPS)) * s["wq"]
        k = k * (1.0 / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS)) * s["wk"]
    q, k = _rotate(q, s, case), _rotate(k, s, case)
    # Every value of the 4-bit format with an exponent above -16 is an E5M2 number.
    k, v = (_decode(*_encode(y)).flatten(1).to(torch.float8_e5m2) for y in (k, v))
    return {"q": q.flatten(1).to(torch.bfloat16), "k": k, "v": v}


def _visible(i, j, prefix, case):
    """Whether the query at position i sees the key at position j."""
    if not case["causal"]:
        return j >= 0
    ok = j <= i
    if case["window"]:
        ok = ok & (j > i - case["window"])
    return ok | (j < prefix) if case["prefix"] else ok


def _plain_attn(s):
    case = s["case"]
    page, heads, kv_heads, hd = case["page"], case["heads"], case["kv_heads"], case["hd"]
    n, max_q, max_kv, dev = case["seqs"], s["max_q"], s["max_kv"], s["q"].device
    group = heads // kv_heads
    j = torch.arange(max_kv, device=dev)
    pages = s["table"][:, j // page].clamp(min=0).long()                    # [n][kv]
    kc, ks, vc, vs = _split(s["cache"], page, hd)
    low = lambda b: torch.stack((b & 15, b >> 4), -1).flatten(-2)           # noqa: E731
    pick = lambda part: part.transpose(1, 2)[pages, j % page]               # noqa: E731  [n][kv][head][..]
    k = _decode(low(pick(kc)), pick(ks)).transpose(1, 2)
    v = _decode(low(pick(vc)), pick(vs)).transpose(1, 2)
    r = torch.arange(max_q, device=dev)
    q_len = s["start"][1:] - s["start"][:-1]
    row = (s["start"][:-1, None] + r).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"].float()[row].unflatten(2, (kv_heads, group, hd)).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).mul_(hd ** -0.5)
    del k
    score = score.unflatten(2, (group, max_q))                              # [n][kvh][g][q][kv]
    if case["cap"]:
        score = score.div_(case["cap"]).tanh_().mul_(case["cap"])
    i = (s["kv_len"] - q_len)[:, None, None] + r[:, None]                   # [n][q][1]
    if case["bias"]:
        slope = s["slopes"].view(kv_heads, group, 1, 1)
        score -= slope * (i - j).abs()[:, None, None].float()
    seen = _visible(i, j, s["prefix"][:, None, None], case) & (j < s["kv_len"][:, None, None])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, max_q))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).flatten(2)                                 # [n][q][heads * hd]
    return o[r < q_len[:, None]].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without


def _pairs(case, fresh, cached):
    """(query, key) pairs that see each other, and the keys that any query sees."""
    pairs, keys = 0, 0
    for f, c in zip(fresh, cached):
        kv = f + c
        if not case["causal"]:
            pairs, keys = pairs + f * kv, keys + kv
            continue
        pre, win = min(case["prefix"], kv), case["window"]
        for i in range(c, kv):
            lo = max(0, i - win + 1) if win else 0
            pairs += i + 1 - lo + max(0, pre - (i + 1)) + min(lo, pre)
        lo = max(0, c - win + 1) if win else 0
        keys += kv - lo + min(lo, pre)
    return pairs, keys


def work(case):
    page = case["page"]
    if case["op"] == "tables":
        fresh, cached = _lengths(case)
        new = sum(_pages(f + c, page) - _pages(c, page) for f, c in zip(fresh, cached))
        old = sum(1 for c in cached if c % page)
        return {"bytes": 16.0 * case["seqs"] + 8.0 * new + 4.0 * old + 8.0 * sum(fresh), "flops": 0.0}
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["hd"]
    if case["op"] == "qkv":
        n, size = case["tokens"], 4 if case["dtype"] == "f32" else 2
        row = (heads + 2 * kv_heads) * hd * size + heads * hd * 2 + kv_heads * (hd + hd // 16)
        return {"bytes": float(n * (row + kv_heads * hd * 2 + 4 + case["axes"] * 4 + case["rot"] * 4)),
                "flops": float(n * (heads + kv_heads) * hd * 8)}
    fresh, cached = _lengths(case)
    pairs, keys = _pairs(case, fresh, cached)
    return {"bytes": float(keys * kv_heads * (hd + hd // 16) + sum(fresh) * heads * hd * 4
                           + 4 * (keys // page) + 12 * case["seqs"]),
            "flops": 4.0 * hd * heads * pairs}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    global own
    if case["op"] == "tables":
        return None  # whole numbers: the plain form's are the definition's
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _exact_qkv(s) if case["op"] == "qkv" else _exact_attn(s)


def _exact_qkv(s):
    case = s["case"]
    heads, kv_heads, hd, rot = case["heads"], case["kv_heads"], case["hd"], case["rot"]
    x = s["qkv"].double()
    q = x[:, :heads * hd].reshape(-1, heads, hd)
    if case["norm"]:
        q = q * (q.pow(2).sum(-1, keepdim=True) / hd + EPS).pow(-0.5) * s["wq"].double()
    out = q.clone()
    first = 0
    for axis, count in enumerate(_sections(rot, case["axes"])):
        for p in range(first, first + count):
            a, b = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + rot // 2)
            cs = s["rope"][s["pos"][axis].long(), p].double()
            out[..., a] = q[..., a] * cs[:, :1] - q[..., b] * cs[:, 1:]
            out[..., b] = q[..., b] * cs[:, :1] + q[..., a] * cs[:, 1:]
        first += count
    # V: the nearest of the format's values times the block's power of two (no arithmetic comes
    # before the rounding, so it is exact). K is rounded after a norm and a rotation: near the
    # middle of two codes either may be right, a whole step apart, so it has no such value.
    v = x[:, (heads + kv_heads) * hd:].reshape(-1, 32)
    e = torch.floor(torch.log2(v.abs().amax(1, keepdim=True).clamp(min=2.0 ** -40))) - 2
    e = e.clamp(E_MIN, E_MAX)
    u = v.abs() / torch.exp2(e)
    step = torch.where(u < 2, 0.5, torch.where(u < 4, 1.0, 2.0)).double()
    u = (torch.round(u / step) * step).clamp(max=6.0)
    v = (torch.sign(v) * u * torch.exp2(e)).reshape(len(x), -1)
    return {"q": out.reshape(len(x), -1), "k": None, "v": v}


def _exact_attn(s):
    case = s["case"]
    page, heads, kv_heads, hd = case["page"], case["heads"], case["kv_heads"], case["hd"]
    group = heads // kv_heads
    dev = s["q"].device
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    rec = s["cache"]

    def values(raw, scales):  # codes s e e m -> (-1)^s * 2^(max(e,1)-1) * (m/2 + (e>0))
        c = torch.stack((raw % 16, raw // 16), -1).reshape(*raw.shape[:-1], -1).double()
        neg, mag = torch.floor(c / 8), c % 8
        e, m = torch.floor(mag / 2), mag % 2
        x = (1 - 2 * neg) * torch.exp2(e.clamp(min=1) - 1) * (m / 2 + (e > 0).double())
        return x * torch.repeat_interleave(torch.exp2(scales.double() - 127), 32, -1)

    for n in range(case["seqs"]):
        a, b, kv = int(s["start"][n]), int(s["start"][n + 1]), int(s["kv_len"][n])
        pages = s["table"][n, :_pages(kv, page)].long()
        j = torch.arange(kv, device=dev)
        i = torch.arange(kv - (b - a), kv, device=dev)[:, None]
        seen = _visible(i, j[None], int(s["prefix"][n]), case)
        for h in range(kv_heads):
            r = rec[pages, h]
            w, z = page * hd // 2, page * hd // 32
            k = values(r[:, :w].reshape(-1, hd // 2), r[:, w:w + z].reshape(-1, hd // 32))[:kv]
            r = r[:, w + z:]
            v = values(r[:, :w].reshape(-1, hd // 2), r[:, w:].reshape(-1, hd // 32))[:kv]
            for g in range(group):
                c = (h * group + g) * hd
                t = s["q"][a:b, c:c + hd].double() @ k.T / math.sqrt(hd)
                if case["cap"]:
                    t = case["cap"] * torch.tanh(t / case["cap"])
                if case["bias"]:
                    t = t - s["slopes"][h * group + g].double() * (i - j[None]).abs()
                p = torch.softmax(t.masked_fill(~seen, -math.inf), -1)
                out[a:b, c:c + hd] = torch.nan_to_num(p) @ v
    return out
