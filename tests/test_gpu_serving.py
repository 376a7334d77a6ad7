"""The serving calls on the GPU (hrb_block_tables, hrb_qkv_append,
hrb_kv_read, hrb_attention) against the plain 64-bit forms of
serving_ref.py, and their refusals.

Tolerances.  Whole numbers and V's codes are equal.  q_out: one BF16 rounding
(8 significant bits: 2^-8 of the value) and FP32 arithmetic on the pair (2^-19 of its two values).
K's codes: equal, except where the 64-bit value lies within 2^-18 of the
middle between two codes or the block's largest value within 2^-18 of a power
of two, where the neighbour is right too.  Attention: one BF16 rounding of
the result (2^-8), and 2^-9 of sum_j p_j |v_j| for the softmax weights' FP16
rounding (2^-11), the scores' FP32 sums and the exponentials.
"""
import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from hotarubi_b200 import capi  # noqa: E402


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def ready():
    """torch's copies and fills run on its own stream."""
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# block tables


def run_tables(hrb, cached, fresh, free, head, table, page, max_tokens, pos=True, stream=0):
    n = len(cached)
    t = {k: dev(np.asarray(v, np.int32)) for k, v in
         dict(cached=cached, fresh=fresh, free=free, table=table, head=[head]).items()}
    out = {k: torch.full((m,), 77, dtype=torch.int32, device="cuda") for k, m in
           dict(start=n + 1, kv=n, slots=max_tokens, pos=max_tokens, head=1).items()}
    ready()
    hrb.block_tables(capi.blocks_desc(
        n, page, cached=t["cached"], fresh=t["fresh"], free_pages=t["free"], nfree=len(free),
        head_in=t["head"], head_out=out["head"], table=t["table"], table_ld=table.shape[1],
        q_start=out["start"], kv_len=out["kv"], slots=out["slots"],
        pos=out["pos"] if pos else None, max_tokens=max_tokens), stream=stream)
    err = None
    try:
        hrb.sync()
    except capi.HrbError as e:
        err = e
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in (t["table"], out["slots"], out["pos"], out["start"],
                                      out["kv"], out["head"])], err


def tables_case(rng, n, page, most_fresh, most_cached, ld_more=2):
    fresh = rng.integers(0, most_fresh + 1, n)
    cached = rng.integers(0, most_cached + 1, n)
    cached[rng.random(n) < 0.2] = 0
    have, total = -(-cached // page), -(-(cached + fresh) // page)
    table = rng.integers(0, 10000, (n, max(1, int(total.max(initial=0)) + ld_more))).astype(np.int32)
    free = rng.permutation(int((total - have).sum()) + 9).astype(np.int32)
    return cached, fresh, free, table


@pytest.mark.parametrize("n,page,most_fresh,most_cached", [
    (1, 16, 1, 0), (1, 16, 1, 15), (3, 32, 0, 100), (8, 16, 1, 2000), (7, 256, 900, 300),
    (300, 16, 40, 500), (1000, 64, 1, 5000), (2000, 16, 3, 50), (257, 128, 700, 10)])
def test_block_tables(hrb, n, page, most_fresh, most_cached):
    rng = np.random.default_rng(n * 31 + page)
    cached, fresh, free, table = tables_case(rng, n, page, most_fresh, most_cached)
    tokens = int(fresh.sum())
    for pad in (0, 5):
        if tokens + pad == 0:
            continue
        want = ref.block_tables(cached, fresh, free, 4, table, page, tokens + pad)
        got, err = run_tables(hrb, cached, fresh, free, 4, table, page, tokens + pad)
        assert err is None
        for name, w, g in zip(("table", "slots", "pos", "start", "kv_len"), want, got):
            assert np.array_equal(w, g), name
        assert got[5][0] == want[5]


@pytest.mark.parametrize("what", ["pages", "tokens", "row", "negative", "hole"])
def test_block_tables_short_of_something(hrb, what):
    rng = np.random.default_rng(5)
    cached, fresh, free, table = tables_case(rng, 40, 16, 50, 100)
    tokens = int(fresh.sum())
    if what == "pages":
        free = free[:10]
    elif what == "tokens":
        tokens -= 30
    elif what == "row":
        table = table[:, :3]
    elif what == "negative":
        fresh[3], cached[7] = -4, -1
        tokens = int(np.maximum(fresh, 0).sum())
    else:
        i = int(np.argmax((cached % 16 != 0) & (fresh > 0)))
        table[i, cached[i] // 16] = -1
    want = ref.block_tables(cached, fresh, free, 2, table, 16, tokens)
    got, err = run_tables(hrb, cached, fresh, free, 2, table, 16, tokens)
    assert err is not None and err.status == capi.HRB_EDATA
    for name, w, g in zip(("table", "slots", "pos", "start", "kv_len"), want, got):
        assert np.array_equal(w, g), name


# ---------------------------------------------------------------------------
# QKV append


def run_qkv(hrb, c, x, heads, bf16=False, w=None, table=None, pos=None, rot=0, interleaved=False,
            sections=(), slots=None, pad=0, shift=0, eps=1e-6):
    """x: q, k, v as [tokens][heads][hd].  pad: extra elements a row; shift:
    elements the rows start off a 16-byte boundary."""
    tokens, hd = x[0].shape[0], c.hd
    flat = np.concatenate([v.reshape(tokens, -1) for v in x] + [np.zeros((tokens, pad), np.float32)], 1)
    ld = flat.shape[1]
    buf = torch.zeros(tokens * ld + shift, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    buf[shift:] = dev(flat.astype(np.float32)).reshape(-1).to(buf.dtype)
    at = buf.data_ptr() + shift * buf.element_size()
    size = buf.element_size()
    data = dev(c.data)
    keep = [None if v is None else dev(v) for v in (w and w[0], w and w[1], table)]
    dpos = None if pos is None else dev(np.asarray(pos, np.int32))
    dslots = dev(np.asarray(slots, np.int32))
    q_out = torch.full((tokens, heads * hd + 4), 9.0, dtype=torch.bfloat16, device="cuda")
    ready()
    hrb.qkv_append(capi.qkv_desc(
        capi.kv_cache(data, c.pages, c.page, c.kv_heads, hd, page_stride=c.stride), tokens, heads,
        dtype=capi.DT_BF16 if bf16 else capi.DT_F32, q=at, k=at + heads * hd * size,
        v=at + (heads + c.kv_heads) * hd * size, ldq=ld, ldk=ld, ldv=ld, q_norm=keep[0],
        k_norm=keep[1], eps=eps, rope=keep[2], max_pos=0 if table is None else len(table), rot=rot,
        interleaved=interleaved, pos=dpos, axes=max(1, len(sections)), sections=sections,
        slots=dslots, q_out=q_out, ldqo=heads * hd + 4))
    err = None
    try:
        hrb.sync()
    except capi.HrbError as e:
        err = e
    assert (q_out[:, heads * hd:] == 9.0).all()
    used = buf[shift:].float().cpu().numpy().reshape(tokens, ld)
    got = ref.Cache(c.pages, c.page, c.kv_heads, hd)
    got.stride, got.data = c.stride, data.cpu().numpy()
    return q_out[:, :heads * hd].float().cpu().numpy().reshape(tokens, heads, hd), got, used, err


def check_codes(got, want, exact):
    """Cached values against the encoding of `want` (64 bits)."""
    code, scale = ref.encode(want)
    value = ref.decode(code, scale)
    if exact:
        assert np.array_equal(got, value)
        return
    near = np.exp2(-18.0)
    up, down = (ref.decode(*ref.encode(want * f)) for f in (1 + near, 1 - near))
    assert ((got == value) | (got == up) | (got == down)).all()


QKV = [
    # heads, kv_heads, hd, page, tokens, bf16, norm, rot, interleaved, sections, pad, shift
    (15, 5, 64, 16, 1, False, True, 64, False, (32,), 0, 0),
    (15, 5, 64, 32, 141, False, True, 64, False, (32,), 0, 0),
    (32, 8, 128, 16, 77, True, True, 128, False, (16, 24, 24), 0, 0),
    (4, 4, 128, 64, 19, False, False, 64, True, (32,), 3, 1),
    (12, 2, 96, 128, 33, True, True, 96, False, (12, 18, 18), 1, 3),
    (6, 1, 96, 16, 300, False, True, 24, True, (12,), 0, 0),
    (8, 8, 32, 256, 65, False, True, 32, False, (10, 6), 0, 2),
    (3, 1, 32, 16, 700, True, False, 8, False, (4,), 4, 0),
    (2, 1, 64, 16, 9, False, True, 0, False, (), 0, 0),
    (28, 4, 128, 16, 1200, True, True, 128, True, (22, 21, 21), 0, 0),
]


@pytest.mark.parametrize("heads,kvh,hd,page,tokens,bf16,norm,rot,inter,sections,pad,shift", QKV)
def test_qkv_append(hrb, heads, kvh, hd, page, tokens, bf16, norm, rot, inter, sections, pad, shift):
    rng = np.random.default_rng(heads * 1000 + hd + tokens)
    pages = -(-tokens // page) + 2
    c = ref.Cache(pages, page, kvh, hd, rng, extra=48)
    before = c.data.copy()
    x = [rng.standard_normal((tokens, h, hd)).astype(np.float32) * s
         for h, s in ((heads, 1.0), (kvh, 3.0), (kvh, 0.02))]
    x[2][0, 0, :32] = 0.0
    x[2][tokens // 2, -1, -32:] = 1e-9      # under the format's smallest value
    w = [(0.5 + rng.random(hd)).astype(np.float32) for _ in range(2)] if norm else None
    table = capi.rope_table(512, rot) if rot else None
    pos = rng.integers(0, 512, (max(1, len(sections)), tokens)) if rot else None
    slots = rng.permutation(pages * page)[:tokens]
    slots[tokens // 3] = -1 if tokens > 2 else slots[tokens // 3]
    q, got, used, err = run_qkv(hrb, c, x, heads, bf16, w, table, pos, rot, inter, sections, slots,
                                pad, shift)
    assert err is None
    split = np.split(used[:, :(heads + 2 * kvh) * hd].reshape(tokens, -1, hd), (heads, heads + kvh), 1)
    args = (1e-6, table, pos, rot, inter, sections)
    want = ref.norm_rotate(split[0], w and w[0], *args)
    spread = np.abs(ref.norm_rotate(split[0], w and w[0], 1e-6, None, None, 0, False, ()))
    pair = spread + np.max(spread, -1, keepdims=True)
    assert (np.abs(q - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -19 * pair).all()
    k = ref.norm_rotate(split[1], w and w[1], *args)
    for t in range(tokens):
        if slots[t] < 0:
            continue
        gk, gv = got.read(slots[t])
        check_codes(gk, k[t], exact=not norm and not rot)
        check_codes(gv, split[2][t].astype(np.float64), exact=True)
    # Nothing else of the cache is touched: other slots, and the gap after a page's records.
    free = np.setdiff1d(np.arange(pages * page), slots)
    old = ref.Cache(pages, page, kvh, hd)
    old.stride, old.data = c.stride, before
    for s in rng.permutation(free)[:50]:
        for h in range(kvh):
            for a, b in zip(got._parts(s // page, h), old._parts(s // page, h)):
                assert np.array_equal(a[s % page], b[s % page])
    assert np.array_equal(got.data[:, kvh * c.record:], before[:, kvh * c.record:])


@pytest.mark.parametrize("what", ["slot", "position", "nan", "inf"])
def test_qkv_append_reports_data_out_of_range(hrb, what):
    rng = np.random.default_rng(8)
    c = ref.Cache(4, 16, 2, 64)
    x = [rng.standard_normal((5, h, 64)).astype(np.float32) for h in (4, 2, 2)]
    slots, pos = np.array([3, 40, 9, 22, 63]), np.array([[1, 2, 3, 4, 5]])
    table = capi.rope_table(16, 64)
    if what == "slot":
        slots[2] = 64
    elif what == "position":
        pos[0, 1] = 16
    else:
        x[2][4, 1, 40] = np.nan if what == "nan" else -np.inf
    q, got, used, err = run_qkv(hrb, c, x, 4, table=table, pos=pos, rot=64, sections=(32,), slots=slots)
    assert err is not None and err.status == capi.HRB_EDATA
    if what == "nan":    # cached as zero, the rest of the row as it is
        v = x[2][4].astype(np.float64)
        v[1, 40] = 0.0
        assert np.array_equal(got.read(63)[1], ref.decode(*ref.encode(v)))
    elif what == "inf":
        assert got.read(63)[1][1, 40] == -6 * 2.0 ** 13
    elif what == "slot":
        assert np.array_equal(got.read(22)[1], ref.decode(*ref.encode(x[2][3].astype(np.float64))))


@pytest.mark.parametrize("dtype", [capi.DT_F32, capi.DT_BF16, capi.DT_E5M2])
@pytest.mark.parametrize("hd", [32, 96, 128])
def test_kv_read(hrb, dtype, hd):
    rng = np.random.default_rng(hd)
    c = ref.Cache(9, 32, 3, hd, rng, extra=16)
    # Every scale byte, those out of the format's range too; E5M2 keeps 2^-16 and above.
    slots = np.concatenate((rng.permutation(9 * 32)[:150], [-1]))
    data, ds = dev(c.data), dev(slots.astype(np.int32))
    t = {capi.DT_F32: torch.float32, capi.DT_BF16: torch.bfloat16,
         capi.DT_E5M2: torch.float8_e5m2}[dtype]
    k, v = (torch.empty(151, 3, hd, dtype=t, device="cuda") for _ in range(2))
    ready()
    cache = capi.kv_cache(data, 9, 32, 3, hd, page_stride=c.stride)
    hrb.kv_read(cache, ds, 151, k, v, dtype=dtype)
    hrb.sync()
    for i, s in enumerate(slots):
        wk, wv = c.read(s) if s >= 0 else (np.zeros((3, hd)),) * 2
        for w, g in ((wk, k[i]), (wv, v[i])):
            w = torch.from_numpy(w).to(t).double() if dtype == capi.DT_E5M2 else torch.from_numpy(w)
            assert torch.equal(w, g.double().cpu())
    ds[7] = 9 * 32
    ready()
    hrb.kv_read(cache, ds, 151, k, None, dtype=dtype)
    with pytest.raises(capi.HrbError) as e:
        hrb.sync()
    assert e.value.status == capi.HRB_EDATA and not k[7].double().any()


# ---------------------------------------------------------------------------
# attention


class Step:
    """One attention call: requests with q rows and kv keys, a cache whose
    other contents are random bytes (every scale byte among them)."""

    def __init__(self, rng, lens, heads, kvh, hd, page, scale=None, extra=0, pad=0, q_scale=1.0,
                 v_scale=1.0):
        self.lens, self.heads, self.kvh, self.hd, self.page = lens, heads, kvh, hd, page
        self.scale = hd ** -0.5 if scale is None else scale
        need = [-(-max(kv, 0) // page) for _, kv in lens]
        self.pages = sum(need) + 3
        c = ref.Cache(self.pages, page, kvh, hd, rng, extra=extra)
        perm = rng.permutation(self.pages)
        self.ld = max(need) + 2
        self.table = np.full((len(lens), self.ld), -1, np.int32)
        self.keys, self.values, at = [], [], 0
        for n, (_, kv) in enumerate(lens):
            self.table[n, :need[n]] = perm[at:at + need[n]]
            at += need[n]
            k = rng.standard_normal((kv, kvh, hd))
            v = rng.standard_normal((kv, kvh, hd)) * v_scale
            k[..., ::16] *= 3.0
            for x, part in ((k, 0), (v, 2)):
                code, sc = ref.encode(x)
                for i in range(-(-kv // page)):
                    m = min(page, kv - i * page)
                    for h in range(kvh):
                        parts = c._parts(self.table[n, i], h)
                        cc = code[i * page:i * page + m, h]
                        parts[part][:m] = cc[:, 0::2] | (cc[:, 1::2] << 4)
                        parts[part + 1][:m] = sc[i * page:i * page + m, h]
                (self.keys if part == 0 else self.values).append(ref.decode(code, sc))
        self.cache = c
        self.start = np.concatenate(([0], np.cumsum([q for q, _ in lens]))).astype(np.int32)
        rows = int(self.start[-1])
        self.ldq = heads * hd + pad
        q = torch.from_numpy(rng.standard_normal((rows, self.ldq)).astype(np.float32) * q_scale)
        self.q = q.to(torch.bfloat16)
        self.rows = rows

    def want(self, **kw):
        q = self.q[:, :self.heads * self.hd].double().numpy().reshape(self.rows, self.heads, self.hd)
        return ref.attention(q, self.start, [max(kv, 0) for _, kv in self.lens], self.keys,
                             self.values, self.scale, **kw)

    def run(self, hrb, prefix=None, slopes=None, oq=False, oquant=capi.QUANT_VEC, out=True, stream=0,
            total_kv=0, workspace=False, sync=True, table=None, max_q=None, max_kv=None, **kw):
        w = self.heads * self.hd
        self.dq, self.dd = self.q.cuda(), dev(self.cache.data)
        lists = [dev(np.asarray(x, np.int32)) for x in
                 (self.start, [kv for _, kv in self.lens], self.table if table is None else table)]
        pre = None if prefix is None else dev(np.asarray(prefix, np.int32))
        slo = None if slopes is None else dev(np.asarray(slopes, np.float32))
        o = torch.full((self.rows, w + 8), 5.0, dtype=torch.bfloat16, device="cuda")
        codes = torch.full((self.rows, w + 32), 99, dtype=torch.int8, device="cuda")
        scales = torch.full((self.rows, w // 32 + 1), 99, dtype=torch.uint8, device="cuda")
        d = capi.attn_desc(
            capi.kv_cache(self.dd, self.pages, self.page, self.kvh, self.hd,
                          page_stride=self.cache.stride), len(self.lens), self.heads, q=self.dq,
            ldq=self.ldq, q_start=lists[0], total_q=self.rows,
            max_q=max(q for q, _ in self.lens) if max_q is None else max_q, kv_len=lists[1],
            max_kv=max(max(kv, 0) for _, kv in self.lens) if max_kv is None else max_kv,
            total_kv=total_kv,
            table=lists[2], table_ld=self.ld, scale=self.scale, prefix=pre, slopes=slo,
            out=o if out else None, ldo=w + 8, oq=codes if oq else None,
            oscale=scales if oq else None, ldoq=w + 32 if oq else 0, oquant=oquant, **kw)
        if workspace:
            n = hrb.attention_workspace(d)
            self.ws = torch.full((max(n, 256) + 256,), 0xFF, dtype=torch.uint8, device="cuda")
            d.workspace, d.workspace_bytes = self.ws.data_ptr(), n
        self.keep = (lists, pre, slo)
        self.out, self.codes, self.scales = o[:, :w], codes, scales
        ready()
        hrb.attention(d, stream=stream)
        if sync:
            hrb.sync()
            torch.cuda.synchronize()
        if workspace:
            assert (self.ws[max(n, 256):] == 0xFF).all()
        assert not out or (o[:, w:] == 5.0).all()
        return o[:, :w].double().cpu().numpy().reshape(self.rows, self.heads, self.hd)


def close(got, want, mass):
    assert np.isfinite(got).all()
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * mass
    bad = np.abs(got - want) > tol
    assert not bad.any(), (f"{bad.sum()} of {bad.size} outputs off, the worst by "
                           f"{(np.abs(got - want) / np.maximum(tol, 1e-30)).max():.2f} tolerances")


SHAPES = [(15, 5, 64, 16), (32, 8, 128, 16), (12, 2, 96, 64), (8, 8, 32, 32), (4, 4, 128, 256),
          (16, 1, 64, 128), (28, 4, 128, 32), (5, 1, 32, 16)]
DECODE = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 100), (1, 255), (1, 700), (1, 64)]


@pytest.mark.parametrize("heads,kvh,hd,page", SHAPES)
def test_attention_single_tokens(hrb, heads, kvh, hd, page):
    rng = np.random.default_rng(heads + hd)
    s = Step(rng, DECODE, heads, kvh, hd, page, extra=32, pad=8)
    close(s.run(hrb), *s.want())


@pytest.mark.parametrize("heads,kvh,hd,page", SHAPES)
def test_attention_prompts(hrb, heads, kvh, hd, page):
    rng = np.random.default_rng(heads + hd + 1)
    s = Step(rng, [(129, 129), (1, 300), (200, 517), (0, 40), (64, 64), (33, 257)], heads, kvh, hd,
             page, pad=8)
    close(s.run(hrb), *s.want())


@pytest.mark.parametrize("q", [2, 3, 4, 5, 8, 13, 21])
def test_attention_a_few_tokens(hrb, q):
    rng = np.random.default_rng(q)
    s = Step(rng, [(q, 333), (1, 1), (q - 1, q + 15), (q, q)], 12, 3, 64, 16)
    close(s.run(hrb), *s.want())


OPTIONS = [
    dict(causal=False),
    dict(window=1), dict(window=40), dict(window=300),
    dict(softcap=2.0), dict(softcap=30.0, window=64),
    dict(prefix="some"), dict(prefix="some", window=17), dict(prefix="all"),
    dict(slopes=True), dict(slopes=True, prefix="some", softcap=5.0, window=90),
    dict(slopes=True, causal=False),
]


@pytest.mark.parametrize("lens", [DECODE, [(70, 70), (150, 411), (3, 290), (1, 128)],
                                  [(3, 200), (4, 4), (2, 65)]], ids=["one", "prompt", "few"])
@pytest.mark.parametrize("option", OPTIONS, ids=str)
def test_attention_masks_and_scores(hrb, lens, option):
    rng = np.random.default_rng(77)
    option = dict(option)
    s = Step(rng, lens, 6, 2, 64, 16)
    if option.get("prefix"):
        kv = np.array([k for _, k in lens])
        option["prefix"] = (kv + 5 if option["prefix"] == "all"
                            else rng.integers(-1, 100, len(lens))).astype(np.int32)
    if option.get("slopes"):
        option["slopes"] = (0.2 * rng.random(6)).astype(np.float32)
    ref_option = dict(option)
    if "prefix" in option:
        ref_option["prefix"] = np.minimum(option["prefix"], [k for _, k in lens])
    close(s.run(hrb, **option), *s.want(**ref_option))


@pytest.mark.parametrize("lens", [[(1, 0), (1, 5), (3, 1), (4, 0)], [(100, 60), (300, 128), (7, 0)]])
def test_attention_rows_that_see_nothing_are_zero(hrb, lens):
    """More rows than keys: the first rows are before the first key."""
    rng = np.random.default_rng(3)
    s = Step(rng, lens, 4, 2, 64, 16)
    want, mass = s.want()
    got = s.run(hrb)
    close(got, want, mass)
    empty = mass.sum(-1) == 0
    assert empty.any() and not got[empty].any()


@pytest.mark.parametrize("q", [1, 90])
def test_attention_a_negative_length_is_no_keys(hrb, q):
    rng = np.random.default_rng(4)
    s = Step(rng, [(q, 130), (q, 0), (q, 150)], 4, 2, 64, 16)
    s.lens = [(q, 130), (q, -3), (q, 150)]
    close(s.run(hrb), *s.want())


@pytest.mark.parametrize("what", ["kv", "rows", "order"])
@pytest.mark.parametrize("q", [1, 90])
def test_attention_leaves_out_requests_past_its_bounds(hrb, what, q):
    rng = np.random.default_rng(5)
    s = Step(rng, [(q, 130), (q, 120), (q, 150)], 4, 2, 64, 16)
    want, mass = s.want()
    if what == "kv":
        s.lens[1] = (q, 1 << 20)
        kw = dict(max_kv=150)
    elif what == "rows":
        s.start[3] += 5
        kw = dict(max_q=q)
    else:
        s.start[1] = -4
        kw = {}
    with pytest.raises(capi.HrbError) as e:
        s.run(hrb, **kw)
    assert e.value.status == capi.HRB_EDATA
    torch.cuda.synchronize()
    out = {"kv": [1], "rows": [2], "order": [0, 1]}[what]
    got = s.out.double().cpu().numpy().reshape(s.rows, s.heads, s.hd)
    for n in range(3):
        a, b = n * q, (n + 1) * q
        if n in out:
            assert (got[a:b] == 5.0).all()
        else:
            close(got[a:b], want[a:b], mass[a:b])


@pytest.mark.parametrize("lens", [[(1, 3000), (1, 2049), (1, 5)], [(5, 4100)], [(140, 2500)]])
def test_attention_long_keys_are_split_and_joined(hrb, lens):
    rng = np.random.default_rng(9)
    s = Step(rng, lens, 8, 2, 128, 16)
    got = s.run(hrb, workspace=True, total_kv=sum(k for _, k in lens))
    close(got, *s.want())
    again = s.run(hrb, workspace=True, total_kv=sum(k for _, k in lens))
    assert np.array_equal(got, again)


@pytest.mark.parametrize("rule", [capi.QUANT_HOST, capi.QUANT_VEC])
@pytest.mark.parametrize("lens", [DECODE, [(150, 200), (1, 90)]], ids=["one", "prompt"])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 64), (6, 2, 96), (3, 1, 32), (8, 2, 128)])
def test_attention_mxint8_copy(hrb, rule, lens, heads, kvh, hd):
    """Codes and scales are the framework's encoding of the result: within
    half a step (plus the result's own tolerance) of the 64-bit value."""
    rng = np.random.default_rng(11)
    s = Step(rng, lens, heads, kvh, hd, 16)
    want, mass = s.want()
    for out in (True, False):
        got = s.run(hrb, oq=True, oquant=rule, out=out)
        if out:
            close(got, want, mass)
        w = heads * hd
        codes = s.codes.cpu().numpy()
        scales = s.scales.cpu().numpy()
        assert (codes[:, w:] == 99).all() and (scales[:, w // 32:] == 99).all()
        step = np.repeat(np.exp2(scales[:, :w // 32].astype(np.float64) - 133), 32, 1)
        value = (codes[:, :w] * step).reshape(want.shape)
        tol = 0.5 * step.reshape(want.shape) + 2.0 ** -9 * mass
        # The largest code is 127: a value that rounds to 128 steps saturates.
        tol = tol + np.where(np.abs(codes[:, :w].reshape(want.shape)) == 127,
                             step.reshape(want.shape), 0)
        assert (np.abs(value - want) <= tol).all()
        assert (np.abs(codes[:, :w].astype(int)).reshape(-1, 32).max(1) >= 63).all() or \
            (mass == 0).any()


@pytest.mark.parametrize("lens", [[(1, 0), (2, 0)], [(100, 0), (7, 0)]])
def test_attention_without_any_key(hrb, lens):
    rng = np.random.default_rng(6)
    s = Step(rng, lens, 4, 2, 64, 16)
    assert not s.run(hrb, oq=True).any()
    assert not s.codes[:, :256].any()


@pytest.mark.parametrize("heads,kvh,hd", [(48, 1, 64), (64, 2, 128), (40, 2, 96), (9, 1, 32)])
@pytest.mark.parametrize("lens", [DECODE, [(40, 90), (2, 400)]], ids=["one", "prompt"])
def test_attention_many_query_heads_a_head(hrb, heads, kvh, hd, lens):
    rng = np.random.default_rng(heads)
    s = Step(rng, lens, heads, kvh, hd, 16)
    close(s.run(hrb), *s.want())


def test_attention_more_keys_than_total_kv_says(hrb):
    """Scratch for 5 tiles: the first request's four fit, the others are left
    out and reported; the next call is not disturbed."""
    rng = np.random.default_rng(7)
    s = Step(rng, [(100, 500), (100, 500), (100, 400)], 4, 2, 64, 16)
    want, mass = s.want()
    with pytest.raises(capi.HrbError) as e:
        s.run(hrb, total_kv=300)
    assert e.value.status == capi.HRB_EDATA
    torch.cuda.synchronize()
    got = s.out.double().cpu().numpy().reshape(s.rows, s.heads, s.hd)
    close(got[:100], want[:100], mass[:100])
    assert (got[100:] == 5.0).all()
    close(s.run(hrb, total_kv=1400), want, mass)


def test_block_tables_refuse_pages_past_31_bits(hrb):
    table = np.full((1, 4), -1, np.int32)
    free = np.array([(1 << 28) + 3, 5], np.int32)
    got, err = run_tables(hrb, [0], [20], free, 0, table, 16, 20)
    assert err is not None and err.status == capi.HRB_EDATA
    assert (got[1][:16] == -1).all() and np.array_equal(got[1][16:], 80 + np.arange(4))


@pytest.mark.parametrize("hd,rot", [(128, 64), (96, 48), (64, 24), (32, 16)])
def test_qkv_append_partial_half_split_rotation(hrb, hd, rot):
    rng = np.random.default_rng(hd + rot)
    c = ref.Cache(4, 16, 2, hd)
    x = [rng.standard_normal((50, h, hd)).astype(np.float32) for h in (5, 2, 2)]
    table, pos = capi.rope_table(64, rot), rng.integers(0, 64, (1, 50))
    slots = rng.permutation(64)[:50]
    q, got, used, err = run_qkv(hrb, c, x, 5, table=table, pos=pos, rot=rot, sections=(rot // 2,), slots=slots)
    assert err is None
    want = ref.norm_rotate(x[0], None, 0, table, pos, rot, False, (rot // 2,))
    pair = np.abs(x[0]) + np.abs(x[0]).max(-1, keepdims=True)
    assert (np.abs(q - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -19 * pair).all()
    k = ref.norm_rotate(x[1], None, 0, table, pos, rot, False, (rot // 2,))
    for t in range(50):
        check_codes(got.read(slots[t])[0], k[t], exact=False)


def test_attention_extreme_scores(hrb):
    """Scores of thousands (one key takes all), and queries near BF16's ends."""
    rng = np.random.default_rng(12)
    for lens in ([(1, 77), (1, 500)], [(90, 90), (40, 300)]):
        s = Step(rng, lens, 4, 2, 64, 16, q_scale=300.0)
        close(s.run(hrb), *s.want())
        s = Step(rng, lens, 4, 2, 64, 16, q_scale=1e30, scale=1e-30)
        close(s.run(hrb), *s.want())
        s = Step(rng, lens, 4, 2, 64, 16, q_scale=1e-30, scale=1e30)
        close(s.run(hrb), *s.want())
        s = Step(rng, lens, 4, 2, 64, 16, scale=-0.3)
        close(s.run(hrb), *s.want())
        s = Step(rng, lens, 4, 2, 64, 16, scale=0.0)
        close(s.run(hrb), *s.want())


@pytest.mark.parametrize("v_scale", [1e-7, 1e-5, 3000.0])
@pytest.mark.parametrize("lens", [DECODE, [(130, 200), (20, 400)]], ids=["one", "prompt"])
def test_attention_small_and_large_values(hrb, lens, v_scale):
    rng = np.random.default_rng(13)
    s = Step(rng, lens, 4, 2, 128, 16, v_scale=v_scale)
    close(s.run(hrb), *s.want())


@pytest.mark.parametrize("lens", [[(1, 90), (1, 200)], [(100, 150), (30, 400)]])
def test_attention_nan_in_one_row_stays_there(hrb, lens):
    rng = np.random.default_rng(14)
    s = Step(rng, lens, 4, 2, 64, 16)
    s.q[0, 5] = float("nan")
    want, mass = s.want()
    got = s.run(hrb)
    assert np.isnan(got[0, 0]).all()
    got[0, 0], want[0, 0] = 0, 0
    close(got, want, mass)


@pytest.mark.parametrize("lens", [[(1, 90), (1, 200)], [(100, 150), (30, 400)]])
def test_attention_reports_a_page_outside_the_cache(hrb, lens):
    rng = np.random.default_rng(15)
    s = Step(rng, lens, 4, 2, 64, 16)
    table = s.table.copy()
    table[1, 3] = s.pages
    for k in (s.keys, s.values):   # reads as a page of zeros
        k[1][48:64] = 0
    with pytest.raises(capi.HrbError) as e:
        s.run(hrb, table=table)
    assert e.value.status == capi.HRB_EDATA
    torch.cuda.synchronize()
    # The rows are written all the same.
    close(s.out.double().cpu().numpy().reshape(s.rows, s.heads, s.hd), *s.want())


def test_attention_cache_beyond_32_bit_offsets(hrb):
    """A cache of over 4 GiB: the request's pages are its last ones."""
    page, kvh, hd = 256, 8, 128
    pages = (5 << 30) // (page * (hd + hd // 16) * kvh)
    rng = np.random.default_rng(16)
    for q in (1, 100):
        s = Step(rng, [(q, 700)], 16, kvh, hd, page)
        big = torch.zeros(pages, s.cache.stride, dtype=torch.uint8, device="cuda")
        big[-s.pages:] = dev(s.cache.data)
        table = dev(np.where(s.table >= 0, s.table + pages - s.pages, -1).astype(np.int32))
        dq, start, kv = s.q.cuda(), dev(s.start), dev(np.array([700], np.int32))
        out = torch.empty(q, 16 * hd, dtype=torch.bfloat16, device="cuda")
        ready()
        hrb.attention(capi.attn_desc(
            capi.kv_cache(big, pages, page, kvh, hd), 1, 16, q=dq, q_start=start, total_q=q, max_q=q,
            kv_len=kv, max_kv=700, table=table, table_ld=s.ld, scale=s.scale, out=out))
        hrb.sync()
        close(out.double().cpu().numpy().reshape(q, 16, hd), *s.want())
        del big


def test_serving_calls_on_another_stream(hrb):
    rng = np.random.default_rng(17)
    side = torch.cuda.Stream()
    for lens in ([(1, 400), (1, 90)], [(130, 200)]):
        s = Step(rng, lens, 8, 2, 64, 16)
        want, mass = s.want()
        s.run(hrb, stream=side.cuda_stream, sync=False, workspace=True)
        side.synchronize()
        close(s.out.double().cpu().numpy().reshape(s.rows, s.heads, s.hd), want, mass)


def test_a_step_in_a_cuda_graph_follows_the_lengths(hrb):
    """Tables, append and attention captured once, replayed with other
    lengths: everything is read on the device."""
    rng = np.random.default_rng(18)
    heads, kvh, hd, page, n, most = 4, 2, 64, 16, 3, 200
    ld = -(-most // page)
    pages = n * ld
    c = ref.Cache(pages, page, kvh, hd)
    data = dev(c.data)
    cached = torch.zeros(n, dtype=torch.int32, device="cuda")
    fresh = torch.ones(n, dtype=torch.int32, device="cuda")
    free = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0).contiguous()
    heads_at = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
    table = torch.full((n, ld), -1, dtype=torch.int32, device="cuda")
    start, kv = (torch.zeros(m, dtype=torch.int32, device="cuda") for m in (n + 1, n))
    slots, pos = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    x = torch.zeros(n, (heads + 2 * kvh) * hd, device="cuda")
    rope = dev(capi.rope_table(most, hd))
    q = torch.zeros(n, heads * hd, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(q)
    kvc = capi.kv_cache(data, pages, page, kvh, hd)
    b = capi.blocks_desc(n, page, cached=cached, fresh=fresh, free_pages=free, nfree=pages,
                         head_in=heads_at[0], head_out=heads_at[1], table=table, table_ld=ld,
                         q_start=start, kv_len=kv, slots=slots, pos=pos, max_tokens=n)
    ldx = x.shape[1]
    d = capi.qkv_desc(kvc, n, heads, q=x, k=x[:, heads * hd:], v=x[:, (heads + kvh) * hd:], ldq=ldx,
                      ldk=ldx, ldv=ldx, rope=rope, max_pos=most, rot=hd, pos=pos, slots=slots, q_out=q)
    a = capi.attn_desc(kvc, n, heads, q=q, q_start=start, total_q=n, max_q=1, kv_len=kv, max_kv=most,
                       table=table, table_ld=ld, scale=hd ** -0.5, out=out)
    ws = torch.zeros(max(256, hrb.attention_workspace(a)), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    side = torch.cuda.Stream()
    ready()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        at = torch.cuda.current_stream().cuda_stream
        hrb.block_tables(b, stream=at)
        hrb.qkv_append(d, stream=at)
        hrb.attention(a, stream=at)
    keys = [np.zeros((0, kvh, hd))] * n
    values = [np.zeros((0, kvh, hd))] * n
    table_h = capi.rope_table(most, hd)
    for step in range(40):
        xs = rng.standard_normal((n, ldx)).astype(np.float32)
        x.copy_(torch.from_numpy(xs))
        ready()
        graph.replay()
        torch.cuda.synchronize()
        split = np.split(xs.reshape(n, -1, hd), (heads, heads + kvh), 1)
        p = np.full((1, n), step)
        for i in range(n):
            # The cache's own keys (their rounding is test_qkv_append's), then the 64-bit attention.
            s = int(slots[i])
            c.data = data.cpu().numpy()
            k1, v1 = c.read(s)
            keys[i] = np.concatenate((keys[i], k1[None]))
            values[i] = np.concatenate((values[i], v1[None]))
            assert np.array_equal(v1, ref.decode(*ref.encode(split[2][i].astype(np.float64))))
        qs = ref.norm_rotate(split[0], None, 0, table_h, p, hd, False, (hd // 2,))
        assert np.abs(qs - q.double().cpu().numpy().reshape(n, heads, hd)).max() < 0.05
        want, mass = ref.attention(q.double().cpu().numpy().reshape(n, heads, hd),
                                   np.arange(n + 1), [step + 1] * n, keys, values, hd ** -0.5)
        close(out.double().cpu().numpy().reshape(n, heads, hd), want, mass)
        cached += 1
        heads_at[0].copy_(heads_at[1])
    hrb.sync()


def test_refusals(hrb):
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = buf.data_ptr()

    def refused(call, desc, **change):
        for k, v in change.items():
            obj = desc
            if k.startswith("cache_"):
                obj, k = desc.cache, k[6:]
            setattr(obj, k, v)
        with pytest.raises(capi.HrbError) as e:
            call(desc)
        assert e.value.status == capi.HRB_EINVAL and e.value.message

    cache = lambda: capi.kv_cache(p, 4, 16, 2, 64)                       # noqa: E731
    attn = lambda: capi.attn_desc(cache(), 2, 4, q=p, q_start=p, total_q=2, max_q=1, kv_len=p,  # noqa: E731
                                  max_kv=30, table=p, table_ld=2, scale=0.1, out=p)
    for change in (dict(cache_page=24), dict(cache_page=8), dict(cache_page=512), dict(cache_hd=48),
                   dict(cache_hd=160), dict(cache_hd=0), dict(cache_kv_heads=0), dict(cache_kv_heads=3),
                   dict(cache_pages=0), dict(cache_data=None), dict(cache_data=p + 8),
                   dict(cache_page_stride=64), dict(cache_page_stride=2 * 1088 + 8), dict(heads=0),
                   dict(heads=5), dict(seqs=70000), dict(seqs=0), dict(max_q=0), dict(max_q=3),
                   dict(q=None), dict(q=p + 2), dict(ldq=255), dict(ldq=260), dict(q_start=None),
                   dict(q_start=p + 1), dict(kv_len=None), dict(table=None), dict(table_ld=1),
                   dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("inf")),
                   dict(causal=0, window=4), dict(causal=0, prefix=p), dict(out=None), dict(out=p + 4),
                   dict(ldo=128), dict(oq=p), dict(oq=p, oscale=p, ldoq=250),
                   dict(oq=p, oscale=p, oquant=2), dict(workspace=p + 16, workspace_bytes=1 << 16)):
        refused(hrb.attention, attn(), **change)
    qkv = lambda: capi.qkv_desc(cache(), 2, 4, q=p, k=p, v=p, slots=p, q_out=p, rope=p,  # noqa: E731
                                max_pos=8, rot=64, pos=p)
    for change in (dict(cache_hd=40), dict(dtype=2), dict(heads=0), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(rot=12), dict(rot=72), dict(rot=0), dict(axes=0),
                   dict(axes=4), dict(axes=2), dict(rope=p + 4), dict(q=None), dict(v=None),
                   dict(pos=None), dict(slots=None), dict(q_out=None), dict(ldq=200), dict(ldk=100),
                   dict(q=p + 2), dict(q_out=p + 2), dict(ldqo=258), dict(slots=p + 2)):
        refused(hrb.qkv_append, qkv(), **change)
    blocks = lambda: capi.blocks_desc(2, 16, cached=p, fresh=p, free_pages=p, nfree=4, table=p,  # noqa: E731
                                      table_ld=4, q_start=p, kv_len=p, slots=p, max_tokens=4)
    for change in (dict(page=20), dict(seqs=70000), dict(cached=None), dict(fresh=None),
                   dict(table=None), dict(q_start=None), dict(kv_len=None), dict(slots=None),
                   dict(free_pages=None), dict(head_in=p, head_out=p), dict(cached=p + 2)):
        refused(hrb.block_tables, blocks(), **change)
    for args in ((p, 2, p, p, 3), (None, 2, p, p, 0), (p + 2, 2, p, p, 0), (p, 2, p + 8, p, 0)):
        with pytest.raises(capi.HrbError):
            hrb.kv_read(cache(), args[0], args[1], args[2], args[3], dtype=args[4])
    # Nothing to do is not an error.
    d = attn()
    d.total_q, d.max_q = 0, 0
    hrb.attention(d)
    d = qkv()
    d.tokens = 0
    hrb.qkv_append(d)
    hrb.kv_read(cache(), None, 0)
    hrb.sync()
