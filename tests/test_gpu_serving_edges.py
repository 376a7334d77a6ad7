"""Edges of the serving calls on the GPU: data and arguments outside what the
calls name, scores and weights near the ends of their types.  Against the
plain 64-bit forms of serving_ref.py, with test_gpu_serving.py's tolerances
unless a test says otherwise."""
import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from hotarubi_b200 import capi  # noqa: E402
from test_gpu_serving import Step, check_codes, close, dev, ready, run_qkv, run_tables  # noqa: E402


def rows_of(s):
    """What a Step's call has written, after an error too."""
    torch.cuda.synchronize()
    return s.out.double().cpu().numpy().reshape(s.rows, s.heads, s.hd)


@pytest.mark.parametrize("entry", ["pages", -1, -2, -(1 << 31)])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("lens", [[(1, 90), (1, 200)], [(100, 150), (30, 400)]], ids=["one", "prompt"])
def test_attention_any_entry_outside_the_cache_reads_as_zeros(hrb, lens, page, entry):
    rng = np.random.default_rng(21)
    s = Step(rng, lens, 4, 2, 64, page)
    table = s.table.copy()
    table[1, 1] = s.pages if entry == "pages" else entry
    for k in (s.keys, s.values):
        k[1][page:2 * page] = 0
    with pytest.raises(capi.HrbError) as e:
        s.run(hrb, table=table)
    assert e.value.status == capi.HRB_EDATA
    close(rows_of(s), *s.want())


def test_attention_more_keys_than_total_kv_says_in_a_split_call(hrb):
    """Scratch for two tiles: the second request's 24, in six chunks, are left
    out, and so are its rows, whatever the chunks' scratch held before."""
    rng = np.random.default_rng(22)
    s = Step(rng, [(40, 100), (200, 3000)], 4, 2, 64, 16)
    want, mass = s.want()
    close(s.run(hrb, total_kv=3100, oq=True), want, mass)   # fills the scratch
    with pytest.raises(capi.HrbError) as e:
        s.run(hrb, total_kv=100, oq=True)
    assert e.value.status == capi.HRB_EDATA
    got = rows_of(s)
    close(got[:40], want[:40], mass[:40])
    assert (got[40:] == 5.0).all()
    assert (s.codes[40:] == 99).all() and (s.scales[40:] == 99).all()


@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_qkv_append_reports_only_what_it_caches(hrb, odd):
    """Rows that pad a step (slot -1) may hold anything."""
    rng = np.random.default_rng(23)
    c = ref.Cache(4, 16, 2, 64)
    x = [rng.standard_normal((9, h, 64)).astype(np.float32) for h in (4, 2, 2)]
    slots = np.array([3, 40, 9, 22, 63, 1, -1, -1, -1])
    for part in x:
        part[6:] = odd
    q, got, used, err = run_qkv(hrb, c, x, 4, slots=slots)
    assert err is None
    for t in range(6):
        assert np.array_equal(got.read(slots[t])[1], ref.decode(*ref.encode(x[2][t].astype(np.float64))))
    x[1][2, 0, 7] = odd
    assert run_qkv(hrb, c, x, 4, slots=slots)[3].status == capi.HRB_EDATA


@pytest.mark.parametrize("sections,bad", [((32,), 0), ((10, 6, 16), 0), ((10, 6, 16), 1),
                                          ((10, 6, 16), 2), ((0, 12, 20), 1), ((32, 0, 0), 0)])
def test_qkv_append_a_position_outside_the_table(hrb, sections, bad):
    """The row keeps its norm, is not rotated on any axis, and nothing is
    cached; positions of axes without pairs do not matter."""
    rng = np.random.default_rng(28)
    tokens = 7
    c = ref.Cache(4, 16, 2, 64)
    x = [rng.standard_normal((tokens, h, 64)).astype(np.float32) for h in (20, 2, 2)]
    w = [(0.5 + rng.random(64)).astype(np.float32) for _ in range(2)]
    table = capi.rope_table(16, 64)
    pos = rng.integers(0, 16, (len(sections), tokens))
    for axis, pairs in enumerate(sections):
        if pairs == 0:
            pos[axis] = 1 << 20
    pos[bad, 3], pos[bad, 5] = 16, -1
    slots = rng.permutation(64)[:tokens]
    q, got, used, err = run_qkv(hrb, c, x, 20, w=w, table=table, pos=pos, rot=64, sections=sections,
                                slots=slots)
    assert err is not None and err.status == capi.HRB_EDATA
    good = np.array([t not in (3, 5) for t in range(tokens)])
    want = ref.norm_rotate(x[0], w[0], 1e-6, None, None, 0, False, ())
    k = ref.norm_rotate(x[1], w[1], 1e-6, None, None, 0, False, ())
    spread = np.abs(want) + np.abs(want).max(-1, keepdims=True)
    inside = np.where((pos >= 0) & (pos < 16), pos, 0)
    want[good] = ref.norm_rotate(x[0], w[0], 1e-6, table, inside, 64, False, sections)[good]
    k[good] = ref.norm_rotate(x[1], w[1], 1e-6, table, inside, 64, False, sections)[good]
    assert (np.abs(q - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -19 * spread).all()
    for t in range(tokens):
        gk, gv = got.read(slots[t])
        if good[t]:
            check_codes(gk, k[t], exact=False)
            check_codes(gv, x[2][t].astype(np.float64), exact=True)
        else:
            assert not gk.any() and not gv.any()


CAPS = [1.0, 30.0, 1e4, 1e6, 1e9, 1e30]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_caps_of_any_size_on_every_last_tile(hrb, cap, hd):
    """Prompts whose last tile of 128 keys holds 1, 64, 65 and 128."""
    rng = np.random.default_rng(24)
    s = Step(rng, [(90, 129), (90, 192), (90, 193), (90, 256), (90, 1)], 4, 2, hd, 16)
    close(s.run(hrb, softcap=cap), *s.want(softcap=cap))


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("hd,page", [(32, 64), (64, 16), (96, 16), (128, 32)])
def test_attention_caps_of_any_size_for_single_tokens(hrb, cap, hd, page):
    rng = np.random.default_rng(25)
    s = Step(rng, [(1, 129), (1, 192), (1, 193), (1, 256), (1, 1), (3, 900)], 4, 2, hd, page)
    close(s.run(hrb, softcap=cap), *s.want(softcap=cap))


@pytest.mark.parametrize("cap", [50.0, 1e4, 1e6, 1e9])
@pytest.mark.parametrize("lens", [[(4, 300)], [(100, 300)]], ids=["few", "prompt"])
def test_attention_a_row_near_the_cap_leaves_the_others_alone(hrb, cap, lens):
    """One row's scores reach the cap, the others' stay small beside it."""
    rng = np.random.default_rng(26)
    s = Step(rng, lens, 4, 2, 64, 16)
    s.q[1] *= cap
    want, mass = s.want(softcap=cap)
    got = s.run(hrb, softcap=cap)
    # FP32 scores as large as the cap are too coarse to compare that row.
    assert np.isfinite(got[1]).all()
    got[1] = want[1]
    close(got, want, mass)


@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1e-30])
@pytest.mark.parametrize("lens", [[(1, 90), (2, 300)], [(100, 200)]], ids=["one", "prompt"])
def test_attention_a_tiny_cap_makes_all_scores_alike(hrb, cap, lens):
    """Products of exactly zero among them."""
    rng = np.random.default_rng(27)
    s = Step(rng, lens, 4, 2, 64, 16)
    s.q[0] = 0.0
    cap = float(np.float32(cap))
    close(s.run(hrb, softcap=cap), *s.want(softcap=cap))


@pytest.mark.parametrize("cap", [1e34, 1e37, 2.9e38])
@pytest.mark.parametrize("lens", [[(1, 90), (2, 300)], [(100, 200)]], ids=["one", "prompt"])
def test_attention_a_cap_near_the_end_of_its_type(hrb, cap, lens):
    rng = np.random.default_rng(31)
    s = Step(rng, lens, 4, 2, 64, 16)
    close(s.run(hrb, softcap=cap), *s.want(softcap=cap))


@pytest.mark.parametrize("lens", [[(1, 3000), (1, 40)], [(60, 200), (9, 70)]], ids=["one", "prompt"])
def test_attention_captured_on_the_contexts_scratch_outlives_larger_calls(hrb, lens):
    """A step captured after a call of its size, a larger call that makes the
    scratch grow, other allocations, and the step's replays."""
    lib = capi.Library()
    rng = np.random.default_rng(32)
    s = Step(rng, lens, 4, 2, 64, 16)
    want = s.want()
    close(s.run(lib), *want)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    lists = [dev(np.asarray(x, np.int32)) for x in (s.start, [kv for _, kv in lens], s.table)]
    out = torch.empty(s.rows, 4 * 64, dtype=torch.bfloat16, device="cuda")
    d = capi.attn_desc(capi.kv_cache(s.dd, s.pages, 16, 2, 64), len(lens), 4, q=s.dq, ldq=s.ldq,
                       q_start=lists[0], total_q=s.rows, max_q=max(q for q, _ in lens),
                       kv_len=lists[1], max_kv=max(kv for _, kv in lens), table=lists[2],
                       table_ld=s.ld, scale=s.scale, out=out)
    ready()
    with torch.cuda.graph(graph, stream=side):
        lib.attention(d, stream=torch.cuda.current_stream().cuda_stream)
    big = Step(rng, [(300, 4000)], 4, 2, 64, 16)
    more = [big]
    for q in (600, 900):   # each larger than all before
        more.append(Step(rng, [(q, 2500 + 10 * q)], 4, 2, 64, 16))
    for b in more:
        close(b.run(lib), *b.want())
        filler = torch.full((1 << 26,), 0xFF, dtype=torch.uint8, device="cuda")
        out.zero_()
        ready()
        graph.replay()
        torch.cuda.synchronize()
        close(out.double().cpu().numpy().reshape(s.rows, 4, 64), *want)
        del filler
    lib.sync()
    del graph
    lib.close()


def test_block_tables_lengths_whose_sums_pass_31_bits(hrb):
    """1200 requests of 2^30 new tokens: the step's slots are the first
    request's, and the sums are held to 2^31 - 1."""
    n, tokens = 1200, 1000
    free = np.random.default_rng(33).permutation(70).astype(np.int32)
    table = np.full((n, 64), -7, np.int32)
    got, err = run_tables(hrb, np.zeros(n), np.full(n, 1 << 30), free, 2, table, 16, tokens)
    assert err is not None and err.status == capi.HRB_EDATA
    t = np.arange(tokens)
    assert np.array_equal(got[1], free[2 + t // 16] * 16 + t % 16) and np.array_equal(got[2], t)
    assert np.array_equal(got[3], np.minimum(np.arange(n + 1) * (1 << 30), 0x7FFFFFFF))
    assert (got[4] == 1 << 30).all()
    table[0, :63] = free[2:65]
    assert np.array_equal(got[0], table)


def test_block_tables_a_length_past_31_bits(hrb):
    table = np.full((3, 4), 5, np.int32)
    got, err = run_tables(hrb, [0, 0x7FFFFFFB, 3], [2, 10, 1], [8, 9], 0, table, 16, 8)
    assert err is not None and err.status == capi.HRB_EDATA
    assert np.array_equal(got[4], [2, 0x7FFFFFFF, 4]) and np.array_equal(got[3], [0, 2, 6, 7])
    assert np.array_equal(got[1], [128, 129, -1, -1, -1, -1, 83, -1])


@pytest.mark.parametrize("long", [(1 << 18) - 1, 1 << 18, 3000000])
def test_block_tables_long_prompts_among_short_ones(hrb, long):
    rng = np.random.default_rng(long)
    fresh = rng.integers(0, 40, 600)
    cached = rng.integers(0, 500, 600)
    fresh[[3, 255, 256, 420]] = long
    table = np.full((600, (long + 500) // 64 + 2), -1, np.int32)
    table[:, :8] = rng.integers(0, 10000, (600, 8))
    need = -(-(cached + fresh) // 64) - -(-cached // 64)
    free = rng.permutation(int(need.sum()) + 9).astype(np.int32)
    start = np.concatenate(([0], np.cumsum(fresh)))
    tokens = int(start[-1]) + 5
    got, err = run_tables(hrb, cached, fresh, free, 4, table, 64, tokens)
    assert err is None
    seq = np.repeat(np.arange(600), fresh)
    pos = np.arange(tokens - 5) - start[seq] + cached[seq]
    base = 4 + np.cumsum(need) - need
    have = -(-cached // 64)
    for i in range(600):
        table[i, have[i]:have[i] + need[i]] = free[base[i]:base[i] + need[i]]
    assert np.array_equal(got[0], table) and np.array_equal(got[3], start)
    assert np.array_equal(got[2], np.concatenate((pos, np.zeros(5, int))))
    assert np.array_equal(got[1], np.concatenate((table[seq, pos // 64] * 64 + pos % 64, [-1] * 5)))
    assert got[5][0] == 4 + need.sum()


def test_block_tables_refuse_an_output_that_is_an_input(hrb):
    """Blocks still read the lists that others would be writing."""
    buf = torch.zeros(16, 64, dtype=torch.int32, device="cuda")
    at = {name: buf[i].data_ptr() for i, name in enumerate(
        ("cached", "fresh", "free_pages", "head_in", "head_out", "table", "q_start", "kv_len", "slots", "pos"))}
    ready()
    for out in ("table", "q_start", "kv_len", "slots", "pos", "head_out"):
        for into in ("cached", "fresh", "free_pages", "head_in"):
            d = capi.blocks_desc(2, 16, nfree=4, table_ld=4, max_tokens=4, **at)
            hrb.block_tables(d)
            setattr(d, out, at[into])
            with pytest.raises(capi.HrbError) as e:
                hrb.block_tables(d)
            assert e.value.status == capi.HRB_EINVAL, (out, into)
    hrb.sync()


def test_attention_single_tokens_over_close_to_2_to_the_31_keys(hrb):
    """One page, seen 2^23 - 2 times, and a last one whose keys' scores stand
    40 over the others': it takes all but 2^-20 of the weights."""
    rng = np.random.default_rng(34)
    page, heads, hd = 256, 4, 32
    kv = (1 << 31) - page
    c = ref.Cache(3, page, 1, hd)
    keys, values = np.zeros((2, page, 1, hd)), rng.standard_normal((2, page, 1, hd))
    keys[:, :, 0, 1:] = rng.standard_normal((2, page, hd - 1))
    keys[1, :, 0, 0] = 6.0
    for p in range(2):
        for t in range(page):
            c.write(p * page + t, keys[p, t], values[p, t])
    read = [c.read(page + t) for t in range(page)]
    q = torch.from_numpy(0.1 * rng.standard_normal((1, heads, hd)).astype(np.float32)).to(torch.bfloat16)
    q[..., 0] = 7.0
    table = torch.zeros(1, kv // page, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    data, dq, start = dev(c.data), q.cuda(), dev(np.array([0, 1], np.int32))
    lens = dev(np.array([kv], np.int32))
    out = torch.empty(1, heads * hd, dtype=torch.bfloat16, device="cuda")
    ready()
    hrb.attention(capi.attn_desc(capi.kv_cache(data, 3, page, 1, hd), 1, heads, q=dq, q_start=start,
                                 total_q=1, max_q=1, kv_len=lens, max_kv=kv, table=table,
                                 table_ld=kv // page, scale=1.0, out=out))
    hrb.sync()
    want, mass = ref.attention(q.double().numpy(), [0, 1], [page], [np.stack([k for k, _ in read])],
                               [np.stack([v for _, v in read])], 1.0)
    close(out.double().cpu().numpy().reshape(1, heads, hd), want, mass)


def test_attention_prompt_with_the_largest_bound_on_keys(hrb):
    """max_kv says 2^31 - 1; the request has 300 keys."""
    rng = np.random.default_rng(35)
    s = Step(rng, [(100, 300)], 2, 1, 32, 256)
    s.ld = 1 << 23
    table = np.full((1, s.ld), -1, np.int32)
    table[0, :2] = s.table[0, :2]
    close(s.run(hrb, table=table, max_kv=0x7FFFFFFF, total_kv=300), *s.want())


@pytest.mark.parametrize("lens", [[(1, 700), (1, 3000)], [(60, 700), (9, 3000)]], ids=["one", "prompt"])
def test_attention_total_kv_past_all_requests_together(hrb, lens):
    rng = np.random.default_rng(36)
    s = Step(rng, lens, 4, 2, 64, 16)
    for total in (6001, 1 << 60, (1 << 64) - 1):
        close(s.run(hrb, total_kv=total, workspace=True), *s.want())


@pytest.mark.parametrize("total", [0, 1 << 40, 1 << 60, (1 << 64) - 1])
def test_attention_refuses_scratch_past_all_memory(hrb, total):
    """300 requests of up to 2^31 - 1 keys: bytes that passed 64 bits came out
    as a few megabytes.  Refused on the host."""
    buf = torch.zeros(1 << 12, dtype=torch.uint8, device="cuda")
    p = buf.data_ptr()
    d = capi.attn_desc(capi.kv_cache(p, 1, 256, 2, 64), 300, 4, q=p, q_start=p, total_q=30000, max_q=100,
                       kv_len=p, max_kv=0x7FFFFFFF, total_kv=total, table=p, table_ld=1 << 23, scale=0.1,
                       out=p)
    for call in (hrb.attention_workspace, hrb.attention):
        with pytest.raises(capi.HrbError) as e:
            call(d)
        assert e.value.status == capi.HRB_ENOMEM and e.value.message


@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens", [[(3, 1), (1, 40)], [(100, 60), (30, 400)]], ids=["few", "prompt"])
def test_attention_nan_in_a_row_without_keys_gives_zeros(hrb, lens, odd):
    rng = np.random.default_rng(30)
    s = Step(rng, lens, 4, 2, 64, 16)
    want, mass = s.want()
    s.q[0, 5] = odd
    assert not mass[0].any()
    close(s.run(hrb), want, mass)


@pytest.mark.parametrize("q", [1, 60])
@pytest.mark.parametrize("drop", [20, 26, 30])
def test_attention_small_weights_beside_a_large_one(hrb, q, drop):
    """One key's score stands `drop` powers of two over all others', whose
    weights are all there is to see: its value is zero, theirs are one.  A
    weight of 2^-30 is still an FP16 number of one significant bit after the
    factor of 2^7 that all weights carry, and the score's FP32 error (30 ln 2
    of 2^-23 each for scale, product and exponent) moves it by 2^-17, so what is
    left is the output's BF16 rounding, 2^-8."""
    rng = np.random.default_rng(29)
    kv = 700
    s = Step(rng, [(q, kv)], 2, 1, 32, 16)
    zero, one = np.zeros((1, 32)), np.ones((1, 32))
    for j in range(kv):
        k = zero.copy()
        k[0, 0] = 4.0 if j == 3 else 0.0
        s.cache.write(int(s.table[0, j // 16]) * 16 + j % 16, k, zero if j == 3 else one)
    s.q[:] = 0.0
    s.q[:, 0] = s.q[:, 32] = 8.0
    s.scale = drop * np.log(2.0) / 32.0
    got = s.run(hrb, causal=False)
    want = (kv - 1) * 2.0 ** -drop / (1 + (kv - 1) * 2.0 ** -drop)
    assert (np.abs(got - want) <= 2.0 ** -8 * want).all()


# ---------------------------------------------------------------------------
# kernels and forms that the dispatch takes by size


def again(s, n):
    """n more requests like a Step's first: its rows, its pages."""
    q = s.lens[0][0]
    s.lens = s.lens + [s.lens[0]] * n
    s.table = np.concatenate((s.table, np.repeat(s.table[:1], n, 0)))
    s.q = torch.cat((s.q, s.q[:q].repeat(n, 1)))
    s.start = np.concatenate((s.start, s.start[-1] + q * np.arange(1, n + 1))).astype(np.int32)
    s.rows = int(s.start[-1])


LONG = {   # requests of more than 1024 keys: two halves of 128 rows a block
    "plain": {}, "open": dict(causal=False), "window": dict(window=300),
    "prefix": dict(window=200, prefix=(300, 0, 2000)), "cap": dict(softcap=4.0),
    "bias": dict(slopes=True), "all": dict(softcap=20.0, slopes=True, window=700, prefix=(130, 1, 0)),
}


@pytest.mark.parametrize("hd,page", [(32, 16), (64, 64), (96, 32), (128, 16)])
@pytest.mark.parametrize("option", LONG)
def test_attention_prompts_over_long_histories(hrb, option, hd, page):
    """Blocks of one and of two halves, several requests, one tile's end."""
    rng = np.random.default_rng(40 + hd)
    s = Step(rng, [(150, 1500), (70, 1153), (129, 129)], 6, 3, hd, page)
    kw = dict(LONG[option])
    if "slopes" in kw:
        kw["slopes"] = (0.05 * rng.random(6)).astype(np.float32)
    ref_kw = dict(kw)
    if "prefix" in kw:
        ref_kw["prefix"] = np.minimum(kw["prefix"], [kv for _, kv in s.lens])
    got = s.run(hrb, **kw)
    close(got, *s.want(**ref_kw))
    assert np.array_equal(got, s.run(hrb, **kw))


@pytest.mark.parametrize("hd,page", [(32, 32), (64, 16), (96, 16), (128, 64)])
@pytest.mark.parametrize("option", LONG)
def test_attention_prompts_over_long_histories_unsplit(hrb, option, hd, page):
    """Enough rows for every SM: a block takes all keys."""
    rng = np.random.default_rng(45 + hd)
    s = Step(rng, [(160, 1100), (90, 1300), (20, 1037)], 16, 8, hd, page)
    kw = dict(LONG[option])
    if "slopes" in kw:
        kw["slopes"] = (0.05 * rng.random(16)).astype(np.float32)
    ref_kw = dict(kw)
    if "prefix" in kw:
        ref_kw["prefix"] = np.minimum(kw["prefix"], [kv for _, kv in s.lens])
        kw["prefix"] = tuple(kw["prefix"]) + (kw["prefix"][0],) * 7
    want, mass = s.want(**ref_kw)
    again(s, 7)
    got = s.run(hrb, **kw)
    close(got[:270], want, mass)
    for i in range(7):
        assert np.array_equal(got[270 + 160 * i:430 + 160 * i], got[:160])


@pytest.mark.parametrize("lens,heads,kvh,hd", [
    ([(5, 1100), (2, 1300)], 8, 1, 128),                 # 40 rows, in chunks of keys
    ([(4, 1200), (4, 1025), (3, 40)], 16, 1, 64),        # 64 rows
    ([(6, 1100), (1, 1500)], 16, 1, 64),                 # 96 rows
    ([(24, 1030), (20, 1200)], 8, 2, 32),                # 96 rows of two heads
    ([(16, 1040), (9, 1028)], 6, 2, 96),                 # 48 rows
    ([(8, 1030)] * 90, 32, 8, 32),                       # 32 rows, one chunk
    ([(16, 1030)] * 48, 32, 8, 32),                      # 64 rows, one chunk
])
@pytest.mark.parametrize("option", ["plain", "all"])
def test_attention_rows_in_blocks_over_long_histories(hrb, lens, heads, kvh, hd, option):
    rng = np.random.default_rng(len(lens) + hd)
    few = lens[:3]
    s = Step(rng, few, heads, kvh, hd, 16)
    kw = {}
    if option == "all":
        kw = dict(softcap=20.0, slopes=(0.05 * rng.random(heads)).astype(np.float32), window=700,
                  prefix=(130, 1, 0)[:len(few)])
    ref_kw = dict(kw)
    if "prefix" in kw:
        ref_kw["prefix"] = np.minimum(kw["prefix"], [kv for _, kv in few])
    want, mass = s.want(**ref_kw)
    n, q = len(lens) - len(few), few[0][0]
    again(s, n)
    if "prefix" in kw:
        kw["prefix"] = tuple(kw["prefix"]) + (kw["prefix"][0],) * n
    got = s.run(hrb, **kw)
    rows = len(want)
    close(got[:rows], want, mass)
    for i in range(n):
        close(got[rows + i * q:rows + (i + 1) * q], want[:q], mass[:q])


@pytest.mark.parametrize("hd,page", [(32, 64), (96, 64), (128, 64), (128, 16)])
@pytest.mark.parametrize("lens", [[(1, 90), (1, 700)], [(3, 130), (2, 300)], [(90, 200), (33, 257)]],
                         ids=["one", "few", "prompt"])
@pytest.mark.parametrize("option", [dict(softcap=3.0), dict(slopes=True),
                                    dict(softcap=300.0, slopes=True, window=50)], ids=str)
def test_attention_shaped_scores_at_every_head_size(hrb, option, lens, hd, page):
    rng = np.random.default_rng(50 + hd)
    s = Step(rng, lens, 6, 2, hd, page)
    kw = dict(option)
    if "slopes" in kw:
        kw["slopes"] = (0.1 * rng.random(6)).astype(np.float32)
    close(s.run(hrb, **kw), *s.want(**kw))


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_attention_mxint8_copy_of_joined_and_two_half_rows(hrb, hd):
    """The MXINT8 copy alone and beside BF16 rows, within half a step of the
    64-bit value."""
    rng = np.random.default_rng(60 + hd)
    for lens in ([(1, 3000), (1, 2049)], [(140, 1500), (100, 1100)]):
        s = Step(rng, lens, 4, 2, hd, 16)
        want, mass = s.want()
        for out in (True, False):
            s.run(hrb, oq=True, out=out)
            codes, scales = s.codes.cpu().numpy()[:, :4 * hd], s.scales.cpu().numpy()[:, :hd // 8]
            step = np.repeat(np.exp2(scales.astype(np.float64) - 133), 32, 1).reshape(want.shape)
            value = codes.reshape(want.shape) * step
            tol = 0.5 * step + 2.0 ** -9 * mass + np.where(np.abs(codes.reshape(want.shape)) == 127, step, 0)
            assert (np.abs(value - want) <= tol).all()


@pytest.mark.parametrize("power", [10, 19, 20, 24, 27, 28, 30, 40, 100])
@pytest.mark.parametrize("lens", [[(1, 300), (3, 700)], [(90, 300)], [(70, 1200)]], ids=["few", "prompt", "long"])
@pytest.mark.parametrize("form", ["plain", "cap", "bias"])
def test_attention_equal_scores_of_any_size(hrb, lens, power, form):
    """Scores are 0, 4 or 6 times 2^power, without rounding: the keys of 6
    share all the weight (the others' is under 2^-1000).  Left is the output's
    BF16 rounding, 2^-8, and the weights' FP16 rounding, 2^-11 of the values."""
    rng = np.random.default_rng(70)
    s = Step(rng, lens, 2, 1, 32, 16)
    s.q[:] = 0.0
    s.q[:, 0] = s.q[:, 32] = 2.0 ** power
    s.scale = 1.0
    for n, (_, kv) in enumerate(lens):
        big = rng.random(kv)
        for j in range(kv):
            key = np.zeros((1, 32))
            key[0, 0] = 6.0 if big[j] < 0.1 or j == kv // 2 else rng.choice((0.0, 4.0))
            s.cache.write(int(s.table[n, j // 16]) * 16 + j % 16, key, s.values[n][j])
            s.keys[n][j] = key
    want, mass = s.want(causal=False)
    kw = {"plain": {}, "cap": dict(softcap=2e38), "bias": dict(slopes=np.zeros(2, np.float32))}[form]
    got = s.run(hrb, causal=False, **kw)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -11 * mass).all()
