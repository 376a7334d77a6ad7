"""CPU-only checks of the serving calls' host parts: record sizes, the
rotation table, and the 64-bit reference's own encoding (against a search
over all codes)."""
import numpy as np

import serving_ref as ref
from hotarubi_b200 import capi


def test_record_bytes():
    lib = capi.load()
    for page in (16, 32, 64, 128, 256):
        for hd in (32, 64, 96, 128):
            assert lib.hrb_kv_record_bytes(page, hd) == capi.kv_record_bytes(page, hd)
            assert capi.kv_record_bytes(page, hd) == ref.Cache(1, page, 1, hd).record
            assert capi.kv_record_bytes(page, hd) % 16 == 0


def test_rope_table():
    t = capi.rope_table(50, 8, theta=100.0)
    assert t.shape == (50, 4, 2) and t.dtype == np.float32
    angle = 37 * 100.0 ** (-2 * 3 / 8)
    assert np.allclose(t[37, 3], (np.cos(angle), np.sin(angle)), rtol=0, atol=2 ** -24)


def test_reference_encoding():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((20, 64)) * np.exp2(rng.integers(-30, 30, (20, 1)))
    x[3, :32] = 0
    x[4, 0] = 5 * 2.0 ** 3           # a tie between 4 and 6
    code, scale = ref.encode(x)
    value = ref.decode(code, scale)
    e = scale.astype(int) - 127
    assert e.min() >= -23 and e.max() <= 13
    step = np.repeat(np.exp2(e.astype(float)), 32, -1)
    every = ref.VALUES[:, None, None] * step
    gap = np.abs(np.abs(x) - every).min(0)
    assert np.array_equal(np.abs(np.abs(value) - np.abs(x)), gap)
    assert np.array_equal(ref.decode(*ref.encode(value)), value)


def test_cache_write_read():
    rng = np.random.default_rng(1)
    c = ref.Cache(3, 16, 2, 64)
    k, v = rng.standard_normal((2, 2, 64))
    c.write(37, k, v)
    got = c.read(37)
    assert np.array_equal(got[0], ref.decode(*ref.encode(k)))
    assert np.array_equal(got[1], ref.decode(*ref.encode(v)))
    assert not c.read(36)[0].any() and not c.read(38)[1].any()
