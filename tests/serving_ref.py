"""Plain 64-bit forms of the serving calls (hrb_gemm.h section 11), written
from their formulas: the 4-bit cache's encoding and records, norm and
rotation, block tables, attention."""
import numpy as np

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
E_MIN, E_MAX = -23, 13


def encode(x):
    """x [..., 32 n] -> codes [..., 32 n], scale bytes [..., n]: the nearest
    E2M1 value of x / 2^e, ties to the even code."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(b).max(-1)
    e = np.full(top.shape, E_MIN)
    e[top > 0] = np.clip(np.frexp(top[top > 0])[1] - 3, E_MIN, E_MAX)
    u = np.abs(b) / np.exp2(e)[..., None]
    gap = np.abs(u[..., None] - VALUES)
    near = gap == gap.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1)) | ((b < 0) * 8)
    return code.reshape(x.shape).astype(np.uint8), (e + 127).astype(np.uint8)


def decode(code, scale):
    v = np.where(code & 8, -1.0, 1.0) * VALUES[code & 7]
    e = np.clip(scale.astype(np.int64) - 127, E_MIN, E_MAX)
    return v * np.repeat(np.exp2(e.astype(np.float64)), 32, -1)


class Cache:
    """A cache in host memory: data [pages][stride], records as documented."""

    def __init__(self, pages, page, kv_heads, hd, rng=None, extra=0):
        self.pages, self.page, self.kv_heads, self.hd = pages, page, kv_heads, hd
        self.record = page * (hd + hd // 16)
        self.stride = kv_heads * self.record + extra
        self.data = (np.zeros((pages, self.stride), np.uint8) if rng is None
                     else rng.integers(0, 256, (pages, self.stride), dtype=np.uint8))

    def _parts(self, p, h):
        r = self.data[p, h * self.record:(h + 1) * self.record]
        w, z = self.page * self.hd // 2, self.page * self.hd // 32
        return [r[:w].reshape(self.page, -1), r[w:w + z].reshape(self.page, -1),
                r[w + z:2 * w + z].reshape(self.page, -1), r[2 * w + z:].reshape(self.page, -1)]

    def write(self, slot, k, v):
        """k, v [kv_heads][hd] at a slot."""
        for h in range(self.kv_heads):
            parts = self._parts(slot // self.page, h)
            for i, x in ((0, k), (2, v)):
                code, scale = encode(x[h])
                parts[i][slot % self.page] = code[0::2] | (code[1::2] << 4)
                parts[i + 1][slot % self.page] = scale

    def read(self, slot):
        """(k, v) [kv_heads][hd] of a slot."""
        out = ([], [])
        for h in range(self.kv_heads):
            parts = self._parts(slot // self.page, h)
            for i, o in ((0, out[0]), (2, out[1])):
                b = parts[i][slot % self.page]
                code = np.stack((b & 15, b >> 4), -1).reshape(-1)
                o.append(decode(code, parts[i + 1][slot % self.page]))
        return np.stack(out[0]), np.stack(out[1])


def norm_rotate(x, w, eps, table, pos, rot, interleaved, sections):
    """x [tokens][heads][hd] -> the same, normed (w not None) and rotated;
    pos [axes][tokens], table [max_pos][rot / 2][2] or None."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    if table is None:
        return x
    out = x.copy()
    axis = np.repeat(np.arange(len(sections)), sections)
    for p in range(rot // 2):
        a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + rot // 2)
        c, s = (table[pos[axis[p]], p, i].astype(np.float64)[:, None] for i in (0, 1))
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def attention(q, q_start, kv_len, keys, values, scale, causal=True, window=0, prefix=None,
              softcap=0.0, slopes=None):
    """q [rows][heads][hd]; keys and values: one [kv][kv_heads][hd] a request.
    Returns the output and its error scale: sum_j p_j |v_j|, what relative
    roundings of the weights p scale with, plus 2^-16 sum_j |v_j| (FP16 weights
    end at 2^-24, half a step of which is 2^-9 of this term)."""
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    heads = q.shape[1]
    for n, kv in enumerate(kv_len):
        a, b = q_start[n], q_start[n + 1]
        if a == b or kv == 0:
            continue
        i = (kv - (b - a) + np.arange(b - a))[:, None]
        j = np.arange(kv)[None]
        seen = np.ones((b - a, kv), bool)
        if causal:
            seen = j <= i
            if window:
                seen &= j > i - window
            if prefix is not None:
                seen |= j < prefix[n]
        for h in range(heads):
            g = h // (heads // keys[n].shape[1])
            s = scale * (q[a:b, h].astype(np.float64) @ keys[n][:, g].T)
            if softcap:
                s = softcap * np.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * np.abs(i - j)
            s = np.where(seen, s, -np.inf)
            top = s.max(-1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(top), top, 0))
            l = p.sum(-1, keepdims=True)
            p = np.divide(p, l, out=np.zeros_like(p), where=l > 0)
            out[a:b, h] = p @ values[n][:, g]
            mass[a:b, h] = (p + 2.0 ** -16 * seen) @ np.abs(values[n][:, g])
    return out, mass


def block_tables(cached, fresh, free, head, table, page, max_tokens):
    table = table.copy()
    slots, pos = np.full(max_tokens, -1), np.zeros(max_tokens, int)
    start, at = [0], head
    for i, (c, f) in enumerate(zip(cached, fresh)):
        c, f = max(int(c), 0), max(int(f), 0)
        for r in range(f):
            p, t = c + r, start[-1] + r
            n = p // page
            if p % page == 0:
                got = int(free[at]) if at < len(free) else -1
                at += 1
                if t < max_tokens and n < table.shape[1]:
                    table[i, n] = got
            if t < max_tokens:
                pos[t] = p
                if n < table.shape[1] and table[i, n] >= 0:
                    slots[t] = table[i, n] * page + p % page
        start.append(start[-1] + f)
    kv_len = np.maximum(cached, 0) + np.maximum(fresh, 0)
    return table, slots, pos, np.array(start), kv_len, at
