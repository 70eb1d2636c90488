"""Ragged batches over a paged cache for the tests of rope, kv_append_paged and attn_paged, and their definitions in 64 bits."""
import numpy as np

from tessl_b200 import nn, synth

U16, U32 = 2.0 ** -8, 2.0 ** -24  # half a step of bf16 and of f32, relative


def bf16(a):
    return synth.f32_to_bf16_bits(np.asarray(a, np.float32))


def f64(bits):
    return synth.bf16_bits_to_f32(np.asarray(bits, np.uint16)).astype(np.float64)


NAN16 = 0x7FC1
SENTINEL16 = 0x4B4D


class Batch:
    """`lens` tokens of each sequence, the last `news` of them new. Pages are dealt in a shuffled order; every slot that no token
    has, and every page that no sequence has, holds NaN; table entries past a sequence's pages are ids outside the cache."""

    def __init__(self, seed, lens, news, kv_heads, group, dim, page, head_major=False, spare=3, std=1.0, starts=True, tail=0):
        r = self.rng = np.random.default_rng(seed)
        self.lens, self.news, self.kv_heads, self.group, self.dim, self.page = lens, news, kv_heads, group, dim, page
        self.heads, self.head_major, self.n = kv_heads * group, head_major, len(lens)
        need = [-(-max(n, 0) // page) for n in lens]
        self.pages, self.width = sum(need) + spare, max(need + [1]) + 1
        order = r.permutation(self.pages).astype(np.int32)
        self.table = r.choice(np.array([-1, self.pages, 2**31 - 1, -2**31], np.int32), (self.n, self.width))
        at = 0
        for s, c in enumerate(need):
            self.table[s, :c] = order[at:at + c]
            at += c
        self.starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32) if starts else None
        self.live = int(sum(news))
        self.total = self.live + tail  # rows behind the last sequence
        shape = (self.pages, kv_heads, page, dim) if head_major else (self.pages, page, kv_heads, dim)
        self.k, self.v = np.full(shape, NAN16, np.uint16), np.full(shape, NAN16, np.uint16)
        for s in range(self.n):
            for name in ("k", "v"):
                self.put(name, s, 0, bf16(r.standard_normal((max(lens[s], 0), kv_heads, dim)) * (std if name == "k" else 1.0)))
        self.q = bf16(r.standard_normal((self.total, self.heads, dim)) * std)

    def slots(self, s, first, last):
        t = np.arange(first, last)
        return self.table[s, t // self.page], t % self.page

    def put(self, name, s, first, rows):
        page, slot = self.slots(s, first, first + len(rows))
        if self.head_major:
            getattr(self, name)[page, :, slot] = rows
        else:
            getattr(self, name)[page, slot] = rows

    def get(self, name, s, last):
        page, slot = self.slots(s, 0, last)
        a = getattr(self, name)
        return a[page, :, slot] if self.head_major else a[page, slot]

    def upload(self, rt):
        self.b_k, self.b_v, self.b_q = rt.buffer_from(self.k), rt.buffer_from(self.v), rt.buffer_from(self.q)
        self.cache = nn.PagedKv(self.b_k, self.b_v, self.pages, self.page, self.kv_heads, self.dim,
                                nn.KV_HEAD_MAJOR if self.head_major else nn.KV_TOKEN_MAJOR)
        self.seqs = nn.PagedSeqs(rt.buffer_from(self.table), rt.buffer_from(np.array(self.lens, np.int32)),
                                 None if self.starts is None else rt.buffer_from(self.starts), self.n, self.width)
        self.out = rt.buffer_from(np.full(self.q.size + 64, SENTINEL16, np.uint16))
        return self

    def attend(self, rt, scale=None, causal=True, window=0, work=None):
        scale = self.dim ** -0.5 if scale is None else scale
        if work is None:
            work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, self.total, self.heads, self.cache, self.seqs))
            work.write(np.full(work.nbytes // 4, np.nan, np.float32))
        out = self.out.view(0, self.q.size * 2)
        nn.attn_paged(rt, self.b_q, self.cache, self.seqs, out, work, self.total, self.heads, scale, causal, window)
        rt.synchronize()
        return self.out.read(np.uint16, self.q.size + 64)

    def exact(self, scale=None, causal=True, window=0, holes=()):
        """(out, tolerance) f64 [live, heads, dim]. `holes`: (sequence, column) of table entries that point outside.

        Tolerance: the result's rounding to bf16 (U16 of it); the weights' rounding to bf16 (U16 of sum p |v| / sum p); a score is a sum
        of dim products in f32 and one multiplication (each step off by U32 of the sum of magnitudes, twice that for a sum that
        truncates), an error of a weight's exponent and so a relative one of the weight, which counts in the sum and in the divisor; the
        exponential (2^-21, in both) and the f32 sums over the keys and the parts (U32 a step)."""
        scale = self.dim ** -0.5 if scale is None else scale
        out, tol = np.zeros((self.live, self.heads, self.dim)), np.zeros((self.live, self.heads, self.dim))
        for s in range(self.n):
            n = min(max(self.lens[s], 0), self.width * self.page)
            row0 = int(self.starts[s]) if self.starts is not None else s
            if n == 0 or self.news[s] == 0:
                continue
            t = np.arange(n)
            there = ~np.isin(t // self.page, [c for (i, c) in holes if i == s])
            page, slot = self.table[s, t // self.page].copy(), t % self.page
            page[~there] = 0
            k, v = (f64(a[page, :, slot] if self.head_major else a[page, slot]) for a in (self.k, self.v))
            k[~there], v[~there] = 0.0, 0.0
            pos = self.lens[s] - self.news[s] + np.arange(self.news[s])
            seen = there[None, :] & ((t[None, :] <= pos[:, None]) if causal else np.ones((self.news[s], n), bool))
            if window:
                seen &= t[None, :] > pos[:, None] - window
            for h in range(self.heads):
                q = f64(self.q[row0:row0 + self.news[s], h])
                e = h // self.group
                z = np.where(seen, scale * (q @ k[:, e].T), -np.inf)
                top = z.max(axis=1, keepdims=True)
                w = np.where(seen, np.exp(z - np.where(np.isfinite(top), top, 0.0)), 0.0)
                den = w.sum(axis=1, keepdims=True)
                den[den == 0] = 1.0
                o, a = (w @ v[:, e]) / den, (w @ np.abs(v[:, e])) / den
                mag = np.where(seen, abs(scale) * (np.abs(q) @ np.abs(k[:, e]).T), 0.0).max(axis=1, keepdims=True)
                off = 2 * (self.dim + 8) * 2 * U32 * mag + 2 * 2.0 ** -21 + (n + 64) * 2 * U32
                out[row0:row0 + self.news[s], h] = o
                tol[row0:row0 + self.news[s], h] = U16 * np.abs(o) * (1 + U16) + (U16 + off) * a * (1 + U16) + 1e-30
        return out, tol

    def check(self, got, what="", **how):
        want, tol = self.exact(**how)
        live = self.live * self.heads * self.dim
        assert (got[live:] == SENTINEL16).all(), f"{what}: rows that belong to no sequence were written"
        g = f64(got[:live]).reshape(want.shape)
        bad = ~(np.abs(g - want) <= tol)
        assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} outside, first at {np.argwhere(bad)[0]}: got {g[bad][0]}, want "
                               f"{want[bad][0]} +- {tol[bad][0]}")


def turn(x, positions, rot, theta, interleaved, factor=1.0, w=None):
    """x f64 [tokens, heads, dim], the first `rot` columns turned."""
    if rot == 0:
        return x.copy()
    if w is None:
        w = theta ** (-2.0 * np.arange(rot // 2) / rot)
    angle = np.asarray(positions, np.float64)[:, None] * w
    z = factor * np.exp(1j * angle)[:, None, :]
    y = x.copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    r = (x[..., a] + 1j * x[..., b]) * z
    y[..., a], y[..., b] = r.real, r.imag
    return y


def turn_size(x, rot, interleaved, factor=1.0):
    """Per value: the magnitudes that its turn adds up."""
    y = np.abs(x)
    if rot == 0:
        return y
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    s = factor * (np.abs(x[..., a]) + np.abs(x[..., b]))
    y = y.copy()
    y[..., a], y[..., b] = s, s
    return y


def normed(x, w, eps):
    return x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * (1.0 + w)
