"""attn_paged on values that are not finite: they reach the rows that see their token, in their column, and no others."""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import NAN16, Batch, f64

pytestmark = pytest.mark.gpu

INF, NINF = 0x7F80, 0xFF80


def plant(b, seed, count):
    """`count` values of each sequence and key head made infinite or NaN, a third of them in its new tokens: (sequence, token, key head, column)."""
    r, at = np.random.default_rng(seed), []
    for s, n in enumerate(b.lens):
        v = np.array(b.get("v", s, n))
        for e in range(b.kv_heads):
            for i in range(count):
                t = int(r.integers(max(n - b.news[s], 0), n) if i % 3 == 0 else r.integers(0, n))
                c = int(r.integers(b.dim))
                v[t, e, c] = (INF, NINF, NAN16)[i % 3]
                at.append((s, t, e, c))
        b.put("v", s, 0, v)
    return at


def check(rt, b, at, **how):
    """Finite results against the definition with these values left out; the others are the sum of the infinities and NaN that the row sees."""
    clean = np.array(b.v)
    clean[(clean & 0x7F80) == 0x7F80] = 0
    kept, b.v = b.v, clean
    want, tol = b.exact(**how)
    b.v = kept
    extra = np.zeros_like(want)
    with np.errstate(invalid="ignore"):
        for s, t, e, c in set(at):
            page, slot = b.table[s, t // b.page], t % b.page
            x = f64(np.array([(kept[page, e, slot, c] if b.head_major else kept[page, slot, e, c])]))[0]
            for i in range(b.news[s]):
                pos = b.lens[s] - b.news[s] + i
                w = how.get("window", 0)
                if (t <= pos or not how.get("causal", True)) and not (w and t <= pos - w):
                    extra[int(b.starts[s]) + i if b.starts is not None else s, e * b.group:(e + 1) * b.group, c] += x
    got = f64(b.upload(rt).attend(rt, **how)[:b.live * b.heads * b.dim]).reshape(want.shape)
    hit = ~np.isfinite(extra) | (extra != 0)
    assert hit.any() and not hit.all()
    assert (np.isnan(got) == np.isnan(extra)).all()
    inf = np.isinf(extra)
    assert (got[inf] == extra[inf]).all()
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("lens,news,kvh,g,d,page", [
    ([70, 33, 200], [6, 3, 1], 2, 3, 64, 16), ([40], [8], 1, 4, 128, 100), ([90, 61], [4, 4], 1, 2, 256, 32), ([3000], [5], 2, 2, 128, 64),
    ([150, 260], [150, 70], 2, 4, 128, 16), ([130, 300], [100, 200], 1, 2, 64, 32), ([200, 90], [180, 64], 1, 3, 256, 64),
    ([3000, 500], [90, 120], 2, 2, 128, 64), ([900], [140], 1, 2, 192, 8)])
def test_hidden_from_some_rows(rt, lens, news, kvh, g, d, page, window):
    b = Batch(41, lens, news, kvh, g, d, page)
    check(rt, b, plant(b, 42, 6), window=window)


@pytest.mark.parametrize("new", [1, 7, 80])
def test_outside_the_window_of_all_rows(rt, new):
    b = Batch(43, [500], [new], 2, 2, 128, 16, head_major=True)
    check(rt, b, plant(b, 44, 9), window=100)


@pytest.mark.parametrize("new", [1, 9, 90])
def test_without_causality(rt, new):
    b = Batch(45, [300, 120], [new, new], 1, 2, 64, 16)
    check(rt, b, plant(b, 46, 3), causal=False)


@pytest.mark.parametrize("new", [3, 100])
def test_keys_hidden_from_some_rows(rt, new):
    """A NaN in k of a token makes the scores of the rows that see it NaN, and no others."""
    b = Batch(47, [400], [new], 1, 2, 128, 16)
    t = 400 - new // 2 - 1
    k = np.array(b.get("k", 0, 400))
    k[t, 0, 5] = NAN16
    clean, tol = b.exact()
    b.put("k", 0, 0, k)
    got = f64(b.upload(rt).attend(rt)[:b.q.size]).reshape(clean.shape)
    sees = 400 - new + np.arange(new) >= t
    assert np.isnan(got[sees]).all()
    assert (np.abs(got - clean)[~sees] <= tol[~sees]).all()
