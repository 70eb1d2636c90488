"""attn_paged over long cuts, counted: queries of zero give every key the same weight, and the values say in which column a key counts, so a
row of the result is the number of keys of each column over the number of all. Keys that are left out, or taken twice, are seen where random
values would hide them in the mean of thousands. (A dropped unit of 64 keys of 40000 changes a column by a tenth, dropped 16 by 2.6 %; the
tolerance is 0.4 %.)"""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import SENTINEL16, U16, U32, Batch, bf16, f64

STEP = 16  # keys that count in one column: the fewest that a kernel takes at a time

# lens, news, kv heads, group, dim, page, head major, window
BATCHES = [
    ([40000], [1], 1, 1, 64, 64, False, 0),       # an item, a part for each block
    ([30000], [16], 1, 16, 64, 64, True, 0),      # 256 rows, a part for each block: tiles
    ([20000], [64], 1, 2, 256, 128, False, 0),    # 128 rows of wide heads
    ([15000], [30], 1, 1, 128, 16, False, 0),     # two items of few rows
    ([9000], [1], 2, 2, 64, 16, False, 0),
    ([12000], [3], 1, 4, 128, 10, True, 0),       # pages that come by rows
    ([3000], [1], 8, 4, 128, 16, False, 0),
    ([2000, 2000], [1, 1], 8, 2, 64, 32, False, 0), ([1500] * 5, [1] * 5, 3, 1, 256, 16, False, 0),  # items of the same length
    ([640] * 37, [1] * 37, 4, 2, 128, 16, False, 0),
    ([20000, 300, 7000], [1, 1, 1], 4, 2, 192, 64, False, 0),
    ([20000, 300, 7000], [90, 300, 40], 2, 2, 128, 32, True, 0),
    ([9000, 4000], [200, 100], 2, 4, 96, 64, False, 0),
    ([9000], [700], 1, 1, 256, 64, True, 0),
    ([20000, 9000], [1, 2], 2, 4, 128, 64, False, 6000), ([20000, 9000], [150, 90], 1, 4, 64, 64, False, 6000),
]


def column(t, head, dim):
    return (t // STEP + 5 * head) % dim


def batch(case):
    lens, news, kvh, g, d, page, major, _ = BATCHES[case]
    b = Batch(300 + case, lens, news, kvh, g, d, page, major)
    b.q[:] = 0
    for s, n in enumerate(lens):
        v = np.zeros((n, kvh, d), np.float32)
        for e in range(kvh):
            v[np.arange(n), e, column(np.arange(n), e, d)] = 1.0
        b.put("v", s, 0, bf16(v))
    return b


def shares(length, pos, window, head, dim, times=None):
    """What a row at position `pos` sees of each column; `times`: how often each key counts."""
    t = np.arange(max(0, pos + 1 - window) if window else 0, min(pos + 1, length))
    w = np.ones(len(t)) if times is None else times[t]
    return np.bincount(column(t, head, dim), weights=w, minlength=dim) / max(w.sum(), 1.0)


def tolerance(want):
    """The rounding of the result, and U32 for each of at most 300 parts, the quotient and the product. Weights are 1 and counts below
    2^24: all sums of them are exact, columns without keys are zeros."""
    return want * (U16 * (1 + U16) + 310 * U32)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(BATCHES)))
def test_every_key_counts_once(rt, case):  # noqa: F811
    b, window = batch(case).upload(rt), BATCHES[case][-1]
    got = b.attend(rt, window=window)
    assert (got[b.q.size:] == SENTINEL16).all()
    g = f64(got[:b.q.size]).reshape(b.total, b.heads, b.dim)
    row = 0
    for s, n in enumerate(b.lens):
        for i in range(b.news[s]):
            for e in range(b.kv_heads):
                want = shares(n, n - b.news[s] + i, window, e, b.dim)
                off = np.abs(g[row, e * b.group:(e + 1) * b.group] - want)
                assert (off <= tolerance(want)).all(), (s, i, e, np.argwhere(off > tolerance(want))[:4])
            row += 1


@pytest.mark.parametrize("case", range(len(BATCHES)))
def test_a_step_left_out_or_taken_twice_is_outside(case):
    """The same tolerance against results that have it wrong: one step of keys, or a part's border off by one step."""
    lens, news, kvh, _, d, _, _, window = BATCHES[case]
    r = np.random.default_rng(case)
    for s, n in enumerate(lens[:3]):
        pos = n - 1
        first = max(0, pos + 1 - window) if window else 0
        want = shares(n, pos, window, 0, d)
        for _ in range(12):
            u = int(r.integers(-(-first // STEP), n // STEP))
            for factor in (0.0, 2.0):
                times = np.ones(n)
                times[u * STEP:(u + 1) * STEP] = factor
                wrong = f64(bf16(shares(n, pos, window, 0, d, times)))
                assert (np.abs(wrong - want) > tolerance(want)).any(), (s, u, factor)
