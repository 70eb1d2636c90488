"""Offsets and lengths that point outside: what is left of them after they are cut to the call's rows is done as if it had been given, and
nothing else is read or written. Descending offsets: attention does nothing, an append at most what one of the sequences asks for."""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import SENTINEL16, Batch, bf16, f64
from tessl_b200 import nn

pytestmark = pytest.mark.gpu

FAR = 2 ** 31 - 1
# offsets as given and as they count, in sixths of the call's rows (FAR: as it is)
OFFSETS = [([0, 2, FAR, 6], [0, 2, 6, 6]), ([-5, 2, 4, 6], [0, 2, 4, 6]), ([0, 2, 4, FAR], [0, 2, 4, 6]), ([-5, -3, -1, 0], [0, 0, 0, 0]),
           ([FAR, FAR, FAR, FAR], [6, 6, 6, 6]), ([2, 2, 5, 5], [2, 2, 5, 5]), ([0, 0, 0, 6], [0, 0, 0, 6]), ([0, 6, 6, 6], [0, 6, 6, 6])]
# one offset behind its successor at least
DESCENDING = [[0, 2, 1, 6], [0, 4, 2, 0], [6, 0, 6, 0], [FAR, 0, 0, 0], [0, 0, 6, -5]]
LENGTHS = [[30, 48, 50], [-3, -2 ** 31, FAR], [FAR, 0, 17], [0, 0, 0], [64, 1, 4]]


def batch(rt, third, dim, lens=(64, 64, 64), major=False):
    """Three sequences of `third` new tokens and four full pages each: every slot that a length can reach holds a token."""
    b = Batch(501, list(lens), [third] * 3, 2, 2, dim, 16, major)
    b.table, b.width = np.ascontiguousarray(b.table[:, :4]), 4
    return b.upload(rt)


def scaled(offsets, third):
    """Sixths of the call's rows in rows."""
    return [o if abs(o) > 6 else o * third // 2 for o in offsets]


def given(rt, b, starts=None, lens=None):
    b.seqs = nn.PagedSeqs(b.seqs.page_table, b.seqs.kv_lens if lens is None else rt.buffer_from(np.array(lens, np.int32)),
                          b.seqs.q_starts if starts is None else rt.buffer_from(np.array(starts, np.int32)), 3, 4)


def check(rt, b, got, starts, lens):
    """Rows of starts[s] .. starts[s + 1] by the definition, all others as they were; nothing else has changed."""
    b.starts, b.lens, b.news = np.array(starts, np.int32), list(lens), [int(n) for n in np.diff(starts)]
    want, tol = b.exact()
    rows = got[:b.q.size].reshape(b.total, b.heads, b.dim)
    mine = np.zeros(b.total, bool)
    mine[starts[0]:starts[3]] = True
    assert (rows[~mine] == SENTINEL16).all(), "rows of no sequence were written"
    assert (np.abs(f64(rows[mine]) - want[mine]) <= tol[mine]).all()
    unchanged(rt, b, got)


def unchanged(rt, b, got):
    assert (got[b.q.size:] == SENTINEL16).all(), "behind the output something was written"
    for buf, was in ((b.b_k, b.k), (b.b_v, b.v), (b.b_q, b.q)):
        assert np.array_equal(buf.read(np.uint16, was.size), was.reshape(-1))
    assert np.array_equal(b.seqs.page_table.read(np.int32, b.table.size), b.table.reshape(-1))
    assert not rt.is_poisoned()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("third", [2, 50])
@pytest.mark.parametrize("offsets,counted", OFFSETS)
def test_offsets_are_cut_to_the_rows(rt, offsets, counted, third, dim):
    b = batch(rt, third, dim)
    given(rt, b, scaled(offsets, third))
    check(rt, b, b.attend(rt), scaled(counted, third), b.lens)


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("third", [2, 50])
@pytest.mark.parametrize("offsets", DESCENDING)
def test_descending_offsets_do_nothing(rt, offsets, third, dim):
    b = batch(rt, third, dim)
    given(rt, b, scaled(offsets, third))
    got = b.attend(rt)
    assert (got == SENTINEL16).all()
    unchanged(rt, b, got)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("third", [2, 50])
@pytest.mark.parametrize("lens", LENGTHS)
def test_lengths_are_cut_to_the_table(rt, lens, third, dim):
    b = batch(rt, third, dim)
    given(rt, b, lens=lens)
    check(rt, b, b.attend(rt), b.starts, lens)


@pytest.mark.parametrize("major", [False, True])
@pytest.mark.parametrize("offsets,counted", OFFSETS + [(o, None) for o in DESCENDING])
@pytest.mark.parametrize("lens", LENGTHS)
def test_an_append_stays_inside(rt, lens, offsets, counted, major):
    """Values as they are, without turn and norm: each slot holds what was there, or the row that belongs there, bit by bit."""
    third, dim = 4, 64
    b = batch(rt, third, dim, major=major)
    starts = scaled(offsets, third)
    given(rt, b, starts, lens)
    r = np.random.default_rng(7)
    new = {n: bf16(r.standard_normal((b.total, h, dim))) for n, h in (("q", b.heads), ("k", 2), ("v", 2))}
    bufs = {n: rt.buffer_from(a) for n, a in new.items()}
    nn.kv_append_paged(rt, bufs["q"], bufs["k"], bufs["v"], b.out.view(0, b.q.size * 2), b.cache, b.seqs, None, None, b.total, b.heads, in_as_bf16=True)
    rt.synchronize()
    got = b.out.read(np.uint16, b.q.size + 64)
    cut = [min(max(s, 0), b.total) for s in starts]
    assert counted is None or cut == scaled(counted, third)
    places = {}  # slot -> the row that goes there; of descending offsets: that may
    may = np.zeros(b.total, bool)
    for s in range(3):
        for row in range(cut[s], cut[s + 1]):
            may[row] = True
            pos = max(lens[s], 0) - (cut[s + 1] - row)
            if 0 <= pos < 64:
                places.setdefault((s, pos), row)
    rows = got[:b.q.size].reshape(b.total, -1)
    put = (rows == new["q"].reshape(b.total, -1)).all(axis=1)
    assert (put | (rows == SENTINEL16).all(axis=1)).all() and not put[~may].any() and (counted is None or put[may].all())
    want = {n: getattr(b, n).copy() for n in "kv"}
    for name, buf in (("k", b.b_k), ("v", b.b_v)):
        after = buf.read(np.uint16, b.k.size).reshape(b.k.shape)
        for (s, pos), row in places.items():
            at = (b.table[s, pos // 16], slice(None), pos % 16) if major else (b.table[s, pos // 16], pos % 16)
            if counted is not None or np.array_equal(after[at], new[name][row]):
                want[name][at] = new[name][row]
        assert np.array_equal(after, want[name]), name
    assert (got[b.q.size:] == SENTINEL16).all() and not rt.is_poisoned()
    for n, a in new.items():
        assert np.array_equal(bufs[n].read(np.uint16, a.size), a.reshape(-1))
