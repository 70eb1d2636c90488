"""attn_paged against its definition in 64 bits: head layouts, lengths from none to long, windows, masks that leave rows empty, pages
that end anywhere, ids and lengths that point outside, NaN wherever no token is, parts of a key range in several blocks."""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import NAN16, SENTINEL16, Batch, bf16
from tessl_b200 import nn

pytestmark = pytest.mark.gpu


# lens, news, kv heads, group, dim, page, head major
SHAPES = [
    ([1], [1], 1, 1, 64, 16, False),
    ([1, 2, 17, 64, 65], [1] * 5, 2, 4, 128, 16, False),
    ([777], [1], 8, 4, 128, 16, True),
    ([2049, 3, 700], [1] * 3, 4, 4, 256, 64, True),
    ([4000], [1], 1, 8, 128, 64, False),
    ([515, 1030], [1, 1], 3, 5, 96, 48, False),
    ([100, 333], [1, 1], 2, 1, 192, 1, False),
    ([90, 41], [1, 1], 2, 3, 8, 7, True),
    ([70, 200, 31], [1, 1, 1], 1, 20, 72, 256, False),
    ([70, 0, 200, 5], [3, 0, 7, 5], 2, 4, 128, 32, True),
    ([300, 129, 64], [129, 129, 64], 2, 4, 128, 16, False),
    ([260, 1000], [260, 77], 1, 7, 64, 24, True),
    ([131, 400], [131, 200], 2, 2, 256, 128, False),
    ([200, 90], [33, 90], 1, 3, 160, 16, True),
    ([300], [300], 1, 1, 40, 10, False),
    ([9000], [1], 2, 2, 64, 16, False),
    ([5000, 100], [40, 100], 2, 6, 128, 64, True),
]


@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_against_the_definition(rt, case):
    lens, news, kvh, g, d, page, hm = SHAPES[case]
    b = Batch(100 + case, lens, news, kvh, g, d, page, hm, tail=2).upload(rt)
    b.check(b.attend(rt), SHAPES[case])


@pytest.mark.parametrize("window", [1, 2, 16, 63, 100, 5000])
@pytest.mark.parametrize("lens,news,kvh,g,d", [([400, 90, 1], [1, 1, 1], 2, 4, 128), ([400, 90], [200, 90], 1, 3, 64),
                                               ([300], [170], 1, 2, 256)])
def test_a_window(rt, lens, news, kvh, g, d, window):
    b = Batch(31 + window, lens, news, kvh, g, d, 16).upload(rt)
    b.check(b.attend(rt, window=window), window=window)


@pytest.mark.parametrize("lens,news,g", [([40, 300], [40, 130], 4), ([70, 5], [1, 1], 2)])
def test_without_causality_every_row_sees_its_sequence(rt, lens, news, g):
    b = Batch(7, lens, news, 2, g, 128, 32).upload(rt)
    b.check(b.attend(rt, causal=False), causal=False)


def test_one_token_each_without_offsets(rt):
    b = Batch(8, [50, 0, 1, 900, 33], [1] * 5, 2, 4, 128, 16, starts=False).upload(rt)
    b.check(b.attend(rt))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,news", [([0, 3, 20], [4, 9, 20]), ([0], [1]), ([5, 40], [140, 200])])
def test_rows_that_see_nothing_are_zeros(rt, lens, news, d):
    """More new tokens than the cache holds: the first ones stand before position 0."""
    b = Batch(9, lens, news, 2, 4, d, 16).upload(rt)
    got = b.attend(rt)
    b.check(got)
    empty = news[0] - lens[0]
    assert (got[:empty * b.heads * d] == 0).all()


@pytest.mark.parametrize("new", [1, 5, 150])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 100), (256, 32)])
def test_pages_outside_the_cache_hold_no_tokens(rt, d, page, new):
    b = Batch(10, [400, 230], [new, new], 2, 4, d, page)
    holes = [(0, 1), (1, 0), (1, 230 // page)]
    for i, (s, c) in enumerate(holes):
        b.table[s, c] = (-1, b.pages, -2**31)[i]
    b.upload(rt)
    b.check(b.attend(rt), holes=holes)


def test_lengths_and_offsets_that_point_outside(rt):
    """Lengths past the table's row: the tokens there do not exist. Offsets past the call's rows, or descending: no row of theirs."""
    b = Batch(11, [64, 40], [1, 1], 1, 4, 128, 16)
    b.table = np.ascontiguousarray(b.table[:, :4])
    b.width = 4
    b.lens = [64 + 1000, 40]
    b.upload(rt)
    b.check(b.attend(rt))
    b = Batch(12, [30, 40, 50], [2, 2, 2], 1, 2, 64, 16).upload(rt)
    good = b.attend(rt)
    b.check(good)
    for starts in ([0, 2, 1, 6], [0, 2, 2**31 - 1, 6], [-5, 2, 4, 6], [0, 2, 4, 2**30]):
        b.seqs = nn.PagedSeqs(b.seqs.page_table, b.seqs.kv_lens, rt.buffer_from(np.array(starts, np.int32)), 3, b.width)
        b.attend(rt)
    b.seqs = nn.PagedSeqs(b.seqs.page_table, rt.buffer_from(np.array([-3, -2**31, 2**31 - 1], np.int32)), rt.buffer_from(b.starts), 3, b.width)
    b.attend(rt)
    b.upload(rt)
    assert np.array_equal(b.attend(rt), good)


@pytest.mark.parametrize("news", [1, 3, 90])
@pytest.mark.parametrize("std,scale", [(1.0, 1.0), (6.0, None), (1.0, 0.0), (1.0, -0.3), (30.0, 0.05)])
def test_sharp_flat_and_negative_scores(rt, std, scale, news):
    b = Batch(13, [500, 200], [news, news], 2, 2, 128, 16, std=std).upload(rt)
    b.check(b.attend(rt, scale=scale), scale=scale)


def test_q_rows_apart(rt):
    """Queries at the front of wider rows."""
    b = Batch(14, [300, 70], [9, 70], 2, 2, 64, 16).upload(rt)
    want = b.attend(rt)
    stride = b.heads * b.dim + 40
    wide = np.full((b.total, stride), NAN16, np.uint16)
    wide[:, :b.heads * b.dim] = b.q.reshape(b.total, -1)
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, b.total, b.heads, b.cache, b.seqs))
    nn.attn_paged(rt, rt.buffer_from(wide), b.cache, b.seqs, b.out.view(0, b.q.size * 2), work, b.total, b.heads, b.dim ** -0.5, True, 0, stride)
    assert np.array_equal(b.out.read(np.uint16, b.q.size + 64), want)


@pytest.mark.parametrize("n,new,length", [(300, 1, 90), (1100, 1, 40), (70, 9, 300)])
def test_many_sequences(rt, n, new, length):
    lens = [new + (i * 37) % length for i in range(n)]
    b = Batch(15, lens, [new] * n, 1, 2, 64, 16).upload(rt)
    b.check(b.attend(rt))


def test_the_same_call_gives_the_same_bits(rt):
    for lens, news in (([9000, 100, 3000], [1, 1, 1]), ([3000, 900], [200, 300])):
        b = Batch(16, lens, news, 2, 4, 128, 64).upload(rt)
        first = b.attend(rt)
        for _ in range(5):
            assert np.array_equal(b.attend(rt), first)


def test_infinite_values_reach_the_rows_that_see_them(rt):
    b = Batch(17, [200], [1], 1, 2, 64, 16)
    v = np.array(b.get("v", 0, 200))
    v[50, 0, 3], v[60, 0, 4], v[61, 0, 5], v[62, 0, 5] = 0x7F80, NAN16, 0x7F80, 0xFF80
    b.put("v", 0, 0, v)
    b.upload(rt)
    got = b.attend(rt)[:b.q.size].reshape(b.heads, b.dim)
    assert (got[:, 3] == 0x7F80).all()
    assert ((got[:, 4:6] & 0x7FFF) > 0x7F80).all()
    rest = np.delete(got, [3, 4, 5], axis=1)
    assert ((rest & 0x7F80) != 0x7F80).all()


def test_captured_calls_replay_on_new_inputs(rt):
    """Two graphs, each with a workspace of its own, replayed at once on two streams after the lengths changed."""
    import torch

    st = torch.cuda.ExternalStream(rt.stream)
    made = []
    rt.set_encode_only(True)
    try:
        for seed, news in ((18, [1, 1, 1]), (19, [150, 1, 40])):
            b = Batch(seed, [900, 300, 4000], news, 2, 4, 128, 16).upload(rt)
            work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, b.total, b.heads, b.cache, b.seqs))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                nn.attn_paged(rt, b.b_q, b.cache, b.seqs, b.out.view(0, b.q.size * 2), work, b.total, b.heads, b.dim ** -0.5)
            made.append((b, g, work))
        for lens in ([900, 300, 4000], [151, 1, 77], [700, 40, 3999]):
            for b, _, _ in made:
                b.lens = lens
                b.seqs.kv_lens.write(np.array(lens, np.int32))
                b.out.write(np.full(b.q.size + 64, SENTINEL16, np.uint16))
            rt.synchronize()
            streams = [torch.cuda.Stream() for _ in made]
            for _ in range(3):
                for (_, g, _), s in zip(made, streams):
                    with torch.cuda.stream(s):
                        g.replay()
            torch.cuda.synchronize()
            for b, _, _ in made:
                b.check(b.out.read(np.uint16, b.q.size + 64))
    finally:
        rt.set_encode_only(False)


def test_nothing_is_launched_for_nothing(rt):
    b = Batch(20, [5], [1], 1, 1, 64, 16).upload(rt)
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, 1, 1, b.cache, b.seqs))
    rt.take_dispatch_count()
    empty = nn.PagedSeqs(b.seqs.page_table, b.seqs.kv_lens, None, 0, b.width)
    nn.attn_paged(rt, b.b_q, b.cache, empty, b.out, work, 0, 1, 0.1)
    assert rt.take_dispatch_count() == 0
