"""attn_paged and kv_append_paged where the division of work, the joining of parts and the addressing can go wrong: items cut into
as many parts as there are blocks, items of the same length, more items than SMs, caches past 2^32 values, pages that sequences share, a
workspace that calls hand on to one another."""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import SENTINEL16, Batch, bf16, f64
from tessl_b200 import nn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,news,kvh,g,d,page", [
    ([40000], [1], 1, 1, 64, 64),      # an item, a part for each block
    ([30000], [16], 1, 16, 64, 64),    # 256 rows, a part for each block: tiles
    ([20000], [64], 1, 2, 256, 128),   # 128 rows of wide heads
    ([15000], [30], 1, 1, 128, 16),    # 30 rows: two items of few rows
    ([3000], [1], 8, 4, 128, 16), ([2000, 2000], [1, 1], 8, 2, 64, 32), ([1500] * 5, [1] * 5, 3, 1, 256, 16),  # items of the same length
    ([640] * 37, [1] * 37, 4, 2, 128, 16),  # as many as the SMs
])
def test_cuts(rt, lens, news, kvh, g, d, page):
    b = Batch(61, lens, news, kvh, g, d, page).upload(rt)
    b.check(b.attend(rt))


@pytest.mark.parametrize("d,page,major", [(64, 16, False), (128, 16, True), (128, 10, False), (192, 64, True), (256, 48, False)])
def test_more_items_than_sms(rt, d, page, major):
    r = np.random.default_rng(62)
    lens = [int(n) for n in r.integers(0, 900, 44)] + [0, 1, 2500]
    b = Batch(63, lens, [1] * len(lens), 4, 3, d, page, head_major=major).upload(rt)
    b.check(b.attend(rt))


def test_more_sequences_than_threads_on_a_shared_sm(rt):
    r = np.random.default_rng(64)
    news = [int(n) for n in r.integers(0, 4, 400)]
    lens = [n + int(x) for n, x in zip(news, r.integers(0, 120, 400))]
    b = Batch(65, lens, news, 2, 2, 64, 16, tail=5).upload(rt)
    b.check(b.attend(rt))


def test_sequences_that_share_pages(rt):
    b = Batch(66, [64, 100, 200], [1, 1, 70], 2, 2, 128, 16)
    b.table[1, :4], b.table[2, :4] = b.table[0, :4], b.table[0, :4]  # the first 64 tokens of all
    b.table[2, 4] = b.table[1, 4]
    b.upload(rt)
    b.check(b.attend(rt))


def test_one_workspace_handed_on(rt):
    """Calls of both kinds and of other sizes, and replays of one of them, one behind the other in one workspace."""
    import torch

    bs = [Batch(70 + i, *how).upload(rt) for i, how in enumerate([([3000], [1], 2, 2, 64, 16), ([2000, 90], [200, 90], 2, 2, 64, 16),
                                                                  ([5000], [1], 1, 4, 64, 16), ([700] * 90, [1] * 90, 2, 2, 64, 16)])]
    work = rt.alloc_buffer(max(nn.attn_paged_workspace_bytes(rt, b.total, b.heads, b.cache, b.seqs) for b in bs))
    work.write(np.full(work.nbytes // 4, 0xFFFFFFFF, np.uint32))
    first = [b.attend(rt, work=work) for b in bs]
    for b, got in zip(bs, first):
        b.check(got)
    st = torch.cuda.ExternalStream(rt.stream)
    rt.set_encode_only(True)
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for b in bs[:2]:
                nn.attn_paged(rt, b.b_q, b.cache, b.seqs, b.out.view(0, b.q.size * 2), work, b.total, b.heads, b.dim ** -0.5)
    finally:
        rt.set_encode_only(False)
    for _ in range(3):
        for b in bs:
            b.out.write(np.full(b.q.size + 64, SENTINEL16, np.uint16))
        with torch.cuda.stream(st):
            g.replay()
            g.replay()
        torch.cuda.synchronize()
        for b, want in zip(bs[:2], first):
            assert np.array_equal(b.out.read(np.uint16, b.q.size + 64), want)
        for b, want in zip(bs, first):
            assert np.array_equal(b.attend(rt, work=work), want)


def test_two_runtimes_and_one_workspace(rt):
    b = Batch(75, [4000, 77], [1, 1], 2, 4, 128, 16).upload(rt)
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, b.total, b.heads, b.cache, b.seqs))
    with nn.Runtime() as other:
        want = b.attend(rt, work=work)
        b.check(want)
        for _ in range(3):
            for r in (other, rt):
                assert np.array_equal(b.attend(r, work=work), want)


@pytest.mark.parametrize("news", [[1, 1], [40, 3], [150, 90]])
@pytest.mark.parametrize("major", [False, True])
def test_a_cache_of_more_than_2_32_values(rt, major, news):
    """Pages at both ends of caches of 2^32 values and some: append, then attention."""
    import torch

    page, kvh, dim, g = 64, 4, 128, 2
    each = page * kvh * dim
    pages = 2**32 // each + 9
    lens = [333, 150]
    small = Batch(80, lens, news, kvh, g, dim, page, head_major=major, spare=0)
    far = np.concatenate([np.arange(pages - small.pages + 3, pages), np.arange(3)]).astype(np.int32)  # where the pages of `small` lie
    caches = [torch.empty(pages * each, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for c, a in zip(caches, (small.k, small.v)):
        c.view(pages, each)[torch.from_numpy(far).cuda().long()] = torch.from_numpy(a.reshape(-1, each).view(np.int16).copy()).cuda().view(torch.bfloat16)
    torch.cuda.synchronize()
    k, v = (nn.GpuBuffer.from_torch(c) for c in caches)
    table = np.full_like(small.table, -1)
    for s, n in enumerate(lens):
        table[s, :-(-n // page)] = far[small.table[s, :-(-n // page)]]
    small.upload(rt)
    cache = nn.PagedKv(k, v, pages, page, kvh, dim, nn.KV_HEAD_MAJOR if major else nn.KV_TOKEN_MAJOR)
    seqs = nn.PagedSeqs(rt.buffer_from(table), small.seqs.kv_lens, small.seqs.q_starts, 2, small.width)
    # new keys and values take the places of those there
    r = np.random.default_rng(81)
    new = [bf16(r.standard_normal((small.total, kvh, dim))) for _ in range(2)]
    at = 0
    for s, n in enumerate(news):
        for name, rows in zip("kv", new):
            small.put(name, s, lens[s] - n, rows[at:at + n])
        at += n
    bufs = [rt.buffer_from(a) for a in new]
    q = rt.buffer_from(small.q)
    nn.kv_append_paged(rt, None, bufs[0], bufs[1], None, cache, seqs, None, None, small.total, 0, in_as_bf16=True)
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, small.total, small.heads, cache, seqs))
    nn.attn_paged(rt, q, cache, seqs, small.out.view(0, small.q.size * 2), work, small.total, small.heads, dim ** -0.5)
    rt.synchronize()
    small.check(small.out.read(np.uint16, small.q.size + 64))
    got = caches[0].view(pages, each)[torch.from_numpy(far).cuda().long()].view(torch.int16).cpu().numpy().view(np.uint16)
    live = small.k.reshape(-1, each) != 0x7FC1
    assert np.array_equal(got[live], small.k.reshape(-1, each)[live])
    assert np.isfinite(f64(got[live])).all()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("pages,width", [(0, 3), (3, 0), (0, 0)])
def test_no_pages_or_no_table(rt, pages, width, new):
    b = Batch(90, [70, 20], [new, new], 2, 2, 64, 16).upload(rt)
    none = nn.GpuBuffer(0, 0)
    cache = nn.PagedKv(b.b_k if pages else none, b.b_v if pages else none, pages, 16, 2, 64)
    seqs = nn.PagedSeqs(b.seqs.page_table if width else none, b.seqs.kv_lens, b.seqs.q_starts, 2, width)
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, b.total, b.heads, cache, seqs))
    nn.attn_paged(rt, b.b_q, cache, seqs, b.out.view(0, b.q.size * 2), work, b.total, b.heads, 0.125)
    kv = rt.buffer_from(bf16(np.ones((b.total, 2, 64))))
    nn.kv_append_paged(rt, None, kv, rt.buffer_from(bf16(np.ones((b.total, 2, 64)))), None, cache, seqs, None, None, b.total, 0, in_as_bf16=True)
    rt.synchronize()
    got = b.out.read(np.uint16, b.q.size + 64)
    if pages == 0 or width == 0:
        assert (got[:b.q.size] & 0x7FFF == 0).all() and (got[b.q.size:] == SENTINEL16).all()


def test_offsets_that_go_back_and_forth_count_to_an_end(rt):
    """Descending offsets may not be given; the work that they add up to is more than the kernels count, and nothing is done."""
    n, tokens, page = 1200, 1024, 1 << 20
    cache = nn.PagedKv(rt.buffer_from(np.zeros(page * 8, np.uint16)), rt.buffer_from(np.zeros(page * 8, np.uint16)), 1, page, 1, 8)
    starts = np.zeros(n + 1, np.int32)
    starts[1::2] = tokens
    seqs = nn.PagedSeqs(rt.buffer_from(np.zeros(n, np.int32)), rt.buffer_from(np.full(n, page, np.int32)), rt.buffer_from(starts), n, 1)
    q = rt.buffer_from(np.zeros(tokens * 16 * 8, np.uint16))
    out = rt.buffer_from(np.full(tokens * 16 * 8, SENTINEL16, np.uint16))
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, tokens, 16, cache, seqs))
    nn.attn_paged(rt, q, cache, seqs, out, work, tokens, 16, 0.3, causal=False)
    rt.synchronize()
    assert not rt.is_poisoned()
    assert (out.read(np.uint16, tokens * 16 * 8) == SENTINEL16).all()
