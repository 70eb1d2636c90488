"""attn_paged: which sizes it takes, and the workspace that it asks for. No GPU: every call ends in a refusal, that of its workspace at the
latest."""
import re
from dataclasses import replace

import pytest

from tessl_b200 import nn
from test_attn_paged_refusals import host_rt  # noqa: F401


def sizes(n, pages_each, page=2048, kvh=8, dim=128, starts=True):
    """A cache and sequences whose buffers are never touched, far apart and as large as they have to be."""
    far = iter(range(1 << 48, 1 << 56, 1 << 46))
    pages = 1 << 10
    cache = nn.PagedKv(nn.GpuBuffer(next(far), 1 << 45), nn.GpuBuffer(next(far), 1 << 45), pages, page, kvh, dim)
    return cache, nn.PagedSeqs(nn.GpuBuffer(next(far), 1 << 45), nn.GpuBuffer(next(far), 1 << 45),
                               nn.GpuBuffer(next(far), 1 << 45) if starts else None, n, pages_each)


def refusal(rt, cache, seqs, total, heads, work=16, **how):
    """What a call with a workspace of 16 bytes is refused for."""
    big = 1 << 45
    with pytest.raises(nn.TesslError) as e:
        nn.attn_paged(rt, nn.GpuBuffer(1 << 57, big), cache, seqs, nn.GpuBuffer(1 << 58, big), nn.GpuBuffer(1 << 59, work), total, heads,
                      how.pop("scale", 0.125), **how)
    return str(e.value)


# sequences, new tokens, heads, pages of 2048 for each, head_dim
TAKEN = [(1, 65536, 64, 512, 128),    # a prompt of 65536 with room for 2^20 tokens
         (16, 65536, 64, 512, 256),
         (4, 200000, 32, 1024, 64)]


@pytest.mark.parametrize("n,total,heads,each,dim", TAKEN)
def test_long_prompts_with_room_for_long_contexts_are_taken(host_rt, n, total, heads, each, dim):  # noqa: F811
    cache, seqs = sizes(n, each, dim=dim)
    assert "workspace has 16 bytes" in refusal(host_rt, cache, seqs, total, heads)


@pytest.mark.parametrize("dim,rows", [(64, 256), (128, 256), (136, 128), (256, 128)])
def test_a_call_is_refused_from_2_32_units_on(host_rt, dim, rows):  # noqa: F811
    """A sequence, 8 query heads on each of 8 key heads: 8 (8 t / rows + 1) (c / 128 + 1) units of t new tokens and c tokens of room; with a
    scale of 0 they are of 16 rows and 64 keys."""
    each = 1024  # 2^21 tokens, 16385 units of 128 keys, 32769 of 64
    cache, seqs = sizes(1, each, dim=dim)
    for scale, r, units in ((0.125, rows, 16385), (-0.1, rows, 16385), (0.0, 16, 32769)):
        total = -(-(2 ** 32 - 8 * units) * r // (64 * units))  # the first that is refused
        assert "more rows and keys" in refusal(host_rt, cache, seqs, total, 64, scale=scale)
        assert "workspace has 16 bytes" in refusal(host_rt, cache, seqs, total - 1, 64, scale=scale)


def test_few_rows_are_counted_by_16_and_64(host_rt):  # noqa: F811
    for page, starts in ((2048, False), (2044, True)):  # a token each, or pages that are no multiple of 8
        n = 40000
        units = -(-(1 << 21) // 64) + 1
        each = -(-((units - 1) * 64) // page)
        cache, seqs = sizes(n, each, page=page, starts=starts, kvh=1)
        blocks = n * 64 / 16 + n
        most = each * page / 64 + 1
        assert blocks * most >= 2 ** 32
        assert "more rows and keys" in refusal(host_rt, cache, seqs, n, 64)
        few = int((2 ** 32 - 1) // (most * 5))
        cache, seqs = sizes(few, each, page=page, starts=starts, kvh=1)
        assert "workspace has 16 bytes" in refusal(host_rt, cache, seqs, few, 64)


@pytest.mark.parametrize("change,match", [
    (dict(layout=2), "layout 2"), (dict(head_dim=0), "head_dim 0"), (dict(head_dim=60), "head_dim 60"), (dict(head_dim=264), "head_dim 264"),
    (dict(n_kv_heads=0), "n_kv_heads 0"), (dict(n_kv_heads=65536), "n_kv_heads 65536"), (dict(page_size=0), "page_size"),
    (dict(page_size=1 << 25), "too large"), (dict(num_pages=1 << 31), "page id"), (dict(n_kv_heads=3), "not a multiple"),
])
def test_the_workspace_of_a_cache_that_is_refused_is_none(host_rt, change, match):  # noqa: F811
    cache, seqs = sizes(3, 4, page=16)
    bad = replace(cache, **change)
    heads = max(16, change.get("n_kv_heads", 0))
    assert match in refusal(host_rt, bad, seqs, 3, heads)
    assert nn.attn_paged_workspace_bytes(host_rt, 3, heads, bad, seqs) == 0


def test_the_workspace_of_a_call_that_is_refused_is_none(host_rt):  # noqa: F811
    cache, seqs = sizes(3, 4, page=16)
    ask = lambda total, heads, c=cache, s=seqs: nn.attn_paged_workspace_bytes(host_rt, total, heads, c, s)
    assert ask(3, 16) > 0
    for heads in (0, 12, 1 << 30):
        assert ask(3, heads) == 0 and refusal(host_rt, cache, seqs, 3, heads)
    for total in (1 << 31, (1 << 32) - 1):
        assert ask(total, 8) == 0 and "int32 offset" in refusal(host_rt, cache, seqs, total, 8)
    assert ask(3, 8, s=replace(seqs, num_seqs=1 << 31)) == 0
    # rows of 2^24 heads of 256 columns: 2^32 values
    wide, one = sizes(1, 4, page=16, dim=256)
    assert ask(1, 1 << 24, wide, one) == 0 and "too long" in refusal(host_rt, wide, one, 1, 1 << 24)
    assert ask(1, (1 << 24) - 8, wide, one) > 0
    # more units than are counted
    long, s = sizes(1, 1024)
    last = -(-(2 ** 32 - 8 * 16385) * 256 // (64 * 16385)) - 1
    assert ask(last, 64, long, s) > 0 and ask(last + 1, 64, long, s) == 0
    assert "more rows and keys" in refusal(host_rt, long, s, last + 1, 64)


def test_a_workspace_can_be_asked_for_before_there_are_buffers(host_rt):  # noqa: F811
    cache, seqs = sizes(3, 4, page=16)
    none = nn.GpuBuffer(0, 0)
    early = replace(seqs, page_table=none, kv_lens=none, q_starts=None)
    for total in (200, 3):
        want = nn.attn_paged_workspace_bytes(host_rt, total, 64, cache, seqs if total == 200 else replace(seqs, q_starts=None))
        assert 0 < want == nn.attn_paged_workspace_bytes(host_rt, total, 64, replace(cache, k=none, v=none), early)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("kvh,heads", [(8, 32), (1, 16), (4, 4), (2, 80)])
def test_the_workspace_of_a_batch_serves_every_smaller_one(host_rt, dim, kvh, heads):  # noqa: F811
    """What a call needs, by its refusal of 16 bytes, against what the query says of larger batches."""
    tokens, counts = (1, 2, 3, 9, 33, 64, 65, 300, 4096), (1, 2, 19, 37, 64, 75, 300)
    need, asked = {}, {}
    for n in counts:
        for total in tokens:
            for starts in (True, False) if total == n else (True,):
                cache, seqs = sizes(n, 4, page=16, kvh=kvh, dim=dim, starts=starts)
                need[total, n, starts] = int(re.search(r"needs (\d+)", refusal(host_rt, cache, seqs, total, heads)).group(1))
                if starts:
                    asked[total, n] = nn.attn_paged_workspace_bytes(host_rt, total, heads, cache, seqs)
    for (t, n, _), least in need.items():
        for (total, most), size in asked.items():
            if t <= total and n <= most:
                assert size >= least > 0, ((t, n), (total, most))
    for (t, n, starts), least in need.items():  # a token each, without offsets: no more than such calls want
        if not starts:
            cache, seqs = sizes(n, 4, page=16, kvh=kvh, dim=dim, starts=False)
            assert nn.attn_paged_workspace_bytes(host_rt, t, heads, cache, seqs) == least
