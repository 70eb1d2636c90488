"""Chunks of prompts beside single tokens in one batch: one call for all, whichever kernel its mean number of rows picks, and a call for the
chunks and one for the tokens, over parts of the same buffers."""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import SENTINEL16, Batch
from tessl_b200 import nn

pytestmark = pytest.mark.gpu

# lens, news (the chunks first), chunks, key heads, group, head_dim
MIXED = [([1500] + [7 + 90 * i for i in range(30)], [130] + [1] * 30, 1, 2, 4, 128),        # few rows on average
         ([900, 300, 40, 800, 1], [300, 300, 1, 1, 1], 2, 2, 4, 128),                      # many
         ([700, 90] + [33 * i for i in range(1, 20)], [200, 60] + [1] * 19, 2, 1, 4, 256),
         ([600, 500, 400], [90, 1, 1], 1, 2, 2, 64)]


@pytest.mark.parametrize("empty", [0, 40])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("case", range(len(MIXED)))
def test_one_call_for_all(rt, case, window, empty):
    """`empty` sequences behind, as they pad a captured batch, lower the mean."""
    lens, news, _, kvh, g, d = MIXED[case]
    b = Batch(600 + case, lens + [0] * empty, news + [0] * empty, kvh, g, d, 16, tail=3).upload(rt)
    b.check(b.attend(rt, window=window), window=window)


@pytest.mark.parametrize("case", range(len(MIXED)))
def test_a_call_for_the_chunks_and_one_for_the_tokens(rt, case):
    lens, news, chunks, kvh, g, d = MIXED[case]
    b = Batch(600 + case, lens, news, kvh, g, d, 16).upload(rt)
    row, rows = b.heads * d * 2, int(b.starts[chunks])
    table, lengths = b.seqs.page_table, b.seqs.kv_lens
    tokens = b.total - rows
    # the workspace of the whole batch serves both
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, b.total, b.heads, b.cache, b.seqs))
    for first, n, at, count, starts in ((0, chunks, 0, rows, rt.buffer_from(b.starts[:chunks + 1])), (chunks, b.n - chunks, rows, tokens, None)):
        seqs = nn.PagedSeqs(table.view(first * b.width * 4, n * b.width * 4), lengths.view(first * 4, n * 4), starts, n, b.width)
        nn.attn_paged(rt, b.b_q.view(at * row, count * row), b.cache, seqs, b.out.view(at * row, count * row), work, count, b.heads, d ** -0.5)
    rt.synchronize()
    b.check(b.out.read(np.uint16, b.q.size + 64))
    assert (b.out.read(np.uint16, b.q.size + 64)[b.q.size:] == SENTINEL16).all()
