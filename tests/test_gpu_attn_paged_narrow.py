"""attn_paged on heads narrower than the 64 columns of a copy, over pages of a multiple of eight tokens: the copies reach past the head, what
lies there are other heads' and tokens' values and must not count."""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("major", [False, True])
@pytest.mark.parametrize("page", [8, 16, 24, 64])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 56])
def test_few_rows(rt, dim, page, major):
    b = Batch(401, [300, 77, 1], [1, 3, 1], 3, 2, dim, page, major, tail=2).upload(rt)
    b.check(b.attend(rt))


@pytest.mark.parametrize("major", [False, True])
@pytest.mark.parametrize("page", [8, 16, 24, 64])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 56])
def test_many_rows(rt, dim, page, major):
    b = Batch(402, [300, 77], [150, 77], 3, 2, dim, page, major, tail=2).upload(rt)
    b.check(b.attend(rt))


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("dim", [8, 40])
def test_one_key_head_and_one_page(rt, dim, new):
    """Neighbours in memory are the tokens in front and behind, and the end of the cache."""
    for lens in ([64], [1], [63]):
        b = Batch(403, lens, [min(new, lens[0])], 1, 2 if new == 1 else 40, dim, 64, spare=0).upload(rt)
        b.check(b.attend(rt), lens)


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("dim", [8, 24, 56])
def test_neighbours_that_are_not_finite(rt, dim, new):
    """Key head 1 of three is not finite throughout: heads 0 and 2 are as if it were not there."""
    b = Batch(404, [300], [new], 3, 2, dim, 16)
    for name, worst in (("k", 0x7F80), ("v", 0x7FC1)):
        rows = np.array(b.get(name, 0, 300))
        rows[:, 1] = worst
        b.put(name, 0, 0, rows)
    b.upload(rt)
    got = b.attend(rt)[:b.q.size].reshape(b.total, b.heads, dim)
    clean = Batch(404, [300], [new], 3, 2, dim, 16).upload(rt)
    want = clean.attend(rt)
    clean.check(want)
    want = want[:b.q.size].reshape(got.shape)
    keep = [0, 1, 4, 5]
    assert np.array_equal(got[:, keep], want[:, keep])
    assert ((got[:, 2:4] & 0x7FFF) > 0x7F80).all()
