"""The cosines and sines of rope: each angle of a turn in 2^32 steps, against 64 bits."""
import numpy as np
import pytest

from gpu_util import rt  # noqa: F401
from paged_util import U32
from tessl_b200 import nn

pytestmark = pytest.mark.gpu


def exact(angle):
    """(cos, sin) of angle / 2^32 turns, relative to themselves: the quadrant is taken off in whole numbers."""
    quadrant = (angle + (1 << 29)) >> 30
    x = (angle - (quadrant << 30)).astype(np.float64) * (2 * np.pi / 2 ** 32)
    c, s = np.cos(x), np.sin(x)
    q = quadrant & 3
    return np.choose(q, [c, -s, -c, s]), np.choose(q, [s, c, -s, -c])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [2, 256])
@pytest.mark.parametrize("kind", ["all around", "near the axes", "near the diagonals"])
def test_angles(rt, kind, dim, interleaved):
    """Pairs (1, 0) turned: what comes out is the cosine and the sine alone.

    Relative error, u = 2^-24, x half a turn's fraction of at most 1/4: the angle to f32 u, which counts as pi x cot(pi x) <= 1 (sine) or
    pi x tan(pi x) <= 0.79 (cosine). Sine: beside pi, the polynomial is 0.11 of it at most; the square of x, its
    product with x, the last rounding of the polynomial and its product 4 * 0.11 u; the polynomial itself 0.06 u; the last sum u. At x = 1/4, 0.79 + 0.44 + 0.06 + 1;
    towards 0, where the polynomial vanishes, 1 + 1. Cosine: 1 - cos is 0.42 of it at most, off by the square's rounding and the last
    sum's before the end, 2 * 0.42 u, and 0.1 of that by the sums before; the polynomial 0.01 u; the last sum 0.71 u (2^-25 of a value
    from 0.70 on): 0.79 + 0.92 + 0.01 + 0.71. Both below 2.5 u."""
    r = np.random.default_rng(5)
    tokens, pairs = 4096, dim // 2
    pos = np.arange(-tokens // 2, tokens // 2)
    if kind == "all around":
        step = r.integers(0, 2 ** 32, pairs)
    else:  # of position p: p of a quarter or half quarter turn, and p * 2^0 to 2^18 angles more
        step = (2.0 ** r.uniform(0, 18, pairs)).astype(np.int64) + (2 ** 30 if kind == "near the axes" else 2 ** 29)
    angle = (pos[:, None] * step[None, :]) % 2 ** 32
    x = np.zeros((tokens, 1, dim), np.float32)
    first, second = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, pairs), slice(pairs, dim))
    x[..., first] = 1.0
    plan = nn.Rope(rt.buffer_from(step.astype(np.uint64) << np.uint64(32)), dim, interleaved, 1.0)
    out = rt.buffer_from(np.full(x.size, 7.0, np.float32))
    nn.rope(rt, rt.buffer_from(x), rt.buffer_from(pos.astype(np.int32)), out, plan, tokens, 1, dim, False, False)
    got = out.read(np.float32, x.size).reshape(tokens, dim).astype(np.float64)
    for g, want, name in zip((got[:, first], got[:, second]), exact(angle), ("cosine", "sine")):
        off, size = np.abs(g - want), np.abs(want)
        assert (off <= 2.5 * U32 * size).all(), f"{name}: off by {(off[size > 0] / size[size > 0]).max() / U32} * 2^-24 of itself"
