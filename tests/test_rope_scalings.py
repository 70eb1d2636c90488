"""rope_steps: each way of stretching the frequencies against its formula, written out in 64 bits and from the waves' side: how often a pair
turns within the trained context. No GPU."""
import math

import numpy as np
import pytest

from tessl_b200 import capi, nn

try:
    capi.load()
except ImportError:
    pytest.skip("the library is not built", allow_module_level=True)

SHAPES = [(128, 10000.0), (64, 500000.0), (256, 1e7), (20, 1e6), (2, 10000.0)]


def plain(rot, theta):
    """Radians a position of each pair."""
    return np.array([theta ** (-i / (rot // 2)) for i in range(rot // 2)])


def check(rot, theta, scaling, want):
    """2^64 / 2 pi times the radians: the relative accuracy of this side's power and few steps in 64 bits (64 * 2^-53; differences of
    near values in a blend count as values of the blend's own size), and half a step."""
    got = np.asarray(nn.rope_steps(rot, theta, scaling)[0], np.float64)
    size = want / (2 * math.pi) * 2.0 ** 64
    assert (np.abs(got - size) <= size * 64 * 2.0 ** -53 + 1).all()


@pytest.mark.parametrize("factor", [1.0, 2.5, 8.0])
@pytest.mark.parametrize("rot,theta", SHAPES)
def test_linear(rot, theta, factor):
    check(rot, theta, nn.RopeScaling("linear", factor), plain(rot, theta) / factor)
    assert nn.rope_steps(rot, theta, nn.RopeScaling("linear", factor))[1] == 1.0


@pytest.mark.parametrize("factor", [1.0, 2.5, 8.0])
@pytest.mark.parametrize("rot,theta", SHAPES[:-1])
def test_ntk(rot, theta, factor):
    """The first pair as it is, the last one slower by the factor, the powers of one base between them."""
    pairs = rot // 2
    want = plain(rot, theta) * factor ** (-np.arange(pairs) / (pairs - 1))
    check(rot, theta, nn.RopeScaling("ntk", factor), want)
    assert nn.rope_steps(rot, theta, nn.RopeScaling("ntk", factor))[1] == 1.0


def test_ntk_of_one_pair_changes_nothing():
    check(2, 10000.0, nn.RopeScaling("ntk", 8.0), plain(2, 10000.0))


@pytest.mark.parametrize("factor,original,low,high", [(8.0, 8192, 0, 0), (32.0, 8192, 1, 4), (4.0, 4096, 2, 16), (2.0, 300, 0.5, 0.75)])
@pytest.mark.parametrize("rot,theta", SHAPES)
def test_wavelength(rot, theta, factor, original, low, high):
    turns_low, turns_high = low or 1.0, high or 4.0
    want = []
    for w in plain(rot, theta):
        wave = 2 * math.pi / w
        if wave < original / turns_high:
            want.append(w)
        elif wave > original / turns_low:
            want.append(w / factor)
        else:
            smooth = (original / wave - turns_low) / (turns_high - turns_low)
            want.append((1 - smooth) * w / factor + smooth * w)
    check(rot, theta, nn.RopeScaling("wavelength", factor, original, low, high), np.array(want))
    assert nn.rope_steps(rot, theta, nn.RopeScaling("wavelength", factor, original, low, high))[1] == 1.0


@pytest.mark.parametrize("factor,original,low,high", [(4.0, 32768, 0, 0), (40.0, 4096, 1, 32), (16.0, 8192, 2, 8), (1.0, 4096, 0, 0)])
@pytest.mark.parametrize("rot,theta", SHAPES)
def test_yarn(rot, theta, factor, original, low, high):
    def pair_that_turns(times):  # original * theta^(-i / pairs) = 2 pi times, for i
        return (rot / 2) * math.log(original / (2 * math.pi * times)) / math.log(theta)

    first = max(math.floor(pair_that_turns(high or 32.0)), 0)
    last = min(math.ceil(pair_that_turns(low or 1.0)), rot - 1)
    want = []
    for i, w in enumerate(plain(rot, theta)):
        kept = 1.0 if i <= first else 0.0 if i >= last else 1 - (i - first) / (last - first)
        want.append(w * kept + w / factor * (1 - kept))
    check(rot, theta, nn.RopeScaling("yarn", factor, original, low, high), np.array(want))
    # 0.1 ln(factor) + 1 in f32
    assert nn.rope_steps(rot, theta, nn.RopeScaling("yarn", factor, original, low, high))[1] == np.float32(0.1 * math.log(factor) + 1.0)


def test_values_by_hand():
    """Bases that make the powers whole: 65536 and four pairs turn by 1, 1/16, 1/256 and 1/4096 radians a position."""
    def radians(s=None):
        return np.asarray(nn.rope_steps(8, 65536.0, s)[0], np.float64) * 2.0 ** -64 * 2 * math.pi

    near = lambda got, want: (np.abs(got - np.array(want)) <= 2.0 ** -40 * np.array(want)).all()
    assert near(radians(), [1, 1 / 16, 1 / 256, 1 / 4096])
    assert near(radians(nn.RopeScaling("linear", 4.0)), [1 / 4, 1 / 64, 1 / 1024, 1 / 16384])
    # the base times 8^(4/3) = 16: powers of 2^-5
    assert near(radians(nn.RopeScaling("ntk", 8.0)), [1, 1 / 32, 1 / 1024, 1 / 32768])
    # within 512 pi positions the pairs turn 256, 16, 1 and 1/16 times; kept from 31, divided up to 1: the second is half and half
    assert near(radians(nn.RopeScaling("wavelength", 4.0, 512 * math.pi, 1.0, 31.0)), [1, (1 / 16 + 1 / 64) / 2, 1 / 1024, 1 / 16384])
    # kept up to the pair that turns 256 times (0), divided from that which turns 1/16 times (3), thirds between them
    assert near(radians(nn.RopeScaling("yarn", 4.0, 512 * math.pi * (1 + 1e-9), 1 / 16 * (1 + 2e-9), 256.0)),
                [1, 1 / 16 * 2 / 3 + 1 / 64 / 3, 1 / 256 / 3 + 1 / 1024 * 2 / 3, 1 / 16384])
