"""YaRN's frequencies against numbers worked out by hand from its definition.

Base 10^4, 64 values that turn, 4096 positions at first.  The pair that turns n times over them is
64 ln(4096 / (2 pi n)) / (2 ln 10^4):
    n = 32: ln(20.3718) = 3.01415, 64 * 3.01415 / 18.42068 = 10.472, down to 10
    n = 1:  ln(651.899) = 6.47988, 64 * 6.47988 / 18.42068 = 22.513, up to 23
so pairs up to 10 stay, those from 23 on are divided by the factor, and pair i between them is f (1 - r) + f / factor r with
r = (i - 10) / 13.  With 8 times the context the turned values grow by 1 + 0.1 ln 8 = 1.2079441541679836.
"""
import pytest

from qwen35_amd import ops


def turns(**more):
    table = ops.RopeTable(64, 1e4, device="cpu", **more)
    return [s % 2 ** 64 for s in table.steps.tolist()], table.gain


def test_range_ramp_and_gain():
    plain, one = turns()
    yarn, gain = turns(scaling="yarn", factor=8.0, original=4096)
    assert one == 1.0 and abs(gain - 1.2079441541679836) < 2.0 ** -24
    for i in range(32):
        # (each is rounded to 2^-64 turns, the factors to 64 bits)
        kept = 13 * 8 if i <= 10 else 13 if i >= 23 else 13 * 8 - 7 * (i - 10)  # in parts of 13 * 8
        assert abs(yarn[i] - plain[i] * kept / (13 * 8)) <= plain[i] * 2.0 ** -50 + 2, i
    assert yarn[10] == plain[10] and yarn[11] < plain[11] and yarn[22] > plain[22] / 8 + 2 ** 20


def test_ends_of_the_range():
    """fast and slow move the ends: n = 2 pi at 4096 positions is pair 64 ln(651.899 / 2 pi) / 18.42068 = 16.128 -> 16, up to 17."""
    plain, _ = turns()
    yarn, _ = turns(scaling="yarn", factor=4.0, original=4096, fast=6.283185307179586, slow=6.2)
    assert yarn[16] == plain[16]
    assert [abs(yarn[i] - plain[i] / 4) <= 2 for i in (17, 18, 31)] == [True] * 3


@pytest.mark.parametrize("factor", [1.0, 2.0, 40.0])
def test_factors(factor):
    plain, _ = turns()
    yarn, _ = turns(scaling="yarn", factor=factor, original=4096)
    assert yarn[:11] == plain[:11]
    for i in range(23, 32):
        assert abs(yarn[i] - plain[i] / factor) <= plain[i] * 2.0 ** -50 + 2
