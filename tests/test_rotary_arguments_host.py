"""Norms and rotation of heads, where no device is needed: arguments that would be left out of account or changed on their way are refused."""
import numpy as np
import pytest


class Host:      # takes uploads, runs nothing
    def upload(self, array, buf=None, offset=0):
        return type("Buffer", (), {"ptr": 0})()


@pytest.mark.parametrize("positions", [np.array([2 ** 31, 0, 1], np.int64), np.array([-2 ** 31 - 1, 0, 1], np.int64), np.array([2 ** 32 + 5, 0, 1], np.uint64), np.array([0.0, 0.5, 1.0]),
                                       np.array([0.0, np.nan, 1.0])], ids=str)
def test_positions_that_32_bits_do_not_hold(pkg, positions):
    turn = pkg.ops.Rotary(Host(), 4, 2, 64, np.zeros(32, np.float32))
    with pytest.raises(ValueError, match="positions"):
        turn(np.zeros((3, 4, 64), np.float16), np.zeros((3, 2, 64), np.float16), positions)


@pytest.mark.parametrize("given", [dict(factor=8.0), dict(trained=8192.0), dict(factor=8.0, trained=8192.0, slow=1.0, fast=4.0)], ids=str)
def test_a_stretch_of_no_kind(pkg, given):
    """(they were left out of account, and the frequencies those of no stretch)"""
    with pytest.raises(ValueError, match="kind"):
        pkg.ops.rotary_frequencies(1e4, 64, **given)
