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


@pytest.mark.parametrize("theta,dim,more", [(1e-45, 64, ()), (1e-300, 4, ()), (5e-324, 128, (1, 2.0))], ids=str)
def test_bases_whose_frequencies_f32_does_not_hold(pkg, theta, dim, more):
    """theta^(-2i / dim) past f32's numbers: an infinite frequency would make NaN of every row."""
    with pytest.raises(pkg.HipComputeError) as e:
        pkg.ops.rotary_frequencies(theta, dim, *more)
    assert e.value.code == 1 and "hipc_rotary_frequencies" in e.value.message


def test_bases_below_one(pkg):
    assert np.allclose(pkg.ops.rotary_frequencies(0.25, 4), [1, 2], rtol=2 ** -23) and np.all(np.isfinite(pkg.ops.rotary_frequencies(1e-38, 64)))
