"""Norms and rotation of heads where no GPU is: the kernel's addresses and refusals on the CPU model, and the frequencies."""
import os
import subprocess

import numpy as np
import pytest


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_addresses_and_refusals_on_the_cpu_model(tmp_path):
    """tests/host/rotary_model.cpp: the kernel thread by thread, every access checked, in every layout and alignment; and what the entry
    points refuse."""
    out = str(tmp_path / "model")
    build = subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "host"), "OUT=" + out, "rotary_model"], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-2000:] + build.stderr[-2000:]
    run = subprocess.run([os.path.join(out, "rotary_model")], capture_output=True, text=True, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout[-2000:] + run.stderr[-2000:]


@pytest.mark.parametrize("dim", [2, 64, 128, 250])
def test_frequencies(pkg, dim):
    """Formed in 64 bits, rounded once: at most half a step (2^-24 of a frequency) and the 64-bit formula's own few steps off."""
    ops, theta, i = pkg.ops, 5e5, np.arange(dim // 2)
    f = theta ** (-2.0 * i / dim)

    def near(got, want):
        assert got.dtype == np.float32 and np.all(np.abs(got - want) <= want * (2.0 ** -24 + 2.0 ** -45))
    near(ops.rotary_frequencies(theta, dim), f)
    near(ops.rotary_frequencies(theta, dim, ops.ROTARY_LINEAR, 8.0), f / 8)
    base = theta * (4.0 ** (dim / (dim - 2)) if dim > 2 else 1)
    near(ops.rotary_frequencies(theta, dim, ops.ROTARY_BASE, 4.0), base ** (-2.0 * i / dim))
    turns = 8192 * f / (2 * np.pi)
    keep = np.clip((turns - 1) / (32 - 1), 0, 1)
    near(ops.rotary_frequencies(theta, dim, ops.ROTARY_BY_PARTS, 16.0, 8192, 1, 32), f / 16 * (1 - keep) + f * keep)
    if dim > 2:   # the slowest pair is slowed by the whole factor, the fastest by nothing
        slow = ops.rotary_frequencies(theta, dim, ops.ROTARY_BASE, 4.0)
        assert slow[0] == 1 and abs(slow[-1] * 4 / f[-1] - 1) < 1e-6


def test_frequencies_refused(pkg):
    ops = pkg.ops
    assert ops.rotary_frequencies(1e4, 0).size == 0
    for args, code in (((0.0, 64), 1), ((-1.0, 64), 1), ((float("nan"), 64), 1), ((float("inf"), 64), 1), ((1e4, 63), 1), ((1e4, -2), 1), ((1e4, 64, 4), 2), ((1e4, 64, 0), 2),
                       ((1e4, 64, 1, 0.5), 1), ((1e4, 64, 1, float("inf")), 1), ((1e4, 64, 1, float("nan")), 1), ((1e4, 64, 3, 2.0, 0.0, 1, 32), 1),
                       ((1e4, 64, 3, 2.0, 8192, 32, 32), 1), ((1e4, 64, 3, 2.0, 8192, -1, 32), 1), ((1e4, 64, 3, 2.0, float("inf"), 1, 32), 1)):
        with pytest.raises(pkg.HipComputeError) as e:
            ops.rotary_frequencies(*args)
        assert e.value.code == code and "hipc_rotary_frequencies" in e.value.message


def test_calls_without_a_context_are_refused(pkg):
    lib, heads, cache = pkg.load_library(), pkg.RotaryHeads(1, 1, 64, 0, 0, 0.0, 0.0, None, None, None), pkg.Kv4Cache()
    assert lib.hipc_rotary(None, heads, pkg.F16, None, 1, None, 64, None, 64, None, 64, None, 64) == 1
    assert lib.hipc_kv4_append_rotary(None, cache, heads, pkg.F16, None, 1, None, 64, None, 64, None, 64, None, 64) == 1


def test_operands_that_do_not_fit_each_other(pkg):
    ops = pkg.ops

    class Host:      # takes uploads, runs nothing
        def upload(self, array, buf=None, offset=0):
            return type("Buffer", (), {"ptr": 0})()
    with pytest.raises(ValueError):
        ops.Rotary(Host(), 4, 2, 64, np.zeros((2, 16), np.float32))
    with pytest.raises(ValueError):
        ops.Rotary(Host(), 4, 2, 64, np.zeros(32, np.float32), q_norm=np.ones(32))
    turn = ops.Rotary(Host(), 4, 2, 64, np.zeros(32, np.float32), k_norm=np.ones(64))
    q, k, at = np.zeros((6, 4, 64), np.float16), np.zeros((6, 2, 64), np.float16), np.zeros(6, np.int32)
    pages = ops.Kv4Pages(Host(), 2, 16, 2, 64, np.zeros((2, 1), np.int32))
    for call in (lambda: turn(q, k, at[:5]), lambda: turn(q, k[:5], at), lambda: turn(q, k.astype(np.float32), at), lambda: turn(q[:, :3], k, at), lambda: turn(q[..., :32], k, at),
                 lambda: pages.append_rotary(turn, q, k, k, [6]), lambda: pages.append_rotary(turn, q, k, k, [4, 3]), lambda: pages.append_rotary(turn, q, k, k[:, :1], [3, 3]),
                 lambda: pages.append_rotary(turn, q[:, :2], k, k, [3, 3]), lambda: pages.append_rotary(turn, q, k, k.astype(np.float32), [3, 3])):
        with pytest.raises(ValueError):
            call()
