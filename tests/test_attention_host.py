"""Attention, the 4-bit cache and token log-probabilities where no GPU is: refusals, and the cache's addresses on the CPU model."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cache_addresses_and_refusals_on_the_cpu_model(tmp_path):
    """tests/host/kv4_model.cpp: the storing and reading kernels thread by thread, every access checked: page numbers that are none,
    lengths past the table and below zero, rows outside the sequence; and what the entry points refuse."""
    out = str(tmp_path / "model")
    build = subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "host"), "OUT=" + out, "kv4_model"], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-2000:] + build.stderr[-2000:]
    run = subprocess.run([os.path.join(out, "kv4_model")], capture_output=True, text=True, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout[-2000:] + run.stderr[-2000:]


def test_a_call_without_a_context_is_refused(pkg):
    lib, heads, cache = pkg.load_library(), pkg.AttentionHeads(1, 1, 64, 1, 0, 0.0), pkg.Kv4Cache()
    assert lib.hipc_prompt_attention(None, heads, pkg.F16, None, 64, None, 64, None, 64, None, None, 1, 1, 1, None, 64) == 1
    assert lib.hipc_kv4_append(None, cache, pkg.F16, None, 1, None, 64, None, 64) == 1
    assert lib.hipc_kv4_read(None, cache, pkg.F16, None, 1, None, 64, None, 64) == 1
    assert lib.hipc_kv4_attention(None, cache, heads, pkg.F16, 1, None, 64, None, 64) == 1
    assert lib.hipc_token_logprobs(None, pkg.F32, None, 8, 1, 8, None, None, None, 0, None, None) == 1


def test_operands_that_do_not_fit_each_other(pkg):
    """The numpy calls refuse them before anything is enqueued (there is no context here to enqueue on)."""
    ops, x = pkg.ops, np.zeros((6, 2, 64), np.float16)
    for q, k, v, lengths in ((x, x.astype(np.float32), x, [6]), (x, x, x[:5], [5]), (x, x[:, :, :32], x[:, :, :32], [6]), (x, x, x, [7]),
                             (x, x, x, [4, -1]), (x, x, x[:, :1], [6])):
        with pytest.raises(ValueError):
            ops.prompt_attention(None, q, k, v, lengths)
    with pytest.raises(ValueError):
        ops.prompt_attention(None, x, x, x, [3, 3], [6])
    with pytest.raises(ValueError):
        ops.token_logprobs(None, np.zeros((2, 8), np.float32), [1])
    with pytest.raises(ValueError):
        ops.Kv4Pages(None, 2, 16, 2, 64, np.zeros(3, np.int32))

    class Host:      # takes uploads, runs nothing
        def upload(self, array, buf=None, offset=0):
            return type("Buffer", (), {"ptr": 0})()
    pages = ops.Kv4Pages(Host(), 2, 16, 2, 64, np.zeros((2, 1), np.int32))
    pages.set_lengths([3, 4]), pages.set_table([[1], [0]])
    for call in (lambda: pages.set_lengths([3]), lambda: pages.set_lengths([3, 4, 5]), lambda: pages.set_table([[0, 1], [0, 1]]),
                 lambda: pages.append(x, x, [6]), lambda: pages.append(x, x, [5, 2]), lambda: pages.append(x, x.astype(np.float32), [3, 3]),
                 lambda: pages.append(x[:, :1], x[:, :1], [3, 3]), lambda: pages.read([1, 1, 1]), lambda: pages.read([2, -1]),
                 lambda: pages.attention(x), lambda: pages.attention(x[:2, :, :32])):
        with pytest.raises(ValueError):
            call()
