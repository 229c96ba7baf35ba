"""Attention of packed new rows over the 4-bit cache, where no device is needed: what is refused without one."""
import numpy as np
import pytest


def test_a_call_without_a_context_is_refused(pkg):
    assert pkg.load_library().hipc_kv4_prompt_attention(None, pkg.Kv4Cache(), pkg.AttentionHeads(4, 2, 64, 1, 0, 0.0), 0, pkg.F16, None, 1, None, 256, None, 256) == 1


def test_rows_that_do_not_fit_the_cache(pkg):
    class Host:      # takes uploads, runs nothing
        def upload(self, array, buf=None, offset=0):
            return type("Buffer", (), {"ptr": 0})()
    pages = pkg.ops.Kv4Pages(Host(), 4, 16, 2, 64, np.zeros((2, 2), np.int32))
    q = np.zeros((6, 4, 64), np.float16)
    for rows, new in ((q[..., :32], [3, 3]), (q, [6]), (q, [3, 4]), (q, [-1, 3]), (q, [1, 2, 3])):
        with pytest.raises(ValueError):
            pages.prompt_attention(rows, new)
    with pytest.raises(KeyError):      # (no element type of the library)
        pages.prompt_attention(q.astype(np.float64), [3, 3])
