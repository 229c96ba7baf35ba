"""Rows that are turned where they lie: at the same distance from each other, or the call is refused (rows would be read after others had been written over them)."""
import numpy as np
import pytest

from test_kv4_gpu import bits
from test_rotary_gpu import table

pytestmark = pytest.mark.gpu


def test_another_distance_is_refused(ctx, pkg):
    rng = np.random.default_rng(1)
    turn = pkg.ops.Rotary(ctx, 2, 2, 64, table(64))
    pages = pkg.ops.Kv4Pages(ctx, 1, 16, 2, 64, [[0]])
    pages.set_lengths([4])
    x = rng.standard_normal((4, 256)).astype(np.float16)
    d, other, at, starts = ctx.upload(x), ctx.upload(x), ctx.upload(np.arange(4, dtype=np.int32)), ctx.upload(np.array([0, 4], np.int32))

    def rotary(rows, q, qo, ko, q_to=d, k_to=other):
        return ctx.lib.hipc_rotary(ctx.handle, turn.heads, pkg.F16, at.ptr, rows, d.ptr, q, other.ptr, 256, q_to.ptr, qo, k_to.ptr, ko)

    def append(q, qo, q_to=d):
        return ctx.lib.hipc_kv4_append_rotary(ctx.handle, pages.cache, turn.heads, pkg.F16, starts.ptr, 4, d.ptr, q, other.ptr, 256, other.ptr, 256, q_to.ptr, qo)
    assert rotary(4, 256, 128, 256) == 1 and rotary(4, 128, 256, 256) == 1 and rotary(4, 256, 256, 128) == 1 and append(256, 128) == 1
    assert b"hipc_kv4_append_rotary" in ctx.lib.hipc_last_error(ctx.handle)
    assert np.array_equal(bits(ctx.download(d, np.float16, x.shape)), bits(x)) and np.array_equal(bits(ctx.download(other, np.float16, x.shape)), bits(x))
    spare = [ctx.alloc(x.nbytes) for _ in range(2)]
    assert rotary(1, 256, 128, 128) == 0 and rotary(4, 256, 128, 128, *spare) == 0 and append(256, 128, spare[0]) == 0 and rotary(4, 256, 256, 256) == 0 and append(256, 256) == 0
    ctx.flush()
    for b in (d, other, at, starts, *spare):
        b.free()
    pages.free(), turn.free()
