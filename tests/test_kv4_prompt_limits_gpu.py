"""Rotation and attention of packed rows over the 4-bit cache where single calls of ordinary size do not go: offsets past 2^31 elements and 2^32 bytes, recorded
calls that share scratch memory, two contexts, wavefronts that share rows, and what is refused."""
import threading

import numpy as np
import pytest

from oracle import attention as ref
from test_kv4_gpu import Pair, bits
from test_kv4_prompt_gpu import case, starts_of
from test_rotary_gpu import table as frequencies

pytestmark = pytest.mark.gpu


def heads(pkg, q_heads, kv, dim, window=0):
    return pkg.AttentionHeads(q_heads, kv, dim, 1, window, 0.0)


def test_a_cache_of_ten_gigabytes(ctx, pkg):
    """Pages past 2^32 bytes of codes: turned, stored and attended to as in a small cache, by either kernel. (Only the pages in use are ever touched.)"""
    kv, dim, page, pages, new = 8, 128, 64, 140001, [150, 129]
    rows, rng = pages * kv * page, np.random.default_rng(2)
    small = pkg.ops.Kv4Pages(ctx, 6, page, kv, dim, [[5, 0, 2], [3, 4, 1]])
    buffers = [ctx.alloc(rows * dim // 2), ctx.alloc(rows * dim // 32 * 4), ctx.alloc(rows * dim // 2), ctx.alloc(rows * dim // 32 * 4)]
    dT = ctx.upload(np.array([[pages - 1, 0, 70001], [139000, pages - 2, 5]], np.int32))
    small.set_lengths(new)
    cache = pkg.Kv4Cache(*(b.ptr for b in buffers), pages, page, kv, dim, 2, small.lengths.ptr, dT.ptr, 3)
    turn = pkg.ops.Rotary(ctx, 32, kv, dim, frequencies(dim))
    q = rng.standard_normal((279, 32, dim)).astype(np.float16)
    k, v = (rng.standard_normal((279, kv, dim)).astype(np.float16) for _ in range(2))
    want_q = small.append_rotary(turn, q, k, v, new)
    dQ, dK, dV, dS, dY = (ctx.upload(x) for x in (q, k, v, starts_of(new), np.zeros_like(q)))
    pkg.ops.kv4_append_rotary_device(ctx, cache, turn.heads, pkg.F16, dS, 279, dQ, 32 * dim, dK, kv * dim, dV, kv * dim, dQ, 32 * dim)
    assert np.array_equal(bits(ctx.download(dQ, np.float16, q.shape)), bits(want_q))
    pkg.ops.kv4_read_device(ctx, cache, pkg.F16, dS, 279, dK, kv * dim, dV, kv * dim)
    for d, want in zip((dK, dV), small.read(new)):
        assert np.array_equal(bits(ctx.download(d, np.float16, k.shape)), bits(want)) and want.any()
    for options in ({}, dict(HIPC_PROMPT_WAVES=4), dict(HIPC_PROMPT_WAVES=8)):
        for few in ([150, 129], [3, 1]):
            n = sum(few)
            ctx.upload(starts_of(few), dS)
            with ctx.options(**options):
                pkg.ops.kv4_prompt_attention_device(ctx, cache, heads(pkg, 32, kv, dim), 0, pkg.F16, dS, n, dQ, 32 * dim, dY, 32 * dim)
                got = ctx.download(dY, np.float16, (n, 32, dim))
                assert np.array_equal(bits(got), bits(small.prompt_attention(want_q[:n], few))) and got.any()
    for b in buffers + [dT, dQ, dK, dV, dS, dY]:
        b.free()
    small.free()


@pytest.mark.parametrize("waves", [1, 4, 8])
def test_rows_far_apart(ctx, pkg, waves):
    """Rows of queries and results 2^25 elements apart: the last of 70 lie more than 2^32 bytes behind the first, for attention and rotation alike."""
    c, stride, new = case(ctx, pkg, [90], 16, 2, 64), 1 << 25, [70]
    q = c.rng.standard_normal((70, 4, 64)).astype(np.float16)
    dQ, dY = (ctx.alloc(2 * (69 * stride + 256)) for _ in range(2))
    for i in range(70):
        ctx.upload(q[i], dQ, 2 * stride * i)
    dS, dP = ctx.upload(starts_of(new)), ctx.upload(np.arange(70, dtype=np.int32))

    def rows():
        return np.stack([ctx.download(dY, np.float16, (4, 64), 2 * stride * i) for i in range(70)])
    with ctx.options(HIPC_PROMPT_WAVES=waves):
        pkg.ops.kv4_prompt_attention_device(ctx, c.gpu.cache, heads(pkg, 4, 2, 64), 0, pkg.F16, dS, 70, dQ, stride, dY, stride)
        assert np.array_equal(bits(rows()), bits(c.gpu.prompt_attention(q, new)))
    turn = pkg.ops.Rotary(ctx, 4, 2, 64, frequencies(64))
    alone = pkg.RotaryHeads(4, 0, 64, 64, 0, 0.0, 0.0, turn.heads.frequencies, None, None)
    pkg.ops.rotary_device(ctx, alone, pkg.F16, dP, 70, dQ, stride, None, 0, dY, stride, None, 0)
    near, _ = turn(q, np.zeros((70, 2, 64), np.float16), np.arange(70, dtype=np.int32))
    assert np.array_equal(bits(rows()), bits(near))
    for b in (dQ, dY, dS, dP):
        b.free()
    c.gpu.free()


def test_recorded_calls_that_share_scratch_memory(ctx, pkg):
    """Two graphs of one context, each with its own shapes and number of workgroups to a tile, replayed in turn with eager calls between: every replay is the eager result."""
    c, rng = case(ctx, pkg, [700, 300], 16, 4, 128), np.random.default_rng(5)
    held = []
    for new, options in (([200, 90], dict(HIPC_PROMPT_WAVES=4, HIPC_PROMPT_SPLIT=3)), ([1, 64], {}), ([300, 0], dict(HIPC_PROMPT_WAVES=8, HIPC_PROMPT_SPLIT=2))):
        q = rng.standard_normal((sum(new), 8, 128)).astype(np.float16)
        dQ, dY, dS = ctx.upload(q), ctx.upload(np.zeros_like(q)), ctx.upload(starts_of(new))
        with ctx.options(**options):
            eager = c.gpu.prompt_attention(q, new)
            ctx.capture_begin()
            pkg.ops.kv4_prompt_attention_device(ctx, c.gpu.cache, heads(pkg, 8, 4, 128), 0, pkg.F16, dS, sum(new), dQ, 1024, dY, 1024)
            held.append((ctx.capture_end(), q, new, options, eager, (dQ, dY, dS)))
    for turn in range(4):
        for graph, q, new, options, eager, (_, dY, _) in held:
            ctx.upload(np.zeros_like(q), dY)
            ctx.graph_launch(graph)
            assert np.array_equal(bits(ctx.download(dY, np.float16, q.shape)), bits(eager))
            with ctx.options(**options):
                assert np.array_equal(bits(c.gpu.prompt_attention(q, new)), bits(eager))
    for graph, *_, buffers in held:
        ctx.graph_destroy(graph)
        for b in buffers:
            b.free()
    c.gpu.free()


def test_two_contexts_turn_and_store_at_once(pkg):
    """Calls of two contexts overlap on the device; each gets what it gets alone."""
    ctxs = [pkg.Context(0) for _ in range(2)]
    rng = np.random.default_rng(8)
    cases = [(rng.standard_normal((n, 8, 128)).astype(np.float16), rng.standard_normal((n, 2, 128)).astype(np.float16)) for n in (300, 170)]

    def run(i, pages, turn):
        q, k = cases[i]
        return pages.append_rotary(turn, q, k, k, [len(q)]), *pages.read([len(q)]), pages.prompt_attention(q, [len(q)])
    made = []
    for i, ctx in enumerate(ctxs):
        n = len(cases[i][0])
        pages, turn = pkg.ops.Kv4Pages(ctx, 20, 16, 2, 128, [list(range(20))]), pkg.ops.Rotary(ctx, 8, 2, 128, frequencies(128), q_norm=np.full(128, 1.5, np.float32))
        pages.set_lengths([n])
        made.append((pages, turn, run(i, pages, turn)))
    wrong = []

    def work(i):
        for _ in range(10):
            got = run(i, *made[i][:2])
            if not all(np.array_equal(bits(x), bits(y)) for x, y in zip(got, made[i][2])):
                wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for (pages, *_), ctx in zip(made, ctxs):
        pages.free()
        ctx.close()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("split", [1, 3])
@pytest.mark.parametrize("waves", [4, 8])
def test_wavefronts_that_share_rows_repeat(ctx, pkg, dtype, split, waves):
    """Heads of 256: two wavefronts of a row exchange their halves of every tile's scores. Many tiles, some of which rows skip: the same bits every time."""
    c = case(ctx, pkg, [900, 500], 32, 1, 256)
    with ctx.options(HIPC_PROMPT_WAVES=waves, HIPC_PROMPT_SPLIT=split):
        q, first = c.attend(4, [400, 333], dtype)
        _, windowed = c.attend(4, [400, 333], dtype, 100, 5)
        for _ in range(8):
            assert np.array_equal(bits(c.gpu.prompt_attention(q, [400, 333])), bits(first))
    assert windowed.any()
    c.gpu.free()


def test_refusals(ctx, pkg):
    p = Pair(ctx, pkg, np.random.default_rng(1), 2, 1, 16, 2, 64)
    d = ctx.alloc(65536)
    good = {n: getattr(p.gpu.cache, n) for n, _ in pkg.Kv4Cache._fields_}

    def attend(shape=(4, 2, 64, 1, 0, 0.0), sinks=0, dtype=pkg.F16, starts=d.ptr, total=2, q=d.ptr, qs=256, y=d.ptr, ys=256, cache=True, **change):
        return ctx.lib.hipc_kv4_prompt_attention(ctx.handle, pkg.Kv4Cache(**{**good, **change}) if cache else None, pkg.AttentionHeads(*shape) if shape else None, sinks, dtype,
                                                 starts, total, q, qs, y, ys)
    assert attend(cache=False) == 1 and attend(shape=None) == 1 and attend(dtype=pkg.U8) == 2
    assert attend(head_dim=48) == 2 and attend(page_size=24) == 2 and attend(n_kv_heads=0) == 1 and attend(n_seqs=-1) == 1 and attend(lengths=None) == 1 and attend(table=None) == 1
    assert attend(shape=(4, 2, 64, 0, 0, 0.0)) == 1                       # not causal
    assert attend(shape=(4, 4, 64, 1, 0, 0.0)) == 1 and attend(shape=(4, 2, 32, 1, 0, 0.0)) == 1 and attend(shape=(3, 2, 64, 1, 0, 0.0)) == 1
    assert attend(shape=(4, 2, 64, 1, -1, 0.0)) == 1 and attend(shape=(4, 2, 64, 1, 0, float("nan"))) == 1 and attend(sinks=-1) == 1
    assert attend(total=-1) == 1 and attend(total=(1 << 30) + 1) == 1 and attend(total=1 << 30) == 2   # (two heads to a kv head: 2^31 query rows)
    assert attend(starts=None) == 1 and attend(starts=d.ptr + 2) == 1
    assert attend(q=None) == 1 and attend(y=None) == 1 and attend(q=d.ptr + 1) == 1 and attend(y=d.ptr + 1) == 1 and attend(qs=255) == 1 and attend(ys=0) == 1
    assert attend(qs=(1 << 40) + 1) == 1 and attend(dtype=pkg.F32, q=d.ptr + 2) == 1
    assert b"hipc_kv4_prompt_attention" in ctx.lib.hipc_last_error(ctx.handle)
    assert attend(total=0, starts=None, q=None, y=None) == 0 and attend(n_seqs=0, starts=None, q=None, y=None) == 0
    d.free()
    p.gpu.free()


def test_a_cache_without_pages(ctx, pkg):
    """No pages, and a table of no width: every row of a sequence is zero, by either kernel; what a rotation on the way would store is stored nowhere."""
    lengths, starts = ctx.upload(np.array([40, 3], np.int32)), ctx.upload(starts_of([40, 3]))
    cache = pkg.Kv4Cache(None, None, None, None, 0, 16, 2, 64, 2, lengths.ptr, None, 0)
    q = np.ones((45, 4, 64), np.float16)
    dQ, dY = ctx.upload(q), ctx.alloc(q.nbytes)
    for waves in (1, 4, 8):
        ctx.upload(q, dY)
        with ctx.options(HIPC_PROMPT_WAVES=waves):
            pkg.ops.kv4_prompt_attention_device(ctx, cache, heads(pkg, 4, 2, 64, 7), 2, pkg.F16, starts, 45, dQ, 256, dY, 256)
        got = ctx.download(dY, np.float16, q.shape)
        assert not got[:43].any() and np.all(got[43:] == 1)
    turn = pkg.ops.Rotary(ctx, 4, 2, 64, frequencies(64))
    pkg.ops.kv4_append_rotary_device(ctx, cache, turn.heads, pkg.F16, starts, 45, dQ, 256, dQ, 256, dQ, 256, dY, 256)
    want, _ = turn(q[:43], q[:43, :2], np.r_[np.arange(40), np.arange(3)].astype(np.int32))
    got = ctx.download(dY, np.float16, q.shape)
    assert np.array_equal(bits(got[:43]), bits(want)) and np.all(got[43:] == 1)
    for b in (lengths, starts, dQ, dY):
        b.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("waves", [1, 4, 8])
@pytest.mark.parametrize("q_heads,kv,dim", [(4, 2, 64), (2, 1, 128), (4, 1, 256)], ids=str)
def test_queries_that_are_no_numbers(ctx, pkg, dtype, waves, q_heads, kv, dim):
    """A head's row with a NaN or infinities is NaN (in f16, where every score is -inf, zero), a row that sees nothing is zero all the same, and every other row is as before."""
    c = case(ctx, pkg, [140, 30], 16, kv, dim)
    new = [90, 40]                                        # (the second sequence's first ten rows lie in front of it)
    q = c.rng.standard_normal((130, q_heads, dim)).astype(dtype)
    bad = q.copy()
    odd = {(3, 0): np.nan, (17, 1): np.inf, (60, 0): -np.inf, (89, 1): np.nan, (93, 0): np.nan, (95, 1): np.inf, (129, 1): -np.inf}
    for (row, head), x in odd.items():
        bad[row, head, 5] = x
    with ctx.options(HIPC_PROMPT_WAVES=waves):
        clean, got = c.gpu.prompt_attention(q, new), c.gpu.prompt_attention(bad, new)
    for row, head in odd:
        y = got[row, head]
        assert not y.any() if row in (93, 95) else np.isnan(y).all() or (dtype == np.float16 and not y.any())
        got[row, head] = clean[row, head]
    assert np.array_equal(bits(got), bits(clean)) and not clean[90:100].any()
    c.gpu.free()


@pytest.mark.parametrize("waves", [1, 4, 8])
@pytest.mark.parametrize("q_heads,kv,dim", [(4, 2, 64), (4, 1, 128), (2, 1, 256)], ids=str)
@pytest.mark.parametrize("scale", [0.0, 1.0, 1e-30, -1e-38, 3e-45])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)], ids=str)
def test_queries_and_scales_of_next_to_nothing(ctx, pkg, waves, q_heads, kv, dim, scale, window, sinks):
    """f32 rows down to the least number there is beside ordinary ones, with scales as small: scores of 0 to working precision make a row the mean of what it sees. The tolerance is
    test_kv4_prompt_gpu.py's for f32, with this scale in the place of 1 / sqrt(dim)."""
    c = case(ctx, pkg, [130, 65, 7], 32, kv, dim)
    new = [70, 33, 7]
    q = c.rng.standard_normal((110, q_heads, dim))
    sizes = np.array([0.0, 1e-45, 1e-42, 1e-39, 1e-35, 1e-20, 1.0])
    q = (q * sizes[np.arange(110 * q_heads) % len(sizes)].reshape(110, q_heads, 1)).astype(np.float32)
    with ctx.options(HIPC_PROMPT_WAVES=waves):
        got = c.gpu.prompt_attention(q, new, window, sinks, scale)
    want, weight, size, most = c.ref.prompt_attention(q, starts_of(new), c.lengths, window, sinks, scale or None)
    k_most = max(float(np.abs(ref.values(np.full((1, 1, 1), code, np.uint8), p[..., :1], p[..., 1:])).max()) for p in (c.ref.params[0].reshape(-1, 1, 2),) for code in (0, 15))
    relative = 2 * (dim + 2) * 2.0 ** -24 * size + (16 + 130) * 2.0 ** -24 + 2.0 ** -22
    relative = relative + 2 * 2.0 ** -22 * np.abs(q.astype(np.float64)).max(-1, keepdims=True) * dim * k_most * (abs(scale) or 1 / np.sqrt(dim))
    off = np.abs(got.astype(np.float64) - want) - (weight * relative + 130 * 2.0 ** -32 * most + 1e-37)
    assert np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))
    c.gpu.free()
