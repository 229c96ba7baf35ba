"""Norms of heads and their rotation on the GPU against the formulas in 64 bits, and their way into the 4-bit cache against the two calls that
it stands for.

Tolerances, of a result y with |x^_a cos| + |x^_b sin| = S (the oracle's second result):
  angles   position * frequency is off by 2^-51 of itself (stated), sine and cosine by a few steps of 64 bits more: A (|x^_a| + |x^_b|) (2^-51 angle + 2^-50);
           |x^_a| + |x^_b| is at most 2 S A^-1 / max(|cos|, |sin|) <= 2 sqrt(2) S_pair / A, S_pair the larger of the pair's two S
  values   f32: the sum of dim squares and the mean, off by (dim + 2) 2^-24 and halved by the root, which rounds with its reciprocal (3 steps); two products, cosine
           and sine times the amplitude, two products and a sum: (dim / 2 + 12) 2^-24 S, then the rounding to the type
"""
import numpy as np
import pytest

from oracle import attention as ref
from test_kv4_gpu import Pair, bits

pytestmark = pytest.mark.gpu

HALF_STEP = {np.dtype(np.float16): (2.0 ** -11, 2.0 ** -25), np.dtype(np.float32): (2.0 ** -24, 2.0 ** -150)}


def table(dim, base=1e4):
    return (base ** (-2.0 * np.arange(dim // 2) / max(dim, 1))).astype(np.float32)


def check(got, x, positions, frequencies, norm, eps=1e-6, interleaved=False, amplitude=1.0):
    want, size = ref.rotary(x, positions, frequencies, norm, eps, interleaved, amplitude)
    n, dim = len(frequencies), x.shape[2]
    pair = size.copy()
    angle = np.zeros(size.shape)
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        pair[..., a] = pair[..., b] = np.maximum(size[..., a], size[..., b])
        angle[..., a] = angle[..., b] = np.abs(positions.astype(np.float64) * np.float64(frequencies[i]))[:, None]
    step, least = HALF_STEP[x.dtype]
    allowed = 2 * 2 ** 0.5 * pair * (angle * 2.0 ** -51 + 2.0 ** -50) + (dim / 2 + 12) * 2.0 ** -24 * size
    allowed = allowed * (1 + step) + np.abs(want) * step + least
    off = np.abs(got.astype(np.float64) - want) - allowed
    assert got.dtype == x.dtype and np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("heads,kv,dim,turn", [(32, 8, 128, 128), (4, 1, 256, 256), (9, 3, 64, 32), (5, 5, 96, 24), (3, 1, 100, 36), (2, 7, 33, 10), (1, 1, 512, 512), (1, 2, 510, 0), (3, 2, 2, 2)],
                         ids=lambda v: str(v))
@pytest.mark.parametrize("rows", [1, 37], ids=str)
def test_against_the_formulas(ctx, pkg, dtype, interleaved, heads, kv, dim, turn, rows):
    rng = np.random.default_rng(dim * 3 + turn + rows)
    f = table(turn)
    norms = [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
    q, k = (2 * rng.standard_normal((rows, h, dim)).astype(dtype) for h in (heads, kv))
    at = rng.integers(-1000, 100000, rows).astype(np.int32)
    for qn, kn, amplitude in ((norms[0], norms[1], 1.0), (None, norms[1], 1.25), (norms[0], None, -0.5)):
        turning = pkg.ops.Rotary(ctx, heads, kv, dim, f, qn, kn, 1e-6, interleaved, amplitude)
        got_q, got_k = turning(q, k, at)
        turning.free()
        check(got_q, q, at, f, qn, 1e-6, interleaved, amplitude)
        check(got_k, k, at, f, kn, 1e-6, interleaved, amplitude)


def test_positions_far_out(ctx, pkg):
    """Up to the last 32-bit position on either side: angles of a billion and more."""
    rng = np.random.default_rng(1)
    at = np.array([0, 1, -1, 2 ** 20 + 1, 10 ** 9 + 7, 2 ** 31 - 1, -2 ** 31, 16777217], np.int32)
    f = table(128, 1e6)
    q, k = (rng.standard_normal((8, h, 128)).astype(np.float32) for h in (2, 1))
    turning = pkg.ops.Rotary(ctx, 2, 1, 128, f)
    got_q, got_k = turning(q, k, at)
    turning.free()
    check(got_q, q, at, f, None)
    check(got_k, k, at, f, None)
    assert np.array_equal(bits(got_q[0]), bits(q[0])) and np.array_equal(bits(got_k[0]), bits(k[0]))   # position 0 turns nothing


def test_many_rows(ctx, pkg):
    """A row a wavefront, and as many as leave the device's last workgroup in part."""
    rng = np.random.default_rng(2)
    rows, f = 2051, table(64)
    q, k = (rng.standard_normal((rows, h, 64)).astype(np.float16) for h in (10, 3))
    at = np.arange(rows, dtype=np.int32)
    w = (1 + 0.2 * rng.standard_normal(64)).astype(np.float32)
    turning = pkg.ops.Rotary(ctx, 10, 3, 64, f, w, w)
    got_q, got_k = turning(q, k, at)
    turning.free()
    check(got_q, q, at, f, w)
    check(got_k, k, at, f, w)


def test_unusual_values(ctx, pkg):
    """Zero heads, infinities and NaN stay with their head (and, not normed, with their pair); least and largest numbers."""
    f = table(32)
    x = np.ones((1, 6, 64), np.float16)
    x[0, 0] = 0
    x[0, 1, 3], x[0, 2, 40] = np.nan, np.inf
    x[0, 3], x[0, 4] = 65504, 2.0 ** -24
    at = np.array([5], np.int32)
    w = np.ones(64, np.float32)
    for norm in (None, w):
        turning = pkg.ops.Rotary(ctx, 6, 6, 64, f, norm, norm, 1e-6)
        q, k = turning(x, x, at)
        turning.free()
        for got in (q, k):
            assert not got[0, 0].any()
            nan = np.isnan(got.astype(np.float32))
            if norm is None:
                assert nan[0, 1].sum() == 2 and nan[0, 1, 3] and nan[0, 1, 19]       # channels 3 and 16 + 3 turn together
                assert np.isposinf(got[0, 2, 40].astype(np.float32)) and np.isfinite(got[0, 2, :40].astype(np.float32)).all()   # channel 40 does not turn
            else:
                assert nan[0, 1].all() and nan[0, 2, 40] and not got[0, 2, 0]        # an infinite mean
            assert np.isfinite(got[0, 5].astype(np.float32)).all()
            check(got[:, [0, 4, 5]], x[:, [0, 4, 5]], at, f, norm)


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("off,pad", [(0, 0), (8, 24), (4, 4), (1, 3)], ids=str)
def test_rows_of_a_projection_in_place(ctx, pkg, dtype, off, pad):
    """q|k|v side by side, at any alignment, turned where they lie: values and what lies between rows stay as they are."""
    rng = np.random.default_rng(off + pad)
    heads, kv, dim, rows = 4, 2, 64, 9
    width = (heads + 2 * kv) * dim + pad
    flat = rng.standard_normal(off + rows * width).astype(dtype)
    rowed = flat[off:].reshape(rows, width)
    q, k = (np.ascontiguousarray(rowed[:, a * dim:b * dim]).reshape(rows, -1, dim) for a, b in ((0, heads), (heads, heads + kv)))
    f, w, at = table(64), (1 + 0.1 * rng.standard_normal(64)).astype(np.float32), rng.integers(0, 5000, rows).astype(np.int32)
    turning = pkg.ops.Rotary(ctx, heads, kv, dim, f, w, None)
    size = flat.itemsize
    d, dP = ctx.upload(flat), ctx.upload(at)
    dq, dk = d.at(off * size), d.at((off + heads * dim) * size)
    pkg.ops.rotary_device(ctx, turning.heads, pkg.runtime.hipc_dtype(flat.dtype), dP, rows, dq, width, dk, width, dq, width, dk, width)
    got = ctx.download(d, dtype, flat.shape)
    want_q, want_k = turning(q, k, at)
    out = got[off:].reshape(rows, width)
    close = [np.ascontiguousarray(out[:, a * dim:b * dim]).reshape(rows, -1, dim) for a, b in ((0, heads), (heads, heads + kv))]
    check(close[0], q, at, f, w)
    assert np.array_equal(bits(close[1]), bits(want_k))
    assert np.array_equal(bits(out[:, (heads + kv) * dim:]), bits(rowed[:, (heads + kv) * dim:])) and np.array_equal(bits(got[:off]), bits(flat[:off]))
    for b in (d, dP):
        b.free()
    turning.free()


def test_queries_or_keys_alone(ctx, pkg):
    rng = np.random.default_rng(4)
    f, at = table(64), np.arange(5, dtype=np.int32) * 100
    x = rng.standard_normal((5, 3, 64)).astype(np.float16)
    turning = pkg.ops.Rotary(ctx, 3, 3, 64, f)
    both = turning(x, x, at)
    dX, dP, dY = ctx.upload(x), ctx.upload(at), ctx.upload(np.zeros_like(x))
    for which in range(2):
        heads = pkg.RotaryHeads(3 * (1 - which), 3 * which, 64, 64, 0, 0.0, 0.0, turning.heads.frequencies, None, None)
        args = [dX, 192, None, 0, dY, 192, None, 0] if which == 0 else [None, 0, dX, 192, None, 0, dY, 192]
        pkg.ops.rotary_device(ctx, heads, pkg.F16, dP, 5, *args)
        assert np.array_equal(bits(ctx.download(dY, np.float16, x.shape)), bits(both[which]))
    for b in (dX, dP, dY):
        b.free()
    turning.free()


def test_turning_by_parts_adds_up(ctx, pkg):
    """By 700 and then by -300 is by 400 (in f32: two roundings of 2^-24 more, and queries' products)."""
    rng = np.random.default_rng(5)
    f, x = table(64), rng.standard_normal((4, 2, 64)).astype(np.float32)
    turning = pkg.ops.Rotary(ctx, 2, 2, 64, f)
    _, far = turning(x, x, np.full(4, 700, np.int32))
    _, back = turning(far, far, np.full(4, -300, np.int32))
    turning.free()
    want, size = ref.rotary(x, np.full(4, 400), f)
    assert np.all(np.abs(back - want) <= 6 * 2.0 ** -24 * (np.abs(x).max() * 2))


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("heads,kv,dim,turn,page", [(32, 8, 128, 128, 16), (4, 1, 256, 64, 64), (3, 3, 96, 24, 16), (14, 2, 64, 64, 32), (5, 5, 160, 36, 16), (6, 9, 32, 10, 16)], ids=str)
def test_into_the_cache_is_the_two_calls(ctx, pkg, dtype, interleaved, heads, kv, dim, turn, page):
    """Bit for bit: queries, codes and parameters; also where pages are missing, rows lie in front of a sequence, and sequences bring nothing."""
    rng = np.random.default_rng(dim + turn)
    new, lengths = [5, 0, 40, 1], [5, 3, 97, 33]
    one, two = (Pair(ctx, pkg, np.random.default_rng(9), 4, -(-100 // page), page, kv, dim) for _ in range(2))
    lost = one.ref.table.copy()
    lost[2, 60 // page] = -1      # a page of the third sequence is given back
    for c in (one, two):
        c.gpu.set_table(lost)
        c.gpu.set_lengths(lengths)
    rows = sum(new)
    q, k, v = (rng.standard_normal((rows, h, dim)).astype(dtype) for h in (heads, kv, kv))
    w = [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
    turning = pkg.ops.Rotary(ctx, heads, kv, dim, table(turn), w[0], w[1], 1e-5, interleaved)
    at = np.concatenate([np.arange(n - m, n) for m, n in zip(new, lengths)]).astype(np.int32)
    want_q, want_k = turning(q, k, at)
    got_q = one.gpu.append_rotary(turning, q, k, v, new)
    two.gpu.append(want_k, v, new)
    assert np.array_equal(bits(got_q), bits(want_q))
    for a, b in zip(one.gpu.buffers, two.gpu.buffers):
        a, b = (ctx.download(x, np.uint8, (x.nbytes,)) for x in (a, b))
        assert np.array_equal(a, b) and a.any()
    # ... and what is stored is the definition's, of the turned keys
    three = ref.Cache(one.ref.codes[0].shape[0], page, kv, dim, lost)
    i = 0
    for s, (m, n) in enumerate(zip(new, lengths)):
        for p in range(n - m, n):
            three.store(s, p, (want_k[i], v[i]))
            i += 1
    for b, want in zip(one.gpu.buffers, (three.codes[0], three.params[0], three.codes[1], three.params[1])):
        assert np.array_equal(ctx.download(b, want.dtype, want.shape).view(np.uint8), want.view(np.uint8))
    one.gpu.free(), two.gpu.free(), turning.free()


def test_rows_outside_every_sequence_are_left(ctx, pkg):
    rng = np.random.default_rng(6)
    pages = pkg.ops.Kv4Pages(ctx, 4, 16, 2, 64, [[0, 1], [2, 3]])
    pages.set_lengths([6, 3])
    turning = pkg.ops.Rotary(ctx, 4, 2, 64, table(64))
    q, k, v = (rng.standard_normal((12, h, 64)).astype(np.float16) for h in (4, 2, 2))
    d = [ctx.upload(x) for x in (q, k, v, np.full_like(q, 7), np.array([2, 5, 10], np.int32))]   # rows 0, 1, 10 and 11 are nobody's; two lie in front of position 0
    pkg.ops.kv4_append_rotary_device(ctx, pages.cache, turning.heads, pkg.F16, d[4], 12, d[0], 256, d[1], 128, d[2], 128, d[3], 256)
    got = ctx.download(d[3], np.float16, q.shape)
    at = np.concatenate([np.arange(3, 6), np.arange(-2, 3)]).astype(np.int32)
    want, _ = turning(q[2:10], k[2:10], at)
    assert np.all(got[[0, 1, 10, 11]] == 7) and np.array_equal(bits(got[2:10]), bits(want))
    for b in d:
        b.free()
    pages.free(), turning.free()


def test_recorded_steps_follow_positions_and_lengths(ctx, pkg):
    """A recorded pair of calls, replayed with other positions and lengths, gives what the calls give."""
    rng = np.random.default_rng(7)
    f = table(128)
    turning = pkg.ops.Rotary(ctx, 8, 2, 128, f)
    pages, again = (pkg.ops.Kv4Pages(ctx, 12, 16, 2, 128, np.arange(12).reshape(3, 4)) for _ in range(2))
    q, k, v = (rng.standard_normal((3, h, 128)).astype(np.float16) for h in (8, 2, 2))
    at = np.array([3, 4, 5], np.int32)
    d = [ctx.upload(x) for x in (q, k, v, at, np.arange(4, dtype=np.int32), np.zeros_like(q), np.zeros_like(q), np.zeros_like(k))]

    def enqueue(cache):
        pkg.ops.rotary_device(ctx, turning.heads, pkg.F16, d[3], 3, d[0], 1024, d[1], 256, d[5], 1024, d[7], 256)
        pkg.ops.kv4_append_rotary_device(ctx, cache, turning.heads, pkg.F16, d[4], 3, d[0], 1024, d[1], 256, d[2], 256, d[6], 1024)

    def results():
        return [bits(ctx.download(b, np.float16, s)) for b, s in ((d[5], q.shape), (d[6], q.shape), (d[7], k.shape))]
    ctx.capture_begin()
    enqueue(pages.cache)
    graph = ctx.capture_end()
    for n in ([1, 1, 1], [20, 33, 64], [2, 34, 7]):
        for p in (pages, again):
            p.set_lengths(n)
        ctx.upload(at + np.array(n, np.int32), d[3])
        ctx.graph_launch(graph)
        got = results()
        enqueue(again.cache)
        for x, y in zip(got, results()):
            assert np.array_equal(x, y)
        for x, y in zip(pages.read([1, 1, 1]), again.read([1, 1, 1])):
            assert np.array_equal(bits(x), bits(y))
    ctx.graph_destroy(graph)
    for b in d:
        b.free()
    pages.free(), again.free(), turning.free()


def test_prompts_are_turned_as_the_decode_step_turns(ctx, pkg):
    """The decode step's own norm and rotation (the oracle's, angles in f32: off by up to 2^-21 of themselves, frequencies included) of the same rows."""
    from oracle import decoder
    rng = np.random.default_rng(8)
    q, k = (rng.standard_normal((40, h, 256)).astype(np.float32) for h in (4, 1))
    w = [(1 + 0.1 * rng.standard_normal(256)).astype(np.float32) for _ in range(2)]
    at = (np.arange(40) * 50).astype(np.int32)
    turning = pkg.ops.Rotary(ctx, 4, 1, 256, pkg.ops.rotary_frequencies(1e4, 256), w[0], w[1], 1e-6)
    for got, x, norm in zip(turning(q, k, at), (q, k), w):
        for r in range(40):
            for h in range(x.shape[1]):
                want = decoder.rope_half(decoder.rmsnorm(x[r, h], norm, 1e-6), int(at[r]), 1e4)
                size = np.abs(x[r, h]).max() * 2
                assert np.all(np.abs(got[r, h] - want) <= size * (float(at[r]) * 2.0 ** -21 + 2.0 ** -18))
    turning.free()
