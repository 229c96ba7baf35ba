"""Attention of packed new rows over the 4-bit cache on the GPU against its definition in 64 bits.

Tolerance, from y = sum w v: with A = sum w |v| and S = scale * sum |q| |k| (both from the reference),
  * a score sums dim products in f32, off by at most (dim + 2) 2^-24 S, which moves every weight by twice that; an f32 query enters with 22 bits of its
    row's largest value: 2^-22 max|q| sum |k| scale more, sum |k| <= dim max |k|;
  * an exponential, a running rescale and the sums over the keys add less than (16 + keys) 2^-24 relative;
  * f16: a weight may be rounded to f16 for the second product, half a step (2^-11), or 2^-32 of the row's heaviest where it is smaller than 2^-21 of that; the
    result once more. f32: weights with 22 bits, 2^-22, or 2^-32 of the heaviest alike.
"""
import numpy as np
import pytest

from oracle import attention as ref
from test_kv4_gpu import Pair, bits
from test_rotary_gpu import check

pytestmark = pytest.mark.gpu


ROUTES = {"by size": {}, "four wavefronts": dict(HIPC_PROMPT_WAVES=4), "eight wavefronts": dict(HIPC_PROMPT_WAVES=8), "shared": dict(HIPC_PROMPT_WAVES=4, HIPC_PROMPT_SPLIT=3)}


@pytest.fixture(params=list(ROUTES))
def route(request, ctx):
    """Who takes sequences of more than 64 query rows: whoever the sizes ask for, or the kernel for many rows with so many wavefronts, its keys shared or not."""
    with ctx.options(**ROUTES[request.param]):
        yield request.param


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def check_rows(got, q, cache, starts, lengths, window=0, sinks=0, rows=None):
    want, weight, size, most = cache.prompt_attention(q, starts, lengths, window, sinks)
    rows = ~np.isnan(want).any((1, 2)) if rows is None else rows
    dim, keys = q.shape[2], max([int(n) for n in lengths] + [1])
    relative = 2 * (dim + 2) * 2.0 ** -24 * size + (16 + keys) * 2.0 ** -24
    if q.dtype == np.float32:
        k_most = max(float(np.abs(ref.values(np.full((1, 1, 1), c, np.uint8), p[..., :1], p[..., 1:])).max()) for p in (cache.params[0].reshape(-1, 1, 2),) for c in (0, 15))
        relative = relative + 2 * 2.0 ** -22 * np.abs(q.astype(np.float64)).max(-1, keepdims=True) * dim * k_most / np.sqrt(dim) + 2.0 ** -22
        tol = weight * relative + keys * 2.0 ** -32 * most + 1e-37
    else:
        tol = weight * (relative + 2.0 ** -11) + keys * 2.0 ** -32 * most + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    off = np.abs(got.astype(np.float64) - want) - tol
    assert np.all(off[rows] <= 0), (float(np.nanmax(off[rows])), np.argwhere(~(off <= 0) & rows[:, None, None])[:3])
    return want


class Case(Pair):
    def attend(self, heads, new, dtype, window=0, sinks=0, gain=1.5):
        q = (gain * self.rng.standard_normal((int(np.sum(new)), heads, self.dim))).astype(dtype)
        got = self.gpu.prompt_attention(q, new, window, sinks)
        check_rows(got, q, self.ref, starts_of(new), self.lengths, window, sinks)
        return q, got


def case(ctx, pkg, lengths, page, kv, dim, seed=0, table=None):
    c = Case(ctx, pkg, np.random.default_rng(sum(lengths) + dim + seed), len(lengths), -(-max(lengths) // page) + 1, page, kv, dim, table)
    c.append(lengths)
    return c


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("new,lengths", [([1], [1]), ([5], [5]), ([64], [64]), ([65, 1, 17], [65, 200, 80]), ([0, 3, 1, 0], [9, 3, 64, 0]), ([130], [131]), ([257, 1], [300, 513])], ids=str)
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 1, 256, 512), (8, 2, 128, 16), (3, 3, 64, 32)], ids=str)
def test_pieces_prompts_and_tokens(ctx, pkg, route, dtype, new, lengths, heads, kv, dim, page):
    c = case(ctx, pkg, lengths, page, kv, dim)
    c.attend(heads, new, dtype)
    c.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (4, 2, 96), (2, 2, 32), (5, 5, 160), (6, 1, 192), (3, 1, 224), (40, 1, 64), (7, 1, 128), (1, 1, 256)], ids=str)
def test_head_layouts(ctx, pkg, route, dtype, heads, kv, dim):
    c = case(ctx, pkg, [150, 40, 70], 16, kv, dim)
    c.attend(heads, [90, 2, 70], dtype)
    c.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 0), (64, 1), (1, 1), (100, 4), (64, 64), (20, 70), (128, 200), (1000, 4), (7, 1 << 30), (1 << 30, 3)], ids=str)
@pytest.mark.parametrize("new,lengths,heads,kv,dim", [([1, 1, 1], [400, 3, 70], 8, 2, 128), ([70, 5, 1], [380, 5, 66], 4, 1, 256), ([150, 40], [310, 41], 4, 4, 64)], ids=str)
def test_windows_and_first_positions(ctx, pkg, route, dtype, window, sinks, new, lengths, heads, kv, dim):
    c = case(ctx, pkg, lengths, 32, kv, dim, window + sinks)
    c.attend(heads, new, dtype, window, sinks)
    c.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
def test_rows_that_see_nothing_and_rows_that_are_nobodys(ctx, pkg, route, dtype):
    """Rows in front of the first sequence and behind the last, positions below 0, sequences without keys, starts out of range."""
    c = case(ctx, pkg, [30, 90, 5, 1], 16, 2, 64)
    for starts, lengths, total in (([3, 20, 70, 80, 81], [10, 90, 0, 1], 90), ([-5, 10, 40, 40, 60], [30, 90, 5, 1], 50), ([0, 50, 30, 30, 35], [30, 90, 5, 1], 40), ([0, 200, 200, 200, 200], [30, 9, 5, 1], 200)):
        q = c.rng.standard_normal((total, 4, 64)).astype(dtype)
        c.gpu.set_lengths(lengths)
        d = [ctx.upload(x) for x in (q, np.full_like(q, 7), np.array(starts, np.int32))]
        pkg.ops.kv4_prompt_attention_device(ctx, c.gpu.cache, pkg.AttentionHeads(4, 2, 64, 1, 0, 0.0), 0, pkg.runtime.hipc_dtype(q.dtype), d[2], total, d[0], 256, d[1], 256)
        got = ctx.download(d[1], dtype, q.shape)
        # (starts that do not ascend give a row to two sequences: which of the two answers it holds is left open, here rows 30 to 34 of the third call)
        owners = sum(((np.arange(total) >= a) & (np.arange(total) < b)).astype(int) for a, b in zip(starts, starts[1:]))
        want = check_rows(got, q, c.ref, starts, lengths, rows=owners == 1)
        nobody = np.isnan(want).any((1, 2))
        assert np.array_equal(nobody, owners == 0)
        assert np.all(got[nobody] == 7)
        unseen = (owners == 1) & ~want.any((1, 2))
        assert unseen.any() and not got[unseen].any()
        for b in d:
            b.free()
    c.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("new", [[1, 1], [90, 70], [3, 150]], ids=str)
def test_pages_that_are_no_pages(ctx, pkg, route, dtype, new):
    table = np.array([[3, -1, 0, 1 << 30, 9, 4, 17, 15, 16, 11, 14], [-7, 5, 99, 6, 7, 8, 1, 2, 10, -1, 12]], np.int32)
    c = case(ctx, pkg, [160, 150], 16, 2, 128, table=table)
    for window, sinks in ((0, 0), (20, 0), (64, 30), (100, 4)):
        c.attend(8, new, dtype, window, sinks)
    c.gpu.free()


@pytest.mark.parametrize("new", [[3, 1], [100, 90]], ids=str)
def test_lengths_past_the_table_and_below_zero(ctx, pkg, route, new):
    """Positions behind the table are not seen, though they count where a window does; a length below 0 counts as 0."""
    c = case(ctx, pkg, [100, 96], 32, 1, 64)
    held = c.ref.table.shape[1] * 32
    q = c.rng.standard_normal((sum(new), 4, 64)).astype(np.float16)
    for lengths, window, sinks in (([held + 2, -5], 0, 0), ([held + 2, 96], 40, 5), ([held + 100, 2], 50, 0), ([1 << 30, 2147483647], 0, 0), ([2147483647, -2147483648], 100, 3)):
        c.gpu.set_lengths(lengths)
        got = c.gpu.prompt_attention(q, new, window, sinks)
        want, _, _, _ = c.ref.prompt_attention(q, starts_of(new), lengths, window, sinks)
        near = [min(n, held + 200) for n in lengths]
        if lengths[0] <= held + 100:
            check_rows(got, q, c.ref, starts_of(new), near, window, sinks)
        assert np.array_equal(got.any((1, 2)), want.any((1, 2)))
    c.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("which", [0, 1], ids=["keys", "values"])
@pytest.mark.parametrize("new", [[4], [120]], ids=str)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_parameters_that_are_not_finite(ctx, pkg, route, dtype, which, new, value):
    """A position in the rows' midst: rows behind it are NaN (of a value: in its channels; infinite parameters make lowest + c * scale infinite for c > 0, and
    a weight times that is no NaN: there the result may be the infinity), rows in front of it are as without."""
    c = case(ctx, pkg, [150], 16, 2, 96)
    q = c.rng.standard_normal((new[0], 4, 96)).astype(dtype)
    want = c.gpu.prompt_attention(q, new)
    at = 150 - new[0] // 2
    page, place = c.ref.place(0, at)
    params = ctx.download(c.gpu.buffers[1 + 2 * which], np.float16, c.ref.params[which].shape)
    params[page, 1, place, 1, :] = value
    ctx.upload(params, c.gpu.buffers[1 + 2 * which])
    got = c.gpu.prompt_attention(q, new)
    before, behind = slice(0, new[0] - new[0] // 2), slice(new[0] - new[0] // 2, None)
    assert np.array_equal(bits(got[before]), bits(want[before])) and np.array_equal(bits(got[:, :2]), bits(want[:, :2]))
    nan = np.isnan(got[behind, 2:].astype(np.float32)) if which == 0 or np.isnan(value) else ~np.isfinite(got[behind, 2:].astype(np.float32))
    if which == 0:
        assert nan.all()
    else:
        assert nan[:, :, 32:64].all() and not nan[:, :, :32].any() and not nan[:, :, 64:].any()
        assert np.array_equal(bits(got[behind, 2:, :32]), bits(want[behind, 2:, :32]))
    # a window of 20 leaves it behind for later rows
    if new[0] > 60:
        got = c.gpu.prompt_attention(q, new, 20)
        assert not np.isnan(got[new[0] - new[0] // 2 + 20:].astype(np.float32)).any()
    c.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("new", [[5, 1], [80, 40]], ids=str)
@pytest.mark.parametrize("off,pad", [(0, 8), (1, 0), (0, 3), (3, 5)], ids=str)
def test_rows_anywhere(ctx, pkg, route, dtype, new, off, pad):
    """Rows apart by odd numbers of elements and off 16 bytes give what rows side by side give; what lies between them stays."""
    c = case(ctx, pkg, [130, 40], 32, 2, 64)
    rows, width = sum(new), 6 * 64 + pad
    q = c.rng.standard_normal((rows, 6, 64)).astype(dtype)
    flat, out = np.zeros(off + rows * width, dtype), np.full(off + rows * width, 7, dtype)
    flat[off:].reshape(rows, width)[:, :384] = q.reshape(rows, 384)
    d = [ctx.upload(x) for x in (flat, out, starts_of(new))]
    size = flat.itemsize
    pkg.ops.kv4_prompt_attention_device(ctx, c.gpu.cache, pkg.AttentionHeads(6, 2, 64, 1, 30, 0.0), 4, pkg.runtime.hipc_dtype(q.dtype), d[2], rows, d[0].at(off * size), width, d[1].at(off * size), width)
    got, want = ctx.download(d[1], dtype, out.shape), c.gpu.prompt_attention(q, new, 30, 4)
    inside = got[off:].reshape(rows, width)
    assert np.array_equal(bits(np.ascontiguousarray(inside[:, :384])), bits(want.reshape(rows, 384))) and np.all(inside[:, 384:] == 7) and np.all(got[:off] == 7)
    for b in d:
        b.free()
    c.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
def test_many_sequences_of_every_kind(ctx, pkg, route, dtype):
    """More sequences than a wavefront has lanes: some bring nothing, most one token, a few whole prompts and pieces."""
    rng = np.random.default_rng(3)
    seqs = 150
    new = np.where(rng.random(seqs) < 0.2, 0, np.where(rng.random(seqs) < 0.85, 1, rng.integers(2, 120, seqs)))
    lengths = [int(n + rng.integers(0, 60)) for n in new]
    c = case(ctx, pkg, lengths, 16, 2, 64, 1)
    for window, sinks in ((0, 0), (30, 3)):
        c.attend(4, [int(n) for n in new], dtype, window, sinks)
    c.gpu.free()


@pytest.mark.parametrize("scale", [0.0, 0.02, -0.1])
@pytest.mark.parametrize("new", [[3], [100]], ids=str)
@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
def test_scales_and_heavy_weights(ctx, pkg, route, dtype, new, scale):
    """Scores of several hundred (one key has all the weight), of either sign, and next to none."""
    c = case(ctx, pkg, [160], 32, 1, 64)
    for gain in (0.001, 40.0):
        q = (gain * c.rng.standard_normal((new[0], 2, 64))).astype(dtype)
        got = c.gpu.prompt_attention(q, new, 0, 0, scale)
        want, weight, size, most = c.ref.prompt_attention(q, starts_of(new), [160], scale=scale or None)
        step = 2.0 ** -11 if dtype == np.float16 else 2.0 ** -22
        size = size + 0.0
        tol = weight * (2 * 66 * 2.0 ** -24 * size + 180 * 2.0 ** -24 + step + (2 * 2.0 ** -22 * size * 64 if dtype == np.float32 else 0)) + np.abs(want) * step + 160 * 2.0 ** -32 * most + 2.0 ** -25
        assert np.all(np.abs(got.astype(np.float64) - want) <= tol)
    c.gpu.free()


def test_the_newest_tokens_call_agrees(ctx, pkg, route):
    """As many tokens of every sequence: hipc_kv4_attention's case, whatever the route."""
    c = case(ctx, pkg, [300, 64, 2, 0], 16, 2, 128)
    for tokens in (1, 2, 33):
        q = c.rng.standard_normal((4 * tokens, 8, 128)).astype(np.float32)
        a, b = c.gpu.attention(q, tokens), c.gpu.prompt_attention(q, [tokens] * 4)
        assert np.all(np.abs(a - b) <= 2.0 ** -18 * np.abs(a).max())
    c.gpu.free()


def test_results_repeat_and_recorded_calls_follow_what_is_written(ctx, pkg, route):
    """Starts, lengths and table are read when the kernels run: a recorded call, replayed with others of as many rows, gives what the call gives, bit for bit."""
    c = case(ctx, pkg, [400, 380, 300], 16, 2, 128)
    q = c.rng.standard_normal((300, 8, 128)).astype(np.float16)
    d = [ctx.upload(x) for x in (q, np.zeros_like(q), starts_of([298, 1, 1]))]
    heads = pkg.AttentionHeads(8, 2, 128, 1, 150, 0.0)

    def enqueue():
        pkg.ops.kv4_prompt_attention_device(ctx, c.gpu.cache, heads, 4, pkg.F16, d[2], 300, d[0], 1024, d[1], 1024)

    def result():
        got = ctx.download(d[1], np.float16, q.shape)
        ctx.fill(d[1], 0, d[1].nbytes, 0x7e007e00)
        return bits(got)
    enqueue()
    first = result()
    ctx.capture_begin()
    enqueue()
    graph = ctx.capture_end()
    for new, lengths in (([298, 1, 1], [400, 380, 300]), ([1, 1, 298], [17, 380, 299]), ([100, 100, 100], [100, 200, 300]), ([0, 0, 300], [9, 9, 300]), ([298, 1, 1], [400, 380, 300])):
        ctx.upload(starts_of(new), d[2])
        c.gpu.set_lengths(lengths)
        ctx.graph_launch(graph)
        got = result()
        enqueue()
        assert np.array_equal(got, result())
    assert np.array_equal(got, first)
    ctx.graph_destroy(graph)
    for b in d:
        b.free()
    c.gpu.free()


def test_two_contexts_at_once(pkg):
    """Calls of two contexts overlap on the device; each gets what it gets alone."""
    with pkg.Context(0) as one, pkg.Context(0) as two:
        sides = []
        for i, ctx in enumerate((one, two)):
            c = case(ctx, pkg, [900, 700, 80], 16, 2, 128, i)
            new = [200, 1, 80]
            q = c.rng.standard_normal((281, 8, 128)).astype(np.float16)
            d = [ctx.upload(x) for x in (q, np.zeros_like(q), starts_of(new))]
            sides.append((ctx, c, d, q, bits(c.gpu.prompt_attention(q, new))))
        heads = pkg.AttentionHeads(8, 2, 128, 1, 0, 0.0)
        for _ in range(20):
            for ctx, c, d, q, _ in sides:
                pkg.ops.kv4_prompt_attention_device(ctx, c.gpu.cache, heads, 0, pkg.F16, d[2], 281, d[0], 1024, d[1], 1024)
        for ctx, c, d, q, alone in sides:
            assert np.array_equal(bits(ctx.download(d[1], np.float16, q.shape)), alone)
            for b in d:
                b.free()
            c.gpu.free()


def test_recorded_on_a_context_that_has_run_none(pkg):
    """The call needs its scratch memory: refused in a recording before any ran, and the recording goes on."""
    with pkg.Context(0) as ctx:
        pages = pkg.ops.Kv4Pages(ctx, 4, 16, 1, 64, [[0, 1, 2, 3]])
        pages.set_lengths([20])
        q = np.ones((20, 2, 64), np.float16)
        d = [ctx.upload(x) for x in (q, np.zeros_like(q), starts_of([20]))]
        ctx.flush()
        ctx.capture_begin()
        with pytest.raises(pkg.HipComputeError):
            pkg.ops.kv4_prompt_attention_device(ctx, pages.cache, pkg.AttentionHeads(2, 1, 64, 1, 0, 0.0), 0, pkg.F16, d[2], 20, d[0], 128, d[1], 128)
        ctx.fill(d[1], 0, 4, 0)
        ctx.graph_destroy(ctx.capture_end())
        assert not pages.prompt_attention(q, [20]).any()      # (an empty cache's values are zeros)
        for b in d:
            b.free()
        pages.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 4)], ids=str)
def test_a_layer_of_prompts_in_pieces_and_tokens(ctx, pkg, route, dtype, window, sinks):
    """The calls as a program makes them: rows of a projection are normed, turned and stored, then attended with, piece by piece and token by token, beside
    other sequences; every step against the definition: queries and keys by the formulas, the cache by the oracle's from these keys, and attention on that."""
    rng = np.random.default_rng(11)
    heads, kv, dim, page = 8, 2, 64, 16
    f = pkg.ops.rotary_frequencies(1e4, dim, pkg.ops.ROTARY_BY_PARTS, 4.0, 64, 1, 8)
    norms = [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
    turning = pkg.ops.Rotary(ctx, heads, kv, dim, f, norms[0], norms[1], 1e-6, amplitude=1.1)
    c = Case(ctx, pkg, rng, 3, 12, page, kv, dim)
    for new in ([70, 0, 33], [50, 90, 1], [1, 1, 1], [0, 1, 1], [1, 20, 1]):
        rows = sum(new)
        q, k, v = (rng.standard_normal((rows, h, dim)).astype(dtype) for h in (heads, kv, kv))
        c.lengths = c.lengths + np.asarray(new)
        c.gpu.set_lengths(c.lengths)
        turned = c.gpu.append_rotary(turning, q, k, v, new)
        got = c.gpu.prompt_attention(turned, new, window, sinks)
        at = np.concatenate([np.arange(int(n) - m, int(n)) for m, n in zip(new, c.lengths)])
        again, key = turning(q, k, at)
        assert np.array_equal(bits(again), bits(turned))
        check(turned, q, at, f, norms[0], amplitude=1.1), check(key, k, at, f, norms[1], amplitude=1.1)
        i = 0
        for s, m in enumerate(new):
            for p in range(int(c.lengths[s]) - m, int(c.lengths[s])):
                c.ref.store(s, p, (key[i], v[i]))
                i += 1
        held = [int(n) for n in c.lengths]
        for x, which in zip(c.gpu.read(held), (0, 1)):
            assert np.array_equal(bits(x), bits(c.rows(which, held)))
        check_rows(got, turned, c.ref, starts_of(new), c.lengths, window, sinks)
    c.gpu.free(), turning.free()
