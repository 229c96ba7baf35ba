"""Attention, the 4-bit cache and token log-probabilities where single calls of ordinary size do not go: offsets past 2^32 bytes, two contexts at
once, calls recorded on a context that has run none, pages that sequences share, and rows left alone by workgroups that share keys."""
import numpy as np
import pytest

from oracle import attention as ref
from test_prompt_attention_gpu import check, operands

pytestmark = pytest.mark.gpu


def bits(x):
    return x.view(np.uint16 if x.dtype == np.float16 else np.uint32)


def test_keys_and_values_far_apart(ctx, pkg):
    """300 keys 16 MB apart: the last ones lie 4.8 GB behind the first."""
    rng = np.random.default_rng(1)
    heads, kv, dim = 4, 1, 64
    for rows, waves in ((5, 1), (300, 4)):
        q, k, v = operands(rng, np.float16, rows, 300, heads, kv, dim)
        stride = 1 << 23
        dK, dV = ctx.alloc(2 * (299 * stride + dim)), ctx.alloc(2 * (299 * stride + dim))
        for i in range(300):
            ctx.upload(k[i], dK, 2 * stride * i), ctx.upload(v[i], dV, 2 * stride * i)
        dQ, dY = ctx.upload(q), ctx.upload(np.zeros_like(q))
        qs, ks = ctx.upload(np.array([0, rows], np.int32)), ctx.upload(np.array([0, 300], np.int32))
        with ctx.options(HIPC_PROMPT_WAVES=waves):
            pkg.ops.prompt_attention_device(ctx, pkg.AttentionHeads(heads, kv, dim, 1, 0, 0.0), pkg.F16, dQ, heads * dim, dK, stride, dV, stride, qs, ks, 1, rows, 300, dY,
                                            heads * dim)
            got, near = ctx.download(dY, np.float16, q.shape), pkg.ops.prompt_attention(ctx, q, k, v, [rows], [300])
        for b in (dK, dV, dQ, dY, qs, ks):
            b.free()
        assert np.array_equal(bits(got), bits(near))
        check(got, q, k, v, [rows], [300])


def test_a_cache_of_ten_gigabytes(ctx, pkg):
    """Pages past 2^32 bytes of codes: stored, read and attended to as in a small cache. (Only the pages in use are ever touched.)"""
    kv, dim, page, pages = 8, 128, 64, 140001
    rows = pages * kv * page
    rng = np.random.default_rng(2)
    table = np.array([[pages - 1, 0, 70001], [139000, pages - 2, 5]], np.int32)
    small = pkg.ops.Kv4Pages(ctx, 6, page, kv, dim, [[5, 0, 2], [3, 4, 1]])
    buffers = [ctx.alloc(rows * dim // 2), ctx.alloc(rows * dim // 32 * 4), ctx.alloc(rows * dim // 2), ctx.alloc(rows * dim // 32 * 4)]
    dT, lengths = ctx.upload(table), [150, 129]
    small.set_lengths(lengths)
    cache = pkg.Kv4Cache(*(b.ptr for b in buffers), pages, page, kv, dim, 2, small.lengths.ptr, dT.ptr, 3)
    k, v = (rng.standard_normal((279, kv, dim)).astype(np.float32) for _ in range(2))
    small.append(k, v, lengths)
    dK, dV, dS = ctx.upload(k), ctx.upload(v), ctx.upload(np.array([0, 150, 279], np.int32))
    pkg.ops.kv4_append_device(ctx, cache, pkg.F32, dS, 279, dK, kv * dim, dV, kv * dim)
    pkg.ops.kv4_read_device(ctx, cache, pkg.F32, dS, 279, dK, kv * dim, dV, kv * dim)
    for d, want in zip((dK, dV), small.read(lengths, np.float32)):
        assert np.array_equal(bits(ctx.download(d, np.float32, k.shape)), bits(want)) and want.any()
    q = rng.standard_normal((2, 32, dim)).astype(np.float16)
    dQ, dY = ctx.upload(q), ctx.upload(np.zeros_like(q))
    pkg.ops.kv4_attention_device(ctx, cache, pkg.AttentionHeads(32, kv, dim, 1, 0, 0.0), pkg.F16, 1, dQ, 32 * dim, dY, 32 * dim)
    assert np.array_equal(bits(ctx.download(dY, np.float16, q.shape)), bits(small.attention(q)))
    for b in buffers + [dT, dK, dV, dS, dQ, dY]:
        b.free()
    small.free()


def test_rows_of_logits_far_apart(ctx, pkg):
    rng = np.random.default_rng(3)
    x, tokens, stride = rng.standard_normal((2, 5003)).astype(np.float16), np.array([7, 4000], np.int32), (1 << 31) + 5
    dX, dT, dL = ctx.alloc(2 * (stride + 5003)), ctx.upload(tokens), ctx.upload(np.zeros(2, np.float32))
    dI, dP = ctx.upload(np.zeros((2, 3), np.int32)), ctx.upload(np.zeros((2, 3), np.float32))
    for r in range(2):
        ctx.upload(x[r], dX, 2 * stride * r)
    pkg.ops.token_logprobs_device(ctx, pkg.F16, dX, stride, 2, 5003, dT, dL, None, 3, dI, dP)
    got = ctx.download(dL, np.float32, (2,)), ctx.download(dI, np.int32, (2, 3))
    for b in (dX, dT, dL, dI, dP):
        b.free()
    want = ref.token_logprobs(x, tokens, 3)
    assert np.array_equal(got[1], want[2]) and np.allclose(got[0], want[0], rtol=1e-5, atol=0)


def _calls(ctx, pkg, seed):
    """A call of each operator whose work several workgroups share, on buffers of its own: (enqueue, results, free)."""
    rng = np.random.default_rng(seed)
    q, k, v = operands(rng, np.float16, 40, 4000, 4, 1, 128)
    up = [ctx.upload(x) for x in (q, k, v, np.zeros_like(q), np.array([0, 40], np.int32), np.array([0, 4000], np.int32))]
    pages = pkg.ops.Kv4Pages(ctx, 40, 64, 2, 128, np.arange(40).reshape(1, 40))
    pages.set_lengths([2500])
    kk, vv = (rng.standard_normal((2500, 2, 128)).astype(np.float16) for _ in range(2))
    pages.append(kk, vv, [2500])
    cq = rng.standard_normal((1, 8, 128)).astype(np.float16)
    cu = [ctx.upload(cq), ctx.upload(np.zeros_like(cq))]
    x = rng.standard_normal((1, 200000)).astype(np.float32)
    lu = [ctx.upload(x), ctx.upload(np.array([3], np.int32)), ctx.upload(np.zeros(1, np.float32)), ctx.upload(np.zeros(1, np.float32)), ctx.upload(np.zeros(5, np.int32)),
          ctx.upload(np.zeros(5, np.float32))]
    heads = pkg.AttentionHeads(4, 1, 128, 1, 0, 0.0), pkg.AttentionHeads(8, 2, 128, 1, 0, 0.0)
    enqueue = [lambda: pkg.ops.prompt_attention_device(ctx, heads[0], pkg.F16, up[0], 512, up[1], 128, up[2], 128, up[4], up[5], 1, 40, 4000, up[3], 512),
               lambda: pkg.ops.kv4_attention_device(ctx, pages.cache, heads[1], pkg.F16, 1, cu[0], 1024, cu[1], 1024),
               lambda: pkg.ops.token_logprobs_device(ctx, pkg.F32, lu[0], 200000, 1, 200000, lu[1], lu[2], lu[3], 5, lu[4], lu[5])]

    def results():
        return [bits(ctx.download(up[3], np.float16, q.shape)), bits(ctx.download(cu[1], np.float16, cq.shape)),
                np.concatenate([ctx.download(b, np.uint32, (n,)) for b, n in zip(lu[2:], (1, 1, 5, 5))])]

    def clear():
        for b in (up[3], cu[1], *lu[2:]):
            ctx.fill(b, 0, b.nbytes, 0xffffffff)

    def free():
        for b in up + cu + lu:
            b.free()
        pages.free()
    return enqueue, results, clear, free


def test_two_contexts_at_once(pkg):
    """Their calls overlap on the device; each has scratch memory of its own, and gets what it gets alone."""
    with pkg.Context(0) as one, pkg.Context(0) as two:
        sides = [_calls(c, pkg, 10 + i) for i, c in enumerate((one, two))]
        alone = []
        for enqueue, results, clear, _ in sides:
            for call in enqueue:
                call()
            alone.append(results())
            clear()
        one.flush(), two.flush()
        for _ in range(20):
            for call in range(3):
                for enqueue, *_ in sides:
                    enqueue[call]()
        for (_, results, _, free), want in zip(sides, alone):
            for a, b in zip(results(), want):
                assert np.array_equal(a, b)
            free()


def test_recorded_before_any_ran(pkg):
    """No scratch memory is there and none may be made: the cache's attention is refused (and works afterwards), the others take a way without,
    and what they record stays right beside the program's own calls."""
    with pkg.Context(0) as ctx:
        enqueue, results, clear, free = _calls(ctx, pkg, 20)
        ctx.capture_begin()
        enqueue[0]()
        with pytest.raises(pkg.HipComputeError) as e:
            enqueue[1]()
        assert e.value.code == 2
        enqueue[2]()
        g = ctx.capture_end()
        for call in enqueue:
            call()
        want = results()
        for _ in range(3):
            clear()
            ctx.graph_launch(g)
            got = results()
            for call in enqueue:
                call()
            assert all(np.array_equal(a, b) for a, b in zip(results(), want))
            # another order of the sums: near, and the same ids
            a, b = got[0].view(np.float16).astype(np.float64), want[0].view(np.float16).astype(np.float64)
            assert np.all(np.abs(a - b) <= 2.0 ** -9 * (np.abs(b) + np.abs(b).max()))
            assert np.array_equal(got[2][2:7], want[2][2:7]) and np.allclose(got[2][:2].view(np.float32), want[2][:2].view(np.float32), rtol=1e-5)
        ctx.graph_destroy(g)
        free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("off,pad,dim", [(1, 3, 64), (0, 0, 36), (0, 1, 250), (2, 2, 9)])
def test_rows_of_any_kind_with_and_without_scratch_memory(pkg, dtype, off, pad, dim):
    """Head widths off 8, rows apart by odd numbers of elements and off 16 bytes: recorded on a context that has no scratch memory, eagerly, and
    recorded again; rows of Y in front of and behind the sequences stay, whatever rows of Q and K there hold."""
    heads, kv, rows, keys = 6, 2, 70, 150
    rng = np.random.default_rng(dim)
    q, k, v = operands(rng, dtype, rows, keys, heads, kv, dim)
    q[:2], q[66:], k[:3], v[:3], k[140:], v[140:] = np.nan, np.nan, np.nan, np.inf, np.inf, np.nan
    code, size = pkg.runtime.hipc_dtype(np.dtype(dtype)), np.dtype(dtype).itemsize

    def strided(x):
        w = x.shape[1] * x.shape[2]
        buf = np.full(off + x.shape[0] * (w + pad), 7, dtype)
        buf[off:].reshape(x.shape[0], w + pad)[:, :w] = x.reshape(x.shape[0], w)
        return buf
    with pkg.Context(0) as ctx:
        up = [ctx.upload(strided(x)) for x in (q, k, v, np.full_like(q, 7))]
        qs, ks = ctx.upload(np.array([2, 30, 30, 66], np.int32)), ctx.upload(np.array([3, 31, 50, 140], np.int32))
        h, wq, wk = pkg.AttentionHeads(heads, kv, dim, 1, 0, 0.0), heads * dim + pad, kv * dim + pad
        at = [b.at(off * size) for b in up]

        def call():
            pkg.ops.prompt_attention_device(ctx, h, code, at[0], wq, at[1], wk, at[2], wk, qs, ks, 3, rows, keys, at[3], wq)

        def result():
            buf = ctx.download(up[3], dtype, (off + rows * wq,))
            assert np.all(buf[:off] == 7)
            y = buf[off:].reshape(rows, wq)
            assert np.all(y[:, heads * dim:] == 7) and np.all(y[:2] == 7) and np.all(y[66:] == 7)
            y = y[2:66, :heads * dim].reshape(64, heads, dim)
            check(y, q[2:66], k[3:140], v[3:140], [28, 0, 36], [28, 19, 90])
            ctx.upload(strided(np.full_like(q, 7)), up[3])
            return bits(np.ascontiguousarray(y))

        def recorded():
            ctx.capture_begin()
            call()
            g = ctx.capture_end()
            for _ in range(2):
                ctx.graph_launch(g)
                y = result()
                call()
                assert np.array_equal(result(), eager) if eager is not None else True
            ctx.graph_destroy(g)
            return y
        eager = None
        recorded()
        call()
        eager = result()
        assert np.array_equal(recorded(), eager)
        for b in up + [qs, ks]:
            b.free()


@pytest.mark.parametrize("waves,dtype,dim", [(-1, np.float16, 64), (4, np.float16, 128), (2, np.float32, 64), (-1, np.float16, 20)])
def test_seven_hundred_prompts(ctx, pkg, waves, dtype, dim):
    """More sequences than are looked up at once, many of them empty, one of some length; parts of them behind earlier keys."""
    rng = np.random.default_rng(5)
    q_lengths = np.where(rng.random(700) < 0.4, 0, rng.integers(1, 4, 700))
    q_lengths[[0, 333, 699]] = 0, 90, 5
    k_lengths = np.where(rng.random(700) < 0.5, q_lengths, q_lengths + rng.integers(0, 9, 700))
    q, k, v = operands(rng, dtype, int(q_lengths.sum()), int(k_lengths.sum()), 4, 2, dim)
    with ctx.options(HIPC_PROMPT_WAVES=waves):
        got = pkg.ops.prompt_attention(ctx, q, k, v, q_lengths, k_lengths)
    check(got, q, k, v, q_lengths, k_lengths)


def test_pages_that_sequences_share(ctx, pkg):
    """Two sequences with one beginning: the same pages in both rows of the table."""
    rng = np.random.default_rng(4)
    kv, dim = 2, 64
    apart = pkg.ops.Kv4Pages(ctx, 8, 16, kv, dim, [[0, 1, 2, 3], [4, 5, 6, 7]])
    shared = pkg.ops.Kv4Pages(ctx, 8, 16, kv, dim, [[0, 1, 2, 3], [0, 1, 6, 7]])
    k, v = (rng.standard_normal((32, kv, dim)).astype(np.float16) for _ in range(2))
    tail = [rng.standard_normal((25, kv, dim)).astype(np.float16) for _ in range(2)]
    for pages in (apart, shared):
        pages.set_lengths([32, 32])
        if pages is apart:
            pages.append(np.concatenate([k, k]), np.concatenate([v, v]), [32, 32])
        else:
            pages.append(k, v, [32, 0])
        pages.set_lengths([50, 39])
        pages.append(*tail, [18, 7])
    q = rng.standard_normal((2, 8, dim)).astype(np.float16)
    assert np.array_equal(bits(apart.attention(q)), bits(shared.attention(q)))
    for a, b in zip(apart.read([50, 39]), shared.read([50, 39])):
        assert np.array_equal(bits(a), bits(b))
    apart.free(), shared.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("split", [2, 5, 70])
@pytest.mark.parametrize("heads,dim", [(2, 8), (1, 64), (6, 136)])
def test_rows_outside_the_sequences_when_keys_are_shared(ctx, pkg, dtype, split, heads, dim):
    """The join leaves rows of no sequence as they were, among them rows between two sequences and ones that share a wavefront with others."""
    rng = np.random.default_rng(split + dim)
    q, k, v = operands(rng, dtype, 60, 500, heads, 1, dim)
    dQ, dK, dV, dY = ctx.upload(q), ctx.upload(k), ctx.upload(v), ctx.upload(np.full_like(q, 7))
    qs, ks = ctx.upload(np.array([3, 20, 20, 51], np.int32)), ctx.upload(np.array([0, 300, 300, 480], np.int32))
    with ctx.options(HIPC_PROMPT_SPLIT=split):
        pkg.ops.prompt_attention_device(ctx, pkg.AttentionHeads(heads, 1, dim, 1, 0, 0.0), pkg.runtime.hipc_dtype(np.dtype(dtype)), dQ, heads * dim, dK, dim, dV, dim, qs, ks, 3, 60,
                                        500, dY, heads * dim)
    y = ctx.download(dY, dtype, q.shape)
    assert np.all(y[:3] == 7) and np.all(y[51:] == 7)
    check(y[3:51], q[3:51], k[:480], v[:480], [17, 0, 31], [300, 0, 180])
    for b in (dQ, dK, dV, dY, qs, ks):
        b.free()


def test_copies_that_the_device_has_no_room_for(pkg):
    """Operands that pass through scratch memory, declared so large (the rows behind the sequences are never touched) that it is not to be had: the call takes the way
    without, and the ones behind it know nothing of that."""
    rng = np.random.default_rng(6)
    heads, dim, keys, total = 16, 250, 40, (1 << 26) - 4
    q, k, v = operands(rng, np.float32, keys, keys, heads, heads, dim)
    with pkg.Context(0) as ctx:
        dQ, dK, dV, dY, dS = (ctx.upload(x) for x in (q, k, v, np.zeros_like(q), np.array([0, 7, keys], np.int32)))
        h, w = pkg.AttentionHeads(heads, heads, dim, 1, 0, 0.0), heads * dim
        for most in (total, keys, total):
            ctx.fill(dY, 0, dY.nbytes, 0)
            pkg.ops.prompt_attention_device(ctx, h, pkg.F32, dQ, w, dK, w, dV, w, dS, dS, 2, keys, most, dY, w)
            check(ctx.download(dY, np.float32, q.shape), q, k, v, [7, keys - 7], [7, keys - 7])
        for b in (dQ, dK, dV, dY, dS):
            b.free()
