"""The 4-bit cache on the GPU: what is stored and read back is the definition's, bit for bit; attention over it against the
definition in 64 bits.

Tolerance of the attention: as for prompts (see test_prompt_attention_gpu.py), the cache's values being exact; an f32 query enters with 22
bits of its row's largest value (2^-22 max|q| sum |k| scale, bounded by 2^-22 S dim), weights with 22 bits.
"""
import numpy as np
import pytest

from oracle import attention as ref

pytestmark = pytest.mark.gpu


def tolerance(dtype, q, keys, y, weight, size, k_most):
    dim = q.shape[2]
    score = (dim + 2) * 2.0 ** -24 * size
    if dtype == np.float32:
        score = score + 2.0 ** -22 * np.abs(q).max(-1, keepdims=True) * dim * k_most / np.sqrt(dim)
    relative = 2 * score + (16 + keys) * 2.0 ** -24 + 2.0 ** -21
    if dtype == np.float16:
        return weight * relative + np.abs(y) * 2.0 ** -11 + 2.0 ** -25
    return weight * relative + 1e-37


def bits(x):
    return x.view(np.uint16 if x.dtype == np.float16 else np.uint32)


class Pair:
    """A cache on the device and the oracle's, filled with the same rows."""

    def __init__(self, ctx, pkg, rng, seqs, width, page, kv, dim, table=None):
        n = seqs * width + 2
        table = rng.permutation(n)[:seqs * width].reshape(seqs, width).astype(np.int32) if table is None else table
        self.kv, self.dim, self.rng, self.seqs = kv, dim, rng, seqs
        self.gpu, self.ref = pkg.ops.Kv4Pages(ctx, n, page, kv, dim, table), ref.Cache(n, page, kv, dim, table)
        self.lengths = np.zeros(seqs, np.int64)

    def append(self, new, dtype=np.float16, change=None):
        k, v = (self.rng.standard_normal((int(np.sum(new)), self.kv, self.dim)).astype(dtype) for _ in range(2))
        if change is not None:
            change(k, v)
        self.lengths = self.lengths + np.asarray(new)
        self.gpu.set_lengths(self.lengths)
        self.gpu.append(k, v, new)
        at = 0
        for s, n in enumerate(new):
            for i in range(n):
                self.ref.store(s, int(self.lengths[s]) - n + i, (k[at + i], v[at + i]))
            at += n
        return k, v

    def rows(self, which, count):
        return np.concatenate([np.stack([self.ref.load(which, s, int(self.lengths[s]) - n + i) for i in range(n)])
                               for s, n in enumerate(count) if n], 0)

    def check(self, ctx, pkg, heads, tokens, dtype, window=0, gain=1.0):
        q = (gain * self.rng.standard_normal((self.seqs * tokens, heads, self.dim))).astype(dtype)
        got = self.gpu.attention(q, tokens, window)
        want, weight, size = self.ref.attention(q, self.lengths, tokens, window)
        k_most = max(float(np.nanmax(np.abs(ref.values(np.full((1, 1, 32), 15, np.uint8), p[..., :1], p[..., 1:]).astype(np.float64)))) +
                     float(np.nanmax(np.abs(p[..., 1].astype(np.float64)))) for p in (self.ref.params[0].reshape(1, -1, 2),))
        off = np.abs(got.astype(np.float64) - want) - tolerance(dtype, q.astype(np.float64), int(self.lengths.max()), want, weight, size, k_most)
        assert np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))
        return got


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("kv,dim", [(1, 256), (8, 128), (3, 96), (2, 32), (5, 160), (3, 64)])
def test_what_is_stored_reads_back_as_defined(ctx, pkg, dtype, kv, dim):
    p = Pair(ctx, pkg, np.random.default_rng(dim + kv), 3, 5, 16, kv, dim)

    def change(k, v):
        k[0, 0, :32] = 0.25                              # a group of one value
        k[1, 0, :32] = np.arange(32) / 31 * 15           # some fall on the border between two codes
        v[0, 0, :16], v[0, 0, 16:32] = -1, 14            # scale 1 exactly: values .5 between codes below
        v[1, 0, :32] = np.repeat(np.arange(16) - 0.5, 2)
        v[1, 0, 0], v[1, 0, 1] = 0, 15
        k[2] *= dtype(1000)
        v[2] *= dtype(1e-6)
        if dtype == np.float32:
            k[3, 0, 0], k[3, 0, 1] = 3e38, -np.inf       # held to the largest values that read back

    new = [40, 1, 17]
    p.append(new, dtype, change)
    for count in (new, [3, 0, 17], [0, 1, 0]):
        for out in (np.float16, np.float32):
            k, v = p.gpu.read(count, out)
            for got, which in ((k, 0), (v, 1)):
                want = p.rows(which, count).astype(out)
                assert np.array_equal(bits(got), bits(want)), np.argwhere(got != want)[:4]
    for b, want in zip(p.gpu.buffers, (p.ref.codes[0], p.ref.params[0], p.ref.codes[1], p.ref.params[1])):
        got = ctx.download(b, want.dtype, want.shape)
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    p.gpu.free()


def test_steps_one_token_at_a_time_fill_the_same_cache(ctx, pkg):
    rng = np.random.default_rng(5)
    a, b = (Pair(ctx, pkg, np.random.default_rng(6), 2, 4, 16, 2, 64) for _ in range(2))
    k, v = a.append([33, 20])
    seen = [0, 0]
    while sum(seen) < 53:
        new = [int(rng.random() < 0.7 and seen[0] < 33), int(rng.random() < 0.7 and seen[1] < 20)]
        rows = [r for s, n, base in ((0, new[0], 0), (1, new[1], 33)) for r in range(base + seen[s], base + seen[s] + n)]
        seen = [seen[0] + new[0], seen[1] + new[1]]
        if rows:
            b.gpu.set_lengths(seen)
            b.gpu.append(k[rows], v[rows], new)
    for x, y in zip(a.gpu.read([33, 20]), b.gpu.read([33, 20])):
        assert np.array_equal(bits(x), bits(y))
    a.gpu.free(), b.gpu.free()


def test_nan_rows_read_back_as_nan_and_nothing_else_does(ctx, pkg):
    p = Pair(ctx, pkg, np.random.default_rng(7), 1, 2, 16, 2, 64)

    def change(k, v):
        k[3, 1, 40] = np.nan

    p.append([20], np.float32, change)
    k, v = p.gpu.read([20])
    nan = np.isnan(k.astype(np.float32))
    assert nan[3, 1, 32:].all() and nan.sum() == 32 and not np.isnan(v.astype(np.float32)).any()
    p.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [64, 63, 65, 0], [1, 300, 2], [700]], ids=str)
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 1, 256, 512), (8, 2, 128, 16), (3, 3, 64, 32), (14, 2, 96, 16)])
def test_attention_of_single_tokens(ctx, pkg, dtype, lengths, heads, kv, dim, page):
    width = -(-max(lengths) // page) + 1
    p = Pair(ctx, pkg, np.random.default_rng(sum(lengths) + dim), len(lengths), width, page, kv, dim)
    p.append(lengths)
    y = p.check(ctx, pkg, heads, 1, dtype, gain=1.5)
    for s, n in enumerate(lengths):
        assert n or not y[s].any()
    p.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,tokens,window", [(4, 1, 64, 3, 0), (2, 2, 32, 5, 0), (16, 1, 64, 2, 0), (6, 2, 128, 4, 20), (4, 4, 160, 1, 1), (5, 1, 256, 7, 64), (1, 1, 224, 2, 100)])
def test_several_tokens_windows_and_short_sequences(ctx, pkg, dtype, heads, kv, dim, tokens, window):
    lengths = [130, 2, 65, 1]           # some shorter than the tokens asked for
    p = Pair(ctx, pkg, np.random.default_rng(dim + tokens), 4, 5, 32, kv, dim)
    p.append(lengths)
    y = p.check(ctx, pkg, heads, tokens, dtype, window)
    if tokens > 2:
        assert not y[tokens:tokens + tokens - 2].any()
    p.gpu.free()


@pytest.mark.parametrize("tokens,group", [(1, 17), (1, 32), (33, 1), (20, 7), (1, 1)])
def test_many_query_rows_of_a_kv_head(ctx, pkg, tokens, group):
    p = Pair(ctx, pkg, np.random.default_rng(tokens), 2, 3, 32, 1, 64)
    p.append([90, 40])
    p.check(ctx, pkg, group, tokens, np.float16)
    p.gpu.free()


def test_pages_that_are_no_pages(ctx, pkg):
    """Numbers outside the cache: not stored, zero when read, not seen; the same with a window that has left them behind."""
    table = np.array([[3, -1, 0, 1 << 30], [-7, -1, 99, -1]], np.int32)
    p = Pair(ctx, pkg, np.random.default_rng(2), 2, 4, 16, 2, 64, table=table)
    p.append([60, 20])
    k, _ = p.gpu.read([60, 20])
    assert k[:16].any() and not k[16:32].any() and k[32:48].any() and not k[48:].any()
    for window in (0, 20):
        y = p.check(ctx, pkg, 4, 1, np.float16, window)
        assert not y[1].any()
    p.gpu.free()


def test_lengths_past_the_table_and_below_zero(ctx, pkg):
    """Positions behind the table lie on no page: rows that would go there are not stored (and nothing else is written over), read as
    zeros, and are not seen, though they count where a window does."""
    p = Pair(ctx, pkg, np.random.default_rng(4), 2, 2, 16, 1, 64)
    p.append([32, 32])
    q = p.rng.standard_normal((2, 2, 64)).astype(np.float16)
    want, held = p.gpu.attention(q), p.gpu.read([32, 32])
    p.gpu.set_lengths([1 << 30, -5])
    got = p.gpu.attention(q)
    assert np.array_equal(bits(got[0]), bits(want[0])) and not got[1].any()
    k, _ = p.gpu.read([2, 2])
    assert not k.any()
    p.gpu.set_lengths([35, 0])
    rows = p.rng.standard_normal((6, 1, 64)).astype(np.float16)
    p.gpu.append(rows[:5], rows[:5], [5, 0])              # positions 30 .. 34: two of them lie in the table
    k, _ = p.gpu.read([35, 0])
    assert np.array_equal(bits(k[:30]), bits(held[0][:30])) and k[30].any() and not np.array_equal(k[30], held[0][30]) and not k[32:].any()
    for s, n in ((0, 35), (1, 0)):
        p.lengths[s] = n
    for i in range(2):
        p.ref.store(0, 30 + i, (rows[i], rows[i]))
    for window in (0, 10, 3):
        y = p.check(ctx, pkg, 4, 1, np.float16, window)
        assert y[0].any() == (window != 3)
    p.gpu.set_lengths([-5, 2147483647])
    assert not p.gpu.attention(q)[0].any()
    p.gpu.free()


def test_a_nan_that_only_the_newest_token_sees(ctx, pkg):
    """Parameters that are not finite at the last position: that token's rows are NaN in their channels, the token before it is as without."""
    p = Pair(ctx, pkg, np.random.default_rng(14), 2, 5, 16, 1, 96)
    p.append([70, 3])
    q = p.rng.standard_normal((4, 3, 96)).astype(np.float16)
    want = p.gpu.attention(q, tokens=2)
    page, place = p.ref.place(0, 69)
    params = ctx.download(p.gpu.buffers[3], np.float16, p.ref.params[1].shape)
    params[page, 0, place, 1] = np.nan                     # channels 32 .. 63 of the value
    ctx.upload(params, p.gpu.buffers[3])
    got = p.gpu.attention(q, tokens=2).astype(np.float32)
    assert np.array_equal(got[[0, 2, 3]], want[[0, 2, 3]].astype(np.float32))
    assert np.isnan(got[1, :, 32:64]).all() and np.array_equal(got[1, :, :32], want[1, :, :32].astype(np.float32)) and np.array_equal(got[1, :, 64:], want[1, :, 64:].astype(np.float32))
    p.gpu.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("off,pad", [(0, 0), (1, 0), (0, 3), (3, 5)])
def test_rows_anywhere(ctx, pkg, dtype, off, pad):
    """Rows apart by odd numbers of elements and off 16 bytes: stored, read and attended to as if they were side by side."""
    kv, dim, heads, n = 2, 64, 6, 37
    p, r = (Pair(ctx, pkg, np.random.default_rng(15), 1, 3, 16, kv, dim) for _ in range(2))
    k, v = r.append([n], dtype)
    width, size, code = kv * dim + pad, np.dtype(dtype).itemsize, pkg.runtime.hipc_dtype(dtype)
    def strided(x, w):
        buf = np.full(off + x.shape[0] * w + 8, 7, dtype)
        for i in range(x.shape[0]):
            buf[off + i * w:off + i * w + x[i].size] = x[i].reshape(-1)
        return buf
    dK, dV, dS = ctx.upload(strided(k, width)), ctx.upload(strided(v, width)), ctx.upload(np.array([0, n], np.int32))
    p.gpu.set_lengths([n])
    pkg.ops.kv4_append_device(ctx, p.gpu.cache, code, dS, n, dK.at(off * size), width, dV.at(off * size), width)
    dB = ctx.upload(strided(np.zeros_like(k), width)), ctx.upload(strided(np.zeros_like(k), width))
    pkg.ops.kv4_read_device(ctx, p.gpu.cache, code, dS, n, dB[0].at(off * size), width, dB[1].at(off * size), width)
    for d, want in zip(dB, r.gpu.read([n], dtype)):
        assert np.array_equal(bits(ctx.download(d, dtype, (off + n * width + 8,))), bits(strided(want, width)))
    q = np.random.default_rng(16).standard_normal((1, heads, dim)).astype(dtype)
    w = heads * dim + pad
    dQ, dY = ctx.upload(strided(q, w)), ctx.upload(strided(np.zeros_like(q), w))
    pkg.ops.kv4_attention_device(ctx, p.gpu.cache, pkg.AttentionHeads(heads, kv, dim, 1, 0, 0.0), code, 1, dQ.at(off * size), w, dY.at(off * size), w)
    assert np.array_equal(bits(ctx.download(dY, dtype, (off + w + 8,))), bits(strided(r.gpu.attention(q), w)))
    for b in (dK, dV, dS, dQ, dY) + dB:
        b.free()
    p.gpu.free(), r.gpu.free()


def test_many_sequences(ctx, pkg):
    """More sequences than a wavefront has lanes, most of them empty, and more units than workgroups."""
    rng = np.random.default_rng(17)
    seqs = 150
    lengths = np.where(rng.random(seqs) < 0.5, 0, rng.integers(1, 40, seqs))
    p = Pair(ctx, pkg, rng, seqs, 3, 16, 2, 32)
    p.append([int(n) for n in lengths])
    y = p.check(ctx, pkg, 4, 1, np.float16)
    assert not y[lengths == 0].any()
    p.check(ctx, pkg, 34, 2, np.float32)                   # 34 query rows a kv head: three blocks, 450 units and more
    k, v = p.gpu.read([int(n) for n in lengths])
    assert np.array_equal(bits(k), bits(p.rows(0, lengths))) and np.array_equal(bits(v), bits(p.rows(1, lengths)))
    p.gpu.free()


@pytest.mark.parametrize("dtype,kv,dim,heads,tokens,window", [(np.float16, 4, 128, 16, 1, 0), (np.float32, 4, 64, 8, 2, 0), (np.float16, 4, 96, 4, 3, 50),
                                                               (np.float32, 4, 256, 4, 1, 100), (np.float16, 6, 32, 36, 4, 0)])
def test_more_units_than_workgroups(ctx, pkg, dtype, kv, dim, heads, tokens, window):
    """A wavefront to a unit, runs of tiles dealt over sequences of very different lengths, some of which several wavefronts have parts of: against the
    definition, and twice the same."""
    rng = np.random.default_rng(dim + tokens)
    seqs = 100
    lengths = np.where(rng.random(seqs) < 0.2, 0, rng.integers(1, 40, seqs))
    lengths[[7, 50, 99]] = 900, 257, 600
    p = Pair(ctx, pkg, rng, seqs, 57, 16, kv, dim)
    p.append([int(n) for n in lengths])
    assert seqs * kv * -(-tokens * heads // kv // 16) >= 384      # (256 CUs)
    q = rng.standard_normal((seqs * tokens, heads, dim)).astype(dtype)
    want, weight, size = p.ref.attention(q, p.lengths, tokens, window)
    got = p.gpu.attention(q, tokens, window)
    k_most = float(np.nanmax(np.abs(p.ref.params[0].astype(np.float64)))) * 16
    off = np.abs(got.astype(np.float64) - want) - tolerance(dtype, q.astype(np.float64), 900, want, weight, size, k_most)
    assert np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))
    assert not got.reshape(seqs, tokens, -1)[lengths == 0].any()
    assert np.array_equal(bits(p.gpu.attention(q, tokens, window)), bits(got))
    # pages that are given back, and one that never was
    table = p.ref.table.copy()
    table[50, 3], table[99, :10], table[7, 30] = -1, 1 << 30, -5
    p.gpu.set_table(table)
    p.ref.table = table
    want, weight, size = p.ref.attention(q, p.lengths, tokens, window)
    off = np.abs(p.gpu.attention(q, tokens, window).astype(np.float64) - want) - tolerance(dtype, q.astype(np.float64), 900, want, weight, size, k_most)
    assert np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))
    p.gpu.free()


def test_what_lies_behind_a_sequence_does_not_reach_it(ctx, pkg):
    """Positions behind the length, and pages of nobody, hold NaN parameters; so does a position outside the window."""
    p = Pair(ctx, pkg, np.random.default_rng(9), 2, 6, 16, 2, 64)
    p.append([70, 21])
    q = p.rng.standard_normal((2, 4, 64)).astype(np.float16)
    want = {w: p.gpu.attention(q, window=w) for w in (0, 30)}
    for which in (0, 1):
        shape = p.ref.params[which].shape
        params = ctx.download(p.gpu.buffers[1 + 2 * which], np.float16, shape)
        held = np.zeros(shape[:1] + shape[2:3], bool)
        for s, n in enumerate((70, 21)):
            for t in range(n):
                held[p.ref.place(s, t)] = True
        params[~held.repeat(shape[1], 0).reshape(shape[0], shape[1], shape[2])] = np.nan
        ctx.upload(params, p.gpu.buffers[1 + 2 * which])
    for w in (0, 30):
        assert np.array_equal(bits(p.gpu.attention(q, window=w)), bits(want[w]))
    page, place = p.ref.place(0, 10)                        # outside a window of 30 at position 69
    for which in (0, 1):
        params = ctx.download(p.gpu.buffers[1 + 2 * which], np.float16, p.ref.params[which].shape)
        params[page, :, place] = np.inf
        ctx.upload(params, p.gpu.buffers[1 + 2 * which])
    assert np.array_equal(bits(p.gpu.attention(q, window=30)), bits(want[30]))
    assert np.isnan(p.gpu.attention(q)[0].astype(np.float32)).all()
    p.gpu.free()


def test_results_repeat_and_follow_the_lengths_when_recorded(ctx, pkg):
    """A recorded step replayed as the lengths grow, with the program's own calls between the replays: bit for bit the eager results."""
    p = Pair(ctx, pkg, np.random.default_rng(10), 3, 20, 16, 2, 128)
    p.append([300, 5, 77])
    q = p.rng.standard_normal((3, 8, 128)).astype(np.float32)
    heads = pkg.AttentionHeads(8, 2, 128, 1, 0, 0.0)
    dQ, dY = ctx.upload(q), ctx.upload(np.zeros_like(q))
    call = lambda: pkg.ops.kv4_attention_device(ctx, p.gpu.cache, heads, pkg.F32, 1, dQ, 1024, dY, 1024)  # noqa: E731
    call()
    ctx.capture_begin()
    call()
    g = ctx.capture_end()
    for lengths in ([300, 5, 77], [12, 5, 1], [0, 0, 0], [299, 4, 64], [300, 5, 77]):
        p.gpu.set_lengths(lengths)
        for _ in range(2):
            ctx.fill(dY, 0, dY.nbytes, 0xffffffff)
            ctx.graph_launch(g)
            got = ctx.download(dY, np.float32, q.shape)
            assert np.array_equal(bits(got), bits(p.gpu.attention(q)))
    ctx.graph_destroy(g)
    dQ.free(), dY.free(), p.gpu.free()


def test_prompt_then_steps_then_probabilities(ctx, pkg):
    """As a program uses them: a prompt in two pieces into the cache (the second piece attends to the first as the cache holds it),
    then single tokens, then the probabilities of what came out."""
    rng = np.random.default_rng(20)
    heads, kv, dim, piece = 4, 2, 64, [30, 9]
    p = Pair(ctx, pkg, rng, 2, 6, 16, kv, dim)
    q = rng.standard_normal((39, heads, dim)).astype(np.float16)
    k, v = p.append(piece)
    first = pkg.ops.prompt_attention(ctx, q, k, v, piece)
    assert np.isfinite(first.astype(np.float32)).all()
    p.append(piece)
    both = [60, 18]
    kk, vv = p.gpu.read(both)
    second = pkg.ops.prompt_attention(ctx, q, kk, vv, piece, both)
    want, weight, size = ref.prompt(q, p.rows(0, both), p.rows(1, both), piece, both)
    tol = weight * (2 * 66 * 2.0 ** -24 * size + 76 * 2.0 ** -24 + 2.0 ** -11) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    assert np.all(np.abs(second.astype(np.float64) - want) <= tol)
    # the last row of each piece, once more as a single token over the cache
    last = p.gpu.attention(q[[29, 38]])
    assert np.all(np.abs(last.astype(np.float64) - want[[29, 38]]) <= tol[[29, 38]])
    for _ in range(3):
        p.append([1, 1])
        y = p.check(ctx, pkg, heads, 1, np.float32)
        logits = (y.reshape(2, -1) @ rng.standard_normal((heads * dim, 1000))).astype(np.float32)
        logprob, entropy, ids, best = pkg.ops.token_logprobs(ctx, logits, logits.argmax(1), 3)
        assert np.array_equal(ids[:, 0], logits.argmax(1)) and np.array_equal(logprob, best[:, 0]) and np.all(entropy > 0)
    p.gpu.free()


def test_refusals(ctx, pkg):
    p = Pair(ctx, pkg, np.random.default_rng(1), 1, 1, 16, 2, 64)
    d = ctx.alloc(65536)
    good = {n: getattr(p.gpu.cache, n) for n, _ in pkg.Kv4Cache._fields_}

    def rows(fn="hipc_kv4_append", dtype=None, starts=d.ptr, total=2, k=d.ptr, ks=128, vs=128, cache=True, **change):
        c = pkg.Kv4Cache(**{**good, **change}) if cache else None
        return getattr(ctx.lib, fn)(ctx.handle, c, pkg.F16 if dtype is None else dtype, starts, total, k, ks, d.ptr, vs)

    for fn in ("hipc_kv4_append", "hipc_kv4_read"):
        assert rows(fn, cache=False) == 1
        assert rows(fn, dtype=pkg.U8) == 2
        assert rows(fn, head_dim=48) == 2 and rows(fn, head_dim=288) == 2 and rows(fn, head_dim=0) == 2
        assert rows(fn, page_size=8) == 2 and rows(fn, page_size=48) == 2
        assert rows(fn, n_kv_heads=0) == 1 and rows(fn, n_seqs=-1) == 1 and rows(fn, n_pages=-1) == 1 and rows(fn, table_width=-1) == 1
        assert rows(fn, table_width=1 << 27) == 1
        assert rows(fn, k_codes=None) == 1 and rows(fn, v_params=good["v_params"] + 4) == 1
        assert rows(fn, lengths=None) == 1 and rows(fn, table=None) == 1
        assert rows(fn, starts=None) == 1 and rows(fn, k=None) == 1 and rows(fn, k=d.ptr + 1) == 1
        assert rows(fn, ks=127) == 1 and rows(fn, vs=0) == 1 and rows(fn, total=-1) == 1
        assert rows(fn, total=0) == 0 and rows(fn, n_seqs=0) == 0

    def attend(heads=(4, 2, 64, 1, 0, 0.0), dtype=None, tokens=1, q=d.ptr, qs=256, y=d.ptr, **change):
        return ctx.lib.hipc_kv4_attention(ctx.handle, pkg.Kv4Cache(**{**good, **change}), pkg.AttentionHeads(*heads), pkg.F16 if dtype is None else dtype,
                                          tokens, q, qs, y, 256)

    assert attend(heads=(4, 2, 64, 0, 0, 0.0)) == 1           # not causal
    assert attend(heads=(4, 1, 64, 1, 0, 0.0)) == 1 and attend(heads=(4, 2, 128, 1, 0, 0.0)) == 1
    assert attend(heads=(3, 2, 64, 1, 0, 0.0)) == 1 and attend(heads=(4, 2, 64, 1, -1, 0.0)) == 1
    assert attend(tokens=0) == 1 and attend(tokens=513) == 2 and attend(dtype=pkg.I8) == 2
    assert attend(q=None) == 1 and attend(y=None) == 1 and attend(q=d.ptr + 1) == 1 and attend(qs=255) == 1
    assert attend(page_size=24) == 2
    assert b"hipc_kv4_attention" in ctx.lib.hipc_last_error(ctx.handle)
    assert attend(n_seqs=0) == 0
    d.free(), p.gpu.free()


@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (128, 8, 1), (256, 4, 1)])
@pytest.mark.parametrize("scale", [0.0, 1.0, 1e-30, -1e-38, 3e-45])
@pytest.mark.parametrize("tokens,window", [(1, 0), (3, 20)])
def test_queries_and_scales_of_next_to_nothing(ctx, pkg, dim, heads, kv, scale, tokens, window):
    """f32 queries down to the least number there is, with scales as small: scores of 0 to working precision, so a row is the mean of what it sees.
    Rows of every size stand beside each other."""
    p = Pair(ctx, pkg, np.random.default_rng(dim + tokens), 3, 5, 32, kv, dim)
    p.append([130, 65, 7])
    q = p.rng.standard_normal((3 * tokens, heads, dim))
    sizes = np.array([0.0, 1e-45, 1e-42, 1e-39, 1e-35, 1e-20, 1.0])
    q = (q * sizes[np.arange(q.shape[0] * heads) % len(sizes)].reshape(q.shape[0], heads, 1)).astype(np.float32)
    got = p.gpu.attention(q, tokens, window, scale)
    want, weight, size = p.ref.attention(q, p.lengths, tokens, window, scale or None)
    k_most = 2 * float(np.nanmax(np.abs(p.ref.params[0].astype(np.float64)))) * 16
    factor = abs(scale) * np.sqrt(dim) if scale else 1.0            # (the tolerance has the scale 1 / sqrt(dim) in it)
    off = np.abs(got.astype(np.float64) - want) - tolerance(np.float32, q.astype(np.float64) * max(factor, 1e-30), int(p.lengths.max()), want, weight, size, k_most)
    assert np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))
    p.gpu.free()


def test_an_infinite_query(ctx, pkg):
    """f16: NaN, or zero where all its scores are -inf; f32: NaN. The rows beside it are as without."""
    p = Pair(ctx, pkg, np.random.default_rng(31), 2, 4, 16, 1, 64)

    def change(k, v):
        k[..., 0] = -1 - np.abs(k[..., 0])

    p.append([50, 20], np.float16, change)
    for dtype in (np.float16, np.float32):
        q = p.rng.standard_normal((2, 3, 64)).astype(dtype)
        want = p.gpu.attention(q)
        q[0, 1] = 0
        q[0, 1, 0] = np.inf
        got = p.gpu.attention(q)
        assert not got[0, 1].any() if dtype == np.float16 else np.isnan(got[0, 1]).all()
        q[0, 1, 0] = -np.inf
        assert np.isnan(p.gpu.attention(q)[0, 1]).all()
        got[0, 1] = want[0, 1]
        assert np.array_equal(bits(got), bits(want))
    p.gpu.free()
