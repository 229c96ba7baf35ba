"""Attention over packed prompts on the GPU against its definition in 64 bits.

Tolerance, from the formula y = sum w v: with A = sum w |v| and S = scale * sum |q| |k| (both from the reference),
  * a score sums dim products in f32: it is off by at most (dim + 2) 2^-24 S, which moves every weight by twice that (its own score
    and the sum it is divided by). f32 factors are three bf16 terms of 8 bits, which sum to them; of the products of terms those of a second
    and a third (below 2^-7 and 2^-15 of the factor) and of two thirds are left out: 2 * 2^-22 + 2^-30 < 9 * 2^-24, in the second product too;
  * an exponential, a running rescale and the sums over the keys add less than (16 + keys) 2^-24 relative (one rounding a key at most);
  * f16 rounds each weight for the second product, half a step of 2^-11, and the result once more.
"""
import numpy as np
import pytest

from oracle import attention as ref

pytestmark = pytest.mark.gpu


def tolerance(dtype, dim, keys, y, weight, size):
    relative = 2 * (dim + 2) * 2.0 ** -24 * size + (16 + keys) * 2.0 ** -24
    if dtype == np.float32:
        relative = relative + 2 * 9 * 2.0 ** -24 * size + 9 * 2.0 ** -24
    if dtype == np.float16:
        return weight * (relative + 2.0 ** -11) + np.abs(y) * 2.0 ** -11 + 2.0 ** -25
    return weight * relative + 1e-37


def operands(rng, dtype, nq, nk, heads, kv, dim, gain=1.5):
    return ((gain * rng.standard_normal((nq, heads, dim))).astype(dtype), rng.standard_normal((nk, kv, dim)).astype(dtype),
            rng.standard_normal((nk, kv, dim)).astype(dtype))


def check(got, q, k, v, q_lengths, k_lengths, **how):
    want, weight, size = ref.prompt(q, k, v, q_lengths, k_lengths, **how)
    tol = tolerance(q.dtype, q.shape[2], max(list(k_lengths) + [1]), want, weight, size)
    off = np.abs(got.astype(np.float64) - want) - tol
    assert np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("lengths", [[1], [2, 1, 3], [31, 33], [64], [65, 1, 130], [257], [300, 7]], ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 256), (4, 2, 128), (3, 3, 64)])
def test_whole_prompts(ctx, pkg, dtype, lengths, heads, kv, dim):
    q, k, v = operands(np.random.default_rng(sum(lengths) + dim), dtype, sum(lengths), sum(lengths), heads, kv, dim)
    check(pkg.ops.prompt_attention(ctx, q, k, v, lengths), q, k, v, lengths, lengths)


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (9, 3, 80), (12, 1, 96), (5, 1, 32), (2, 1, 8), (3, 1, 7), (2, 2, 33), (16, 2, 160), (2, 1, 248),
                                          (1, 1, 264), (2, 1, 512), (1, 1, 1), (40, 1, 64)])
def test_head_layouts(ctx, pkg, dtype, heads, kv, dim):
    lengths = [70, 5]
    q, k, v = operands(np.random.default_rng(dim), dtype, 75, 75, heads, kv, dim)
    check(pkg.ops.prompt_attention(ctx, q, k, v, lengths), q, k, v, lengths, lengths)


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("q_lengths,k_lengths", [([5], [200]), ([1, 1], [513, 2]), ([64, 3], [65, 300]), ([40], [17]), ([9, 4], [0, 4]), ([0, 6, 0], [3, 6, 9]), ([130], [700])], ids=str)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 33), (True, 64)])
def test_pieces_windows_and_rows_that_see_nothing(ctx, pkg, dtype, q_lengths, k_lengths, causal, window):
    q, k, v = operands(np.random.default_rng(sum(k_lengths) + window), dtype, sum(q_lengths), sum(k_lengths), 4, 2, 64)
    got = pkg.ops.prompt_attention(ctx, q, k, v, q_lengths, k_lengths, causal=causal, window=window)
    check(got, q, k, v, q_lengths, k_lengths, causal=causal, window=window)
    if q_lengths == [40]:
        assert causal is False or not got[:23].any()     # positions below 0


@pytest.mark.parametrize("dtype,waves,dim,many", [(np.float16, 4, 16, True), (np.float16, 8, 16, False), (np.float16, 4, 136, False), (np.float32, 2, 16, True),
                                                  (np.float32, 4, 72, False)])
def test_more_tiles_than_run_at_once(ctx, pkg, dtype, waves, dim, many):
    """Tiles of all sequences are started in the order of the keys they see: sequences of very different lengths, empty ones, ones behind
    earlier keys and with fewer keys than rows; every row is there."""
    rng = np.random.default_rng(dim + many)
    if many:
        q_lengths = rng.integers(0, 70, 64)
        k_lengths = np.where(rng.random(64) < 0.3, q_lengths, np.maximum(q_lengths + rng.integers(-20, 90, 64), 0))
    else:
        q_lengths, k_lengths = np.array([0, 700, 1, 333, 0, 64, 1005]), np.array([5, 700, 41, 900, 3, 20, 1134])
    heads, kv = (40, 40) if dim <= 128 else (16, 8)
    rows, keys = int(q_lengths.sum()), int(k_lengths.sum())
    tile = 32 * waves // (2 if dim > 128 else 1)
    assert (-(-rows * (heads // kv) // tile) + len(q_lengths)) * kv > 2 * 256      # (of 256 CUs)
    q, k, v = operands(rng, dtype, rows, keys, heads, kv, dim)
    with ctx.options(HIPC_PROMPT_WAVES=waves):
        got = pkg.ops.prompt_attention(ctx, q, k, v, q_lengths, k_lengths)
    check(got, q, k, v, q_lengths, k_lengths)


@pytest.mark.parametrize("dtype,dim", [(np.float16, 64), (np.float16, 256), (np.float32, 128), (np.float16, 33)])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, pkg, dtype, dim):
    """Infinities and NaN in keys and values behind the causal border, in front of the window and in other sequences."""
    lengths, window = [90, 70], 40
    rng = np.random.default_rng(3)
    q, k, v = operands(rng, dtype, 160, 160, 2, 1, dim)
    bad_k, bad_v = k.copy(), v.copy()
    bad_k[60], bad_v[60] = np.nan, np.inf
    bad_v[61, 0, dim // 2], bad_k[62, 0, 0] = -np.inf, np.inf
    bad_v[63] = np.nan
    for hidden in (bad_k, bad_v):
        hidden[159] = np.nan          # the last key of the last sequence: its last row alone sees it
    got = pkg.ops.prompt_attention(ctx, q, bad_k, bad_v, lengths, window=window)
    want = pkg.ops.prompt_attention(ctx, q, k, v, lengths, window=window)
    clean = np.ones(160, bool)
    clean[60:90] = clean[159] = False      # rows at 60.. of the first sequence see one of the four (a window of 40)
    assert np.array_equal(got[clean].view(np.uint8), want[clean].view(np.uint8))
    assert np.isnan(got[60:90].astype(np.float32)).any(axis=(1, 2)).all() and np.isnan(got[159].astype(np.float32)).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
def test_large_and_small_scores(ctx, pkg, dtype):
    """Scores of some hundreds (one key takes the whole weight) and of nearly nothing, and values near the type's ends."""
    rng = np.random.default_rng(8)
    for gain in (60.0, 1e-4):
        q, k, v = operands(rng, dtype, 100, 100, 4, 2, 64, gain)
        v = (v * dtype(1000.0 if dtype == np.float16 else 1e30)).astype(dtype)
        check(pkg.ops.prompt_attention(ctx, q, k, v, [100]), q, k, v, [100], [100])


def test_scale_argument(ctx, pkg):
    q, k, v = operands(np.random.default_rng(9), np.float32, 40, 40, 2, 1, 64)
    for scale in (0.5, -0.25):
        check(pkg.ops.prompt_attention(ctx, q, k, v, [40], scale=scale), q, k, v, [40], [40], scale=scale)


@pytest.mark.parametrize("dtype,dim,pad", [(np.float16, 64, 0), (np.float16, 64, 3), (np.float32, 128, 0), (np.float32, 128, 1)])
def test_parts_of_one_projection_and_rows_left_alone(ctx, pkg, dtype, dim, pad):
    """q|k|v side by side in rows of one buffer (with `pad` odd values behind, also off 16 bytes); rows in front of the first and
    behind the last sequence of Y keep what they held."""
    heads, kv, total, lengths = 4, 2, 50, [20, 11]
    width = (heads + 2 * kv) * dim + pad
    rng = np.random.default_rng(dim + pad)
    rows = rng.standard_normal((total, width)).astype(dtype)
    size = rows.itemsize
    dX, dY = ctx.upload(rows), ctx.upload(np.full((total, heads * dim), 7, dtype))
    starts = np.array([4, 24, 35], np.int32)
    dS = ctx.upload(starts)
    h = pkg.AttentionHeads(heads, kv, dim, 1, 0, 0.0)
    pkg.ops.prompt_attention_device(ctx, h, pkg.runtime.hipc_dtype(dtype), dX, width, dX.at(heads * dim * size), width, dX.at((heads + kv) * dim * size), width,
                                    dS, dS, 2, total, total, dY, heads * dim)
    y = ctx.download(dY, dtype, (total, heads, dim))
    assert np.all(y[:4] == 7) and np.all(y[35:] == 7)
    cut = rows[4:35, :(heads + 2 * kv) * dim].reshape(31, heads + 2 * kv, dim)
    check(y[4:35], cut[:, :heads], cut[:, heads:heads + kv], cut[:, heads + kv:], lengths, lengths)
    for b in (dX, dY, dS):
        b.free()


def test_starts_that_say_too_much_are_held_to_the_totals(ctx, pkg):
    """Sequences that would end behind the rows, and starts that do not ascend: nothing outside is read or written."""
    q, k, v = operands(np.random.default_rng(11), np.float16, 64, 64, 2, 1, 64)
    dQ, dK, dV, dY = ctx.upload(q), ctx.upload(k), ctx.upload(v), ctx.upload(np.full_like(q, 7))
    h = pkg.AttentionHeads(2, 1, 64, 1, 0, 0.0)
    for starts, rows in (([0, 64, 1 << 30], slice(0, 64)), ([-5, 64], slice(0, 64))):
        dS = ctx.upload(np.array(starts, np.int32))
        ctx.upload(np.full_like(q, 7), dY)
        pkg.ops.prompt_attention_device(ctx, h, pkg.F16, dQ, 128, dK, 64, dV, 64, dS, dS, len(starts) - 1, 64, 64, dY, 128)
        check(ctx.download(dY, np.float16, q.shape)[rows], q, k, v, [64], [64])
        dS.free()
    for b in (dQ, dK, dV, dY):
        b.free()


def test_a_recorded_call_follows_the_starts(ctx, pkg):
    """Replayed with other lengths in the same memory, with the program's own work between the replays."""
    rng = np.random.default_rng(12)
    q, k, v = operands(rng, np.float16, 400, 400, 4, 1, 128)
    dQ, dK, dV, dY = ctx.upload(q), ctx.upload(k), ctx.upload(v), ctx.upload(np.zeros_like(q))
    dS = ctx.upload(np.array([0, 200, 400], np.int32))
    h = pkg.AttentionHeads(4, 1, 128, 1, 0, 0.0)
    call = lambda: pkg.ops.prompt_attention_device(ctx, h, pkg.F16, dQ, 512, dK, 128, dV, 128, dS, dS, 2, 400, 400, dY, 512)  # noqa: E731
    call()
    ctx.capture_begin()
    call()
    g = ctx.capture_end()
    for cut in (1, 399, 130):
        ctx.upload(np.array([0, cut, 400], np.int32), dS)
        ctx.graph_launch(g)
        got = ctx.download(dY, np.float16, q.shape)
        want = pkg.ops.prompt_attention(ctx, q, k, v, [cut, 400 - cut])
        assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
    ctx.graph_destroy(g)
    for b in (dQ, dK, dV, dY, dS):
        b.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("waves", [1, 2, 4, 8])
@pytest.mark.parametrize("split", [1, 2, 5])
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 256), (6, 2, 128), (3, 1, 64)])
def test_every_launch_shape(ctx, pkg, dtype, waves, split, heads, kv, dim):
    """Workgroups of 4 and 8 wavefronts, of four that share 32 rows (1) and of one (2), alone with their keys or sharing them, over sequences that end anywhere in a tile."""
    q_lengths, k_lengths = [70, 3, 1], [200, 3, 90]
    q, k, v = operands(np.random.default_rng(dim + split), dtype, 74, 293, heads, kv, dim)
    with ctx.options(HIPC_PROMPT_WAVES=waves, HIPC_PROMPT_SPLIT=split):
        for how in (dict(), dict(window=50), dict(causal=False)):
            check(pkg.ops.prompt_attention(ctx, q, k, v, q_lengths, k_lengths, **how), q, k, v, q_lengths, k_lengths, **how)


def test_refusals(ctx, pkg):
    d = ctx.alloc(4096)

    def call(heads=(2, 1, 64, 1, 0, 0.0), dtype=None, q=d.ptr, qs=128, ks=64, starts=d.ptr, n=1, total=4, y=d.ptr):
        h = None if heads is None else pkg.AttentionHeads(*heads)
        return ctx.lib.hipc_prompt_attention(ctx.handle, h, pkg.F16 if dtype is None else dtype, q, qs, d.ptr, ks, d.ptr, 64, starts, starts, n, total, total, y, 128)

    assert call(heads=None) == 1
    assert call(heads=(3, 2, 64, 1, 0, 0.0)) == 1          # query heads no multiple of the kv heads
    assert call(heads=(2, 0, 64, 1, 0, 0.0)) == 1
    assert call(heads=(2, 1, 0, 1, 0, 0.0)) == 1
    assert call(heads=(2, 1, 513, 1, 0, 0.0), qs=2000, ks=2000) == 2
    assert call(heads=(2, 1, 64, 0, 5, 0.0)) == 1          # a window without a causal mask
    assert call(heads=(2, 1, 64, 1, -1, 0.0)) == 1
    assert call(heads=(2, 1, 64, 1, 0, float("nan"))) == 1
    assert call(dtype=pkg.I32) == 2
    assert call(q=None) == 1 and call(y=None) == 1 and call(starts=None) == 1
    assert call(qs=127) == 1 and call(ks=63) == 1
    assert call(q=d.ptr + 1) == 1 and call(starts=d.ptr + 2) == 1
    assert call(total=-1) == 1 and call(n=-1) == 1 and call(total=(1 << 30) + 1) == 1
    assert b"hipc_prompt_attention" in ctx.lib.hipc_last_error(ctx.handle)
    assert call(n=0) == 0 and call(total=0) == 0           # nothing to do
    d.free()


@pytest.mark.parametrize("waves,split", [(1, 1), (1, 4), (2, 1), (4, 1), (4, 3), (8, 1), (-1, -1)])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_many_keys_far_below_one(ctx, pkg, waves, split, dim, at):
    """One key e^18 times as heavy as each of 60000 others, which together weigh 9e-4: they are not lost. A weight in f16 is off by half a step, 2^-11 of
    itself, or where it is subnormal by 2^-25; weights are kept 2^7 times as large, so that is 2^-32 of the heaviest one a key,
    in the weighted sum (times |v|) and in the sum it is divided by."""
    rng = np.random.default_rng(dim)
    keys, heads, rows = 60001, 2, 3
    q, k, v = np.zeros((rows, heads, dim), np.float16), np.zeros((keys, 1, dim), np.float16), np.zeros((keys, 1, dim), np.float16)
    q[:, :, 0] = np.sqrt(dim)                                   # a score is the key's first channel
    k[:, 0, 0] = rng.uniform(-0.2, 0.2, keys)
    v[:, 0, :] = 1 + np.arange(dim) / dim
    one = {"first": 5, "middle": 31007, "last": keys - 7}[at]
    k[one, 0, 0], v[one] = 18.0, 0.0
    v[one, 0, ::3] = 0.01
    with ctx.options(HIPC_PROMPT_WAVES=waves, HIPC_PROMPT_SPLIT=split):
        got = pkg.ops.prompt_attention(ctx, q, k, v, [rows], [keys])
    want, weight, size = ref.prompt(q, k, v, [rows], [keys])
    assert 8e-4 < want[0, 0, 1] < 4e-3
    tol = tolerance(np.float16, dim, keys, want, weight, size) + keys * 2.0 ** -32 * (2.0 + np.abs(want))
    off = np.abs(got.astype(np.float64) - want) - tol
    assert np.all(off <= 0), (float(off.max()), float(got[0, 0, 1]), want[0, 0, 1])


@pytest.mark.parametrize("dtype,waves,split,dim", [(np.float16, w, s, d) for w in (1, 2, 4, 8) for s in (1, 3) for d in (64, 256)] +
                         [(np.float32, w, s, d) for w in (4, 8) for s in (1, 3) for d in (64, 256)] + [(np.float16, -1, -1, 264), (np.float32, -1, -1, 264), (np.float16, -1, -1, 100)])
@pytest.mark.parametrize("kind", ["light", "outweighed later", "outweighed before"])
def test_an_infinity_that_is_seen_reaches_the_row(ctx, pkg, dtype, waves, split, dim, kind):
    """Whatever its key weighs: e^-30 of the others in a tile that all rows see, or e^-150 of one that comes later, or before. The channels it is not in are
    as without."""
    rng = np.random.default_rng(dim)
    rows, keys, heads = 5, 700, 2
    q, k, v = np.zeros((rows, heads, dim), dtype), np.zeros((keys, 1, dim), dtype), rng.standard_normal((keys, 1, dim)).astype(dtype)
    q[:, :, 0] = np.sqrt(dim).astype(dtype)
    k[:, 0, 0] = rng.uniform(-0.5, 0.5, keys)
    odd = np.array([10, 11, 12, 13, 14]) + (500 if kind == "outweighed before" else 0)
    if kind == "light":
        k[odd, 0, 0] = -30.0
    else:
        k[20 if kind == "outweighed before" else 600, 0, 0] = 150.0
    v[odd[0], 0, 0], v[odd[1], 0, 1] = np.inf, -np.inf
    v[odd[2], 0, 2], v[odd[3], 0, 2] = np.inf, -np.inf
    v[odd[4], 0, dim - 1] = np.nan
    with ctx.options(HIPC_PROMPT_WAVES=waves, HIPC_PROMPT_SPLIT=split):
        got = pkg.ops.prompt_attention(ctx, q, k, v, [rows], [keys]).astype(np.float64)
    assert np.all(got[..., 0] == np.inf) and np.all(got[..., 1] == -np.inf) and np.isnan(got[..., 2]).all() and np.isnan(got[..., dim - 1]).all()
    v[odd, 0, :3], v[odd, 0, dim - 1] = 0, 0
    want, weight, size = ref.prompt(q, k, v, [rows], [keys])
    off = np.abs(got - want) - tolerance(q.dtype, dim, keys, want, weight, size)
    assert np.all(off[..., 3:dim - 1] <= 0), float(off[..., 3:dim - 1].max())


@pytest.mark.parametrize("dtype,waves,split,dim", [(np.float16, w, s, 64) for w in (1, 2, 4, 8) for s in (1, 3)] + [(np.float16, 4, 1, 256), (np.float16, -1, -1, 264),
                                                   (np.float32, -1, -1, 264), (np.float32, -1, -1, 64)])
def test_rows_whose_scores_are_all_minus_infinity(ctx, pkg, dtype, waves, split, dim):
    """They have no weights and are zero (f32 on the matrix cores: NaN, as whatever sees an infinite query); a NaN among the scores makes NaN."""
    rng = np.random.default_rng(dim)
    q, k, v = operands(rng, dtype, 9, 200, 2, 1, dim)
    q[3], k[:, 0, 0] = 0, -1 - rng.random(200).astype(dtype)
    q[3, :, 0] = np.inf                                       # against -1 .. -2
    q[5] = q[3]
    q[5, :, 1] = np.nan
    with ctx.options(HIPC_PROMPT_WAVES=waves, HIPC_PROMPT_SPLIT=split):
        got = pkg.ops.prompt_attention(ctx, q, k, v, [9], [200])
    if dtype == np.float32 and dim == 64:
        assert np.isnan(got[3]).all()
    else:
        assert not got[3].any()
    assert np.isnan(got[5]).all()
    q[[3, 5]], got[[3, 5]] = 0, 0
    keep = [0, 1, 2, 4, 6, 7, 8]
    want, weight, size = ref.prompt(q, k, v, [9], [200])
    assert np.all(np.abs(got.astype(np.float64) - want)[keep] <= tolerance(q.dtype, dim, 200, want, weight, size)[keep])
