"""Log probabilities, entropy and alternatives on the GPU against 64 bits. Ids are equal; numbers are off by at most
  logprob  x - lse: the sum of exponentials, its logarithm and two roundings at the size of lse: 2^-24 (8 + 4 |lse| + 2 |x|), plus what the
           exponentials' arguments lose (they are scaled before the exponential: 2^-23 of themselves, at most ln(vocab) + 20 where they count)
  entropy  the same, with sum p |x - m| in the place of x
"""
import numpy as np
import pytest

from oracle import attention as ref

pytestmark = pytest.mark.gpu


def allowed(x, value):
    v = x.astype(np.float64)
    m = np.where(np.isfinite(v), v, 0.0).max(1)
    lse = m + np.log(np.exp(np.where(np.isfinite(v), v, -np.inf) - m[:, None]).sum(1))
    size = 8 + 4 * np.abs(lse) + 2 * (np.log(x.shape[1]) + 20)
    return 2.0 ** -23 * (size[:, None] + np.abs(value)) if value.ndim == 2 else 2.0 ** -23 * (size + np.abs(value))


def check(ctx, pkg, x, tokens, top):
    got = pkg.ops.token_logprobs(ctx, x, tokens, top)
    want = ref.token_logprobs(x, tokens, top)
    assert np.array_equal(got[2], want[2]), np.argwhere(got[2] != want[2])[:4]
    for g, w in ((got[0], want[0]), (got[1], want[1]), (got[3], want[3])):
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(np.isinf(g), np.isinf(w))
        fine = np.isfinite(w)
        assert np.all(np.abs(np.where(fine, g.astype(np.float64) - w, 0.0)[fine]) <= allowed(x, np.where(fine, w, 0.0))[fine])
    return got


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 3), (3, 63, 5), (2, 64, 32), (5, 1000, 20), (2, 4097, 0), (1, 100003, 20), (3, 65536, 1), (1, 262144, 32), (40, 9001, 4)])
def test_rows_of_logits(ctx, pkg, dtype, rows, vocab, top):
    rng = np.random.default_rng(vocab + rows)
    x = (3 * rng.standard_normal((rows, vocab))).astype(dtype)
    check(ctx, pkg, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("kind", ["equal", "few values", "ascending", "descending", "one of many", "banned", "all but three banned", "large", "lowest"])
def test_ties_orders_and_masks(ctx, pkg, dtype, kind):
    rng = np.random.default_rng(3)
    n = 30011
    x = {"equal": np.full(n, 1.5), "few values": rng.integers(0, 4, n), "ascending": np.arange(n) / n, "descending": -np.arange(n) / n,
         "one of many": np.where(np.arange(n) == 17777, 9.0, -9.0), "banned": np.where(rng.random(n) < 0.5, -np.inf, rng.standard_normal(n)),
         "all but three banned": np.where(np.isin(np.arange(n), (5, 20000, 30010)), 1.0, -np.inf), "large": 60000 * (rng.random(n) - 0.5),
         "lowest": np.where(rng.random(n) < 0.9, np.finfo(dtype).min, rng.standard_normal(n))}[kind]
    x = np.stack([x, np.roll(x, 77)]).astype(dtype)
    check(ctx, pkg, x, np.array([5, 20000]), 32)


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 131077), (300, 9001), (300, 20021), (100, 90001)], ids=["shared", "alone", "alone, streamed", "shared, streamed"])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_every_way_through_a_row(ctx, pkg, dtype, rows, vocab, top):
    """Rows that one workgroup has or several, held in registers or streamed, with values that are equal, few, in order or banned."""
    rng = np.random.default_rng(top + vocab)
    i = np.arange(vocab)
    kinds = [np.full(vocab, -2.5), rng.integers(0, 3, vocab), i / vocab, -i / vocab, rng.standard_normal(vocab),
             np.where(rng.random(vocab) < 0.999, -np.inf, rng.standard_normal(vocab)), np.where(np.isin(i, (5, vocab // 2, vocab - 1)), 1.0, -np.inf),
             np.where(rng.random(vocab) < 0.9, np.finfo(dtype).min, rng.standard_normal(vocab)), np.where(i < vocab - 7, 0.0, np.nan), np.full(vocab, -np.inf)]
    x, tokens = np.stack(kinds).astype(dtype), np.full(len(kinds), 5)
    with np.errstate(all="ignore"):
        want = ref.token_logprobs(x, tokens, top)
        bound = [allowed(x, np.where(np.isfinite(want[j]), want[j], 0.0)) for j in (0, 1, 3)]
    for first in range(0, len(kinds), min(rows, len(kinds))):
        pick = (first + np.arange(rows)) % len(kinds)
        got = pkg.ops.token_logprobs(ctx, x[pick], tokens[pick], top)
        assert np.array_equal(got[2], want[2][pick]), np.argwhere(got[2] != want[2][pick])[:4]
        for j, limit in zip((0, 1, 3), bound):
            w = want[j][pick]
            assert np.array_equal(np.isnan(got[j]), np.isnan(w)) and np.array_equal(np.isinf(got[j]), np.isinf(w))
            fine = np.isfinite(w)
            assert np.all(np.abs(got[j][fine].astype(np.float64) - w[fine]) <= limit[pick][fine])


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
def test_rows_without_a_distribution(ctx, pkg, dtype):
    """All -inf, a +inf, a NaN, nothing but NaN: NaN, with the ids of what compares; the rows around them are untouched by it."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 5000)).astype(dtype)
    x[1], x[2, 77], x[3, 4000], x[4] = -np.inf, np.inf, np.nan, np.nan
    got = check(ctx, pkg, x, np.array([1, 2, 3, 4, 5, 6]), 4)
    assert np.isnan(got[0][1:5]).all() and np.isnan(got[1][1:5]).all() and np.isfinite(got[0][[0, 5]]).all()
    assert got[2][1].tolist() == [0, 1, 2, 3] and got[2][2][0] == 77 and got[2][4].tolist() == [-1] * 4


def test_tokens_that_are_none(ctx, pkg):
    x = np.random.default_rng(5).standard_normal((5, 100)).astype(np.float32)
    got = check(ctx, pkg, x, np.array([-1, 100, -2, 99, 1 << 30]), 2)
    assert got[0][0] == 0 and np.isnan(got[0][[1, 2, 4]]).all() and got[0][3] < 0


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
def test_strides_offsets_and_parts_of_the_answer(ctx, pkg, dtype):
    """Rows apart by an odd number of elements, off 16 bytes; any of the outputs alone; the rest is left as it was."""
    rng = np.random.default_rng(6)
    rows, vocab, stride, off = 7, 1003, 1011, 3
    buf = rng.standard_normal(off + rows * stride).astype(dtype)
    x = np.stack([buf[off + r * stride: off + r * stride + vocab] for r in range(rows)])
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    want = pkg.ops.token_logprobs(ctx, x, tokens, 3)
    dX, dT, dO = ctx.upload(buf), ctx.upload(tokens), ctx.upload(np.zeros(16 * rows, np.float32))
    code, at = pkg.runtime.hipc_dtype(dtype), dX.at(off * buf.itemsize)
    part = lambda i: dO.at(4 * rows * i)  # noqa: E731
    pkg.ops.token_logprobs_device(ctx, code, at, stride, rows, vocab, dT, part(0), None, 0, None, None)
    pkg.ops.token_logprobs_device(ctx, code, at, stride, rows, vocab, None, None, part(1), 0, None, None)
    pkg.ops.token_logprobs_device(ctx, code, at, stride, rows, vocab, None, None, None, 3, part(2), part(5))
    got = ctx.download(dO, np.float32, (16, rows))
    # (the same sums in another order of lanes)
    for g, w in ((got[0], want[0]), (got[1], want[1]), (got[5:8].reshape(rows, 3), want[3])):
        assert np.all(np.abs(g.astype(np.float64) - w) <= 2 * allowed(x, w.astype(np.float64)))
    assert np.array_equal(got[2:5].reshape(rows, 3).view(np.int32), want[2]) and not got[8:].any()
    for b in (dX, dT, dO):
        b.free()


def test_of_a_decode_step_where_its_logits_lie(ctx, pkg):
    """The probabilities of the token a decode step picked, read from the decoder's own logits."""
    dec = pkg.decoder
    cfg = dict(dec.GEMMA3_1B, n_layers=1, hidden=256, ffn=512, n_q_heads=2, n_kv_heads=1, head_dim=64, vocab=1003, embed_scale=1.0)
    d = dec.Decoder(ctx, cfg, 16)
    d.load(dec.build_weights(cfg, 3))
    d.reset(5)
    dT, dL, dI, dP = ctx.alloc(4), ctx.alloc(8), ctx.alloc(12), ctx.alloc(12)
    for _ in range(3):
        d.step()
        token, _, logits, _ = d.read(want_logits=True)
        ctx.upload(np.array([token], np.int32), dT)
        pkg.ops.token_logprobs_device(ctx, pkg.F32, d.logits(), cfg["vocab"], 1, cfg["vocab"], dT, dL, dL.at(4), 3, dI, dP)
        want = ref.token_logprobs(logits[None], [token], 3)
        got = ctx.download(dL, np.float32, (2,))
        assert ctx.download(dI, np.int32, (3,))[0] == token and np.array_equal(ctx.download(dI, np.int32, (3,)), want[2][0])
        assert abs(got[0] - want[0][0]) <= allowed(logits[None], want[0])[0] and abs(got[1] - want[1][0]) <= allowed(logits[None], want[1])[0]
    for b in (dT, dL, dI, dP):
        b.free()
    d.destroy()


def test_recorded_and_replayed(ctx, pkg):
    rng = np.random.default_rng(7)
    for rows, vocab in ((1, 200000), (9, 5000)):
        x = rng.standard_normal((rows, vocab)).astype(np.float32)
        dX, dT = ctx.upload(x), ctx.upload(np.zeros(rows, np.int32))
        dL, dE, dI, dP = (ctx.alloc(4 * rows), ctx.alloc(4 * rows), ctx.alloc(20 * rows), ctx.alloc(20 * rows))
        call = lambda: pkg.ops.token_logprobs_device(ctx, pkg.F32, dX, vocab, rows, vocab, dT, dL, dE, 5, dI, dP)  # noqa: E731
        call()
        ctx.capture_begin()
        call()
        g = ctx.capture_end()
        for _ in range(3):
            x = rng.standard_normal((rows, vocab)).astype(np.float32)
            tokens = rng.integers(0, vocab, rows).astype(np.int32)
            ctx.upload(x, dX), ctx.upload(tokens, dT)
            ctx.graph_launch(g)
            got = (ctx.download(dL, np.float32, (rows,)), ctx.download(dE, np.float32, (rows,)), ctx.download(dI, np.int32, (rows, 5)), ctx.download(dP, np.float32, (rows, 5)))
            want = pkg.ops.token_logprobs(ctx, x, tokens, 5)
            for a, b in zip(got, want):
                assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
        ctx.graph_destroy(g)
        for b in (dX, dT, dL, dE, dI, dP):
            b.free()


def test_refusals(ctx, pkg):
    d = ctx.alloc(4096)

    def call(dtype=None, x=d.ptr, stride=100, rows=2, vocab=100, tokens=d.ptr, logprob=d.ptr, entropy=d.ptr, top=1, ids=d.ptr, best=d.ptr):
        return ctx.lib.hipc_token_logprobs(ctx.handle, pkg.F32 if dtype is None else dtype, x, stride, rows, vocab, tokens, logprob, entropy, top, ids, best)

    assert call(dtype=pkg.I32) == 2
    assert call(x=None) == 1 and call(x=d.ptr + 2) == 1 and call(entropy=d.ptr + 1) == 1
    assert call(stride=99) == 1 and call(rows=-1) == 1 and call(vocab=0) == 1 and call(vocab=(1 << 30) + 1, stride=1 << 31) == 1
    assert call(top=-1) == 1 and call(top=33) == 1
    assert call(tokens=None) == 1 and call(logprob=None) == 1
    assert call(ids=None) == 1 and call(best=None) == 1 and call(top=0) == 1
    assert b"hipc_token_logprobs" in ctx.lib.hipc_last_error(ctx.handle)
    assert call(rows=0) == 0 and call(rows=0, x=None, ids=None, best=None) == 0
    d.free()


def places(vocab):
    """Ids all over a row: in the first chunks, in later ones of the same wavefront, in other wavefronts and workgroups, and the last."""
    return sorted({1, 700, 1024, 1500, 3000, vocab // 3, vocab // 2, vocab - 1030, vocab - 1})


def check_rows(ctx, pkg, x, rows, top):
    """`x` in batches of `rows` rows (which decides how a row is shared): ids, and where there is a distribution the numbers."""
    tokens = np.full(len(x), 3)
    with np.errstate(all="ignore"):
        want = ref.token_logprobs(x, tokens, top)
        bound = [allowed(x, np.where(np.isfinite(want[j]), want[j], 0.0)) for j in (0, 1, 3)]
    for first in range(0, len(x), min(rows, len(x))):
        pick = (first + np.arange(rows)) % len(x)
        got = pkg.ops.token_logprobs(ctx, x[pick], tokens[pick], top)
        wrong = np.argwhere((got[2] != want[2][pick]).any(1)).ravel()
        assert not len(wrong), (pick[wrong[0]], got[2][wrong[0]], want[2][pick[wrong[0]]])
        for j, limit in zip((0, 1, 3), bound):
            w = want[j][pick]
            assert np.array_equal(np.isnan(got[j]), np.isnan(w)) and np.array_equal(np.isinf(got[j]), np.isinf(w))
            fine = np.isfinite(w)
            assert np.all(np.abs(got[j][fine].astype(np.float64) - w[fine]) <= limit[pick][fine])


WAYS = pytest.mark.parametrize("rows,vocab", [(1, 131077), (300, 9001), (300, 20021), (100, 90001)], ids=["shared", "alone", "alone, streamed", "shared, streamed"])


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@WAYS
@pytest.mark.parametrize("top", [1, 5, 32])
def test_one_step_above_many_equal_logits(ctx, pkg, dtype, rows, vocab, top):
    """Rows of one value with a few that are the next larger number of the type, anywhere: these are the best, not the equal ones in front of them."""
    lines = []
    for base in (1.0, -1.5, 0.0, -0.0):
        base = dtype(base)
        above = np.nextafter(base, dtype(np.inf), dtype=dtype)
        for p in places(vocab):
            x = np.full(vocab, base, dtype)
            x[p] = above
            lines.append(x)
        x = np.full(vocab, base, dtype)
        x[places(vocab)] = above
        lines.append(x)
    x = lines[0].copy()
    x[::977] = np.nextafter(x[0], dtype(np.inf), dtype=dtype)
    x[vocab - 5] = np.nextafter(x[977], dtype(np.inf), dtype=dtype)      # two steps
    check_rows(ctx, pkg, np.stack(lines + [x]), rows, top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@WAYS
@pytest.mark.parametrize("top", [1, 5, 32])
def test_banned_logits_beside_the_lowest_number(ctx, pkg, dtype, rows, vocab, top):
    """-inf and the type's lowest value (another way to ban): the lowest value is the larger one, also where few are."""
    rng = np.random.default_rng(vocab)
    lowest, lines = np.finfo(dtype).min, []
    for some in (1, 3, 40, 300):
        x = np.full(vocab, -np.inf, dtype)
        x[rng.choice(vocab, some, replace=False)] = lowest
        lines.append(x.copy())
        x[rng.choice(vocab, 2, replace=False)] = 1.0
        lines.append(x)
    for p in places(vocab):
        x = np.full(vocab, -np.inf, dtype)
        x[p] = lowest
        lines.append(x)
    check_rows(ctx, pkg, np.stack(lines), rows, top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@WAYS
@pytest.mark.parametrize("top", [1, 5, 32])
def test_nan_in_front_of_banned_logits(ctx, pkg, dtype, rows, vocab, top):
    """Rows that begin (or go on for a while) with NaN: the ids are those of what compares, -inf too."""
    lines = []
    for n in (1, 63, 1024, 1030, 4096, vocab - 3):
        x = np.full(vocab, -np.inf, dtype)
        x[:n] = np.nan
        lines.append(x.copy())
        x[n // 2::1500] = -np.inf
        x[min(n + 2000, vocab - 1)] = 2.0
        lines.append(x)
    x = np.full(vocab, np.nan, dtype)
    x[::700] = -np.inf
    lines.append(x)
    check_rows(ctx, pkg, np.stack(lines), rows, top)


@pytest.mark.parametrize("rows,vocab", [(1, 131077), (300, 9001), (300, 20021), (100, 90001)], ids=["shared", "alone", "alone, streamed", "shared, streamed"])
@pytest.mark.parametrize("dtype,step,shift", [(np.float32, 2.0 ** -8, 2.0 ** 14), (np.float32, 2.0 ** -4, -2.0 ** 18), (np.float16, 2.0 ** -5, 32.0), (np.float16, 8.0, -8192.0)])
def test_rows_far_from_zero(ctx, pkg, dtype, step, shift, rows, vocab):
    """A distribution does not know by how much its logits are shifted: where the type holds the shifted logits exactly, the same bits come out. The
    numbers are off by x - m (one rounding), the logarithm of the sum (8 roundings with its own) and what the exponentials' arguments lose (as above):
    nothing at the size of the logits. No log-probability is above 0: x - m is not, and the sum has the largest logit's own 1 in it."""
    rng = np.random.default_rng(vocab)
    x = (np.round(3 * rng.standard_normal((min(rows, 4), vocab)) / step) * step).astype(dtype)
    x[:, 77] = x.max(1) + dtype(40 * step)
    pick = np.arange(rows) % len(x)
    far = (x.astype(np.float64) + shift).astype(dtype)
    assert np.array_equal(far.astype(np.float64) - shift, x.astype(np.float64))
    tokens = np.where(pick % 2, 77, 5)
    near = pkg.ops.token_logprobs(ctx, x[pick], tokens, 5)
    got = pkg.ops.token_logprobs(ctx, far[pick], tokens, 5)
    for a, b in zip(got, near):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    want = ref.token_logprobs(x, tokens[:len(x)], 5)
    size = 8 + 2 * (np.log(vocab) + 20)
    for j in (0, 1, 3):
        w = want[j][pick]
        assert np.all(np.abs(got[j].astype(np.float64) - w) <= 2.0 ** -23 * (size + np.abs(w)))
    assert np.array_equal(got[2], want[2][pick]) and np.all(got[0] <= 0) and np.all(got[3] <= 0)
