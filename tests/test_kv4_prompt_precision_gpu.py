"""Attention of packed f16 rows over the 4-bit cache: its weights hold 22 bits, whichever kernel takes a row and whatever rows stand beside it.

Tolerance, from y = sum w v, with A = sum w |v|, S = scale * sum |q| |k| (both from the reference): scores, exponentials and sums as in
test_kv4_prompt_gpu.py; a weight is two f16 terms, the second within half a step of what the first (2^-11 at most) left, 2^-22 of the weight, or
2^-32 of the row's heaviest; and the result is rounded to f16 once: half the distance of the f16 numbers around it. (Weights of one term, off by up to
2^-11, pass that half distance in one of some fifty results.)
"""
import numpy as np
import pytest

from test_kv4_prompt_gpu import ROUTES, case, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("route", list(ROUTES))
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 1, 96), (8, 2, 128), (4, 1, 256)], ids=str)
@pytest.mark.parametrize("new,lengths", [([80], [80]), ([70, 1], [300, 200]), ([3], [40])], ids=str)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)], ids=str)
def test_weights_have_22_bits(ctx, pkg, route, heads, kv, dim, new, lengths, window, sinks):
    c = case(ctx, pkg, lengths, 16, kv, dim)
    q = (1.5 * c.rng.standard_normal((sum(new), heads, dim))).astype(np.float16)
    with ctx.options(**ROUTES[route]):
        got = c.gpu.prompt_attention(q, new, window, sinks)
    want, weight, size, most = c.ref.prompt_attention(q, starts_of(new), c.lengths, window, sinks)
    keys = max(lengths)
    tol = weight * (2 * (dim + 2) * 2.0 ** -24 * size + (16 + keys) * 2.0 ** -24 + 2.0 ** -22) + keys * 2.0 ** -32 * most
    tol = tol + 0.5 * np.spacing((np.abs(want) + tol).astype(np.float16)).astype(np.float64)
    off = np.abs(got.astype(np.float64) - want) - tol
    assert np.all(off <= 0), (float(off.max()), float((off > 0).mean()))
    c.gpu.free()
