"""Norms and rotation of heads step by step, to the bit: a cache stores what keys are quantized to, and a key next to the border between two codes falls where these f32 steps put it.

    squares summed four side by side, then neighbours by twos; the mean, + eps; the reciprocal root right to half a step; x times that, times w; two products of a pair and their
    sum or difference; the result once to the rows' type -- in this order however many channels turn (powers of two) and however the rows are aligned (vectors of 8 or 16 bytes)

The reciprocal root's own error before its last rounding is below 2^-45 of itself, a Newton step behind a root that is off by 2^-22 at most, and a step is 2^-24 to 2^-23: no head here
lies within 2^-21 steps of the middle between two numbers (asserted), so that there is one right number. Sine and cosine are formed in 64 bits and rounded: the same f32 numbers as NumPy's
except within some 2^-27 steps of a middle.
"""
import numpy as np
import pytest

from test_kv4_gpu import bits
from test_rotary_gpu import table

pytestmark = pytest.mark.gpu
f32, f64 = np.float32, np.float64


def normed(x, w, eps):
    s = (x * x).reshape(*x.shape[:-1], -1, 4)
    s = ((s[..., 0] + s[..., 1]) + s[..., 2]) + s[..., 3]
    while s.shape[-1] > 1:
        s = s[..., 0::2] + s[..., 1::2]
    mean = s / f32(x.shape[-1]) + f32(eps)
    root = 1 / np.sqrt(mean.astype(f64))
    by = root.astype(f32)
    off = np.abs(root - by) / np.spacing(by)
    assert mean.dtype == f32 and np.all(np.abs(off - 0.5) > 2.0 ** -21)
    return x * by * w


def turned(y, positions, frequencies, interleaved, amplitude):
    turn = positions.astype(f64)[:, None] * frequencies.astype(f64) * 0.15915494309189533577
    angle = 2 * np.pi * (turn - np.rint(turn))
    cos, sin = (f(angle).astype(f32)[:, None] * f32(amplitude) for f in (np.cos, np.sin))
    n = len(frequencies)
    a, b = (np.s_[..., 0:2 * n:2], np.s_[..., 1:2 * n:2]) if interleaved else (np.s_[..., :n], np.s_[..., n:2 * n])
    out = y.copy()
    out[a], out[b] = y[a] * cos - y[b] * sin, y[b] * cos + y[a] * sin
    assert out.dtype == f32
    return out


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("dim,turn", [(64, 64), (64, 32), (128, 0), (128, 32), (128, 64), (128, 128), (256, 0), (256, 64), (256, 128), (256, 256), (512, 256)], ids=str)
@pytest.mark.parametrize("pad", [0, 4], ids=str)
@pytest.mark.parametrize("rows", [3, 700], ids=str)
def test_step_by_step(ctx, pkg, dtype, interleaved, dim, turn, pad, rows):
    rng = np.random.default_rng(dim + turn)
    heads, width, f = 3, 3 * dim + pad, table(turn)
    x = (2 * rng.standard_normal((rows, heads, dim))).astype(dtype)
    w = (1 + 0.2 * rng.standard_normal(dim)).astype(f32)
    at = rng.integers(0, 100000, rows).astype(np.int32)
    flat = np.zeros((rows, width), dtype)
    flat[:, :heads * dim] = x.reshape(rows, -1)
    turning = pkg.ops.Rotary(ctx, heads, 0, dim, f, w, None, 1e-5, interleaved, 1.25)
    d, dP = ctx.upload(flat), ctx.upload(at)
    pkg.ops.rotary_device(ctx, turning.heads, pkg.runtime.hipc_dtype(x.dtype), dP, rows, d, width, None, 0, d, width, None, 0)
    got = ctx.download(d, dtype, flat.shape)[:, :heads * dim].reshape(x.shape)
    for b in (d, dP):
        b.free()
    turning.free()
    want = turned(normed(x.astype(f32), w, 1e-5), at, f, interleaved, 1.25).astype(dtype)
    assert np.array_equal(bits(got), bits(want)), float((bits(got) != bits(want)).mean())
