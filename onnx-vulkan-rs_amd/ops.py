"""Operator entry points over the C ABI.

Two levels: ``*_device`` functions take device pointers / ``Buffer`` objects and only
enqueue (what a benchmark or a captured graph calls); the plain functions take and return
numpy arrays in the ONNX layouts (what the parity tests call) and flush before returning.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from .runtime import (AttentionHeads, Buffer, Context, ConvGeom, F16, F32, HipComputeError, I8, Kv4Cache, RotaryHeads, RotaryScaling, U8, _ptr,
                      hipc_dtype, load_library)

_vp = C.c_void_p


# ------------------------------------------------------------------ MatMulNBits

class NBitsWeight:
    """A prepacked MatMulNBits weight (``hipc_nbits_weight``)."""

    def __init__(self, ctx: Context, B, scales, zp, K: int, N: int, block_size: int):
        """B / scales / zp: numpy arrays in the ONNX layout (zp may be None)."""
        self.ctx, self.K, self.N, self.block_size = ctx, K, N, block_size
        B = np.ascontiguousarray(B, np.uint8)
        scales = np.ascontiguousarray(scales)
        dB, dS = ctx.upload(B), ctx.upload(scales)
        dZ = None if zp is None else ctx.upload(np.ascontiguousarray(zp, np.uint8))
        h = _vp()
        ctx._check(ctx.lib.hipc_prepack_matmul_nbits(
            ctx.handle, dB.ptr, B.size, dS.ptr, hipc_dtype(scales.dtype), scales.size,
            _ptr(dZ), 0 if zp is None else zp.size, K, N, block_size, C.byref(h)))
        ctx.flush()
        for b in (dB, dS, dZ):
            if b is not None:
                b.free()
        self.handle = h

    @property
    def nbytes(self) -> int:
        return self.ctx.lib.hipc_nbits_weight_bytes(self.handle)

    def destroy(self):
        if self.handle:
            self.ctx.lib.hipc_nbits_weight_destroy(self.ctx.handle, self.handle)
            self.handle = None


def matmul_nbits_device(ctx, A, a_dtype, B, b_len, scales, scale_dtype, scales_len, zp, zp_len, Y, M, K, N,
                        block_size, accuracy_level=0):
    ctx._check(ctx.lib.hipc_matmul_nbits(ctx.handle, _ptr(A), a_dtype, _ptr(B), b_len, _ptr(scales), scale_dtype,
                                         scales_len, _ptr(zp), zp_len, _ptr(Y), M, K, N, block_size, accuracy_level))


def matmul_nbits_packed_device(ctx, A, a_dtype, weight: NBitsWeight, Y, M, accuracy_level=0):
    ctx._check(ctx.lib.hipc_matmul_nbits_packed(ctx.handle, _ptr(A), a_dtype, weight.handle, _ptr(Y), M,
                                                accuracy_level))


def matmul_nbits(ctx: Context, A, B, scales, zp, K, N, block_size, accuracy_level=0, weight: NBitsWeight = None):
    """``MatMulNBits`` on numpy operands. With ``weight`` the prepacked path runs."""
    A = np.ascontiguousarray(A)
    M = A.size // K if K else 0
    dA = ctx.upload(A)
    dY = ctx.alloc(max(M * N * A.dtype.itemsize, 4))
    if weight is not None:
        matmul_nbits_packed_device(ctx, dA, hipc_dtype(A.dtype), weight, dY, M, accuracy_level)
        tmp = []
    else:
        B = np.ascontiguousarray(B, np.uint8)
        scales = np.ascontiguousarray(scales)
        dB, dS = ctx.upload(B), ctx.upload(scales)
        dZ = None if zp is None else ctx.upload(np.ascontiguousarray(zp, np.uint8))
        matmul_nbits_device(ctx, dA, hipc_dtype(A.dtype), dB, B.size, dS, hipc_dtype(scales.dtype), scales.size,
                            dZ, 0 if zp is None else zp.size, dY, M, K, N, block_size, accuracy_level)
        tmp = [dB, dS, dZ]
    Y = ctx.download(dY, A.dtype, (M, N))
    for b in [dA, dY] + tmp:
        if b is not None:
            b.free()
    return Y.reshape(A.shape[:-1] + (N,)) if A.ndim >= 1 else Y


# -------------------------------------------------------- DynamicQuantizeLinear

def dynamic_quantize_linear_device(ctx, X, n, Y, scale_out, zp_out, range_slot=None, range_ready=False):
    ctx._check(ctx.lib.hipc_dynamic_quantize_linear(ctx.handle, _ptr(X), n, _ptr(Y), _ptr(scale_out), _ptr(zp_out),
                                                    _ptr(range_slot), int(range_ready)))


def dynamic_quantize_linear(ctx: Context, x):
    """Returns (y uint8 like x, scale float32, zero_point int)."""
    x = np.ascontiguousarray(x, np.float32)
    dX = ctx.upload(x)
    dY = ctx.alloc(max(x.size, 4))
    dP = ctx.alloc(8)
    dynamic_quantize_linear_device(ctx, dX if x.size else None, x.size, dY if x.size else None, dP, dP.at(4))
    y = ctx.download(dY, np.uint8, x.shape)
    scale = ctx.download(dP, np.float32, (1,))[0]
    zp = int(ctx.download(dP, np.uint8, (1,), offset=4)[0])
    for b in (dX, dY, dP):
        b.free()
    return y, scale, zp


def dynamic_quantize_linear_static(ctx: Context, x):
    """The same through the entry point that allocates nothing (``hipc_dynamic_quantize_linear_static``)."""
    x = np.ascontiguousarray(x, np.float32)
    dX = ctx.upload(x)
    dY = ctx.alloc(max(x.size, 4))
    dP = ctx.alloc(8)
    ctx._check(ctx.lib.hipc_dynamic_quantize_linear_static(ctx.handle, dX.ptr if x.size else None, x.size,
                                                           dY.ptr if x.size else None, dP.ptr, dP.ptr + 4))
    y = ctx.download(dY, np.uint8, x.shape)
    scale = ctx.download(dP, np.float32, (1,))[0]
    zp = int(ctx.download(dP, np.uint8, (1,), offset=4)[0])
    for b in (dX, dY, dP):
        b.free()
    return y, scale, zp


SQRT2_F32 = float(np.float32(np.sqrt(2.0)))


def decomposed_gelu(ctx: Context, x, divisor=SQRT2_F32, offset=1.0, factor=0.5, factor_first=False):
    """The exact GELU as Div, Erf, Add, Mul, Mul in one kernel (``DecomposedGelu``)."""
    x = np.ascontiguousarray(x, np.float32)
    dX, dY = ctx.upload(x), ctx.alloc(max(x.nbytes, 4))
    ctx._check(ctx.lib.hipc_decomposed_gelu(ctx.handle, dX.ptr, x.size, divisor, offset, factor, int(factor_first), dY.ptr))
    y = ctx.download(dY, np.float32, x.shape)
    dX.free(), dY.free()
    return y


def dynamic_quantize_linear_gelu(ctx: Context, x, divisor=SQRT2_F32, offset=1.0, factor=0.5, factor_first=False):
    """DynamicQuantizeLinear(DecomposedGelu(x)) in two passes over x (``DecomposedGeluQuantize``)."""
    x = np.ascontiguousarray(x, np.float32)
    dX = ctx.upload(x)
    dY = ctx.alloc(max(x.size, 4))
    dP = ctx.alloc(8)
    ctx._check(ctx.lib.hipc_dynamic_quantize_linear_gelu(ctx.handle, dX.ptr if x.size else None, x.size, divisor, offset, factor,
                                                         int(factor_first), dY.ptr if x.size else None, dP.ptr, dP.ptr + 4, None))
    y = ctx.download(dY, np.uint8, x.shape)
    scale = ctx.download(dP, np.float32, (1,))[0]
    zp = int(ctx.download(dP, np.uint8, (1,), offset=4)[0])
    for b in (dX, dY, dP):
        b.free()
    return y, scale, zp


# ------------------------------------------------------------------ MatMulInteger

class Int8Weight:
    """A prepacked MatMulInteger / QLinearMatMul B (``hipc_int8_weight``)."""

    def __init__(self, ctx: Context, B):
        B = np.ascontiguousarray(B)
        assert B.dtype in (np.uint8, np.int8) and B.ndim == 2
        self.ctx, self.K, self.N, self.dtype = ctx, B.shape[0], B.shape[1], B.dtype
        dB = ctx.upload(B)
        h = _vp()
        ctx._check(ctx.lib.hipc_prepack_int8_b(ctx.handle, dB.ptr, hipc_dtype(B.dtype), self.K, self.N, C.byref(h)))
        ctx.flush()
        dB.free()
        self.handle = h

    def destroy(self):
        if self.handle:
            self.ctx.lib.hipc_int8_weight_destroy(self.ctx.handle, self.handle)
            self.handle = None


def matmul_integer_device(ctx, A, a_dtype, weight: Int8Weight, a_zp, b_zp, Y, M):
    ctx._check(ctx.lib.hipc_matmul_integer(ctx.handle, _ptr(A), a_dtype, weight.handle, _ptr(a_zp), _ptr(b_zp),
                                           _ptr(Y), M))


def matmul_integer_scale_bias_device(ctx, A, a_dtype, weight, a_zp, b_zp, scale, scale_step, product, product_step,
                                     bias, bias_step, relu, range_slot, Y, M):
    ctx._check(ctx.lib.hipc_matmul_integer_scale_bias(
        ctx.handle, _ptr(A), a_dtype, weight.handle, _ptr(a_zp), _ptr(b_zp), _ptr(scale), scale_step, _ptr(product),
        product_step, _ptr(bias), bias_step, int(bool(relu)), _ptr(range_slot), _ptr(Y), M))


def _zp_buffer(ctx, value, dtype):
    return None if value is None else ctx.upload(np.array([value]).astype(dtype))


def matmul_integer(ctx: Context, A, B, a_zp=None, b_zp=None, weight: Int8Weight = None, raw: bool = False):
    """``MatMulInteger`` -> int32 [.., M, N]. ``raw`` packs B inside the call."""
    A = np.ascontiguousarray(A)
    B = np.ascontiguousarray(B)
    K, N = B.shape
    M = A.size // K if K else 0
    dA = ctx.upload(A)
    dY = ctx.alloc(max(M * N * 4, 4))
    dza, dzb = _zp_buffer(ctx, a_zp, A.dtype), _zp_buffer(ctx, b_zp, B.dtype)
    own = None
    tmp = [dA, dY, dza, dzb]
    if raw:
        dB = ctx.upload(B)
        tmp.append(dB)
        ctx._check(ctx.lib.hipc_matmul_integer_raw(ctx.handle, dA.ptr, hipc_dtype(A.dtype), dB.ptr, hipc_dtype(B.dtype),
                                                   _ptr(dza), _ptr(dzb), dY.ptr, M, K, N))
    else:
        if weight is None:
            weight = own = Int8Weight(ctx, B)
        matmul_integer_device(ctx, dA, hipc_dtype(A.dtype), weight, dza, dzb, dY, M)
    Y = ctx.download(dY, np.int32, (M, N))
    for b in tmp:
        if b is not None:
            b.free()
    if own:
        own.destroy()
    return Y.reshape(A.shape[:-1] + (N,))


def matmul_integer_scale_bias(ctx: Context, A, B, a_zp, b_zp, scale, bias=None, product=None, relu=False,
                              fold_range=False, weight: Int8Weight = None):
    """The fused dequantising linear layer; returns float32 [M, N] (and the folded range bits)."""
    A = np.ascontiguousarray(A)
    B = np.ascontiguousarray(B)
    K, N = B.shape
    M = A.size // K
    own = None
    if weight is None:
        weight = own = Int8Weight(ctx, B)
    dA = ctx.upload(A)
    dY = ctx.alloc(max(M * N * 4, 4))
    dza, dzb = _zp_buffer(ctx, a_zp, A.dtype), _zp_buffer(ctx, b_zp, B.dtype)

    def vec(v):
        if v is None:
            return None, 0
        a = np.ascontiguousarray(np.atleast_1d(v), np.float32)
        return ctx.upload(a), (0 if a.size == 1 else 1)

    (ds, ss), (dp, ps), (db, bs) = vec(scale), vec(product), vec(bias)
    dr = None
    if fold_range:
        dr = ctx.alloc(8)
        ctx.fill(dr, 0, 8, 0)
    matmul_integer_scale_bias_device(ctx, dA, hipc_dtype(A.dtype), weight, dza, dzb, ds, ss, dp, ps, db, bs, relu, dr,
                                     dY, M)
    Y = ctx.download(dY, np.float32, (M, N))
    rng = ctx.download(dr, np.uint32, (2,)) if dr else None
    for b in (dA, dY, dza, dzb, ds, dp, db, dr):
        if b is not None:
            b.free()
    if own:
        own.destroy()
    return (Y, rng) if fold_range else Y


def requantize(ctx: Context, acc, bias, ratio, inner, y_zp, out_signed=False):
    acc = np.ascontiguousarray(acc, np.int32)
    ratio = np.ascontiguousarray(np.atleast_1d(ratio), np.float32)
    dA, dR = ctx.upload(acc), ctx.upload(ratio)
    dB = None if bias is None else ctx.upload(np.ascontiguousarray(bias, np.int32))
    dO = ctx.alloc(max(acc.size, 4))
    ctx._check(ctx.lib.hipc_requantize(ctx.handle, dA.ptr, _ptr(dB), dR.ptr, acc.size, inner, ratio.size, int(y_zp),
                                       I8 if out_signed else U8, dO.ptr))
    out = ctx.download(dO, np.int8 if out_signed else np.uint8, acc.shape)
    for b in (dA, dR, dB, dO):
        if b is not None:
            b.free()
    return out


def _f32_vector(v):
    """`v` as a contiguous float32 vector: itself where it is one."""
    if type(v) is np.ndarray and v.dtype == np.float32 and v.ndim == 1 and v.flags.c_contiguous:
        return v
    return np.ascontiguousarray(np.atleast_1d(v), np.float32)


def qlinear_matmul_device(ctx, A, a_dtype, a_scale, a_zp, weight: Int8Weight, b_scale, b_zp, y_scale, y_zp, y_dtype, Y, M):
    bs = _f32_vector(b_scale)
    ctx._check(ctx.lib.hipc_qlinear_matmul(
        ctx.handle, _ptr(A), a_dtype, float(a_scale), int(a_zp), weight.handle, bs, bs.size, int(b_zp), float(y_scale),
        int(y_zp), y_dtype, _ptr(Y), M))


def qlinear_matmul(ctx: Context, A, a_scale, a_zp, B, b_scale, b_zp, y_scale, y_zp, y_signed=False,
                   weight: Int8Weight = None):
    A = np.ascontiguousarray(A)
    B = np.ascontiguousarray(B)
    K, N = B.shape
    M = A.size // K
    own = None
    if weight is None:
        weight = own = Int8Weight(ctx, B)
    bs = np.ascontiguousarray(np.atleast_1d(b_scale), np.float32)
    dA = ctx.upload(A)
    dY = ctx.alloc(max(M * N, 4))
    ctx._check(ctx.lib.hipc_qlinear_matmul(
        ctx.handle, dA.ptr, hipc_dtype(A.dtype), float(a_scale), int(a_zp), weight.handle,
        bs.ctypes.data_as(C.POINTER(C.c_float)), bs.size, int(b_zp), float(y_scale), int(y_zp),
        I8 if y_signed else U8, dY.ptr, M))
    Y = ctx.download(dY, np.int8 if y_signed else np.uint8, (M, N))
    dA.free(), dY.free()
    if own:
        own.destroy()
    return Y


# ------------------------------------------------------ ConvInteger / QLinearConv

class ConvWeight:
    """A prepacked convolution weight (``hipc_conv_weight``)."""

    def __init__(self, ctx: Context, W, geom: ConvGeom):
        W = np.ascontiguousarray(W)
        assert W.dtype in (np.uint8, np.int8) and W.ndim == 4
        self.ctx, self.dtype = ctx, W.dtype
        dW = ctx.upload(W)
        h = _vp()
        ctx._check(ctx.lib.hipc_prepack_conv_w(ctx.handle, dW.ptr, hipc_dtype(W.dtype), C.byref(geom), C.byref(h)))
        ctx.flush()
        dW.free()
        self.handle = h

    def destroy(self):
        if self.handle:
            self.ctx.lib.hipc_conv_weight_destroy(self.ctx.handle, self.handle)
            self.handle = None


def conv_out_shape(ctx_or_lib, geom: ConvGeom):
    lib = ctx_or_lib.lib if isinstance(ctx_or_lib, Context) else ctx_or_lib
    ho, wo = C.c_int64(), C.c_int64()
    rc = lib.hipc_conv_out_shape(C.byref(geom), C.byref(ho), C.byref(wo))
    if rc != 0:
        raise ValueError("the kernel window does not fit the padded input")
    return (geom.n, geom.c_out, ho.value, wo.value)


def conv_integer(ctx: Context, X, W, x_zp, w_zp, geom: ConvGeom, weight: ConvWeight = None):
    X = np.ascontiguousarray(X)
    W = np.ascontiguousarray(W)
    own = None
    if weight is None:
        weight = own = ConvWeight(ctx, W, geom)
    shape = conv_out_shape(ctx, geom)
    dX = ctx.upload(X)
    dY = ctx.alloc(max(int(np.prod(shape)) * 4, 4))
    dzx, dzw = _zp_buffer(ctx, x_zp, X.dtype), _zp_buffer(ctx, w_zp, W.dtype)
    ctx._check(ctx.lib.hipc_conv_integer(ctx.handle, dX.ptr, hipc_dtype(X.dtype), weight.handle, _ptr(dzx), _ptr(dzw),
                                         C.byref(geom), dY.ptr))
    Y = ctx.download(dY, np.int32, shape)
    for b in (dX, dY, dzx, dzw):
        if b is not None:
            b.free()
    if own:
        own.destroy()
    return Y


def qlinear_conv_device(ctx, X, x_dtype, x_scale, x_zp, weight: ConvWeight, w_scale: np.ndarray, w_zp, y_scale, y_zp,
                        y_dtype, bias, geom: ConvGeom, Y):
    ws = _f32_vector(w_scale)
    ctx._check(ctx.lib.hipc_qlinear_conv(
        ctx.handle, _ptr(X), x_dtype, float(x_scale), int(x_zp), weight.handle, ws, ws.size, int(w_zp), float(y_scale),
        int(y_zp), y_dtype, _ptr(bias), geom, _ptr(Y)))


def qlinear_conv(ctx: Context, X, x_scale, x_zp, W, w_scale, w_zp, y_scale, y_zp, bias, geom: ConvGeom,
                 y_signed=False, weight: ConvWeight = None):
    X = np.ascontiguousarray(X)
    W = np.ascontiguousarray(W)
    own = None
    if weight is None:
        weight = own = ConvWeight(ctx, W, geom)
    shape = conv_out_shape(ctx, geom)
    dX = ctx.upload(X)
    dY = ctx.alloc(max(int(np.prod(shape)), 4))
    dB = None if bias is None else ctx.upload(np.ascontiguousarray(bias, np.int32))
    qlinear_conv_device(ctx, dX, hipc_dtype(X.dtype), x_scale, x_zp, weight, w_scale, w_zp, y_scale, y_zp,
                        I8 if y_signed else U8, dB, geom, dY)
    Y = ctx.download(dY, np.int8 if y_signed else np.uint8, shape)
    for b in (dX, dY, dB):
        if b is not None:
            b.free()
    if own:
        own.destroy()
    return Y


# ------------------------------------------ norms and positions of queries and keys

ROTARY_LINEAR, ROTARY_BASE, ROTARY_BY_PARTS = 1, 2, 3


def rotary_frequencies(theta, rotary_dim, kind=None, factor=1.0, trained=0.0, slow=1.0, fast=32.0):
    """The frequencies of a rotation, ``[rotary_dim / 2]`` float32 on the host, stretched ``factor``-fold in one of the kinds above
    (``hipc_rotary_frequencies``)."""
    if kind is None and (factor, trained) != (1.0, 0.0):
        raise ValueError(f"rotary_frequencies: a factor of {factor} over {trained} positions and no kind")
    lib, out = load_library(), np.zeros(max(int(rotary_dim), 0) // 2, np.float32)
    scaling = None if kind is None else C.byref(RotaryScaling(kind, factor, trained, slow, fast))
    rc = lib.hipc_rotary_frequencies(theta, rotary_dim, scaling, out.ctypes.data)
    if rc != 0:
        raise HipComputeError(rc, lib.hipc_host_error().decode())
    return out


def rotary_device(ctx, heads: RotaryHeads, dtype, positions, rows, Q, q_stride, K, k_stride, Q_out, q_out_stride, K_out, k_out_stride):
    ctx._check(ctx.lib.hipc_rotary(ctx.handle, heads, dtype, _ptr(positions), rows, _ptr(Q), q_stride, _ptr(K), k_stride, _ptr(Q_out), q_out_stride,
                                   _ptr(K_out), k_out_stride))


def kv4_append_rotary_device(ctx, cache: Kv4Cache, heads: RotaryHeads, dtype, starts, total, Q, q_stride, K, k_stride, V, v_stride, Q_out, q_out_stride):
    ctx._check(ctx.lib.hipc_kv4_append_rotary(ctx.handle, cache, heads, dtype, _ptr(starts), total, _ptr(Q), q_stride, _ptr(K), k_stride, _ptr(V), v_stride,
                                              _ptr(Q_out), q_out_stride))


class Rotary:
    """Norms and rotation of a layer's heads as a program keeps them: frequencies and norm weights on the device."""

    def __init__(self, ctx: Context, n_q_heads, n_kv_heads, head_dim, frequencies, q_norm=None, k_norm=None, eps=1e-6, interleaved=False, amplitude=0.0):
        frequencies = np.ascontiguousarray(frequencies, np.float32)
        if frequencies.ndim != 1:
            raise ValueError(f"Rotary: frequencies of shape {frequencies.shape}")
        norms = [None if w is None else np.ascontiguousarray(w, np.float32) for w in (q_norm, k_norm)]
        for w in norms:
            if w is not None:
                _rows_match("Rotary", (w,), ((head_dim,),), np.float32)
        self.ctx, self.n_q_heads, self.n_kv_heads, self.head_dim = ctx, n_q_heads, n_kv_heads, head_dim
        self.buffers = [None if x is None else ctx.upload(x) for x in (frequencies, *norms)]
        self.heads = RotaryHeads(n_q_heads, n_kv_heads, head_dim, 2 * frequencies.size, int(interleaved), eps, amplitude,
                                 *(None if b is None else b.ptr for b in self.buffers))

    def rows_match(self, what, q, k):
        _rows_match(what, (q, k), ((q.shape[0], self.n_q_heads, self.head_dim), (q.shape[0], self.n_kv_heads, self.head_dim)), q.dtype)

    def __call__(self, q, k, positions):
        """``q [rows, heads, dim]`` and ``k [rows, kv heads, dim]`` at ``positions [rows]``: both normed and turned."""
        q, k, positions = np.ascontiguousarray(q), np.ascontiguousarray(k), np.asarray(positions)
        if positions.size and (positions.dtype.kind not in "iu" or positions.min() < -2 ** 31 or positions.max() >= 2 ** 31):
            raise ValueError(f"Rotary: positions ({positions.dtype}) that are no whole numbers of 32 bits")
        positions = np.ascontiguousarray(positions, np.int32)
        self.rows_match("Rotary", q, k)
        _rows_match("Rotary", (positions,), ((q.shape[0],),), np.int32)
        dQ, dK, dP = (self.ctx.upload(x) for x in (q, k, positions))
        qw, kw = self.n_q_heads * self.head_dim, self.n_kv_heads * self.head_dim
        rotary_device(self.ctx, self.heads, hipc_dtype(q.dtype), dP, q.shape[0], dQ, qw, dK, kw, dQ, qw, dK, kw)
        out = self.ctx.download(dQ, q.dtype, q.shape), self.ctx.download(dK, k.dtype, k.shape)
        for b in (dQ, dK, dP):
            b.free()
        return out

    def free(self):
        for b in self.buffers:
            if b is not None:
                b.free()


# ------------------------------------------ attention over prompts and a cache in 4 bits

KV4_GROUP = 32   # channels that share a scale and a lowest value


def prompt_attention_device(ctx, heads: AttentionHeads, dtype, Q, q_stride, K, k_stride, V, v_stride, q_starts, k_starts, n_seqs,
                            total_q, total_k, Y, y_stride):
    ctx._check(ctx.lib.hipc_prompt_attention(ctx.handle, heads, dtype, _ptr(Q), q_stride, _ptr(K), k_stride, _ptr(V), v_stride,
                                             _ptr(q_starts), _ptr(k_starts), n_seqs, total_q, total_k, _ptr(Y), y_stride))


def kv4_append_device(ctx, cache: Kv4Cache, dtype, starts, total, K, k_stride, V, v_stride):
    ctx._check(ctx.lib.hipc_kv4_append(ctx.handle, cache, dtype, _ptr(starts), total, _ptr(K), k_stride, _ptr(V), v_stride))


def kv4_read_device(ctx, cache: Kv4Cache, dtype, starts, total, K, k_stride, V, v_stride):
    ctx._check(ctx.lib.hipc_kv4_read(ctx.handle, cache, dtype, _ptr(starts), total, _ptr(K), k_stride, _ptr(V), v_stride))


def kv4_attention_device(ctx, cache: Kv4Cache, heads: AttentionHeads, dtype, tokens, Q, q_stride, Y, y_stride):
    ctx._check(ctx.lib.hipc_kv4_attention(ctx.handle, cache, heads, dtype, tokens, _ptr(Q), q_stride, _ptr(Y), y_stride))


def kv4_prompt_attention_device(ctx, cache: Kv4Cache, heads: AttentionHeads, sinks, dtype, starts, total, Q, q_stride, Y, y_stride):
    ctx._check(ctx.lib.hipc_kv4_prompt_attention(ctx.handle, cache, heads, sinks, dtype, _ptr(starts), total, _ptr(Q), q_stride, _ptr(Y), y_stride))


def _rows_match(what, arrays, shapes, dtype):
    """The device reads every operand by the first one's type and shape."""
    for x, shape in zip(arrays, shapes):
        if x.dtype != dtype or x.shape != shape:
            raise ValueError(f"{what}: {x.dtype} {x.shape} beside {dtype} {shape}")


def _starts(what, lengths, n_seqs, rows):
    n = np.asarray(lengths, np.int64)
    if n.shape != (n_seqs,) or (n < 0).any() or n.sum() > rows:
        raise ValueError(f"{what}: lengths {list(lengths)} of {n_seqs} sequences in {rows} rows")
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def prompt_attention(ctx: Context, q, k, v, q_lengths, k_lengths=None, causal=True, window=0, scale=0.0):
    """Attention over packed prompts on numpy operands: ``q [rows, heads, dim]``, ``k`` / ``v [keys, kv heads, dim]``, float16 or
    float32; the lengths of the sequences in rows and in keys (by default the same)."""
    q, k, v = (np.ascontiguousarray(x) for x in (q, k, v))
    if k_lengths is None:
        k_lengths = q_lengths
    _rows_match("prompt_attention", (k, v), (k.shape[:2] + q.shape[2:],) * 2, q.dtype)
    heads = AttentionHeads(q.shape[1], k.shape[1], q.shape[2], int(causal), window, scale)
    starts = [_starts("prompt_attention", n, len(q_lengths), x.shape[0]) for n, x in ((q_lengths, q), (k_lengths, k))]
    dQ, dK, dV, dqs, dks = (ctx.upload(x) for x in (q, k, v, *starts))
    dY = ctx.upload(np.zeros_like(q))
    row = [x.shape[1] * x.shape[2] for x in (q, k, v)]
    prompt_attention_device(ctx, heads, hipc_dtype(q.dtype), dQ, row[0], dK, row[1], dV, row[2], dqs, dks, len(q_lengths),
                            q.shape[0], k.shape[0], dY, row[0])
    y = ctx.download(dY, q.dtype, q.shape)
    for b in (dQ, dK, dV, dqs, dks, dY):
        b.free()
    return y


class Kv4Pages:
    """The memory of a paged 4-bit cache, its page table and its lengths, kept by a context (``hipc_kv4_cache``)."""

    def __init__(self, ctx: Context, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, table):
        """``table [sequences, width]``: the page numbers of every sequence."""
        table = np.ascontiguousarray(table, np.int32)
        if table.ndim != 2:
            raise ValueError(f"Kv4Pages: a table of shape {table.shape}")
        self.ctx, self.n_kv_heads, self.head_dim, self.n_seqs, self.width = ctx, n_kv_heads, head_dim, *table.shape
        rows = n_pages * n_kv_heads * page_size
        codes, params = np.zeros(rows * head_dim // 2, np.uint8), np.zeros(rows * (head_dim // KV4_GROUP) * 2, np.float16)
        self.buffers = [ctx.upload(x) for x in (codes, params, codes, params)]
        self.table, self.lengths = ctx.upload(table), ctx.upload(np.zeros(table.shape[0], np.int32))
        p = [b.ptr for b in self.buffers]
        self.cache = Kv4Cache(p[0], p[1], p[2], p[3], n_pages, page_size, n_kv_heads, head_dim, table.shape[0], self.lengths.ptr,
                              self.table.ptr, table.shape[1])

    def set_lengths(self, lengths):
        lengths = np.ascontiguousarray(lengths, np.int32)
        _rows_match("set_lengths", (lengths,), ((self.n_seqs,),), np.int32)
        self.ctx.upload(lengths, self.lengths)

    def set_table(self, table):
        table = np.ascontiguousarray(table, np.int32)
        _rows_match("set_table", (table,), ((self.n_seqs, self.width),), np.int32)
        self.ctx.upload(table, self.table)

    def append(self, k, v, new):
        """Packed rows ``[sum(new), kv heads, dim]`` become the last ``new[s]`` positions of sequence s (lengths count them already)."""
        k, v = np.ascontiguousarray(k), np.ascontiguousarray(v)
        _rows_match("append", (k, v), ((k.shape[0], self.n_kv_heads, self.head_dim),) * 2, k.dtype)
        starts = _starts("append", new, self.n_seqs, k.shape[0])
        dK, dV, ds = self.ctx.upload(k), self.ctx.upload(v), self.ctx.upload(starts)
        row = self.n_kv_heads * self.head_dim
        kv4_append_device(self.ctx, self.cache, hipc_dtype(k.dtype), ds, k.shape[0], dK, row, dV, row)
        for b in (dK, dV, ds):
            b.free()

    def append_rotary(self, rotary: Rotary, q, k, v, new):
        """``append`` of keys that ``rotary`` norms and turns on their way; returns the queries, turned by the same positions."""
        q, k, v = (np.ascontiguousarray(x) for x in (q, k, v))
        rotary.rows_match("append_rotary", q, k)
        _rows_match("append_rotary", (k, v), ((q.shape[0], self.n_kv_heads, self.head_dim),) * 2, q.dtype)
        starts = _starts("append_rotary", new, self.n_seqs, k.shape[0])
        dQ, dK, dV, ds = (self.ctx.upload(x) for x in (q, k, v, starts))
        qw, row = q.shape[1] * q.shape[2], self.n_kv_heads * self.head_dim
        kv4_append_rotary_device(self.ctx, self.cache, rotary.heads, hipc_dtype(k.dtype), ds, k.shape[0], dQ, qw, dK, row, dV, row, dQ, qw)
        out = self.ctx.download(dQ, q.dtype, q.shape)
        for b in (dQ, dK, dV, ds):
            b.free()
        return out

    def read(self, count, dtype=np.float16):
        """The last ``count[s]`` positions of every sequence, packed: (keys, values)."""
        shape = (int(np.sum(count)), self.n_kv_heads, self.head_dim)
        starts, zero = _starts("read", count, self.n_seqs, shape[0]), np.zeros(shape, dtype)
        dK, dV, ds = self.ctx.upload(zero), self.ctx.upload(zero), self.ctx.upload(starts)
        row = self.n_kv_heads * self.head_dim
        kv4_read_device(self.ctx, self.cache, hipc_dtype(np.dtype(dtype)), ds, shape[0], dK, row, dV, row)
        out = self.ctx.download(dK, dtype, shape), self.ctx.download(dV, dtype, shape)
        for b in (dK, dV, ds):
            b.free()
        return out

    def attention(self, q, tokens=1, window=0, scale=0.0):
        """``q [sequences * tokens, heads, dim]``: the newest tokens of every sequence over its cache."""
        q = np.ascontiguousarray(q)
        _rows_match("attention", (q,), ((self.n_seqs * tokens, q.shape[1], self.head_dim),), q.dtype)
        heads = AttentionHeads(q.shape[1], self.n_kv_heads, self.head_dim, 1, window, scale)
        dQ, dY = self.ctx.upload(q), self.ctx.upload(np.zeros_like(q))
        row = q.shape[1] * q.shape[2]
        kv4_attention_device(self.ctx, self.cache, heads, hipc_dtype(q.dtype), tokens, dQ, row, dY, row)
        y = self.ctx.download(dY, q.dtype, q.shape)
        dQ.free(), dY.free()
        return y

    def prompt_attention(self, q, new, window=0, sinks=0, scale=0.0):
        """Packed rows ``q [sum(new), heads, dim]``, the last ``new[s]`` positions of sequence s, over its cache; with a window the first ``sinks``
        positions stay visible."""
        q = np.ascontiguousarray(q)
        _rows_match("prompt_attention", (q,), ((q.shape[0], q.shape[1], self.head_dim),), q.dtype)
        starts = _starts("prompt_attention", new, self.n_seqs, q.shape[0])
        heads = AttentionHeads(q.shape[1], self.n_kv_heads, self.head_dim, 1, window, scale)
        dQ, dY, ds = self.ctx.upload(q), self.ctx.upload(np.zeros_like(q)), self.ctx.upload(starts)
        row = q.shape[1] * q.shape[2]
        kv4_prompt_attention_device(self.ctx, self.cache, heads, sinks, hipc_dtype(q.dtype), ds, q.shape[0], dQ, row, dY, row)
        y = self.ctx.download(dY, q.dtype, q.shape)
        for b in (dQ, dY, ds):
            b.free()
        return y

    def free(self):
        for b in self.buffers + [self.table, self.lengths]:
            b.free()


# ----------------------------------------------------- probabilities of the answers

TOP_MAX = 32


def token_logprobs_device(ctx, dtype, logits, row_stride, rows, vocab, tokens, logprob, entropy, top, top_ids, top_logprobs):
    ctx._check(ctx.lib.hipc_token_logprobs(ctx.handle, dtype, _ptr(logits), row_stride, rows, vocab, _ptr(tokens), _ptr(logprob),
                                           _ptr(entropy), top, _ptr(top_ids), _ptr(top_logprobs)))


def token_logprobs(ctx: Context, logits, tokens, top=0):
    """``logits [rows, vocab]`` float16 or float32, ``tokens [rows]``: (logprob, entropy, ids and log probabilities of the ``top``
    best)."""
    logits, tokens = np.ascontiguousarray(logits), np.ascontiguousarray(tokens, np.int32)
    rows, vocab = logits.shape
    _rows_match("token_logprobs", (tokens,), ((rows,),), np.int32)
    dX, dT = ctx.upload(logits), ctx.upload(tokens)
    dL, dE = ctx.alloc(max(4 * rows, 4)), ctx.alloc(max(4 * rows, 4))
    dI, dP = (ctx.alloc(4 * rows * top), ctx.alloc(4 * rows * top)) if rows * top else (None, None)
    token_logprobs_device(ctx, hipc_dtype(logits.dtype), dX, vocab, rows, vocab, dT, dL, dE, top, dI, dP)
    out = [ctx.download(dL, np.float32, (rows,)), ctx.download(dE, np.float32, (rows,))]
    out += [ctx.download(dI, np.int32, (rows, top)), ctx.download(dP, np.float32, (rows, top))] if dI else \
        [np.zeros((rows, top), np.int32), np.zeros((rows, top), np.float32)]
    for b in (dX, dT, dL, dE, dI, dP):
        if b is not None:
            b.free()
    return tuple(out)
