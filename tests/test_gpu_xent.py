"""Softmax cross entropy of a linear classifier (mi_xent_forward, mi_xent_backward) against the formula
in 64 bits, elementwise.

Bounds, with u = 2^-24 (half a step of fp32) and h = half a step of the result's type (bf16 2^-8):
  z       ez = (K + 8) u (|x| . |w| + |b|) per element: K products and sums in fp32
  lse     |error| <= max_j ez + (2 |z - max| + 400) u + 2 u |lse|: exp of a rounded argument, sums along a path of
          at most a few hundred additions, one logarithm
  loss    twice that (lse and z_t)
  g       d p (ez + error of the argument) =: eg, elementwise; bf16 operands add h |g|
  dX      sum_j (eg + h |g|) |w| + (V + 8) u sum_j |g| |w| + h |dX|,  dW likewise over the rows
The sums over j and i are exact worst cases of the terms, so the bounds hold element by element."""
import ctypes

import numpy as np
import pytest

from tbb_test_amd import capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
H16 = 2.0 ** -8
FILL = 0x7B  # what buffers hold before a call


def bf16_bits(a):
    u = np.ascontiguousarray(a, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def widen(h):
    return (np.asarray(h, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Strided:
    """A matrix on the device with its own leading dimension and element offset; what surrounds it is checked."""

    def __init__(self, rows, cols, ld, offset, dtype, values=None):
        self.rows, self.cols, self.ld, self.offset, self.dtype = rows, cols, ld, offset, np.dtype(dtype)
        self.count = offset + rows * ld + 8
        self.host = np.full(self.count * self.dtype.itemsize, FILL, np.uint8).view(self.dtype)
        if values is not None:
            self._inside(self.host)[...] = values
        self.buf = capi.DeviceBuffer.from_numpy(self.host)

    def _inside(self, flat):
        return flat[self.offset:self.offset + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    @property
    def ptr(self):
        return self.buf.ptr + self.offset * self.dtype.itemsize

    def get(self):
        flat = self.buf.to_numpy((self.count,), self.dtype)
        inside = self._inside(flat).copy()
        self._inside(flat)[...] = self._inside(self.host)
        assert np.array_equal(flat.view(np.uint8), self.host.view(np.uint8)), "written outside the matrix"
        return inside


class Problem:
    def __init__(self, dtype, M, V, K, bias=True, seed=0, pad=0, offset=0, ignored=0.2, tweak=None, shift=0):
        rng = np.random.default_rng(seed + 7 * M + 11 * V + 13 * K)
        self.dtype, self.M, self.V, self.K = dtype, M, V, K
        self.bf16 = dtype == capi.MI_BF16
        X = rng.standard_normal((M, K)).astype(np.float32)
        W = (2.0 / np.sqrt(K) * rng.standard_normal((V, K))).astype(np.float32)
        t = rng.integers(0, V, M).astype(np.int32)
        X[::2] += (3.0 * W[t[::2]]).astype(np.float32)
        b = rng.standard_normal(V).astype(np.float32) if bias else None
        t[rng.random(M) < ignored] = -100
        if M > 4:
            t[3] = V  # just behind the last class
            t[4] = V - 1
        d = rng.uniform(0.1, 1.0, M).astype(np.float32)
        if tweak:
            tweak(X, W, b, t, d)
        if self.bf16:
            X, W = widen(bf16_bits(X)), widen(bf16_bits(W))
        self.X, self.W, self.b, self.t, self.d = X, W, b, t, d
        el = np.uint16 if self.bf16 else np.float32
        enc = bf16_bits if self.bf16 else (lambda a: a)
        self.dX_, self.dW_ = Strided(M, K, K + pad, offset, el, enc(X)), Strided(V, K, K + pad, offset, el, enc(W))
        self.dWt = Strided(K, V, V + pad, offset, el, enc(W.T)) if self.bf16 else None
        vec = lambda a: Strided(1, a.size, a.size, shift, a.dtype, a)  # noqa: E731
        self.db_, self.dt_, self.dd_ = vec(b) if bias else None, vec(t), vec(d)
        self.loss, self.lse = Strided(1, M, M, shift, np.float32), Strided(1, M, M, shift, np.float32)
        self.pad, self.offset = pad, offset
        f, w = ctypes.c_size_t(), ctypes.c_size_t()
        capi.check(capi.lib().mi_xent_workspace(dtype, M, V, K, ctypes.byref(f), ctypes.byref(w)))
        self.nf, self.nw = f.value, w.value
        self.ws = capi.DeviceBuffer(max(self.nf, self.nw) + 256)
        capi.check(capi.lib().mi_memset(self.ws.ptr, 0xFF, max(self.nf, self.nw) + 256))  # NaN in every type

    def forward(self, stream=None):
        capi.check(capi.lib().mi_xent_forward(
            self.dtype, self.M, self.V, self.K, self.dX_.ptr, self.dX_.ld, self.dW_.ptr, self.dW_.ld,
            self.db_.ptr if self.db_ else None, self.dt_.ptr, self.loss.ptr, self.lse.ptr, self.ws.ptr, self.nf, stream))

    def make_outputs(self, dw_dtype):
        el = np.uint16 if self.bf16 else np.float32
        self.gX = Strided(self.M, self.K, self.K + self.pad, self.offset, el)
        self.gW = Strided(self.V, self.K, self.K + self.pad, self.offset, np.uint16 if dw_dtype == capi.MI_BF16 else np.float32)
        self.gb = Strided(1, self.V, self.V, 0, np.float32) if self.b is not None else None
        self.dw_dtype = dw_dtype

    def backward(self, use_wt=True, dloss=True, stream=None):
        wt = self.dWt if use_wt and self.dWt is not None else None
        capi.check(capi.lib().mi_xent_backward(
            self.dtype, self.M, self.V, self.K, self.dX_.ptr, self.dX_.ld, self.dW_.ptr, self.dW_.ld,
            wt.ptr if wt else None, wt.ld if wt else 0, self.db_.ptr if self.db_ else None, self.dt_.ptr, self.lse.ptr,
            self.dd_.ptr if dloss else None, self.gX.ptr, self.gX.ld, self.dw_dtype, self.gW.ptr, self.gW.ld,
            self.gb.ptr if self.gb else None, self.ws.ptr, self.nw, stream))

    # the formula in 64 bits
    def oracle(self):
        X, W = self.X.astype(np.float64), self.W.astype(np.float64)
        b = np.zeros(self.V) if self.b is None else self.b.astype(np.float64)
        z = X @ W.T + b
        top = z.max(1, keepdims=True)
        self.lse_ref = (np.log(np.exp(z - top).sum(1)) + top[:, 0])
        self.counts = (self.t >= 0) & (self.t < self.V)
        rows = np.arange(self.M)
        zt = z[rows, np.where(self.counts, self.t, 0)]
        self.loss_ref = np.where(self.counts, self.lse_ref - zt, 0.0)
        self.ez = (self.K + 8) * U * (np.abs(X) @ np.abs(W).T + np.abs(b))
        self.span = np.abs(z - top)
        self.z = z
        return self

    def lse_bound(self):
        # exp of the far columns is not felt; 40 below the maximum it is 2^-57
        return self.ez.max(1) + (2 * np.minimum(self.span.max(1), 40.0) + 400) * U + 2 * U * np.abs(self.lse_ref)


def check_forward(p):
    p.oracle()
    p.forward()
    capi.check(capi.lib().mi_stream_sync(None))
    loss, lse = p.loss.get()[0], p.lse.get()[0]
    bound = p.lse_bound()
    assert np.all(np.abs(lse - p.lse_ref) <= bound), np.max(np.abs(lse - p.lse_ref) / bound)
    assert np.all(np.abs(loss - p.loss_ref) <= 2 * bound), np.max(np.abs(loss - p.loss_ref) / bound)
    assert np.all(loss[~p.counts] == 0.0)


def check_backward(p, dw_dtype, use_wt=True, dloss=True):
    p.make_outputs(dw_dtype)
    p.backward(use_wt, dloss)
    capi.check(capi.lib().mi_stream_sync(None))
    lse = p.lse.get()[0].astype(np.float64)  # what the call was given
    d = np.where(p.counts, p.d if dloss else 1.0, 0.0).astype(np.float64)
    x = p.z - lse[:, None]
    prob = np.exp(x)
    g = prob.copy()
    rows = np.flatnonzero(p.counts)
    g[rows, p.t[rows]] -= 1.0
    g *= d[:, None]
    eg = d[:, None] * prob * (p.ez + (4 * np.minimum(np.abs(x), 100.0) + 8) * U) + 4 * U * np.abs(g)
    h = H16 if p.bf16 else 0.0
    ag, W, X = np.abs(g), p.W.astype(np.float64), p.X.astype(np.float64)
    term = eg + (h * (1 + 2 * h) + (p.V + 8) * U) * ag + 1e-38
    gX = widen(p.gX.get()) if p.bf16 else p.gX.get()
    ref = g @ W
    bound = (term @ np.abs(W)) * (1 + 2 * h) + h * np.abs(ref) + 1e-37
    assert np.all(np.abs(gX - ref) <= bound), np.max(np.abs(gX - ref) / bound)
    assert np.all(gX[~p.counts] == 0.0)
    out16 = dw_dtype == capi.MI_BF16
    gW = widen(p.gW.get()) if out16 else p.gW.get()
    ref = g.T @ X
    term = eg + (h * (1 + 2 * h) + (p.M + 8) * U) * ag + 1e-38
    bound = (term.T @ np.abs(X)) * (1 + 2 * h) + (H16 if out16 else 0.0) * np.abs(ref) + 1e-37
    assert np.all(np.abs(gW - ref) <= bound), np.max(np.abs(gW - ref) / bound)
    if p.gb is not None:
        bound = (eg + (p.M + 8) * U * ag).sum(0) + 1e-37
        assert np.all(np.abs(p.gb.get()[0] - g.sum(0)) <= bound), np.max(np.abs(p.gb.get()[0] - g.sum(0)) / bound)


SHAPES = [(1, 1, 1), (1, 1000, 64), (5, 7, 3), (16, 64, 64), (128, 128, 128), (130, 257, 64), (129, 640, 192),
          (200, 1000, 100), (64, 4099, 65), (300, 513, 520), (513, 1030, 256)]


@pytest.mark.parametrize("M,V,K", SHAPES)
@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("bias", [True, False], ids=["bias", "plain"])
def test_loss_and_gradients(M, V, K, dtype, bias):
    p = Problem(dtype, M, V, K, bias)
    check_forward(p)
    check_backward(p, dtype)


@pytest.mark.parametrize("M,V,K", [(1, 300, 37), (9, 1000, 300), (16, 333, 31), (17, 700, 515), (33, 129, 1001), (64, 2000, 260)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 1)])
def test_few_rows_against_unaligned_classes(M, V, K, pad, offset):
    p = Problem(capi.MI_BF16, M, V, K, pad=pad, offset=offset)
    check_forward(p)


@pytest.mark.parametrize("M,V,K", [(1, 4100, 37), (9, 5000, 300), (16, 4333, 31), (17, 4700, 515), (32, 33000, 70), (33, 8200, 1001),
                                   (64, 9000, 260), (64, 33000, 90)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 1)])
@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_few_rows_against_many_classes(dtype, M, V, K, pad, offset):
    p = Problem(dtype, M, V, K, pad=pad, offset=offset)
    check_forward(p)


# pieces of whole rounds, of whole tiles and what is left over; parts of dX's sum in each
@pytest.mark.parametrize("M,V,K", [(50, 20500, 1664), (200, 20100, 512), (130, 33000, 64), (256, 17000, 1999), (5, 9000, 3776),
                                   (3000, 500, 64), (8000, 260, 130)])
def test_fp32_gradients_in_pieces(M, V, K):
    p = Problem(capi.MI_F32, M, V, K)
    check_forward(p)
    check_backward(p, capi.MI_F32)


def test_fp32_classes_that_are_no_whole_tiles():
    p = Problem(capi.MI_F32, 40, 66000, 128)  # most read in place, 80 left over
    check_forward(p)
    check_backward(p, capi.MI_F32)


@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (0, 1), (3, 0), (5, 3)])
@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_strides_and_alignment(dtype, pad, offset):
    p = Problem(dtype, 150, 384, 128, pad=pad, offset=offset)
    check_forward(p)
    check_backward(p, dtype)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_vectors_that_start_anywhere(dtype):
    p = Problem(dtype, 150, 384, 128, shift=1)  # bias, target, dloss, loss and lse at odd multiples of 4 bytes
    check_forward(p)
    check_backward(p, dtype)


@pytest.mark.parametrize("V,use_wt", [(1024, True), (1024, False), (1032, True), (1030, True)])
@pytest.mark.parametrize("dw", [capi.MI_F32, capi.MI_BF16], ids=["dw32", "dw16"])
def test_transposed_copy_and_type_of_the_weight_gradient(V, use_wt, dw):
    p = Problem(capi.MI_BF16, 260, V, 128)
    check_forward(p)
    check_backward(p, dw, use_wt, dloss=False)


def test_vocabulary_in_several_pieces_bf16():
    # wide enough that the copies of W's piece are cut: 2^27 / 16384 = 8192 classes each
    p = Problem(capi.MI_BF16, 130, 9000, 16384, bias=True)
    check_forward(p)
    check_backward(p, capi.MI_BF16, use_wt=False)
    check_backward(p, capi.MI_F32, use_wt=True)


def test_packed_weights_in_several_launches():
    # K no multiple of 64: the forward call packs 2^24 / 2112 = 7936 classes at a time
    p = Problem(capi.MI_BF16, 70, 8200, 2100)
    check_forward(p)


def test_more_rows_than_fit_at_once():
    # statistics of 2^25 / 1563 = 21248 rows at a time; the formula for the rows around the cut and at the ends
    M, V, K = 21800, 100000, 64
    rng = np.random.default_rng(11)
    X, W = widen(bf16_bits(rng.standard_normal((M, K)))), widen(bf16_bits(0.25 * rng.standard_normal((V, K))))
    t = rng.integers(-1, V, M).astype(np.int32)
    lib, dev = capi.lib(), capi.DeviceBuffer.from_numpy
    dX, dW, dt = dev(bf16_bits(X)), dev(bf16_bits(W)), dev(t)
    loss, lse = Strided(1, M, M, 0, np.float32), Strided(1, M, M, 0, np.float32)
    n = ctypes.c_size_t()
    capi.check(lib.mi_xent_workspace(capi.MI_BF16, M, V, K, ctypes.byref(n), None))
    assert n.value < 300 << 20
    ws = capi.DeviceBuffer(n.value)
    capi.check(lib.mi_xent_forward(capi.MI_BF16, M, V, K, dX.ptr, K, dW.ptr, K, None, dt.ptr, loss.ptr, lse.ptr, ws.ptr, n.value, None))
    capi.check(lib.mi_stream_sync(None))
    rows = np.r_[0:100, 21200:21300, M - 100:M]
    z = X[rows].astype(np.float64) @ W.T.astype(np.float64)
    top = z.max(1)
    want = np.log(np.exp(z - top[:, None]).sum(1)) + top
    counts = t[rows] >= 0
    ez = (K + 8) * U * (np.abs(X[rows]) @ np.abs(W).T).max(1)
    bound = ez + (2 * 40.0 + 400) * U + 2 * U * np.abs(want)
    assert np.all(np.abs(lse.get()[0][rows] - want) <= bound)
    picked = z[np.arange(len(rows)), np.where(counts, t[rows], 0)]
    assert np.all(np.abs(loss.get()[0][rows] - np.where(counts, want - picked, 0.0)) <= 2 * bound)


@pytest.mark.parametrize("M,V,K", [(2000, 64, 64), (4096, 130, 128)])
def test_long_batch_against_few_classes(M, V, K):
    p = Problem(capi.MI_BF16, M, V, K)
    check_forward(p)
    check_backward(p, capi.MI_F32)
    check_backward(p, capi.MI_BF16)


def test_fp32_logits_in_several_pieces():
    # 2^28 / 70000 rows -> 3776 classes a piece
    p = Problem(capi.MI_F32, 70000, 4000, 4, bias=True)
    check_forward(p)
    check_backward(p, capi.MI_F32)


@pytest.mark.parametrize("M,V,K", [(4000, 3400, 64),    # the tiles of the logits fill the device
                                   (300, 4090, 3600),   # those of the weight gradient do
                                   (4090, 200, 3400),   # those of the input gradient do
                                   (4090, 4300, 64),    # a whole round of tiles and some classes more: two launches
                                   (3900, 4300, 64)])   # the same, but the rows are padded differently by the two
def test_large_tiles(M, V, K):
    p = Problem(capi.MI_BF16, M, V, K)
    check_forward(p)
    check_backward(p, capi.MI_BF16)
    check_backward(p, capi.MI_F32, dloss=False)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_classes_and_rows_that_are_switched_off(dtype):
    def tweak(X, W, b, t, d):
        b[10:300] = -np.inf      # whole blocks of 64 classes among them
        b[5] = np.finfo(np.float32).min
        t[:] = np.where((t >= 10) & (t < 300), 301, t)
        d[7] = 0.0
    with np.errstate(all="ignore"):
        p = Problem(dtype, 140, 500, 64, tweak=tweak)
        b = p.b.copy()
        p.oracle()
        p.ez[:, np.isinf(b) | (b == np.finfo(np.float32).min)] = 0.0  # those logits are exact
        p.span = np.where(np.isfinite(p.span), p.span, 0.0)
        p.forward()
        capi.check(capi.lib().mi_stream_sync(None))
        bound = p.lse_bound()
        assert np.all(np.abs(p.lse.get()[0] - p.lse_ref) <= bound)
        assert np.all(np.abs(p.loss.get()[0] - p.loss_ref) <= 2 * bound)
        p.make_outputs(dtype)
        p.backward()
        capi.check(capi.lib().mi_stream_sync(None))
    gX = widen(p.gX.get()) if p.bf16 else p.gX.get()
    gW = widen(p.gW.get()) if p.bf16 else p.gW.get()
    assert np.all(np.isfinite(gX)) and np.all(np.isfinite(gW))
    assert np.all(gW[10:300] == 0.0) and np.all(p.gb.get()[0][10:300] == 0.0)
    assert np.all(gX[7] == 0.0)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_infinite_and_nan_logits_stay_in_their_row(dtype):
    def tweak(X, W, b, t, d):
        X[1, 0] = np.nan
        X[2, 0] = np.inf
        t[:] = 3
        t[6] = -1
        X[6, 0] = np.nan  # a row that does not count
    with np.errstate(all="ignore"):
        p = Problem(dtype, 20, 300, 64, tweak=tweak, ignored=0.0)
        p.forward()
        p.make_outputs(dtype)
        p.backward()
        capi.check(capi.lib().mi_stream_sync(None))
        loss, lse = p.loss.get()[0], p.lse.get()[0]
        gX = widen(p.gX.get()) if p.bf16 else p.gX.get()
    assert np.isnan(loss[1]) and np.isnan(lse[1])
    assert not np.isfinite(lse[2])
    assert loss[6] == 0.0 and np.isnan(lse[6]) and np.all(gX[6] == 0.0)
    fine = np.ones(20, bool)
    fine[[1, 2, 6]] = False
    assert np.all(np.isfinite(loss[fine])) and np.all(np.isfinite(gX[fine]))


@pytest.mark.parametrize("M,V,K", [(20, 300, 64), (33, 77, 50), (300, 700, 256), (256, 128, 128), (70, 1000, 1000)])
@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_rows_that_do_not_count_may_hold_anything(dtype, M, V, K):
    """What stands in padding rows leaves no trace in dW, db and the other rows of dX: bit for bit as with zeros there."""
    dead = [0, 5, M // 2, M - 1]

    def run(values):
        def tweak(X, W, b, t, d):
            t[dead] = [-100, V, -1, 2 ** 31 - 1]
            X[dead] = values
            d[dead] = values[:, 0]
        with np.errstate(all="ignore"):
            p = Problem(dtype, M, V, K, tweak=tweak, ignored=0.0)
        p.forward()
        p.make_outputs(dtype)
        p.backward(use_wt=False)
        capi.check(capi.lib().mi_stream_sync(None))
        assert np.all(p.loss.get()[0][dead] == 0.0)
        return p.gX.get(), p.gW.get(), p.gb.get(), np.delete(p.lse.get()[0], dead)
    zero = run(np.zeros((4, K), np.float32))
    rest = np.full((4, K), np.nan, np.float32)
    rest[1] = np.inf
    rest[2, ::2] = -np.inf
    for a, b in zip(zero, run(rest)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_rows_so_far_apart_that_a_tile_passes_32_bits(dtype):
    """W and dW with rows of 9 M elements (128 of them span more than 2^32 bytes): the same bits as dense ones."""
    M, V, K, ld = 128, 256, 64, 9 << 20
    p = Problem(dtype, M, V, K)
    p.forward()
    p.make_outputs(dtype)
    p.backward(use_wt=False)
    capi.check(capi.lib().mi_stream_sync(None))
    dense = [p.loss.get(), p.lse.get(), p.gX.get(), p.gW.get()]
    size = np.dtype(p.dX_.dtype).itemsize
    rows = p.dW_.get()

    class Far:
        def __init__(self):
            self.buf, self.ld = capi.DeviceBuffer(((V - 1) * ld + K) * size), ld
            self.ptr = self.buf.ptr

        def get(self):
            out = np.empty((V, K), rows.dtype)
            for i in range(V):
                capi.check(capi.lib().mi_memcpy_d2h(out[i].ctypes.data_as(ctypes.c_void_p), self.ptr + i * ld * size, K * size))
            return out

    p.dW_, p.gW = Far(), Far()
    for i in range(V):
        row = np.ascontiguousarray(rows[i])
        capi.check(capi.lib().mi_memcpy_h2d(p.dW_.ptr + i * ld * size, row.ctypes.data_as(ctypes.c_void_p), K * size))
    p.loss, p.lse = Strided(1, M, M, 0, np.float32), Strided(1, M, M, 0, np.float32)
    p.gX = Strided(M, K, K, 0, p.dX_.dtype)
    p.forward()
    p.backward(use_wt=False)
    capi.check(capi.lib().mi_stream_sync(None))
    for a, b in zip(dense, [p.loss.get(), p.lse.get(), p.gX.get(), p.gW.get()]):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_no_class_possible(dtype):
    def tweak(X, W, b, t, d):
        b[:] = -np.inf
        t[:] = -1
        t[2] = 5
    with np.errstate(all="ignore"):
        p = Problem(dtype, 8, 100, 64, tweak=tweak, ignored=0.0)
        p.forward()
        capi.check(capi.lib().mi_stream_sync(None))
    assert np.all(p.lse.get()[0] == -np.inf)
    loss = p.loss.get()[0]
    assert np.isnan(loss[2]) and np.all(np.delete(loss, 2) == 0.0)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_every_row_ignored(dtype):
    p = Problem(dtype, 33, 200, 64, ignored=2.0)
    p.t[:] = -1
    p.dt_ = capi.DeviceBuffer.from_numpy(p.t)
    check_forward(p)
    p.make_outputs(dtype)
    p.backward()
    capi.check(capi.lib().mi_stream_sync(None))
    assert not p.gX.get().any() and not p.gW.get().any() and not p.gb.get().any()


def test_a_sure_answer_keeps_its_small_loss():
    """loss = softplus(lse of the others - z_t): a loss of 1e-7 is still right to fp32, where lse - z_t is 0 or 2e-6."""
    M, V, K = 4, 256, 64
    X = np.zeros((M, K), np.float32)
    X[:, 0] = 1.0
    W = np.zeros((V, K), np.float32)
    W[9, 0] = 21.5
    p = Problem(capi.MI_BF16, M, V, K, bias=False)
    p.dX_, p.dW_ = Strided(M, K, K, 0, np.uint16, bf16_bits(X)), Strided(V, K, K, 0, np.uint16, bf16_bits(W))
    p.dt_ = capi.DeviceBuffer.from_numpy(np.full(M, 9, np.int32))
    p.forward()
    capi.check(capi.lib().mi_stream_sync(None))
    want = np.log1p(255.0 * np.exp(-21.5))
    # logf(255) and the subtraction round at 16: 2^-20 absolute in the exponent, the rest in ulps
    np.testing.assert_allclose(p.loss.get()[0], want, rtol=2.0 ** -19)


def test_gradient_agrees_with_differences():
    """fp32: the loss's own differences along random directions of X, W and b.  Central differences of step s on
    a loss rounded at 2^-24 of about 10: error <= 2^-20 / s + s^2 / 6 |third derivative|; s = 2^-5 leaves 2^-14."""
    M, V, K = 24, 90, 20
    p = Problem(capi.MI_F32, M, V, K)
    check_forward(p)
    p.make_outputs(capi.MI_F32)
    p.backward()
    capi.check(capi.lib().mi_stream_sync(None))
    gX, gW, gb = p.gX.get().astype(np.float64), p.gW.get().astype(np.float64), p.gb.get()[0].astype(np.float64)
    rng = np.random.default_rng(5)
    counts = p.counts

    def total(X, W, b):
        q = Problem(capi.MI_F32, M, V, K, tweak=lambda X_, W_, b_, t_, d_: (X_.__setitem__(Ellipsis, X), W_.__setitem__(Ellipsis, W),
                                                                          b_.__setitem__(Ellipsis, b)))
        q.forward()
        capi.check(capi.lib().mi_stream_sync(None))
        return float((q.loss.get()[0].astype(np.float64) * np.where(counts, p.d, 0.0)).sum())

    s = 2.0 ** -5
    for _ in range(3):
        vX, vW, vb = (rng.standard_normal(a.shape) / np.sqrt(a.size) for a in (p.X, p.W, p.b))
        up = total(p.X + s * vX, p.W + s * vW, p.b + s * vb)
        down = total(p.X - s * vX, p.W - s * vW, p.b - s * vb)
        slope = (gX * vX).sum() + (gW * vW).sum() + (gb * vb).sum()
        # M losses of rounding 2^-20 each over 2 s, and the third-order term of a softmax along a unit direction
        assert abs((up - down) / (2 * s) - slope) <= M * 2.0 ** -20 / s + s * s * M


def test_same_bits_every_time_and_on_two_streams_at_once():
    rt = ctypes.CDLL("libamdhip64.so")
    rt.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    a, b = (Problem(capi.MI_BF16, 300, 2000, 256, seed=s) for s in (1, 2))
    want = []
    for p in (a, b):
        check_forward(p)
        check_backward(p, capi.MI_F32)
        want.append([x.get() for x in (p.loss, p.lse, p.gX, p.gW, p.gb)])
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        assert rt.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0
    for _ in range(5):
        for p, s in zip((a, b), streams):
            p.forward(s)
            p.backward(stream=s)
    for s in streams:
        capi.check(capi.lib().mi_stream_sync(s))
    for p, w in zip((a, b), want):
        for x, y in zip((p.loss, p.lse, p.gX, p.gW, p.gb), w):
            assert np.array_equal(x.get().view(np.uint8), y.view(np.uint8))
    for s in streams:
        rt.hipStreamDestroy(s)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_captured_and_replayed(dtype):
    rt = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    stream, graph, run = vp(), vp(), vp()
    assert rt.hipStreamCreateWithFlags(ctypes.byref(stream), ctypes.c_uint(1)) == 0
    p = Problem(dtype, 200, 700, 100)
    check_forward(p)
    check_backward(p, dtype)
    want = [x.get() for x in (p.loss, p.lse, p.gX, p.gW, p.gb)]
    assert rt.hipStreamBeginCapture(stream, ctypes.c_int(1)) == 0
    p.forward(stream)
    p.backward(stream=stream)
    assert rt.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        capi.check(capi.lib().mi_memset(p.ws.ptr, 0xFF, p.ws.nbytes))
        capi.check(capi.lib().mi_memset(p.gX.buf.ptr, FILL, p.gX.buf.nbytes))
        capi.check(capi.lib().mi_stream_sync(None))
        assert rt.hipGraphLaunch(run, stream) == 0
        capi.check(capi.lib().mi_stream_sync(stream))
        for x, y in zip((p.loss, p.lse, p.gX, p.gW, p.gb), want):
            assert np.array_equal(x.get().view(np.uint8), y.view(np.uint8))
        other = Problem(dtype, 50, 80, 64)  # the program's own work between replays
        check_forward(other)
    rt.hipGraphExecDestroy(run)
    rt.hipGraphDestroy(graph)
    rt.hipStreamDestroy(stream)


# A cut in two (a whole round of 256 x 256 tiles and some classes more) of a call so small that dX, dW and db share a
# launch: both parts' column sums have to reach db.  In the first three the left-over classes are on 64 x 64 tiles,
# in the last two on 128 x 128.
@pytest.mark.parametrize("M,V,K", [(4096, 4300, 192), (4096, 4097, 128), (4300, 4300, 128), (6592, 5107, 96), (5376, 4096, 192)])
def test_bias_gradient_of_classes_cut_in_two(M, V, K):
    p = Problem(capi.MI_BF16, M, V, K)
    check_forward(p)
    check_backward(p, capi.MI_BF16)
    check_backward(p, capi.MI_F32, dloss=False)


# (M, V, K) by how dX is written: one launch for all results, tiles of one piece, sums over several pieces (2^27 / 16384 = 8192
# classes each), fp32 sums folded, fp32 products straight into dX
@pytest.mark.parametrize("dtype,M,V,K", [(capi.MI_BF16, 20, 300, 64), (capi.MI_BF16, 300, 700, 2048), (capi.MI_BF16, 16, 8300, 16384),
                                         (capi.MI_F32, 20, 300, 64), (capi.MI_F32, 1024, 256, 4096), (capi.MI_F32, 1000, 256, 4096)])
def test_rows_that_do_not_count_have_a_zero_gradient_whatever_the_weights_hold(dtype, M, V, K):
    dead = [0, 5, M // 2, M - 1]

    def tweak(X, W, b, t, d):
        t[dead] = [-100, V, -1, 2 ** 31 - 1]
        W[7, 3] = np.inf
        W[V - 1, 0] = np.nan
    with np.errstate(all="ignore"):
        p = Problem(dtype, M, V, K, tweak=tweak, ignored=0.0)
    p.forward()
    p.make_outputs(dtype)
    for use_wt in (True, False):
        p.backward(use_wt)
        capi.check(capi.lib().mi_stream_sync(None))
        gX = widen(p.gX.get()) if p.bf16 else p.gX.get()
        assert np.all(gX[dead] == 0.0)
        alive = np.setdiff1d(np.arange(M), dead + ([3] if M > 4 else []))  # (row 3 of a Problem has the target V)
        assert np.all(np.isnan(gX[alive]).any(1))  # a NaN logit makes lse NaN, and that every element of the row's g


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,V,K", [(12, 300, 64), (12, 4400, 70), (300, 513, 64)])  # tiles, few rows, tiles of fp32 models
def test_an_infinite_logit_of_the_target_is_no_small_loss(dtype, M, V, K):
    """loss = lse - z_t: inf - inf is NaN, as the gradient is; the other rows lose infinitely much."""
    def tweak(X, W, b, t, d):
        b[9] = np.inf
        t[:] = 8
        t[::3] = 9
        t[5] = -1
    with np.errstate(all="ignore"):
        p = Problem(dtype, M, V, K, tweak=tweak, ignored=0.0)
    p.forward()
    capi.check(capi.lib().mi_stream_sync(None))
    loss, lse = p.loss.get()[0], p.lse.get()[0]
    want = np.full(M, np.inf)
    want[p.t == 9] = np.nan
    want[p.t == -1] = 0.0
    assert np.array_equal(loss, want, equal_nan=True)
    assert np.all(lse == np.inf)


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_the_only_class_left_costs_nothing(dtype):
    def tweak(X, W, b, t, d):
        b[:] = -np.inf
        b[4] = 0.5
        t[:] = 4
    with np.errstate(all="ignore"):
        p = Problem(dtype, 9, 300, 64, tweak=tweak, ignored=0.0)
    p.forward()
    p.make_outputs(dtype)
    p.backward()
    capi.check(capi.lib().mi_stream_sync(None))
    assert not p.loss.get().any() and not p.gX.get().any() and not p.gW.get().any() and not p.gb.get().any()


class FarRows:
    """A matrix whose rows lie `ld` elements apart, nothing between them touched from the host."""

    def __init__(self, values, ld):
        self.values, self.ld = np.ascontiguousarray(values), ld
        size = self.values.dtype.itemsize
        self.buf = capi.DeviceBuffer(((len(values) - 1) * ld + values.shape[1]) * size)
        self.ptr, self.step = self.buf.ptr, ld * size
        for i, row in enumerate(self.values):
            capi.check(capi.lib().mi_memcpy_h2d(self.ptr + i * self.step, row.ctypes.data_as(ctypes.c_void_p), row.nbytes))

    def get(self):
        out = np.empty_like(self.values)
        for i in range(len(out)):
            capi.check(capi.lib().mi_memcpy_d2h(out[i].ctypes.data_as(ctypes.c_void_p), self.ptr + i * self.step, out[i].nbytes))
        return out


@pytest.mark.parametrize("dtype", [capi.MI_BF16, capi.MI_F32], ids=["bf16", "f32"])
def test_far_rows_of_more_than_128_rows_of_x(dtype):
    """As test_rows_so_far_apart_that_a_tile_passes_32_bits, with so many rows of X that an fp32 dW comes out of dense tiles
    (up to 128 the product writes dW itself)."""
    p = Problem(dtype, 256, 192, 64)
    check_forward(p)
    check_backward(p, dtype)
    dense = [x.get() for x in (p.loss, p.lse, p.gX, p.gW, p.gb)]
    p.dW_, p.gW = FarRows(p.dW_.get(), 9 << 20), FarRows(np.full((p.V, p.K), 7, p.dW_.dtype), 9 << 20)
    p.loss, p.lse = Strided(1, p.M, p.M, 0, np.float32), Strided(1, p.M, p.M, 0, np.float32)
    p.gX, p.gb = Strided(p.M, p.K, p.K, 0, p.dX_.dtype), Strided(1, p.V, p.V, 0, np.float32)
    p.forward()
    p.backward()
    capi.check(capi.lib().mi_stream_sync(None))
    for a, b in zip(dense, [x.get() for x in (p.loss, p.lse, p.gX, p.gW, p.gb)]):
        assert np.array_equal(a, b)
