"""Orthogonalised update (mi_orthogonalize, mi_ortho_update_raw) against the iteration in 64 bits.

Bounds.  Every product rounds its operands to fp16: relative errors uniform within 2^-11, 2^-11 / sqrt(3) = 2.8e-4
root mean square, independent.  An iteration has three such operands (X, A, the polynomial), each entering X with a
factor of about one relative to |X|_F once X is near its limit, and later iterations do not grow what earlier ones
left (the slope of a s + b s^3 + c s^5 is below 1.6 in size where the singular values settle).  Three operands,
the last two or three iterations: sqrt(9) 2.8e-4 = 9e-4; twice that is the bound on |error|_F / |O|_F, 2e-3.  The result's
rounding to bf16 adds 2^-8 / sqrt(3) = 2.3e-3 at worst: sqrt(2^2 + 2.3^2) = 3.1e-3.  Single elements: six of those
root mean squares, plus half a bf16 step of the element."""
import ctypes

import numpy as np
import pytest

from tbb_test_amd import capi
from test_gpu_xent import Problem, Strided, bf16_bits, widen

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
NS = 2e-3            # of |O|_F, before the result is rounded
OUT = 3.1e-3         # after rounding to bf16


def newton_schulz(G, steps=5):
    a, b, c = COEF
    X = np.asarray(G, np.float64)
    flip = X.shape[0] > X.shape[1]
    X = X.T if flip else X
    norm = np.linalg.norm(X)
    X = X / norm if norm else X
    for _ in range(steps):
        A = X @ X.T
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.T if flip else X


def gradient(rng, rows, cols, kind="mixed"):
    r = max(1, min(rows, cols) // 8)
    if kind == "noise":
        G = rng.standard_normal((rows, cols))
    else:
        floor = {"mixed": 0.3, "steep": 0.02}[kind]
        G = rng.standard_normal((rows, r)) @ rng.standard_normal((r, cols)) / np.sqrt(r) + floor * rng.standard_normal((rows, cols))
    return (1e-3 * G).astype(np.float32)


def workspace(batch, rows, cols):
    n = ctypes.c_size_t()
    capi.check(capi.lib().mi_ortho_workspace(batch, rows, cols, ctypes.byref(n)))
    ws = capi.DeviceBuffer(n.value)
    capi.check(capi.lib().mi_memset(ws.ptr, 0xFF, n.value))
    return ws


def near(got, want, rel, half_step):
    norm = np.linalg.norm(want)
    rms = norm / np.sqrt(want.size)
    err = np.abs(got - want)
    assert np.linalg.norm(err) <= rel * norm, np.linalg.norm(err) / norm
    assert np.all(err <= 6 * NS * rms * 1.5 + half_step * np.abs(want)), np.max(err / rms)


class Stack:
    """`batch` matrices of one shape on the device, gaps between rows and between matrices checked."""

    def __init__(self, batch, rows, cols, ld, stride, dtype, values=None, offset=0):
        self.shape = (batch, rows, cols)
        self.ld, self.stride, self.dtype, self.offset = ld, stride, np.dtype(dtype), offset
        self.host = np.full((offset + batch * stride + rows * ld + 8) * self.dtype.itemsize, 0x7B, np.uint8).view(self.dtype)
        if values is not None:
            for i in range(batch):
                self.inside(self.host, i)[...] = values[i]
        self.buf = capi.DeviceBuffer.from_numpy(self.host)

    def inside(self, flat, i):
        _, rows, cols = self.shape
        at = self.offset + i * self.stride
        return flat[at:at + rows * self.ld].reshape(rows, self.ld)[:, :cols]

    @property
    def ptr(self):
        return self.buf.ptr + self.offset * self.dtype.itemsize

    def get(self):
        flat = self.buf.to_numpy(self.host.shape, self.dtype)
        out = np.stack([self.inside(flat, i).copy() for i in range(self.shape[0])])
        for i in range(self.shape[0]):
            self.inside(flat, i)[...] = self.inside(self.host, i)
        assert np.array_equal(flat.view(np.uint8), self.host.view(np.uint8)), "written outside the matrices"
        return out


def run(G, dtype, steps=5, pad=0, gap=0, offset=0, stream=None):
    batch, rows, cols = G.shape
    enc = bf16_bits if dtype == capi.MI_BF16 else (lambda a: a)
    src = Stack(batch, rows, cols, cols + pad, rows * (cols + pad) + gap, np.uint16 if dtype == capi.MI_BF16 else np.float32,
                [enc(g) for g in G], offset)
    dst = Stack(batch, rows, cols, cols + pad, rows * (cols + pad) + gap, np.uint16, None, offset)
    ws = workspace(batch, rows, cols)
    capi.check(capi.lib().mi_orthogonalize(dtype, batch, rows, cols, src.ptr, src.ld, src.stride, dst.ptr, dst.ld, dst.stride,
                                           steps, ws.ptr, ws.nbytes, stream))
    capi.check(capi.lib().mi_stream_sync(stream))
    return widen(dst.get())


SHAPES = [(1, 1), (1, 50), (50, 1), (3, 7), (64, 64), (100, 60), (128, 128), (129, 257), (257, 130), (300, 1000), (1000, 300),
          (512, 512), (70, 3001)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [capi.MI_F32, capi.MI_BF16], ids=["f32", "bf16"])
def test_orthogonalize(rows, cols, dtype):
    G = gradient(np.random.default_rng(rows + 3 * cols), rows, cols)
    if dtype == capi.MI_BF16:
        G = widen(bf16_bits(G))
    near(run(G[None], dtype)[0], newton_schulz(G), OUT, 2.0 ** -8)


@pytest.mark.parametrize("kind", ["noise", "mixed", "steep"])
def test_spectra(kind):
    G = gradient(np.random.default_rng(4), 320, 448, kind)
    near(run(G[None], capi.MI_F32)[0], newton_schulz(G), OUT, 2.0 ** -8)


@pytest.mark.parametrize("steps", [1, 2, 8])
def test_number_of_steps(steps):
    G = gradient(np.random.default_rng(9), 200, 150)
    near(run(G[None], capi.MI_F32, steps)[0], newton_schulz(G, steps), OUT, 2.0 ** -8)


@pytest.mark.parametrize("dtype", [capi.MI_F32, capi.MI_BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(130, 200), (200, 130)])
def test_batch_with_strides(rows, cols, dtype):
    rng = np.random.default_rng(3)
    G = np.stack([gradient(rng, rows, cols) * 10.0 ** i for i in range(-1, 3)])
    if dtype == capi.MI_BF16:
        G = widen(bf16_bits(G))
    got = run(G, dtype, pad=3, gap=17, offset=5)
    for o, g in zip(got, G):
        near(o, newton_schulz(g), OUT, 2.0 ** -8)


@pytest.mark.parametrize("rows,cols", [(300, 520), (520, 300)])
def test_large_tiles(rows, cols):
    rng = np.random.default_rng(12)
    G = np.stack([gradient(rng, rows, cols) for _ in range(70)])  # together enough 256 x 256 tiles to fill the device
    for o, g in zip(run(G, capi.MI_F32), G):
        near(o, newton_schulz(g), OUT, 2.0 ** -8)


def test_singular_values_end_near_one():
    G = gradient(np.random.default_rng(8), 256, 400, "noise")
    s = np.linalg.svd(run(G[None], capi.MI_F32)[0], compute_uv=False)
    # the limit cycle of the polynomial stays within 0.68 .. 1.21; half a percent for the roundings
    assert s.min() > 0.67 and s.max() < 1.22


@pytest.mark.parametrize("scale", [1e-36, 1e-20, 1e20, 1e37])
def test_scale_of_the_gradient_does_not_matter(scale):
    G = gradient(np.random.default_rng(2), 140, 96)
    G = (G / np.abs(G).max()).astype(np.float32)
    big = (G.astype(np.float64) * scale).astype(np.float32)
    near(run(big[None], capi.MI_F32)[0], newton_schulz(big), OUT, 2.0 ** -8)


def test_zero_and_not_finite():
    rng = np.random.default_rng(6)
    G = np.stack([np.zeros((96, 70), np.float32), gradient(rng, 96, 70), gradient(rng, 96, 70), gradient(rng, 96, 70)])
    G[1, 5, 6] = np.nan
    G[2, 0, 0] = np.inf
    O = run(G, capi.MI_F32)
    assert not O[0].any() and np.all(np.isnan(O[1])) and np.all(np.isnan(O[2]))
    near(O[3], newton_schulz(G[3]), OUT, 2.0 ** -8)


def test_in_place_bf16():
    G = widen(bf16_bits(gradient(np.random.default_rng(1), 150, 220)))
    buf = capi.DeviceBuffer.from_numpy(bf16_bits(G))
    ws = workspace(1, 150, 220)
    capi.check(capi.lib().mi_orthogonalize(capi.MI_BF16, 1, 150, 220, buf.ptr, 220, 0, buf.ptr, 220, 0, 5, ws.ptr, ws.nbytes, None))
    capi.check(capi.lib().mi_stream_sync(None))
    near(widen(buf.to_numpy((150, 220), np.uint16)), newton_schulz(G), OUT, 2.0 ** -8)


class Update:
    def __init__(self, batch, rows, cols, R, gap=0, copies=True, seed=0):
        rng = np.random.default_rng(seed + rows + cols)
        n = rows * cols
        self.batch, self.rows, self.cols, self.R = batch, rows, cols, R
        self.layer, self.replica = n + gap, batch * (n + gap) + gap
        common = [gradient(rng, rows, cols) for _ in range(batch)]
        self.G = np.stack([np.stack([c / R + 1e-4 * rng.standard_normal(c.shape) for c in common]) for _ in range(R)]).astype(np.float32)
        self.W0 = (rng.standard_normal((batch, rows, cols)) / np.sqrt(cols)).astype(np.float32)
        self.M0 = np.stack([3 * c for c in common]).astype(np.float32)
        flat = np.full(self.R * self.replica + 8, 9.0, np.float32)
        for r in range(R):
            for i in range(batch):
                at = r * self.replica + i * self.layer
                flat[at:at + n] = self.G[r, i].ravel()
        self.g = capi.DeviceBuffer.from_numpy(flat)
        self.w = Stack(batch, rows, cols, cols, self.layer, np.float32, self.W0)
        self.m = Stack(batch, rows, cols, cols, self.layer, np.float32, self.M0)
        self.w16 = Stack(batch, rows, cols, cols, self.layer, np.uint16) if copies else None
        self.wt16 = Stack(batch, cols, rows, rows, self.layer, np.uint16) if copies else None
        self.ws = workspace(batch, rows, cols)

    def call(self, lr, scale, decay, mu, nesterov, stream=None):
        capi.check(capi.lib().mi_ortho_update_raw(
            self.batch, self.rows, self.cols, self.w.ptr, self.w16.ptr if self.w16 else None, self.wt16.ptr if self.wt16 else None,
            self.m.ptr, self.g.ptr, self.layer, self.replica, self.R, lr, scale, decay, mu, nesterov, 5, self.ws.ptr,
            self.ws.nbytes, stream))

    def check(self, lr, scale, decay, mu, nesterov, times=1):
        capi.check(capi.lib().mi_stream_sync(None))
        g = self.G.astype(np.float64).sum(0)
        M, W = self.M0.astype(np.float64), self.W0.astype(np.float64)
        for _ in range(times):
            M = np.float64(np.float32(mu)) * M + g
            u = g + np.float64(np.float32(mu)) * M if nesterov else M
            O = np.stack([newton_schulz(x) for x in u])
            W = W * (1 - lr * decay) - lr * scale * O
        m = self.m.get()
        # R + 1 roundings per call in sums whose terms are at most |G| R + |M|
        room = times * (self.R + 2) * 2.0 ** -24 * (np.abs(self.G).sum(0) + np.abs(self.M0) + np.abs(M))
        assert np.all(np.abs(m - M) <= room)
        w = self.w.get()
        for i in range(self.batch):
            err = w[i] - W[i]
            step = times * lr * scale * np.linalg.norm(O[i])
            assert np.linalg.norm(err) <= NS * step + times * 4 * 2.0 ** -24 * np.linalg.norm(W[i]), np.linalg.norm(err) / step
        if self.w16:
            assert np.array_equal(self.w16.get(), bf16_bits(w))
            assert np.array_equal(self.wt16.get(), bf16_bits(w).transpose(0, 2, 1))


@pytest.mark.parametrize("batch,rows,cols,R,gap", [(1, 64, 64, 1, 0), (1, 130, 257, 3, 0), (3, 257, 130, 2, 64), (2, 256, 256, 8, 4),
                                                  (2, 33, 40, 2, 7)])
@pytest.mark.parametrize("nesterov", [0, 1])
def test_update(batch, rows, cols, R, gap, nesterov):
    p = Update(batch, rows, cols, R, gap)
    p.call(0.02, 0.5, 0.1, 0.95, nesterov)
    p.check(0.02, 0.5, 0.1, 0.95, nesterov)


def test_update_without_copies_twice():
    p = Update(2, 100, 80, 2, copies=False)
    p.call(0.02, 1.0, 0.0, 0.9, 1)
    p.call(0.02, 1.0, 0.0, 0.9, 1)
    p.check(0.02, 1.0, 0.0, 0.9, 1, times=2)


def test_same_bits_every_time_and_captured():
    rt = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    args = (0.01, 1.0, 0.1, 0.95, 1)
    want = Update(2, 200, 300, 2)
    for _ in range(4):
        want.call(*args)
    capi.check(capi.lib().mi_stream_sync(None))
    p = Update(2, 200, 300, 2)
    stream, graph, exe = vp(), vp(), vp()
    assert rt.hipStreamCreateWithFlags(ctypes.byref(stream), ctypes.c_uint(1)) == 0
    p.call(*args, stream=stream)
    assert rt.hipStreamBeginCapture(stream, ctypes.c_int(1)) == 0
    p.call(*args, stream=stream)
    assert rt.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        assert rt.hipGraphLaunch(exe, stream) == 0
        capi.check(capi.lib().mi_stream_sync(stream))
        Update(1, 64, 90, 1).call(*args)  # other work between the replays
        capi.check(capi.lib().mi_stream_sync(None))
    for a, b in ((p.w, want.w), (p.m, want.m), (p.w16, want.w16), (p.wt16, want.wt16)):
        assert np.array_equal(a.get().view(np.uint8), b.get().view(np.uint8))
    rt.hipGraphExecDestroy(exe)
    rt.hipGraphDestroy(graph)
    rt.hipStreamDestroy(stream)


def test_two_streams_at_once():
    rt = ctypes.CDLL("libamdhip64.so")
    args = (0.01, 1.0, 0.1, 0.95, 1)
    want = []
    for seed in (1, 2):
        p = Update(2, 200, 300, 2, seed=seed)
        for _ in range(4):
            p.call(*args)
        capi.check(capi.lib().mi_stream_sync(None))
        want.append([x.get() for x in (p.w, p.m, p.w16, p.wt16)])
    pair = [Update(2, 200, 300, 2, seed=seed) for seed in (1, 2)]
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        assert rt.hipStreamCreateWithFlags(ctypes.byref(s), ctypes.c_uint(1)) == 0
    for _ in range(4):
        for p, s in zip(pair, streams):
            p.call(*args, stream=s)
    for s in streams:
        capi.check(capi.lib().mi_stream_sync(s))
        rt.hipStreamDestroy(s)
    for p, w in zip(pair, want):
        for x, y in zip((p.w, p.m, p.w16, p.wt16), w):
            assert np.array_equal(x.get().view(np.uint8), y.view(np.uint8))


def test_one_training_step_of_a_classifier_head():
    """The operators as they are used together, on one stream with nothing waited for in between: loss and
    gradients of a linear head per replica, then the update from both replicas' weight gradients, then the loss with the
    updated bf16 copies."""
    R, B, V, K = 2, 150, 384, 256
    lib = capi.lib()
    heads = [Problem(capi.MI_BF16, B, V, K, bias=False, seed=s) for s in range(R)]
    W0 = heads[0].W.astype(np.float32)
    n = V * K
    w, w16, wt16 = Stack(1, V, K, K, n, np.float32, [W0]), Stack(1, V, K, K, n, np.uint16, [bf16_bits(W0)]), Stack(1, K, V, V, n, np.uint16, [bf16_bits(W0.T)])
    m = Stack(1, V, K, K, n, np.float32, [np.zeros_like(W0)])
    grads = Stack(R, V, K, K, n, np.float32)
    dX = [Strided(B, K, K, 0, np.uint16) for _ in range(R)]
    ws = workspace(1, V, K)
    for r, p in enumerate(heads):
        p.W = W0
        capi.check(lib.mi_xent_forward(capi.MI_BF16, B, V, K, p.dX_.ptr, K, w16.ptr, K, None, p.dt_.ptr, p.loss.ptr, p.lse.ptr,
                                       p.ws.ptr, p.nf, None))
        capi.check(lib.mi_xent_backward(capi.MI_BF16, B, V, K, p.dX_.ptr, K, w16.ptr, K, wt16.ptr, V, None, p.dt_.ptr, p.lse.ptr,
                                        p.dd_.ptr, dX[r].ptr, K, capi.MI_F32, grads.ptr + r * n * 4, K, None, p.ws.ptr, p.nw, None))
    capi.check(lib.mi_ortho_update_raw(1, V, K, w.ptr, w16.ptr, wt16.ptr, m.ptr, grads.ptr, n, n, R, 0.02, 0.5, 0.0, 0.95, 1, 5,
                                       ws.ptr, ws.nbytes, None))
    after = [Strided(1, B, B, 0, np.float32) for _ in range(2 * R)]
    for r, p in enumerate(heads):
        capi.check(lib.mi_xent_forward(capi.MI_BF16, B, V, K, p.dX_.ptr, K, w16.ptr, K, None, p.dt_.ptr, after[2 * r].ptr,
                                       after[2 * r + 1].ptr, p.ws.ptr, p.nf, None))
    capi.check(lib.mi_stream_sync(None))
    # gradients from the formula with the weights before the step
    total = np.zeros((V, K))
    for r, p in enumerate(heads):
        p.oracle()
        g = np.exp(p.z - p.lse_ref[:, None])
        rows = np.flatnonzero(p.counts)
        g[rows, p.t[rows]] -= 1.0
        g *= np.where(p.counts, p.d, 0.0)[:, None]
        ref = g.T @ p.X.astype(np.float64)
        got = grads.get()[r]
        assert np.linalg.norm(got - ref) <= 2.0 ** -8 * np.linalg.norm(np.abs(g).T @ np.abs(p.X))
        total += got.astype(np.float64)
        assert np.linalg.norm(widen(dX[r].get()) - g @ W0) <= 2.0 ** -7 * np.linalg.norm(np.abs(g) @ np.abs(W0))
    O = newton_schulz(total + np.float64(np.float32(0.95)) * total)
    W1 = W0 - 0.02 * 0.5 * O
    got = w.get()[0]
    assert np.linalg.norm(got - W1) <= NS * 0.01 * np.linalg.norm(O) + 4 * 2.0 ** -24 * np.linalg.norm(W1)
    assert np.array_equal(w16.get()[0], bf16_bits(got)) and np.array_equal(wt16.get()[0], bf16_bits(got).T)
    for r, p in enumerate(heads):
        p.W = widen(bf16_bits(got))
        p.oracle()
        assert np.all(np.abs(after[2 * r + 1].get()[0] - p.lse_ref) <= p.lse_bound())
        assert np.all(np.abs(after[2 * r].get()[0] - p.loss_ref) <= 2 * p.lse_bound())
