"""What stands around the int8 products, on every kernel: results of 16 bits are those of 32 bits rounded once, bit by bit; activations
over their whole range, held to bounds that are counted step by step; residuals that are also the tokens or the results."""
import ctypes
import math

import numpy as np
import pytest

import i8_layer_ref as lref
import i8_ref as ref
import i8_shapes as shapes
import test_gpu_i8 as base
from oxidize_amd import _lib, int8
from oxidize_amd import matvec as mv
from test_gpu_i8_layer import Case, Gate, Step, listed, up_to_16

pytestmark = pytest.mark.gpu
F32, F16, BF16 = int8.F32, int8.F16, int8.BF16
KINDS = pytest.mark.parametrize("kind", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
ACTS = list(lref.ACTS.values())


def rounded_once(got, kind, wide):
    """got in `kind`'s encoding: the bits of the f32 values `wide` rounded to nearest; NaN where those are."""
    nan = np.isnan(wide)
    assert np.isnan(ref.decode(got, kind)[nan]).all()
    return base.same_bits(np.where(nan, 0, got).astype(got.dtype), ref.encode(np.where(nan, np.float32(0), wide), kind))


# ─── bits ───────────────────────────────────────────────────────────────


def stated(c, residual):
    """the f32 results where every step is stated: no activation, or max(v, 0)"""
    v = ref.product(c.q, c.qs, c.w, c.ws, c.bias)
    v = np.where(v < 0, np.float32(0), v) if c.e.desc.act == lref.RELU else v
    return v + residual


@pytest.mark.parametrize("n,rows,cols", listed(lref.EX))
def test_results_of_every_kernel_are_rounded_once(oxh, n, rows, cols):
    c = Case(n, rows, cols, n + cols, int8.NONE, w_stride=up_to_16(cols) + 16)
    acts = [(int8.NONE, lref.RELU)[(n + rows) % 2], (lref.SILU, lref.GELU, lref.GELU_TANH)[(n + cols) % 3]]
    for kind in (F16, BF16):
        res = base.floats(n, rows, kind, 5)
        for act in acts:
            c.e.desc.act = act
            c.kind = kind
            c.d["res"].upload(ref.padded(res, c.res_stride, 1))
            got = c.matmul_ex(rows + 1)
            c.kind = F32
            c.d["res"].upload(ref.padded(ref.decode(res, kind), c.res_stride, 1))
            wide = c.matmul_ex(rows + 1)
            assert rounded_once(got, kind, wide)
            if act in (int8.NONE, lref.RELU) and kind == F16:
                assert base.same_bits(wide, stated(c, ref.decode(res, kind)))


@pytest.mark.parametrize("n,rows,cols", listed(lref.GATED))
def test_gated_results_of_every_kernel_are_rounded_once(oxh, n, rows, cols):
    c = Gate(n, rows, cols, n + cols, pad=1)
    acts = [(int8.NONE, lref.RELU)[(n + rows) % 2], (lref.SILU, lref.GELU, lref.GELU_TANH)[(n + cols) % 3]]
    for act in acts:
        c.g.desc.act = act
        c.kind = F32
        wide = c.run(rows + 1)
        if act in (int8.NONE, lref.RELU):
            g, u = (ref.product(c.q, c.qs, *m) for m in c.mats)
            assert base.same_bits(wide, (np.where(g < 0, np.float32(0), g) if act == lref.RELU else g) * u)
        for kind in (F16, BF16):
            c.kind = kind
            assert rounded_once(c.run(rows + 1), kind, wide)


# ─── activations ────────────────────────────────────────────────────────

_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def bound(act, v):
    """The activation in 64 bits and how far the steps that the kernels take may be from it.

    In units of 2^-24 relative: a rounding is 1, the instructions for 2^x and 1/x are good to a unit in the last place, 2.

    SILU and GELU_TANH, v / (1 + 2^t): the sum 1, the reciprocal 2, the product 1; 2^t counts by its share w = 2^t / (1 + 2^t) only: 2, and
    what t is off times |t| ln 2.  SILU: t rounded once, its factor carried in two numbers: 1.01 |v|.  GELU_TANH: v v, a constant off by a third and one
    by a tenth of a rounding, the sum, the product: 3.4 times 2u = 2 sqrt(2 / pi) (v + 0.044715 v^3).
    GELU, v P with P = 2^(c v v) R(|v|) below 0 and 1 minus that above: the polynomial is fitted to 2.4; its argument 1 / (1 + 0.3 |v|) is off by 3,
    which R takes over 2.66-fold at most (R's condition, largest at 0): 8; Horner's roundings weigh 3.1 together; the products r t and 2^x
    (r t) 2, the exponential 2: 17.5.  c v v: the constant 0.23, two products: 2.23 of v^2 / 2: 1.12 v^2.  Above 0 those weigh
    (1 - P) / P; the subtraction and the product with v 2.

    And lref.LOST, for what the instructions count as 0 below 2^-126."""
    e, _ = lref.activation(act, v)
    x = v.astype(np.float64)
    with np.errstate(all="ignore"):
        if act == lref.SILU:
            d = 4 + (2 + 1.01 * np.abs(x)) / (1 + np.exp(x))
        elif act == lref.GELU_TANH:
            u2 = 2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)
            d = 4 + (2 + 3.4 * np.abs(u2)) / (1 + np.exp(u2))
        elif act == lref.GELU:
            above = 0.5 * _erfc(np.abs(x) / math.sqrt(2.0))
            d = 2 + np.where(x > 0, above / (1 - above), 1.0) * (17.5 + 1.12 * x * x)
        else:
            return e, np.zeros(x.shape)
        return e, np.where(np.abs(e) > 0, d * lref.HALF * np.abs(e), 0.0) + lref.LOST


def values(count, seed):
    """of any size, most of them where an activation bends, and what is no number last"""
    rng = np.random.default_rng(seed)
    some = np.concatenate([rng.uniform(-14, 14, 4 * count), rng.uniform(-110, 110, count), rng.choice([-1, 1], count) * np.exp(rng.uniform(-87, 88, count)),
                           np.zeros(20)]).astype(np.float32)
    v = rng.choice(some, count)
    v[-4:] = np.array([0.0, np.nan, np.inf, -np.inf], np.float32)[-min(4, count):]
    return v


def near(got, act, v):
    want, far = bound(act, v)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)
    return lref.same_or_near(got, F32, want, far)


class Codes:
    """Tokens with one code, 1, in the last column and scale 1 against rows that have the sign of v there, and its size as their scale: every token's
    sums are v."""

    def __init__(self, n, rows, cols):
        self.n, self.rows, self.cols, self.stride, self.v = n, rows, cols, up_to_16(cols), values(rows, n + rows)
        w, up, q = base.codes(rows, cols, 1), base.codes(rows, cols, 2), np.zeros((n, cols), np.int8)
        q[:, -1], up[:, -1], w[:, -1] = 1, 1, np.where(np.isnan(self.v), 1, np.sign(self.v))
        ones = np.ones(max(n, rows), np.float32)
        self.d = {k: mv.DeviceBuffer.from_host(a) for k, a in dict(w=ref.padded(w, self.stride, 7), up=ref.padded(up, self.stride, 9), q=ref.padded(q, self.stride, 5),
                                                                  ws=np.abs(self.v), ones=ones).items()}
        self.out = mv.DeviceBuffer(4 * n * rows)

    def check(self, act, call):
        call(act)
        mv.sync()
        got = self.out.download(np.float32, self.n * self.rows).reshape(self.n, self.rows)
        assert near(got[0], act, self.v)
        for row in got[1:]:
            assert np.array_equal(row, got[0], equal_nan=True)


@pytest.mark.parametrize("n,rows,cols", listed(lref.EX))
def test_activations_over_their_whole_range_on_every_kernel(oxh, n, rows, cols):
    c = Codes(n, rows, cols)
    m = int8.Matrix(c.d["w"].ptr, c.d["ws"].ptr, rows, cols, c.stride)
    need = m.matmul_workspace(n)
    ws = mv.DeviceBuffer(max(16, need))
    for act in ACTS[1:]:
        c.check(act, lambda a: m.matmul_ex(c.d["q"].ptr, c.stride, c.d["ones"].ptr, n, int8.Epilogue(act=a), F32, c.out.ptr, rows, ws.ptr, need))


@pytest.mark.parametrize("n,rows,cols", listed(lref.GATED))
def test_gated_activations_over_their_whole_range_on_every_kernel(oxh, n, rows, cols):
    c = Codes(n, rows, cols)
    for act in ACTS[1:]:
        g = int8.Gated(c.d["w"].ptr, c.d["ws"].ptr, c.d["up"].ptr, c.d["ones"].ptr, rows, cols, c.stride, act)
        need = g.workspace(n)
        ws = mv.DeviceBuffer(max(16, need))
        c.check(act, lambda a: g.matmul(c.d["q"].ptr, c.stride, c.d["ones"].ptr, n, F32, c.out.ptr, rows, ws.ptr, need))


# ─── the same memory twice ──────────────────────────────────────────────


def linear_over(c, kind, x_ptr, res_ptr, res_stride, out_ptr, out_stride):
    need = c.m.linear_workspace(c.n)
    ws = mv.DeviceBuffer(max(16, need))
    e = int8.Epilogue(c.d_bias, c.act, res_ptr, res_stride)
    c.m.linear_ex(kind, x_ptr, c.cols, c.n, e, kind, out_ptr, out_stride, ws.ptr, need)
    mv.sync()


@KINDS
@pytest.mark.parametrize("n,size", [(1, 1), (1, 50), (3, 300), (1, 4096), (1, 5000), (16, 700), (40, 700), (130, 257), (333, 1000)])
def test_tokens_that_are_the_residual(oxh, kind, n, size):
    c, x = Case(n, size, size, n + size, int8.GELU, kind=kind), base.floats(n, size, kind, 3)
    d_x, d_res, out, dt = mv.DeviceBuffer.from_host(x), mv.DeviceBuffer.from_host(x), mv.DeviceBuffer(4 * n * size), ref.np_type(kind)
    linear_over(c, kind, d_x.ptr, d_res.ptr, size, out.ptr, size)
    want = out.download(dt, n * size)
    c.res = x
    c.check(want.reshape(n, size), *ref.quantize(ref.decode(x, kind)))
    linear_over(c, kind, d_x.ptr, d_x.ptr, size, out.ptr, size)
    assert base.same_bits(out.download(dt, n * size), want) and base.same_bits(d_x.download(dt, n * size), x.reshape(-1))


@KINDS
@pytest.mark.parametrize("n,rows,cols", listed(shapes.LINEAR) + [pytest.param(n, r, c, id="%dx%dx%d" % (n, r, c)) for n, r, c in
                                                                 ((16, 300, 500), (17, 300, 500), (8, 4096, 14336), (24, 4096, 14336), (200, 500, 700))])
def test_float_tokens_with_results_over_the_residual(oxh, kind, n, rows, cols):
    c, x, dt = Case(n, rows, cols, n + rows, int8.SILU, kind=kind), base.floats(n, cols, kind, 3), ref.np_type(kind)
    d_x, out, over = mv.DeviceBuffer.from_host(x), mv.DeviceBuffer(4 * n * rows), mv.DeviceBuffer.from_host(ref.padded(c.res, c.res_stride, 1))
    linear_over(c, kind, d_x.ptr, c.d["res"].ptr, c.res_stride, out.ptr, rows)
    linear_over(c, kind, d_x.ptr, over.ptr, c.res_stride, over.ptr, c.res_stride)
    got = over.download(dt, n * c.res_stride).reshape(n, -1)
    assert base.same_bits(got[:, :rows], out.download(dt, n * rows).reshape(n, rows)) and (got[:, rows:] == 1).all()


# ─── eager calls between replays ────────────────────────────────────────


@pytest.mark.parametrize("n", [1, 24, 130])
def test_eager_calls_between_replays_keep_their_results(oxh, n):
    stream = ctypes.c_void_p()
    _lib.check(oxh.oxh_stream_create(ctypes.byref(stream)))
    other, step = Step(n, 70, None), Step(n, 10, stream)
    other.run()
    alone = other.results()
    step.run()
    mv.sync(stream)
    with mv.Graph(stream) as g:
        step.run()
    for _ in range(4):
        g.launch()
        other.run()
        g.launch()
        assert all(np.array_equal(a, b) for a, b in zip(other.results(), alone))
    mv.sync(stream)
    g.destroy()
    oxh.oxh_stream_destroy(stream)
