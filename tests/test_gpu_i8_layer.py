"""The norm, the products with an epilogue, the gated product and the feed-forward block on the device, against the definitions in 64
bits (i8_layer_ref).

Sums are exact integers and the float steps up to an activation are stated, so the host repeats their bits; behind an
activation results are held to the bounds derived in i8_layer_ref.  Results that go two ways (in place, on another kernel, with
less workspace, replayed) are equal bit by bit.
"""
import ctypes

import numpy as np
import pytest

import i8_layer_ref as lref
import i8_ref as ref
import i8_shapes as shapes
import test_gpu_i8 as base
from oxidize_amd import _lib, int8
from oxidize_amd import matvec as mv

pytestmark = pytest.mark.gpu
F32, F16, BF16 = int8.F32, int8.F16, int8.BF16
KINDS = pytest.mark.parametrize("kind", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
ACTS = pytest.mark.parametrize("act", list(lref.ACTS.values()), ids=list(lref.ACTS))
same_bits, up_to_16 = base.same_bits, base.up_to_16


def filled_like(n, stride, kind):
    dt = ref.np_type(kind)
    return np.full((n, stride), np.frombuffer(b"\x5a" * np.dtype(dt).itemsize, dt)[0], dt)


def rows_of(buf, n, stride, width, kind, what="wrote outside its rows"):
    """The rows of a buffer that was filled_like() with one row more; nothing beside them may be written."""
    dt = ref.np_type(kind)
    got, was = buf.download(dt, (n + 1) * stride).reshape(n + 1, stride), filled_like(1, 1, kind)[0, 0]
    assert (got[n] == was).all() and (got[:n, width:] == was).all(), what
    return got[:n, :width]


# ─── norm ───────────────────────────────────────────────────────────────


def run_norm(x, kind, weight=None, eps=1e-5, add=None, pad=0, want_sum=True, want_y=True, in_place=None, stream=None):
    """(codes, scales, sum, y) of encoded rows.  in_place: which of "x" and "add" the sum goes over."""
    n, cols = x.shape
    strides = dict(x=cols + pad, add=cols + 2 * pad, sum=cols + 3 * pad, y=cols + pad)
    q_stride = up_to_16(cols) + 16 * (pad % 3)
    d = dict(x=mv.DeviceBuffer.from_host(ref.padded(np.vstack([x, x[:1]]), strides["x"], 1)), q=mv.DeviceBuffer.from_host(np.full((n + 1, q_stride), 0x55, np.int8)),
             scale=mv.DeviceBuffer(4 * n))
    if add is not None:
        d["add"] = mv.DeviceBuffer.from_host(ref.padded(np.vstack([add, add[:1]]), strides["add"], 1))
    if weight is not None:
        d["weight"] = mv.DeviceBuffer.from_host(weight)
    if want_sum and not in_place:
        d["sum"] = mv.DeviceBuffer.from_host(filled_like(n + 1, strides["sum"], kind))
    if want_y:
        d["y"] = mv.DeviceBuffer.from_host(filled_like(n + 1, strides["y"], kind))
    if in_place:
        d["sum"], strides["sum"] = d[in_place], strides[in_place]

    def ptr(name):
        return d[name].ptr if name in d else None

    norm = int8.Norm(ptr("weight"), eps, ptr("add"), strides["add"], ptr("sum"), strides["sum"], ptr("y"), strides["y"])
    norm.quantize(kind, ptr("x"), strides["x"], n, cols, ptr("q"), q_stride, ptr("scale"), stream)
    mv.sync(stream)
    q = d["q"].download(np.int8, (n + 1) * q_stride).reshape(n + 1, q_stride)
    assert (q[n] == 0x55).all() and (q[:n, up_to_16(cols):] == 0x55).all() and not q[:n, cols:up_to_16(cols)].any()
    total = None
    if in_place:
        total = d["sum"].download(ref.np_type(kind), (n + 1) * strides["sum"]).reshape(n + 1, -1)
        assert same_bits(total[n:, :cols], (x if in_place == "x" else add)[:1]) and (total[:, cols:] == 1).all()
        total = total[:n, :cols]
    elif want_sum:
        total = rows_of(d["sum"], n, strides["sum"], cols, kind)
    return q[:n, :cols], d["scale"].download(np.float32, n), total, rows_of(d["y"], n, strides["y"], cols, kind) if want_y else None


def check_norm(got, x, kind, weight, eps, add):
    """y is its f64 value rounded once to f32 (HALF), and r's sum of squares may be added in another order (n 2^-53, below 2^-36 of
    it): 1.001 HALF.  The scale adds its own rounding, and a code is within half of one and 127 times both of y / scale."""
    q, scale, total, y = got
    s, want = lref.norm(ref.decode(x, kind), weight, eps, None if add is None else ref.decode(add, kind))
    if total is not None:
        assert same_bits(total, ref.encode(s, kind))
    ok = np.isfinite(want).all(axis=1)
    assert np.isnan(scale[~ok]).all() and not q[~ok].any()
    want, q, scale = want[ok], q[ok], scale[ok]
    s64 = np.abs(want).max(axis=1) / 127.0
    small = s64 < 2.0 ** -126 * (1 + 2.0 ** -20)
    assert np.all((np.abs(scale - s64) <= 2.001 * lref.HALF * s64) | small)
    ratio = want / np.where(s64 > 0, s64, 1.0)[:, None]
    assert np.all((np.abs(q - ratio) <= 0.5 + 127 * 4 * lref.HALF) | ((scale == 0) & small)[:, None])
    if y is not None:
        tiny = {F32: 1e-44, F16: 2.0 ** -25, BF16: 1e-40}[kind]
        g = ref.decode(y[ok], kind).astype(np.float64)
        with np.errstate(invalid="ignore"):
            near = np.abs(g - want) <= (1.001 * lref.HALF + (ref.EPS[kind] if kind != F32 else 0.0)) * np.abs(want) + tiny
        assert np.all(near | (np.isinf(g) & (np.abs(want) > 65504)))


NORMS = [(1, 1, 0), (3, 2, 1), (2, 15, 3), (5, 16, 0), (4, 17, 2), (9, 511, 1), (3, 512, 0), (2, 513, 5), (7, 1024, 0), (2, 2047, 1), (2, 2049, 3),
         (1, 4096, 0), (3, 4095, 1), (2, 8192, 0), (2, 8200, 8), (2, 14336, 0), (1, 16384, 0), (2, 16385, 1), (2, 40001, 3), (1, 131071, 0), (1500, 64, 0),
         (70, 1025, 1), (600, 2050, 0), (1100, 4096, 8), (1030, 8190, 0)]


@KINDS
@pytest.mark.parametrize("n,cols,pad", NORMS)
def test_norm(oxh, kind, n, cols, pad):
    rng = np.random.default_rng(n + cols)
    x, add = (base.floats(n, cols, kind, s, 2.0) for s in (1, 2))
    weight = rng.normal(1, 0.3, cols).astype(np.float32)
    check_norm(run_norm(x, kind, weight, 1e-5, add, pad), x, kind, weight, 1e-5, add)


@KINDS
@pytest.mark.parametrize("n,cols", [(3, 300), (2, 5000), (2, 20000)])
@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("add", [False, True])
def test_norm_without_its_options(oxh, kind, n, cols, weight, add):
    x = base.floats(n, cols, kind, 5)
    w = np.random.default_rng(3).normal(1, 0.3, cols).astype(np.float32) if weight else None
    a = base.floats(n, cols, kind, 6) if add else None
    whole = run_norm(x, kind, w, 1e-6, a, 1)
    check_norm(whole, x, kind, w, 1e-6, a)
    bare = run_norm(x, kind, w, 1e-6, a, 0, want_sum=False, want_y=False)
    assert np.array_equal(bare[0], whole[0]) and same_bits(bare[1], whole[1])


@KINDS
@pytest.mark.parametrize("n,cols", [(5, 60), (3, 512), (40, 1000), (3, 4096), (2, 9000), (1, 30000), (2, 131071)])
@pytest.mark.parametrize("over", ["x", "add"])
def test_norm_in_place(oxh, kind, n, cols, over):
    x, add = (base.floats(n, cols, kind, s) for s in (1, 2))
    w = np.random.default_rng(3).normal(1, 0.3, cols).astype(np.float32)
    a, b = run_norm(x, kind, w, 1e-5, add, 2), run_norm(x, kind, w, 1e-5, add, 2, in_place=over)
    for u, v in zip(a, b):
        assert same_bits(u, v) if u.dtype != np.int8 else np.array_equal(u, v)


def test_norm_does_not_depend_on_the_rows_beside_it(oxh):
    for cols in (700, 2000, 4096, 8192, 14336):
        x = base.floats(1100, cols, BF16, 4)
        all_, some = run_norm(x, BF16), run_norm(x[7:9], BF16)
        for u, v in zip(all_, some):
            assert np.array_equal(u[7:9], v)


@KINDS
@pytest.mark.parametrize("cols", [70, 3000, 20001])
def test_norm_rows_without_codes(oxh, kind, cols):
    x = np.random.default_rng(1).normal(size=(12, cols)).astype(np.float32)
    x[1], x[5] = 0.0, np.float32(1e-7) * np.sign(x[5])
    if kind != F16:
        x[6], x[7], x[8], x[9] = x[6] * np.float32(1e-39), x[7] * np.float32(3e37), np.float32(1e-30) * np.sign(x[8]), np.float32(1e38) * np.sign(x[9])
    enc = ref.encode(x, kind)
    inf, nan = (ref.encode(np.array([v], np.float32), kind)[0] if kind != BF16 else np.uint16(b) for v, b in ((np.inf, 0x7F80), (np.nan, 0x7FC0)))
    enc[2, cols - 1], enc[3, 0], enc[4, 33] = nan, inf, inf
    for eps in (1e-5, 0.0):
        got = run_norm(enc, kind, None, eps)
        check_norm(got, enc, kind, None, eps, None)
        assert np.isnan(got[1][2:5]).all() and (got[1][1] == 0 if eps else np.isnan(got[1][1]))
    lone = run_norm(ref.encode(np.eye(3, cols, dtype=np.float32) * 5, kind), kind, None, 0.0)        # one value a row: sqrt(cols), the largest y
    assert np.allclose(lone[1] * 127, np.sqrt(cols), rtol=1e-6) and (lone[0].max(axis=1) == 127).all()


# ─── products with an epilogue ──────────────────────────────────────────


class Case(base.Case):
    def __init__(self, n, rows, cols, seed, act, bias=True, residual=True, kind=F32, **kw):
        super().__init__(n, rows, cols, seed, bias=bias, kind=kind, **kw)
        self.act, self.res_stride = act, rows + n % 5
        self.res = base.floats(n, rows, kind, seed + 9) if residual else None
        self.d["res"] = mv.DeviceBuffer.from_host(ref.padded(self.res, self.res_stride, 1) if residual else np.zeros(4, np.float32))
        self.e = int8.Epilogue(self.d_bias, act, self.d["res"].ptr if residual else None, self.res_stride)

    def want_ex(self, q=None, qs=None):
        """(f64 results, how far) of the epilogue."""
        return lref.epilogue(self.q if q is None else q, self.qs if qs is None else qs, self.w, self.ws, self.bias, self.act,
                             None if self.res is None else ref.decode(self.res, self.kind))

    def check(self, got, q=None, qs=None):
        want, far = self.want_ex(q, qs)
        assert lref.same_or_near(got, self.kind, want, far)
        if not far.any():                               # nothing but stated f32 steps
            v = ref.product(self.q if q is None else q, self.qs if qs is None else qs, self.w, self.ws, self.bias)
            with np.errstate(invalid="ignore"):
                v = np.where(v < 0, np.float32(0), v) if self.act == lref.RELU else v
                v = v if self.res is None else v + ref.decode(self.res, self.kind)
            assert same_bits(np.where(got == 0, 0, got), np.where(ref.encode(v, self.kind) == 0, 0, ref.encode(v, self.kind))) or self.kind != F32

    def matmul_ex(self, out_stride=None, ws=True, stream=None):
        need = self.m.matmul_workspace(self.n) if ws else 0
        buf = mv.DeviceBuffer(max(16, need))
        return self.out(lambda d, s: self.m.matmul_ex(self.d["q"].ptr, self.q_stride, self.d["qs"].ptr, self.n, self.e, self.kind, d, s,
                                                      buf.ptr if ws else None, need, stream), out_stride)

    def linear_ex(self, x, kind, stride=None, stream=None):
        need = self.m.linear_workspace(self.n)
        buf, d_x = mv.DeviceBuffer(max(16, need)), mv.DeviceBuffer.from_host(ref.padded(x, stride or self.cols, 1))
        return self.out(lambda d, s: self.m.linear_ex(kind, d_x.ptr, stride or self.cols, self.n, self.e, self.kind, d, s, buf.ptr, need, stream))


def listed(table):
    return [pytest.param(*size, id="-".join(str(int(v)) for v in (key if isinstance(key, tuple) else (key,))) + ":" + "x".join(map(str, size))) for key, sizes in table.items() for size in sizes]


@pytest.mark.parametrize("n,rows,cols", listed(lref.EX))
def test_matmul_ex_in_every_kernel(oxh, n, rows, cols):
    kind = (BF16, F32, F16)[(n + rows) % 3]
    c = Case(n, rows, cols, n + cols, list(lref.ACTS.values())[(n + cols) % 5], kind=kind, w_stride=up_to_16(cols) + 16, q_stride=up_to_16(cols) + 32)
    c.check(c.matmul_ex(rows + 3))


@ACTS
@KINDS
@pytest.mark.parametrize("n,rows,cols,bias,residual", [(1, 1, 1, True, True), (1, 50, 64, False, True), (5, 130, 1003, True, False), (40, 70, 90, True, True),
                                                       (70, 96, 9000, False, False), (130, 257, 300, True, True), (9, 16, 4230, True, True)])
def test_matmul_ex(oxh, act, kind, n, rows, cols, bias, residual):
    c = Case(n, rows, cols, n + rows, act, bias, residual, kind)
    got = c.matmul_ex(rows + 1)
    c.check(got)
    assert same_bits(c.matmul_ex(ws=False), got)


@KINDS
@pytest.mark.parametrize("n,rows,cols", listed(shapes.LINEAR) + [pytest.param(n, r, c, id="%dx%dx%d" % (n, r, c)) for n, r, c in ((3, 1000, 1025), (17, 1000, 500), (100, 200, 300))])
def test_linear_ex_is_the_quantiser_and_the_product(oxh, kind, n, rows, cols):
    c = Case(n, rows, cols, n + cols, list(lref.ACTS.values())[n % 5], kind=kind)
    x = base.floats(n, cols, kind, 11)
    got = c.linear_ex(x, kind, cols + 3)
    q, qs = ref.quantize(ref.decode(x, kind))
    c.check(got, q, qs)
    c.d["q"].upload(ref.padded(q, c.q_stride))
    c.d["qs"].upload(qs)
    assert same_bits(c.matmul_ex(), got)


@pytest.mark.parametrize("n,rows,cols", [(1, 4096, 4096), (3, 50, 70), (33, 100, 64), (9, 16, 4230), (200, 300, 500), (514, 4000, 132), (130, 3000, 8238)])
def test_no_epilogue_is_the_product(oxh, n, rows, cols):
    c = Case(n, rows, cols, 4, int8.NONE, bias=True, residual=False, kind=BF16)
    want = c.matmul()
    assert same_bits(c.matmul_ex(), want)
    c.e = int8.Epilogue()
    c.d_bias = c.bias = None
    want = c.matmul()
    assert same_bits(c.matmul_ex(), want)
    c.e = None
    assert same_bits(c.matmul_ex(), want)


@KINDS
@pytest.mark.parametrize("n,rows,cols", [(1, 33, 64), (1, 2048, 11008), (16, 200, 4096), (40, 70, 900), (48, 4096, 14336), (300, 131, 500), (825, 8133, 274), (776, 23320, 386)])
def test_residual_in_place(oxh, kind, n, rows, cols):
    c = Case(n, rows, cols, 6, int8.GELU, kind=kind)
    want = c.matmul_ex()
    need = c.m.matmul_workspace(n)
    ws, d = mv.DeviceBuffer(max(16, need)), mv.DeviceBuffer.from_host(ref.padded(c.res, c.res_stride, 1))
    e = int8.Epilogue(c.d_bias, c.act, d.ptr, c.res_stride)
    c.m.matmul_ex(c.d["q"].ptr, c.q_stride, c.d["qs"].ptr, n, e, kind, d.ptr, c.res_stride, ws.ptr, need)
    mv.sync()
    got = d.download(ref.np_type(kind), n * c.res_stride).reshape(n, -1)
    assert same_bits(got[:, :rows], want) and (got[:, rows:] == 1).all()


@ACTS
def test_activations_over_their_whole_range(oxh, act):
    """One token of code 1 against rows of code 1, 0, -1: v is the row's scale times the token's, of any size."""
    v = np.concatenate([np.linspace(-110, 110, 20001), np.geomspace(1e-38, 3e38, 4000), -np.geomspace(1e-38, 3e38, 4000), [0.0, np.nan, np.inf, -np.inf]]).astype(np.float32)
    rows = v.size
    w, q = mv.DeviceBuffer.from_host(ref.padded(np.sign(np.nan_to_num(v, nan=1.0)).astype(np.int8)[:, None], 16)), mv.DeviceBuffer.from_host(ref.padded(np.ones((1, 1), np.int8), 16))
    ws, qs, out = mv.DeviceBuffer.from_host(np.abs(v)), mv.DeviceBuffer.from_host(np.ones(1, np.float32)), mv.DeviceBuffer(4 * rows)
    int8.Matrix(w.ptr, ws.ptr, rows, 1, 16).matmul_ex(q.ptr, 16, qs.ptr, 1, int8.Epilogue(act=act), F32, out.ptr, rows)
    mv.sync()
    want, far = lref.activation(act, v)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)
    got = out.download(np.float32, rows)
    assert lref.same_or_near(got, F32, want, far)
    assert np.isnan(got[-3]) and got[-2] == np.inf


def test_tokens_and_rows_without_numbers_spoil_their_own_results_only(oxh):
    n, rows, cols = 40, 200, 500
    x = np.random.default_rng(2).normal(size=(n, cols)).astype(np.float32)
    x[7, 3], x[20, 499], x[33] = np.nan, np.inf, 0.0
    for act in lref.ACTS.values():
        c = Case(n, rows, cols, 9, act, residual=True)
        c.res[5, 17] = np.nan
        c.d["res"].upload(ref.padded(c.res, c.res_stride, 1))
        got = c.linear_ex(x, F32)
        assert np.isnan(got[[7, 20]]).all() and np.isnan(got[5, 17])
        got[5, 17] = 0
        assert np.isfinite(np.delete(got, [7, 20], axis=0)).all()


# ─── gated products and the block ───────────────────────────────────────


class Gate:
    def __init__(self, n, rows, cols, seed, act=int8.SILU, bias=True, kind=F32, pad=0):
        rng = np.random.default_rng(seed)
        self.n, self.rows, self.cols, self.act, self.kind = n, rows, cols, act, kind
        self.stride, self.q_stride = up_to_16(cols) + 16 * pad, up_to_16(cols) + 16 * (pad % 2)
        self.q, self.qs = base.codes(n, cols, seed + 2), (rng.uniform(0.5, 2, size=n) / 30).astype(np.float32)
        self.mats = []
        for i in range(2):
            self.mats.append((base.codes(rows, cols, seed + 3 + i), (rng.normal(size=rows) / np.sqrt(cols) / 30).astype(np.float32),
                              rng.normal(size=rows).astype(np.float32) if bias else None))
        self.d = dict(q=mv.DeviceBuffer.from_host(ref.padded(self.q, self.q_stride, -99)), qs=mv.DeviceBuffer.from_host(self.qs))
        ptrs = []
        for i, (w, s, b) in enumerate(self.mats):
            for name, a in (("w%d" % i, ref.padded(w, self.stride, 77)), ("s%d" % i, s), ("b%d" % i, b if bias else np.zeros(1, np.float32))):
                self.d[name] = mv.DeviceBuffer.from_host(a)
            ptrs.append((self.d["w%d" % i].ptr, self.d["s%d" % i].ptr, self.d["b%d" % i].ptr if bias else None))
        self.g = int8.Gated(ptrs[0][0], ptrs[0][1], ptrs[1][0], ptrs[1][1], rows, cols, self.stride, act, ptrs[0][2], ptrs[1][2])

    def run(self, out_stride=None, ws=True, stream=None):
        out_stride, need = out_stride or self.rows, self.g.workspace(self.n) if ws else 0
        buf, d = mv.DeviceBuffer(max(16, need)), mv.DeviceBuffer.from_host(filled_like(self.n + 1, out_stride, self.kind))
        self.g.matmul(self.d["q"].ptr, self.q_stride, self.d["qs"].ptr, self.n, self.kind, d.ptr, out_stride, buf.ptr if ws else None, need, stream)
        mv.sync(stream)
        return rows_of(d, self.n, out_stride, self.rows, self.kind)

    def check(self, got):
        want, far = lref.gated(self.q, self.qs, self.mats[0], self.mats[1], self.act)
        assert lref.same_or_near(got, self.kind, want, far)


@pytest.mark.parametrize("n,rows,cols", listed(lref.GATED))
def test_gated_in_every_kernel(oxh, n, rows, cols):
    c = Gate(n, rows, cols, n + cols, list(lref.ACTS.values())[(n + cols) % 5], kind=(BF16, F32, F16)[(n + rows) % 3], pad=n % 3)
    got = c.run(rows + 3)
    c.check(got)


@ACTS
@KINDS
@pytest.mark.parametrize("n,rows,cols,bias,pad", [(1, 1, 1, True, 0), (1, 50, 64, False, 1), (5, 130, 1003, True, 2), (17, 66, 90, True, 0), (40, 70, 90, True, 3),
                                                  (70, 95, 9000, False, 0), (130, 257, 300, True, 1), (9, 16, 4230, True, 0)])
def test_gated(oxh, act, kind, n, rows, cols, bias, pad):
    c = Gate(n, rows, cols, n + rows, act, bias, kind, pad)
    got = c.run(rows + n % 4)
    c.check(got)
    assert same_bits(c.run(ws=False), got)


def test_gated_with_one_bias(oxh):
    c = Gate(20, 100, 300, 3)
    for name, i in (("d_b_gate", 0), ("d_b_up", 1)):
        kept, m = getattr(c.g.desc, name), list(c.mats[i])
        setattr(c.g.desc, name, None)
        c.mats[i] = (m[0], m[1], None)
        c.check(c.run())
        setattr(c.g.desc, name, kept)
        c.mats[i] = tuple(m)


class Block:
    """norm -> feed-forward -> residual, with every buffer its own."""

    def __init__(self, n, hidden, ffn, seed, act=int8.SILU, bias=True, kind=BF16, pad=0, max_tok=None, stream=None):
        rng = np.random.default_rng(seed)
        self.gate = Gate(n, ffn, hidden, seed, act, bias, F32, pad)
        self.n, self.hidden, self.ffn, self.kind, self.stream = n, hidden, ffn, kind, stream
        self.down = (base.codes(hidden, ffn, seed + 7), (rng.normal(size=hidden) / np.sqrt(ffn) / 30).astype(np.float32), rng.normal(size=hidden).astype(np.float32) if bias else None)
        stride = up_to_16(ffn) + 16 * pad
        self.d = dict(w=mv.DeviceBuffer.from_host(ref.padded(self.down[0], stride, 9)), s=mv.DeviceBuffer.from_host(self.down[1]),
                      b=mv.DeviceBuffer.from_host(self.down[2] if bias else np.zeros(1, np.float32)))
        self.m = int8.Matrix(self.d["w"].ptr, self.d["s"].ptr, hidden, ffn, stride)
        self.block = int8.FeedForward(self.gate.g, self.m, max_tok or n)
        self.res = base.floats(n, hidden, kind, seed + 8)
        self.d["res"] = mv.DeviceBuffer.from_host(self.res)
        self.e = int8.Epilogue(self.d["b"].ptr if bias else None, int8.NONE, self.d["res"].ptr, hidden)

    def run(self, out_stride=None):
        stride, c = out_stride or self.hidden, self.gate
        d = mv.DeviceBuffer.from_host(filled_like(self.n + 1, stride, self.kind))
        self.block.forward(c.d["q"].ptr, c.q_stride, c.d["qs"].ptr, self.n, self.e, self.kind, d.ptr, stride, self.stream)
        mv.sync(self.stream)
        return rows_of(d, self.n, stride, self.hidden, self.kind)

    def check(self, got):
        c = self.gate
        want, far = lref.ffn(c.q, c.qs, c.mats[0], c.mats[1], c.act, self.down, ref.decode(self.res, self.kind))
        assert lref.same_or_near(got, self.kind, want, far)


FFN = [(1, 1, 1), (1, 64, 96), (2, 33, 50), (16, 256, 512), (40, 100, 300), (65, 130, 257), (300, 200, 130), (1, 4096, 1000), (3, 1000, 4096), (17, 64, 9000),
       (130, 520, 1030), (1, 300, 20000)]


@KINDS
@pytest.mark.parametrize("n,hidden,ffn", FFN)
def test_ffn(oxh, kind, n, hidden, ffn):
    c = Block(n, hidden, ffn, n + hidden, list(lref.ACTS.values())[(n + ffn) % 5], n % 2 == 0, kind, n % 3)
    got = c.run(hidden + n % 4)
    c.check(got)
    h = c.gate.run()                                            # the two calls one by one
    d_h, need = mv.DeviceBuffer.from_host(h), c.m.linear_workspace(n)
    ws, d = mv.DeviceBuffer(max(16, need)), mv.DeviceBuffer.from_host(filled_like(n + 1, hidden, kind))
    c.m.linear_ex(F32, d_h.ptr, ffn, n, c.e, kind, d.ptr, hidden, ws.ptr, need)
    mv.sync()
    assert same_bits(rows_of(d, n, hidden, hidden, kind), got)


def test_a_workspace_for_more_tokens_serves_fewer(oxh):
    for n in (1, 2, 17, 64, 65, 130, 333):
        few, many = Block(n, 300, 5000, 1), Block(n, 300, 5000, 1, max_tok=700)
        assert same_bits(few.run(), many.run())


def test_a_layer_step_by_step(oxh):
    """A sub-layer as a program runs it, the residual stream brought up to date in place twice: stream += attention; codes = norm(stream);
    stream += block(codes); codes and floats of the next norm."""
    for n in (1, 5, 70):
        hidden, ffn, kind = 256, 700, BF16
        c = Block(n, hidden, ffn, n, kind=kind, bias=False)
        w = np.random.default_rng(1).normal(1, 0.2, hidden).astype(np.float32)
        attention, x = base.floats(n, hidden, kind, 2), base.floats(n, hidden, kind, 3)
        d = dict(x=mv.DeviceBuffer.from_host(x), a=mv.DeviceBuffer.from_host(attention), w=mv.DeviceBuffer.from_host(w), q=mv.DeviceBuffer(n * 256), s=mv.DeviceBuffer(4 * n),
                 y=mv.DeviceBuffer(2 * n * hidden))
        first = int8.Norm(d["w"].ptr, 1e-5, d["a"].ptr, hidden, d["x"].ptr, hidden)
        second = int8.Norm(d["w"].ptr, 1e-5, d_y=d["y"].ptr, y_stride=hidden)
        e = int8.Epilogue(None, int8.NONE, d["x"].ptr, hidden)

        def step():
            first.quantize(kind, d["x"].ptr, hidden, n, hidden, d["q"].ptr, 256, d["s"].ptr)
            c.block.forward(d["q"].ptr, 256, d["s"].ptr, n, e, kind, d["x"].ptr, hidden)
            second.quantize(kind, d["x"].ptr, hidden, n, hidden, d["q"].ptr, 256, d["s"].ptr)

        step()
        mv.sync()
        q, s, total, _ = run_norm(x, kind, w, 1e-5, attention)
        check_norm((q, s, total, None), x, kind, w, 1e-5, attention)
        want, far = lref.ffn(q, s, c.gate.mats[0], c.gate.mats[1], c.gate.act, c.down, ref.decode(total, kind))
        after = d["x"].download(np.uint16, n * hidden).reshape(n, hidden)
        assert lref.same_or_near(after, kind, want, far)
        check_norm((d["q"].download(np.int8, n * 256).reshape(n, 256), d["s"].download(np.float32, n), None, d["y"].download(np.uint16, n * hidden).reshape(n, hidden)),
                   after, kind, w, 1e-5, None)


# ─── streams, graphs, large offsets ─────────────────────────────────────


class Step:
    """Norm, block, gated product and a product with an epilogue of new inputs, in one stream."""

    def __init__(self, n, seed, stream):
        self.n, self.stream, self.seed = n, stream, seed
        self.hidden, self.ffn = 300, 5000
        self.b = Block(n, self.hidden, self.ffn, 1, stream=stream)              # the same matrices for every seed
        self.w = mv.DeviceBuffer.from_host(np.ones(self.hidden, np.float32))
        self.d = {k: mv.DeviceBuffer(v) for k, v in dict(x=2 * n * 300, a=2 * n * 300, sum=2 * n * 300, out=2 * n * 300, h=2 * n * 5000, lin=2 * n * 300, q=n * 304, s=4 * n).items()}
        self.need = (self.b.gate.g.workspace(n), self.b.m.linear_workspace(n))
        self.ws = mv.DeviceBuffer(max(16, *self.need))                          # one for both: calls of one stream
        d = self.d
        self.norm = int8.Norm(self.w.ptr, 1e-5, d["a"].ptr, 300, d["sum"].ptr, 300)
        self.e = int8.Epilogue(None, int8.GELU, d["sum"].ptr, 300)
        self.load(seed)

    def load(self, seed):
        for i, k in enumerate(("x", "a")):
            self.d[k].upload(base.floats(self.n, 300, BF16, seed + i))

    def run(self):
        d, n, st, b = self.d, self.n, self.stream, self.b
        self.norm.quantize(BF16, d["x"].ptr, 300, n, 300, d["q"].ptr, 304, d["s"].ptr, st)
        b.block.forward(d["q"].ptr, 304, d["s"].ptr, n, self.e, BF16, d["out"].ptr, 300, st)
        b.gate.g.matmul(d["q"].ptr, 304, d["s"].ptr, n, BF16, d["h"].ptr, 5000, self.ws.ptr, self.need[0], st)
        b.m.linear_ex(BF16, d["h"].ptr, 5000, n, self.e, BF16, d["lin"].ptr, 300, self.ws.ptr, self.need[1], st)

    def results(self):
        mv.sync(self.stream)
        return [self.d[k].download(np.uint16, self.d[k].nbytes // 2) for k in ("sum", "out", "h", "lin")]


@pytest.mark.parametrize("n", [1, 9, 40, 130])
def test_graphs_on_two_streams_replayed_between_eager_calls(oxh, n):
    streams = []
    for _ in range(2):
        s = ctypes.c_void_p()
        _lib.check(oxh.oxh_stream_create(ctypes.byref(s)))
        streams.append(s)
    steps = [Step(n, 10 * (i + 1), s) for i, s in enumerate(streams)]
    eager = {}
    for seed in (10, 20, 30, 40, 50):
        steps[0].load(seed)
        steps[0].run()
        eager[seed] = steps[0].results()
    graphs = []
    for st in steps:
        with mv.Graph(st.stream) as g:
            st.run()
        graphs.append(g)
    other = Step(n, 70, None)
    for seeds in ((10, 20), (30, 40), (50, 10)):
        for st, seed in zip(steps, seeds):
            st.load(seed)
        for g in graphs:
            g.launch()
        other.run()
        for st, seed in zip(steps, seeds):
            for got, want in zip(st.results(), eager[seed]):
                assert np.array_equal(got, want)
        other.results()
    for g in graphs:
        g.destroy()
    for s in streams:
        oxh.oxh_stream_destroy(s)


@pytest.mark.parametrize("n", [1, 24, 130])
def test_two_graphs_of_one_stream_share_workspaces(oxh, n):
    stream = ctypes.c_void_p()
    _lib.check(oxh.oxh_stream_create(ctypes.byref(stream)))
    steps = [Step(n, seed, stream) for seed in (10, 20)]
    want = []
    for st in steps:
        st.run()
        want.append(st.results())
    steps[1].ws, steps[1].b.block.workspace = steps[0].ws, steps[0].b.block.workspace
    graphs = []
    for st in steps:
        with mv.Graph(stream) as g:
            st.run()
        graphs.append(g)
    for _ in range(3):
        for g in graphs + graphs[::-1]:
            g.launch()
        for st, w in zip(steps, want):
            assert all(np.array_equal(a, b) for a, b in zip(st.results(), w))
        steps[0].run()                                  # eager work in the same workspaces between the replays
    for g in graphs:
        g.destroy()
    mv.sync(stream)
    oxh.oxh_stream_destroy(stream)


def test_rows_residual_and_results_of_more_than_4_gib(oxh):
    """300000 tokens whose rows lie 16 KB apart: the last ones are far behind 4 GiB in x, add, sum, residual and results."""
    n, cols, stride, last = 300000, 33, 4096, 200
    x, add, total = (base.filled(oxh, 4 * n * stride, b) for b in (0x3F, 0x3E, 0x11))
    tail = [base.floats(last, cols, F32, s) for s in (1, 2)]
    for d, t in ((x, tail[0]), (add, tail[1])):
        d.upload(ref.padded(t, stride, 7), 4 * (n - last) * stride)
    q, s = mv.DeviceBuffer(n * 48), mv.DeviceBuffer(4 * n)
    int8.Norm(None, 1e-5, add.ptr, stride, total.ptr, stride, x.ptr, stride).quantize(F32, x.ptr, stride, n, cols, q.ptr, 48, s.ptr)
    mv.sync()
    got = total.download(np.float32, last * stride, 4 * (n - last) * stride).reshape(last, stride)
    y = x.download(np.float32, last * stride, 4 * (n - last) * stride).reshape(last, stride)
    codes = q.download(np.int8, last * 48, (n - last) * 48).reshape(last, 48)[:, :cols]
    scales = s.download(np.float32, last, 4 * (n - last))
    check_norm((codes, scales, got[:, :cols], y[:, :cols]), tail[0], F32, None, 1e-5, tail[1])
    assert (got[:, cols:].view(np.uint32) == 0x11111111).all() and (y[:, cols:] == 7).all()
    c = Case(last, 20, cols, 8, int8.NONE, kind=F32)
    need = c.m.matmul_workspace(n)
    ws = mv.DeviceBuffer(max(16, need))
    res = total.download(np.float32, last * stride, 4 * (n - last) * stride).reshape(last, stride)[:, :20]
    c.m.matmul_ex(q.ptr, 48, s.ptr, n, int8.Epilogue(c.d_bias, int8.NONE, total.ptr, stride), F32, total.ptr, stride, ws.ptr, need)
    mv.sync()
    got = total.download(np.float32, last * stride, 4 * (n - last) * stride).reshape(last, stride)
    assert same_bits(got[:, :20], ref.product(codes, scales, c.w, c.ws, c.bias) + res) and (got[:, 33:].view(np.uint32) == 0x11111111).all()


def test_matrices_of_more_than_4_gib(oxh):
    rows, cols, stride, last, n = 1100000, 70, 4096, 130, 3
    bufs, tails = [], []
    for i in range(2):
        w = base.filled(oxh, rows * stride, 1)
        tails.append(base.codes(last, cols, 5 + i))
        w.upload(ref.padded(tails[i], stride, 3), (rows - last) * stride)
        bufs.append(w)
    s, q, qs = np.full(rows, 0.01, np.float32), base.codes(n, cols, 9), np.arange(1, n + 1, dtype=np.float32) / 50
    d_s, d_q, d_qs, out = mv.DeviceBuffer.from_host(s), mv.DeviceBuffer.from_host(ref.padded(q, 80, 9)), mv.DeviceBuffer.from_host(qs), mv.DeviceBuffer(4 * n * rows)
    int8.Gated(bufs[0].ptr, d_s.ptr, bufs[1].ptr, d_s.ptr, rows, cols, stride, int8.SILU).matmul(d_q.ptr, 80, d_qs.ptr, n, F32, out.ptr, rows)
    mv.sync()
    mats = [(np.concatenate([np.ones((1, cols), np.int8), t]), s[:last + 1], None) for t in tails]
    want, far = lref.gated(q, qs, mats[0], mats[1], int8.SILU)
    for t in range(n):
        got = out.download(np.float32, rows, 4 * t * rows)
        assert lref.same_or_near(got[rows - last:], F32, want[t, 1:], far[t, 1:])
        assert (got[:rows - last] == got[0]).all() and lref.same_or_near(got[:1], F32, want[t, :1], far[t, :1])


# ─── calls that the documentation allows and the rest does not make ─────


@KINDS
@pytest.mark.parametrize("n,rows,cols", [(1, 100, 600), (7, 97, 333), (40, 131, 500), (130, 259, 700), (16, 130, 9000)])
def test_pointers_aligned_to_their_elements_only(oxh, kind, n, rows, cols):
    """Everything but codes lies one element behind a 16-byte border."""
    e_ = ref.np_type(kind)().itemsize
    c = Case(n, rows, cols, 3, int8.SILU, kind=kind)
    want = c.matmul_ex()

    def shifted(a, by):
        d = mv.DeviceBuffer(a.nbytes + by)
        d.upload(np.ascontiguousarray(a), by)
        return d

    ws, bias, qs, res = shifted(c.ws, 4), shifted(c.bias, 4), shifted(c.qs, 4), shifted(ref.padded(c.res, c.res_stride, 1), e_)
    out = mv.DeviceBuffer(n * (rows + 1) * e_ + e_)
    m = int8.Matrix(c.d["w"].ptr, ws.ptr + 4, rows, cols, c.m.desc.stride)
    e = int8.Epilogue(bias.ptr + 4, c.act, res.ptr + e_, c.res_stride)
    need = m.matmul_workspace(n)
    buf = mv.DeviceBuffer(max(16, need))
    m.matmul_ex(c.d["q"].ptr, c.q_stride, qs.ptr + 4, n, e, kind, out.ptr + e_, rows + 1, buf.ptr, need)
    mv.sync()
    got = out.download(ref.np_type(kind), n * (rows + 1), e_).reshape(n, rows + 1)[:, :rows]
    assert same_bits(got, want)
    x, add = (base.floats(n, cols, kind, i) for i in (1, 2))
    w = np.random.default_rng(3).normal(1, 0.3, cols).astype(np.float32)
    d_x, d_a, d_w = shifted(x, e_), shifted(add, e_), shifted(w, 4)
    total, y = mv.DeviceBuffer(n * cols * e_ + e_), mv.DeviceBuffer(n * cols * e_ + e_)
    q, s = mv.DeviceBuffer(n * up_to_16(cols)), mv.DeviceBuffer(4 * n + 4)
    int8.Norm(d_w.ptr + 4, 1e-5, d_a.ptr + e_, cols, total.ptr + e_, cols, y.ptr + e_, cols).quantize(kind, d_x.ptr + e_, cols, n, cols, q.ptr, up_to_16(cols), s.ptr + 4)
    mv.sync()
    dt = ref.np_type(kind)
    check_norm((q.download(np.int8, n * up_to_16(cols)).reshape(n, -1)[:, :cols], s.download(np.float32, n, 4), total.download(dt, n * cols, e_).reshape(n, cols),
                y.download(dt, n * cols, e_).reshape(n, cols)), x, kind, w, 1e-5, add)


@pytest.mark.parametrize("cols", [300, 4096, 20000])
def test_norm_over_both_inputs_at_once(oxh, cols):
    n, kind = 5, BF16
    x, add = (base.floats(n, cols, kind, i) for i in (1, 2))
    want = run_norm(x, kind, None, 1e-5, add)
    d_x, d_a, q, s = mv.DeviceBuffer.from_host(x), mv.DeviceBuffer.from_host(add), mv.DeviceBuffer(n * up_to_16(cols)), mv.DeviceBuffer(4 * n)
    int8.Norm(None, 1e-5, d_a.ptr, cols, d_a.ptr, cols, d_x.ptr, cols).quantize(kind, d_x.ptr, cols, n, cols, q.ptr, up_to_16(cols), s.ptr)
    mv.sync()
    assert same_bits(d_a.download(np.uint16, n * cols).reshape(n, cols), want[2]) and same_bits(d_x.download(np.uint16, n * cols).reshape(n, cols), want[3])
    assert np.array_equal(q.download(np.int8, n * up_to_16(cols)).reshape(n, -1)[:, :cols], want[0])


def test_x_added_to_itself(oxh):
    x = base.floats(3, 700, F32, 4)
    d, q, s = mv.DeviceBuffer.from_host(x), mv.DeviceBuffer(3 * 704), mv.DeviceBuffer(12)
    int8.Norm(None, 1e-5, d.ptr, 700, d.ptr, 700).quantize(F32, d.ptr, 700, 3, 700, q.ptr, 704, s.ptr)
    mv.sync()
    assert same_bits(d.download(np.float32, 3 * 700).reshape(3, 700), x + x)


@pytest.mark.parametrize("rows,cols", [(20, 40), (70, 5000)])
def test_more_tokens_than_a_grid_has_rows(oxh, rows, cols):
    """70000 tokens: beyond what the join of parts could take, so the columns stay together."""
    n = 70000
    c = Gate(n, rows, cols, 5, kind=BF16)
    got = c.run()
    some = np.r_[0:5, 65530:65540, n - 5:n]
    want, far = lref.gated(c.q[some], c.qs[some], c.mats[0], c.mats[1], c.act)
    assert lref.same_or_near(got[some], BF16, want, far)
    e = Case(n, rows, cols, 6, int8.GELU, kind=F16)
    got = e.matmul_ex()
    want, far = lref.epilogue(e.q[some], e.qs[some], e.w, e.ws, e.bias, e.act, ref.decode(e.res[some], F16))
    assert lref.same_or_near(got[some], F16, want, far)


def test_two_threads_at_once(oxh):
    """Calls from two host threads, each on a stream and buffers of its own."""
    import threading
    streams = []
    for _ in range(2):
        s = ctypes.c_void_p()
        _lib.check(oxh.oxh_stream_create(ctypes.byref(s)))
        streams.append(s)
    steps = [Step(40, 10 * (i + 1), s) for i, s in enumerate(streams)]
    want = []
    for st in steps:
        st.run()
        want.append(st.results())
    got, wrong = [None, None], []

    def work(i):
        try:
            for _ in range(20):
                steps[i].run()
            got[i] = steps[i].results()
        except Exception as e:                          # shown by the assertion below
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for g, w in zip(got, want):
        assert all(np.array_equal(a, b) for a, b in zip(g, w))
    for s in streams:
        oxh.oxh_stream_destroy(s)


def test_ffn_in_place_at_every_few_tokens(oxh):
    for n in (1, 2, 5, 17, 33, 65, 200):
        c = Block(n, 520, 700, n, kind=F16)
        want = c.run()
        c.e = int8.Epilogue(c.d["b"].ptr, int8.NONE, c.d["res"].ptr, c.hidden)
        g = c.gate
        c.block.forward(g.d["q"].ptr, g.q_stride, g.d["qs"].ptr, n, c.e, F16, c.d["res"].ptr, c.hidden)
        mv.sync()
        assert same_bits(c.d["res"].download(np.float16, n * c.hidden).reshape(n, -1), want)
