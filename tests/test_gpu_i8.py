"""int8 rows with a scale per row on the device, against the definitions in 64 bits (i8_ref).

Codes and scales of the quantiser are exact.  A product is an exact integer followed by stated f32 steps, which the host
repeats: equal bits, in f32 and after the one rounding to f16 or bf16.  The expert layer is held to a bound that is
derived in i8_ref.experts: f32 steps, and codes of h next to a half.
"""
import ctypes

import numpy as np
import pytest

import i8_ref as ref
from oxidize_amd import _lib, int8, synth
from oxidize_amd import matvec as mv

pytestmark = pytest.mark.gpu
F32, F16, BF16 = int8.F32, int8.F16, int8.BF16
KINDS = pytest.mark.parametrize("kind", [F32, F16, BF16], ids=["f32", "f16", "bf16"])


def floats(n, cols, kind, seed, spread=1.0):
    x = np.random.default_rng(seed).normal(size=(n, cols)).astype(np.float32) * np.float32(spread)
    return ref.encode(x, kind)


def codes(rows, cols, seed):
    return np.random.default_rng(seed).integers(-128, 128, size=(rows, cols)).astype(np.int8)


def up_to_16(cols):
    return (cols + 15) // 16 * 16


def run_quantize(x, kind, stride=None, q_stride=None, up=None):
    """(codes with their padding, scales) of encoded rows; the rest of the output rows must stay as it was."""
    n, cols = x.shape
    stride, q_stride = stride or cols, q_stride or up_to_16(cols) + 16
    bufs = [mv.DeviceBuffer.from_host(ref.padded(a, stride, 1)) for a in ((x,) if up is None else (x, up))]
    d_q, d_s = mv.DeviceBuffer.from_host(np.full((n + 1, q_stride), 0x55, np.int8)), mv.DeviceBuffer(4 * n)
    int8.quantize(kind, bufs[0].ptr, stride, n, cols, d_q.ptr, q_stride, d_s.ptr, None if up is None else bufs[1].ptr)
    mv.sync()
    q = d_q.download(np.int8, (n + 1) * q_stride).reshape(n + 1, q_stride)
    assert (q[n] == 0x55).all() and (q[:n, up_to_16(cols):] == 0x55).all(), "wrote outside its rows"
    assert not q[:n, cols:up_to_16(cols)].any()
    return q[:n, :cols], d_s.download(np.float32, n)


def same_scale(a, b):
    return np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)])


@KINDS
@pytest.mark.parametrize("n,cols,stride", [(1, 1, 1), (3, 2, 7), (2, 15, 15), (5, 16, 17), (4, 17, 32), (9, 255, 255), (1, 4096, 4096),
                                           (300, 100, 103), (2, 8191, 8200), (3, 14336, 14336), (2, 16384, 16384), (2, 16385, 16390),
                                           (2, 40001, 40001), (1, 131071, 131071), (2000, 64, 64), (70, 1024, 1025), (513, 2050, 2050), (1100, 2049, 2051),
                                           (1024, 8192, 8192)])
def test_quantize(oxh, kind, n, cols, stride):
    x = floats(n, cols, kind, n * 31 + cols)
    q, s = run_quantize(x, kind, stride)
    want_q, want_s = ref.quantize(ref.decode(x, kind))
    assert np.array_equal(s, want_s)
    assert np.array_equal(q, want_q)


def test_quantize_next_to_halves(oxh):
    """Rows whose quotients lie on halves, or one unit in the last place beside them, for scales of many mantissas."""
    rng = np.random.default_rng(5)
    rows = []
    for i in range(400):
        top = np.float32(127.0 if i == 0 else 2.0 ** rng.integers(-100, 100) * rng.uniform(1, 2))
        s = np.float32(float(top) / 127.0)
        v = (np.arange(-126, 126, dtype=np.float64) + 0.5) * float(s)
        v = v.astype(np.float32)
        rows.append(np.concatenate([[top], v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(-np.inf))]))
    x = np.array(rows, np.float32)
    q, s = run_quantize(x, F32)
    want_q, want_s = ref.quantize(x)
    assert np.array_equal(s, want_s) and np.array_equal(q, want_q)


@KINDS
def test_quantize_rows_without_codes(oxh, kind):
    x = np.random.default_rng(1).normal(size=(10, 70)).astype(np.float32)
    x[1], x[2, 69], x[3, 0], x[4, 33] = 0.0, np.nan, np.inf, -np.inf
    x[5] = np.float32(1e-7) * np.sign(x[5])
    if kind == F32:
        x[6], x[7], x[8] = x[6] * np.float32(1e-39), x[7] * np.float32(3e37), np.float32(1.5e-36) * np.sign(x[8])
    enc = ref.encode(np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0), kind)
    inf, nan = (ref.encode(np.array([v], np.float32), kind)[0] if kind != BF16 else np.uint16(b) for v, b in
                ((np.inf, 0x7F80), (np.nan, 0x7FC0)))
    enc[2, 69], enc[3, 0], enc[4, 33] = nan, inf, inf
    q, s = run_quantize(enc, kind)
    want_q, want_s = ref.quantize(ref.decode(enc, kind))
    assert same_scale(s, want_s) and np.array_equal(q, want_q)
    assert np.isnan(s[2:5]).all() and s[1] == 0


@KINDS
@pytest.mark.parametrize("n,cols,stride", [(1, 1, 1), (3, 100, 101), (40, 4096, 4096), (2, 20000, 20000), (1030, 2500, 2501)])
def test_quantize_swiglu(oxh, kind, n, cols, stride):
    """v = silu(x) * up in f32 is within 12 * 2^-24 of itself (an exponential of two units in the last place whose argument is
    exact, a sum, a quotient, a product), so the scale within 13 and a code within half of one and 127 * 25 * 2^-24 of v / scale."""
    x, up = floats(n, cols, kind, 3, 4.0), floats(n, cols, kind, 4)
    q, s = run_quantize(x, kind, stride, up=up)
    v = ref.silu(ref.decode(x, kind).astype(np.float64)) * ref.decode(up, kind).astype(np.float64)
    want = np.abs(v).max(axis=1) / 127.0
    assert np.all(np.abs(s - want) <= 13 * 2.0 ** -24 * want)
    assert np.all(np.abs(q - v / want[:, None]) <= 0.5 + 127 * 25 * 2.0 ** -24)


# ─── products ───────────────────────────────────────────────────────────


class Case:
    def __init__(self, n, rows, cols, seed, w_stride=None, q_stride=None, bias=False, kind=F32):
        rng = np.random.default_rng(seed)
        self.n, self.rows, self.cols, self.kind = n, rows, cols, kind
        self.w, self.q = codes(rows, cols, seed + 1), codes(n, cols, seed + 2)
        self.ws = (rng.normal(size=rows) / np.sqrt(cols) / 30).astype(np.float32)
        self.qs = (rng.uniform(0.5, 2, size=n) / 30).astype(np.float32)
        self.bias = rng.normal(size=rows).astype(np.float32) if bias else None
        w_stride, self.q_stride = w_stride or up_to_16(cols), q_stride or up_to_16(cols)
        # what lies behind a row's columns must not matter
        self.d = {k: mv.DeviceBuffer.from_host(a) for k, a in
                  dict(w=ref.padded(self.w, w_stride, 77), q=ref.padded(self.q, self.q_stride, -99), ws=self.ws, qs=self.qs,
                       bias=self.bias if bias else np.zeros(1, np.float32)).items()}
        self.m = int8.Matrix(self.d["w"].ptr, self.d["ws"].ptr, rows, cols, w_stride)
        self.d_bias = self.d["bias"].ptr if bias else None

    def want(self, q=None, qs=None):
        return ref.encode(ref.product(self.q if q is None else q, self.qs if qs is None else qs, self.w, self.ws, self.bias), self.kind)

    def out(self, call, out_stride=None):
        """`call(d_out, out_stride)`; nothing between the rows may be written."""
        out_stride = out_stride or self.rows
        dt = ref.np_type(self.kind)
        fill = np.frombuffer(b"\x5a" * np.dtype(dt).itemsize, dt)[0]
        d = mv.DeviceBuffer.from_host(np.full((self.n + 1, out_stride), fill, dt))
        call(d.ptr, out_stride)
        mv.sync()
        got = d.download(dt, (self.n + 1) * out_stride).reshape(self.n + 1, out_stride)
        assert (got[self.n] == fill).all() and (got[:self.n, self.rows:] == fill).all(), "wrote outside its rows"
        return got[:self.n, :self.rows]

    def matmul(self, out_stride=None, ws=True, stream=None):
        need = self.m.matmul_workspace(self.n) if ws else 0
        buf = mv.DeviceBuffer(max(16, need))
        return self.out(lambda d, s: self.m.matmul(self.d["q"].ptr, self.q_stride, self.d["qs"].ptr, self.n, self.kind, d, s, self.d_bias,
                                                   buf.ptr if ws else None, need, stream), out_stride)


def same_bits(a, b):
    u = {4: np.uint32, 2: np.uint16}[a.dtype.itemsize]
    return np.array_equal(np.ascontiguousarray(a).view(u), np.ascontiguousarray(b).view(u))


SIZES = [(1, 1, 1), (1, 16, 16), (2, 17, 64), (3, 5, 100), (16, 64, 65), (17, 100, 128), (1, 4096, 4096), (5, 1000, 1003), (33, 130, 2049),
         (64, 256, 256), (65, 257, 300), (128, 128, 128), (129, 384, 1024), (257, 513, 777), (300, 1024, 1000), (1, 33, 131071),
         (70, 96, 20000), (48, 512, 14336), (1000, 64, 64), (2, 3001, 16), (512, 2048, 512), (700, 1500, 640), (9, 40000, 48)]


@pytest.mark.parametrize("n,rows,cols", SIZES)
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_matmul(oxh, n, rows, cols, bias):
    c = Case(n, rows, cols, n + rows + cols, bias=bias)
    want = c.want()
    assert same_bits(c.matmul(), want)
    assert same_bits(c.matmul(ws=False), want)


@KINDS
@pytest.mark.parametrize("n,rows,cols,w_pad,q_pad,o_pad", [(1, 100, 200, 16, 32, 1), (40, 70, 90, 48, 0, 3), (200, 300, 500, 16, 16, 5),
                                                           (6, 4096, 1024, 0, 64, 8), (333, 512, 1040, 0, 0, 0),
                                                           (1500, 1025, 130, 16, 16, 7)])
def test_matmul_types_and_strides(oxh, kind, n, rows, cols, w_pad, q_pad, o_pad):
    c = Case(n, rows, cols, 7, up_to_16(cols) + w_pad, up_to_16(cols) + q_pad, bias=True, kind=kind)
    assert same_bits(c.matmul(rows + o_pad), c.want())


def test_matmul_of_the_largest_sums(oxh):
    """-128 * -128 over the widest row: the int32 sum reaches 2147467264."""
    cols = int8.MAX_COLS
    c = Case(2, 3, cols, 1)
    c.q[:], c.w[:] = -128, -128
    c.w[1] = 127
    c.d["q"].upload(ref.padded(c.q, c.q_stride))
    c.d["w"].upload(ref.padded(c.w, up_to_16(cols)))
    assert same_bits(c.matmul(), c.want())


def test_a_token_without_codes_spoils_its_own_row_only(oxh):
    n, rows, cols = 40, 200, 500
    x = np.random.default_rng(2).normal(size=(n, cols)).astype(np.float32)
    x[7, 3], x[20, 499], x[33] = np.nan, np.inf, 0.0
    c = Case(n, rows, cols, 9)
    got = linear(c, x, F32)
    assert np.isnan(got[[7, 20]]).all() and not got[33].any()
    assert np.isfinite(np.delete(got, [7, 20], axis=0)).all()


def linear(c, x, kind, stride=None, stream=None):
    need = c.m.linear_workspace(c.n)
    buf, d_x = mv.DeviceBuffer(max(16, need)), mv.DeviceBuffer.from_host(ref.padded(x, stride or c.cols, 1))
    return c.out(lambda d, s: c.m.linear(kind, d_x.ptr, stride or c.cols, c.n, c.kind, d, s, c.d_bias, buf.ptr, need, stream))


@KINDS
@pytest.mark.parametrize("n,rows,cols,pad", [(1, 1, 1, 0), (1, 4096, 4096, 0), (2, 100, 77, 1), (3, 1000, 1025, 3), (4, 64, 14336, 0),
                                             (5, 513, 16384, 0), (8, 300, 4000, 2), (9, 300, 4000, 0), (1, 50, 20001, 0), (1, 7, 131071, 0),
                                             (16, 64, 256, 0), (17, 1000, 500, 0), (100, 200, 300, 5), (6, 30000, 512, 0)])
def test_linear_is_the_quantiser_and_the_product(oxh, kind, n, rows, cols, pad):
    c = Case(n, rows, cols, n + cols, bias=n % 2 == 0, kind=kind)
    x = floats(n, cols, kind, 11)
    assert same_bits(linear(c, x, kind, cols + pad), c.want(*ref.quantize(ref.decode(x, kind))))


def test_from_packed(oxh):
    """A Q4_K matrix: the int8 form holds oxh_get_rows' values to half a code."""
    rows, cols = 300, 512
    w = synth.weights(13, rows, cols, seed=3, stream=1)
    d_w, d_ids = mv.DeviceBuffer.from_host(w), mv.DeviceBuffer.from_host(np.arange(rows, dtype=np.uint32))
    d_f = mv.DeviceBuffer(4 * rows * cols)
    mv.get_rows(13, d_w.ptr, rows, cols, d_ids.ptr, rows, d_f.ptr, cols)
    mv.sync()
    f = d_f.download(np.float32, rows * cols).reshape(rows, cols)
    m, keep = int8.from_packed(13, d_w.ptr, rows, cols)
    q, s = ref.quantize(f)
    assert np.array_equal(keep[0].download(np.int8, rows * m.desc.stride).reshape(rows, -1)[:, :cols], q)
    assert np.array_equal(keep[1].download(np.float32, rows), s)


WIDE = [(17, 1, 1), (18, 500, 3001), (32, 4096, 4096), (33, 1000, 900), (40, 17, 8192), (47, 16, 16), (48, 2048, 2049), (49, 64, 130),
        (63, 4095, 4090), (64, 300, 8100), (64, 4097, 128)]


@pytest.mark.parametrize("n,rows,cols", WIDE)
@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
def test_matmul_of_17_to_64_tokens_on_small_matrices(oxh, kind, n, rows, cols):
    c = Case(n, rows, cols, n + rows, up_to_16(cols) + 16 * (n % 3), up_to_16(cols) + 16 * (n % 2), bias=n % 2 == 0, kind=kind)
    assert same_bits(c.matmul(rows + n % 4), c.want())
    x = floats(n, cols, kind, 12)
    assert same_bits(linear(c, x, kind), c.want(*ref.quantize(ref.decode(x, kind))))


@pytest.mark.parametrize("n,rows,cols", [(4400, 4400, 144), (4099, 4500, 130), (8193, 257, 64), (191, 4090, 14300),
                                         (333, 28600, 700), (1000, 4090, 1100), (1400, 3000, 1100), (450, 4096, 14300),
                                         (4400, 5001, 1100), (40, 70000, 200), (33, 15000, 900)])
def test_matmul_in_every_tile(oxh, n, rows, cols):
    c = Case(n, rows, cols, 3, bias=True, kind=BF16)
    assert same_bits(c.matmul(), c.want())


def test_a_workspace_for_more_tokens_serves_fewer(oxh):
    big = Case(700, 600, 5000, 1)
    need = big.m.linear_workspace(700)
    buf = mv.DeviceBuffer(need)
    for n in (1, 17, 64, 65, 130, 333, 699):
        c = Case(n, 600, 5000, 1)
        x = floats(n, 5000, F32, n)
        d_x = mv.DeviceBuffer.from_host(x)
        for size in (need, (5000 + 63) // 64 * 64 * n + (4 * n + 15) // 16 * 16):      # the least: codes and scales
            got = c.out(lambda d, s: c.m.linear(F32, d_x.ptr, 5000, n, F32, d, s, None, buf.ptr, size))
            assert same_bits(got, c.want(*ref.quantize(x)))


# ─── offsets that pass 32 bits ──────────────────────────────────────────


def filled(oxh, size, byte):
    d = mv.DeviceBuffer(size)
    _lib.check(oxh.oxh_memset(d.ptr, byte, size, None))
    return d


@pytest.mark.parametrize("n", [3, 40, 150])
def test_a_matrix_of_more_than_4_gib(oxh, n):
    rows, cols, stride, last = 1100000, 70, 4096, 130
    w = filled(oxh, rows * stride, 1)
    tail, q = codes(last, cols, 5), codes(n, cols, 6)
    w.upload(ref.padded(tail, stride, 3), (rows - last) * stride)
    ws, qs = np.full(rows, 0.5, np.float32), np.arange(1, n + 1, dtype=np.float32)
    d_ws, d_q, d_qs = (mv.DeviceBuffer.from_host(a) for a in (ws, ref.padded(q, 80, 9), qs))
    out = mv.DeviceBuffer(2 * n * rows)
    m = int8.Matrix(w.ptr, d_ws.ptr, rows, cols, stride)
    m.matmul(d_q.ptr, 80, d_qs.ptr, n, F16, out.ptr, rows)
    mv.sync()
    for t in (0, n - 1):
        got = out.download(np.uint16, rows, 2 * t * rows)
        whole = np.concatenate([np.ones((1, cols), np.int8), tail])
        want = ref.encode(ref.product(q[t:t + 1], qs[t:t + 1], whole, ws[:last + 1]), F16).view(np.uint16)[0]
        assert (got[:rows - last] == want[0]).all() and np.array_equal(got[rows - last:], want[1:])


def test_tokens_and_results_of_more_than_4_gib(oxh):
    n, rows, cols, x_stride, out_stride, last = 300000, 20, 33, 4096, 4000, 300
    d_x, out = filled(oxh, 4 * n * x_stride, 0x3F), filled(oxh, 4 * n * out_stride, 0x5A)
    c = Case(n, rows, cols, 8)
    x = floats(last, cols, F32, 9)
    d_x.upload(ref.padded(x, x_stride, 7), 4 * (n - last) * x_stride)
    buf = mv.DeviceBuffer(c.m.linear_workspace(n))
    c.m.linear(F32, d_x.ptr, x_stride, n, F32, out.ptr, out_stride, None, buf.ptr, c.m.linear_workspace(n))
    mv.sync()
    first = np.full((1, cols), np.frombuffer(b"\x3f" * 4, np.float32)[0])
    want = c.want(*ref.quantize(np.concatenate([first, x])))
    got = out.download(np.float32, last * out_stride, 4 * (n - last) * out_stride).reshape(last, out_stride)
    assert same_bits(got[:, :rows], want[1:]) and (got[:, rows:].view(np.uint32) == 0x5A5A5A5A).all()
    got = out.download(np.float32, 1000 * out_stride).reshape(1000, out_stride)
    assert same_bits(got[:, :rows], np.repeat(want[:1], 1000, axis=0)) and (got[:, rows:].view(np.uint32) == 0x5A5A5A5A).all()


# ─── experts ────────────────────────────────────────────────────────────


class Layer:
    def __init__(self, e, k, hidden, ffn, max_tok, seed=1, pad=0):
        rng = np.random.default_rng(seed)
        self.e, self.k, self.hidden, self.ffn = e, k, hidden, ffn
        self.host, bufs = {}, []
        for name, rows, cols in (("gate", ffn, hidden), ("up", ffn, hidden), ("down", hidden, ffn)):
            w = rng.integers(-127, 128, size=(e * rows, cols)).astype(np.int8)
            s = (rng.uniform(0.5, 1.5, size=e * rows) / 70 / np.sqrt(cols)).astype(np.float32)
            self.host[name] = (w.reshape(e, rows, cols), s.reshape(e, rows))
            bufs += [mv.DeviceBuffer.from_host(ref.padded(w, up_to_16(cols) + pad, 55)), mv.DeviceBuffer.from_host(s)]
        self.keep = bufs
        self.layer = int8.MoeLayer(*[b.ptr for b in bufs], e, k, hidden, ffn, up_to_16(hidden) + pad, up_to_16(ffn) + pad, max_tok)

    def route(self, ids, weights):
        """A routing on the device made from given choices."""
        counts, offsets, perm, slot = ref.group(ids, self.e)
        d = [mv.DeviceBuffer.from_host(np.ascontiguousarray(a)) for a in
             (ids.astype(np.int32), weights.astype(np.float32), counts.astype(np.uint32), offsets.astype(np.uint32),
              perm.astype(np.uint32), slot.astype(np.uint32))]
        return mv.make_routing(*[b.ptr for b in d]), d

    def run(self, x, kind, routing, out_kind, x_stride=None, out_stride=None, stream=None):
        n = x.shape[0]
        xs, os_ = x_stride or self.hidden, out_stride or self.hidden
        dt = ref.np_type(out_kind)
        fill = np.frombuffer(b"\x5a" * np.dtype(dt).itemsize, dt)[0]
        d_x, d_o = mv.DeviceBuffer.from_host(ref.padded(x, xs, 1)), mv.DeviceBuffer.from_host(np.full((n + 1, os_), fill, dt))
        self.layer.forward(routing, kind, d_x.ptr, n, out_kind, d_o.ptr, xs, os_, stream)
        mv.sync(stream)
        got = d_o.download(dt, (n + 1) * os_).reshape(n + 1, os_)
        assert (got[n] == fill).all() and (got[:n, self.hidden:] == fill).all(), "wrote outside its rows"
        return ref.decode(got[:n, :self.hidden], out_kind).astype(np.float64)

    def check(self, got, x, kind, ids, weights, out_kind):
        want, far = ref.experts(ref.decode(x, kind), ids, weights.astype(np.float64), *[self.host[n] for n in ("gate", "up", "down")])
        tiny = {F32: 1e-40, F16: 2.0 ** -25, BF16: 1e-40}[out_kind]
        assert np.all(np.abs(got - want) <= far + ref.EPS[out_kind] * (np.abs(want) + far) + tiny)


def choices(rng, n, e, k, skew=False):
    """Distinct experts per token; `skew`: most tokens go to the first experts."""
    p = 1.0 / (1.0 + np.arange(e)) ** 2 if skew else np.ones(e)
    ids = np.array([rng.choice(e, size=k, replace=False, p=p / p.sum()) for _ in range(n)])
    w = rng.uniform(0.1, 1.0, size=(n, k)).astype(np.float32)
    return ids, w / w.sum(1, keepdims=True)


@pytest.mark.parametrize("n,e,k,hidden,ffn", [(1, 1, 1, 1, 1), (1, 8, 2, 64, 96), (2, 4, 3, 33, 50), (16, 8, 2, 256, 512), (7, 128, 8, 128, 48),
                                              (100, 3, 2, 200, 130), (300, 16, 4, 128, 160), (65, 512, 16, 96, 32), (64, 2, 1, 1000, 520),
                                              (150, 5, 5, 300, 257), (1, 300, 16, 2048, 768), (3, 2, 2, 4096, 64), (2, 8, 2, 64, 5000), (1030, 4, 1, 2100, 40)])
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16), (F16, F32)], ids=["f32", "bf16", "f16-f32"])
def test_expert_layer(oxh, n, e, k, hidden, ffn, kind, out_kind):
    rng = np.random.default_rng(n + e + hidden)
    lay = Layer(e, k, hidden, ffn, n + 3, pad=16 * (n % 3))
    ids, w = choices(rng, n, e, k)
    routing, keep = lay.route(ids, w)
    x = floats(n, hidden, kind, 5)
    got = lay.run(x, kind, routing, out_kind, hidden + n % 4, hidden + n % 3)
    lay.check(got, x, kind, ids, w, out_kind)


@pytest.mark.parametrize("n,e,k,hidden,ffn", [(1, 8, 2, 64, 96), (3, 32, 5, 200, 1000), (1, 16, 16, 130, 77), (2, 12, 1, 2048, 8000), (5, 64, 8, 2048, 768),
                                              (1, 4, 3, 8190, 2500), (4, 40, 6, 1111, 1408), (1, 1, 1, 1, 1), (16, 8, 1, 48, 4100)])
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16), (F16, F16)], ids=["f32", "bf16", "f16"])
def test_few_pairs_give_the_same_bits_both_ways(oxh, n, e, k, hidden, ffn, kind, out_kind):
    """With the choices' ids the layer may go pair by pair, without them it goes by the sorted pairs."""
    lay = Layer(e, k, hidden, ffn, n, pad=16 * (n % 2))
    ids, w = choices(np.random.default_rng(n + k), n, e, k)
    x = floats(n, hidden, kind, 6)
    routing, keep = lay.route(ids, w)
    got = lay.run(x, kind, routing, out_kind, hidden + n % 3, hidden + n % 2)
    sorted_ = mv.make_routing(0, *[b.ptr for b in keep[1:]])
    assert np.array_equal(got, lay.run(x, kind, sorted_, out_kind))
    lay.check(got, x, kind, ids, w, out_kind)


def test_few_pairs_with_spoiled_tokens_and_ids_out_of_range(oxh):
    n, e, k = 4, 16, 2
    lay = Layer(e, k, 100, 70, n)
    x = floats(n, 100, F32, 1)
    x[1, 3], x[2] = np.nan, 0.0
    ids, w = choices(np.random.default_rng(2), n, e, k)
    w[3] = 0.0
    routing, keep = lay.route(ids, w)
    got = lay.run(x, F32, routing, F32)
    assert np.isnan(got[1]).all() and not got[2].any() and not got[3].any()
    lay.check(got[[0, 2, 3]], x[[0, 2, 3]], F32, ids[[0, 2, 3]], w[[0, 2, 3]], F32)
    keep[0].upload(np.array([-1, 16, 2 ** 31 - 1, -2 ** 31, 5, 999, 0, 15], np.int32))
    lay.run(x, F32, routing, F32)


@pytest.mark.parametrize("n", [40, 200])
def test_expert_layer_with_uneven_loads(oxh, n):
    """Most tokens on the first expert, several without any; and all of them on one."""
    lay = Layer(24, 2, 144, 80, n)
    x = floats(n, 144, F32, 8)
    for ids, w in (choices(np.random.default_rng(n), n, 24, 2, skew=True),
                   (np.tile([[23, 4]], (n, 1)), np.full((n, 2), 0.5, np.float32))):
        routing, keep = lay.route(ids, w)
        lay.check(lay.run(x, F32, routing, F32), x, F32, ids, w, F32)


def test_expert_layer_with_spoiled_and_weightless_tokens(oxh):
    n = 30
    lay = Layer(8, 2, 100, 70, n)
    x = np.random.default_rng(1).normal(size=(n, 100)).astype(np.float32)
    ids, w = choices(np.random.default_rng(2), n, 8, 2)
    w[5], x[11, 4], x[12] = 0.0, np.nan, 0.0
    routing, keep = lay.route(ids, w)
    got = lay.run(x, F32, routing, F32)
    assert np.isnan(got[11]).all() and not got[5].any() and not got[12].any()
    rest = np.delete(np.arange(n), 11)
    lay.check(got[rest], x[rest], F32, ids[rest], w[rest], F32)


def test_the_layer_takes_the_routing_of_moe_route_too(oxh):
    n, e, k = 50, 8, 2
    lay = Layer(e, k, 128, 64, n)
    logits = np.random.default_rng(4).normal(size=(n, e)).astype(np.float32)
    d_l, x = mv.DeviceBuffer.from_host(logits), floats(n, 128, F32, 3)
    d = [mv.DeviceBuffer(4 * max(n * k, e + 1)) for _ in range(6)]
    mv.moe_route(d_l.ptr, n, e, k, True, *[b.ptr for b in d])
    got = lay.run(x, F32, mv.make_routing(*[b.ptr for b in d]), F32)
    ids, w = d[0].download(np.int32, n * k).reshape(n, k), d[1].download(np.float32, n * k).reshape(n, k)
    lay.check(got, x, F32, ids, w, F32)


@pytest.mark.parametrize("n", [3, 60, 300])
def test_a_routing_that_is_none_stays_in_bounds(oxh, n):
    """Offsets that fall, positions behind the last pair: clamped; the layer's next call is not touched by it."""
    e, k = 8, 2
    lay = Layer(e, k, 64, 48, n)
    x, (ids, w) = floats(n, 64, F32, 3), choices(np.random.default_rng(n), n, e, k)
    routing, keep = lay.route(ids, w)
    good = [b.download(np.uint32, b.nbytes // 4) for b in keep]
    for offsets in ([0, n * k] * 4 + [0], [0xFFFFFFFF] * 9, [0, 0, 0xFFFFFFFF, 1, n * k, 0, n * k, 2, n * k], [n * k] * 9):
        keep[3].upload(np.array(offsets, np.uint32))
        keep[4].upload(np.random.default_rng(1).integers(0, 2 ** 32, size=n * k).astype(np.uint32))
        keep[5].upload(np.random.default_rng(2).integers(0, 2 ** 32, size=n * k).astype(np.uint32))
        lay.run(x, F32, routing, F32)
    for b, a in zip(keep, good):
        b.upload(a)
    lay.check(lay.run(x, F32, routing, F32), x, F32, ids, w, F32)


@pytest.mark.parametrize("n", [2, 50, 200])
def test_expert_stacks_of_more_than_4_gib(oxh, n):
    """All tokens go to the last expert of 512; a layer of that expert alone has to give the same bits."""
    e, hidden, ffn, stride = 512, 64, 2100, 4112
    one = Layer(1, 1, hidden, ffn, n)
    stacks = []
    for name, rows in (("gate", ffn), ("up", ffn), ("down", hidden)):
        wide = stride if name != "down" else 2112 + 65536 * 2
        d = filled(oxh, e * rows * wide, 0)
        d.upload(ref.padded(one.host[name][0][0], wide), (e - 1) * rows * wide)
        s = mv.DeviceBuffer.from_host(np.concatenate([np.zeros((e - 1) * rows, np.float32), one.host[name][1][0]]))
        stacks += [d, s]
    all_ = Layer.__new__(Layer)
    all_.e, all_.k, all_.hidden, all_.ffn = e, 1, hidden, ffn
    all_.layer = int8.MoeLayer(*[b.ptr for b in stacks], e, 1, hidden, ffn, stride, 2112 + 65536 * 2, n)
    x = floats(n, hidden, F32, 3)
    got = []
    for lay in (one, all_):
        routing, keep = lay.route(np.full((n, 1), lay.e - 1), np.full((n, 1), 0.75))
        got.append(lay.run(x, F32, routing, F32))
    assert np.array_equal(got[0], got[1]) and np.abs(got[0]).max() > 0


@pytest.mark.parametrize("e,by_ids", [(1, False), (10, False), (100, False), (150, True)], ids=["tiles-128", "tiles-64", "few", "pairs"])
def test_silu_keeps_its_bits_far_from_zero(oxh, e, by_ids):
    """One column of h: its code is 127 or -127 and its scale |h| / 127, so that the output is h itself but for three roundings, and
    h = silu(g) * g for a g that the host knows to the bit.  Units of 2^-24: an exponential of two units in the last place 4, a sum, a quotient and a
    product 3, the scale 1, its way back 1, none of them growing with g."""
    n = 300
    x = np.linspace(-87, 88, n).astype(np.float32)[np.random.default_rng(1).permutation(n)][:, None]
    ones = mv.DeviceBuffer.from_host(np.full((e, 16), 1, np.int8))
    unit = mv.DeviceBuffer.from_host(np.ones(e, np.float32))
    lay = Layer.__new__(Layer)
    lay.e, lay.k, lay.hidden, lay.ffn = e, 1, 1, 1
    lay.layer = int8.MoeLayer(*[b.ptr for b in (ones, unit) * 3], e, 1, 1, 1, 16, 16, n)
    routing, keep = lay.route(np.arange(n)[:, None] % e, np.ones((n, 1)))
    got = lay.run(x, F32, routing if by_ids else mv.make_routing(0, *[b.ptr for b in keep[1:]]), F32)[:, 0]
    q, s = ref.quantize(x)
    g = (q[:, 0].astype(np.float32) * s).astype(np.float64)
    want = ref.silu(g) * g
    assert (np.abs(got - want) / np.abs(want)).max() <= 9.001 * 2.0 ** -24


@pytest.mark.parametrize("n,by_ids", [(2, True), (4, False), (44, False), (4000, False)], ids=["pairs", "few", "tiles-64", "tiles-128"])
def test_codes_of_h_are_the_quantisers(oxh, n, by_ids):
    """Down is the identity and one expert has all weight, so the output is code times scale: those of the quantiser and the products, called one
    after the other."""
    hidden = ffn = 512
    lay = Layer(1, 1, hidden, ffn, n)
    eye, unit = mv.DeviceBuffer.from_host(np.eye(ffn, dtype=np.int8)), mv.DeviceBuffer.from_host(np.ones(ffn, np.float32))
    d_gate, d_up = lay.keep[:2], lay.keep[2:4]
    d_gate[1].upload(lay.host["gate"][1][0] * np.float32(2))             # |g| up to about 10
    lay.layer = int8.MoeLayer(*[b.ptr for b in (*d_gate, *d_up, eye, unit)], 1, 1, hidden, ffn, hidden, ffn, n)
    routing, keep = lay.route(np.zeros((n, 1), np.int64), np.ones((n, 1)))
    x = floats(n, hidden, F32, 12)
    got = lay.run(x, F32, routing if by_ids else mv.make_routing(0, *[b.ptr for b in keep[1:]]), F32)
    d_x, glu = mv.DeviceBuffer.from_host(x), [mv.DeviceBuffer(4 * n * ffn) for _ in range(2)]
    for (w, s), out in zip((d_gate, d_up), glu):
        m = int8.Matrix(w.ptr, s.ptr, ffn, hidden)
        need = m.linear_workspace(n)
        ws = mv.DeviceBuffer(max(16, need))
        m.linear(F32, d_x.ptr, hidden, n, F32, out.ptr, ffn, None, ws.ptr, need)
        mv.sync()
    d_q, d_s = mv.DeviceBuffer(n * ffn), mv.DeviceBuffer(4 * n)
    int8.quantize(F32, glu[0].ptr, ffn, n, ffn, d_q.ptr, ffn, d_s.ptr, glu[1].ptr)
    mv.sync()
    q, s = d_q.download(np.int8, n * ffn).reshape(n, ffn), d_s.download(np.float32, n)
    assert np.array_equal(got.astype(np.float32), q.astype(np.float32) * s[:, None])


# ─── as they are used together ──────────────────────────────────────────


class Block:
    """A router's product, the selection and the expert layer of `n` tokens, in one stream; every buffer is its own."""

    def __init__(self, lay, n, seed, stream=None):
        rng = np.random.default_rng(seed)
        e, k, h = lay.e, lay.k, lay.hidden
        self.lay, self.n, self.stream = lay, n, stream
        self.bias = rng.normal(size=e).astype(np.float32) * np.float32(0.1)
        self.x = rng.normal(size=(n, h)).astype(np.float32)
        w, self.router_scale = codes(e, h, seed), (rng.uniform(0.5, 1, size=e) / 70 / np.sqrt(h)).astype(np.float32)
        self.router_w = w
        self.d = {name: mv.DeviceBuffer.from_host(a) for name, a in dict(x=self.x, w=ref.padded(w, up_to_16(h)), ws=self.router_scale,
                                                                         bias=self.bias).items()}
        self.m = int8.Matrix(self.d["w"].ptr, self.d["ws"].ptr, e, h, up_to_16(h))
        self.router = mv.MoeRouter(e, k, "sigmoid", n_group=4, top_group=2, group_best=2, d_bias=self.d["bias"].ptr, scale=1.5)
        self.lin_ws, self.sel_ws = self.m.linear_workspace(n), self.router.workspace_bytes(n)
        for name, size in dict(logits=4 * n * e, out=4 * n * h, lin=max(16, self.lin_ws), sel=max(16, self.sel_ws), ids=4 * n * k,
                               wts=4 * n * k, counts=4 * e, offsets=4 * e + 4, perm=4 * n * k, slot=4 * n * k).items():
            self.d[name] = mv.DeviceBuffer(size)
        self.routing = mv.make_routing(*[self.d[i].ptr for i in ("ids", "wts", "counts", "offsets", "perm", "slot")])
        self.layer = int8.MoeLayer(*[b.ptr for b in lay.keep], e, k, h, lay.ffn, lay.layer.desc.gate_up_stride,
                                   lay.layer.desc.down_stride, n)

    def launch(self):
        d, n, h = self.d, self.n, self.lay.hidden
        self.m.linear(F32, d["x"].ptr, h, n, F32, d["logits"].ptr, self.lay.e, None, d["lin"].ptr, self.lin_ws, self.stream)
        self.router.select(F32, d["logits"].ptr, self.lay.e, n, self.routing, d["sel"].ptr, self.sel_ws, self.stream)
        self.layer.forward(self.routing, F32, d["x"].ptr, n, F32, d["out"].ptr, stream=self.stream)

    def new_input(self, seed):
        self.x = np.random.default_rng(seed).normal(size=self.x.shape).astype(np.float32)
        self.d["x"].upload(self.x)

    def results(self):
        mv.sync(self.stream)
        return self.d["out"].download(np.float32, self.n * self.lay.hidden).reshape(self.n, -1)

    def check(self):
        got, e, k = self.results(), self.lay.e, self.lay.k
        logits = self.d["logits"].download(np.float32, self.n * e).reshape(self.n, e)
        assert same_bits(logits, ref.product(*ref.quantize(self.x), self.router_w, self.router_scale))
        ids, w = ref.select(logits, k, "sigmoid", 4, 2, 2, self.bias, True, 1.5)
        assert np.array_equal(self.d["ids"].download(np.int32, self.n * k).reshape(self.n, k), ids)
        self.lay.check(got, self.x, F32, ids, w, F32)
        return got


@pytest.mark.parametrize("n", [1, 20, 90, 260])
def test_router_selection_and_experts_together(oxh, n):
    b = Block(Layer(32, 4, 160, 96, 4), n, n)
    b.launch()
    b.check()


@pytest.mark.parametrize("n", [2, 90])
def test_captured_replayed_and_beside_each_other(oxh, n):
    """Two blocks captured on two streams with workspaces of their own, replayed on new inputs while the other runs, eager
    work and synchronisations between; every replay equals the eager result."""
    lay = Layer(32, 4, 160, 96, 4)
    streams = []
    for _ in range(2):
        s = ctypes.c_void_p()
        _lib.check(oxh.oxh_stream_create(ctypes.byref(s)))
        streams.append(s)
    blocks = [Block(lay, n, 10 + i, s) for i, s in enumerate(streams)]
    for b in blocks:
        b.launch()
        b.check()
    graphs = []
    for b in blocks:
        with mv.Graph(b.stream) as g:
            b.launch()
        graphs.append(g)
    for turn in range(4):
        for i, b in enumerate(blocks):
            b.new_input(100 * turn + i)
        for g in graphs:
            g.launch()
        got = [b.check() for b in blocks]
        for b, first in zip(blocks, got):
            b.launch()
            assert same_bits(b.results(), first)
    for g in graphs:
        g.destroy()
    for s in streams:
        oxh.oxh_stream_destroy(s)
