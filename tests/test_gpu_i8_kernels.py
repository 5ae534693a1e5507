"""Every kernel of the int8 products, the quantiser, the expert layer and the selection at sizes that are known to run on it
(i8_shapes), against the definitions in 64 bits."""
import numpy as np
import pytest

import i8_ref as ref
import i8_shapes as shapes
import test_gpu_i8 as base
import test_gpu_select as sel
from oxidize_amd import int8, synth
from oxidize_amd import matvec as mv

pytestmark = pytest.mark.gpu
F32, F16, BF16 = int8.F32, int8.F16, int8.BF16
KINDS = pytest.mark.parametrize("kind", [F32, F16, BF16], ids=["f32", "f16", "bf16"])


def listed(table):
    return [pytest.param(*size, id="-".join(str(int(v)) for v in (key if isinstance(key, tuple) else (key,))) + ":" + "x".join(map(str, size)))
            for key, sizes in table.items() for size in sizes]


@pytest.mark.parametrize("n,rows,cols", listed(shapes.MATMUL))
def test_matmul(oxh, n, rows, cols):
    c = base.Case(n, rows, cols, n + cols, up_to(cols, 16) + 16, up_to(cols, 16) + 32, bias=True, kind=BF16)
    assert base.same_bits(c.matmul(rows + 3), c.want())


def up_to(v, m):
    return (v + m - 1) // m * m


@pytest.mark.parametrize("n,rows,cols", [s for key, sizes in shapes.MATMUL.items() if key[0] != int8.TILES for s in sizes])
@pytest.mark.parametrize("kind", [F32, F16], ids=["f32", "f16"])
def test_few_tokens_in_other_types(oxh, kind, n, rows, cols):
    c = base.Case(n, rows, cols, n + cols, kind=kind)
    assert base.same_bits(c.matmul(), c.want())


@KINDS
@pytest.mark.parametrize("n,rows,cols", listed(shapes.LINEAR))
def test_linear_in_one_launch(oxh, kind, n, rows, cols):
    c = base.Case(n, rows, cols, n + cols, bias=kind == F16, kind=kind)
    x = base.floats(n, cols, kind, 11)
    assert c.m.linear_workspace(n) == 0
    assert base.same_bits(base.linear(c, x, kind, cols + 3), c.want(*ref.quantize(ref.decode(x, kind))))


@pytest.mark.parametrize("n,e,k,hidden,ffn", listed({key: sizes for key, sizes in shapes.EXPERTS.items() if key[0]}))
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16), (F16, F16)], ids=["f32", "bf16", "f16"])
def test_experts_pair_by_pair(oxh, n, e, k, hidden, ffn, kind, out_kind):
    run_experts(n, e, k, hidden, ffn, kind, out_kind, True)


@pytest.mark.parametrize("n,e,k,hidden,ffn", listed({key: sizes for key, sizes in shapes.EXPERTS.items() if not key[0]}))
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16)], ids=["f32", "bf16"])
def test_experts_sorted(oxh, n, e, k, hidden, ffn, kind, out_kind):
    run_experts(n, e, k, hidden, ffn, kind, out_kind, False)


def run_experts(n, e, k, hidden, ffn, kind, out_kind, ids):
    lay = base.Layer(e, k, hidden, ffn, n, pad=16)
    chosen, w = base.choices(np.random.default_rng(n + e), n, e, k)
    routing, keep = lay.route(chosen, w)
    if not ids:
        routing = mv.make_routing(0, *[b.ptr for b in keep[1:]])
    x = base.floats(n, hidden, kind, 5)
    got = lay.run(x, kind, routing, out_kind, hidden + 3, hidden + 1)
    lay.check(got, x, kind, chosen, w, out_kind)


@KINDS
@pytest.mark.parametrize("n,cols", [(3, 512), (3, 1000), (5, 1500), (2, 2048), (1025, 3000), (4, 3000), (2, 17000)])
@pytest.mark.parametrize("glu", [False, True], ids=["plain", "swiglu"])
def test_quantize(oxh, kind, n, cols, glu):
    """64 threads and one or two steps, 256 and one or four, 1024 and two; the bound of silu * up as in test_gpu_i8."""
    x, up = base.floats(n, cols, kind, 3, 4.0), base.floats(n, cols, kind, 4)
    q, s = base.run_quantize(x, kind, cols + 1, up=up if glu else None)
    if not glu:
        want_q, want_s = ref.quantize(ref.decode(x, kind))
        assert np.array_equal(s, want_s) and np.array_equal(q, want_q)
        return
    v = ref.silu(ref.decode(x, kind).astype(np.float64)) * ref.decode(up, kind).astype(np.float64)
    want = np.abs(v).max(axis=1) / 127.0
    assert np.all(np.abs(s - want) <= 13 * 2.0 ** -24 * want)
    assert np.all(np.abs(q - v / want[:, None]) <= 0.5 + 127 * 25 * 2.0 ** -24)


@KINDS
@pytest.mark.parametrize("e", [40, 128, 250, 512])
@pytest.mark.parametrize("n", [9, 70])
def test_select(oxh, kind, e, n):
    """One, two, four and eight experts to a lane, in one launch and in two."""
    logits = ref.encode(np.random.default_rng(e).normal(size=(n, e)).astype(np.float32), kind)
    got = sel.select(logits, kind, 7, e + 3, score="sigmoid", n_group=2, top_group=1, group_best=2)
    sel.check(got, ref.decode(logits, kind), 7, "sigmoid", 2, 1, 2)


def test_calls_of_one_stream_share_a_workspace(oxh):
    """An expert layer under several token counts, pair by pair, by few pairs and by tiles, and products of one matrix, each in one workspace that
    holds the call before: outputs of their own, one wait at the end."""
    lay, rng = base.Layer(20, 2, 200, 300, 700), np.random.default_rng(2)
    m = base.Case(700, 600, 5000, 1)
    need = m.m.linear_workspace(700)
    ws, calls = mv.DeviceBuffer.from_host(np.full(need, 0xFF, np.uint8)), []
    for n in (700, 3, 40, 400, 1, 200, 60):
        ids, w = base.choices(rng, n, 20, 2)
        x, y = base.floats(n, 200, F32, n), base.floats(n, 5000, F32, n)
        calls.append((n, x, ids, w, *lay.route(ids, w), mv.DeviceBuffer.from_host(x), mv.DeviceBuffer(4 * n * 200), y,
                      mv.DeviceBuffer.from_host(y), mv.DeviceBuffer(4 * n * 600)))
    for n, x, ids, w, routing, keep, d_x, d_o, y, d_y, d_p in calls:
        lay.layer.forward(routing, F32, d_x.ptr, n, F32, d_o.ptr)
        m.m.linear(F32, d_y.ptr, 5000, n, F32, d_p.ptr, 600, None, ws.ptr, need)
    mv.sync()
    for n, x, ids, w, routing, keep, d_x, d_o, y, d_y, d_p in calls:
        lay.check(d_o.download(np.float32, n * 200).reshape(n, 200).astype(np.float64), x, F32, ids, w, F32)
        assert base.same_bits(d_p.download(np.float32, n * 600).reshape(n, 600), ref.product(*ref.quantize(y), m.w, m.ws))


def test_from_packed_in_several_blocks_of_rows(oxh):
    """More rows than one expansion takes (65535), the last block a short one."""
    rows, cols = 65535 + 700, 256
    w = synth.weights(13, rows, cols, seed=3, stream=1)
    d_w, d_ids = mv.DeviceBuffer.from_host(w), mv.DeviceBuffer.from_host(np.arange(rows, dtype=np.uint32))
    m, keep = int8.from_packed(13, d_w.ptr, rows, cols)
    q = keep[0].download(np.int8, rows * m.desc.stride).reshape(rows, -1)[:, :cols]
    s = keep[1].download(np.float32, rows)
    d_f = mv.DeviceBuffer(4 * 1000 * cols)
    for r in (0, 65000, rows - 1000):
        mv.get_rows(13, d_w.ptr, rows, cols, d_ids.ptr + 4 * r, 1000, d_f.ptr, cols)
        mv.sync()
        want_q, want_s = ref.quantize(d_f.download(np.float32, 1000 * cols).reshape(1000, cols))
        n = min(1000, rows - r)
        assert np.array_equal(q[r:r + n], want_q[:n]) and np.array_equal(s[r:r + n], want_s[:n])


@pytest.mark.parametrize("qtype", [13, 15, 16, 7], ids=["q4_k", "q5_k", "q6_k", "q8_0"])
def test_what_one_scale_a_row_costs(oxh, qtype):
    """A weight moves by at most half a code, the row's largest magnitude / 254 (and its f32 roundings)."""
    rows, cols = 64, 4096
    w = synth.weights(qtype, rows, cols, seed=5, stream=1)
    d_w, d_ids = mv.DeviceBuffer.from_host(w), mv.DeviceBuffer.from_host(np.arange(rows, dtype=np.uint32))
    d_f = mv.DeviceBuffer(4 * rows * cols)
    mv.get_rows(qtype, d_w.ptr, rows, cols, d_ids.ptr, rows, d_f.ptr, cols)
    m, keep = int8.from_packed(qtype, d_w.ptr, rows, cols)
    f = d_f.download(np.float32, rows * cols).reshape(rows, cols).astype(np.float64)
    q, s = keep[0].download(np.int8, rows * m.desc.stride).reshape(rows, -1)[:, :cols], keep[1].download(np.float32, rows)
    off = np.abs(q * s[:, None].astype(np.float64) - f)
    assert np.all(off <= np.abs(f).max(axis=1, keepdims=True) / 254 * (1 + 256 * 2.0 ** -24))
    print("relative to the rows' rms: %.4f" % np.sqrt((off ** 2).mean() / (f ** 2).mean()))
