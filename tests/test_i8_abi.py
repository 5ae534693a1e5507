"""The int8 entry points and the expert selection without a device: struct layout, workspaces, refusals."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import i8_ref as ref
import i8_shapes as shapes
from oxidize_amd import _lib, int8
from oxidize_amd import matvec as mv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20                     # an address no refused call follows


def test_bindings_lay_the_new_structs_out_as_the_header_does(tmp_path):
    structs = {n: getattr(_lib, n) for n in ("OxhMoeRouter", "OxhRouting", "OxhI8Matrix", "OxhMoeI8")}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "oxhip.h"', 'int main(void) {']
    for name, cls in structs.items():
        lines.append('printf("%s size %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f) for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, value = line.split()
        cls = structs[name]
        assert int(value) == (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset), (name, field)


def refused(fn, *args, status=_lib.ERR_ARG, **kw):
    with pytest.raises(_lib.OxhError) as e:
        fn(*args, **kw)
    assert e.value.status == status, e.value
    assert len(str(e.value)) > 30           # says what is wrong


QUANT = dict(x_type=int8.F32, d_x=A, x_stride=64, n_vec=2, cols=64, d_q=A, q_stride=64, d_scale=A)


@pytest.mark.parametrize("change", [dict(x_type=3), dict(d_x=0), dict(d_x=A + 2), dict(x_type=int8.BF16, d_x=A + 1), dict(x_stride=63),
                                    dict(cols=0), dict(d_q=0), dict(d_q=A + 8), dict(q_stride=72), dict(q_stride=48), dict(d_scale=0),
                                    dict(d_up=A + 2), dict(n_vec=(1 << 23) + 1)])
def test_quantize_refuses(change):
    refused(int8.quantize, **{**QUANT, **change})


def test_sizes_that_are_too_wide_or_empty():
    refused(int8.quantize, **{**QUANT, "cols": 131072, "x_stride": 131072, "q_stride": 131072}, status=_lib.ERR_TOO_WIDE)
    m = int8.Matrix(A, A, 8, 131072)
    refused(m.matmul, A, 131072, A, 1, int8.F32, A, 8, status=_lib.ERR_TOO_WIDE)
    int8.quantize(**{**QUANT, "n_vec": 0})          # nothing to do, no device needed
    int8.Matrix(A, A, 0, 64).matmul(A, 64, A, 1, int8.F32, A, 8)
    int8.Matrix(A, A, 8, 64).linear(int8.F32, A, 64, 0, int8.F32, A, 8)


MAT = dict(d_w=A, d_scale=A, rows=8, cols=100, stride=128)
MUL = dict(d_q=A, q_stride=128, d_q_scale=A, n_vec=3, out_type=int8.F32, d_out=A, out_stride=8)


@pytest.mark.parametrize("mat,mul", [(dict(d_w=0), {}), (dict(d_w=A + 4), {}), (dict(stride=120), {}), (dict(stride=96), {}),
                                     (dict(d_scale=0), {}), (dict(cols=0), {}), (dict(rows=(1 << 23) + 1), dict(out_stride=1 << 24)),
                                     ({}, dict(d_q=0)), ({}, dict(d_q=A + 1)), ({}, dict(q_stride=100)), ({}, dict(q_stride=96)),
                                     ({}, dict(d_q_scale=0)), ({}, dict(out_type=7)), ({}, dict(d_out=0)), ({}, dict(d_out=A + 2)),
                                     ({}, dict(out_type=int8.F16, d_out=A + 1)), ({}, dict(out_stride=7)),
                                     ({}, dict(d_ws=A + 4, ws_bytes=64)), ({}, dict(n_vec=(1 << 23) + 1))])
def test_matmul_refuses(mat, mul):
    refused(int8.Matrix(**{**MAT, **mat}).matmul, **{**MUL, **mul})


@pytest.mark.parametrize("change", [dict(d_x=0), dict(x_stride=99), dict(x_type=9), dict(d_out=0), dict(ws_bytes=-1), dict(d_ws=0),
                                    dict(d_ws=A + 8), dict(out_stride=7)])
def test_linear_refuses(change):
    m = int8.Matrix(**MAT)
    need = m.linear_workspace(300)
    assert need > 0
    args = dict(x_type=int8.F32, d_x=A, x_stride=100, n_vec=300, out_type=int8.F32, d_out=A, out_stride=8, d_ws=A, ws_bytes=need)
    if change.get("ws_bytes") == -1:
        change = dict(ws_bytes=need - 1)
    refused(m.linear, **{**args, **change})


ROUTER = dict(n_expert=64, top_k=4)


@pytest.mark.parametrize("change", [dict(n_expert=0), dict(n_expert=513), dict(top_k=0), dict(top_k=17), dict(n_expert=3),
                                    dict(n_group=7, top_group=2), dict(n_group=128, n_expert=512, top_group=2),
                                    dict(n_group=8, top_group=0), dict(n_group=8, top_group=9),
                                    dict(n_group=8, top_group=2, group_best=3), dict(n_group=32, top_group=1)])
def test_routers_refused(change):
    r = mv.MoeRouter(**{**ROUTER, **change})
    refused(r.workspace_bytes, 10)
    refused(r.select, int8.F32, A, 512, 10, mv.make_routing(A, A, A, A, A, A), A, 1 << 20)


def test_select_refuses():
    r, rt = mv.MoeRouter(**ROUTER), mv.make_routing(A, A, A, A, A, A)
    assert r.workspace_bytes(16) == 0
    need = r.workspace_bytes(1000)
    assert 0 < need <= 1000 * 64
    refused(r.workspace_bytes, 65536)
    for args in ((3, A, 64, 10, rt), (0, 0, 64, 10, rt), (0, A + 2, 64, 10, rt), (2, A + 1, 64, 10, rt), (0, A, 63, 10, rt),
                 (0, A, 64, 65536, rt, A, 1 << 30), (0, A, 64, 1000, rt), (0, A, 64, 1000, rt, A, need - 1),
                 (0, A, 64, 1000, rt, A + 8, need)):
        refused(r.select, *args)
    for i in range(6):
        refused(r.select, 0, A, 64, 10, mv.make_routing(*[0 if j == i else A for j in range(6)]))
    bad = mv.MoeRouter(**ROUTER)
    bad.desc.score = 2
    refused(bad.select, 0, A, 64, 10, rt)
    r.select(0, A, 64, 0, rt)                       # no tokens: nothing to do


class Layer(int8.MoeLayer):
    """The descriptor without a workspace of its own, as there is no device to hold one."""

    def __init__(self, **change):
        p = dict(d_w_gate=A, d_w_up=A, d_w_down=A, d_s_gate=A, d_s_up=A, d_s_down=A, gate_up_stride=112, down_stride=48, n_expert=8,
                 top_k=2, hidden=100, ffn=33)
        p.update(change)
        self.desc = _lib.OxhMoeI8(**p)


def test_expert_layers_refused():
    need = ctypes.c_size_t()
    lib, rt = _lib.lib(), mv.make_routing(A, A, A, A, A, A)

    def call(layer, routing=rt, x_type=0, d_x=A, x_stride=100, n=5, out_type=0, d_out=A, out_stride=100, ws=A, bytes_=1 << 30):
        return lib.oxh_moe_ffn_i8(ctypes.byref(layer.desc), ctypes.byref(routing) if routing else None, x_type, d_x, x_stride, n,
                                  out_type, d_out, out_stride, ws, bytes_, None)

    for change in (dict(n_expert=0), dict(n_expert=513), dict(top_k=0), dict(top_k=9), dict(top_k=17, n_expert=64), dict(hidden=0),
                   dict(ffn=0)):
        assert lib.oxh_moe_i8_workspace_bytes(ctypes.byref(Layer(**change).desc), 5, ctypes.byref(need)) == _lib.ERR_ARG
        assert call(Layer(**change)) == _lib.ERR_ARG, change
    assert call(Layer(ffn=131072, down_stride=131072)) == _lib.ERR_TOO_WIDE
    for change in (dict(d_w_gate=0), dict(d_w_up=A + 1), dict(d_w_down=0), dict(d_s_gate=0), dict(d_s_up=0), dict(d_s_down=0),
                   dict(gate_up_stride=100), dict(gate_up_stride=96), dict(down_stride=40), dict(down_stride=32)):
        assert call(Layer(**change)) == _lib.ERR_ARG, change
    assert lib.oxh_moe_i8_workspace_bytes(ctypes.byref(Layer().desc), 5, ctypes.byref(need)) == _lib.OK
    for kw in (dict(x_type=4), dict(d_x=0), dict(d_x=A + 2), dict(x_stride=99), dict(n=0), dict(n=65536), dict(out_type=4), dict(d_out=0),
               dict(out_stride=99), dict(ws=0), dict(ws=A + 16), dict(bytes_=need.value - 1), dict(routing=None)):
        assert call(Layer(), **kw) == _lib.ERR_ARG, kw
    for i in (1, 3, 4, 5):
        assert call(Layer(), routing=mv.make_routing(*[0 if j == i else A for j in range(6)])) == _lib.ERR_ARG


def test_more_results_than_any_memory_holds_are_refused():
    big = int8.Matrix(A, A, 1 << 21, 64, 64)
    refused(big.matmul, A, 64, A, (1 << 16) + 1, int8.F32, A, 1 << 21)
    refused(big.linear, int8.F32, A, 64, (1 << 16) + 1, int8.F32, A, 1 << 21, d_ws=A, ws_bytes=1 << 40)
    need, wide = ctypes.c_size_t(), Layer(n_expert=64, top_k=16, ffn=131071, down_stride=131072)
    assert _lib.lib().oxh_moe_i8_workspace_bytes(ctypes.byref(wide.desc), 16384, ctypes.byref(need)) == _lib.OK
    assert _lib.lib().oxh_moe_i8_workspace_bytes(ctypes.byref(wide.desc), 16385, ctypes.byref(need)) == _lib.ERR_ARG


def test_workspaces_for_more_tokens_serve_fewer():
    for rows, cols in ((8, 100), (4096, 14336), (600, 5000), (128, 131071), (5000, 64)):
        m = int8.Matrix(A, A, rows, cols, (cols + 15) // 16 * 16)
        least = [n * ((cols + 63) // 64 * 64) + (4 * n + 15) // 16 * 16 for n in range(1, 700)]
        assert all(m.linear_workspace(n) >= least[n - 1] for n in range(17, 700))
    need, last = ctypes.c_size_t(), 0
    for n in range(1, 3000):
        layer = Layer(n_expert=512, top_k=8, hidden=64, ffn=32)
        assert _lib.lib().oxh_moe_i8_workspace_bytes(ctypes.byref(layer.desc), n, ctypes.byref(need)) == _lib.OK
        assert need.value >= last
        last = need.value
    sizes = [mv.MoeRouter(384, 8).workspace_bytes(n) for n in range(1, 20000)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_a_valid_call_without_a_device_says_so():
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    refused(int8.quantize, **QUANT, status=_lib.ERR_NO_DEVICE)


# ─── the oracle itself ──────────────────────────────────────────────────


def test_oracle_rounds_quotients_to_nearest_even():
    codes, scale = ref.quantize(np.array([[127.0, 0.5, 1.5, -2.5, 126.5]], np.float32))
    assert scale[0] == 1.0 and codes[0].tolist() == [127, 0, 2, -2, 126]
    codes, scale = ref.quantize(np.array([[0.0, 0.0], [1.0, np.inf], [np.nan, 1.0], [1e-38, 0.0]], np.float32))
    assert not codes.any() and scale[0] == 0 and np.isnan(scale[1:3]).all() and scale[3] == 0


def test_oracle_selects_by_hand_worked_cases():
    ids, w = ref.select(np.array([[1.0, 3.0, 3.0, 2.0]]), 3, "softmax")
    assert ids[0].tolist() == [1, 2, 3] and abs(w[0].sum() - 1) < 1e-15
    # groups {0,1} {2,3}: 0.5 + 0.5 against 0.73 + 0.12: the sum of two keeps the first, the best one the second
    x = np.array([[0.0, 0.0, 1.0, -2.0]])
    assert ref.select(x, 1, "sigmoid", 2, 1, 2)[0][0, 0] == 0 and ref.select(x, 1, "sigmoid", 2, 1, 1)[0][0, 0] == 2
    # the bias decides the choice and not the weight
    ids, w = ref.select(x, 2, "sigmoid", bias=np.array([0, 0, 0, 1.0]), renorm=False)
    assert ids[0].tolist() == [3, 2] and abs(w[0, 0] - 1 / (1 + np.exp(2.0))) < 1e-15
    ids, w = ref.select(np.array([[-np.inf, np.nan, 0.5, -np.inf]]), 3, "softmax")
    assert ids[0].tolist() == [2, 0, 1] and w[0].tolist() == [1, 0, 0]
    ids, w = ref.select(np.full((1, 4), -np.inf), 2, "softmax")
    assert ids[0].tolist() == [0, 1] and w[0].tolist() == [0, 0]


def test_strides_that_are_not_given_are_those_of_rows_next_to_each_other():
    assert int8.Matrix(A, A, 8, 4096).desc.stride == 4096
    refused(int8.Matrix(A, A, 8, 100).linear, int8.F32, A, 100, 1, int8.F32, A, 8)       # 100 is no multiple of 16
    assert [int8.stride_of(c) for c in (1, 128, 129, 4000, 4096, 8190)] == [128, 128, 256, 4224, 4224, 8320]


# ─── which kernels run ──────────────────────────────────────────────────


def matmul_key(n, rows, cols, ws_bytes=1 << 40):
    kernel, a, b, c = int8.kernel(rows, cols, n, ws_bytes=ws_bytes)
    return (kernel, a, b > 1, c > 0) if kernel == int8.TILES else (kernel, b, c)


def test_listed_sizes_run_on_the_kernels_they_are_listed_for():
    for key, sizes in shapes.MATMUL.items():
        for n, rows, cols in sizes:
            assert matmul_key(n, rows, cols) == key, (n, rows, cols)
            need = int8.Matrix(A, A, rows, cols, (cols + 15) // 16 * 16).matmul_workspace(n)
            assert (need > 0) == (key[0] == int8.TILES and key[2])
            assert matmul_key(n, rows, cols, need) == key
    for held, sizes in shapes.LINEAR.items():
        for n, rows, cols in sizes:
            kernel, _, got, tokens = int8.kernel(rows, cols, n, floats=True)
            assert (kernel, got, tokens) == (int8.FEW_FLOAT, held, n), (n, rows, cols)
    for key, sizes in shapes.EXPERTS.items():
        for n, e, k, hidden, ffn in sizes:
            assert int8.moe_kernels(Layer(n_expert=e, top_k=k, hidden=hidden, ffn=ffn).desc, n, key[0]) == key, (n, e, k, hidden, ffn)


def test_no_size_runs_on_a_kernel_that_has_none_listed():
    """Sizes of all lengths: whatever kernel they run on is among the listed ones."""
    rng = np.random.default_rng(1)
    up, down = ({(key[0], key[1], key[i]) for key in shapes.EXPERTS} for i in (2, 3))

    def length(lo, hi):
        return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))

    for _ in range(20000):
        n, rows, cols = length(1, 5000), length(1, 160000), length(1, int8.MAX_COLS)
        assert matmul_key(n, rows, cols, rng.choice([0, 1 << 40])) in shapes.MATMUL, (n, rows, cols)
        kernel, _, held, _ = int8.kernel(rows, cols, n, floats=True)
        assert kernel != int8.FEW_FLOAT or held in shapes.LINEAR, (n, rows, cols)
        e = length(1, 512)
        k, n = int(rng.integers(1, min(16, e) + 1)), length(1, 3000)
        layer, ids = Layer(n_expert=e, top_k=k, hidden=length(1, 20000), ffn=length(1, 40000)), int(rng.integers(0, 2))
        pairs, tok, up_held, down_held = int8.moe_kernels(layer.desc, n, ids)
        assert (pairs, tok, up_held) in up and (pairs, tok, down_held) in down, (n, e, k, layer.desc.hidden, layer.desc.ffn)


# ─── limits ─────────────────────────────────────────────────────────────


def test_the_limits_are_the_headers(tmp_path):
    names = {"OXH_I8_MAX_COLS": int8.MAX_COLS, "OXH_I8_MAX_ROWS": int8.MAX_ROWS, "OXH_I8_MAX_RESULTS": int8.MAX_RESULTS,
             "OXH_MOE_I8_MAX_VALUES": int8.MOE_MAX_VALUES}
    src, exe = tmp_path / "limits.c", tmp_path / "limits"
    src.write_text('#include <stdio.h>\n#include "oxhip.h"\nint main(void) {' +
                   "".join('printf("%s %%zu\\n", (size_t)%s);' % (n, n) for n in names) + "return 0; }")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert {a: int(b) for a, b in (line.split() for line in out.splitlines())} == names


def test_what_lies_next_to_a_limit():
    """The largest sizes are planned for and one more is refused."""
    most, need = int8.MAX_ROWS, ctypes.c_size_t()
    refused(int8.quantize, **{**QUANT, "n_vec": most + 1})
    m = int8.Matrix(**MAT)
    refused(m.matmul, **{**MUL, "n_vec": most + 1})
    assert m.linear_workspace(most) >= most * 128 and m.linear_workspace(most + 1) == 0 and m.matmul_workspace(most + 1) == 0
    high = dict(MAT, rows=most + 1)
    refused(int8.Matrix(**high).matmul, **{**MUL, "out_stride": most + 1})
    assert int8.Matrix(**dict(MAT, rows=most)).linear_workspace(100) > 0 and int8.Matrix(**high).linear_workspace(100) == 0
    large = int8.Matrix(**dict(MAT, rows=most))                        # 2^21 rows: 2^16 tokens have 2^37 results
    refused(large.matmul, **{**MUL, "n_vec": (1 << 16) + 1, "out_stride": most})
    wide = 1 << 23
    refused(int8.quantize, **{**QUANT, "q_stride": wide + 16})
    refused(int8.Matrix(**dict(MAT, stride=wide + 16)).matmul, **MUL)

    def layer(n, **sizes):
        return _lib.lib().oxh_moe_i8_workspace_bytes(ctypes.byref(Layer(**sizes).desc), n, ctypes.byref(need))

    assert layer(65535, hidden=65536, top_k=1) == _lib.OK and need.value > 65535 * 65536
    assert layer(65535, hidden=65537, top_k=1) == _lib.ERR_ARG         # 65600 bytes of codes a token: more than 4 GiB
    assert layer(1 << 14, n_expert=64, top_k=16, ffn=131071) == _lib.OK
    assert layer((1 << 14) + 1, n_expert=64, top_k=16, ffn=131071) == _lib.ERR_ARG


def test_the_largest_sizes_pass_the_checks():
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is a device")                               # the addresses are not real
    most = int8.MAX_ROWS
    refused(int8.quantize, **{**QUANT, "n_vec": most, "q_stride": 1 << 23}, status=_lib.ERR_NO_DEVICE)
    refused(int8.Matrix(**dict(MAT, rows=most, stride=1 << 23)).matmul, **{**MUL, "n_vec": 1 << 16, "out_stride": most},
            status=_lib.ERR_NO_DEVICE)
