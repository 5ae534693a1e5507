"""The norm, the products with an epilogue, the gated product and the feed-forward block without a device: struct layout, workspaces,
refusals."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import i8_layer_ref as lref
import i8_shapes as shapes
from oxidize_amd import _lib, int8
from test_i8_abi import A, ROOT, refused


def test_bindings_lay_the_new_structs_out_as_the_header_does(tmp_path):
    structs = {n: getattr(_lib, n) for n in ("OxhI8Norm", "OxhI8Epilogue", "OxhI8Gated")}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "oxhip.h"', 'int main(void) {']
    for name, cls in structs.items():
        lines.append('printf("%s size %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f) for f, _ in cls._fields_]
    lines += ['printf("acts %u%u%u%u%u\\n", OXH_ACT_NONE, OXH_ACT_RELU, OXH_ACT_SILU, OXH_ACT_GELU, OXH_ACT_GELU_TANH);', "return 0; }"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    said = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert said.pop() == "acts " + "".join(str(v) for v in (int8.NONE, int8.RELU, int8.SILU, int8.GELU, int8.GELU_TANH))
    for line in said:
        name, field, value = line.split()
        cls = structs[name]
        assert int(value) == (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset), (name, field)


NORM = dict(d_weight=A, eps=1e-5)
ROWS = dict(x_type=int8.F32, d_x=A, x_stride=64, n_vec=2, cols=64, d_q=A, q_stride=64, d_scale=A)


@pytest.mark.parametrize("norm,rows", [(dict(eps=-1e-9), {}), (dict(eps=float("nan")), {}), (dict(d_weight=A + 2), {}),
                                       (dict(d_add=A + 2, add_stride=64), {}), (dict(d_add=A, add_stride=63), {}),
                                       (dict(d_sum=A + 1, sum_stride=64), {}), (dict(d_sum=A, sum_stride=0), {}),
                                       (dict(d_y=A + 3, y_stride=64), {}), (dict(d_y=A, y_stride=10), {}),
                                       (dict(d_y=4 * A, d_sum=4 * A, sum_stride=64, y_stride=64), {}),
                                       (dict(d_sum=A, sum_stride=65), {}), (dict(d_add=2 * A, add_stride=70, d_y=2 * A, y_stride=64), {}),
                                       ({}, dict(x_type=3)), ({}, dict(d_x=0)), ({}, dict(d_x=A + 2)), ({}, dict(x_type=int8.F16, d_x=A + 1)),
                                       ({}, dict(x_stride=63)), ({}, dict(cols=0)), ({}, dict(d_q=0)), ({}, dict(d_q=A + 8)),
                                       ({}, dict(q_stride=72)), ({}, dict(q_stride=48)), ({}, dict(d_scale=0)), ({}, dict(n_vec=(1 << 21) + 1))])
def test_norm_refuses(norm, rows):
    refused(int8.Norm(**{**NORM, **norm}).quantize, **{**ROWS, **rows})


def test_norm_of_nothing_and_of_too_much():
    int8.Norm(A, 0.0).quantize(**{**ROWS, "n_vec": 0})
    refused(int8.Norm(A, 0.0).quantize, **{**ROWS, "cols": 131072, "x_stride": 131072, "q_stride": 131072}, status=_lib.ERR_TOO_WIDE)
    assert _lib.lib().oxh_i8_rmsnorm(None, 0, A, 64, 2, 64, A, 64, A, None) == _lib.ERR_ARG


MAT = dict(d_w=A, d_scale=A, rows=8, cols=100, stride=128)
MUL = dict(d_q=A, q_stride=128, d_q_scale=A, n_vec=3, epilogue=None, out_type=int8.F32, d_out=A, out_stride=8)
LIN = dict(x_type=int8.F32, d_x=2 * A, x_stride=100, n_vec=300, epilogue=None, out_type=int8.F32, d_out=A, out_stride=8, d_ws=A)


def epilogues():
    return [dict(act=5), dict(d_bias=A + 2), dict(d_residual=A + 2, residual_stride=8), dict(d_residual=2 * A, residual_stride=7),
            dict(d_residual=A, residual_stride=9)]


@pytest.mark.parametrize("e", epilogues())
def test_epilogues_refused(e):
    m = int8.Matrix(**MAT)
    refused(m.matmul_ex, **{**MUL, "epilogue": int8.Epilogue(**e)})
    refused(m.linear_ex, **{**LIN, "ws_bytes": m.linear_workspace(300), "epilogue": int8.Epilogue(**e)})


@pytest.mark.parametrize("mat,mul", [(dict(d_w=0), {}), (dict(d_w=A + 4), {}), (dict(stride=120), {}), (dict(stride=96), {}),
                                     (dict(d_scale=0), {}), (dict(cols=0), {}), (dict(rows=(1 << 23) + 1), dict(out_stride=1 << 24)),
                                     ({}, dict(d_q=0)), ({}, dict(d_q=A + 1)), ({}, dict(q_stride=100)), ({}, dict(q_stride=96)),
                                     ({}, dict(d_q_scale=0)), ({}, dict(out_type=7)), ({}, dict(d_out=0)), ({}, dict(d_out=A + 2)),
                                     ({}, dict(out_type=int8.F16, d_out=A + 1)), ({}, dict(out_stride=7)),
                                     ({}, dict(d_ws=A + 4, ws_bytes=64)), ({}, dict(n_vec=(1 << 23) + 1))])
def test_matmul_ex_refuses(mat, mul):
    refused(int8.Matrix(**{**MAT, **mat}).matmul_ex, **{**MUL, **mul})


@pytest.mark.parametrize("change", [dict(d_x=0), dict(x_stride=99), dict(x_type=9), dict(d_out=0), dict(ws_bytes=-1), dict(d_ws=0),
                                    dict(d_ws=A + 8), dict(out_stride=7), dict(d_x=A)])
def test_linear_ex_refuses(change):
    m = int8.Matrix(**MAT)
    need = m.linear_workspace(300)
    if change.get("ws_bytes") == -1:
        change = dict(ws_bytes=need - 1)
    refused(m.linear_ex, **{**LIN, "ws_bytes": need, **change})


GATED = dict(d_w_gate=A, d_s_gate=A, d_w_up=A, d_s_up=A, rows=40, cols=100, stride=128)
GMUL = dict(d_q=A, q_stride=128, d_q_scale=A, n_vec=3, out_type=int8.F32, d_out=A, out_stride=40)


@pytest.mark.parametrize("mat,mul", [(dict(d_w_gate=0), {}), (dict(d_w_up=0), {}), (dict(d_w_up=A + 8), {}), (dict(stride=120), {}),
                                     (dict(stride=96), {}), (dict(d_s_gate=0), {}), (dict(d_s_up=0), {}), (dict(cols=0), {}),
                                     (dict(d_b_gate=A + 1), {}), (dict(d_b_up=A + 2), {}), (dict(act=5), {}),
                                     (dict(rows=(1 << 21) + 1), dict(out_stride=1 << 24)), ({}, dict(d_q=0)), ({}, dict(d_q=A + 1)),
                                     ({}, dict(q_stride=100)), ({}, dict(q_stride=96)), ({}, dict(d_q_scale=0)), ({}, dict(out_type=7)),
                                     ({}, dict(d_out=0)), ({}, dict(out_type=int8.BF16, d_out=A + 1)), ({}, dict(out_stride=39)),
                                     ({}, dict(d_ws=A + 4, ws_bytes=64)), ({}, dict(n_vec=(1 << 21) + 1))])
def test_gated_refuses(mat, mul):
    refused(int8.Gated(**{**GATED, **mat}).matmul, **{**GMUL, **mul})


class Block(int8.FeedForward):
    """The block without a workspace of its own, as there is no device to hold one."""

    def __init__(self, gated=None, down=None, bytes_=None, ptr=A):
        self.gated, self.down, self.max_tok = gated or int8.Gated(**GATED), down or int8.Matrix(A, A, 100, 40, 48), 1 << 30
        need = int(_lib.lib().oxh_i8_ffn_workspace(self.gated._ref, self.down._ref, 3))

        class Ws:
            pass

        self.workspace = Ws()
        self.workspace.ptr, self.workspace.nbytes = ptr, need if bytes_ is None else bytes_


FMUL = dict(d_q=A, q_stride=128, d_q_scale=A, n_tok=3, epilogue=None, out_type=int8.F32, d_out=A, out_stride=100)


def test_ffn_refuses():
    for change in (dict(d_q=0), dict(d_q=A + 4), dict(q_stride=96), dict(d_q_scale=0), dict(out_type=4), dict(d_out=0), dict(out_stride=99),
                   dict(epilogue=int8.Epilogue(act=9)), dict(epilogue=int8.Epilogue(d_residual=A, residual_stride=101)),
                   dict(n_tok=(1 << 21) + 1)):
        refused(Block().forward, **{**FMUL, **change})
    for bad in (Block(down=int8.Matrix(A, A, 100, 41, 48)), Block(down=int8.Matrix(A, 0, 100, 40, 48)), Block(int8.Gated(**{**GATED, "d_s_up": 0})),
                Block(bytes_=3 * 64 * 4 - 1), Block(ptr=A + 128), Block(ptr=0), Block(int8.Gated(**{**GATED, "rows": 0}), int8.Matrix(A, A, 100, 0, 48))):
        refused(bad.forward, **FMUL)
    with pytest.raises(ValueError):
        b = Block()
        b.max_tok = 2
        b.forward(**FMUL)


def test_nothing_to_do_needs_no_device():
    m = int8.Matrix(**MAT)
    m.matmul_ex(**{**MUL, "n_vec": 0})
    m.linear_ex(**{**LIN, "n_vec": 0})
    int8.Matrix(A, A, 0, 64).matmul_ex(A, 64, A, 1, None, int8.F32, A, 8)
    int8.Gated(**GATED).matmul(**{**GMUL, "n_vec": 0})
    int8.Gated(**{**GATED, "rows": 0}).matmul(**GMUL)
    Block().forward(**{**FMUL, "n_tok": 0})


def test_valid_calls_without_a_device_say_so():
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    m, need = int8.Matrix(**MAT), int8.Matrix(**MAT).linear_workspace(300)
    e = int8.Epilogue(A, int8.GELU, A, 8)
    for call, args in ((int8.Norm(A, 1e-6, A, 64, A, 64, 2 * A, 64).quantize, ROWS), (m.matmul_ex, {**MUL, "epilogue": e}),
                       (m.linear_ex, {**LIN, "epilogue": e, "ws_bytes": need}), (int8.Gated(**GATED).matmul, GMUL), (Block().forward, FMUL)):
        refused(call, **args, status=_lib.ERR_NO_DEVICE)


def test_more_results_than_any_memory_holds_are_refused():
    big = 1 << 21
    refused(int8.Matrix(A, A, big, 16).matmul_ex, A, 16, A, big, None, int8.F32, A, big)
    refused(int8.Gated(A, A, A, A, big, 16).matmul, A, 16, A, big, int8.F32, A, big)


def test_workspaces():
    """A workspace for more tokens serves fewer: what a call insists on never shrinks with more of them."""
    lib = _lib.lib()
    for rows, cols in ((300, 5000), (14336, 4096), (64, 16000), (4864, 896)):
        g, down = int8.Gated(A, A, A, A, rows, cols, int8.stride_of(cols)), int8.Matrix(A, A, cols, rows, int8.stride_of(rows))
        for n in (1, 2, 16, 17, 64, 65, 333, 2048):
            need = lib.oxh_i8_ffn_workspace(g._ref, down._ref, n)
            assert need % 16 == 0 and need >= 4 * n * rows
            assert g.workspace(n) <= 64 << 20
    assert lib.oxh_i8_ffn_workspace(None, None, 3) == 0 and lib.oxh_i8_gated_workspace(None, 3) == 0
    assert int8.Gated(**{**GATED, "cols": 131072}).workspace(4) == 0


def key_of(n, rows, cols, gated):
    k = int8.layer_kernel(rows, cols, n, gated)
    return (k[0], k[1], k[2] > 1, k[3] > 0) if k[0] == int8.TILES else (k[0], k[2], k[3])


@pytest.mark.parametrize("gated,table", [(False, lref.EX), (True, lref.GATED)], ids=["epilogue", "gated"])
def test_listed_sizes_run_on_the_kernels_they_are_listed_for(gated, table):
    for key, sizes in table.items():
        for n, rows, cols in sizes:
            assert key_of(n, rows, cols, gated) == key, (n, rows, cols)


@pytest.mark.parametrize("gated,table", [(False, lref.EX), (True, lref.GATED)], ids=["epilogue", "gated"])
def test_no_size_runs_on_a_kernel_that_has_none_listed(gated, table):
    rng = np.random.default_rng(1)
    for _ in range(4000):
        n, rows, cols = (int(np.exp(rng.uniform(np.log(a), np.log(b)))) for a, b in ((1, 5000), (1, 40000), (1, 20000)))
        assert key_of(n, rows, cols, gated) in table, (n, rows, cols)
    assert {key for key in table if key[:2] not in ((0, int8.TILE_64x32_RING), (0, int8.TILE_64x32))} <= set(shapes.MATMUL)


def test_a_product_that_needs_parts_with_an_epilogue_says_so_without():
    """One workspace serves both: where either goes in parts of its columns there is room for them."""
    rng = np.random.default_rng(2)
    for _ in range(2000):
        n, rows, cols = (int(np.exp(rng.uniform(np.log(a), np.log(b)))) for a, b in ((1, 65), (1, 20000), (1, 20000)))
        need = int8.Matrix(A, A, rows, cols, int8.stride_of(cols)).matmul_workspace(n)
        for k in (int8.kernel(rows, cols, n), int8.layer_kernel(rows, cols, n, False)):
            if k[0] == int8.TILES and k[2] > 1:
                assert need >= 4 * k[2] * n * rows
        if need:
            assert int8.layer_kernel(rows, cols, n, False, need) == int8.layer_kernel(rows, cols, n, False)


def test_oracle_activations_at_known_places():
    v = np.array([0.0, 1.0, -1.0, 30.0, -30.0], np.float32)
    assert np.allclose(lref.activation(lref.SILU, v)[0], [0, 0.7310585786300049, -0.2689414213699951, 30, -2.807287e-12], rtol=1e-6)
    assert np.allclose(lref.activation(lref.GELU, v)[0], [0, 0.8413447460685429, -0.15865525393145707, 30, -30 * 4.906713927148187e-198], rtol=1e-6, atol=0)
    assert np.allclose(lref.activation(lref.GELU_TANH, v)[0], [0, 0.8411919906082768, -0.15880800939172324, 30, 0], rtol=1e-6, atol=1e-30)
    assert np.array_equal(lref.activation(lref.RELU, v)[0], [0, 1, 0, 30, 0])
