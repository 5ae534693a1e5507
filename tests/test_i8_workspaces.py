"""Workspaces of the int8 products without a device: what is sized for the largest batch serves every smaller one as its own would,
with the same kernel and the same parts of columns."""
import numpy as np
import pytest

from oxidize_amd import _lib, int8
from test_i8_abi import A, refused
from test_i8_layer_abi import Block


def up(v, to):
    return (v + to - 1) // to * to


def sizes(seed, count, tokens=2048, rows=20000, cols=20000):
    rng = np.random.default_rng(seed)
    return [tuple(int(np.exp(rng.uniform(np.log(a), np.log(b)))) for a, b in ((2, tokens), (1, rows), (1, cols))) for _ in range(count)]


KNOWN = [(2048, 4096, 14336), (1024, 4096, 14336), (1024, 2048, 8192), (333, 300, 5000), (16, 18570, 8070)]


def matrix(rows, cols):
    return int8.Matrix(A, A, rows, cols, int8.stride_of(cols))


def gated(rows, cols):
    return int8.Gated(A, A, A, A, rows, cols, int8.stride_of(cols))


def block(hidden, ffn, n):
    return int(_lib.lib().oxh_i8_ffn_workspace(gated(ffn, hidden)._ref, matrix(hidden, ffn)._ref, n))


def codes_bytes(n, cols):
    return n * up(cols, 64) + up(4 * n, 16)


def fewer(n, seed):
    """some of 1 to n - 1, all of the first ones"""
    return sorted({*range(1, min(n, 70)), *(int(v) for v in np.random.default_rng(seed).integers(1, n, 40))})


@pytest.mark.parametrize("n,rows,cols", KNOWN + sizes(1, 150))
def test_a_smaller_batch_keeps_its_way_in_the_workspace_of_a_larger_one(n, rows, cols):
    m, g = matrix(rows, cols), gated(rows, cols)
    product, linear, both = m.matmul_workspace(n), m.linear_workspace(n), g.workspace(n)
    whole = block(cols, rows, n) if rows <= int8.MAX_COLS else 0        # down: cols rows of `rows` columns
    for k in fewer(n, rows):
        plain, ex, pair = int8.kernel(rows, cols, k), int8.layer_kernel(rows, cols, k, False), int8.layer_kernel(rows, cols, k, True)
        assert int8.kernel(rows, cols, k, ws_bytes=product) == plain and int8.layer_kernel(rows, cols, k, False, product) == ex
        assert int8.layer_kernel(rows, cols, k, True, both) == pair
        if int8.kernel(rows, cols, k, floats=True)[0] != int8.FEW_FLOAT:
            left = linear - codes_bytes(k, cols)
            assert left >= 0 and int8.kernel(rows, cols, k, ws_bytes=left) == plain and int8.layer_kernel(rows, cols, k, False, left) == ex
        if whole:
            left = whole - up(k * up(rows, 64) * 4, 256)
            assert left >= 0 and int8.layer_kernel(rows, cols, k, True, left) == pair
            if int8.kernel(cols, rows, k, floats=True)[0] != int8.FEW_FLOAT:
                left -= codes_bytes(k, rows)
                assert left >= 0 and int8.layer_kernel(cols, rows, k, False, left) == int8.layer_kernel(cols, rows, k, False)


@pytest.mark.parametrize("n,rows,cols", KNOWN + sizes(2, 25, tokens=700))
def test_workspaces_never_shrink_and_hold_no_more_than_some_batch_uses(n, rows, cols):
    m, g, n = matrix(rows, cols), gated(rows, cols), min(n, 700)

    def parts(kernel, of_rows, k):
        return 4 * kernel[2] * k * of_rows if kernel[0] == int8.TILES and kernel[2] > 1 else 0

    product = both = last = 0
    for k in range(1, n + 1):
        product = max(product, parts(int8.kernel(rows, cols, k), up(rows, 4), k), parts(int8.layer_kernel(rows, cols, k, False), up(rows, 4), k))
        both = max(both, parts(int8.layer_kernel(rows, cols, k, True), 2 * up(rows, 4), k))
        assert m.matmul_workspace(k) == product and g.workspace(k) == both
        need = m.linear_workspace(k)
        assert need == (0 if int8.kernel(rows, cols, k, floats=True)[0] == int8.FEW_FLOAT else codes_bytes(k, cols) + product) >= last
        last = need
    if rows <= int8.MAX_COLS:
        wholes = [block(cols, rows, k) for k in range(1, n + 1)]
        assert all(a <= b for a, b in zip(wholes, wholes[1:]))


@pytest.mark.parametrize("n,rows,cols", KNOWN + sizes(3, 40))
def test_calls_accept_the_workspace_of_more_tokens(n, rows, cols):
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    m, down, need = matrix(rows, cols), matrix(cols, min(rows, int8.MAX_COLS)), matrix(rows, cols).linear_workspace(n)
    g = gated(min(rows, int8.MAX_COLS), cols)
    for k in fewer(n, cols):
        refused(m.linear_ex, int8.F32, 2 * A, cols, k, None, int8.F32, A, rows, A, need, status=_lib.ERR_NO_DEVICE)
        refused(m.linear, int8.F32, A, cols, k, int8.F32, A, rows, d_ws=A, ws_bytes=need, status=_lib.ERR_NO_DEVICE)
        b = Block(g, down, int(_lib.lib().oxh_i8_ffn_workspace(g._ref, down._ref, n)))
        refused(b.forward, A, int8.stride_of(cols), A, k, None, int8.F32, A, cols, status=_lib.ERR_NO_DEVICE)


def test_sizes_that_are_refused_have_no_workspace():
    """More than 2^37 results: the calls are refused, and the functions say 0."""
    rows, n = 1 << 21, 1 << 16
    assert matrix(rows, 5000).linear_workspace(n) >= codes_bytes(n, 5000) and matrix(rows, 5000).linear_workspace(n + 1) == 0
    assert matrix(rows, 5000).matmul_workspace(n + 1) == 0 and gated(rows, 5000).workspace(n + 1) == 0
    refused(matrix(rows, 5000).linear, int8.F32, A, 5000, n + 1, int8.F32, A, rows, d_ws=A, ws_bytes=1 << 40)
    assert block(100, 100000, 1 << 20) > 0 and block(100, 131071, (1 << 20) + 16) == 0 and block(1 << 17, 100, (1 << 20) + 1) == 0
