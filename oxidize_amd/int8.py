"""int8 rows with one scale per row: the quantiser, products and the expert layer (oxh_i8_*, oxh_moe_ffn_i8).

Addresses are integers, as everywhere in the device-resident layer; nothing here allocates but :class:`MoeLayer`, which
owns its workspace, and :func:`from_packed`, which returns what it made.
"""
import ctypes

import numpy as np

from . import _lib
from . import matvec as mv
from ._lib import check, lib

F32, F16, BF16 = 0, 1, 2
MAX_COLS, MAX_ROWS, MAX_RESULTS, MOE_MAX_VALUES = 131071, 1 << 21, 1 << 37, 1 << 35


def stride_of(cols):
    """The row stride in bytes that rows of `cols` codes are best kept at: whole lines of memory, and not a multiple of 4096, which sends
    the same columns of all rows to the same channels (28672 x 4096 under 16 tokens: 24.1 us at 4224 bytes, 26.4 at 4096)."""
    stride = (cols + 127) // 128 * 128
    return stride + 128 if stride % 4096 == 0 else stride


def quantize(x_type, d_x, x_stride, n_vec, cols, d_q, q_stride, d_scale, d_up=None, stream=None):
    """Rows of floats (or silu(x) * up of two) to codes and scales."""
    check(lib().oxh_i8_quantize(x_type, d_x, x_stride, n_vec, cols, d_up, d_q, q_stride, d_scale, stream))


TILE_256x256, TILE_128x256, TILE_128x192, TILE_128x128, TILE_64x64_RING, TILE_64x64 = range(6)
TILES, FEW, FEW_WIDE, FEW_FLOAT = range(4)


def kernel(rows, cols, n_vec, floats=False, ws_bytes=1 << 40, n_cu=256):
    """Which kernel a product of these sizes runs on: (TILES, tile, parts, half tiles), or one of FEW.. with (waves to 16 rows, stages
    a wave holds, tokens in sixteens); host arithmetic (include/oxhip_lab.h)."""
    out = (ctypes.c_uint32 * 4)()
    check(_lib.lab().i8_kernel(rows, cols, n_vec, n_cu, ws_bytes, int(floats), ctypes.byref(out)))
    return tuple(out)


def moe_kernels(desc, n_tok, ids=True, n_cu=256):
    """(pair by pair?, pairs of a tile, stages gate and up hold or 0 for tiles, stages down holds) of a layer's launch."""
    out = (ctypes.c_uint32 * 4)()
    check(_lib.lab().moe_i8_kernels(ctypes.byref(desc), n_tok, int(ids), n_cu, ctypes.byref(out)))
    return tuple(out)


class Matrix:
    """An int8 matrix resident on the device, a scale per row; the memory is the caller's.  `stride`: bytes from row to row (cols: rows
    next to each other; :func:`stride_of` is fastest)."""

    def __init__(self, d_w, d_scale, rows, cols, stride=None):
        self.desc = _lib.OxhI8Matrix(d_w, stride or cols, d_scale, rows, cols)
        self._ref = ctypes.byref(self.desc)

    def matmul_workspace(self, n_vec):
        return int(lib().oxh_i8_matmul_workspace(self._ref, n_vec))

    def matmul(self, d_q, q_stride, d_q_scale, n_vec, out_type, d_out, out_stride, d_bias=None, d_ws=None, ws_bytes=0, stream=None):
        """Quantised tokens against the matrix."""
        check(lib().oxh_i8_matmul(self._ref, d_q, q_stride, d_q_scale, n_vec, d_bias, out_type, d_out, out_stride, d_ws, ws_bytes,
                                  stream))

    def linear_workspace(self, n_vec):
        return int(lib().oxh_i8_linear_workspace(self._ref, n_vec))

    def linear(self, x_type, d_x, x_stride, n_vec, out_type, d_out, out_stride, d_bias=None, d_ws=None, ws_bytes=0, stream=None):
        """Float tokens against the matrix, quantised on the way."""
        check(lib().oxh_i8_linear(self._ref, x_type, d_x, x_stride, n_vec, d_bias, out_type, d_out, out_stride, d_ws, ws_bytes,
                                  stream))


def from_packed(qtype, d_w, rows, cols, stream=None):
    """A packed matrix (any type oxh_get_rows expands) as int8 rows: (Matrix, [the buffers it lives in]).

    What one scale a row costs beside the packed format's own: a weight moves by at most half a code, its row's largest magnitude / 254.
    That is 1.3 % of the weights' rms for random Q4_K, Q5_K and Q6_K rows of 4096 columns, 1.1 % for Q8_0."""
    stride, step = stride_of(cols), max(1, min(65535, rows, (256 << 20) // (4 * cols)))
    pad = (cols + 3) // 4 * 4
    codes, scale = mv.DeviceBuffer(rows * stride), mv.DeviceBuffer(4 * rows)
    expanded, ids = mv.DeviceBuffer(4 * step * pad), mv.DeviceBuffer.from_host(np.arange(rows, dtype=np.uint32))
    for r in range(0, rows, step):
        n = min(step, rows - r)
        mv.get_rows(qtype, d_w, rows, cols, ids.ptr + 4 * r, n, expanded.ptr, pad, stream)
        quantize(F32, expanded.ptr, pad, n, cols, codes.ptr + r * stride, stride, scale.ptr + 4 * r, stream=stream)
    mv.sync(stream)
    return Matrix(codes.ptr, scale.ptr, rows, cols, stride), [codes, scale]


class MoeLayer:
    """A mixture-of-experts feed-forward over int8 stacks under a given routing; owns its workspace, sized for
    `max_tok` tokens: calls that overlap in time need a layer each.  Strides as :class:`Matrix`'s."""

    def __init__(self, d_w_gate, d_s_gate, d_w_up, d_s_up, d_w_down, d_s_down, n_expert, top_k, hidden, ffn, gate_up_stride=None,
                 down_stride=None, max_tok=16):
        self.desc = _lib.OxhMoeI8(d_w_gate, d_w_up, d_w_down, d_s_gate, d_s_up, d_s_down, gate_up_stride or hidden,
                                  down_stride or ffn, n_expert, top_k, hidden, ffn)
        self.hidden, self.max_tok = hidden, max_tok
        need = ctypes.c_size_t()
        check(lib().oxh_moe_i8_workspace_bytes(ctypes.byref(self.desc), max_tok, ctypes.byref(need)))
        self.workspace = mv.DeviceBuffer(need.value)

    def forward(self, routing, x_type, d_x, n_tok, out_type, d_out, x_stride=None, out_stride=None, stream=None):
        if n_tok > self.max_tok:
            raise ValueError("n_tok %d beyond the workspace's %d" % (n_tok, self.max_tok))
        check(lib().oxh_moe_ffn_i8(ctypes.byref(self.desc), ctypes.byref(routing), x_type, d_x, x_stride or self.hidden, n_tok,
                                   out_type, d_out, out_stride or self.hidden, self.workspace.ptr, self.workspace.nbytes, stream))
