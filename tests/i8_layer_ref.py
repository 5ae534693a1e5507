"""What stands around the int8 products (norm, epilogues, gated products, the feed-forward block) from the definitions in 64 bits
on the host, and how far the stated arithmetic may be from them.  HALF = 2^-24: half a step of f32, relative."""
import math

import numpy as np

import i8_ref as ref

HALF = 2.0 ** -24
LOST = 1.03e-36             # what an activation may lose next to the smallest numbers (activation())
NONE, RELU, SILU, GELU, GELU_TANH = range(5)
ACTS = {"none": NONE, "relu": RELU, "silu": SILU, "gelu": GELU, "gelu_tanh": GELU_TANH}
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def norm(x, weight, eps, add=None):
    """s (f32), y (f64 product of the f32 s, not rounded) and the f32 r of rows of f32 values."""
    with np.errstate(all="ignore"):
        s = x.astype(np.float32) if add is None else x.astype(np.float32) + add.astype(np.float32)
        wide = s.astype(np.float64)
        squares = np.array([math.fsum(row) if np.isfinite(row).all() else np.nan for row in wide * wide])
        r = 1.0 / np.sqrt(squares / x.shape[1] + np.float64(np.float32(eps)))
        y = wide * r[:, None] * (1.0 if weight is None else weight.astype(np.float64))
    return s, y


def activation(act, v):
    """act of f32 values, exactly, and a bound on an f32 evaluation's error.

    The bounds count roundings of HALF each.  SILU: an exponential of two units in the last place (4), whose argument is |v| or rounded in units
    of |v| HALF on the way to a power of two (|v|), a sum, a reciprocal or quotient of a unit (2), a product: 8 + |v|.  GELU_TANH: the same of
    2u = 1.596 (v + 0.0447 v^3), five roundings of it (a cube, two products, a sum, a constant) and its way to a power of two: 8 + 6 |2u|.  GELU: v times erfc(z) / 2, z =
    -v / sqrt(2) with two roundings (a constant, a product), which move erfc by at most (2 z^2 + 2) times theirs, z^2 = v^2 / 2; an exponential of z^2 (three
    roundings of z^2 as an argument), and 32 for erfc's own: 40 + 4 v^2.

    LOST: an exponential, its reciprocal and erfc count as 0 below 2^-126.  SILU: from v = -126 ln 2 = -87.34 on, where |v| e^v, which falls
    from there, is 87.34 * 2^-126 = 1.027e-36 at most.  GELU_TANH: from 2u = -87.34, v = -10, on: less.  GELU: |v| of it, at v = -13, 1.6e-37."""
    with np.errstate(all="ignore"):
        x = v.astype(np.float64)
        if act == RELU:
            return np.where(x < 0, 0.0, x), np.zeros(x.shape)
        if act == SILU:
            e, d = ref.silu(x), 8 + np.abs(x)
        elif act == GELU:
            e, d = x * 0.5 * _erfc(-x / math.sqrt(2.0)), 40 + 4 * x * x
        elif act == GELU_TANH:
            u2 = 2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)
            e, d = x / (1.0 + np.exp(-u2)), 8 + 6 * np.abs(u2)
        else:
            return x, np.zeros(x.shape)
        return e, np.where(np.abs(e) > 0, d * HALF * np.abs(e), 0.0) + LOST


def epilogue(q, qs, w, ws, bias, act, residual):
    """f64 results of act(product + bias) + residual, and how far f32 results may be; the product's own f32 steps are exact, its bits
    are known."""
    v = ref.product(q, qs, w, ws, bias)
    e, far = activation(act, v)
    if residual is not None:
        e = e + residual.astype(np.float64)
        far = far + np.where(far > 0, HALF * np.abs(e), 0.0)
    return e, far


def same_or_near(got, kind, want, far):
    """got: results in `kind`'s encoding.  Where far is 0 they are the f32 value rounded once, bit by bit (a sum of two f32 values in f64 is exact
    or rounds as in f32 but for a double rounding, which the half step covers)."""
    g = ref.decode(got, kind).astype(np.float64)
    tiny = {ref.F32: 1e-44, ref.F16: 2.0 ** -25, ref.BF16: 1e-40}[kind]
    step = ref.EPS[kind] + (HALF if kind != ref.F32 else 0.0)
    with np.errstate(all="ignore"):
        off = np.abs(g - want) - (far + step * (np.abs(want) + far) + tiny)
    both_nan = np.isnan(g) & np.isnan(want)
    return bool(np.all(both_nan | (off <= 0) | ((g == want) & np.isinf(g))))


def gated(q, qs, gate, up, act):
    """act(g) * u in f64 of the products' f32 bits, and the f32 bound.  gate, up: (codes, scales, bias)."""
    g, u = ref.product(q, qs, *gate), ref.product(q, qs, *up)
    e, far = activation(act, g)
    e = e * u.astype(np.float64)
    return e, far * np.abs(u) + HALF * np.abs(e) + 1e-44


def ffn(q, qs, gate, up, act, down, residual=None):
    """The block in f64 and its bound.  h is known to `far`; a row's scale moves by at most its largest value's share and its own rounding,
    so a value nearer than 127 times both to a half may get the other code, and each code stands for a scale that
    moves.  The product is three roundings, bias and residual one each."""
    h, far = gated(q, qs, gate, up, act)
    codes, scale = ref.quantize(h)
    s = scale.astype(np.float64)[:, None]
    with np.errstate(all="ignore"):
        rel = (far.max(axis=1) / np.abs(h).max(axis=1))[:, None] + 2 * HALF
        move = 127.0 * rel + np.where(s > 0, far / s, 0.0)
        near = np.where(s > 0, np.abs(np.abs(h / s - codes) - 0.5) <= move, False)
    w, ws, bias = down[0].astype(np.float64), down[1].astype(np.float64), down[2]
    y = (codes.astype(np.float64) @ w.T) * s * ws
    off = (near.astype(np.float64) @ np.abs(w).T) * s * np.abs(ws) + np.abs(y) * (rel + 4 * HALF)
    for more in (bias, residual):
        if more is not None:
            y = y + more.astype(np.float64)
            off = off + HALF * np.abs(y)
    return y, off


# Sizes at which each kernel of a product with an epilogue, and of the gated product, runs on 256 compute units, as in i8_shapes:
# [(tokens, rows, columns)]
EX = {
    (1, 2, 1): [(1, 16, 64), (16, 200, 4096), (7, 4096, 1000), (1, 4107, 3588)],
    (1, 4, 1): [(1, 16, 4102), (8, 40, 8192), (9, 16, 4230), (16, 2400, 8064), (3, 5888, 6528)],
    (1, 8, 1): [(1, 3057, 8209), (2, 4096, 14336), (8, 4096, 14336), (8, 3100, 16384)],
    (2, 2, 2): [(17, 16, 64), (32, 50, 4090)],
    (2, 2, 3): [(34, 16, 65), (48, 70, 4096)],
    (2, 2, 4): [(49, 17, 66), (64, 4096, 4000)],
    (0, 0, False, False): [(514, 19821, 132)],
    (0, 0, False, True): [(776, 23320, 386)],
    (0, 0, True, False): [(130, 11042, 8238)],
    (0, 1, False, False): [(825, 8133, 274)],
    (0, 1, True, False): [(3990, 130, 12785)],
    (0, 2, False, False): [(603, 8092, 132)],
    (0, 2, True, False): [(131, 5498, 5051), (333, 4096, 14336)],
    (0, 3, False, False): [(66, 16916, 65)],
    (0, 3, True, False): [(66, 2700, 7728)],
    (0, 4, False, False): [(67, 16, 64), (70, 300, 1030)],
    (0, 4, True, False): [(48, 4096, 14336), (37, 65, 4683)],
    (0, 5, False, False): [(33, 40000, 100)],
    (0, 5, True, False): [(3777, 1, 4214)],
    (0, 6, False, False): [(1, 4110, 1), (5, 14336, 4096), (16, 5001, 700), (32, 6000, 900)],
    (0, 6, True, False): [(1, 1, 8276), (21, 40, 6617), (24, 4096, 14336)],
    (0, 7, False, False): [(1, 32863, 64), (29, 36260, 70)],
    (0, 7, True, False): [(4, 6516, 7118), (1, 6648, 4249)],
}
GATED = {
    (1, 2, 1): [(1, 16, 1300), (8, 200, 2048), (7, 2048, 1700)],
    (1, 4, 1): [(1, 16, 2103), (8, 40, 4096), (5, 4096, 4096)],
    (1, 8, 1): [(1, 1, 4146), (1, 3415, 4949), (2, 4096, 8192), (4, 3912, 4505)],
    (0, 0, False, False): [(514, 10000, 132)],
    (0, 0, False, True): [(707, 14552, 415)],
    (0, 0, True, False): [(155, 5663, 12638)],
    (0, 1, False, False): [(243, 8805, 1433)],
    (0, 1, True, False): [(204, 2816, 13387)],
    (0, 2, False, False): [(275, 5936, 259)],
    (0, 2, True, False): [(158, 2901, 8183)],
    (0, 3, False, False): [(67, 8328, 65), (333, 4864, 896)],
    (0, 3, True, False): [(252, 2299, 9671)],
    (0, 4, False, False): [(67, 16, 64), (70, 150, 1030), (34, 16, 65), (64, 2048, 2000), (260, 1891, 6834)],
    (0, 4, True, False): [(48, 2048, 8000), (66, 1450, 7728)],
    (0, 5, False, False): [(33, 20000, 100)],
    (0, 5, True, False): [(44, 4218, 15900)],
    (0, 6, False, False): [(1, 1, 1), (7, 2048, 1000), (17, 16, 64), (9, 33, 70), (32, 300, 500), (16, 14336, 4096), (5, 14336, 4096)],
    (0, 6, True, False): [(9, 16, 8276), (1, 1, 8543), (32, 200, 9000)],
    (0, 7, False, False): [(1, 17582, 64), (8, 24486, 40)],
    (0, 7, True, False): [(1, 4455, 7576)],
}
