"""The int8 operators and the expert selection from their definitions, in 64 bits on the host."""
import numpy as np

F32, F16, BF16 = 0, 1, 2
EPS = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}          # half a step, relative


def bf16_bits(a):
    """f32 -> bf16 bits, to nearest, ties to even (finite values)."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def encode(a, kind):
    """f32 values in the element type's bytes (bf16 as bits)."""
    a = np.ascontiguousarray(a, np.float32)
    with np.errstate(over="ignore"):
        return a if kind == F32 else a.astype(np.float16) if kind == F16 else bf16_bits(a)


def decode(a, kind):
    return a.astype(np.float32) if kind != BF16 else (a.astype(np.uint32) << 16).view(np.float32)


def np_type(kind):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[kind]


def padded(a, stride, fill=0):
    out = np.full((a.shape[0], stride), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


def quantize(v):
    """Codes and f32 scales of rows of f32 (or f64) values."""
    v = np.asarray(v, np.float64)
    bad = ~np.isfinite(v).all(axis=1)
    v = np.where(bad[:, None], 0.0, v)
    scale = (np.abs(v).max(axis=1) / 127.0).astype(np.float32)
    scale[scale < np.float32(2.0 ** -126)] = 0.0
    div = np.where(scale > 0, scale, 1).astype(np.float64)
    codes = np.where(scale[:, None] > 0, np.rint(v / div[:, None]), 0).astype(np.int8)
    scale[bad] = np.nan
    return codes, scale


def product(q, q_scale, w, w_scale, bias=None):
    """The stated f32 steps on the exact integer sums."""
    acc = q.astype(np.float64) @ w.astype(np.float64).T            # below 2^53: exact
    with np.errstate(invalid="ignore", over="ignore"):
        out = acc.astype(np.float32) * q_scale.astype(np.float32)[:, None] * w_scale.astype(np.float32)[None, :]
        return out if bias is None else out + bias.astype(np.float32)[None, :]


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def select(logits, top_k, score, n_group=1, top_group=1, best=1, bias=None, renorm=True, scale=1.0):
    """ids [n][k], weights [n][k] in f64."""
    n, e = logits.shape
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, float(np.finfo(np.float32).max)))
    ids, weights = np.zeros((n, top_k), np.int64), np.zeros((n, top_k))
    size = e // max(n_group, 1)
    for t in range(n):
        live = x[t] > -np.inf
        p = np.zeros(e)
        if score == "softmax":
            if live.any():
                with np.errstate(over="ignore"):
                    p[live] = np.exp(x[t][live] - x[t][live].max())
                p /= p.sum()
        else:
            with np.errstate(over="ignore"):
                p[live] = 1.0 / (1.0 + np.exp(-x[t][live]))
        key = p + (0.0 if bias is None else bias.astype(np.float64))
        live &= key > -np.inf                                       # a NaN is not
        open_ = np.ones(e, bool)
        if n_group > 1:
            ranks = []
            for g in range(n_group):
                k = np.sort(key[g * size:(g + 1) * size][live[g * size:(g + 1) * size]])[::-1][:best]
                ranks.append(k.sum() if k.size else -np.inf)
            kept = sorted(range(n_group), key=lambda g: (-ranks[g], g))[:top_group]
            open_ = np.repeat(np.isin(np.arange(n_group), kept), size)
        order = sorted(np.flatnonzero(open_), key=lambda i: (not live[i], -key[i] if live[i] else 0.0, i))[:top_k]
        w = np.where(live[order], p[order], 0.0)
        if renorm:
            w = w / w.sum() if w.sum() > 0 else w * 0.0
        ids[t], weights[t] = order, w * np.float64(np.float32(scale))
    return ids, weights


def group(ids, n_expert):
    """counts, offsets, perm, slot_pos: the pairs by expert, token order kept."""
    n, k = ids.shape
    flat = ids.reshape(-1)
    counts = np.bincount(flat, minlength=n_expert)
    order = np.argsort(flat, kind="stable")
    slot = np.empty(n * k, np.int64)
    slot[order] = np.arange(n * k)
    return counts, np.concatenate([[0], np.cumsum(counts)]), order // k, slot


def experts(x, ids, weights, gate, up, down):
    """The layer's output in f64 and how far the stated f32 arithmetic may be from it.  gate, up: (codes [E][ffn][hidden],
    scales [E][ffn]), down: (codes [E][hidden][ffn], scales [E][hidden]).

    The bound.  gate and up are integers times two f32 scales: 3 roundings, 2^-24 each.  silu(g) * u adds those of
    g's own argument (|g| <= 88 moves silu by at most (1 + |g|) times its relative error), an exponential of two units
    in the last place, a sum, a quotient and a product: d = 2^-24 * (3 + 3 * (1 + |g|) + 4 + 3) relative.  The row's
    scale then moves by at most the largest value's d and its own rounding, so that v / scale moves by at most 127 * D,
    D = 2^-24 + the row's d_max + the value's d: a value nearer than that to a half may get the other code, and the code itself
    stands for s_h times itself, which moves with the scale.  Everything after is 3 roundings, and a weighted sum of k
    terms with k + 1."""
    codes, scale = quantize(x)
    n, k = ids.shape
    u24 = 2.0 ** -24
    out, far = np.zeros((n, down[0].shape[1])), np.zeros((n, down[0].shape[1]))
    for t in range(n):
        for j in range(k):
            e = ids[t, j]
            tok = codes[t].astype(np.float64) * float(scale[t])
            g = (gate[0][e].astype(np.float64) @ tok) * gate[1][e].astype(np.float64)
            u = (up[0][e].astype(np.float64) @ tok) * up[1][e].astype(np.float64)
            h = silu(g) * u
            qh, sh = quantize(h[None])
            qh, sh = qh[0].astype(np.float64), float(sh[0])
            d = u24 * (3 + 3 * (1 + np.minimum(np.abs(g), 88.0)) + 7)
            move = 127.0 * (u24 + d.max() + d)
            near = np.abs(np.abs(h / sh - qh) - 0.5) <= move if sh > 0 else np.zeros(h.shape, bool)
            w = down[0][e].astype(np.float64)
            y = (w @ qh) * sh * down[1][e]
            dy = (np.abs(w) @ near.astype(np.float64)) * sh * np.abs(down[1][e]) + np.abs(y) * (u24 * 4 + d.max())
            out[t] += weights[t, j] * y
            far[t] += abs(weights[t, j]) * (dy + np.abs(y) * u24 * (k + 3))
    return out, far
