"""What stands around the int8 products of a layer, as cases that can be timed and compared.

  norm     the residual's addition, a root-mean-square norm and int8 rows with one scale each
  linear   float tokens against an int8 matrix, with bias, activation and residual: the form for single tokens and decode batches
  matmul   quantised tokens against such a matrix, with bias, activation and residual: the form for prompts
  gated    quantised tokens against a gate and an up matrix, and activation(gate) * up
  ffn      the feed-forward block: gated, its rows quantised, the down projection and the residual

Where ``own`` is false ``run`` computes them from elementary torch operations.  Activations are N(0, 1) with every 64th
channel eight times as large; weight codes are round(32 N(0, 1)) within +-127 and their scales 2^-5 / sqrt(cols) on average,
so that outputs are of unit size; norm weights are N(1, 0.2^2), biases N(0, 0.1^2).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one token's norm between two products of a decode step: latency
        dict(name="norm_1x4096", kind="norm", n=1, cols=4096, x="f32", add=True, y=False),
        # a long prompt's, half-precision residual stream; a router beside the layer reads the normed floats too
        dict(name="norm_4096x4096", kind="norm", n=4096, cols=4096, x="bf16", add=True, y=True),
        # a decode step's down projection, added to an f32 residual stream
        dict(name="linear_1", kind="linear", n=1, rows=4096, cols=14336, x="f32", act="none", bias=False, residual=True),
        # the first projection of a block without a gate under six sequences decoding together
        dict(name="linear_6", kind="linear", n=6, rows=14336, cols=4096, x="bf16", act="gelu_tanh", bias=True, residual=False),
        # a prompt whose length fits no tile, over the down projection
        dict(name="matmul_333", kind="matmul", n=333, rows=4096, cols=14336, out="bf16", act="none", bias=True, residual=True),
        # a long prompt over the first projection of a block without a gate
        dict(name="matmul_4096", kind="matmul", n=4096, rows=14336, cols=4096, out="bf16", act="gelu", bias=True, residual=False),
        # one decoding token over the gate and up projections
        dict(name="gated_1", kind="gated", n=1, rows=14336, cols=4096, out="f32", act="silu", bias=False),
        # sixteen sequences decoding together
        dict(name="gated_16", kind="gated", n=16, rows=14336, cols=4096, out="bf16", act="silu", bias=False),
        # a prompt of odd length through a small model
        dict(name="gated_333", kind="gated", n=333, rows=4864, cols=896, out="f16", act="gelu_tanh", bias=True),
        # a long prompt
        dict(name="gated_4096", kind="gated", n=4096, rows=14336, cols=4096, out="bf16", act="silu", bias=False),
        # the block for one decoding token
        dict(name="ffn_1", kind="ffn", n=1, hidden=4096, ffn=14336, out="bf16", act="silu", bias=False, residual=True),
        # and for a prompt
        dict(name="ffn_2048", kind="ffn", n=2048, hidden=4096, ffn=14336, out="bf16", act="silu", bias=False, residual=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "linear", "matmul", "gated", "ffn"))
    out = rng.choice(("f32", "f16", "bf16"))
    if kind == "norm":
        cols = _log_int(rng, 500, 16384)
        return dict(kind=kind, n=min(_log_int(rng, 1, 4096), 4096 * 14336 // cols), cols=cols, x=out, add=rng.random() < 0.7,
                    y=rng.random() < 0.3)
    rows, cols = _log_int(rng, 500, 14336), _log_int(rng, 500, 14336)
    if rng.random() < 0.5:                              # as most models have them
        rows, cols = (rows + 15) // 16 * 16, (cols + 63) // 64 * 64
    act, bias, residual = rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")), rng.random() < 0.5, rng.random() < 0.5
    if kind == "linear":
        return dict(kind=kind, n=_log_int(rng, 1, 64), rows=rows, cols=cols, x=out, act=act, bias=bias, residual=residual)
    most = 4096 * 14336 * 4096
    if kind == "matmul":
        return dict(kind=kind, n=min(_log_int(rng, 1, 4096), most // (rows * cols)), rows=rows, cols=cols, out=out, act=act,
                    bias=bias, residual=residual)
    act = rng.choice(("silu", "silu", "gelu", "gelu_tanh", "relu"))
    if kind == "gated":
        return dict(kind=kind, n=min(_log_int(rng, 1, 4096), 2 * most // (2 * rows * cols)), rows=rows, cols=cols, out=out, act=act,
                    bias=bias)
    return dict(kind=kind, n=min(_log_int(rng, 1, 4096), 2 * most // (3 * rows * cols)), hidden=cols, ffn=rows,
                out=rng.choice(("f16", "bf16")), act=act, bias=bias, residual=residual)


def work(case):
    """Every input read once, every output written once; two operations per multiplication."""
    c, kind = case, case["kind"]
    if kind == "norm":
        e = BYTES[c["x"]]
        return dict(bytes=c["n"] * (c["cols"] * (e * (1 + 2 * c["add"] + c["y"]) + 1) + 4) + 4 * c["cols"], flops=6 * c["n"] * c["cols"])
    n = c["n"]
    if kind in ("linear", "matmul"):
        e = BYTES[c["x"] if kind == "linear" else c["out"]]
        token = c["cols"] * e if kind == "linear" else c["cols"] + 4
        return dict(bytes=c["rows"] * (c["cols"] + 4 + 4 * c["bias"]) + n * (token + c["rows"] * e * (1 + c["residual"])),
                    flops=2 * n * c["rows"] * c["cols"])
    if kind == "gated":
        return dict(bytes=2 * c["rows"] * (c["cols"] + 4 + 4 * c["bias"]) + n * (c["cols"] + 4 + c["rows"] * BYTES[c["out"]]),
                    flops=4 * n * c["rows"] * c["cols"])
    h, f = c["hidden"], c["ffn"]
    return dict(bytes=3 * h * f + (4 + 4 * c["bias"]) * (2 * f + h) + n * (h + 4 + h * BYTES[c["out"]] * (1 + c["residual"])),
                flops=6 * n * h * f)


# ─── inputs ─────────────────────────────────────────────────────────────


class Inputs:
    """Seeded random data on the device."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed * 7919 + 23)

    def normal(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.gen)

    def tokens(self, n, cols, kind="f32"):
        x = self.normal(n, cols)
        x[:, ::64] *= 8.0
        return x.to(TYPES[kind])

    def codes(self, rows, cols):
        """int8 rows at the stride that the kernels like best."""
        w = torch.zeros(rows, _stride(cols), dtype=torch.int8, device="cuda")
        step = max(1, (1 << 28) // cols)
        for r in range(0, rows, step):
            w[r:r + step, :cols] = (self.normal(min(step, rows - r), cols) * 32.0).round_().clamp_(-127, 127)
        return w

    def scales(self, rows, cols):
        return (self.normal(rows) * 0.2 + 1.0).abs() / (32.0 * math.sqrt(cols))


def _stride(cols):
    stride = (cols + 127) // 128 * 128
    return stride + 128 if stride % 4096 == 0 else stride


def _empty(shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    c, inp, kind = case, Inputs(seed), case["kind"]
    s, n = dict(case=c), case["n"]
    if kind == "norm":
        s["x"], s["weight"] = inp.tokens(n, c["cols"], c["x"]), inp.normal(c["cols"]) * 0.2 + 1.0
        s["add"] = inp.tokens(n, c["cols"], c["x"]) if c["add"] else None
    else:
        if kind == "ffn":
            matrices, cols, results = (("gate", c["ffn"], c["hidden"]), ("up", c["ffn"], c["hidden"]), ("down", c["hidden"], c["ffn"])), c["hidden"], c["hidden"]
        elif kind == "gated":
            matrices, cols, results = (("gate", c["rows"], c["cols"]), ("up", c["rows"], c["cols"])), c["cols"], c["rows"]
        else:
            matrices, cols, results = (("w", c["rows"], c["cols"]),), c["cols"], c["rows"]
        for name, rows, width in matrices:
            s[name], s[name + "_scale"] = inp.codes(rows, width), inp.scales(rows, width)
            s[name + "_bias"] = inp.normal(rows) * 0.1 if c["bias"] else None
        if kind == "linear":
            s["x"] = inp.tokens(n, cols, c["x"])
        else:
            s["q"], s["q_scale"] = inp.codes(n, cols), (inp.normal(n) * 0.2 + 1.0).abs() / 32.0
        s["residual"] = inp.tokens(n, results, c["x"] if kind == "linear" else c["out"]) if c.get("residual") else None
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def run(s):
    return (_run_own if own else _run_plain)(s)


# ─── the framework's calls ──────────────────────────────────────────────


def _prepare_own(s):
    """The output buffers, workspaces and handles that a program keeps."""
    from oxidize_amd import _lib, int8
    _lib.check(_lib.lib().oxh_init(0))
    c, kind, n = s["case"], s["case"]["kind"], s["case"]["n"]
    code = {"f32": int8.F32, "f16": int8.F16, "bf16": int8.BF16}
    acts = {"none": int8.NONE, "relu": int8.RELU, "silu": int8.SILU, "gelu": int8.GELU, "gelu_tanh": int8.GELU_TANH}

    def ptr(t):
        return None if t is None else t.data_ptr()

    if kind == "norm":
        cols, kept = c["cols"], dict(dtype=TYPES[c["x"]], device="cuda")
        # the codes are turned into the values they stand for by the program's own next operation: a stream that both are put on
        s["stream"] = torch.cuda.Stream()
        s["sum"] = torch.empty(n, cols, **kept) if c["add"] else None
        s["y"] = torch.empty(n, cols, **kept) if c["y"] else None
        s["q"], s["scale"], s["values"] = torch.zeros(n, _stride(cols), dtype=torch.int8, device="cuda"), _empty((n, 1), torch.float32), _empty((n, cols), torch.float32)
        s["codes"] = s["q"][:, :cols]
        norm = int8.Norm(ptr(s["weight"]), 1e-5, d_add=ptr(s["add"]), add_stride=cols, d_sum=ptr(s["sum"]), sum_stride=cols, d_y=ptr(s["y"]),
                         y_stride=cols)
        s["call"] = lambda: norm.quantize(code[c["x"]], ptr(s["x"]), cols, n, cols, ptr(s["q"]), _stride(cols), ptr(s["scale"]),
                                          s["stream"].cuda_stream)
        return
    results = c["hidden"] if kind == "ffn" else c["rows"]
    out = c["x"] if kind == "linear" else c["out"]
    s["out"] = _empty((n, results), TYPES[out])
    if kind in ("linear", "matmul"):
        rows, cols = c["rows"], c["cols"]
        m = int8.Matrix(ptr(s["w"]), ptr(s["w_scale"]), rows, cols, _stride(cols))
        e = int8.Epilogue(ptr(s["w_bias"]), acts[c["act"]], ptr(s["residual"]), rows)
        need = m.linear_workspace(n) if kind == "linear" else m.matmul_workspace(n)
        s["ws"] = _empty(max(need, 16), torch.uint8)
        if kind == "linear":
            s["call"] = lambda: m.linear_ex(code[c["x"]], ptr(s["x"]), cols, n, e, code[out], ptr(s["out"]), rows, ptr(s["ws"]), need)
        else:
            s["call"] = lambda: m.matmul_ex(ptr(s["q"]), _stride(cols), ptr(s["q_scale"]), n, e, code[out], ptr(s["out"]), rows, ptr(s["ws"]),
                                            need)
        return
    rows, cols = (c["ffn"], c["hidden"]) if kind == "ffn" else (c["rows"], c["cols"])
    gated = int8.Gated(ptr(s["gate"]), ptr(s["gate_scale"]), ptr(s["up"]), ptr(s["up_scale"]), rows, cols, _stride(cols), acts[c["act"]],
                       ptr(s["gate_bias"]), ptr(s["up_bias"]))
    if kind == "gated":
        need = gated.workspace(n)
        s["ws"] = _empty(max(need, 16), torch.uint8)
        s["call"] = lambda: gated.matmul(ptr(s["q"]), _stride(cols), ptr(s["q_scale"]), n, code[out], ptr(s["out"]), rows, ptr(s["ws"]), need)
        return
    block = int8.FeedForward(gated, int8.Matrix(ptr(s["down"]), ptr(s["down_scale"]), cols, rows, _stride(rows)), max_tok=n)
    e = int8.Epilogue(ptr(s["down_bias"]), int8.NONE, ptr(s["residual"]), cols)
    s["call"] = lambda: block.forward(ptr(s["q"]), _stride(cols), ptr(s["q_scale"]), n, e, code[out], ptr(s["out"]), cols)


def _run_own(s):
    s["call"]()
    if s["case"]["kind"] != "norm":
        return s["out"]
    with torch.cuda.stream(s["stream"]):
        torch.mul(s["codes"], s["scale"], out=s["values"])
    return dict(sum=s["sum"], y=s["y"], values=s["values"], scale=s["scale"])


# ─── the plain form ─────────────────────────────────────────────────────


def _quantize(v):
    """Codes and f32 scales of f32 rows; the quotient next to a half needs more than 32 bits."""
    scale = (v.abs().amax(1).double() / 127.0).float()
    return torch.round(v.double() / scale.double()[:, None]).to(torch.int8), scale


def _product(q, q_scale, w, w_scale, bias):
    out = (q.float() @ w.float().t()) * q_scale[:, None] * w_scale[None, :]
    return out if bias is None else out + bias


def _activation(act, v):
    if act == "relu":
        return torch.where(v < 0.0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * torch.special.erfc(v * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _gated(c, s, rows, cols):
    gate, up = (_product(s["q"][:, :cols], s["q_scale"], s[name][:, :cols], s[name + "_scale"], s[name + "_bias"]) for name in ("gate", "up"))
    return _activation(c["act"], gate) * up


def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        v = s["x"].float() if s["add"] is None else s["x"].float() + s["add"].float()
        wide = v.double()                                   # codes next to a half need more than 32 bits of the norm
        wide = wide * (1.0 / torch.sqrt((wide * wide).mean(1, keepdim=True) + 1e-5))
        y = (wide * s["weight"].double()).float()
        codes, scale = _quantize(y)
        scale = scale[:, None]
        return dict(sum=v.to(TYPES[c["x"]]) if c["add"] else None, y=y.to(TYPES[c["x"]]) if c["y"] else None, values=codes * scale, scale=scale)
    if kind == "gated":
        return _gated(c, s, c["rows"], c["cols"]).to(TYPES[c["out"]])
    if kind == "ffn":
        q, q_scale = _quantize(_gated(c, s, c["ffn"], c["hidden"]))
        v, out = _product(q, q_scale, s["down"][:, :c["ffn"]], s["down_scale"], s["down_bias"]), c["out"]
    else:
        out = c["x"] if kind == "linear" else c["out"]
        q, q_scale = _quantize(s["x"].float()) if kind == "linear" else (s["q"][:, :c["cols"]], s["q_scale"])
        v = _activation(c["act"], _product(q, q_scale, s["w"][:, :c["cols"]], s["w_scale"], s["w_bias"]))
    return (v if s["residual"] is None else v + s["residual"].float()).to(TYPES[out])


# ─── in 64 bits ─────────────────────────────────────────────────────────


def _exact_rows(v):
    """A row's scale is stored in 32 bits by definition; everything else stays in 64."""
    scale = torch.div(v.abs().max(dim=1, keepdim=True).values, torch.full((1, 1), 127.0, dtype=torch.float64, device=v.device))
    scale = scale.to(torch.float32).to(torch.float64)
    return torch.round(torch.div(v, scale)), scale


def _exact_activation(act, v):
    if act == "relu":
        return v.clamp(min=0.0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * 0.5 * (1.0 + torch.erf(v / math.sqrt(2.0)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def exact(case, seed):
    c, kind = case, case["kind"]
    s = prepare(case, seed)

    def against(tokens, name, cols):
        w = s[name][:, :cols].double() * s[name + "_scale"].double()[:, None]
        out = torch.matmul(tokens, w.t().contiguous())
        return out if s[name + "_bias"] is None else out + s[name + "_bias"].double()

    if kind == "norm":
        v = s["x"].double()
        if s["add"] is not None:
            v = v + s["add"].double()
        total = v
        if c["add"]:                                        # the sum is formed in 32 bits by definition, and so is what is quantised
            v = v.to(torch.float32).to(torch.float64)
        y = v / torch.sqrt(v.pow(2).sum(dim=1, keepdim=True) / c["cols"] + 1e-5) * s["weight"].double()
        codes, scale = _exact_rows(y.to(torch.float32).to(torch.float64))
        return dict(sum=total if c["add"] else None, y=y if c["y"] else None, values=codes * scale, scale=y.abs().max(dim=1, keepdim=True).values / 127.0)
    if kind == "linear":
        q, scale = _exact_rows(s["x"].double())
        x = q * scale
    else:
        x = s["q"][:, :c["hidden"] if kind == "ffn" else c["cols"]].double() * s["q_scale"].double()[:, None]
    if kind in ("gated", "ffn"):
        width = x.shape[1]
        h = _exact_activation(c["act"], against(x, "gate", width)) * against(x, "up", width)
        if kind == "gated":
            return h
        q, scale = _exact_rows(h)
        v = against(q * scale, "down", c["ffn"])
    else:
        v = _exact_activation(c["act"], against(x, "w", c["cols"]))
    return v if s["residual"] is None else v + s["residual"].double()
