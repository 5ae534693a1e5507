"""The int8 operators and the router of many experts, as cases that can be timed and compared.

  quantize   rows of floats to int8 with one scale per row
  linear     float tokens against an int8 matrix with a scale per row: the form for single tokens and decode batches
  matmul     quantised tokens against such a matrix: the form for prompts
  select     router logits to expert ids, weights and the pairs sorted by expert
  experts    a mixture-of-experts layer over int8 stacks, from router logits to combined output

Where ``own`` is false ``run`` computes them from elementary torch operations.  Activations are N(0, 1) with every 64th
channel eight times as large; weight codes are round(32 N(0, 1)) within +-127 and their scales 2^-5 / sqrt(cols) on average,
so that outputs are of unit size; router logits are N(0, 1.5^2), the balance biases N(0, 0.1^2).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token's activation between two products of a decode step: latency
        dict(name="quantize_1x4096", kind="quantize", n=1, cols=4096, x="f32"),
        # a long prompt's input of the down projection
        dict(name="quantize_4096x14336", kind="quantize", n=4096, cols=14336, x="bf16"),
        # a decode step's attention output projection
        dict(name="linear_1", kind="linear", n=1, rows=4096, cols=4096, x="f32", out="f32", bias=False),
        # the gate projection under five sequences decoding together, half-precision activations
        dict(name="linear_5", kind="linear", n=5, rows=14336, cols=4096, x="bf16", out="bf16", bias=True),
        # a small batch against few rows and many columns: the shape that leaves a device idle
        dict(name="matmul_48", kind="matmul", n=48, rows=4096, cols=14336, out="f32", bias=False),
        # a prompt whose length fits no tile, over the down projection
        dict(name="matmul_333", kind="matmul", n=333, rows=4096, cols=14336, out="f32", bias=True),
        # a long prompt over the gate projection
        dict(name="matmul_4096", kind="matmul", n=4096, rows=14336, cols=4096, out="bf16", bias=False),
        # sixteen decoding tokens over eight experts
        dict(name="select_16x8", kind="select", n=16, experts=8, top_k=2, score="softmax", groups=1, top_groups=1, best=1,
             bias=False, renorm=True, scale=1.0, x="f32"),
        # a long prompt over many experts in groups, balanced by biases
        dict(name="select_4096x256", kind="select", n=4096, experts=256, top_k=8, score="sigmoid", groups=8, top_groups=4,
             best=2, bias=True, renorm=True, scale=2.5, x="f32"),
        # one decoding token over many small experts
        dict(name="experts_1x128", kind="experts", n=1, experts=128, top_k=8, hidden=2048, ffn=768, score="softmax",
             groups=1, top_groups=1, best=1, bias=False, renorm=True, scale=1.0, x="bf16", out="bf16"),
        # sixteen decoding tokens over eight large experts
        dict(name="experts_16x8", kind="experts", n=16, experts=8, top_k=2, hidden=4096, ffn=14336, score="softmax",
             groups=1, top_groups=1, best=1, bias=False, renorm=True, scale=1.0, x="f32", out="bf16"),
        # a prompt over many small experts
        dict(name="experts_2000x128", kind="experts", n=2000, experts=128, top_k=8, hidden=2048, ffn=768, score="sigmoid",
             groups=8, top_groups=4, best=2, bias=True, renorm=True, scale=2.5, x="bf16", out="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _router(rng, experts):
    groups = rng.choice([g for g in (1, 1, 4, 8) if experts % g == 0 and experts // g >= 4])
    top_groups = rng.randint((groups + 1) // 2, groups)
    return dict(experts=experts, top_k=rng.randint(1, min(8, top_groups * (experts // groups))), groups=groups,
                top_groups=top_groups, best=rng.choice((1, 2)), score=rng.choice(("softmax", "sigmoid")),
                bias=rng.random() < 0.5, renorm=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)))


def draw(rng):
    kind = rng.choice(("quantize", "linear", "matmul", "matmul", "select", "experts"))
    x = rng.choice(("f32", "f16", "bf16"))
    if kind == "quantize":
        cols = _log_int(rng, 500, 16384)
        return dict(kind=kind, n=min(_log_int(rng, 1, 4096), 4096 * 14336 // cols), cols=cols, x=x)
    if kind == "linear":
        return dict(kind=kind, n=_log_int(rng, 1, 64), rows=_log_int(rng, 500, 32000), cols=_log_int(rng, 500, 14336), x=x,
                    out=x, bias=rng.random() < 0.5)
    if kind == "matmul":
        rows, cols = _log_int(rng, 500, 14336), _log_int(rng, 500, 14336)
        if rng.random() < 0.5:                          # as most models have them
            rows, cols = (rows + 15) // 16 * 16, (cols + 63) // 64 * 64
        return dict(kind=kind, n=min(_log_int(rng, 1, 4096), 4096 * 14336 * 4096 // (rows * cols)), rows=rows, cols=cols, out=x,
                    bias=rng.random() < 0.5)
    if kind == "select":
        return dict(kind=kind, n=_log_int(rng, 1, 4096), x=x, **_router(rng, rng.choice((8, 16, 60, 64, 128, 160, 256))))
    r = _router(rng, rng.choice((8, 16, 32, 64, 128)))
    hidden = _log_int(rng, 500, 4096)
    ffn = min(_log_int(rng, 384, 14336), 8 * 4096 * 14336 // (r["experts"] * hidden))
    return dict(kind=kind, n=max(1, min(_log_int(rng, 1, 2000), 2000 * 8 * 2048 * 768 // (r["top_k"] * hidden * ffn))), hidden=hidden,
                ffn=ffn, x=x, out=rng.choice(("f16", "bf16")), **r)


def work(case):
    """Every input read once, every output written once; two operations per multiplication."""
    c, kind = case, case["kind"]
    e = {"f32": 4, "f16": 2, "bf16": 2}
    if kind == "quantize":
        return dict(bytes=c["n"] * (c["cols"] * (e[c["x"]] + 1) + 4), flops=4 * c["n"] * c["cols"])
    if kind in ("linear", "matmul"):
        token = c["cols"] * (e[c["x"]] if kind == "linear" else 1) + (4 if kind == "matmul" else 0)
        return dict(bytes=c["rows"] * (c["cols"] + 4 + 4 * c["bias"]) + c["n"] * (token + c["rows"] * e[c["out"]]),
                    flops=2 * c["n"] * c["rows"] * c["cols"])
    n, n_exp, k = c["n"], c["experts"], c["top_k"]
    if kind == "select":
        return dict(bytes=n * n_exp * e[c["x"]] + 4 * n_exp * c["bias"] + 16 * n * k + 8 * n_exp + 4, flops=20 * n * n_exp)
    hit = n_exp * (1.0 - (1.0 - k / n_exp) ** n)        # experts that get a token, on average
    return dict(bytes=hit * (3 * c["hidden"] * c["ffn"] + 4 * (2 * c["ffn"] + c["hidden"])) + n * (4 * n_exp + c["hidden"] * (e[c["x"]] + e[c["out"]])),
                flops=6 * n * k * c["hidden"] * c["ffn"])


# ─── inputs ─────────────────────────────────────────────────────────────


class Inputs:
    """Seeded random data on the device."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed * 7919 + 17)

    def normal(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.gen)

    def tokens(self, n, cols, kind="f32"):
        x = self.normal(n, cols)
        x[:, ::64] *= 8.0
        return x.to(TYPES[kind])

    def codes(self, rows, cols):
        """int8 rows a multiple of 64 bytes apart, as the kernels take them."""
        w = torch.zeros(rows, _stride(cols), dtype=torch.int8, device="cuda")
        step = max(1, (1 << 28) // cols)
        for r in range(0, rows, step):
            w[r:r + step, :cols] = (self.normal(min(step, rows - r), cols) * 32.0).round_().clamp_(-127, 127)
        return w

    def scales(self, rows, cols):
        return (self.normal(rows) * 0.2 + 1.0).abs() / (32.0 * math.sqrt(cols))


def _stride(cols):
    return (cols + 63) // 64 * 64


def _empty(shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    c, inp, kind = case, Inputs(seed), case["kind"]
    s = dict(case=c)
    if kind == "quantize":
        s["x"] = inp.tokens(c["n"], c["cols"], c["x"])
    elif kind in ("linear", "matmul"):
        s["w"], s["w_scale"] = inp.codes(c["rows"], c["cols"]), inp.scales(c["rows"], c["cols"])
        s["bias"] = inp.normal(c["rows"]) * 0.1 if c["bias"] else None
        if kind == "linear":
            s["x"] = inp.tokens(c["n"], c["cols"], c["x"])
        else:
            s["q"], s["q_scale"] = inp.codes(c["n"], c["cols"]), (inp.normal(c["n"]) * 0.2 + 1.0).abs() / 32.0
    else:
        s["logits"] = (inp.normal(c["n"], c["experts"]) * 1.5).to(TYPES[c["x"]] if kind == "select" else torch.float32)
        s["bias"] = inp.normal(c["experts"]) * 0.1 if c["bias"] else None
        if kind == "experts":
            e, h, f = c["experts"], c["hidden"], c["ffn"]
            s["x"] = inp.tokens(c["n"], h, c["x"])
            for name, rows, cols in (("gate", f, h), ("up", f, h), ("down", h, f)):
                s[name], s[name + "_scale"] = inp.codes(e * rows, cols), inp.scales(e * rows, cols)
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
    from oxidize_amd import matvec as mv
    _lib.check(_lib.lib().oxh_init(0))
    c, kind = s["case"], s["case"]["kind"]
    code = {"f32": int8.F32, "f16": int8.F16, "bf16": int8.BF16}

    def ptr(t):
        return None if t is None else t.data_ptr()

    if kind == "quantize":
        n, cols = c["n"], c["cols"]
        s["q"], s["scale"] = torch.zeros(n, _stride(cols), dtype=torch.int8, device="cuda"), _empty(n, torch.float32)
        s["call"] = lambda: int8.quantize(code[c["x"]], ptr(s["x"]), cols, n, cols, ptr(s["q"]), _stride(cols), ptr(s["scale"]))
        return
    if kind in ("linear", "matmul"):
        n, rows, cols = c["n"], c["rows"], c["cols"]
        m = int8.Matrix(ptr(s["w"]), ptr(s["w_scale"]), rows, cols, _stride(cols))
        need = m.linear_workspace(n) if kind == "linear" else m.matmul_workspace(n)
        s["out"], s["ws"] = _empty((n, rows), TYPES[c["out"]]), _empty(max(need, 16), torch.uint8)
        if kind == "linear":
            s["call"] = lambda: m.linear(code[c["x"]], ptr(s["x"]), cols, n, code[c["out"]], ptr(s["out"]), rows, ptr(s["bias"]),
                                         ptr(s["ws"]), need)
        else:
            s["call"] = lambda: m.matmul(ptr(s["q"]), _stride(cols), ptr(s["q_scale"]), n, code[c["out"]], ptr(s["out"]), rows,
                                         ptr(s["bias"]), ptr(s["ws"]), need)
        return
    n, e, k = c["n"], c["experts"], c["top_k"]
    router = mv.MoeRouter(e, k, score=c["score"], n_group=c["groups"], top_group=c["top_groups"], group_best=c["best"],
                          d_bias=ptr(s["bias"]), renorm=c["renorm"], scale=c["scale"])
    r = s["routing"] = dict(ids=_empty((n, k), torch.int32), weights=_empty((n, k), torch.float32),
                            counts=_empty(e, torch.int32), offsets=_empty(e + 1, torch.int32),
                            perm=_empty(n * k, torch.int32), slot_pos=_empty((n, k), torch.int32))
    routing = mv.make_routing(*[ptr(r[name]) for name in ("ids", "weights", "counts", "offsets", "perm", "slot_pos")])
    need = router.workspace_bytes(n)
    s["ws"] = _empty(max(need, 16), torch.uint8)
    logits_type = code[c["x"]] if kind == "select" else int8.F32

    def select():
        router.select(logits_type, ptr(s["logits"]), e, n, routing, ptr(s["ws"]), need)

    if kind == "select":
        s["call"] = select
        return
    h, f = c["hidden"], c["ffn"]
    layer = int8.MoeLayer(*[ptr(s[name + part]) for name in ("gate", "up", "down") for part in ("", "_scale")], e, k, h, f,
                          gate_up_stride=_stride(h), down_stride=_stride(f), max_tok=n)
    s["out"] = _empty((n, h), TYPES[c["out"]])

    def forward():
        select()
        layer.forward(routing, code[c["x"]], ptr(s["x"]), n, code[c["out"]], ptr(s["out"]))

    s["call"] = forward


def _run_own(s):
    s["call"]()
    kind, c = s["case"]["kind"], s["case"]
    if kind == "quantize":
        return dict(codes=s["q"][:, :c["cols"]], scale=s["scale"])
    if kind == "select":
        return s["routing"]
    return s["out"]


# ─── the plain form ─────────────────────────────────────────────────────


def _quantize(v):
    """Codes and f32 scales of f32 rows; the quotient next to a half needs more than 32 bits."""
    scale = (v.abs().amax(1).double() / 127.0).float()
    return torch.round(v.double() / scale.double()[:, None]).to(torch.int8), scale


def _product(q, q_scale, w, w_scale):
    return (q.float() @ w.float().t()) * q_scale[:, None] * w_scale[None, :]


def _swiglu(gate, up):
    return gate / (1.0 + torch.exp(-gate)) * up


def _select(c, logits, bias):
    n, e, k = c["n"], c["experts"], c["top_k"]
    x = logits.double()
    if c["score"] == "softmax":
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-x))
    key = p if bias is None else p + bias.double()
    if c["groups"] > 1:
        g = key.view(n, c["groups"], e // c["groups"])
        rank = torch.sort(g, dim=2, descending=True).values[:, :, :c["best"]].sum(2)
        kept = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        out = torch.ones(n, c["groups"], dtype=torch.bool, device=x.device).scatter_(1, kept, False)
        key = torch.where(out[:, :, None], -math.inf, g).view(n, e)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = (w * c["scale"]).float()
    flat = ids.reshape(-1)
    counts = (flat[:, None] == torch.arange(e, device=x.device)[None, :]).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    order = torch.sort(flat, stable=True).indices
    slot = torch.empty_like(order).scatter_(0, order, torch.arange(n * k, device=x.device))
    return {name: v.to(torch.int32) if v.dtype == torch.int64 else v for name, v in
            dict(ids=ids, weights=w, counts=counts, offsets=offsets, perm=order // k, slot_pos=slot.view(n, k)).items()}


def _experts(c, s, r):
    """Each expert over its own run of the sorted pairs; the sizes of the runs go to the host."""
    e, h, f = c["experts"], c["hidden"], c["ffn"]
    q, q_scale = _quantize(s["x"].float())
    perm, y = r["perm"].long(), torch.empty(c["n"] * c["top_k"], h, device="cuda")
    at = r["offsets"].tolist()
    for i in range(e):
        if at[i] == at[i + 1]:
            continue
        tok = perm[at[i]:at[i + 1]]
        part = {name: _product(q[tok], q_scale[tok], s[name][i * f:(i + 1) * f, :h], s[name + "_scale"][i * f:(i + 1) * f])
                for name in ("gate", "up")}
        qh, h_scale = _quantize(_swiglu(part["gate"], part["up"]))
        y[at[i]:at[i + 1]] = _product(qh, h_scale, s["down"][i * h:(i + 1) * h, :f], s["down_scale"][i * h:(i + 1) * h])
    return (y[r["slot_pos"].long()] * r["weights"][:, :, None]).sum(1).to(TYPES[c["out"]])


def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "quantize":
        codes, scale = _quantize(s["x"].float())
        return dict(codes=codes, scale=scale)
    if kind in ("linear", "matmul"):
        q, q_scale = _quantize(s["x"].float()) if kind == "linear" else (s["q"][:, :c["cols"]], s["q_scale"])
        out = _product(q, q_scale, s["w"][:, :c["cols"]], s["w_scale"])
        return (out if s["bias"] is None else out + s["bias"]).to(TYPES[c["out"]])
    r = _select(c, s["logits"], s["bias"])
    return r if kind == "select" else _experts(c, s, r)


# ─── in 64 bits ─────────────────────────────────────────────────────────


def _exact_rows(v):
    """A row's scale is stored in 32 bits by definition; everything else stays in 64."""
    scale = torch.div(v.abs().max(dim=1, keepdim=True).values, torch.full((1, 1), 127.0, dtype=torch.float64, device=v.device))
    scale = scale.to(torch.float32).to(torch.float64)
    return torch.round(torch.div(v, scale)), scale


def _exact_routing(c, logits, bias):
    """(token, expert) pairs of each token in the order of choice, and their weights, one token at a time on the host."""
    import numpy as np
    x = logits.double().cpu().numpy()
    b = np.zeros(c["experts"]) if bias is None else bias.double().cpu().numpy()
    size = c["experts"] // c["groups"]
    ids, weights = np.zeros((c["n"], c["top_k"]), np.int64), np.zeros((c["n"], c["top_k"]))
    for t in range(c["n"]):
        p = np.exp(x[t] - x[t].max()) / np.exp(x[t] - x[t].max()).sum() if c["score"] == "softmax" else 1.0 / (1.0 + np.exp(-x[t]))
        key = p + b
        ranks = np.array([np.sort(key[g * size:(g + 1) * size])[-c["best"]:].sum() for g in range(c["groups"])])
        open_ = np.argsort(-ranks, kind="stable")[:c["top_groups"]]
        among = np.sort(np.concatenate([np.arange(g * size, (g + 1) * size) for g in open_]))
        ids[t] = among[np.argsort(-key[among], kind="stable")[:c["top_k"]]]
        w = p[ids[t]]
        weights[t] = w / (w.sum() if c["renorm"] else 1.0) * c["scale"]
    return ids, weights


def exact(case, seed):
    c, kind = case, case["kind"]
    s = prepare(case, seed)
    if kind == "quantize":
        return dict(codes=None, scale=s["x"].double().abs().max(dim=1).values / 127.0)
    if kind in ("linear", "matmul"):
        q, scale = _exact_rows(s["x"].double()) if kind == "linear" else (s["q"][:, :c["cols"]].double(), s["q_scale"].double()[:, None])
        out = torch.matmul(q * scale, (s["w"][:, :c["cols"]].double() * s["w_scale"].double()[:, None]).t().contiguous())
        return out if s["bias"] is None else out + s["bias"].double()
    ids, weights = _exact_routing(c, s["logits"], s["bias"])
    if kind == "select":
        return dict(ids=None, weights=torch.from_numpy(weights), counts=None, offsets=None, perm=None, slot_pos=None)
    h, f = c["hidden"], c["ffn"]
    ids, weights = torch.from_numpy(ids).cuda(), torch.from_numpy(weights).cuda()
    q, scale = _exact_rows(s["x"].double())
    x, out = q * scale, torch.zeros(c["n"], h, dtype=torch.float64, device="cuda")

    def expert(name, i, rows, cols):
        return (s[name][i * rows:(i + 1) * rows, :cols].double() * s[name + "_scale"][i * rows:(i + 1) * rows].double()[:, None]).t().contiguous()

    for i in range(c["experts"]):
        tok, place = torch.nonzero(ids == i, as_tuple=True)
        if tok.numel():
            g = torch.matmul(x[tok], expert("gate", i, f, h))
            qh, sh = _exact_rows(g * torch.sigmoid(g) * torch.matmul(x[tok], expert("up", i, f, h)))
            out[tok] += weights[tok, place][:, None] * torch.matmul(qh * sh, expert("down", i, h, f))
    return out
