"""oxh_moe_select on the device against the definition in 64 bits (i8_ref): ids and the grouping are exact, weights are
the 64-bit ones rounded once."""
import numpy as np
import pytest

import i8_ref as ref
from oxidize_amd import _lib
from oxidize_amd import matvec as mv

pytestmark = pytest.mark.gpu
KINDS = [ref.F32, ref.F16, ref.BF16]


def select(logits, kind, k, stride=None, bias=None, **how):
    """What the device makes of encoded logits, as arrays; entries behind the last pair must stay as they were."""
    n, e = logits.shape
    stride = stride or e
    d_l = mv.DeviceBuffer.from_host(ref.padded(logits, stride))
    d_b = None if bias is None else mv.DeviceBuffer.from_host(bias.astype(np.float32))
    r = mv.MoeRouter(e, k, d_bias=None if bias is None else d_b.ptr, **how)
    sizes = dict(ids=n * k, weights=n * k, counts=e, offsets=e + 1, perm=n * k, slot_pos=n * k)
    d = {name: mv.DeviceBuffer.from_host(np.full(size + 4, 0xABCD1234, np.uint32)) for name, size in sizes.items()}
    need = r.workspace_bytes(n)
    ws = mv.DeviceBuffer(need) if need else None
    r.select(kind, d_l.ptr, stride, n, mv.make_routing(*[b.ptr for b in d.values()]), ws.ptr if ws else None, need)
    mv.sync()
    out = {}
    for name, size in sizes.items():
        raw = d[name].download(np.uint32, size + 4)
        assert (raw[size:] == 0xABCD1234).all(), name
        out[name] = raw[:size].view(np.float32) if name == "weights" else raw[:size].astype(np.int64)
    return out


def check(got, logits, k, score, n_group=1, top_group=1, group_best=1, bias=None, renorm=True, scale=1.0):
    n, e = logits.shape
    ids, w = ref.select(logits, k, score, n_group, top_group, group_best, bias, renorm, scale)
    assert np.array_equal(got["ids"].reshape(n, k), ids)
    # 64-bit arithmetic in another order: far inside one more part in 2^24 / 1000
    assert np.all(np.abs(got["weights"].reshape(n, k) - w) <= 2.0 ** -24 * 1.001 * np.abs(w) + 2.0 ** -149)
    counts, offsets, perm, slot = ref.group(ids, e)
    for name, want in (("counts", counts), ("offsets", offsets), ("perm", perm), ("slot_pos", slot)):
        assert np.array_equal(got[name], want), name


@pytest.mark.parametrize("n,e,k,groups,top,best", [
    (1, 1, 1, 1, 1, 1), (1, 8, 2, 1, 1, 1), (16, 8, 8, 1, 1, 1), (16, 300, 9, 1, 1, 1), (17, 300, 9, 6, 4, 2), (32, 64, 5, 1, 1, 1), (33, 64, 5, 2, 1, 1), (63, 60, 4, 4, 2, 2), (64, 64, 6, 8, 3, 1), (65, 64, 6, 8, 3, 2),
    (100, 65, 5, 5, 1, 1), (129, 128, 16, 1, 1, 1), (500, 160, 6, 8, 3, 1), (1000, 256, 8, 8, 4, 2), (4096, 16, 2, 1, 1, 1),
    (4097, 32, 4, 4, 2, 2), (1024, 48, 5, 3, 2, 2), (1025, 48, 5, 1, 1, 1), (2049, 300, 12, 4, 3, 2), (65535, 24, 2, 1, 1, 1), (8200, 12, 3, 3, 2, 2), (300, 512, 16, 64, 2, 2), (77, 511, 7, 7, 3, 2), (17000, 4, 1, 1, 1, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_select(oxh, n, e, k, groups, top, best, score):
    rng = np.random.default_rng(n + e)
    logits = rng.normal(size=(n, e)).astype(np.float32) * np.float32(1.5)
    how = dict(n_group=groups, top_group=top, group_best=best, renorm=n % 2 == 0, scale=2.5 if n % 3 else 1.0)
    bias = rng.normal(size=e).astype(np.float32) * np.float32(0.1) if e % 2 == 0 else None
    got = select(logits, ref.F32, k, e + n % 5, bias, score=score, **how)
    check(got, logits, k, score, bias=bias, **how)


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_logits_go_to_the_lowest_expert(oxh, kind, score):
    """Few distinct values: ties within and across the experts of a lane, and between groups."""
    rng = np.random.default_rng(9)
    for e, k, groups, top in ((200, 9, 1, 1), (96, 4, 8, 3)):
        logits = ref.encode(rng.integers(-2, 3, size=(150, e)).astype(np.float32), kind)
        got = select(logits, kind, k, score=score, n_group=groups, top_group=top, group_best=2)
        check(got, ref.decode(logits, kind), k, score, groups, top, 2)


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top", [(1, 1), (6, 2)])
def test_masked_experts(oxh, kind, score, groups, top):
    """-inf, NaN, +inf and the type's lowest value among the logits; rows with fewer than k experts left, with one, with none."""
    rng = np.random.default_rng(3)
    n, e, k = 120, 72, 6
    x = rng.normal(size=(n, e)).astype(np.float32)
    lowest = {ref.F32: -3.4028235e38, ref.F16: -65504.0, ref.BF16: -3.3895314e38}[kind]
    x[rng.random((n, e)) < 0.3] = lowest
    enc = ref.encode(x, kind)
    ninf, pinf, nan = {ref.F32: (np.float32(-np.inf), np.float32(np.inf), np.float32(np.nan)),
                       ref.F16: (np.float16(-np.inf), np.float16(np.inf), np.float16(np.nan)),
                       ref.BF16: (np.uint16(0xFF80), np.uint16(0x7F80), np.uint16(0x7FC0))}[kind]
    enc[rng.random((n, e)) < 0.3] = ninf
    enc[rng.random((n, e)) < 0.02] = nan
    enc[::10, 5] = pinf
    enc[3], enc[4], enc[5] = ninf, nan, lowest if kind != ref.BF16 else np.uint16(0xFF7F)
    enc[6], enc[6, 70], enc[7], enc[7, 11:13] = ninf, 0, ninf, 0
    enc[8] = pinf
    got = select(enc, kind, k, score=score, n_group=groups, top_group=top, group_best=2)
    check(got, ref.decode(enc, kind), k, score, groups, top, 2)
    w = got["weights"].reshape(n, k)
    assert not w[3].any() and not w[4].any() and np.isfinite(w).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_biases_that_mask_or_force(oxh, score):
    rng = np.random.default_rng(8)
    x = rng.normal(size=(70, 40)).astype(np.float32)
    bias = rng.normal(size=40).astype(np.float32)
    bias[3], bias[4], bias[17], bias[30] = -np.inf, np.nan, np.inf, np.inf
    got = select(x, ref.F32, 5, bias=bias, score=score, n_group=4, top_group=3, group_best=2)
    check(got, x, 5, score, 4, 3, 2, bias)
    assert not np.isin(got["ids"], [3, 4]).any() and (got["ids"] == 17).sum() == 70


def test_two_keys_closer_than_32_bits_tell(oxh):
    """Keys 2^-40 apart: score 0.5 plus biases, summed in 64 bits."""
    x = np.zeros((5, 64), np.float32)
    bias = np.zeros(64, np.float32)
    bias[40], bias[9] = 2.0 ** -39, 2.0 ** -40
    got = select(x, ref.F32, 3, bias=bias, score="sigmoid")
    assert got["ids"].reshape(5, 3).tolist() == [[40, 9, 0]] * 5


def test_calls_may_follow_each_other_over_one_workspace(oxh):
    rng = np.random.default_rng(1)
    for n in (5000, 200, 30, 900):
        x = rng.normal(size=(n, 64)).astype(np.float32)
        check(select(x, ref.F32, 4, score="softmax"), x, 4, "softmax")


def test_logits_of_more_than_4_gib(oxh):
    n, e, k, stride, last = 65535, 40, 3, 20000, 50
    d_l = mv.DeviceBuffer(4 * n * stride)
    _lib.check(oxh.oxh_memset(d_l.ptr, 0, 4 * n * stride, None))
    x = np.random.default_rng(3).normal(size=(last, e)).astype(np.float32)
    d_l.upload(ref.padded(x, stride, 9), 4 * (n - last) * stride)
    r = mv.MoeRouter(e, k)
    sizes = dict(ids=n * k, weights=n * k, counts=e, offsets=e + 1, perm=n * k, slot_pos=n * k)
    d = {name: mv.DeviceBuffer(4 * size) for name, size in sizes.items()}
    ws = mv.DeviceBuffer(r.workspace_bytes(n))
    r.select(ref.F32, d_l.ptr, stride, n, mv.make_routing(*[b.ptr for b in d.values()]), ws.ptr, ws.nbytes)
    mv.sync()
    got = {name: d[name].download(np.float32 if name == "weights" else np.int32, size) for name, size in sizes.items()}
    check(got, np.concatenate([np.zeros((n - last, e), np.float32), x]), k, "softmax")


@pytest.mark.parametrize("e", [64, 130, 500])
def test_keys_that_differ_in_their_last_bits(oxh, e):
    """Sigmoids between 1 - 2^-43 and 1, and scores of 0.5 with biases down to the last bit of the sum, 2^-53: largest first,
    wherever the experts lie among the lanes; equal ones by their number."""
    rng = np.random.default_rng(e)
    x = np.zeros((40, e), np.float32)
    far = np.linspace(29.8, 35.8, 16).astype(np.float32)              # neighbours 4e-14 to 1e-16 apart
    for t in range(40):
        x[t, rng.choice(e, size=16, replace=False)] = far
    got = select(x, ref.F32, 12, score="sigmoid", renorm=False)
    check(got, x, 12, "sigmoid", renorm=False)
    assert np.array_equal(np.take_along_axis(x, got["ids"].reshape(40, 12), 1), np.tile(far[:3:-1], (40, 1)))
    bias, at = np.zeros(e, np.float32), rng.choice(e, size=8, replace=False)
    bias[at] = np.arange(1, 9) * 2.0 ** -53
    got = select(np.zeros((40, e), np.float32), ref.F32, 10, bias=bias, score="sigmoid")
    zeros = np.setdiff1d(np.arange(e), at)[:2]
    assert got["ids"].reshape(40, 10).tolist() == [at[::-1].tolist() + zeros.tolist()] * 40


def test_rows_of_counts_with_a_choice_for_every_thread(oxh):
    """64 tokens of 16 choices to a workgroup, the last one with a single token; ids that cover a row's 1024 threads."""
    x = np.random.default_rng(6).normal(size=(8193 + 64, 20)).astype(np.float32)
    check(select(x, ref.F32, 16, score="sigmoid"), x, 16, "sigmoid")


def test_calls_of_one_stream_share_a_workspace(oxh):
    """Large and small calls over several expert counts, one after the other on one stream into ONE workspace, which holds other counts before
    each; outputs of their own, one wait at the end."""
    rng = np.random.default_rng(4)
    calls, need = [], 0
    for n, e, k in ((5000, 64, 4), (200, 64, 4), (30, 300, 5), (900, 20, 3), (5000, 500, 8), (17, 64, 4), (2100, 33, 16), (70, 512, 2)):
        x, r = rng.normal(size=(n, e)).astype(np.float32), mv.MoeRouter(e, k, "sigmoid")
        sizes = dict(ids=n * k, weights=n * k, counts=e, offsets=e + 1, perm=n * k, slot_pos=n * k)
        calls.append((x, k, r, mv.DeviceBuffer.from_host(x), {name: mv.DeviceBuffer(4 * size) for name, size in sizes.items()}, sizes))
        need = max(need, r.workspace_bytes(n))
    ws = mv.DeviceBuffer.from_host(np.full(need, 0xFF, np.uint8))
    for x, k, r, d_x, d, sizes in calls:
        r.select(ref.F32, d_x.ptr, x.shape[1], x.shape[0], mv.make_routing(*[b.ptr for b in d.values()]), ws.ptr, need)
    mv.sync()
    for x, k, r, d_x, d, sizes in calls:
        got = {name: d[name].download(np.float32 if name == "weights" else np.int32, size) for name, size in sizes.items()}
        check(got, x, k, "sigmoid")
