"""GPU tests of the scoring operators against plain implementations in 64 bits.

Tolerances count roundings.  H is half a step of the output's type (2^-11 for
f16, 2^-24 for f32, relative), E = 2^-24 that of the f32 arithmetic inside; a
sum of n terms in f32 is off by at most about n E times the sum of magnitudes
(the longest chain of a thread, plus the few steps of the join)."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {"fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
TINY = {"fp16": 2.0 ** -25, "fp32": 2.0 ** -150}  # half a step of the smallest numbers
SENTINEL = 12345.0


def _dtype(profile):
    import torch

    return torch.float16 if profile == "fp16" else torch.float32


def _np(t):
    import torch

    torch.cuda.synchronize()
    return t.detach().cpu().numpy()


# ====================================================================== token scores

class Scores:
    """A token-scores dispatch with its own output buffers, filled with sentinels."""

    def __init__(self, pk, device, logits, columns, profile, targets=None, top_k=0, slots=None, **kw):
        import torch

        rows = kw.pop("rows", logits.shape[0])
        slots = rows if slots is None else slots
        f = dict(dtype=torch.float32, device="cuda")
        self.out = dict(log_probs=torch.full((slots,), SENTINEL, **f), log_sums=torch.full((slots,), SENTINEL, **f),
                        entropies=torch.full((slots,), SENTINEL, **f),
                        top_ids=torch.full((slots, top_k), -7, dtype=torch.int32, device="cuda"),
                        top_log_probs=torch.full((slots, top_k), SENTINEL, **f))
        targets = torch.zeros(slots, dtype=torch.int32, device="cuda") if targets is None else targets
        self.call = pk.kernels.TokenScoresKernel.create(device, None, 0, profile).create_dispatch(dict(
            label="scores", logits=logits, rows=rows, columns=columns, targets=targets, top_k=top_k, slots=slots,
            row_stride=kw.pop("row_stride", logits.shape[-1]), **self.out, **kw))

    def __call__(self, stream=None):
        self.call.encode(stream)
        return self

    def host(self):
        return {k: _np(v) for k, v in self.out.items()}


def _score_reference(x, targets, k):
    """x: float64 [rows, columns] (no NaN or +inf)."""
    top = x.max(axis=1, keepdims=True)
    empty = np.isneginf(top[:, 0])
    away = np.where(empty[:, None], -np.inf, x - np.where(np.isneginf(top), 0.0, top))
    e = np.exp(away)
    s = np.where(empty, 1.0, e.sum(axis=1))
    log_s = np.log(s)
    share = np.where(e > 0, e * np.where(e > 0, away, 0.0), 0.0).sum(axis=1) / s
    ids = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -x), axis=1)[:, :k]
    rows = np.arange(x.shape[0])
    return dict(log_probs=away[rows, targets] - log_s, log_sums=np.where(empty, -np.inf, top[:, 0] + log_s),
                entropies=np.where(empty, 0.0, log_s - share), top_ids=ids,
                top_log_probs=np.take_along_axis(away, ids, axis=1) - log_s[:, None])


def _check_scores(got, x, targets, k, rows=slice(None)):
    """Errors: a column's exponential is off by 2 ulp of ex2.approx, the rounding of x - m and of the product
    with log2(e) (|d| E each, and e^d |d| <= 1); a thread's chain has columns / 32 terms at most; log s is off
    by s's relative error.  Every output then rounds at its own size."""
    ref = _score_reference(x[rows], targets[rows], k)
    np.testing.assert_array_equal(got["top_ids"][rows], ref["top_ids"])
    rel = (x.shape[1] / 32 + 64) * E
    finite = np.where(np.isfinite(x), np.abs(x), 0.0)[rows].max(axis=1)
    for name in ("log_probs", "log_sums", "top_log_probs"):
        g, r = got[name][rows].astype(np.float64), ref[name]
        lim = np.isneginf(r)
        np.testing.assert_array_equal(np.isneginf(g), lim, err_msg=name)
        tol = rel + 4 * E * np.where(lim, 0.0, np.abs(r))
        size = finite if r.ndim == 1 else finite[:, None]
        assert np.all(np.abs(np.where(lim, 0.0, g - np.where(lim, 0.0, r))) <= tol + 2 * E * size), name
    # u = sum e^d d: every term's error is |d| times that of its exponential, and |u| / s = log s - entropy.
    g, r = got["entropies"][rows].astype(np.float64), ref["entropies"]
    log_s = np.where(np.isneginf(ref["log_sums"]), 0.0, np.log(np.maximum(1.0, x.shape[1])))
    assert np.all(np.abs(g - r) <= rel * (4 + log_s + np.abs(log_s - r)))


def _logits(rng, rows, stride, profile, std=2.5):
    x = (rng.standard_normal((rows, stride)) * std).astype(np.float16 if profile == "fp16" else np.float32)
    return x


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,columns,stride,first,k", [
    (1, 1, 1, 0, 1), (3, 5, 1032, 1025, 5), (9, 33, 33, 0, 32), (5, 31, 40, 3, 31), (17, 1025, 1032, 0, 4),
    (2, 4097, 4099, 1, 8), (1, 32000, 32000, 0, 8), (150, 9000, 9001, 0, 5), (3, 131075, 131077, 2, 16), (300, 70, 72, 1, 1),
    (2, 640, 640, 0, 0),
])
def test_token_scores(pk, device, profile, rows, columns, stride, first, k):
    import torch

    rng = np.random.default_rng(rows * 7 + columns)
    x = _logits(rng, rows, stride, profile)
    targets = rng.integers(0, columns, rows)
    s = Scores(pk, device, torch.from_numpy(x).cuda(), columns, profile, torch.from_numpy(targets.astype(np.int32)).cuda(),
               k, first_column=first)
    _check_scores(s().host(), x[:, first:first + columns].astype(np.float64), targets, k)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("columns", [7, 1025, 20000])
def test_token_scores_masks_and_orders(pk, device, profile, columns):
    """Rows that a mask leaves with half, one or none of their columns, rows of the type's lowest value, equal
    rows, rows in ascending order (every value is the best so far) and signed zeros."""
    import torch

    rng = np.random.default_rng(columns)
    x = _logits(rng, 9, columns, profile)
    lowest = np.finfo(x.dtype).min
    x[0, rng.random(columns) < 0.5] = -np.inf
    x[1, :] = -np.inf
    x[2, :] = -np.inf
    x[2, columns // 2] = 1.5
    x[3, :] = lowest
    x[4, 1:] = lowest
    x[5, :] = 0.25
    x[6] = np.sort(x[6])
    x[7] = np.sort(x[7])[::-1]
    x[8] = np.where(rng.random(columns) < 0.5, 0.0, -0.0)
    targets = rng.integers(0, columns, 9)
    targets[2] = columns // 2
    k = min(columns, 8)
    s = Scores(pk, device, torch.from_numpy(x).cuda(), columns, profile, torch.from_numpy(targets.astype(np.int32)).cuda(), k)
    got = s().host()
    _check_scores(got, x.astype(np.float64) + 0.0, targets, k)
    assert got["entropies"][1] == 0.0 and np.all(np.isneginf(got["top_log_probs"][1]))
    np.testing.assert_array_equal(got["top_ids"][1], np.arange(k))


@pytest.mark.parametrize("columns", [40, 5000])
def test_token_scores_of_rows_without_a_distribution(pk, device, columns):
    """NaN or +inf anywhere: NaN scores; the alternatives still rank, NaN last.  A target outside the row: NaN."""
    import torch

    rng = np.random.default_rng(3)
    x = _logits(rng, 5, columns, "fp32")
    x[0, columns - 1] = np.nan
    x[1, 3] = np.inf
    x[2, :] = np.nan
    targets = np.array([0, 1, 2, columns, -1], np.int32)
    got = Scores(pk, device, torch.from_numpy(x).cuda(), columns, "fp32", torch.from_numpy(targets).cuda(), 4)().host()
    for r in (0, 1, 2):
        for name in ("log_probs", "log_sums", "entropies", "top_log_probs"):
            assert np.all(np.isnan(got[name][r])), (name, r)
    rank = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    ids = np.lexsort((np.broadcast_to(np.arange(columns), x.shape), -rank), axis=1)[:, :4]
    np.testing.assert_array_equal(got["top_ids"], ids)
    assert np.all(np.isnan(got["log_probs"][3:])) and np.all(np.isfinite(got["log_sums"][3:]))


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,columns,stride,first,k", [
    (4801, 1, 1, 0, 1), (4801, 100, 101, 0, 5), (2600, 1025, 1032, 0, 32), (4800, 1025, 1033, 3, 17), (2500, 2100, 2100, 0, 0),
    (5000, 4099, 4104, 5, 8), (2400, 9000, 9000, 0, 20), (1300, 21000, 21001, 1, 6),
])
def test_token_scores_of_many_rows(pk, device, profile, rows, columns, stride, first, k):
    """Rows by the thousand: one or more warps to a row, streamed."""
    test_token_scores(pk, device, profile, rows, columns, stride, first, k)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
def test_token_scores_of_many_rows_with_masks_and_ties(pk, device, profile):
    """Masked columns, rows of equal values (whose candidates overflow the pool) and rows without a distribution
    give the same among thousands of rows as in a call of their own."""
    import torch

    rng = np.random.default_rng(61)
    x = _logits(rng, 4800, 3001, profile)
    x[7], x[1200] = -np.inf, x.dtype.type(1.5)
    x[2400, 1:] = -np.inf
    x[3000, ::3] = x[3000, 0]
    x[4000, 17], x[4799, 5] = np.nan, np.inf
    targets = rng.integers(0, 3001, 4800).astype(np.int32)
    names = ("log_probs", "log_sums", "entropies", "top_ids", "top_log_probs")
    for k in (4, 24):
        many = Scores(pk, device, torch.from_numpy(x).cuda(), 3001, profile, torch.from_numpy(targets).cuda(), k)().host()
        at = np.array([7, 1200, 2400, 3000, 4000, 4799, 11])
        few = Scores(pk, device, torch.from_numpy(np.ascontiguousarray(x[at])).cuda(), 3001, profile,
                     torch.from_numpy(targets[at]).cuda(), k)().host()
        for n in names:
            if n == "top_ids":
                np.testing.assert_array_equal(many[n][at], few[n])
            else:  # two orders of the same f32 sums of 3001 terms: 2 * (3001 / 32 + 40) roundings at most, log sum below 13
                np.testing.assert_allclose(many[n][at], few[n], rtol=0, atol=2 * (3001 / 32 + 40) * E * 13, equal_nan=True)


def test_token_scores_row_count_and_row_map(pk, device):
    """Rows behind the device's count, slots outside the buffers and slots nobody maps to stay as they were."""
    import torch

    rng = np.random.default_rng(4)
    x = _logits(rng, 12, 1032, "fp32")
    slots = 20
    rmap = rng.permutation(slots)[:12].astype(np.int32)
    rmap[2] = slots + 5
    targets = rng.integers(0, 1025, slots).astype(np.int32)
    s = Scores(pk, device, torch.from_numpy(x).cuda(), 1025, "fp32", torch.from_numpy(targets).cuda(), 4, slots,
               row_map=torch.from_numpy(rmap).cuda(), row_count=torch.tensor([9], dtype=torch.int32, device="cuda"))
    got = s().host()
    live = [r for r in range(9) if r != 2]
    at = rmap[live]
    _check_scores({k: v[at] for k, v in got.items()}, x[live][:, :1025].astype(np.float64), targets[at].astype(np.int64), 4)
    rest = np.setdiff1d(np.arange(slots), at)
    for name, v in got.items():
        assert np.all(v[rest] == (-7 if name == "top_ids" else SENTINEL)), name


def test_token_scores_single_outputs(pk, device):
    import torch

    x = torch.randn(3, 100, device="cuda")
    full = Scores(pk, device, x, 100, "fp32", top_k=4)().host()
    for name in ("log_sums", "entropies", "top_ids", "top_log_probs"):
        shape = full[name].shape
        out = torch.zeros(shape, dtype=torch.int32 if name == "top_ids" else torch.float32, device="cuda")
        pk.kernels.TokenScoresKernel.create(device, None, 0, "fp32").create_dispatch(dict(
            label="one", logits=x, rows=3, columns=100, top_k=4, **{name: out})).encode()
        np.testing.assert_array_equal(_np(out), full[name])


def test_token_scores_offsets_past_32_bits(pk, device):
    import torch

    stride = (1 << 30) + 8
    x = torch.zeros(2 * stride + 100, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(5)
    rows = _logits(rng, 3, 100, "fp16")
    for r in range(3):
        x[r * stride:r * stride + 100] = torch.from_numpy(rows[r]).cuda()
    targets = rng.integers(0, 100, 3)
    s = Scores(pk, device, x, 100, "fp16", torch.from_numpy(targets.astype(np.int32)).cuda(), 8, rows=3, row_stride=stride)
    _check_scores(s().host(), rows.astype(np.float64), targets, 8)


def test_token_scores_repeat_bit_for_bit(pk, device):
    import torch

    x = torch.randn(4, 70001, device="cuda").half()
    first = Scores(pk, device, x, 70001, "fp16", top_k=16)().host()
    for _ in range(5):
        again = Scores(pk, device, x, 70001, "fp16", top_k=16)().host()
        for name in first:
            np.testing.assert_array_equal(again[name], first[name])


# ====================================================================== residual norm

def _norm64(v, kind, gamma, beta, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(axis=1, keepdims=True)
    return v / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps) * gamma + (beta if kind == "layer" else 0.0)


def _norm_error(v, dv, kind, gamma, beta, eps):
    """Bound of the f32 norm's error where v is off by at most dv (per row)."""
    if kind == "none":
        return dv
    n = v.shape[1] / 32 + 32  # a thread's chain at its longest, and the join
    dmean = n * E * np.abs(v).mean(axis=1, keepdims=True) + dv.max(axis=1, keepdims=True) if kind == "layer" else 0.0
    c = v - v.mean(axis=1, keepdims=True) if kind == "layer" else v
    rstd = 1.0 / np.sqrt((c * c).mean(axis=1, keepdims=True) + eps)
    dc = dv + dmean + 2 * E * np.abs(v)
    # 1 / deviation is off, relatively, by the sum's chain and by the centred values' error over the deviation.
    drel = n * E + 2 * dc.max(axis=1, keepdims=True) * rstd
    out = c * rstd * gamma
    return dc * rstd * np.abs(gamma) + np.abs(out) * (drel + 4 * E) + (2 * E * np.abs(out + beta) if kind == "layer" else 0.0)


def _residual_norm(pk, device, x, f, profile, post="none", pre="none", gate=None, gate_rows=0, scale=1.0, eps=1e-5, seed=0,
                   place=None, run=True):
    import torch

    rows, channels = x.shape
    rng = np.random.default_rng(seed)
    dt = _dtype(profile)
    par = {}
    for at, kind in (("post", post), ("pre", pre)):
        if kind != "none":
            par[f"{at}_gamma"] = (1 + 0.3 * rng.standard_normal(channels)).astype(np.float32)
        if kind == "layer":
            par[f"{at}_beta"] = (0.3 * rng.standard_normal(channels)).astype(np.float32)
    dev = {k: torch.from_numpy(v).cuda() for k, v in par.items()}
    tx, tf = torch.from_numpy(x).cuda(), torch.from_numpy(f).cuda()
    y = torch.full((rows, channels), SENTINEL, dtype=dt, device="cuda")
    h = torch.full((rows, channels), SENTINEL, dtype=dt, device="cuda") if pre != "none" else None
    if place == "input":
        y = tx
    if place == "both":
        y, h = tx, tf if pre != "none" else None
    if place == "swapped":
        y, h = tf, tx if pre != "none" else None
    d = dict(label="norm", input=tx, block=tf, output=y, rows=rows, channels=channels, post=post, pre=pre, epsilon=eps,
             residual_scale=scale, gate_rows=gate_rows, **dev)
    if h is not None:
        d["normalized"] = h
    if gate is not None:
        d["gate"] = torch.from_numpy(gate).cuda()
    call = pk.kernels.ResidualNormKernel.create(device, None, 0, profile).create_dispatch(d)
    call.encode()
    got = (_np(y), None if h is None else _np(h))
    g = 1.0 if gate is None else gate.astype(np.float64)[np.arange(rows) // gate_rows if gate_rows else np.zeros(rows, int)]
    p64 = {k: v.astype(np.float64) for k, v in par.items()}
    f64, x64 = f.astype(np.float64), x.astype(np.float64)
    u = _norm64(f64, post, p64.get("post_gamma"), p64.get("post_beta"), eps)
    du = _norm_error(f64, np.zeros_like(f64), post, p64.get("post_gamma"), p64.get("post_beta"), eps)
    ref = x64 + scale * g * u
    dref = np.abs(scale * g) * (du + 2 * E * np.abs(u)) + 2 * E * np.abs(ref)
    H, T = HALF[profile], TINY[profile]
    assert np.all(np.abs(got[0] - ref) <= dref + H * (np.abs(ref) + dref) + T)
    if pre != "none":
        want = _norm64(ref, pre, p64["pre_gamma"], p64.get("pre_beta"), eps)
        dw = _norm_error(ref, dref, pre, p64["pre_gamma"], p64.get("pre_beta"), eps)
        assert np.all(np.abs(got[1] - want) <= dw + H * (np.abs(want) + dw) + T)
    return got


def _rows(rng, rows, channels, profile, std=1.0, mean=0.0):
    return (rng.standard_normal((rows, channels)) * std + mean).astype(np.float16 if profile == "fp16" else np.float32)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,channels", [(1, 4), (1, 640), (9, 1024), (3, 68), (2, 1500), (5, 2048), (3, 4100), (2, 8192),
                                           (1, 16388), (2, 32768), (1000, 64), (2401, 640), (5003, 264), (2370, 1024),
                                           (1201, 2048), (20001, 16)])
def test_residual_norm_shapes(pk, device, profile, rows, channels):
    rng = np.random.default_rng(rows + channels)
    x, f = _rows(rng, rows, channels, profile, 2.0), _rows(rng, rows, channels, profile, 1.5, 0.3)
    _residual_norm(pk, device, x, f, profile, "layer", "layer", scale=0.5)
    _residual_norm(pk, device, x, f, profile, "rms", "rms")


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("post", ["none", "layer", "rms"])
@pytest.mark.parametrize("pre", ["none", "layer", "rms"])
@pytest.mark.parametrize("gate_rows", [None, 0, 3, 7])
@pytest.mark.parametrize("rows", [13, 4099])
def test_residual_norm_kinds_and_gates(pk, device, profile, post, pre, gate_rows, rows):
    rng = np.random.default_rng(11)
    x, f = _rows(rng, rows, 320, profile, 2.0), _rows(rng, rows, 320, profile)
    gate = None
    if gate_rows is not None:
        gate = rng.standard_normal((1 if gate_rows == 0 else -(-rows // gate_rows), 320)).astype(np.float32)
    _residual_norm(pk, device, x, f, profile, post, pre, gate, gate_rows or 0, scale=0.25)


@pytest.mark.parametrize("place", ["input", "both", "swapped"])
@pytest.mark.parametrize("pre", ["none", "layer"])
@pytest.mark.parametrize("rows,channels", [(11, 640), (11, 4096), (2500, 640)])
def test_residual_norm_in_place(pk, device, place, pre, rows, channels):
    rng = np.random.default_rng(12)
    x, f = _rows(rng, rows, channels, "fp16", 2.0), _rows(rng, rows, channels, "fp16")
    want = _residual_norm(pk, device, x, f, "fp16", "layer", pre, scale=0.5)
    got = _residual_norm(pk, device, x, f, "fp16", "layer", pre, scale=0.5, place=place)
    np.testing.assert_array_equal(got[0], want[0])
    if pre != "none":
        np.testing.assert_array_equal(got[1], want[1])


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
def test_residual_norm_large_mean_and_constant_rows(pk, device, profile):
    """A mean a thousand deviations away, and rows without deviation (the norm is then 0, or beta)."""
    rng = np.random.default_rng(13)
    x = _rows(rng, 4, 1024, profile)
    f = _rows(rng, 4, 1024, "fp32", 1.0, 1000.0).astype(x.dtype)
    f[1] = 7.0
    f[2] = 0.0
    _residual_norm(pk, device, x, f, profile, "layer", "rms", scale=0.5)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("channels", [64, 1000, 9000])
def test_residual_norm_unaligned_buffers(pk, device, profile, channels):
    """Rows that start one element into their buffers: the element-wise route, the same numbers."""
    import torch

    rng = np.random.default_rng(14)
    x, f = _rows(rng, 3, channels, profile), _rows(rng, 3, channels, profile)
    want = _residual_norm(pk, device, x, f, profile, pre="rms", scale=0.5)
    dt = _dtype(profile)
    bufs = [torch.zeros(3 * channels + 1, dtype=dt, device="cuda") for _ in range(4)]
    bufs[0][1:] = torch.from_numpy(x).cuda().flatten()
    bufs[1][1:] = torch.from_numpy(f).cuda().flatten()
    gamma = torch.from_numpy((1 + 0.3 * np.random.default_rng(0).standard_normal(channels)).astype(np.float32)).cuda()
    pk.kernels.ResidualNormKernel.create(device, None, 0, profile).create_dispatch(dict(
        label="n", input=bufs[0][1:], block=bufs[1][1:], output=bufs[2][1:], normalized=bufs[3][1:], rows=3,
        channels=channels, pre="rms", pre_gamma=gamma, residual_scale=0.5)).encode()
    np.testing.assert_array_equal(_np(bufs[2])[1:].reshape(3, channels), want[0])
    # The threads of a row sum in another order.
    H = HALF[profile]
    got = _np(bufs[3])[1:].reshape(3, channels).astype(np.float64)
    assert np.all(np.abs(got - want[1]) <= (2 * H + 2 * (channels / 32 + 32) * E) * np.abs(want[1]) + TINY[profile])
    assert _np(bufs[2])[0] == 0 and _np(bufs[3])[0] == 0


# ====================================================================== int4 products

def _int4(pk, device, rows, inner, columns, group, profile, epilogue="none", seed=0, a=None, scale=0.5):
    import torch

    rng = np.random.default_rng(seed + rows + inner + columns)
    codes = rng.integers(0, 16, (inner, columns)).astype(np.uint8)
    npd = np.float16 if profile == "fp16" else np.float32
    scales = ((0.5 + rng.random((inner // group, columns))) * 0.05).astype(npd)
    a = rng.standard_normal((rows, inner)).astype(npd) if a is None else a
    weight = pk.kernels.Int4Weight.from_words(torch.from_numpy(pk.runtime_plan.pack_int4(codes).view(np.int32)).cuda(),
                                              torch.from_numpy(scales).cuda(), inner, group)
    out = torch.full((rows, columns), SENTINEL, dtype=_dtype(profile), device="cuda")
    d = dict(label="int4", a=torch.from_numpy(a).cuda(), weight=weight, output=out, rows=rows)
    bias = rng.standard_normal(columns).astype(np.float32)
    res = rng.standard_normal((rows, columns)).astype(npd)
    if epilogue in ("bias", "silu", "relu"):
        d["bias"] = torch.from_numpy(bias).cuda()
        d["activation"] = epilogue if epilogue != "bias" else "none"
    if epilogue.startswith("residual"):
        d["residual"], d["residual_scale"] = torch.from_numpy(res).cuda(), scale
        if epilogue == "residual in place":
            out.copy_(d["residual"])
            d["residual"] = out
    pk.kernels.Int4GemvKernel.create(device, None, 0, profile).create_dispatch(d).encode()
    got = _np(out).astype(np.float64)
    w = (codes.astype(np.float64) - 8.0) * np.repeat(scales.astype(np.float64), group, axis=0)
    a64 = a.astype(np.float64)
    mass = np.abs(a64) @ np.abs(w)
    v = a64 @ w
    # f32 accumulation, up to one step (2^-23) per product instruction and join; FP32 inputs as two f16 parts
    # lose at most 2^-22 of each input and, relative to a tile's largest, 2^-39.
    dv = (inner / 16 + 64) * 2 * E * mass
    if profile == "fp32":
        dv = dv + 2.0 ** -22 * mass + 2.0 ** -38 * np.abs(a64).max() * np.abs(w).sum(axis=0)
    if epilogue in ("bias", "silu", "relu"):
        v = v + bias
        dv = dv + E * np.abs(v)
        if epilogue == "relu":
            v = np.maximum(v, 0.0)
        elif epilogue == "silu":
            sig = 1.0 / (1.0 + np.exp(-v))
            v, dv = v * sig, dv * 1.1 + 8 * E * np.abs(v * sig)  # |silu'| < 1.1
    elif epilogue.startswith("residual"):
        v, dv = res + scale * v, scale * dv + 2 * E * np.abs(res + scale * v)
    H = HALF[profile]
    err = np.abs(got - v) - (dv + H * (np.abs(v) + dv) + TINY[profile])
    assert np.all(err <= 0), (float(err.max()), float(np.abs(got - v).max()))


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,columns,group", [
    (1, 32, 1, 32), (1, 640, 640, 64), (2, 640, 1032, 128), (3, 96, 17, 32), (7, 1280, 250, 64), (8, 256, 16, 256),
    (9, 4096, 48, 128), (16, 1024, 333, 32), (17, 512, 40, 512), (32, 8192, 24, 128), (33, 640, 100, 64), (64, 2048, 80, 32),
    (64, 320, 2600, 64), (1, 16384, 64, 128), (5, 384, 5000, 384),
])
def test_int4_gemv(pk, device, profile, rows, inner, columns, group):
    _int4(pk, device, rows, inner, columns, group, profile)


# Enough rows and tiles for the tcgen05 route: five tiles of 128 x 128 weights per SM and 32 columns.
@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,columns,group,epilogue", [
    (17, 1056, 12005, 32, "none"), (17, 640, 19000, 64, "bias"), (32, 4096, 4001, 128, "silu"), (33, 128, 97000, 128, "none"),
    (64, 8192, 1500, 512, "residual"), (20, 32768, 300, 128, "residual in place"), (19, 2208, 6100, 32, "relu"),
    (64, 96, 50000, 32, "none"), (23, 16384, 1000, 64, "none"), (17, 65536, 260, 128, "none"), (33, 262144, 50, 4096, "none"),
])
def test_int4_gemv_many_rows(pk, device, profile, rows, inner, columns, group, epilogue):
    _int4(pk, device, rows, inner, columns, group, profile, epilogue)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("epilogue", ["bias", "silu", "relu", "residual", "residual in place"])
@pytest.mark.parametrize("rows", [1, 12])
def test_int4_gemv_epilogues(pk, device, profile, epilogue, rows):
    _int4(pk, device, rows, 640, 136, 64, profile, epilogue)


def test_int4_gemv_wide_range_of_inputs(pk, device):
    """FP32 rows whose inputs span many powers of two, zero rows and rows near the ends of the range."""
    rng = np.random.default_rng(21)
    a = (rng.standard_normal((6, 512)) * 10.0 ** rng.uniform(-6, 6, (6, 512))).astype(np.float32)
    a[1] = 0.0
    a[2] *= np.float32(1e25)
    a[3] *= np.float32(1e-30)
    a[4, ::2] = 0.0
    for r in (slice(0, 2), slice(2, 3), slice(3, 4), slice(4, 6)):
        _int4(pk, device, a[r].shape[0], 512, 48, 64, "fp32", a=np.ascontiguousarray(a[r]))


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
def test_int4_gemv_infinities_and_nan_stay_in_their_rows(pk, device, profile):
    import torch

    rng = np.random.default_rng(22)
    npd = np.float16 if profile == "fp16" else np.float32
    codes = rng.integers(9, 16, (256, 32)).astype(np.uint8)  # positive weights
    weight = pk.kernels.Int4Weight.from_words(torch.from_numpy(pk.runtime_plan.pack_int4(codes).view(np.int32)).cuda(),
                                              torch.full((4, 32), 0.25, dtype=_dtype(profile), device="cuda"), 256, 64)
    a = rng.standard_normal((4, 256)).astype(npd)
    a[1, 77], a[2, 200] = np.inf, np.nan
    out = torch.zeros((4, 32), dtype=_dtype(profile), device="cuda")
    pk.kernels.Int4GemvKernel.create(device, None, 0, profile).create_dispatch(dict(
        label="g", a=torch.from_numpy(a).cuda(), weight=weight, output=out, rows=4)).encode()
    got = _np(out)
    assert np.all(np.isposinf(got[1])) and np.all(np.isnan(got[2])) and np.all(np.isfinite(got[[0, 3]]))


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,columns,group", [(3, 256, 40, 64), (9, 1024, 17, 128), (20, 96, 33, 32), (2, 8192, 16, 256), (20, 2048, 6000, 128)])
def test_int4_gemv_infinities_take_the_weights_signs(pk, device, profile, rows, inner, columns, group):
    """An infinity of every place of a word meets weights of both signs and zeros: the formula's signs and NaNs,
    and the rows beside them keep the values that they have alone."""
    import torch

    rng = np.random.default_rng(31 + inner)
    npd = np.float16 if profile == "fp16" else np.float32
    codes = rng.integers(0, 16, (inner, columns)).astype(np.uint8)
    scales = ((0.5 + rng.random((inner // group, columns))) * 0.05).astype(npd)
    weight = pk.kernels.Int4Weight.from_words(torch.from_numpy(pk.runtime_plan.pack_int4(codes).view(np.int32)).cuda(),
                                              torch.from_numpy(scales).cuda(), inner, group)
    kernel = pk.kernels.Int4GemvKernel.create(device, None, 0, profile)

    def run(a):
        out = torch.zeros((rows, columns), dtype=_dtype(profile), device="cuda")
        kernel.create_dispatch(dict(label="g", a=torch.from_numpy(a).cuda(), weight=weight, output=out, rows=rows)).encode()
        return _np(out)

    a = rng.standard_normal((rows, inner)).astype(npd)
    plain = run(a)
    w = codes.astype(np.float64) - 8.0
    for place in range(8):
        b = a.copy()
        k = int(rng.integers(0, inner // 8)) * 8 + place
        b[1, k] = -np.inf if place % 3 == 0 else np.inf
        if place == 5:
            b[1, (k + 8) % inner] = np.nan
        got = run(b)
        with np.errstate(invalid="ignore"):
            want = np.full(columns, np.nan) if place == 5 else float(b[1, k]) * w[k]
        np.testing.assert_array_equal(got[1], want)
        keep = np.arange(rows) != 1
        np.testing.assert_array_equal(got[keep], plain[keep])


def test_int4_quantized_weight(pk, device):
    """Int4Weight.quantize end to end: the product is that of the rounded weight."""
    import torch

    rng = np.random.default_rng(23)
    w = (rng.standard_normal((640, 72)) * 0.05).astype(np.float32)
    weight = pk.kernels.Int4Weight.quantize(w, 64, "fp16")
    words, scales = pk.runtime_plan.quantize_int4(w, 64, "fp16")
    back = (pk.runtime_plan.unpack_int4(words).astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), 64, axis=0)
    a = rng.standard_normal((3, 640)).astype(np.float16)
    out = torch.zeros((3, 72), dtype=torch.float16, device="cuda")
    pk.kernels.Int4GemvKernel.create(device).create_dispatch(dict(
        label="g", a=torch.from_numpy(a).cuda(), weight=weight, output=out, rows=3)).encode()
    a64 = a.astype(np.float64)
    v, mass = a64 @ back, np.abs(a64) @ np.abs(back)
    assert np.all(np.abs(_np(out) - v) <= (640 / 16 + 64) * 2 * E * mass + 2.0 ** -11 * (np.abs(v) + 1e-3 * mass) + 2.0 ** -25)


# ====================================================================== joint logits

def _joint(pk, device, counts, frames, max_tokens, inner, columns, profile, bias=True, seed=0, big_frame=False):
    import torch

    rng = np.random.default_rng(seed + inner + columns + len(counts))
    npd = np.float16 if profile == "fp16" else np.float32
    batch = len(counts)
    enc = rng.standard_normal((batch, frames, inner)).astype(npd)
    pred = rng.standard_normal((batch, max_tokens, inner)).astype(np.float32)
    at = rng.integers(0, frames, (batch, max_tokens)).astype(np.int32)
    if big_frame:
        at[0, 0] = frames + 9
    w = (rng.standard_normal((inner, columns)) / math.sqrt(inner)).astype(npd)
    b = rng.standard_normal(columns).astype(np.float32) if bias else None
    cu = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    logits = torch.full((batch * max_tokens, columns), SENTINEL, dtype=_dtype(profile), device="cuda")
    rmap = torch.full((batch * max_tokens,), -7, dtype=torch.int32, device="cuda")
    total = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    d = dict(label="joint", encoder_projected=cu(enc), predictor=cu(pred), joint_frames=cu(at),
             counts=cu(np.asarray(counts, np.int32)), weight=cu(w), logits=logits, row_map=rmap, row_count=total,
             batch_size=batch, frames=frames, max_tokens=max_tokens, inner=inner, columns=columns)
    if bias:
        d["bias"] = cu(b)
    pk.kernels.JointLogitsKernel.create(device, None, 0, profile).create_dispatch(d).encode()
    places = [(i, u) for i, n in enumerate(counts) for u in range(min(n, max_tokens))]
    n = len(places)
    assert int(total.item()) == n
    np.testing.assert_array_equal(_np(rmap)[:n], [i * max_tokens + u for i, u in places])
    assert np.all(_np(rmap)[n:] == -7) and np.all(_np(logits)[n:] == np.asarray(SENTINEL, npd))
    if not n:
        return
    i, u = np.array(places).T
    h = np.maximum(enc[i, np.minimum(at[i, u], frames - 1)].astype(np.float64) + pred[i, u], 0.0)
    w64 = w.astype(np.float64)
    v, mass = h @ w64 + (b if bias else 0.0), h @ np.abs(w64)
    # FP16: hidden's rounding, and a step of 2^-23 per product instruction (16 inputs).  FP32: three tf32
    # products a term, each of 8 inputs an instruction; the two low parts are cut at 2^-22 of their value and
    # the product of the two is left out.
    dv = (2.0 ** -11 + (inner / 16 + 8) * 2 * E if profile == "fp16" else 3 * 4 * E + (3 * inner / 8 + 8) * 2 * E) * mass
    dv = dv + 2 * E * np.abs(v)
    err = np.abs(_np(logits)[:n] - v) - (dv + HALF[profile] * (np.abs(v) + dv) + TINY[profile])
    assert np.all(err <= 0), float(err.max())
    device.status()  # no bounded wait ran out


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("counts,frames,max_tokens,inner,columns", [
    ([1], 1, 1, 32, 8), ([61], 188, 256, 640, 1032), ([0, 5, 0, 130, 1], 20, 200, 640, 1032), ([0, 0], 3, 4, 64, 16),
    ([128, 128], 188, 128, 96, 72), ([129, 40, 300], 50, 300, 1280, 264), ([7] * 40, 188, 2048, 640, 1032),
    ([3, 9, 2] * 100, 2, 16, 64, 40), ([300] * 33, 64, 300, 128, 2064),
])
def test_joint_logits(pk, device, profile, counts, frames, max_tokens, inner, columns):
    _joint(pk, device, counts, frames, max_tokens, inner, columns, profile)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
def test_joint_logits_without_bias_and_beyond_its_bounds(pk, device, profile):
    """Counts above max_tokens and frames behind the window are held to their bounds."""
    _joint(pk, device, [40, 3, 99], 6, 24, 160, 48, profile, bias=False, big_frame=True)


# ====================================================================== together, streams, graphs

def _chain(pk, device, profile, seed=0):
    """Norm -> 4-bit projector -> joint -> scores of the tokens and of the durations, as one program; returns
    (dispatches, buffers, inputs in 64 bits)."""
    import torch

    rng = np.random.default_rng(seed)
    npd = np.float16 if profile == "fp16" else np.float32
    dt, K = _dtype(profile), pk.kernels
    batch, tokens, frames, width, columns = 3, 16, 20, 640, 1032
    rows = batch * tokens
    cu = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()  # noqa: E731
    x, f = (rng.standard_normal((rows, width)).astype(npd) for _ in range(2))
    gamma, beta = (1 + 0.1 * rng.standard_normal(width)).astype(np.float32), (0.1 * rng.standard_normal(width)).astype(np.float32)
    w4 = (rng.standard_normal((width, width)) / 25).astype(np.float32)
    enc = rng.standard_normal((batch, frames, width)).astype(npd)
    at = rng.integers(0, frames, (batch, tokens)).astype(np.int32)
    counts = np.array([16, 0, 9], np.int32)
    head = (rng.standard_normal((width, columns)) * 0.1).astype(npd)
    bias = rng.standard_normal(columns).astype(np.float32)
    ids, durations = rng.integers(0, 1025, rows).astype(np.int32), rng.integers(0, 5, rows).astype(np.int32)
    buf = dict(y=torch.zeros((rows, width), dtype=dt, device="cuda"), h=torch.zeros((rows, width), dtype=dt, device="cuda"),
               q=torch.zeros((rows, width), dtype=dt, device="cuda"), p=torch.zeros((rows, width), device="cuda"),
               logits=torch.zeros((rows, columns), dtype=dt, device="cuda"),
               rmap=torch.zeros(rows, dtype=torch.int32, device="cuda"), n=torch.zeros(1, dtype=torch.int32, device="cuda"))
    outs = [{k: torch.full((rows,), SENTINEL, device="cuda") for k in ("log_probs", "entropies")} for _ in range(2)]
    steps = [
        K.ResidualNormKernel.create(device, None, 0, profile).create_dispatch(dict(
            label="norm", input=cu(x), block=cu(f), output=buf["y"], normalized=buf["h"], rows=rows, channels=width,
            pre="layer", pre_gamma=cu(gamma), pre_beta=cu(beta), residual_scale=0.5)),
        K.Int4GemvKernel.create(device, None, 0, profile).create_dispatch(dict(
            label="projector", a=buf["h"], weight=K.Int4Weight.quantize(w4, 64, profile), output=buf["q"], rows=rows)),
        lambda stream=None: buf["p"].copy_(buf["q"]),
        K.JointLogitsKernel.create(device, None, 0, profile).create_dispatch(dict(
            label="joint", encoder_projected=cu(enc), predictor=buf["p"], joint_frames=cu(at), counts=cu(counts),
            weight=cu(head), bias=cu(bias), logits=buf["logits"], row_map=buf["rmap"], row_count=buf["n"],
            batch_size=batch, frames=frames, max_tokens=tokens, inner=width, columns=columns)),
    ]
    kernel = K.TokenScoresKernel.create(device, None, 0, profile)
    for first, n, given, out in ((0, 1025, ids, outs[0]), (1025, 5, durations, outs[1])):
        steps.append(kernel.create_dispatch(dict(
            label="scores", logits=buf["logits"], rows=rows, columns=n, first_column=first, row_stride=columns,
            targets=cu(given), row_count=buf["n"], row_map=buf["rmap"], **out)))
    host = dict(x=x, f=f, gamma=gamma, beta=beta, w4=w4, enc=enc, at=at, counts=counts, head=head, bias=bias, ids=ids,
                durations=durations, tokens=tokens)
    return steps, buf, outs, host


def _run_chain(steps):
    for s in steps:
        s() if callable(s) else s.encode()


def _chain_reference(pk, h, profile):
    c = {k: v.astype(np.float64) if v.dtype.kind == "f" else v for k, v in h.items() if isinstance(v, np.ndarray)}
    y = c["x"] + 0.5 * c["f"]
    n = _norm64(y, "layer", c["gamma"], c["beta"], 1e-5)
    words, scales = pk.runtime_plan.quantize_int4(h["w4"], 64, profile)
    q = n @ ((pk.runtime_plan.unpack_int4(words).astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), 64, axis=0))
    places = [(i, u) for i, k in enumerate(h["counts"]) for u in range(k)]
    rows = np.array([i * h["tokens"] + u for i, u in places])
    i, u = np.array(places).T
    hid = np.maximum(c["enc"][i, h["at"][i, u]] + q[rows], 0.0)
    logits = hid @ c["head"] + c["bias"]
    return rows, [_score_reference(logits[:, a:b], t[rows], 0) for a, b, t in ((0, 1025, h["ids"]), (1025, 1030, h["durations"]))]


def _check_chain(pk, outs, host, profile):
    rows, refs = _chain_reference(pk, host, profile)
    rest = np.setdiff1d(np.arange(48), rows)
    # FP16: y, h, q, hidden and the logits (up to 16 in magnitude: half a step of 2^-8) round once each; the
    # first four move a logit by about 2^-11 of sqrt(640) terms of size 0.1: 4 * 2^-11 * 2.6 and, four deviations
    # out, 0.02.  A log probability then moves by at most twice the largest logit's error, the entropy by
    # that times the spread of the logits (about 8).
    tol = 2 * (0.02 + 2.0 ** -7) if profile == "fp16" else 2 * 2.0 ** -11 * (0.02 + 2.0 ** -7)
    for out, ref in zip(outs, refs):
        got = {k: _np(v) for k, v in out.items()}
        for k in ("log_probs", "entropies"):
            assert np.all(got[k][rest] == SENTINEL)
            assert np.max(np.abs(got[k][rows] - ref[k])) <= tol * (1 if k == "log_probs" else 8), k


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
def test_a_run_of_the_operators(pk, device, profile):
    steps, buf, outs, host = _chain(pk, device, profile)
    _run_chain(steps)
    _check_chain(pk, outs, host, profile)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
def test_a_captured_run_replays(pk, device, profile):
    """The run as a CUDA graph: replayed on new counts, new ids and new inputs it gives what the calls give."""
    import torch

    steps, buf, outs, host = _chain(pk, device, profile, seed=1)
    _run_chain(steps)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _run_chain(steps)
    for out in outs:
        for t in out.values():
            t.fill_(SENTINEL)
    graph.replay()
    _check_chain(pk, outs, host, profile)
    want = [{k: _np(v).copy() for k, v in out.items()} for out in outs]
    graph.replay()
    for out, w in zip(outs, want):
        for k in w:
            np.testing.assert_array_equal(_np(out[k]), w[k])


def test_two_runs_on_two_streams(pk, device):
    """No operator keeps a workspace: two programs run side by side give what each gives alone."""
    import torch

    progs = [_chain(pk, device, "fp16", seed=s) for s in (2, 3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in progs]
    for _ in range(20):
        for (steps, *_), stream in zip(progs, streams):
            with torch.cuda.stream(stream):
                _run_chain(steps)
    torch.cuda.synchronize()
    for _, _, outs, host in progs:
        _check_chain(pk, outs, host, "fp16")


def test_an_explicit_stream_and_a_destroyed_dispatch(pk, device):
    import torch

    x = torch.randn(2, 64, device="cuda")
    s = Scores(pk, device, x, 64, "fp32", top_k=2)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    s(stream)
    stream.synchronize()
    want = Scores(pk, device, x, 64, "fp32", top_k=2)().host()
    for k, v in s.host().items():
        np.testing.assert_array_equal(v, want[k])
    s.call.destroy()
    with pytest.raises(pk.kernels.ParakeetError, match="destroyed"):
        s()
