"""The scoring operators on numbers far from one: large finite logits.

E = 2^-24 is half a step of f32 arithmetic, relative."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_scoring import E, Scores, _logits, _score_reference

pytestmark = pytest.mark.gpu


# ====================================================================== token scores

MASKS = {"fp16": (-300.0, -1e4, -6e4, -65504.0),
         "fp32": (-300.0, -1e4, -65535.0, -65537.0, -1e5, -1e9, -1e10, -1e20, -1e30, -0.9e37, -1e37, -1.1e37,
                  float(np.finfo(np.float32).min))}
PEAKS = {"fp16": (300.0, 2e4, 65504.0),
         "fp32": (300.0, 65535.0, 65537.0, 1e5, 1e9, 1e10, 1e20, 1e30, 0.9e37, 1e37, 1.1e37, float(np.finfo(np.float32).max) / 2)}


def _wide_rows(rng, columns, profile):
    """Rows with finite masks and peaks of every size, ties of them, values of all sizes and rows about 2^16."""
    dt = np.float16 if profile == "fp16" else np.float32
    base = lambda: _logits(rng, 1, columns, profile)[0].astype(np.float64)  # noqa: E731
    rows = []
    for m in MASKS[profile]:
        for share in (0.5, 0.95):
            x = base()
            x[:int(share * columns)] = m  # a contiguous part: whole warps see nothing else
            rows.append(x)
        x = base()
        x[rng.random(columns) < 0.95] = m
        rows.append(x)
        rows.append(np.full(columns, m))
        x = np.full(columns, m)
        x[columns // 3] = 1.5
        rows.append(x)
        x = np.full(columns, m)
        x[::2] = -np.inf
        rows.append(x)
    for p in PEAKS[profile]:
        x = base()
        x[columns // 5] = p
        rows.append(x)
        x = base()
        x[[columns // 7, columns - 1]] = p  # a tie, in different warps
        rows.append(x)
        x = base()
        x[columns - 1], x[0] = p, 0.9 * p  # two sizes in different warps
        rows.append(x)
        x = base()
        x[0], x[columns - 1] = p, 0.9 * p
        rows.append(x)
    top = 4.0 if profile == "fp16" else 37.0
    for sign in (-1.0, 1.0):
        rows.append(sign * 10.0 ** rng.uniform(-3, top, columns))
        rows.append(sign * np.sort(10.0 ** rng.uniform(-3, top, columns)))
        middle = 60000.0 if profile == "fp16" else 65536.0
        rows.append(sign * middle + base() * (8.0 if profile == "fp16" else 0.5))  # neighbours about 2^16
        rows.append(sign * middle + np.sort(base()) * (8.0 if profile == "fp16" else 0.5))
    return np.array(rows).astype(dt)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,columns,k", [
    (0, 2, 0), (0, 200, 4), (0, 1999, 8), (0, 9001, 5), (2600, 1025, 4), (1300, 9000, 3),
])
def test_token_scores_of_large_finite_logits(pk, device, profile, rows, columns, k):
    """Held by one warp and by several, streamed by one warp and by several (`rows` at least in one call)."""
    x = _wide_rows(np.random.default_rng(71 + columns), columns, profile)
    _check_wide(pk, device, np.resize(x, (max(rows, len(x)), columns)), len(x), columns, k, profile)


@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("columns", [20000, 131075])
def test_token_scores_of_large_finite_logits_over_clusters(pk, device, profile, columns):
    """A row over a cluster of CTAs, held and streamed: three rows a call."""
    x = _wide_rows(np.random.default_rng(72 + columns), columns, profile)
    for r in range(0, len(x), 3):
        _check_wide(pk, device, x[r:r + 3], len(x[r:r + 3]), columns, 4, profile)


def _check_wide(pk, device, x, n, columns, k, profile):
    import torch

    rng = np.random.default_rng(5)
    targets = rng.integers(0, columns, len(x))
    targets[::2] = x[::2].argmax(axis=1)
    got = Scores(pk, device, torch.from_numpy(x).cuda(), columns, profile, torch.from_numpy(targets.astype(np.int32)).cuda(),
                 k)().host()
    got = {name: v[:n].astype(np.float64) for name, v in got.items()}
    ref = _score_reference(x[:n].astype(np.float64) + 0.0, targets[:n], k)
    np.testing.assert_array_equal(got["top_ids"], ref["top_ids"])
    # d = x - m, its product with log2 e and the exponential round at their own sizes: e^d is off by
    # e^d (|d| 3 E + 4 E) at most, of which |d| e^d <= 1/e, so s by under 6 E of itself, beside its sums (a thread's
    # chain of columns / 32 terms at most, and the joins).  log p = d - log s and log sum = m + log s round at their
    # own sizes; no error grows with the logits.
    rel = (columns / 32 + 64) * E
    for name in ("log_probs", "log_sums", "top_log_probs"):
        g, r = got[name], ref[name]
        gone = np.isneginf(r)
        np.testing.assert_array_equal(np.isneginf(g), gone, err_msg=name)
        g, r = np.where(gone, 0.0, g), np.where(gone, 0.0, r)
        bad = ~(np.abs(g - r) <= rel + 4 * E * np.abs(r))
        assert not bad.any(), (name, np.argwhere(bad)[:5].tolist(), g[bad][:5], r[bad][:5])
    # u = sum e^d d, relative to s: its terms' errors are |d| times those of the exponentials, and |u| / s is
    # log s - entropy, below log columns.
    g, r, span = got["entropies"], ref["entropies"], np.log(columns)
    bad = ~(np.abs(g - r) <= rel * (4 + 2 * span))
    assert not bad.any(), ("entropies", np.argwhere(bad)[:5].tolist(), g[bad][:5], r[bad][:5])


# ====================================================================== residual norm

@pytest.mark.parametrize("profile", ["fp16", "fp32"])
@pytest.mark.parametrize("channels", [64, 1000, 1002 * 4, 9000, 32768])
@pytest.mark.parametrize("unaligned", [False, True])
def test_residual_norm_of_rows_whose_squares_leave_f32(pk, device, profile, channels, unaligned):
    """The mean square is infinite where a value is, or where its square is in f32: finite values over its root are
    0, by the formula, an infinite one is NaN, and the rows beside keep what they have alone."""
    import torch

    dt = torch.float16 if profile == "fp16" else torch.float32
    rng = np.random.default_rng(channels)
    x, f = (_logits(rng, 6, channels, profile, 1.0) for _ in range(2))
    f[1, 7] = np.inf
    x[3, 11] = -np.inf
    if profile == "fp32":
        f[4, channels - 1] = 1e20
        x[5, 0] = 1e20
    gamma = rng.uniform(0.5, 1.5, channels).astype(np.float32)

    def run(x, f, post, pre):
        n, skip = x.size, int(unaligned)
        bufs = [torch.zeros(n + skip, dtype=dt, device="cuda") for _ in range(4)]
        for b, v in zip(bufs, (x, f)):
            b[skip:] = torch.from_numpy(v).cuda().flatten()
        beta = torch.full((channels,), 0.25, device="cuda")
        d = dict(label="n", input=bufs[0][skip:], block=bufs[1][skip:], output=bufs[2][skip:], normalized=bufs[3][skip:],
                 rows=x.shape[0], channels=channels, post=post, pre=pre)
        for at, kind in (("post", post), ("pre", pre)):
            d[at + "_gamma"] = torch.from_numpy(gamma).cuda()
            if kind == "layer":
                d[at + "_beta"] = beta
        pk.kernels.ResidualNormKernel.create(device, None, 0, profile).create_dispatch(d).encode()
        torch.cuda.synchronize()
        return [b[skip:].cpu().numpy().reshape(x.shape) for b in bufs[2:]]

    y, h = run(x, f, "rms", "rms")
    rest = lambda row, at: np.delete(row, at)  # noqa: E731
    # Row 1: u is 0 but for the infinite channel, so y is the input itself there; the pre norm of a row with NaN is NaN.
    assert np.isnan(y[1, 7]) and np.array_equal(rest(y[1], 7), rest(x[1], 7)) and np.isnan(h[1]).all()
    # Row 3: y has an infinite channel; h is 0 elsewhere.
    assert np.isneginf(y[3, 11]) and np.isnan(h[3, 11]) and np.isfinite(rest(y[3], 11)).all() and not rest(h[3], 11).any()
    if profile == "fp32":
        assert np.array_equal(y[4], x[4]) and np.isfinite(h[4]).all() and h[4].any()
        assert np.isfinite(y[5]).all() and not h[5].any()
    yl, hl = run(x, f, "layer", "layer")
    assert np.isnan(yl[1]).all() and np.isnan(hl[1]).all()  # inf - inf in the centred values
    if profile == "fp32":
        # The mean of row 4 is 1e20 / channels; what is left of the others' squares does not count.
        assert np.array_equal(yl[4], x[4] + np.float32(0.25)) and np.array_equal(hl[5], np.full(channels, 0.25, np.float32))
    keep = [0, 2] if profile == "fp32" else [0, 2, 4, 5]
    for got, want in zip((y, h, yl, hl), run(x[keep], f[keep], "rms", "rms") + run(x[keep], f[keep], "layer", "layer")):
        np.testing.assert_array_equal(got[keep], want)


# ====================================================================== int4 products

# mma.sync (one and two column tiles, four in two passes) and tcgen05 (16 and 32 columns, groups of every kind).
@pytest.mark.parametrize("rows,inner,columns,group", [
    (1, 640, 640, 64), (5, 512, 48, 128), (12, 1024, 200, 32), (17, 640, 19000, 64), (10, 4096, 6000, 128),
    (40, 1056, 12005, 32),
])
@pytest.mark.parametrize("inputs,weights", [(1e-34, 1.0), (1e-37, 1.0), (1e-20, 1e-17), (1e-38, 1e3), (1e35, 1.0), (1e37, 1e-4),
                                            (1e30, 1e6), (1.0, 1e-30), (1.0, 1e33)])
def test_int4_gemv_of_small_and_large_numbers(pk, device, rows, inner, columns, group, inputs, weights):
    """FP32 inputs and scales near the ends of the type: as near to the formula as those near one, as far as f32
    has numbers for the products."""
    import torch

    rng = np.random.default_rng(rows + inner)
    codes = rng.integers(0, 16, (inner, columns)).astype(np.uint8)
    scales = ((0.5 + rng.random((inner // group, columns))) * 0.05 * weights).astype(np.float32)
    a = (rng.standard_normal((rows, inner)) * inputs).astype(np.float32)
    out = torch.zeros((rows, columns), device="cuda")
    weight = pk.kernels.Int4Weight.from_words(torch.from_numpy(pk.runtime_plan.pack_int4(codes).view(np.int32)).cuda(),
                                              torch.from_numpy(scales).cuda(), inner, group)
    pk.kernels.Int4GemvKernel.create(device, None, 0, "fp32").create_dispatch(dict(
        label="g", a=torch.from_numpy(a).cuda(), weight=weight, output=out, rows=rows)).encode()
    got = out.double().cpu().numpy()
    w = (codes.astype(np.float64) - 8.0) * np.repeat(scales.astype(np.float64), group, axis=0)
    a64 = a.astype(np.float64)
    v, mass = a64 @ w, np.abs(a64) @ np.abs(w)
    assert np.abs(v).max() < 1e38  # sums of terms of both signs: none on the way leaves f32
    # f32 accumulation, up to one step (2^-23) per product instruction and join; inputs as two f16 parts lose at most
    # 2^-22 of each and, relative to a tile's largest, 2^-38.  A product instruction's or group's sum below the
    # smallest numbers is off by half a step of 2^-149.
    dv = (inner / 16 + 64) * 2 * E * mass + 2.0 ** -22 * mass + 2.0 ** -38 * np.abs(a64).max() * np.abs(w).sum(axis=0)
    dv = dv + (inner / 16 + 64) * 2.0 ** -150
    err = np.abs(got - v) - dv * (1 + E) - E * np.abs(v)
    assert np.all(err <= 0), (float(err.max()), float(np.abs(got - v).max()), float(np.abs(v).max()))


# ====================================================================== optional operands

def test_token_scores_take_none_for_what_is_not_wanted(pk, device):
    """None stands for an output or operand that is left out, as the key's absence does."""
    import torch

    x = torch.randn(3, 100, device="cuda")
    kernel = pk.kernels.TokenScoresKernel.create(device, None, 0, "fp32")
    outs = [torch.zeros(3, device="cuda") for _ in range(2)]
    left_out = dict(log_probs=None, targets=None, entropies=None, top_ids=None, top_log_probs=None, row_count=None, row_map=None)
    for out, extra in zip(outs, ({}, left_out)):
        kernel.create_dispatch(dict(label="s", logits=x, rows=3, columns=100, log_sums=out, **extra)).encode()
    torch.cuda.synchronize()
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    with pytest.raises(pk.kernels.ParakeetError, match="needs targets"):
        kernel.create_dispatch(dict(label="s", logits=x, rows=3, columns=100, log_probs=outs[0], targets=None))
    with pytest.raises(pk.kernels.RangeError, match="outputs hold"):
        kernel.create_dispatch(dict(label="s", logits=x, rows=3, columns=100, log_sums=outs[0], slots=2, row_map=None))
