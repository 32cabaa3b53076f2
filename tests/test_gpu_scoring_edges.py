"""The scoring operators at the ends of their ranges: offsets past 32 bits, first calls inside a capture, one
dispatch on two streams, another thread."""
from __future__ import annotations

import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("channels,rows", [(32768, (1 << 16) + 5), (4096, (1 << 19) + 3)])
def test_residual_norm_offsets_past_32_bits(pk, device, channels, rows):
    """More than 2^31 elements: the last rows against the formula, both ways to split rows over threads."""
    import torch

    half = dict(dtype=torch.float16, device="cuda")
    x, h = (torch.zeros((rows, channels), **half) for _ in range(2))
    f = torch.randn((rows, channels), **half)
    gamma = torch.rand(channels, device="cuda") + 0.5
    last = f[-4:].double().cpu().numpy()
    pk.kernels.ResidualNormKernel.create(device).create_dispatch(dict(
        label="n", input=x, block=f, output=x, normalized=h, rows=rows, channels=channels, pre="rms", pre_gamma=gamma,
        residual_scale=0.5)).encode()
    y = 0.5 * last
    want = y / np.sqrt((y * y).mean(axis=1, keepdims=True) + 1e-5) * gamma.double().cpu().numpy()
    assert np.array_equal(x[-4:].double().cpu().numpy(), y.astype(np.float16).astype(np.float64))  # one rounding
    # h: one rounding (2^-11) and an f32 sum of squares, at most 200 roundings deep, under a root: 100 * 2^-24.
    got = h[-4:].double().cpu().numpy()
    assert np.all(np.abs(got - want) <= (2.0 ** -11 + 1e-5) * np.abs(want) + 2.0 ** -25)
    assert int(torch.count_nonzero(h.abs().amax(dim=1) == 0)) == 0  # every row was written


def test_joint_logits_offsets_past_32_bits(pk, device):
    """2^18 + 5 rows of 8192 columns, ragged: the last rows against the formula."""
    import torch

    batch, tokens, inner, columns, frames = 257, 1024, 32, 8192, 3
    counts = torch.full((batch,), tokens, dtype=torch.int32, device="cuda")
    counts[-1] = 5
    total = (batch - 1) * tokens + 5
    enc = torch.randn((batch, frames, inner), device="cuda").half()
    pred = torch.randn((batch, tokens, inner), device="cuda")
    at = torch.randint(0, frames, (batch, tokens), dtype=torch.int32, device="cuda")
    w = torch.randn((inner, columns), device="cuda").half()
    logits = torch.empty((batch * tokens, columns), dtype=torch.float16, device="cuda")
    logits[total:] = -7.0
    rmap = torch.full((batch * tokens,), -1, dtype=torch.int32, device="cuda")
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    pk.kernels.JointLogitsKernel.create(device).create_dispatch(dict(
        label="j", encoder_projected=enc, predictor=pred, joint_frames=at, counts=counts, weight=w, logits=logits,
        row_map=rmap, row_count=n, batch_size=batch, frames=frames, max_tokens=tokens, inner=inner, columns=columns)).encode()
    assert int(n) == total and bool((logits[total:] == -7.0).all()) and bool((rmap[total:] == -1).all())
    assert torch.equal(rmap[:total], torch.arange(total, dtype=torch.int32, device="cuda"))
    rows = torch.arange(total - 100, total, device="cuda")
    win, u = rows // tokens, rows % tokens
    hidden = (enc[win, at[win, u].long()].double() + pred[win, u].double()).clamp(min=0)
    want, mass = hidden @ w.double(), hidden @ w.double().abs()
    got = logits[rows].double()
    # hidden rounds once (2^-11), an f32 sum of 32 products, the logit rounds once.
    dv = (2.0 ** -11 + 32 * 2.0 ** -23) * mass
    assert bool(((got - want).abs() <= dv + 2.0 ** -11 * (want.abs() + dv) + 2.0 ** -25).all())


def test_int4_gemv_codes_past_32_bits(pk, device):
    """2^22 outputs of 4096 inputs, 8 GB of codes: zero weights but for the last tile of outputs."""
    import torch

    inner, columns, group = 4096, 1 << 22, 128
    K, rp = pk.kernels, pk.runtime_plan
    rng = np.random.default_rng(41)
    last = rng.integers(0, 16, (inner, 16)).astype(np.uint8)
    scales = ((0.5 + rng.random((inner // group, 16))) * 0.05).astype(np.float16)
    tile = K.Int4Weight.from_words(torch.from_numpy(rp.pack_int4(last).view(np.int32)).cuda(),
                                   torch.from_numpy(scales).cuda(), inner, group)
    codes = torch.full((columns * inner // 8,), -0x77777778, dtype=torch.int32, device="cuda")
    laid = torch.ones((columns * inner // group,), dtype=torch.float16, device="cuda")
    codes[-tile.codes.tensor.numel():] = tile.codes.tensor
    laid[-tile.scales.tensor.numel():] = tile.scales.tensor
    weight = K.Int4Weight(inner, columns, group, K.GpuTensor("c", "uint32", (inner, columns), rp.INT4_TILE_LAYOUT, codes),
                          K.GpuTensor("s", "float16", (inner // group, columns), rp.INT4_TILE_SCALE_LAYOUT, laid))
    for rows in (1, 12, 64):
        a = rng.standard_normal((rows, inner)).astype(np.float16)
        out = torch.full((rows, columns), 3.0, dtype=torch.float16, device="cuda")
        K.Int4GemvKernel.create(device).create_dispatch(dict(
            label="g", a=torch.from_numpy(a).cuda(), weight=weight, output=out, rows=rows)).encode()
        # A weight of zero is code 8: (64 + 8) x - 72 x in f32, up to the rounding of sums of 64 times the inputs.
        slack = (inner / 16 + 64) * 2.0 ** -23 * 144 * float(np.abs(a.astype(np.float64)).sum(axis=1).max())
        assert float(out[:, :-16].abs().max()) <= slack + 2.0 ** -25
        w = (last.astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), group, axis=0)
        a64 = a.astype(np.float64)
        v, mass = a64 @ w, np.abs(a64) @ np.abs(w)
        dv = (inner / 16 + 64) * 2.0 ** -23 * mass
        got = out[:, -16:].double().cpu().numpy()
        assert np.all(np.abs(got - v) <= dv + 2.0 ** -11 * (np.abs(v) + dv) + 2.0 ** -25)


FIRST = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import __graft_entry__, torch
pk = __graft_entry__.load()
import test_gpu_scoring as t
device = pk.kernels.Device(0)
for profile in ("fp16", "fp32"):
    steps, buf, outs, host = t._chain(pk, device, profile, seed=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t._run_chain(steps)
    graph.replay()
    t._check_chain(pk, outs, host, profile)
    del graph
device.close()
print("captured first")
"""


def test_first_calls_in_a_capture():
    """A process whose first calls are captured: what a first call sets up does not break the capture."""
    tests = Path(__file__).resolve().parent
    out = subprocess.run([sys.executable, "-c", FIRST.format(root=str(tests.parent), tests=str(tests))], text=True,
                         capture_output=True, timeout=600)
    assert out.returncode == 0 and "captured first" in out.stdout, out.stdout[-2000:] + out.stderr[-2000:]


def test_one_dispatch_on_two_streams(pk, device):
    """The same dispatches of fixed inputs, queued on two streams at once from two threads: every launch writes the
    same values, so the outputs are those of one call."""
    import torch

    import test_gpu_scoring as t

    steps, buf, outs, host = t._chain(pk, device, "fp16", seed=5)
    steps = [steps[0], steps[1]]  # the norm and the product: each writes what no other step of the other stream reads
    for s in steps:
        s.encode()
    torch.cuda.synchronize()
    want = [buf[k].clone() for k in ("y", "h", "q")]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def run(stream):
        for _ in range(50):
            for s in steps:
                s.encode(stream)

    threads = [threading.Thread(target=run, args=(s,)) for s in streams]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    for k, w in zip(("y", "h", "q"), want):
        assert torch.equal(buf[k], w)


def test_scores_repeat_while_their_graph_replays_elsewhere(pk, device):
    """Two captured graphs of the same operators, replayed side by side on two streams."""
    import torch

    import test_gpu_scoring as t

    progs = [t._chain(pk, device, "fp32", seed=s) for s in (6, 7)]
    graphs = []
    for steps, *_ in progs:
        t._run_chain(steps)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            t._run_chain(steps)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, _, outs, host in progs:
        t._check_chain(pk, outs, host, "fp32")


def test_int4_gemv_repeats_bit_for_bit_on_streams_and_in_graphs(pk, device):
    """The tcgen05 route (32 columns, 32 tiles per SM) on two streams at once and replayed: always the same bits."""
    import torch

    rng = np.random.default_rng(51)
    inner, columns, group = 4096, 16384, 128
    K = pk.kernels
    weight = K.Int4Weight.quantize((rng.standard_normal((inner, columns)) * 0.02).astype(np.float32), group, "fp16")
    a = torch.randn((32, inner), device="cuda").half()
    outs = [torch.zeros((32, columns), dtype=torch.float16, device="cuda") for _ in range(3)]
    calls = [K.Int4GemvKernel.create(device).create_dispatch(dict(label="g", a=a, weight=weight, output=o, rows=32)) for o in outs]
    calls[0].encode()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for c, s in zip(calls[1:], streams):
            c.encode(s)
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls[1].encode()
        calls[2].encode()
    for o in outs[1:]:
        o.zero_()
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    device.status()
