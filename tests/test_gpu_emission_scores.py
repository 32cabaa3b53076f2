"""Scores of the decoder's emissions: the traced decode against the untraced
one and a 64-bit prediction net, and the engine's scores against the joint
computed in 64 bits from that trace."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import cuda, host

pytestmark = pytest.mark.gpu


def _decode(pk, device, enc, lengths, dec, precision, max_tokens, traced, flush=None):
    import torch

    K, (b, t) = pk.kernels, enc.shape[:2]
    u32 = lambda a, d: cuda(np.asarray(np.full(b, d) if a is None else a, np.uint32))  # noqa: E731
    wdtype = "float16" if precision == "fp16" else "float32"
    model = {name: K.GpuTensor(name, wdtype if profiled else "float32", shape, layout, cuda(dec[name]))
             for name, (profiled, shape, layout) in K.TDT_DECODER_TENSORS.items()}
    out = lambda: torch.full((b, max_tokens), 0xEEEE, dtype=torch.int32, device="cuda")  # noqa: E731
    d = dict(encoder_projected=cuda(enc), encoded_lengths=u32(lengths, t), decode_starts=u32(None, 0),
             decode_ends=u32(None, t), flush_finals=u32(flush, 0), tokens=out(), token_frames=out(), token_durations=out(),
             metadata=torch.full((2 * b,), -1, dtype=torch.int32, device="cuda"), batch_size=b, frames=t,
             max_tokens=max_tokens)
    if traced:
        d["trace_predictor"] = torch.full((b, max_tokens, 640), float("nan"), device="cuda")
        d["trace_joint_frames"] = out()
    K.PersistentTdtDecoderKernel.create(device, None, model, precision).create_dispatch(d).encode()
    meta = host(d["metadata"])
    res = dict(tokens=host(d["tokens"]), frames=host(d["token_frames"]), durations=host(d["token_durations"]),
               counts=meta[:b], flags=meta[b:])
    if traced:
        res.update(predictor=host(d["trace_predictor"]), joint_frames=host(d["trace_joint_frames"]))
    return res


def _predictor64(dec, tokens):
    """The prediction net before each of `tokens`, in 64 bits."""
    w = {k: v.astype(np.float64) for k, v in dec.items()}
    sig = lambda v: 1.0 / (1.0 + np.exp(-v))  # noqa: E731
    h, c = [np.zeros(640), np.zeros(640)], [np.zeros(640), np.zeros(640)]
    out = []
    for u in range(len(tokens)):
        x = None if u == 0 else w["decoder.embedding.weight"][tokens[u - 1]]
        for layer in (0, 1):
            m = w[f"decoder.lstm.weight_l{layer}"]
            g = w[f"decoder.lstm.bias_l{layer}"].copy()
            if x is not None:
                g += x @ m[:640]
            if u:
                g += h[layer] @ m[640:]
            i, f, z, o = g[:640], g[640:1280], g[1280:1920], g[1920:]
            c[layer] = sig(f) * c[layer] + sig(i) * np.tanh(z)
            h[layer] = sig(o) * np.tanh(c[layer])
            x = h[layer]
        out.append(h[1] @ w["decoder.decoder_projector.weight"] + w["decoder.decoder_projector.bias"])
    return np.array(out)


def _logits64(enc, res, dec, w):
    n = int(res["counts"][w])
    hidden = np.maximum(enc[w, res["joint_frames"][w, :n]].astype(np.float64) + res["predictor"][w, :n], 0.0)
    return hidden, hidden @ dec["joint.head.weight"].astype(np.float64) + dec["joint.head.bias"]


LENGTHS, FLUSH = [188, 150, 0, 5, 188], [0, 1, 0, 1, 1]


@pytest.mark.parametrize("precision,route", [("fp16", "resident"), ("fp16", "cluster"), ("fp32", "cluster")])
@pytest.mark.parametrize("max_tokens", [400, 7])
def test_traced_decode(pk, device, precision, route, max_tokens):
    dt = np.float16 if precision == "fp16" else np.float32
    enc = np.random.default_rng(31).normal(0, 1, (5, 188, 640)).astype(dt)
    dec = {k: v["data"] for k, v in pk.synthetic.make_decoder(precision, seed=3).items()}
    pk.kernels.set_decoder_route(route)
    try:
        plain = _decode(pk, device, enc, LENGTHS, dec, precision, max_tokens, False, FLUSH)
        res = _decode(pk, device, enc, LENGTHS, dec, precision, max_tokens, True, FLUSH)
        if route == "resident":
            pk.kernels.set_decoder_route("cluster")
            other = _decode(pk, device, enc, LENGTHS, dec, precision, max_tokens, True, FLUSH)
            for w, n in enumerate(res["counts"]):
                np.testing.assert_array_equal(res["predictor"][w, :n], other["predictor"][w, :n])
                np.testing.assert_array_equal(res["joint_frames"][w, :n], other["joint_frames"][w, :n])
    finally:
        pk.kernels.set_decoder_route("auto")
    for key in plain:
        np.testing.assert_array_equal(res[key], plain[key])
    assert res["counts"][2] == 0 and max(res["counts"]) == max_tokens if max_tokens == 7 else sum(res["counts"]) > 50
    for w, n in enumerate(res["counts"]):
        # FP32: rounding errors of a gate's 1280 products are about sqrt(1280) E 13 = 3e-5 (13: their magnitudes'
        # sum); recurrence, second layer and projector multiply that by about 20.  FP16: chains of 640 f16 sums
        # are off by about sqrt(640) 2^-11 of partial sums near 1, 0.012 a gate, and as much further on.
        want = _predictor64(dec, res["tokens"][w, :n])
        if n:
            assert np.abs(res["predictor"][w, :n] - want).max() <= (2e-3 if precision == "fp32" else 0.25)
        # The decoder took the joint's best token and duration: within the error of its own head chains (FP16:
        # 640 f16 sums of partial sums up to about 4, sqrt(640) 2^-11 4 / 2 = 0.025; ten of these).
        _, logits = _logits64(enc, res, dec, w)
        slack = 1e-3 if precision == "fp32" else 0.25
        rows = np.arange(n)
        assert np.all(logits[rows, res["tokens"][w, :n]] >= logits[:, :1025].max(axis=1, initial=-np.inf) - slack)
        assert np.all(logits[rows, 1025 + res["durations"][w, :n]] >= logits[:, 1025:1030].max(axis=1, initial=-np.inf) - slack)


def _log_softmax(x):
    m = x.max(axis=1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(axis=1, keepdims=True))


@pytest.mark.parametrize("precision", ["fp16", "fp32"])
@pytest.mark.parametrize("alternatives", [0, 5])
def test_engine_scores_its_emissions(pk, device, precision, alternatives):
    package = pk.synthetic.make_package(precision, seed=0)
    decoder = pk.synthetic.make_decoder(precision, seed=0)
    package.update(decoder)
    dec = {k: v["data"] for k, v in decoder.items()}
    pcm = pk.synthetic.make_pcm(40.0, seed=9)
    plans = pk.windows.plan_stateless_windows(len(pcm))
    windows = [(pcm[p.source_start_sample:p.source_end_sample], p) for p in plans]
    assert len(windows) >= 3
    plain = pk.engine.ParakeetEngine(device, package, precision, capacity=4)
    try:
        want = plain.transcribe_windows(windows[:3])
        merged = plain.transcribe(pcm)
    finally:
        plain.destroy()
    assert all(r.scores is None for r in want)
    eng = pk.engine.ParakeetEngine(device, package, precision, capacity=4, alternatives=alternatives)
    try:
        for batch in (3, 1, 3):  # the dispatches of a batch size are kept
            got = eng.transcribe_windows(windows[:batch])
            assert [r.tokens for r in got] == [r.tokens for r in want[:batch]]
        projected = host(eng.graph.decoder_input()).reshape(-1, 188, 640)
        predictor, frames = host(eng._scorer._predictor), host(eng._scorer._frames)
        total = 0
        for w, r in enumerate(got):
            n, s = len(r.tokens), r.scores
            total += n
            hidden = np.maximum(projected[w, frames[w, :n]].astype(np.float64) + predictor[w, :n], 0.0)
            head = dec["joint.head.weight"].astype(np.float64)
            logits = hidden @ head + dec["joint.head.bias"]
            # A logit's error: FP16 rounds hidden (2^-11 of each term) and itself; FP32 as in the joint's own test.
            E = 2.0 ** -24
            part = 2.0 ** -11 + 48 * 2 * E if precision == "fp16" else 12 * E + 248 * 2 * E
            half = 2.0 ** -11 if precision == "fp16" else E
            err = (hidden @ np.abs(head)) * part + half * np.abs(logits) + 4 * E * np.abs(logits)
            # A log probability moves by at most twice the largest of its logits' errors, and its own f32 rounding
            # and sums (1025 terms: under 128 E); the entropy, the mean of -log p, by that times 1 + the spread
            # of log p under p, which is below its largest value.
            tokens = np.array([t.token_id for t in r.tokens], int)
            durations = np.array([t.duration_frames for t in r.tokens], int)
            rows = np.arange(n)
            for x, e, ids, got_lp in ((logits[:, :1025], err[:, :1025], tokens, s.token_log_probs),
                                      (logits[:, 1025:1030], err[:, 1025:1030], durations, s.duration_log_probs)):
                lp = _log_softmax(x)
                tol = 2 * e.max(axis=1) + 128 * E * (1 + np.abs(lp).max(axis=1))
                assert np.all(np.abs(got_lp - lp[rows, ids]) <= tol)
            lp = _log_softmax(logits[:, :1025])
            tol = 2 * err[:, :1025].max(axis=1) + 128 * E * (1 + np.abs(lp).max(axis=1))
            entropy = -(np.exp(lp) * lp).sum(axis=1)
            assert np.all(np.abs(s.token_entropies - entropy) <= tol * (1 + np.abs(lp).max(axis=1)))
            assert s.alternatives.shape == s.alternative_log_probs.shape == (n, alternatives)
            if alternatives:
                taken = np.take_along_axis(lp, s.alternatives.astype(int), axis=1)
                assert np.all(np.abs(s.alternative_log_probs - taken) <= tol[:, None])
                best = -np.sort(-lp, axis=1)[:, :alternatives]
                assert np.all(np.abs(s.alternative_log_probs - best) <= 2 * tol[:, None])
                assert np.all(np.diff(s.alternative_log_probs, axis=1) <= 0)
                assert all(len(set(row)) == alternatives for row in s.alternatives)
        assert total > 10
        # Long-form transcription does not score, and is the same.
        assert eng.transcribe(pcm).tokens == merged.tokens
        assert device.status() == 0
    finally:
        eng.destroy()
