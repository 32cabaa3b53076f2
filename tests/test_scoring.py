"""CPU-side checks of the scoring operators: what their dispatches and C entry
points refuse, and the 4-bit weight format.  No compute runs here."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest


class _FakeDevice:
    handle = None
    ordinal = 0


def _handle():
    """Stands in for a device handle in calls that are refused before it is read."""
    return ctypes.create_string_buffer(4096)


def _refuse(pk, entry, desc, status, match):
    buf = _handle()
    with pytest.raises(pk.PkError, match=match) as e:
        pk._lib.call(entry, ctypes.cast(buf, ctypes.c_void_p), ctypes.byref(desc), None)
    assert e.value.status == status


# ------------------------------------------------------------------ C entry points

def test_null_arguments(pk):
    lib = pk._lib.load()
    for entry in ("pk_token_scores", "pk_residual_norm", "pk_int4_gemv", "pk_joint_logits"):
        assert getattr(lib, entry)(None, None, None) == -1


P = 1 << 20  # an address that no refused call reads


def _scores(pk, **kw):
    d = dict(precision=0, top_k=4, rows=3, columns=10, row_stride=10, logits=P, targets=P, slots=3, log_probs=P,
             top_ids=P, top_log_probs=P)
    return pk._lib.TokenScoresDesc(**{**d, **kw})


@pytest.mark.parametrize("change,status,match", [
    (dict(logits=None), -1, "null"), (dict(precision=2), -1, "precision"), (dict(rows=0), -2, "rows"),
    (dict(rows=(1 << 30) + 1), -2, "rows"), (dict(columns=0), -2, "columns"), (dict(row_stride=9), -2, "stride"),
    (dict(top_k=33), -2, "top_k"), (dict(top_k=-1), -2, "top_k"), (dict(top_k=11, columns=10), -2, "top_k"),
    (dict(slots=2), -2, "outputs hold"), (dict(targets=None), -1, "target"), (dict(logits=P + 1), -3, "aligned"),
    (dict(log_probs=None, top_ids=None, top_log_probs=None), -1, "without an output"),
])
def test_token_scores_refuses(pk, change, status, match):
    _refuse(pk, "pk_token_scores", _scores(pk, **change), status, match)


def _norm(pk, **kw):
    d = dict(precision=0, post=1, pre=2, rows=4, channels=64, gate_rows=0, residual_scale=1.0, epsilon=1e-5, input=P,
             block=2 * P, post_gamma=P, post_beta=P, pre_gamma=P, output=3 * P, normalized=4 * P)
    return pk._lib.ResidualNormDesc(**{**d, **kw})


@pytest.mark.parametrize("change,status,match", [
    (dict(block=None), -1, "null"), (dict(precision=7), -1, "precision"), (dict(rows=0), -2, "rows"),
    (dict(channels=66), -2, "channels"), (dict(channels=32772), -2, "channels"), (dict(gate_rows=-1), -2, "gate"),
    (dict(post=3), -1, "unknown post"), (dict(post_beta=None), -1, "gamma and beta"),
    (dict(pre_beta=P), -1, "gamma alone"), (dict(pre=0), -1, "no parameters"),
    (dict(pre=0, pre_gamma=None), -1, "belong together"), (dict(normalized=None), -1, "belong together"),
    (dict(normalized=3 * P), -1, "same buffer"), (dict(input=P + 1), -3, "aligned"),
    (dict(output=P + 64), -1, "overlap"), (dict(normalized=2 * P + 128), -1, "overlap"),
    (dict(normalized=3 * P + 256), -1, "overlap"),
])
def test_residual_norm_refuses(pk, change, status, match):
    _refuse(pk, "pk_residual_norm", _norm(pk, **change), status, match)


def _gemv(pk, **kw):
    d = dict(precision=0, rows=2, inner=128, columns=24, group=64, activation=0, residual_scale=1.0, a=P, codes=P,
             scales=P, c=P)
    return pk._lib.Int4GemvDesc(**{**d, **kw})


@pytest.mark.parametrize("change,status,match", [
    (dict(codes=None), -1, "null"), (dict(precision=-1), -1, "precision"), (dict(rows=0), -2, "rows"),
    (dict(rows=65), -2, "rows"), (dict(inner=100), -2, "K%32"), (dict(columns=0), -2, "K%32"),
    (dict(group=48), -3, "groups"), (dict(inner=192, group=128), -3, "groups"), (dict(group=0), -3, "groups"),
    (dict(activation=3), -1, "activation"), (dict(bias=P, residual=P), -4, "bias and residual"),
    (dict(a=P + 8), -3, "aligned"), (dict(codes=P + 4), -3, "aligned"),
])
def test_int4_gemv_refuses(pk, change, status, match):
    _refuse(pk, "pk_int4_gemv", _gemv(pk, **change), status, match)


def _joint(pk, **kw):
    d = dict(precision=0, batch=2, frames=4, max_tokens=8, inner=64, columns=16, encoder_projected=P, predictor=P,
             joint_frames=P, counts=P, weight=P, bias=P, logits=P, row_map=P, row_count=P)
    return pk._lib.JointLogitsDesc(**{**d, **kw})


@pytest.mark.parametrize("change,status,match", [
    (dict(counts=None), -1, "null"), (dict(precision=3), -1, "precision"), (dict(batch=0), -2, "geometry"),
    (dict(frames=0), -2, "geometry"), (dict(max_tokens=0), -2, "geometry"),
    (dict(batch=65535, max_tokens=1 << 20), -2, "geometry"), (dict(inner=48), -2, "joint shape"),
    (dict(columns=12), -2, "joint shape"), (dict(weight=P + 8), -3, "aligned"), (dict(bias=P + 4), -3, "aligned"),
])
def test_joint_logits_refuses(pk, change, status, match):
    _refuse(pk, "pk_joint_logits", _joint(pk, **change), status, match)


SCORES = ("logits", "targets", "row_count", "row_map", "log_probs", "log_sums", "entropies", "top_ids", "top_log_probs")
GEMV = ("a", "codes", "scales", "residual", "c")
JOINT = ("encoder_projected", "predictor", "joint_frames", "counts", "weight", "bias", "logits", "row_map", "row_count")
NORM = ("input", "block", "post_gamma", "post_beta", "pre_gamma", "gate", "output", "normalized")


@pytest.mark.parametrize("entry,make,names,a,b,shift", [
    ("pk_token_scores", _scores, SCORES, "log_probs", "logits", 4),
    ("pk_token_scores", _scores, SCORES, "log_probs", "targets", 0),
    ("pk_token_scores", _scores, SCORES, "top_ids", "top_log_probs", 8),
    ("pk_token_scores", _scores, SCORES, "entropies", "row_map", 8),
    ("pk_token_scores", _scores, SCORES, "log_sums", "row_count", -8),
    ("pk_int4_gemv", _gemv, GEMV, "c", "a", 0),
    ("pk_int4_gemv", _gemv, GEMV, "c", "residual", 2),
    ("pk_int4_gemv", _gemv, GEMV, "c", "codes", 1024),
    ("pk_int4_gemv", _gemv, GEMV, "c", "scales", 0),
    ("pk_joint_logits", _joint, JOINT, "logits", "encoder_projected", 512),
    ("pk_joint_logits", _joint, JOINT, "logits", "predictor", 16),
    ("pk_joint_logits", _joint, JOINT, "row_map", "joint_frames", 0),
    ("pk_joint_logits", _joint, JOINT, "row_count", "counts", 4),
    ("pk_joint_logits", _joint, JOINT, "row_map", "row_count", -4),
    ("pk_residual_norm", _norm, NORM, "output", "pre_gamma", 0),
    ("pk_residual_norm", _norm, NORM, "normalized", "gate", 128),
])
def test_outputs_over_other_buffers_are_refused(pk, entry, make, names, a, b, shift):
    at = {n: (100 + i) * P for i, n in enumerate(names)}
    at[a] = at[b] + shift
    _refuse(pk, entry, make(pk, **at), -1, "overlap")


@pytest.mark.parametrize("entry,make,names,name,by", [
    ("pk_token_scores", _scores, SCORES, "targets", 2), ("pk_token_scores", _scores, SCORES, "top_ids", 1),
    ("pk_token_scores", _scores, SCORES, "row_map", 2), ("pk_int4_gemv", _gemv, GEMV, "c", 1),
    ("pk_int4_gemv", _gemv, GEMV, "scales", 1), ("pk_int4_gemv", _gemv, GEMV, "residual", 1),
    ("pk_joint_logits", _joint, JOINT, "counts", 2), ("pk_joint_logits", _joint, JOINT, "row_count", 2),
    ("pk_joint_logits", _joint, JOINT, "logits", 8), ("pk_residual_norm", _norm, NORM, "gate", 2),
])
def test_buffers_off_their_elements_are_refused(pk, entry, make, names, name, by):
    at = {n: (100 + i) * P for i, n in enumerate(names)}
    at[name] += by
    _refuse(pk, entry, make(pk, **at), -3, "aligned")


def test_token_scores_refuses_sizes_that_no_memory_holds(pk):
    for change in (dict(row_stride=1 << 60), dict(slots=(1 << 32) + 1)):
        _refuse(pk, "pk_token_scores", _scores(pk, **change), -2, "at most")


# ------------------------------------------------------------------ dispatches

def test_dispatches_refuse_shapes_before_buffers(pk):
    K = pk.kernels
    scores = K.TokenScoresKernel.create(_FakeDevice())
    base = dict(label="s", rows=2, columns=10)
    for change, match in ((dict(rows=0), "rows"), (dict(rows=True), "rows"), (dict(columns=0), "columns"),
                          (dict(row_stride=9), "stride"), (dict(first_column=1), "stride"),
                          (dict(top_k=33, columns=64), "top_k"), (dict(top_k=11), "top_k"), (dict(slots=1), "hold")):
        with pytest.raises(K.RangeError, match=match):
            scores.create_dispatch({**base, **change})
    norm = K.ResidualNormKernel.create(_FakeDevice())
    base = dict(label="n", rows=2, channels=64)
    for change, match in ((dict(rows=0), "rows"), (dict(channels=6), "shape"), (dict(channels=40000), "shape"),
                          (dict(gate_rows=-1), "gate_rows")):
        with pytest.raises(K.RangeError, match=match):
            norm.create_dispatch({**base, **change})
    for change, match in ((dict(post="batch"), "unknown post"), (dict(pre="rms"), "gamma alone"),
                          (dict(post_gamma=1), "no parameters"), (dict(normalized=1), "normalized")):
        with pytest.raises(K.ParakeetError, match=match):
            norm.create_dispatch({**base, **change})
    joint = K.JointLogitsKernel.create(_FakeDevice())
    base = dict(label="j", batch_size=1, frames=4, max_tokens=4, inner=64, columns=16)
    for change in (dict(inner=40), dict(columns=20), dict(batch_size=0), dict(frames=-1)):
        with pytest.raises(K.RangeError):
            joint.create_dispatch({**base, **change})


def test_dispatches_refuse_host_buffers_and_unknown_profiles(pk):
    import torch

    K = pk.kernels
    for kernel in (K.TokenScoresKernel, K.ResidualNormKernel, K.Int4GemvKernel, K.JointLogitsKernel):
        with pytest.raises(K.ParakeetError, match="precision"):
            kernel.create(_FakeDevice(), None, 0, "bf16")
    with pytest.raises(K.ParakeetError, match="contiguous tensor on cuda:0"):
        K.TokenScoresKernel.create(_FakeDevice()).create_dispatch(
            dict(label="s", rows=1, columns=4, logits=torch.zeros(4, dtype=torch.float16), log_sums=torch.zeros(1)))
    with pytest.raises(K.ParakeetError, match="needs logits"):
        K.TokenScoresKernel.create(_FakeDevice()).create_dispatch(dict(label="s", rows=1, columns=4))


def test_int4_dispatch_refuses(pk):
    import torch

    K, rp = pk.kernels, pk.runtime_plan
    t = torch.zeros(1024, dtype=torch.float16)

    def weight(**kw):
        w = dict(inner=128, columns=16, group=64, codes=K.GpuTensor("c", "uint32", (128, 16), rp.INT4_TILE_LAYOUT, t),
                 scales=K.GpuTensor("s", "float16", (2, 16), rp.INT4_TILE_SCALE_LAYOUT, t))
        return K.Int4Weight(**{**w, **kw})

    k = K.Int4GemvKernel.create(_FakeDevice())
    base = dict(label="g", a=t, output=t, weight=weight(), rows=1)
    with pytest.raises(K.RangeError, match="rows"):
        k.create_dispatch({**base, "rows": 65})
    for change, match in ((dict(weight=t), "weight format"), (dict(activation="gelu"), "activation"),
                          (dict(weight=weight(codes=K.GpuTensor("c", "uint32", (128, 16), rp.INT4_LAYOUT, t))), "format"),
                          (dict(weight=weight(scales=K.GpuTensor("s", "float32", (2, 16), rp.INT4_TILE_SCALE_LAYOUT,
                                                                 t.float()))), "scales must be"),
                          (dict(bias=t, residual=t), "bias and residual"),
                          (dict(residual_scale=0.5), "residual scale without")):
        with pytest.raises(K.ParakeetError, match=match):
            k.create_dispatch({**base, **change})
    words = torch.zeros((16, 16), dtype=torch.int32)
    with pytest.raises(K.RangeError, match="groups"):
        K.Int4Weight.from_words(words, t[:32].view(2, 16), 128, 48)
    with pytest.raises(K.ParakeetError, match="codes must be"):
        K.Int4Weight.from_words(words[:, :8].contiguous(), t[:32].view(2, 16), 128, 64)
    with pytest.raises(K.ParakeetError, match="scales must be"):
        K.Int4Weight.from_words(words, t[:16].view(1, 16), 128, 64)
    with pytest.raises(K.ParakeetError, match="CUDA"):
        K.Int4Weight.from_words(words, t[:32].view(2, 16), 128, 64)


# ------------------------------------------------------------------ 4-bit format

def test_int4_pack_roundtrip_and_bit_order(pk):
    rp = pk.runtime_plan
    codes = np.random.default_rng(0).integers(0, 16, (64, 24)).astype(np.uint8)
    words = rp.pack_int4(codes)
    assert words.shape == (24, 8)
    np.testing.assert_array_equal(rp.unpack_int4(words), codes)
    one = np.zeros((8, 1), np.uint8)
    one[:, 0] = [1, 2, 3, 4, 5, 6, 7, 8]
    assert int(rp.pack_int4(one)[0, 0]) == 0x87654321
    with pytest.raises(ValueError, match="multiple of 8"):
        rp.pack_int4(codes[:5])
    with pytest.raises(ValueError, match=r"\[0, 16\)"):
        rp.pack_int4(codes + 1)


@pytest.mark.parametrize("precision", ["fp16", "fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_quantization_error(pk, precision, group):
    """|w - (code - 8) scale| is at most half a step, and half of the scale's own rounding for code 1 or 15
    (whose weight is 7 scales before the scale is rounded)."""
    rp = pk.runtime_plan
    w = np.random.default_rng(1).standard_normal((128, 24)).astype(np.float32)
    w[:group, 3] = 0.0
    words, scales = rp.quantize_int4(w, group, precision)
    assert scales.dtype == (np.float16 if precision == "fp16" else np.float32)
    step = np.repeat(scales.astype(np.float64), group, axis=0)
    back = (rp.unpack_int4(words).astype(np.float64) - 8.0) * step
    half = 2.0 ** -11 if precision == "fp16" else 2.0 ** -24
    assert np.all(np.abs(back - w) <= step * (0.5 + 8 * half))
    assert np.all(back[:group, 3] == 0.0)
    for bad in (0, 48, 96):
        with pytest.raises(ValueError, match="groups"):
            rp.quantize_int4(w, bad, precision)


# ------------------------------------------------------------------ trace and engine

def test_trace_and_alternatives_are_refused(pk):
    lib = pk._lib
    desc, trace = lib.TdtDesc(), lib.TdtTrace(P, None)
    buf = _handle()
    for tr in (None, ctypes.byref(trace)):
        with pytest.raises(pk.PkError, match="trace"):
            lib.call("pk_tdt_decode_traced", ctypes.cast(buf, ctypes.c_void_p), ctypes.byref(desc), tr, None)
    for shifted in (lib.TdtTrace(P + 8, P), lib.TdtTrace(P, P + 2)):
        with pytest.raises(pk.PkError, match="aligned"):
            lib.call("pk_tdt_decode_traced", ctypes.cast(buf, ctypes.c_void_p), ctypes.byref(desc), ctypes.byref(shifted), None)
    for k in (-1, 33):
        with pytest.raises(pk.kernels.RangeError, match="alternatives"):
            pk.engine.ParakeetEngine(_FakeDevice(), {}, "fp16", alternatives=k)
