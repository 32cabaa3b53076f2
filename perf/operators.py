"""The scoring operators' cases: what each computes in its plain form, and the framework's calls.

A decoder's last steps, from a block's output to a scored answer:

* ``residual_norm``: the norm after a block, its gate and residual scale, the residual sum and
  the next block's norm in one operator;
* ``int4_gemv``: a few rows times a matrix held in 4 bits with a scale per group of inputs;
* ``joint_logits``: the transducer's joint over the emitted tokens of a batch of windows;
* ``token_scores``: log probability of a given token, log of the normaliser, entropy and the
  best alternatives of every row of logits.

``run`` computes them in elementary torch operations where ``own`` is false, and calls the
framework where it is true.  Inputs are synthetic.
"""
import math

import torch

own = False
EPSILON = 1e-5
DTYPES = {"fp16": torch.float16, "fp32": torch.float32}
_devices = {}


def _framework():
    import __graft_entry__

    pk = __graft_entry__.load()
    if "device" not in _devices:
        _devices["device"] = pk.kernels.Device(0)
    return pk.kernels, _devices["device"]


# ------------------------------------------------------------------------------- cases

def listed():
    token = dict(op="token_scores")
    norm = dict(op="residual_norm")
    gemv = dict(op="int4_gemv")
    joint = dict(op="joint_logits", inner=640, columns=1032)
    return [
        # One step of one stream: the answer's probability with a mask on half of the vocabulary.
        dict(token, name="scores 1x32000 fp16", rows=1, columns=32000, stride=32000, top_k=8, profile="fp16",
             masked=0.5),
        # The confidences of a batch of 32 windows: 1025 token columns of the joint's padded 1032.
        dict(token, name="scores 1953x1025 fp32", rows=1953, columns=1025, stride=1032, top_k=4, profile="fp32",
             masked=0.0),
        # Rescoring a long text with a large, odd vocabulary.
        dict(token, name="scores 4096x50257 fp16", rows=4096, columns=50257, stride=50264, top_k=8, profile="fp16",
             masked=0.01),
        # One token between two blocks of the predictor's width.
        dict(norm, name="norm 1x640 fp16", rows=1, channels=640, post="layer", pre="layer", gate="none",
             gate_rows=0, scale=0.5, profile="fp16"),
        # 32 windows of 188 frames between two Conformer blocks, a learned gate per channel, half residual.
        dict(norm, name="norm 6016x1024 fp16", rows=6016, channels=1024, post="layer", pre="layer", gate="channel",
             gate_rows=0, scale=0.5, profile="fp16"),
        # A long batch between two wide blocks, a gate per sequence and channel, in 32 bits.
        dict(norm, name="norm 16384x4096 fp32", rows=16384, channels=4096, post="rms", pre="rms", gate="group",
             gate_rows=2048, scale=1.0, profile="fp32"),
        # The predictor's projector for one stream: latency.
        dict(gemv, name="int4 1x640x640 fp16", rows=1, inner=640, columns=640, group=64, epilogue="bias",
             profile="fp16"),
        # One token through a wide expanding layer.
        dict(gemv, name="int4 1x4096x16384 fp16", rows=1, inner=4096, columns=16384, group=128, epilogue="silu",
             profile="fp16"),
        # Sixteen streams through a vocabulary-sized product, in 32 bits.
        dict(gemv, name="int4 16x4096x65536 fp32", rows=16, inner=4096, columns=65536, group=128, epilogue="none",
             profile="fp32"),
        # One window's emissions.
        dict(joint, name="joint 1 window fp16", batch=1, frames=188, max_tokens=256, tokens=61, profile="fp16"),
        # A batch of 32 windows.
        dict(joint, name="joint 32 windows fp16", batch=32, frames=188, max_tokens=256, tokens=61, profile="fp16"),
        # The largest batch, dense speech, in 32 bits.
        dict(joint, name="joint 40 windows fp32", batch=40, frames=188, max_tokens=256, tokens=110, profile="fp32"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["token_scores", "residual_norm", "int4_gemv", "joint_logits"])
    profile = rng.choice(["fp16", "fp32"])
    if op == "token_scores":
        columns = _log_int(rng, 5, 131072)
        rows = min(_log_int(rng, 1, 16384), max(1, 100_000_000 // columns))
        return dict(op=op, rows=rows, columns=columns, stride=columns + rng.choice([0, 0, 1, 7, 8]),
                    top_k=min(columns, rng.choice([0, 1, 4, 5, 8, 16, 32])), profile=profile,
                    masked=rng.choice([0.0, 0.0, 0.1, 0.9]))
    if op == "residual_norm":
        channels = 4 * _log_int(rng, 16, 2048)
        rows = min(_log_int(rng, 1, 32768), max(1, 60_000_000 // channels))
        gate = rng.choice(["none", "channel", "group"])
        return dict(op=op, rows=rows, channels=channels, post=rng.choice(["none", "layer", "rms"]),
                    pre=rng.choice(["none", "layer", "rms"]), gate=gate,
                    gate_rows=_log_int(rng, 1, rows) if gate == "group" else 0,
                    scale=rng.choice([0.5, 1.0, 0.25]), profile=profile)
    if op == "int4_gemv":
        group = rng.choice([32, 64, 128, 256])
        inner = group * max(1, _log_int(rng, 64, 8192) // group)
        columns = 8 * min(_log_int(rng, 2, 8192), max(1, 200_000_000 // (8 * inner)))
        return dict(op=op, rows=_log_int(rng, 1, 64), inner=inner, columns=columns, group=group,
                    epilogue=rng.choice(["none", "bias", "silu", "relu", "residual"]), profile=profile)
    max_tokens = _log_int(rng, 8, 512)
    return dict(op=op, inner=32 * rng.randint(4, 40), columns=8 * rng.randint(8, 258), batch=rng.randint(1, 40),
                frames=rng.randint(1, 188), max_tokens=max_tokens, tokens=rng.randint(2, min(max_tokens, 110)),
                profile=profile)


# ------------------------------------------------------------------------------- inputs

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["profile"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std + mean

    def whole(low, high, *shape, dtype=torch.int32):
        return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.int64).to(dtype)

    s = {"case": case}
    if case["op"] == "token_scores":
        rows, columns = case["rows"], case["columns"]
        logits = normal(rows, case["stride"], std=2.5)
        s["targets"] = whole(0, columns, rows)
        # Most given tokens are likely ones.
        at = s["targets"].to(torch.int64).unsqueeze(1)
        logits.scatter_add_(1, at, 6.0 + 3.0 * normal(rows, 1))
        if case["masked"]:
            gone = torch.rand(columns, generator=gen, device="cuda") < case["masked"]
            logits[:, :columns][:, gone] = -math.inf
        s["logits"] = logits.to(dtype)
    elif case["op"] == "residual_norm":
        rows, channels = case["rows"], case["channels"]
        s["input"] = normal(rows, channels, std=2.0).to(dtype)
        s["block"] = normal(rows, channels, std=1.5, mean=0.1).to(dtype)
        for at in ("post", "pre"):
            if case[at] != "none":
                s[at + "_gamma"] = normal(channels, std=0.2, mean=1.0)
            if case[at] == "layer":
                s[at + "_beta"] = normal(channels, std=0.2)
        if case["gate"] != "none":
            groups = 1 if case["gate"] == "channel" else -(-rows // case["gate_rows"])
            s["gate"] = normal(groups, channels, std=0.3, mean=0.7)
    elif case["op"] == "int4_gemv":
        rows, inner, columns, group = case["rows"], case["inner"], case["columns"], case["group"]
        s["a"] = normal(rows, inner).to(dtype)
        # Eight codes to a word, inputs in increasing order from the lowest bits: [columns, inner / 8].
        s["words"] = whole(-2 ** 31, 2 ** 31, columns, inner // 8)
        s["scales"] = ((0.5 + torch.rand(inner // group, columns, generator=gen, device="cuda"))
                       * (0.25 / math.sqrt(inner))).to(dtype)
        if case["epilogue"] != "none":
            s["bias"] = None if case["epilogue"] == "residual" else normal(columns)
        if case["epilogue"] == "residual":
            s["residual"] = normal(rows, columns).to(dtype)
    else:
        batch, frames, most = case["batch"], case["frames"], case["max_tokens"]
        inner, columns = case["inner"], case["columns"]
        s["encoder"] = normal(batch, frames, inner).to(dtype)
        s["predictor"] = normal(batch, most, inner)
        s["joint_frames"] = whole(0, frames, batch, most)
        # Half as many tokens to half as many more, windows of silence among them, in any order.
        window = torch.arange(batch, device="cuda")
        counts = (case["tokens"] * (50 + 37 * window % 101) // 100).clamp(1, most)
        counts[1::5] = 0
        order = torch.randperm(batch, generator=gen, device="cuda")
        s["counts"] = counts[order].to(torch.int32)
        s["weight"] = normal(inner, columns, std=2.0 / math.sqrt(inner)).to(dtype)
        s["bias"] = normal(columns, std=0.5)
        s["total"] = int(s["counts"].sum())
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        kernels, device = _framework()
        dtype = DTYPES[case["profile"]]
        if case["op"] == "token_scores":
            rows, k = case["rows"], case["top_k"]
            f32 = dict(dtype=torch.float32, device="cuda")
            s["out"] = dict(log_probs=torch.empty(rows, **f32), log_sums=torch.empty(rows, **f32),
                            entropies=torch.empty(rows, **f32),
                            top_ids=torch.empty((rows, k), dtype=torch.int32, device="cuda"),
                            top_log_probs=torch.empty((rows, k), **f32))
            kernel = kernels.TokenScoresKernel.create(device, None, 0, case["profile"])
            s["call"] = kernel.create_dispatch(dict(
                label="scores", logits=s["logits"], targets=s["targets"], rows=rows, columns=case["columns"],
                row_stride=case["stride"], top_k=k, **s["out"]))
        elif case["op"] == "residual_norm":
            shape = (case["rows"], case["channels"])
            s["out"] = dict(output=torch.empty(shape, dtype=dtype, device="cuda"))
            if case["pre"] != "none":
                s["out"]["normalized"] = torch.empty(shape, dtype=dtype, device="cuda")
            kernel = kernels.ResidualNormKernel.create(device, None, 0, case["profile"])
            given = {n: s[n] for n in ("post_gamma", "post_beta", "pre_gamma", "pre_beta", "gate") if n in s}
            s["call"] = kernel.create_dispatch(dict(
                label="norm", input=s["input"], block=s["block"], rows=case["rows"], channels=case["channels"],
                post=case["post"], pre=case["pre"], gate_rows=case["gate_rows"], residual_scale=case["scale"],
                epsilon=EPSILON, **given, **s["out"]))
        elif case["op"] == "int4_gemv":
            s["out"] = dict(output=torch.empty((case["rows"], case["columns"]), dtype=dtype, device="cuda"))
            weight = kernels.Int4Weight.from_words(s["words"], s["scales"], case["inner"], case["group"])
            kernel = kernels.Int4GemvKernel.create(device, None, 0, case["profile"])
            given = {n: s[n] for n in ("bias", "residual") if s.get(n) is not None}
            if "residual" in given:
                given["residual_scale"] = 0.5
            s["call"] = kernel.create_dispatch(dict(
                label="int4", a=s["a"], weight=weight, rows=case["rows"],
                activation=case["epilogue"] if case["epilogue"] in ("silu", "relu") else "none", **given,
                **s["out"]))
        else:
            rows = case["batch"] * case["max_tokens"]
            s["out"] = dict(logits=torch.empty((rows, case["columns"]), dtype=dtype, device="cuda"),
                            row_map=torch.empty(rows, dtype=torch.int32, device="cuda"),
                            row_count=torch.empty(1, dtype=torch.int32, device="cuda"))
            kernel = kernels.JointLogitsKernel.create(device, None, 0, case["profile"])
            s["call"] = kernel.create_dispatch(dict(
                label="joint", encoder_projected=s["encoder"], predictor=s["predictor"],
                joint_frames=s["joint_frames"], counts=s["counts"], weight=s["weight"], bias=s["bias"],
                batch_size=case["batch"], frames=case["frames"], max_tokens=case["max_tokens"],
                inner=case["inner"], columns=case["columns"], **s["out"]))
    return s


# ------------------------------------------------------------------------------- plain forms

def _scores(s):
    case = s["case"]
    columns, k = case["columns"], case["top_k"]
    x = s["logits"][:, :columns].float() + 0.0  # one zero: -0 ranks as 0
    top = x.max(dim=1, keepdim=True).values
    # A row whose mask leaves nothing: every probability is 0, the entropy too.
    left = top > -math.inf
    away = torch.where(left, x - top, -math.inf)
    e = torch.exp(away)
    total = e.sum(dim=1, keepdim=True)
    log_total = torch.where(left, torch.log(total), 0.0)
    # Masked columns have no share: 0 times -inf is 0 here.
    share = torch.where(e > 0, e * away, torch.zeros((), device=x.device))
    entropies = (log_total - share.sum(dim=1, keepdim=True) / torch.where(left, total, 1.0)).squeeze(1)
    given = away.gather(1, s["targets"].to(torch.int64).unsqueeze(1))
    # A row's order by value, then by the lower index: one whole number that sorts so.
    bits = x.view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    order = order * 2 ** 20 + (2 ** 20 - 1 - torch.arange(columns, device=x.device))
    ids = torch.topk(order, k, dim=1).indices
    return dict(log_probs=(given - log_total).squeeze(1), log_sums=(top + log_total).squeeze(1),
                entropies=entropies, top_ids=ids.to(torch.int32), top_log_probs=away.gather(1, ids) - log_total)


def _normed(v, kind, gamma, beta):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPSILON) * gamma
    return v + beta if kind == "layer" else v


def _residual_norm(s):
    case = s["case"]
    dtype = DTYPES[case["profile"]]
    u = _normed(s["block"].float(), case["post"], s.get("post_gamma"), s.get("post_beta"))
    if case["gate"] == "channel":
        u = u * s["gate"]
    elif case["gate"] == "group":
        u = u * s["gate"].repeat_interleave(case["gate_rows"], dim=0)[: case["rows"]]
    y = s["input"].float() + case["scale"] * u
    out = dict(output=y.to(dtype))
    if case["pre"] != "none":
        out["normalized"] = _normed(y, case["pre"], s.get("pre_gamma"), s.get("pre_beta")).to(dtype)
    return out


def _int4_gemv(s):
    case = s["case"]
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    codes = ((s["words"].unsqueeze(2) >> shifts) & 15).reshape(case["columns"], case["inner"])
    weight = (codes - 8).float() * s["scales"].float().t().repeat_interleave(case["group"], dim=1)
    y = s["a"].float() @ weight.t()
    if case["epilogue"] == "residual":
        y = s["residual"].float() + 0.5 * y
    elif case["epilogue"] != "none":
        y = y + s["bias"]
        if case["epilogue"] == "silu":
            y = y / (1.0 + torch.exp(-y))
        elif case["epilogue"] == "relu":
            y = y.clamp_min(0.0)
    return dict(output=y.to(DTYPES[case["profile"]]))


def _joint_logits(s):
    case = s["case"]
    live = torch.arange(case["max_tokens"], device="cuda") < s["counts"].unsqueeze(1)
    window, token = live.nonzero(as_tuple=True)
    frame = s["joint_frames"][window, token].to(torch.int64)
    hidden = (s["encoder"][window, frame].float() + s["predictor"][window, token]).clamp_min(0.0)
    logits = hidden @ s["weight"].float() + s["bias"]
    return dict(logits=logits.to(DTYPES[case["profile"]]),
                row_map=(window * case["max_tokens"] + token).to(torch.int32),
                row_count=s["counts"].sum(dtype=torch.int32).reshape(1))


def run(s):
    op = s["case"]["op"]
    if own:
        s["call"].encode()
        if op == "joint_logits":  # rows behind the last window's are not written
            total = s["total"]
            return dict(logits=s["out"]["logits"][:total], row_map=s["out"]["row_map"][:total],
                        row_count=s["out"]["row_count"])
        return s["out"]
    if op == "token_scores":
        return _scores(s)
    if op == "residual_norm":
        return _residual_norm(s)
    if op == "int4_gemv":
        return _int4_gemv(s)
    return _joint_logits(s)


# ------------------------------------------------------------------------------- work and definitions

def work(case):
    size = 2 if case["profile"] == "fp16" else 4
    if case["op"] == "token_scores":
        rows, columns = case["rows"], case["columns"]
        return {"bytes": rows * (columns * size + 4 + 12 + 8 * case["top_k"]), "flops": rows * columns * 5}
    if case["op"] == "residual_norm":
        rows, channels = case["rows"], case["channels"]
        streams = 3 + (case["pre"] != "none")
        groups = {"none": 0, "channel": 1}.get(case["gate"], -(-rows // max(1, case["gate_rows"])))
        params = sum({"none": 0, "rms": 1, "layer": 2}[case[at]] for at in ("post", "pre")) + groups
        return {"bytes": streams * rows * channels * size + params * channels * 4, "flops": rows * channels * 14}
    if case["op"] == "int4_gemv":
        rows, inner, columns = case["rows"], case["inner"], case["columns"]
        params = inner * columns // 2 + inner // case["group"] * columns * size
        extra = columns * 4 if case["epilogue"] in ("bias", "silu", "relu") else 0
        extra += rows * columns * size if case["epilogue"] == "residual" else 0
        return {"bytes": params + extra + rows * (inner + columns) * size, "flops": 2 * rows * inner * columns}
    inner, columns = case["inner"], case["columns"]
    rows = max(1, case["batch"] * case["tokens"])
    # Several tokens may read one frame: each frame that is read counts once.
    frames = min(rows, case["batch"] * case["frames"])
    read = frames * inner * size + rows * (inner * 4 + 4) + inner * columns * size + columns * 4 + case["batch"] * 4
    return {"bytes": read + rows * (columns * size + 4), "flops": 2 * rows * inner * columns}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "token_scores":
        parts = []
        for at in range(0, case["rows"], 512):
            x = s["logits"][at:at + 512, :case["columns"]].double()
            log_sums = torch.logsumexp(x, dim=1)
            logp = torch.where(log_sums[:, None] > -math.inf, x - log_sums[:, None], -math.inf)
            p = torch.exp(logp)
            entropies = -(p * logp.masked_fill(p == 0, 0.0)).sum(dim=1)
            best, ids = torch.sort(x, dim=1, descending=True, stable=True)
            ids = ids[:, :case["top_k"]]
            parts.append((logp.gather(1, s["targets"][at:at + 512, None].long())[:, 0], log_sums, entropies,
                          ids.int(), logp.gather(1, ids)))
        whole = [torch.cat(p) for p in zip(*parts)]
        return dict(zip(("log_probs", "log_sums", "entropies", "top_ids", "top_log_probs"), whole))
    if case["op"] == "residual_norm":
        def norm(v, at):
            if case[at] == "none":
                return v
            gamma = s[at + "_gamma"].double()
            if case[at] == "rms":
                return gamma * v * torch.rsqrt(v.square().mean(1, True) + EPSILON)
            var, mean = torch.var_mean(v, dim=1, correction=0, keepdim=True)
            return gamma * (v - mean) * torch.rsqrt(var + EPSILON) + s[at + "_beta"].double()

        u = norm(s["block"].double(), "post")
        if case["gate"] != "none":
            rows = torch.arange(case["rows"], device="cuda") // (case["gate_rows"] or case["rows"])
            u = u * s["gate"].double()[rows]
        y = s["input"].double() + case["scale"] * u
        return dict(output=y, **({} if case["pre"] == "none" else {"normalized": norm(y, "pre")}))
    if case["op"] == "int4_gemv":
        a, inner, group = s["a"].double(), case["inner"], case["group"]
        y = torch.zeros(case["rows"], case["columns"], dtype=torch.float64, device="cuda")
        for g in range(inner // group):
            words = s["words"][:, g * group // 8:(g + 1) * group // 8].long() % 2 ** 32
            codes = torch.stack([words // 16 ** j % 16 for j in range(8)], dim=2).reshape(case["columns"], group)
            y += (a[:, g * group:(g + 1) * group] @ (codes.double() - 8.0).t()) * s["scales"][g].double()
        kind = case["epilogue"]
        if kind == "residual":
            y = s["residual"].double() + y / 2
        elif kind != "none":
            y = y + s["bias"].double()
            y = y * torch.sigmoid(y) if kind == "silu" else torch.relu(y) if kind == "relu" else y
        return dict(output=y)
    rows = [(w, u) for w, n in enumerate(s["counts"].tolist()) for u in range(n)]
    at = torch.tensor(rows, dtype=torch.int64, device="cuda").reshape(-1, 2)
    frame = s["joint_frames"].long()[at[:, 0], at[:, 1]]
    hidden = torch.relu(s["encoder"].double()[at[:, 0], frame] + s["predictor"].double()[at[:, 0], at[:, 1]])
    return dict(logits=torch.addmm(s["bias"].double(), hidden, s["weight"].double()),
                row_map=(at[:, 0] * case["max_tokens"] + at[:, 1]).int(),
                row_count=torch.tensor([len(rows)], dtype=torch.int32, device="cuda"))
