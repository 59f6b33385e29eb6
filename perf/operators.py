"""Operators at the tail of a decoder step, each in its plain form and as the
framework's call: the norms around a block with its gate and residual, the
product with a 4-bit group-scaled weight, and the scores of given tokens.

A case is a dict of plain values; `kind` says which operator it is:

  norm    out = residual + scale * gate * norm(input) and next = norm(out)
          (pk_block_norm): LayerNorm or RMS norm, gates per row, per run of
          rows or for all rows, rows of wider buffers
  q4      out = residual + scale * act(a @ w + bias), w = scale * (code - 8)
          + offset in groups along the inner dimension (pk_q4)
  score   log probabilities of given tokens, the entropy of each row and its
          best alternatives (pk_score)

`own` false: elementary torch operations in 32 bits, rounded once. `own` true:
the entry points of parakeet_wgsl_amd.palette_abi.
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"f16": torch.float16, "f32": torch.float32}
INF = float("inf")


def listed():
    return [
        # one frame of a live stream between two Conformer blocks
        {"name": "norm-1x1024", "kind": "norm", "precision": "f16", "norm": "layer", "rows": 1, "channels": 1024,
         "gate": "none", "post": True, "next": True, "wide": False, "scale": 0.5},
        # the same place in the full batch: 16 windows of 188 frames, a gate row per window
        {"name": "norm-3008x1024", "kind": "norm", "precision": "f16", "norm": "layer", "rows": 3008,
         "channels": 1024, "gate": "window", "post": True, "next": True, "wide": False, "scale": 0.5},
        # an odd channel count in the fp32 profile: rows without vector alignment
        {"name": "norm-f32-1504x1001", "kind": "norm", "precision": "f32", "norm": "layer", "rows": 1504,
         "channels": 1001, "gate": "all", "post": True, "next": True, "wide": False, "scale": 1.0},
        # a long prompt of a wide decoder: value and gate are the halves of one product's rows
        {"name": "norm-8192x4096", "kind": "norm", "precision": "f16", "norm": "rms", "rows": 8192,
         "channels": 4096, "gate": "row", "post": True, "next": True, "wide": True, "scale": 1.0},
        # the joint head over one frame, fp32 profile
        {"name": "q4-f32-1x640x1032", "kind": "q4", "precision": "f32", "rows": 1, "inner": 640, "columns": 1032,
         "group": 32, "offsets": False, "bias": True, "activation": "none", "residual": False},
        # one token through a wide projection: the weight stream
        {"name": "q4-1x4096x8192", "kind": "q4", "precision": "f16", "rows": 1, "inner": 4096, "columns": 8192,
         "group": 128, "offsets": False, "bias": False, "activation": "none", "residual": False},
        # 64 streams at once through the largest weight, asymmetric codes
        {"name": "q4-64x8192x8192", "kind": "q4", "precision": "f16", "rows": 64, "inner": 8192, "columns": 8192,
         "group": 64, "offsets": True, "bias": False, "activation": "none", "residual": True},
        # the feed-forward expand of 8 windows: many rows, the matrix units' side of the operator
        {"name": "q4-1504x1024x4096", "kind": "q4", "precision": "f16", "rows": 1504, "inner": 1024,
         "columns": 4096, "group": 128, "offsets": False, "bias": True, "activation": "silu", "residual": False},
        # the confidence of one decoded token: rows of the TDT head hold 1025 token columns of 1032
        {"name": "score-1x1025", "kind": "score", "precision": "f16", "rows": 1, "columns": 1025, "stride": 1032,
         "alternatives": 4, "temperature": 1.0, "masked": 0.0},
        # every frame of 16 windows scored at once
        {"name": "score-3008x1025", "kind": "score", "precision": "f16", "rows": 3008, "columns": 1025,
         "stride": 1032, "alternatives": 4, "temperature": 1.0, "masked": 0.0},
        # eight streams over a large vocabulary: few rows, a long axis
        {"name": "score-8x131072", "kind": "score", "precision": "f16", "rows": 8, "columns": 131072,
         "stride": 131072, "alternatives": 8, "temperature": 1.0, "masked": 0.0},
        # rescoring a batch of hypotheses, fp32 logits, a tenth of the vocabulary masked
        {"name": "score-f32-2048x32000", "kind": "score", "precision": "f32", "rows": 2048, "columns": 32000,
         "stride": 32000, "alternatives": 8, "temperature": 0.8, "masked": 0.1},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """A size of the range: mostly a multiple of 8, sometimes any number."""
    n = _log_int(rng, low, high)
    return n if rng.random() < 0.3 else max(8, n // 8 * 8)


def draw(rng):
    kind = rng.choice(["norm", "q4", "score"])
    precision = rng.choice(["f16", "f16", "f32"])
    if kind == "norm":
        channels = _size(rng, 64, 8192)
        most = 8192 * 4096 // (channels * (1 if precision == "f16" else 2))
        return {"kind": kind, "precision": precision, "norm": rng.choice(["layer", "rms"]),
                "rows": _log_int(rng, 1, min(8192, most)), "channels": channels,
                "gate": rng.choice(["none", "row", "window", "all"]), "post": rng.random() < 0.7,
                "next": rng.random() < 0.8, "wide": rng.random() < 0.3, "scale": rng.choice([0.5, 1.0, 0.25])}
    if kind == "q4":
        inner, columns = _size(rng, 64, 8192), _size(rng, 64, 8192)
        most = 1504 * 1024 * 4096 // (inner * columns * (1 if precision == "f16" else 4))
        return {"kind": kind, "precision": precision,
                "rows": _log_int(rng, 1, max(1, min(rng.choice([4, 64, 1504]), most))), "inner": inner,
                "columns": columns, "group": rng.choice([32, 64, 128, 128, 256, 0]), "offsets": rng.random() < 0.4,
                "bias": rng.random() < 0.5, "activation": rng.choice(["none", "silu", "relu"]),
                "residual": rng.random() < 0.5}
    columns = _log_int(rng, 5, 131072)
    return {"kind": kind, "precision": precision, "rows": _log_int(rng, 1, min(4096, 2048 * 32000 // columns)),
            "columns": columns, "stride": columns + rng.choice([0, 0, 1, 7, 8]),
            "alternatives": min(columns, rng.choice([0, 1, 4, 8, 16])), "temperature": rng.choice([1.0, 0.7, 1.5]),
            "masked": rng.choice([0.0, 0.0, 0.3])}


# ------------------------------------------------------------------ inputs

def _inputs(case, seed):
    """The seeded tensors of a case, made on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind, rows = DTYPE[case["precision"]], case["kind"], case["rows"]

    def normal(*shape, std=1.0, mean=0.0, dtype=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    if kind == "norm":
        c, f32 = case["channels"], torch.float32
        t = {"residual": normal(rows, c, std=2.0, mean=0.1)}
        gates = {"none": 0, "row": rows, "window": (rows + 187) // 188, "all": 1}[case["gate"]]
        t["gate_rows"] = {"none": 1, "row": 1, "window": 188, "all": 0}[case["gate"]]
        if case["wide"]:  # the value and its gate side by side, as a product of twice the width leaves them
            both = normal(max(rows, gates), 2 * c, std=0.7)
            t["input"], t["gate"] = both[:rows, :c], both[:gates, c:] if gates else None
        else:
            t["input"], t["gate"] = normal(rows, c, std=1.5), normal(gates, c, std=0.7) if gates else None
        for n in ("", "next_"):
            t[n + "gamma"] = normal(c, std=0.1, mean=1.0, dtype=f32)
            t[n + "beta"] = normal(c, std=0.1, dtype=f32) if case["norm"] == "layer" else None
        return t
    if kind == "q4":
        inner, columns = case["inner"], case["columns"]
        words = (inner * columns + 7) // 8
        groups = -(-inner // (case["group"] or inner))
        packed = torch.randint(-2**31, 2**31, (words,), generator=g, device="cuda", dtype=torch.int64)
        return {"a": normal(rows, inner), "packed": packed.to(torch.int32),
                "scales": (torch.rand((groups, columns), generator=g, device="cuda") * 0.006 + 0.002).to(dtype),
                "offsets": normal(groups, columns, std=0.003) if case["offsets"] else None,
                "bias": normal(columns, std=0.1, dtype=torch.float32) if case["bias"] else None,
                "residual": normal(rows, columns) if case["residual"] else None}
    columns = case["columns"]
    logits = normal(rows, case["stride"], std=2.5, dtype=torch.float32)
    # a peak of its own height in each row: from undecided to certain
    peak = torch.randint(0, columns, (rows, 1), generator=g, device="cuda")
    logits.scatter_add_(1, peak, torch.rand((rows, 1), generator=g, device="cuda") * 14)
    if case["masked"]:
        out = torch.rand((rows, case["stride"]), generator=g, device="cuda") < case["masked"]
        out[rows // 2] = rows > 1  # and one row with nothing left
        logits.masked_fill_(out, -INF)
    tokens = torch.where(torch.rand((rows, 1), generator=g, device="cuda") < 0.7, peak,
                         torch.randint(0, columns, (rows, 1), generator=g, device="cuda")).reshape(-1)
    if rows > 4:
        tokens[rows - 2:] = -1  # positions behind the last token of a padded batch
    return {"logits": logits.to(dtype)[:, :columns], "tokens": tokens.to(torch.int32)}


class Buffer:
    """A torch tensor as a device buffer of the ABI: pointer, bytes up to its
    last element, numpy type."""

    _TYPES = {torch.float16: np.float16, torch.float32: np.float32, torch.int32: np.uint32}

    def __init__(self, tensor):
        self.tensor, self.ptr = tensor, tensor.data_ptr()
        last = sum((n - 1) * s for n, s in zip(tensor.shape, tensor.stride()))
        self.nbytes = (last + 1) * tensor.element_size()
        self.dtype, self.shape = np.dtype(self._TYPES[tensor.dtype]), tuple(tensor.shape)


def _buffer(tensor):
    return None if tensor is None else Buffer(tensor)


_context = None
_LEGACY_STREAM = 1  # hipStreamLegacy: torch's default stream, whose handle 0 stands for the context's own in a call


class State:
    """What a user's program holds between calls: its tensors, and the
    framework's op over them where that is what runs, with the stream that it
    works on, torch's current one when the state was made."""

    op = None
    stream = None

    def __init__(self, case, tensors, outputs):
        self.case, self.tensors, self.outputs = case, tensors, outputs

    def __del__(self):
        if self.op is not None:
            torch.cuda.synchronize()
            self.op.release()


def _op(case, t, outputs):
    """The framework's op over these tensors."""
    import parakeet_wgsl_amd.palette_abi as abi
    global _context
    if _context is None:
        torch.cuda.current_device()
        _context = abi.Context(0)
    torch.cuda.synchronize()  # the library's stream starts after the inputs are there
    b = {n: _buffer(x) for n, x in t.items() if x is None or torch.is_tensor(x)}
    b.update({n: _buffer(x) for n, x in outputs.items()})
    if case["kind"] == "norm":
        post, following = case["post"], case["next"]
        op = abi.BlockNormOp(
            _context, kind=case["norm"], rows=case["rows"], channels=case["channels"], input=b["input"],
            input_stride=t["input"].stride(0), gamma=b["gamma"] if post else None, beta=b["beta"] if post else None,
            gate=b["gate"], gate_stride=0 if t["gate"] is None else t["gate"].stride(0), gate_rows=t["gate_rows"],
            residual=b["residual"], residual_scale=case["scale"], output=b["output"],
            next_gamma=b["next_gamma"] if following else None, next_beta=b["next_beta"] if following else None,
            next_output=b["next"] if following else None)
    elif case["kind"] == "q4":
        op = abi.Q4GemmOp(
            _context, a=b["a"], packed=b["packed"], scales=b["scales"], offsets=b["offsets"], output=b["output"],
            rows=case["rows"], inner=case["inner"], columns=case["columns"], group_size=case["group"],
            bias=b["bias"], residual=b["residual"], residual_scale=0.5 if case["residual"] else None,
            activation=case["activation"])
    else:
        op = abi.TokenScoreOp(
            _context, logits=b["logits"], rows=case["rows"], columns=case["columns"], row_stride=case["stride"],
            tokens=b["tokens"], temperature=case["temperature"], alternatives=case["alternatives"],
            log_probs=b["log_probs"], entropies=b["entropies"], top_tokens=b.get("top_tokens"),
            top_log_probs=b.get("top_log_probs"))
    _context.synchronize()
    return op


def prepare(case, seed):
    t, outputs = _inputs(case, seed), {}
    if own:
        def new(*shape, dtype=DTYPE[case["precision"]]):
            return torch.zeros(shape, dtype=dtype, device="cuda")
        rows = case["rows"]
        if case["kind"] == "norm":
            outputs = {"output": new(rows, case["channels"])}
            if case["next"]:
                outputs["next"] = new(rows, case["channels"])
        elif case["kind"] == "q4":
            outputs = {"output": new(rows, case["columns"])}
        else:
            outputs = {"log_probs": new(rows, dtype=torch.float32), "entropies": new(rows, dtype=torch.float32)}
            if k := case["alternatives"]:
                outputs |= {"top_tokens": new(rows, k, dtype=torch.int32),
                            "top_log_probs": new(rows, k, dtype=torch.float32)}
    state = State(case, t, outputs)
    if own:
        state.op = _op(case, t, outputs)
        state.stream = torch.cuda.current_stream().cuda_stream or _LEGACY_STREAM
    return state


# ------------------------------------------------------------- plain forms

def _plain_norm(x, kind, gamma, beta):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * gamma
    return x if beta is None else x + beta


def _run_norm(case, t):
    dtype, rows = t["residual"].dtype, case["rows"]
    v = t["input"].float()
    if case["post"]:
        v = _plain_norm(v, case["norm"], t["gamma"], t["beta"])
    if t["gate"] is not None:
        at = torch.arange(rows, device=v.device)
        v = v * t["gate"].float()[at // t["gate_rows"] if t["gate_rows"] else at * 0]
    y = t["residual"].float() + case["scale"] * v
    out = {"output": y.to(dtype)}
    if case["next"]:
        out["next"] = _plain_norm(y, case["norm"], t["next_gamma"], t["next_beta"]).to(dtype)
    return out


def _run_q4(case, t):
    inner, columns = case["inner"], case["columns"]
    group = case["group"] or inner
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    codes = ((t["packed"][:, None] >> shifts) & 15).reshape(-1)[:inner * columns].reshape(inner, columns)
    at = torch.arange(inner, device="cuda") // group
    w = (codes - 8).float() * t["scales"].float()[at]
    if t["offsets"] is not None:
        w = w + t["offsets"].float()[at]
    y = t["a"].float() @ w
    if t["bias"] is not None:
        y = y + t["bias"]
    if case["activation"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["activation"] == "relu":
        y = torch.clamp(y, min=0)
    if t["residual"] is not None:
        y = t["residual"].float() + 0.5 * y
    return {"output": y.to(t["a"].dtype)}


def _run_score(case, t):
    raw, tokens, k = t["logits"].float(), t["tokens"].long(), case["alternatives"]
    z = raw / case["temperature"]
    top = z.amax(-1, keepdim=True)
    live = top > -INF  # a row whose mask leaves nothing has no probabilities
    d = z - torch.where(live, top, torch.zeros_like(top))
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(-1, keepdim=True)
    entropies = torch.where(live, log_total - weighted / total, torch.zeros_like(total))[:, 0]
    nothing = torch.full_like(d[:, :1], -INF)
    given = torch.where(live, d.gather(1, tokens.clamp(min=0)[:, None]) - log_total, nothing)[:, 0]
    out = {"log_probs": torch.where(tokens >= 0, given, torch.zeros_like(given)), "entropies": entropies}
    if k:
        # keys in the order of the logits, and of falling indexes where they are equal
        bits = (raw + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
        columns = case["columns"]
        keys = (order << 32) | (columns - 1 - torch.arange(columns, device="cuda"))
        at = columns - 1 - (torch.topk(keys, k, dim=-1).values & 0xFFFFFFFF)
        found = torch.where(live, d.gather(1, at) - log_total, nothing)
        out["top_tokens"] = torch.where(found > -INF, at, torch.full_like(at, -1)).to(torch.int32)
        out["top_log_probs"] = found
    return out


def run(state):
    """One pass, in order with what the stream that was torch's current one in
    `prepare` holds, as the plain form is. `own`: the outputs are the state's,
    which the next pass on that stream writes again."""
    if own:
        state.op.enqueue(0, state.stream)
        return state.outputs
    return {"norm": _run_norm, "q4": _run_q4, "score": _run_score}[state.case["kind"]](state.case, state.tensors)


# ------------------------------------------------------------------- work

def work(case):
    rows, e = case["rows"], 2 if case["precision"] == "f16" else 4
    if case["kind"] == "norm":
        c = case["channels"]
        gates = {"none": 0, "row": rows, "window": (rows + 187) // 188, "all": 1}[case["gate"]]
        vectors = (case["post"] + case["next"]) * (2 if case["norm"] == "layer" else 1)
        return {"bytes": (rows * (3 + case["next"]) + gates) * c * e + vectors * c * 4,
                "flops": rows * c * (3 + 7 * (case["post"] + case["next"]))}
    if case["kind"] == "q4":
        inner, columns = case["inner"], case["columns"]
        groups = -(-inner // (case["group"] or inner))
        weight = inner * columns / 2 + groups * columns * e * (1 + case["offsets"])
        return {"bytes": weight + rows * (inner + columns * (1 + case["residual"])) * e + 4 * columns * case["bias"],
                "flops": 2 * rows * inner * columns}
    return {"bytes": rows * (case["columns"] * e + 12 + 8 * case["alternatives"]),
            "flops": rows * case["columns"] * 6}


# ------------------------------------------------------------------ exact

def _exact_norm(case, t):
    def norm(x, gamma, beta):
        mean = x.sum(1, keepdim=True) / x.shape[1] if case["norm"] == "layer" else 0.0
        power = ((x - mean) ** 2).sum(1, keepdim=True) / x.shape[1]
        y = (x - mean) / torch.sqrt(power + 1e-5) * gamma.double()
        return y if beta is None else y + beta.double()
    v = t["input"].double()
    if case["post"]:
        v = norm(v, t["gamma"], t["beta"])
    if t["gate"] is not None:
        gate, each = t["gate"].double(), t["gate_rows"]
        v = v * (gate.repeat_interleave(each, 0)[:case["rows"]] if each else gate)
    y = t["residual"].double() + v * case["scale"]
    out = {"output": y}
    if case["next"]:
        out["next"] = norm(y, t["next_gamma"], t["next_beta"])
    return out


def _exact_q4(case, t):
    inner, columns, rows = case["inner"], case["columns"], case["rows"]
    group = case["group"] or inner
    groups = -(-inner // group)
    words = t["packed"].long() & 0xFFFFFFFF
    codes = torch.stack([(words >> (4 * i)) & 15 for i in range(8)], 1).reshape(-1)[:inner * columns]
    y = torch.zeros(rows, columns, dtype=torch.float64, device="cuda")
    a, codes = t["a"].double(), codes.reshape(inner, columns)
    for g in range(groups):
        part, c = a[:, g * group:(g + 1) * group], codes[g * group:(g + 1) * group].double()
        y += (part @ c - 8 * part.sum(1, keepdim=True)) * t["scales"][g].double()
        if t["offsets"] is not None:
            y += part.sum(1, keepdim=True) * t["offsets"][g].double()
    if t["bias"] is not None:
        y = y + t["bias"].double()
    if case["activation"] != "none":
        y = y * (torch.sigmoid(y) if case["activation"] == "silu" else (y > 0))
    if t["residual"] is not None:
        y = t["residual"].double() + y / 2
    return {"output": y}


def _exact_score(case, t):
    z, tokens, k = t["logits"].double() / case["temperature"], t["tokens"].long(), case["alternatives"]
    log_p = z - torch.logsumexp(z, 1, keepdim=True)
    log_p[torch.isnan(log_p)] = -INF  # nothing left by the mask
    h = -(torch.special.xlogy(torch.exp(log_p), torch.exp(log_p))).sum(1)
    given = log_p[torch.arange(len(tokens), device="cuda"), tokens.clamp(min=0)]
    out = {"log_probs": given.masked_fill(tokens < 0, 0.0), "entropies": h}
    if k:
        best, at = torch.sort(log_p, dim=1, descending=True, stable=True)
        out["top_tokens"] = at[:, :k].masked_fill(best[:, :k] == -INF, -1).to(torch.int32)
        out["top_log_probs"] = best[:, :k].contiguous()
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    return {"norm": _exact_norm, "q4": _exact_q4, "score": _exact_score}[case["kind"]](case, t)
