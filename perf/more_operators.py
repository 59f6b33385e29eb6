"""Operators of a decoder that keeps what it has read, each in its plain form
and as the framework's call: keys and values appended to a paged cache, the
attention of new tokens over it, and the verification of drafted tokens.

A case is a dict of plain values; `kind` says which operator it is:

  append     rotated queries and keys, keys and values into pages (pk_cache_append)
  attention  new tokens, one, a few or a chunk for each sequence, over the pages,
             causal or not, with a window and a cap of the scores (pk_cache_attention)
  verify     how many drafted tokens stand against the target's probabilities, and
             the token that follows them (pk_draft_verify)

`own` false: elementary torch operations, rounded once. `own` true: the entry
points of parakeet_wgsl_amd.palette_abi.

The rows and lengths of a case's sequences lie between its bounds, spread over
them by their logarithm in an order without pattern.
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"f16": torch.float16, "f32": torch.float32}
INF = float("inf")


def _append(name, precision, sequences, rows, lengths, heads, kv_heads, head_dim, page, rotary_dim, **over):
    return dict({"name": name, "kind": "append", "precision": precision, "sequences": sequences, "rows_low": rows[0],
                 "rows_high": rows[1], "length_low": lengths[0], "length_high": lengths[1], "heads": heads,
                 "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "rotary_dim": rotary_dim,
                 "pairs": "halves", "positions": False, "packed": True}, **over)


def _attention(name, precision, sequences, rows, lengths, heads, kv_heads, head_dim, page, **over):
    return dict({"name": name, "kind": "attention", "precision": precision, "sequences": sequences,
                 "rows_low": rows[0], "rows_high": rows[1], "length_low": lengths[0], "length_high": lengths[1],
                 "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "window": 0, "cap": 0.0,
                 "causal": True}, **over)


def _verify(name, precision, sequences, rows, columns, **over):
    return dict({"name": name, "kind": "verify", "precision": precision, "sequences": sequences,
                 "rows_low": rows[0], "rows_high": rows[1], "columns": columns, "stride": columns, "mode": "sample",
                 "draft": True, "temperature": 1.0}, **over)


def listed():
    return [
        # one token of one live stream
        _append("append-1", "f16", 1, (1, 1), (376, 376), 8, 8, 128, 16, 128, packed=False),
        # a step of 64 streams in the fp32 profile, part of each head rotated, at positions of their own
        _append("append-f32-64", "f32", 64, (1, 1), (100, 30000), 8, 2, 80, 16, 32, pairs="neighbours", positions=True,
                packed=False),
        # chunks of 16 windows of audio, 188 frames each at most
        _append("append-16x188", "f16", 16, (60, 188), (188, 1504), 8, 8, 128, 16, 128, packed=False),
        # a chunk of long prompts of a wide decoder with shared key heads
        _append("append-4x2048", "f16", 4, (2048, 2048), (2048, 32768), 32, 8, 128, 64, 128),
        # one token of one live stream over half a minute of frames
        _attention("attention-1x376", "f16", 1, (1, 1), (376, 376), 8, 8, 128, 16),
        # a step of 64 streams of different ages, four query heads to a key head
        _attention("attention-64-ragged", "f16", 64, (1, 1), (200, 16384), 32, 8, 128, 16),
        # a step of few streams with a very long memory
        _attention("attention-4x131072", "f16", 4, (1, 1), (131072, 131072), 32, 8, 128, 64),
        # drafts of 3 to 7 tokens checked at once: capped scores, a window, pages of an odd size
        _attention("attention-draft-16", "f16", 16, (4, 8), (1500, 6000), 16, 2, 64, 24, window=4096, cap=50.0),
        # chunks of long prompts
        _attention("attention-4x1024", "f16", 4, (700, 1024), (2048, 8192), 32, 8, 128, 64),
        # a streamed window of frames with a left context, fp32 profile
        _attention("attention-f32-16x188", "f32", 16, (60, 188), (188, 752), 8, 8, 128, 16, window=376),
        # four drafted tokens of one stream over the TDT head's token columns
        _verify("verify-1x5x1025", "f16", 1, (5, 5), 1025, stride=1032),
        # 32 streams with drafts of up to 7 tokens over a large vocabulary
        _verify("verify-32x8x131072", "f16", 32, (3, 8), 131072, temperature=0.8),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_heads(rng):
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    return kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 8]), kv_heads, rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 128, 192, 256])


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "verify"])
    precision = rng.choice(["f16", "f16", "f32"])
    if kind == "verify":
        columns = _log_int(rng, 5, 131072)
        rows = rng.choice([1, 4, 8, 12])
        sequences = _log_int(rng, 1, max(1, min(64, 32 * 5 * 131072 // (columns * rows * (1 + (precision == "f32"))))))
        return _verify(None, precision, sequences, (max(1, rows // 2), rows), columns,
                       stride=columns + rng.choice([0, 0, 1, 7, 8]), mode=rng.choice(["sample", "sample", "greedy"]),
                       draft=rng.random() < 0.7, temperature=rng.choice([1.0, 0.7, 1.3])) | {"name": ""}
    heads, kv_heads, head_dim = _draw_heads(rng)
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    width = (heads + 2 * kv_heads) * head_dim * (1 + (precision == "f32"))
    if kind == "append":
        rows = _log_int(rng, 1, 2048)
        sequences = _log_int(rng, 1, max(1, min(64, 8192 * 6144 // (width * rows))))
        longest = _log_int(rng, rows, 32768)
        return _append("", precision, sequences, (max(1, rows // 3), rows), (max(rows, longest // 8), longest), heads,
                       kv_heads, head_dim, page, rng.choice([head_dim, head_dim, head_dim // 2, 0]),
                       pairs=rng.choice(["halves", "neighbours"]), positions=rng.random() < 0.3,
                       packed=rng.random() < 0.6)
    rows = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, 1024)])
    # tokens of cache, and scores, within the longest and the largest of the list
    longest = _log_int(rng, max(rows, 16), 65536)
    most = min(2 ** 29 // (longest * kv_heads * head_dim * (1 + (precision == "f32"))),
               2 ** 33 // (rows * longest * heads * head_dim * (1 if precision == "f16" else 16) // 32))
    sequences = _log_int(rng, 1, max(1, min(64, most)))
    if most < 1:
        rows = 1
    causal = rng.random() < 0.8
    return _attention("", precision, sequences, (max(1, rows // 2), rows), (max(rows, longest // 16), longest), heads,
                      kv_heads, head_dim, page, causal=causal, cap=rng.choice([0.0, 0.0, 30.0]),
                      window=_log_int(rng, 16, 8192) if causal and rng.random() < 0.3 else 0)


# ------------------------------------------------------------------ inputs

def _spread(low, high, count, step):
    """`count` whole numbers over [low, high], by their logarithm."""
    if count == 1:
        return [high]
    return [int(round(low * (high / low) ** ((1 + i * step) % 1.0))) for i in range(count)]


def _rows_of(case):
    return _spread(case["rows_low"], case["rows_high"], case["sequences"], 0.7548776662466927)


def _lengths_of(case):
    return [max(n, rows) for n, rows in zip(_spread(case["length_low"], case["length_high"], case["sequences"],
                                                    0.6180339887498949), _rows_of(case))]


def _starts(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def _ints(values):
    return torch.tensor(values, dtype=torch.int64).to(torch.int32).cuda()


def _paged(case, g, t, shared):
    """Lengths, page table and caches. With `shared`, pages before a sequence's
    new tokens are those of a common prompt: few pages that nothing writes."""
    rows, lengths, page = _rows_of(case), _lengths_of(case), case["page"]
    tables, own_pages, prompt = [], 0, 8 if shared else 0
    for n, length in zip(rows, lengths):
        first = (length - n) // page if shared else 0
        count = -(-length // page)
        tables.append([i % prompt for i in range(first)] + [-2 - own_pages - i for i in range(count - first)])
        own_pages += count - first
    pages = prompt + own_pages + 3  # the pool has more than these sequences hold
    order = torch.randperm(pages - prompt, generator=g, device="cuda")[:own_pages] + prompt
    width = max(len(x) for x in tables)
    table = torch.tensor([x + [-1] * (width - len(x)) for x in tables], dtype=torch.int64).cuda()
    t["page_table"] = torch.where(table < -1, order[(-2 - table).clamp(min=0)], table).to(torch.int32)
    t["row_starts"], t["lengths"] = _ints(_starts(rows)), _ints(lengths)
    shape = (pages, case["kv_heads"], page, case["head_dim"])
    for name in ("key_cache", "value_cache"):
        t[name] = torch.empty(shape, dtype=DTYPE[case["precision"]], device="cuda")
        for part in t[name].split(max(1, 2 ** 26 // (shape[1] * shape[2] * shape[3]))):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    return t


def _inputs(case, seed):
    """The seeded tensors of a case, made on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind, rows = DTYPE[case["precision"]], case["kind"], sum(_rows_of(case))

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    if kind == "append":
        heads, kv, dim, half = case["heads"], case["kv_heads"], case["head_dim"], case["rotary_dim"] // 2
        if case["packed"]:  # queries, keys and values side by side, as one product leaves them
            both = normal(rows, (heads + 2 * kv) * dim)
            t = dict(zip(("queries", "keys", "values"), both.split([heads * dim, kv * dim, kv * dim], 1)))
        else:
            t = {"queries": normal(rows, heads * dim), "keys": normal(rows, kv * dim), "values": normal(rows, kv * dim)}
        _paged(case, g, t, True)
        t["frequencies"] = None
        if half:
            t["frequencies"] = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float32) / half)
        t["positions"] = None
        if case["positions"]:
            t["positions"] = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda").to(torch.int32)
        return t
    if kind == "attention":
        t = {"queries": normal(rows, case["heads"] * case["head_dim"], std=2.0)}
        return _paged(case, g, t, False)
    columns, stride = case["columns"], case["stride"]
    # what both models agree on, with a peak of its own height in each row, and what they do not
    base = normal(rows, stride, std=2.0, dtype=torch.float32)
    peak = torch.randint(0, columns, (rows, 1), generator=g, device="cuda")
    base.scatter_add_(1, peak, uniform(rows, 1) * 14)
    draft = (base + normal(rows, stride, dtype=torch.float32)).to(dtype)[:, :columns]
    t = {"target": (base + normal(rows, stride, dtype=torch.float32)).to(dtype)[:, :columns]}
    del base
    t["draft"] = draft if case["draft"] else None
    # the draft after row r is drawn from the draft model's row r, or is its best
    race = draft.float() / case["temperature"]
    if case["draft"]:
        race = race - torch.log(-torch.log(uniform(rows, columns).clamp(1e-9, 1 - 1e-7)))
    chosen = race.argmax(-1)
    t["tokens"] = torch.cat([torch.zeros_like(chosen[:1]), chosen[:-1]]).to(torch.int32)
    t["row_starts"] = _ints(_starts(_rows_of(case)))
    t["uniforms"], t["draws"] = uniform(rows), uniform(case["sequences"])
    return t


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
    b = {n: _buffer(x) for n, x in t.items()}
    b.update({n: _buffer(x) for n, x in outputs.items()})
    rows, sequences = sum(_rows_of(case)), case["sequences"]
    if case["kind"] == "verify":
        op = abi.DraftVerifyOp(
            _context, target=b["target"], target_stride=case["stride"], draft=b["draft"],
            draft_stride=case["stride"] if case["draft"] else 0, rows=rows, sequences=sequences,
            columns=case["columns"], row_starts=b["row_starts"], tokens=b["tokens"], mode=case["mode"],
            temperature=case["temperature"], uniforms=b["uniforms"], draws=b["draws"], accepted=b["accepted"],
            next_tokens=b["next_tokens"])
    else:
        cache = dict(rows=rows, sequences=sequences, heads=case["heads"], kv_heads=case["kv_heads"],
                     head_dim=case["head_dim"], row_starts=b["row_starts"], lengths=b["lengths"],
                     page_table=b["page_table"], pages_per_sequence=t["page_table"].shape[1], key_cache=b["key_cache"],
                     value_cache=b["value_cache"], pages=t["key_cache"].shape[0], page_size=case["page"])
        if case["kind"] == "append":
            op = abi.CacheAppendOp(
                _context, queries=b["queries"], query_stride=t["queries"].stride(0), query_output=b["rotated"],
                keys=b["keys"], key_stride=t["keys"].stride(0), values=b["values"],
                value_stride=t["values"].stride(0), rotary_dim=case["rotary_dim"], rotary=case["pairs"],
                frequencies=b["frequencies"], positions=b["positions"] if case["rotary_dim"] else None, **cache)
        else:
            op = abi.CacheAttentionOp(
                _context, queries=b["queries"], output=b["output"], causal=case["causal"], window=case["window"],
                score_cap=case["cap"] or None, **cache)
    _context.synchronize()
    return op


def prepare(case, seed):
    t, outputs = _inputs(case, seed), {}
    if own:
        if case["kind"] == "verify":
            outputs = {n: torch.zeros(case["sequences"], dtype=torch.int32, device="cuda")
                       for n in ("accepted", "next_tokens")}
        else:
            name = "rotated" if case["kind"] == "append" else "output"
            outputs = {name: torch.zeros(t["queries"].shape, dtype=t["queries"].dtype, device="cuda")}
    state = State(case, t, outputs)
    if own:
        state.op = _op(case, t, outputs)
        state.stream = torch.cuda.current_stream().cuda_stream or _LEGACY_STREAM
        if case["kind"] == "append":
            state.outputs = outputs | {"keys": t["key_cache"], "values": t["value_cache"]}
    return state


# ------------------------------------------------------------- plain forms

def _places(case, t):
    """Of each row its sequence and its position in it."""
    starts, at = t["row_starts"].long(), torch.arange(t["keys"].shape[0], device="cuda")
    sequence = (at[:, None] >= starts[None, 1:]).sum(1)
    return sequence, t["lengths"].long()[sequence] - starts[sequence + 1] + at


def _run_append(case, t):
    dim, half, kv, page = case["head_dim"], case["rotary_dim"] // 2, case["kv_heads"], case["page"]
    sequence, position = _places(case, t)
    angle = position if t["positions"] is None else t["positions"].long()

    def rotated(x, heads):
        x = x.float().reshape(-1, heads, dim)
        if not half:
            return x
        turn = (angle.double()[:, None] * t["frequencies"].double())[:, None]
        c, s = torch.cos(turn).float(), torch.sin(turn).float()
        out = x.clone()
        first, second = ((slice(0, half), slice(half, 2 * half)) if case["pairs"] == "halves" else
                         (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
        out[..., first] = x[..., first] * c - x[..., second] * s
        out[..., second] = x[..., second] * c + x[..., first] * s
        return out

    dtype = t["keys"].dtype
    number, place = t["page_table"].long()[sequence, position // page], position % page
    t["key_cache"][number, :, place] = rotated(t["keys"], kv).to(dtype)
    t["value_cache"][number, :, place] = t["values"].reshape(-1, kv, dim)
    return {"rotated": rotated(t["queries"], case["heads"]).to(dtype).reshape(-1, case["heads"] * dim),
            "keys": t["key_cache"], "values": t["value_cache"]}


def _run_attention(case, t):
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group, parts = heads // kv, []
    for s, (n, length, start) in enumerate(zip(_rows_of(case), _lengths_of(case), _starts(_rows_of(case)))):
        numbers = t["page_table"][s, :-(-length // page)].long()
        k, v = (t[c][numbers].transpose(0, 1).reshape(kv, -1, dim)[:, :length].float()
                for c in ("key_cache", "value_cache"))
        q = t["queries"][start:start + n].float().reshape(n, kv, group, dim).permute(1, 2, 0, 3)
        at, tokens = torch.arange(length - n, length, device="cuda")[:, None], torch.arange(length, device="cuda")
        hidden = tokens > at if case["causal"] else torch.zeros_like(tokens > at)
        if case["window"]:
            hidden = hidden | (tokens <= at - case["window"])
        out = torch.empty(kv, group, n, dim, device="cuda")
        for h in range(kv):
            z = (q[h].reshape(-1, dim) @ k[h].T).reshape(group, n, length) / math.sqrt(dim)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            z = z.masked_fill(hidden, -INF)
            e = torch.exp(z - z.amax(-1, keepdim=True))
            out[h] = (e.reshape(-1, length) @ v[h]).reshape(group, n, dim) / e.sum(-1, keepdim=True)
        parts.append(out.permute(2, 0, 1, 3).reshape(n, heads * dim))
    return {"output": torch.cat(parts).to(t["queries"].dtype)}


def _probabilities(logits, temperature):
    z = logits.double() / temperature
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _run_verify(case, t):
    columns = case["columns"]
    starts, tokens = t["row_starts"].long(), t["tokens"].long()
    rows = torch.arange(len(tokens), device="cuda")
    drafted = torch.cat([tokens[1:], tokens[:1]])  # the draft that a row judges
    last = torch.zeros_like(rows, dtype=torch.bool)
    last[starts[1:] - 1] = True
    if case["mode"] == "greedy":
        z, index = t["target"].float(), torch.arange(columns, device="cuda")
        best = torch.where(z == z.amax(-1, keepdim=True), index, columns).amin(-1)
        stands = best == drafted
    else:
        p = _probabilities(t["target"], case["temperature"])
        one = torch.zeros_like(p).scatter_(1, drafted[:, None], 1.0)
        q = _probabilities(t["draft"], case["temperature"]) if case["draft"] else one
        stands = t["uniforms"].double() * q[rows, drafted] < p[rows, drafted]
    ends = torch.where(stands & ~last, len(tokens), rows)  # each sequence's first row whose draft does not stand
    sequence = (rows[:, None] >= starts[None, 1:]).sum(1)
    at = torch.full_like(starts[1:], len(tokens)).scatter_reduce(0, sequence, ends, "amin")
    if case["mode"] == "greedy":
        chosen = best[at]
    else:
        w = torch.where(last[at][:, None], p[at], (p[at] - q[at]).clamp(min=0))
        running = torch.cumsum(w, -1)
        want = t["draws"].double() * running[:, -1]
        found = (running <= want[:, None]).sum(-1)
        behind = torch.where(w > 0, torch.arange(columns, device="cuda"), 0).amax(-1)
        chosen = torch.minimum(found, behind)
    return {"accepted": (at - starts[:-1]).to(torch.int32), "next_tokens": chosen.to(torch.int32)}


def run(state):
    """One pass, in order with what the stream that was torch's current one in
    `prepare` holds, as the plain form is. `own`: the outputs are the state's,
    which the next pass on that stream writes again."""
    if own:
        state.op.enqueue(0, state.stream)
        return state.outputs
    form = {"append": _run_append, "attention": _run_attention, "verify": _run_verify}[state.case["kind"]]
    return form(state.case, state.tensors)


# ------------------------------------------------------------------- work

def _seen(case, n, length):
    """Scores of a sequence's rows, and the tokens that any of its rows sees."""
    if not case["causal"]:
        return n * length, length
    window = case["window"] or length
    return sum(min(window, p + 1) for p in range(length - n, length)), min(length, window + n - 1)


def work(case):
    e, counts = 2 if case["precision"] == "f16" else 4, _rows_of(case)
    rows = sum(counts)
    if case["kind"] == "append":
        width = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": rows * (2 * width * e + 4 * case["positions"]),
                "flops": rows * (case["heads"] + case["kv_heads"]) * case["rotary_dim"] * 3}
    if case["kind"] == "attention":
        seen = [_seen(case, n, length) for n, length in zip(counts, _lengths_of(case))]
        return {"bytes": (sum(x[1] for x in seen) * case["kv_heads"] + rows * case["heads"]) * 2 * case["head_dim"] * e,
                "flops": sum(x[0] for x in seen) * case["heads"] * case["head_dim"] * 4}
    drafts = rows - case["sequences"] if case["draft"] and case["mode"] == "sample" else 0
    return {"bytes": (rows + drafts) * case["columns"] * e + rows * 8 + case["sequences"] * 12,
            "flops": (rows + drafts) * case["columns"] * 4}


# ------------------------------------------------------------------ exact

def _exact_append(case, t):
    dim, page, half = case["head_dim"], case["page"], case["rotary_dim"] // 2
    rows, lengths = _rows_of(case), _lengths_of(case)
    position = torch.cat([torch.arange(length - n, length) for n, length in zip(rows, lengths)]).cuda()
    if half:
        angle = position if t["positions"] is None else t["positions"]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           angle.double()[:, None, None] * t["frequencies"].double())

    def rotate(x):
        x = x.double().reshape(len(position), -1, dim)
        if not half:
            return x
        part, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["pairs"] == "halves":
            both = torch.complex(part[..., :half], part[..., half:]) * turn[..., :half]
            return torch.cat([both.real, both.imag, rest], -1)
        both = torch.view_as_complex(part.reshape(len(x), -1, half, 2).contiguous()) * turn[..., :half]
        return torch.cat([torch.view_as_real(both).reshape(part.shape), rest], -1)

    keys, values = t["key_cache"].double(), t["value_cache"].double()
    number = torch.cat([t["page_table"][s].long()[torch.arange(length - n, length, device="cuda") // page]
                        for s, (n, length) in enumerate(zip(rows, lengths))])
    k, v = rotate(t["keys"]), t["values"].double().reshape(len(position), -1, dim)
    for h in range(case["kv_heads"]):
        keys[number, h, position % page] = k[:, h]
        values[number, h, position % page] = v[:, h]
    return {"rotated": rotate(t["queries"]).reshape(len(position), -1), "keys": keys, "values": values}


def _exact_attention(case, t):
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out, start = torch.zeros(sum(_rows_of(case)), heads, dim, dtype=torch.float64, device="cuda"), 0
    for s, (n, length) in enumerate(zip(_rows_of(case), _lengths_of(case))):
        token = torch.arange(length, device="cuda")
        number, place = t["page_table"][s].long()[token // page], token % page
        for h in range(heads):
            k, v = (t[c][number, h // (heads // kv), place].double() for c in ("key_cache", "value_cache"))
            q = t["queries"][start:start + n, h * dim:(h + 1) * dim].double()
            z = q @ k.T.contiguous() * dim ** -0.5
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            ahead = token[None] - torch.arange(length - n, length, device="cuda")[:, None]
            if case["causal"]:
                z[ahead > 0] = -INF
            if case["window"]:
                z[ahead <= -case["window"]] = -INF
            out[start:start + n, h] = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ v
        start += n
    return {"output": out.reshape(len(out), -1)}


def _exact_verify(case, t):
    accepted, chosen, temperature = [], [], case["temperature"]
    starts, tokens = _starts(_rows_of(case)), t["tokens"].tolist()
    uniforms, draws = t["uniforms"].tolist(), t["draws"].tolist()
    for s in range(case["sequences"]):
        taken = 0
        for row in range(starts[s], starts[s + 1]):
            z = t["target"][row].double()
            d = tokens[row + 1] if row + 1 < starts[s + 1] else None
            if case["mode"] == "greedy":
                w = (z == z.max()).double()
                token = int(torch.nonzero(w)[0])
                if d is None or token != d:
                    break
                taken += 1
                continue
            w = torch.softmax(z / temperature, 0)
            if d is not None:
                q = torch.zeros_like(w)
                if case["draft"]:
                    q = torch.softmax(t["draft"][row].double() / temperature, 0)
                else:
                    q[d] = 1
                if float(w[d]) > uniforms[row] * float(q[d]):
                    taken += 1
                    continue
                w = torch.relu(w - q)
            running = torch.cumsum(w, 0)
            token = int(torch.searchsorted(running, draws[s] * running[-1:], right=True))
            token = min(token, int(torch.nonzero(w)[-1]))
            break
        accepted.append(taken)
        chosen.append(token)
    return {"accepted": _ints(accepted), "next_tokens": _ints(chosen)}


def exact(case, seed):
    t = _inputs(case, seed)
    form = {"append": _exact_append, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]]
    return form(case, t)
