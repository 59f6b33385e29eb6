"""The verification of drafted tokens on the GPU. Its outputs are whole numbers
and have to be those of the formulas in float64: the numbers that decide are
set at a margin of 1e-9 of their borders, which both sides' roundings (some
1e-13 for sums of 131072 terms) cannot cross, and the margins are checked."""
import numpy as np
import pytest

from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu

NO_TOKEN = 0xFFFFFFFF
MARGIN = 1e-9


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


def probabilities(z, temperature):
    """softmax in float64, or None where there is none."""
    z = z.astype(np.float64) / temperature
    if np.isnan(z).any() or (z == np.inf).any() or (z == -np.inf).all():
        return None
    e = np.exp(z - z.max())
    return e / e.sum()


def formula(target, draft, tokens, starts, uniforms, draws, temperature, greedy, margins=None):
    """Accepted drafts and next tokens; `margins` collects the distances from the borders."""
    rows, columns = target.shape
    accepted, chosen = [], []
    margins = [] if margins is None else margins
    for s in range(len(starts) - 1):
        start, end = min(int(starts[s]), rows), min(int(starts[s + 1]), rows)
        taken, token = 0, NO_TOKEN
        for row in range(start, end):
            d = int(tokens[row + 1]) if row + 1 < end else NO_TOKEN
            last = d >= columns
            if greedy:
                z = target[row].astype(np.float64).copy()
                z[np.isnan(z)] = -np.inf
                token = int(np.argmax(z)) if z.max() > -np.inf else NO_TOKEN
                if last or token != d:
                    break
                taken += 1
                continue
            p = probabilities(target[row], temperature)
            q = None
            if draft is None:
                q = np.zeros(columns)
                if not last:
                    q[d] = 1
            elif not last:
                q = probabilities(draft[row], temperature)
            if p is None or (q is None and not last):
                token = NO_TOKEN
                break
            if not last:
                if np.isfinite(uniforms[row]) and (p[d] or q[d]):  # two zeros are exact
                    margins.append(abs(float(uniforms[row]) * q[d] - p[d]) / max(p[d], 1e-300))
                if float(uniforms[row]) * q[d] < p[d]:
                    taken += 1
                    continue
            w = p if last else np.maximum(p - q, 0)
            if w.sum() == 0:
                w = p
            running = np.cumsum(w)
            draw = float(draws[s])
            if draw > 0 and draw < 1:
                margins.append(np.abs(running / running[-1] - draw).min())
                token = int(np.argmax((running > draw * running[-1]) & (w > 0)))
            else:
                live = np.flatnonzero(w > 0)
                token = int(live[0] if draw <= 0 else live[-1])
            break
        accepted.append(taken)
        chosen.append(token)
    return np.array(accepted, np.uint32), np.array(chosen, np.uint32)


def make(rng, dtype, counts, columns, agreement=0.5, stride=0, temperature=1.0, drafted=True):
    """Logits of target and draft that agree to some extent, drafts drawn from the draft's."""
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    rows, stride = max(1, int(starts[-1])), stride or columns
    base = rng.standard_normal((rows, stride)) * 2
    base[np.arange(rows), rng.integers(0, columns, rows)] += rng.random(rows) * 14
    draft, target = ((base + rng.standard_normal((rows, stride)) * (1 - agreement)).astype(dtype) for _ in range(2))
    race = draft[:, :columns].astype(np.float64) / temperature
    if drafted:
        race = race - np.log(-np.log(rng.random((rows, columns)).clip(1e-12, 1 - 1e-12)))
    best = race.argmax(1)
    tokens = np.concatenate([[0], best[:-1]]).astype(np.uint32)
    return dict(target=target, draft=draft if drafted else None, tokens=tokens, starts=starts,
                uniforms=rng.random(rows).astype(np.float32), draws=rng.random(len(counts)).astype(np.float32),
                columns=columns)


def run(abi, ctx, scope, case, temperature=None, greedy=False, active=0, repeat=1):
    put = scope.put
    sequences = len(case["starts"]) - 1
    accepted, chosen = (put(np.full(sequences, 77, np.uint32)) for _ in range(2))
    target, draft = case["target"], case["draft"]
    op = abi.DraftVerifyOp(
        ctx, target=put(target), target_stride=target.shape[1], draft=put(draft) if not greedy else None,
        draft_stride=0 if draft is None else draft.shape[1], rows=target.shape[0], sequences=sequences,
        columns=case["columns"], row_starts=put(case["starts"]), tokens=put(case["tokens"]),
        uniforms=None if greedy else put(case["uniforms"]), draws=None if greedy else put(case["draws"]),
        accepted=accepted, next_tokens=chosen, temperature=temperature, mode="greedy" if greedy else "sample")
    for _ in range(repeat):
        op.enqueue(active)
    ctx.synchronize()
    op.release()
    return accepted.download(), chosen.download()


def check(abi, ctx, scope, case, temperature=None, greedy=False, active=0, repeat=1):
    n, margins = case["columns"], []
    # The formulas use the temperature that the op is given, an f32.
    want = formula(case["target"][:, :n], None if case["draft"] is None else case["draft"][:, :n], case["tokens"],
                   case["starts"], case["uniforms"], case["draws"], float(np.float32(temperature or 1.0)), greedy, margins)
    assert not margins or min(margins) > MARGIN, "the inputs lie on a border"
    got = run(abi, ctx, scope, case, temperature, greedy, active, repeat)
    live = slice(0, active or None)
    np.testing.assert_array_equal(got[0][live], want[0][live])
    np.testing.assert_array_equal(got[1][live], want[1][live])
    if active:
        assert (got[0][active:] == 77).all() and (got[1][active:] == 77).all()
    return want


DTYPES = pytest.mark.parametrize("dtype", [np.float16, np.float32])


@DTYPES
@pytest.mark.parametrize("columns", [1, 2, 3, 64, 255, 1025, 8191, 8192, 8193, 32000])
@pytest.mark.parametrize("drafted", [True, False])
def test_sizes(abi, ctx, scope, dtype, columns, drafted):
    rng = np.random.default_rng(columns)
    want = check(abi, ctx, scope, make(rng, dtype, [5, 1, 8, 3, 2, 0, 7], columns, drafted=drafted))
    if columns > 2 and drafted:
        assert want[0].max() > 0


@DTYPES
@pytest.mark.parametrize("columns", [5, 1025, 20000])
def test_greedy(abi, ctx, scope, dtype, columns):
    rng = np.random.default_rng(columns)
    case = make(rng, dtype, [5, 1, 8, 3, 2, 0, 7], columns, agreement=0.9, drafted=False)
    check(abi, ctx, scope, case, greedy=True)
    case["target"][:] = rng.integers(-2, 3, case["target"].shape)  # many equal logits: the lowest index
    best = case["target"][:, :columns].argmax(1)
    case["tokens"][1:] = best[:-1]
    want = check(abi, ctx, scope, case, greedy=True)
    assert list(want[0]) == [4, 0, 7, 2, 1, 0, 6]
    case["target"][3] = -np.inf
    case["target"][6, :] = np.nan
    case["target"][7, columns // 2] = np.inf
    case["target"][8, :columns - 1] = -0.0
    case["target"][8, columns - 1:] = 0.0
    check(abi, ctx, scope, case, greedy=True)


@DTYPES
def test_large_vocabulary(abi, ctx, scope, dtype):
    rng = np.random.default_rng(9)
    for counts in ([4], [3, 8, 5]):
        check(abi, ctx, scope, make(rng, dtype, counts, 131072, temperature=0.8), temperature=0.8)


@DTYPES
@pytest.mark.parametrize("columns", [1025, 40000])
def test_flat_rows(abi, ctx, scope, dtype, columns):
    """Flat distributions: many tokens of nearly one probability, a border every 1 / V."""
    rng = np.random.default_rng(columns)
    case = make(rng, dtype, [3] * 12, columns, drafted=True)
    for name in ("target", "draft"):
        case[name][:] = rng.standard_normal(case[name].shape) * 0.01
    check(abi, ctx, scope, case)


@DTYPES
@pytest.mark.parametrize("stride,temperature", [(1032, 0.5), (1026, 1.7), (1040, 2.0 ** -20), (1033, 2.0 ** 20)])
def test_strides_and_temperatures(abi, ctx, scope, dtype, stride, temperature):
    rng = np.random.default_rng(stride)
    check(abi, ctx, scope, make(rng, dtype, [4, 6], 1025, stride=stride, temperature=temperature), temperature=temperature)


@DTYPES
def test_many_sequences(abi, ctx, scope, dtype):
    rng = np.random.default_rng(10)
    check(abi, ctx, scope, make(rng, dtype, list(rng.integers(0, 6, 300)), 129))
    check(abi, ctx, scope, make(rng, dtype, [40], 700, agreement=1.0))  # all accepted but by chance
    check(abi, ctx, scope, make(rng, dtype, [3, 4, 5], 700), active=2, repeat=3)


@DTYPES
@pytest.mark.parametrize("columns", [300, 20000])
def test_same_logits_accept_all(abi, ctx, scope, dtype, columns):
    case = make(np.random.default_rng(11), dtype, [6, 2], columns)
    case["draft"] = case["target"].copy()
    case["uniforms"][:] = np.float32(1 - 2.0 ** -24)
    n = case["columns"]
    got = run(abi, ctx, scope, case)
    assert list(got[0]) == [5, 1]
    case["uniforms"][:] = 2.0  # beyond the range: refused, and p nowhere above q, so drawn from p
    case["draws"][:] = [0.25, 0.75]
    got = run(abi, ctx, scope, case)
    assert list(got[0]) == [0, 0]
    for s, row in enumerate((0, 6)):
        running = np.cumsum(probabilities(case["target"][row, :n], 1.0))
        assert got[1][s] == np.argmax(running > case["draws"][s] * running[-1])


@DTYPES
@pytest.mark.parametrize("columns", [50, 12000])
def test_masked_and_strange_rows(abi, ctx, scope, dtype, columns):
    rng = np.random.default_rng(12)
    case = make(rng, dtype, [3, 3, 3, 3, 3, 3, 3, 3], columns)
    target, draft = case["target"], case["draft"]
    mask = rng.random(target.shape) < 0.6
    mask[np.arange(len(mask))[:-1], case["tokens"][1:]] = False
    mask[:, 0] = False
    target[mask] = -np.inf
    target[3, case["tokens"][4]] = -np.inf    # a masked draft
    target[6] = -np.inf                       # nothing left
    target[9, 1] = np.nan
    target[12, 2] = np.inf
    draft[15] = -np.inf
    draft[18, 0] = np.nan
    case["tokens"][22] = columns              # no draft: its row is the last
    check(abi, ctx, scope, case)
    draft[21] = np.nan                        # not read then
    check(abi, ctx, scope, case)


@DTYPES
def test_ends_of_the_ranges(abi, ctx, scope, dtype):
    case = make(np.random.default_rng(13), dtype, [2] * 8, 500)
    case["uniforms"][::2] = [0, 0, 1, 1, np.nan, np.inf, -1, 0.5]
    case["draws"][:] = [0, 1, 0, np.nan, 2, -1, np.inf, -np.inf]
    case["uniforms"][4:8] = 1.0
    check(abi, ctx, scope, case)


@DTYPES
def test_lowest_numbers(abi, ctx, scope, dtype):
    """A mask of the type's lowest number, and differences beyond f32."""
    case = make(np.random.default_rng(14), dtype, [3, 4], 600)
    low = np.finfo(dtype).min
    case["target"][:, ::2] = low
    case["draft"][:, ::2] = low
    case["target"][4] = low
    case["target"][5] = np.where(np.arange(600) < 300, low, -low if dtype == np.float32 else 60000)
    check(abi, ctx, scope, case)


def test_starts_are_cut_to_the_rows(abi, ctx, scope):
    case = make(np.random.default_rng(15), np.float16, [3, 4, 2], 100)
    case["starts"][3] = 5000
    check(abi, ctx, scope, case)
    case["starts"][1:] = [9, 9, 9]
    check(abi, ctx, scope, case)
