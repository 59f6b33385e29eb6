"""The paged cache on the GPU against the formulas in float64: appended rows with
their rotation, and the attention of new tokens over what the cache holds.

Tolerances count roundings. Append: sine, cosine, the two products and their sum
round once each, so an output is within 3 * 2^-24 (|x| + |y|) of the formula; 4 *
2^-24 are allowed, and its own rounding adds half a step. Attention: a score
is a sum of D products in f32 (D * 2^-24 of the sum of their magnitudes, of f16
inputs exact products), scaled and, with a cap, through tanh (2^-20 of the cap);
with an error delta of every score, the weights move by a factor within 1 +- 2
delta. f16 rows round each weight by 2^-11 (and weights below 2^-14 of the
running maximum by 2^-25 of it), sums of n terms in f32 add up their n roundings,
which are independent, to 4 sqrt(n) * 2^-24, and the output's rounding adds half a
step: all relative to sum(p |v|) / sum(p), the weights' least step to max |v| / sum(p)."""
import numpy as np
import pytest

from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu

NO_PAGE = 0xFFFFFFFF
HALF_STEP = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24}


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


class Cache:
    """Host copies of a cache and the tables of some sequences."""

    def __init__(self, rng, dtype, counts, lengths, kv_heads, dim, page_size, spare=3, page_stride=0, width=0):
        self.dtype, self.kv_heads, self.dim, self.page_size = dtype, kv_heads, dim, page_size
        self.counts, self.lengths = list(counts), np.array(lengths, np.uint32)
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
        self.rows, self.sequences = int(self.starts[-1]), len(self.counts)
        held = [-(-int(n) // page_size) for n in lengths]
        self.width = max(held + [1, width])
        self.pages = sum(held) + spare
        order = iter(rng.permutation(self.pages))
        self.table = np.full((self.sequences, self.width), NO_PAGE, np.uint32)
        for s, n in enumerate(held):
            self.table[s, :n] = [next(order) for _ in range(n)]
        page = kv_heads * page_size * dim
        self.page_stride = page_stride or page
        shape = (self.pages - 1) * self.page_stride + page
        self.keys, self.values = (rng.standard_normal(shape).astype(dtype) for _ in range(2))

    def place(self, s, token):
        """The element of kv head 0 of a token, or None."""
        if token < 0 or token // self.page_size >= self.width:
            return None
        page = int(self.table[s, token // self.page_size])
        return page * self.page_stride + token % self.page_size * self.dim if page < self.pages else None

    def head(self, cache, s, kv, tokens):
        """Rows of the tokens that have a place, and those tokens."""
        held = [t for t in tokens if self.place(s, t) is not None]
        at = np.array([self.place(s, t) for t in held], np.int64) + kv * self.page_size * self.dim
        return cache[at[:, None] + np.arange(self.dim)].reshape(-1, self.dim).astype(np.float64), np.array(held, np.int64)

    def put(self, scope):
        self.device = {"key_cache": scope.put(self.keys), "value_cache": scope.put(self.values),
                       "row_starts": scope.put(self.starts), "lengths": scope.put(self.lengths),
                       "page_table": scope.put(self.table)}
        return dict(self.device, rows=self.rows, sequences=self.sequences, kv_heads=self.kv_heads, head_dim=self.dim,
                    pages_per_sequence=self.width, pages=self.pages, page_size=self.page_size,
                    page_stride=self.page_stride)

    def start(self, s):
        return min(int(self.starts[s]), self.rows)

    def row_positions(self, active=None):
        return [(s, r, int(self.lengths[s]) - self.start(s + 1) + r)
                for s in range(self.sequences if active is None else active) for r in range(self.start(s), self.start(s + 1))]


# ------------------------------------------------------------------- append


def rotate(x, angle, kind):
    """float64 rotation of [heads, dim] by the angles of its pairs."""
    out, half = x.astype(np.float64), len(angle)
    first, second = ((slice(0, half), slice(half, 2 * half)) if kind == "halves" else
                     (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    a, b = out[:, first].copy(), out[:, second].copy()
    out[:, first] = a * np.cos(angle) - b * np.sin(angle)
    out[:, second] = b * np.cos(angle) + a * np.sin(angle)
    size = np.abs(x.astype(np.float64))
    size[:, first] = size[:, second] = np.abs(a) + np.abs(b)
    return out, size


def exact_angle(position, frequencies):
    """position * frequency less whole turns: in long double, whose 64 bits hold
    the product exactly, with 1 / (2 pi) to 128 bits in two parts."""
    a = np.longdouble(int(position)) * frequencies.astype(np.longdouble)
    high = np.longdouble(0.15915494309189535)
    low = np.longdouble(-9.839338337591835e-18)
    turns = a * high
    whole = np.rint(turns)
    return ((turns - whole) + a * low).astype(np.float64) * (2 * np.pi)


def check_append(cache, got, queries, keys, values, frequencies, kind, positions=None, heads=0, active=None, error=2.0 ** -22):
    """`got`: query output, keys and values of the caches."""
    dtype, dim, kv, half = cache.dtype, cache.dim, cache.kv_heads, HALF_STEP[cache.dtype]
    want_keys, want_values = cache.keys.copy(), cache.values.copy()
    key_size = np.zeros(len(want_keys))
    exact_keys = want_keys.astype(np.float64)
    want_queries = None if not heads else np.zeros((cache.rows, heads * dim))
    for s, r, p in cache.row_positions(active):
        if p < 0:
            continue
        angle = exact_angle(p if positions is None else positions[r], frequencies)
        if heads:
            exact, size = rotate(queries[r].reshape(heads, dim), angle, kind)
            bound = half * np.abs(exact) + error * size + np.finfo(dtype).smallest_subnormal
            off = np.abs(got[0][r].reshape(heads, dim).astype(np.float64) - exact) / bound
            assert off.max() <= 1, (s, r)
            want_queries[r] = 1
        at = cache.place(s, p)
        if at is None:
            continue
        exact, size = rotate(keys[r].reshape(kv, dim), angle, kind)
        for h in range(kv):
            run = slice(at + h * cache.page_size * dim, at + h * cache.page_size * dim + dim)
            exact_keys[run], key_size[run] = exact[h], size[h]
            want_values[run] = values[r].reshape(kv, dim)[h]
    np.testing.assert_array_equal(got[2], want_values)
    touched = key_size > 0
    np.testing.assert_array_equal(got[1][~touched], want_keys[~touched])
    bound = half * np.abs(exact_keys) + error * key_size + np.finfo(dtype).smallest_subnormal
    off = np.abs(got[1].astype(np.float64) - exact_keys) / bound
    assert off.max() <= 1
    return want_queries


def make_rows(rng, cache, heads, packed=False, wide=0, offset=0):
    """Queries, keys and values as arrays of rows, and where they lie: parts of
    one buffer, or buffers of their own with `wide` more columns."""
    dim, kv, rows, dtype = cache.dim, cache.kv_heads, cache.rows, cache.dtype
    widths = [heads * dim, kv * dim, kv * dim]
    if packed:
        both = rng.standard_normal((rows, sum(widths))).astype(dtype)
        return np.split(both, np.cumsum(widths)[:-1], axis=1), both, widths
    return [rng.standard_normal((rows, w + wide)).astype(dtype)[:, :w] for w in widths], None, widths


class Slice:
    def __init__(self, array, offset, nbytes, dtype):
        self.ptr, self.nbytes, self.dtype = array.ptr + offset, nbytes, np.dtype(dtype)


def run_append(abi, ctx, scope, rng, dtype, counts, lengths, heads, kv_heads, dim, page_size, rotary_dim, kind="halves",
               positions=None, packed=False, in_place=False, wide=0, offset=0, page_stride=0, active=0, spoil=None,
               stride_pages=False):
    cache = Cache(rng, dtype, counts, lengths, kv_heads, dim, page_size, page_stride=page_stride)
    if spoil:
        spoil(cache)
    e = np.dtype(dtype).itemsize
    frequencies = (10000.0 ** (-np.arange(rotary_dim // 2) / max(1, rotary_dim // 2))).astype(np.float32)
    (q, k, v), both, widths = make_rows(rng, cache, heads, packed)
    kw = cache.put(scope)
    if packed:
        row = sum(widths)
        device = scope.put(both)
        at = np.concatenate([[0], np.cumsum(widths)]) * e
        binds = [Slice(device, int(at[i]), both.nbytes - int(at[i]), dtype) for i in range(3)]
        strides = [row] * 3
    else:
        binds, strides = [], []
        for x, w in zip((q, k, v), widths):
            host = np.zeros(cache.rows * (w + wide) + offset, dtype)
            host[offset:].reshape(cache.rows, w + wide)[:, :w] = x
            device = scope.put(host) if host.size else None
            binds.append(Slice(device, offset * e, host.nbytes - offset * e, dtype) if w else None)
            strides.append(w + wide)
    output = binds[0] if in_place else (scope.put(np.full((cache.rows, max(heads, 1) * dim), 7, dtype)) if heads else None)
    op = abi.CacheAppendOp(
        ctx, keys=binds[1], key_stride=strides[1], values=binds[2], value_stride=strides[2], heads=heads,
        queries=binds[0] if heads else None, query_stride=strides[0] if heads else 0, query_output=output,
        query_output_stride=strides[0] if in_place else 0, rotary_dim=rotary_dim, rotary=kind,
        frequencies=scope.put(frequencies) if rotary_dim else None,
        positions=scope.put(np.array(positions, np.uint32)) if positions is not None else None, **kw)
    op.enqueue(active)
    ctx.synchronize()
    op.release()
    if in_place:
        assert packed
        out = device.download()[:, :widths[0]]
        np.testing.assert_array_equal(device.download()[:, widths[0]:], both[:, widths[0]:])
    else:
        out = output.download() if heads else None
    got = [out, cache.device["key_cache"].download(), cache.device["value_cache"].download()]
    done = check_append(cache, got, q, k, v, frequencies, kind, positions, heads, active or None)
    if heads:  # rows without a sequence or a position are left as they were
        before = q if in_place else np.full((cache.rows, heads * dim), 7, dtype)
        np.testing.assert_array_equal(out[done[:, 0] == 0], before[done[:, 0] == 0])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary_dim,kind", [
    (8, 8, 128, 128, "halves"), (4, 1, 64, 64, "neighbours"), (5, 5, 80, 32, "halves"), (6, 2, 40, 40, "neighbours"),
    (2, 1, 256, 256, "halves"), (3, 3, 8, 6, "halves"), (0, 2, 96, 48, "neighbours"), (4, 2, 72, 0, "halves"),
    (4, 4, 32, 2, "neighbours"), (1, 1, 24, 20, "halves")])
@pytest.mark.parametrize("packed", [False, True])
def test_append(abi, ctx, scope, dtype, heads, kv_heads, dim, rotary_dim, kind, packed):
    rng = np.random.default_rng(dim + heads)
    run_append(abi, ctx, scope, rng, dtype, [1, 7, 0, 19, 3], [1, 30, 9, 19, 100], heads, kv_heads, dim, 16, rotary_dim,
               kind, packed=packed and heads > 0)


@pytest.mark.parametrize("page_size", [1, 3, 16, 100, 65536])
def test_append_page_sizes(abi, ctx, scope, page_size):
    run_append(abi, ctx, scope, np.random.default_rng(page_size), np.float16, [33, 2], [70, 2], 2, 1, 16, page_size, 16)


def test_append_far_positions(abi, ctx, scope):
    """Positions up to 2^32 - 1: the angle is reduced before it is rounded."""
    positions = [0, 1, 2 ** 16 + 1, 2 ** 24 + 1, 2 ** 30 + 3, 2 ** 31 - 1, 2 ** 32 - 1]
    for kind in ("halves", "neighbours"):
        run_append(abi, ctx, scope, np.random.default_rng(5), np.float32, [3, 4], [50, 4], 2, 2, 128, 16, 128, kind,
                   positions=positions)


def test_append_in_place_and_strided(abi, ctx, scope):
    rng = np.random.default_rng(6)
    for dtype in (np.float16, np.float32):
        run_append(abi, ctx, scope, rng, dtype, [5, 40], [5, 41], 4, 2, 64, 16, 64, packed=True, in_place=True)
        run_append(abi, ctx, scope, rng, dtype, [5, 40], [5, 41], 4, 2, 64, 16, 64, "neighbours", packed=True, in_place=True)
        for wide, offset in ((3, 1), (8, 0), (4, 4), (1, 0)):  # rows and buffers at any element
            run_append(abi, ctx, scope, rng, dtype, [2, 9], [20, 9], 3, 1, 64, 16, 32, wide=wide, offset=offset)


def test_append_page_stride(abi, ctx, scope):
    run_append(abi, ctx, scope, np.random.default_rng(7), np.float16, [9, 30], [9, 64], 2, 2, 32, 8, 32,
               page_stride=2 * 2 * 8 * 32 + 8)


def test_append_active_and_odd_tables(abi, ctx, scope):
    """Rows behind the active sequences, pages that are none, lengths below the
    rows and beyond the table: nothing but what has a place is written."""
    rng = np.random.default_rng(8)
    run_append(abi, ctx, scope, rng, np.float16, [4, 9, 5, 1], [4, 20, 50, 8], 2, 1, 64, 16, 64, active=2)

    def spoil(cache):
        cache.table[1, 0] = NO_PAGE
        cache.table[2, 1] = cache.pages
        cache.lengths[0] = 2       # below its 4 rows
        cache.lengths[3] = 70      # 16 * 4 places
        cache.starts[5] = 4000     # cut to the rows
    run_append(abi, ctx, scope, rng, np.float32, [4, 9, 5, 8, 3], [4, 20, 30, 60, 8], 2, 1, 64, 16, 64, spoil=spoil)


# ---------------------------------------------------------------- attention


def attention_rows(cache, queries, heads, causal=True, window=0, scale=None, cap=0.0, active=None):
    """Of each row: the output [heads, dim], sum(p |v|) / sum(p), the largest sum
    |q k|, and count * max |v| / sum(p)."""
    dim, group = cache.dim, heads // cache.kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = np.zeros((cache.rows, heads, dim))
    size, slack, least = np.zeros_like(out), np.zeros((cache.rows, heads, 1)), np.zeros((cache.rows, heads, 1))
    parts = {}
    for s, r, p in cache.row_positions(active):
        if s not in parts:
            held = range(min(int(cache.lengths[s]), cache.width * cache.page_size))
            parts[s] = [[cache.head(c, s, h, held) for c in (cache.keys, cache.values)] for h in range(cache.kv_heads)]
        for h in range(heads):
            (k, tokens), (v, _) = parts[s][h // group]
            keep = np.ones(len(tokens), bool)
            if causal:
                keep &= tokens <= p
                if window:
                    keep &= tokens > p - window
            if not keep.any():
                continue
            q, k, v = queries[r].reshape(heads, dim)[h].astype(np.float64), k[keep], v[keep]
            z = k @ q * scale
            slack[r, h] = (np.abs(k) @ np.abs(q)).max() * abs(scale)
            if cap:
                z = cap * np.tanh(z / cap)
            e = np.exp(z - z.max())
            out[r, h] = e @ v / e.sum()
            size[r, h] = e @ np.abs(v) / e.sum()
            least[r, h] = len(e) * np.abs(v).max() / e.sum()
    return out, size, slack, least


def check_attention(cache, got, queries, heads, active=None, **kw):
    want, size, slack, least = attention_rows(cache, queries, heads, active=active, **kw)
    half, most = HALF_STEP[cache.dtype], float(cache.lengths.max())
    score = (cache.dim + 4) * 2.0 ** -24 * slack + (kw.get("cap", 0.0) or 0.0) * 2.0 ** -20
    weights = 2 * score + (8 + most ** 0.5 * 4) * 2.0 ** -24
    if cache.dtype == np.float16:
        weights = weights + 2.0 ** -11
        least = least * 2.0 ** -25
    else:
        least = 0
    bound = half * np.abs(want) + (1 + half) * (weights * size + least) + np.finfo(cache.dtype).smallest_subnormal
    rows = cache.start(cache.sequences if active is None else active)
    got = got.reshape(cache.rows, heads, cache.dim).astype(np.float64)
    assert np.isfinite(got[:rows]).all()
    if not rows:
        return
    off = (np.abs(got - want) / bound)[:rows]
    assert off.max() <= 1, np.argwhere(off > 1)[:4]


def run_attention(abi, ctx, scope, rng, dtype, counts, lengths, heads, kv_heads, dim, page_size, page_stride=0, width=0,
                  query_std=2.0, wide=0, offset=0, active=0, spoil=None, check=True, **kw):
    cache = Cache(rng, dtype, counts, lengths, kv_heads, dim, page_size, page_stride=page_stride, width=width)
    queries = (rng.standard_normal((cache.rows, heads * dim)) * query_std).astype(dtype)
    if spoil:
        spoil(cache, queries)
    e, row = np.dtype(dtype).itemsize, heads * dim + wide
    host = np.zeros(cache.rows * row + offset, dtype)
    host[offset:].reshape(cache.rows, row)[:, :heads * dim] = queries
    device = scope.put(host)
    filled = np.full(cache.rows * row + offset, 7, dtype)
    output = scope.put(filled)
    at = lambda x: Slice(x, offset * e, host.nbytes - offset * e, dtype)
    op = abi.CacheAttentionOp(ctx, queries=at(device), query_stride=row, output=at(output), output_stride=row, heads=heads,
                              causal=kw.get("causal", True), window=kw.get("window", 0), scale=kw.get("scale"),
                              score_cap=kw.get("cap"), **cache.put(scope))
    op.enqueue(active)
    ctx.synchronize()
    op.release()
    whole = output.download()
    got = whole[offset:].reshape(cache.rows, row)
    assert (whole[:offset] == 7).all() and (got[:, heads * dim:] == 7).all()
    if active:
        assert (got[int(cache.starts[active]):] == 7).all()
    if check:
        check_attention(cache, got[:, :heads * dim], queries, heads, active or None, **kw)
    return cache, got[:, :heads * dim], queries


DTYPES = pytest.mark.parametrize("dtype", [np.float16, np.float32])


@DTYPES
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 128), (8, 2, 128), (6, 1, 64), (5, 5, 80), (7, 1, 40), (2, 2, 256),
                                                (3, 1, 192), (32, 1, 32), (1, 1, 8), (4, 2, 96)])
def test_decode(abi, ctx, scope, dtype, heads, kv_heads, dim):
    """One new token each, of sequences from one token on."""
    rng = np.random.default_rng(heads * dim)
    lengths = [1, 2, 15, 16, 17, 33, 64, 100, 257, 700]
    run_attention(abi, ctx, scope, rng, dtype, [1] * len(lengths), lengths, heads, kv_heads, dim, 16)


@DTYPES
@pytest.mark.parametrize("page_size", [1, 3, 8, 24, 64, 100, 1000])
def test_pages(abi, ctx, scope, dtype, page_size):
    run_attention(abi, ctx, scope, np.random.default_rng(page_size), dtype, [1, 5, 40], [300, 77, 150], 4, 2, 64, page_size,
                  page_stride=2 * page_size * 64 * 2 + 8)


@DTYPES
@pytest.mark.parametrize("counts,lengths,heads,kv_heads,dim", [
    ([3, 8, 1, 5], [200, 8, 1, 90], 4, 1, 64), ([17, 31], [300, 31], 2, 2, 128), ([64], [64], 4, 2, 128),
    ([130, 1, 65], [130, 500, 400], 4, 2, 128), ([33], [700], 3, 1, 80), ([200], [333], 6, 2, 256), ([70], [70], 1, 1, 8),
    ([150, 0, 20], [151, 50, 21], 5, 1, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(abi, ctx, scope, dtype, counts, lengths, heads, kv_heads, dim, causal):
    """Several new tokens of a sequence, with what it holds before them and without."""
    rng = np.random.default_rng(dim + counts[0])
    run_attention(abi, ctx, scope, rng, dtype, counts, lengths, heads, kv_heads, dim, 16, causal=causal)


@DTYPES
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("page_size", [1, 7, 16, 24, 48, 100])
def test_pages_of_chunks(abi, ctx, scope, dtype, dim, page_size):
    """Pages that end inside a tile, or hold some of its tokens, a page that is missing, and what lies behind a sequence."""
    def spoil(cache, queries):
        held = np.zeros(cache.pages * page_size, bool)
        for s in range(cache.sequences):
            for t in range(int(cache.lengths[s])):
                held[cache.table[s, t // page_size] * page_size + t % page_size] = True
        for x in (cache.keys, cache.values):
            rows = x.reshape(cache.pages, 2, page_size, dim)
            rows[~np.repeat(held.reshape(cache.pages, 1, page_size), 2, 1)] = np.nan
        cache.table[0, 30 // page_size] = NO_PAGE
    run_attention(abi, ctx, scope, np.random.default_rng(dim + page_size), dtype, [140, 66, 3], [150, 200, 77], 4, 2, dim,
                  page_size, spoil=spoil)


@DTYPES
@pytest.mark.parametrize("counts", [[1, 1, 1], [6, 3, 1], [90, 40, 3]])
@pytest.mark.parametrize("window", [1, 5, 32, 100, 10000])
def test_windows(abi, ctx, scope, dtype, counts, window):
    rng = np.random.default_rng(window)
    run_attention(abi, ctx, scope, rng, dtype, counts, [300, 64, 5], 4, 2, 64, 24, window=window)


@DTYPES
@pytest.mark.parametrize("counts", [[1, 1], [70, 4]])
@pytest.mark.parametrize("cap,std", [(30.0, 2.0), (2.0, 8.0), (1.0, 0.01)])
def test_caps(abi, ctx, scope, dtype, counts, cap, std):
    run_attention(abi, ctx, scope, np.random.default_rng(int(cap)), dtype, counts, [200, 90], 2, 1, 128, 16, cap=cap,
                  query_std=std)


@DTYPES
def test_scales_and_large_scores(abi, ctx, scope, dtype):
    """One token takes all: scores of hundreds, falling and rising along the sequence."""
    rng = np.random.default_rng(4)
    for counts in ([1, 1], [40, 80]):
        run_attention(abi, ctx, scope, rng, dtype, counts, [400, 90], 2, 2, 64, 16, scale=0.0)
        run_attention(abi, ctx, scope, rng, dtype, counts, [400, 90], 2, 2, 64, 16, scale=-1.5)

        def slope(sign):
            def spoil(cache, queries):
                for s in range(2):
                    for t in range(int(cache.lengths[s])):
                        for h in range(2):
                            at = cache.place(s, t) + h * 16 * 64
                            cache.keys[at] = sign * t
                queries[:, ::64] = 2
            return spoil
        for sign in (1, -1):
            run_attention(abi, ctx, scope, rng, dtype, counts, [400, 90], 2, 2, 64, 16, spoil=slope(sign), query_std=0.1)


@DTYPES
def test_strides_and_offsets(abi, ctx, scope, dtype):
    rng = np.random.default_rng(11)
    for counts in ([1, 1], [40, 5]):
        for wide, offset in ((3, 1), (8, 8), (0, 1), (4, 2)):
            run_attention(abi, ctx, scope, rng, dtype, counts, [70, 50], 2, 1, 64, 16, wide=wide, offset=offset)


@DTYPES
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [5, 9, 4, 30]])
def test_active_sequences(abi, ctx, scope, dtype, counts):
    run_attention(abi, ctx, scope, np.random.default_rng(12), dtype, counts, [70, 50, 300, 31], 2, 1, 64, 16, active=2)


@DTYPES
@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [7, 3, 9, 4, 6], [60, 40, 33, 70, 5]])
def test_missing_pages_and_odd_lengths(abi, ctx, scope, dtype, counts):
    """Tokens without a page are hidden, a sequence without any gives zeros, rows
    before position 0 too; lengths may pass the table."""
    def spoil(cache, queries):
        cache.table[0, 1] = NO_PAGE
        cache.table[0, 3] = cache.pages
        cache.table[1, :] = NO_PAGE
        cache.lengths[2] = 0
        cache.lengths[3] = 2000   # 20 * 16 places
        cache.lengths[4] = max(1, counts[4] // 2)
    for causal in (True, False):
        run_attention(abi, ctx, scope, np.random.default_rng(13), dtype, counts, [100, 64, 80, 320, 90], 4, 2, 64, 16,
                      spoil=spoil, causal=causal)


@DTYPES
@pytest.mark.parametrize("counts", [[1], [4], [20], [90]])
def test_hidden_infinities_and_nan(abi, ctx, scope, dtype, counts):
    """What a row does not see does not touch it: places behind the length, pages
    of others, tokens before a window, and tokens behind a row of the chunk."""
    def spoil(cache, queries):
        seen = {cache.place(0, t) // 64 for t in range(int(cache.lengths[0]))}
        for name in ("keys", "values"):
            x = getattr(cache, name).reshape(-1, 64)
            heads = 2
            for row in range(len(x)):
                page, place = divmod(row, heads * 16)
                if (page * heads * 16 + place % 16) not in seen:
                    x[row] = (np.nan, np.inf, -np.inf)[row % 3]
    run_attention(abi, ctx, scope, np.random.default_rng(14), dtype, counts, [118], 4, 2, 64, 16, spoil=spoil)
    length, n = 118, counts[0]

    def newest(cache, queries):  # the newest token's values and keys are not numbers: only the last row sees them
        for h in range(2):
            at = cache.place(0, length - 1) + h * 16 * 64
            cache.values[at:at + 64] = np.nan
            cache.keys[at:at + 64] = np.inf
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(15), dtype, counts, [length], 4, 2, 64, 16,
                                        spoil=newest, check=False)
    assert np.isnan(got[n - 1].astype(np.float64)).all()
    if n > 1:
        cache.rows, cache.counts = n - 1, [n - 1]
        cache.starts = np.array([0, n - 1], np.uint32)
        cache.lengths = np.array([length - 1], np.uint32)
        check_attention(cache, got[:n - 1], queries[:n - 1], 4)

    def old(cache, queries):  # a token that only the first rows see, in front of the others' windows
        for h in range(2):
            at = cache.place(0, length - n - 9) + h * 16 * 64
            cache.values[at:at + 64] = np.inf
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(16), dtype, counts, [length], 4, 2, 64, 16,
                                        spoil=old, check=False, window=10)
    assert not np.isfinite(got[0].astype(np.float64)).any()
    if n > 1:
        cache.starts = np.array([0, n - 1], np.uint32)
        cache.rows, cache.counts = n - 1, [n - 1]
        check_attention(cache, got[1:], queries[1:], 4, window=10)


@DTYPES
def test_nan_in_a_query_stays_in_its_row(abi, ctx, scope, dtype):
    for counts in ([3, 1], [50, 2]):
        def spoil(cache, queries):
            queries[1, 64:128] = np.nan
        cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(17), dtype, counts, [80, 20], 4, 2, 64,
                                            16, spoil=spoil, check=False)
        assert np.isnan(got[1, 64:128].astype(np.float64)).all()
        queries[1, 64:128] = 0
        want = attention_rows(cache, queries, 4)[0].reshape(cache.rows, -1)
        got = got.astype(np.float64).copy()
        got[1, 64:128] = want[1, 64:128]
        check_attention(cache, got.astype(dtype), queries, 4)


@DTYPES
@pytest.mark.parametrize("counts,lengths,width", [([1], [20000], 0), ([1, 1, 1], [9000, 3, 5000], 4000),
                                                  ([3, 40], [6000, 9000], 0), ([129, 1], [3000, 9000], 1000)])
def test_long(abi, ctx, scope, dtype, counts, lengths, width):
    run_attention(abi, ctx, scope, np.random.default_rng(lengths[0]), dtype, counts, lengths, 4, 1, 64, 16, width=width)


@DTYPES
@pytest.mark.parametrize("sequences,most_rows,longest", [(64, 1, 700), (65, 1, 700), (65, 40, 90), (130, 3, 400), (1100, 1, 60)])
def test_many_sequences(abi, ctx, scope, dtype, sequences, most_rows, longest):
    """More sequences than a wavefront has lanes are listed by a launch of their own; some have no rows."""
    rng = np.random.default_rng(sequences)
    counts = rng.integers(0, most_rows + 1, sequences)
    lengths = np.maximum(counts, np.exp(rng.uniform(0, np.log(longest), sequences)).astype(int))
    for width in (0, 100):
        run_attention(abi, ctx, scope, rng, dtype, list(counts), list(lengths), 2, 1, 32, 16, width=width)
    run_attention(abi, ctx, scope, rng, dtype, list(counts), list(lengths), 2, 1, 32, 16, active=sequences - 3)


@DTYPES
def test_long_among_many_sequences(abi, ctx, scope, dtype):
    rng = np.random.default_rng(20)
    lengths = [9000 if s % 30 == 7 else 1 + s for s in range(100)]
    run_attention(abi, ctx, scope, rng, dtype, [1] * 100, lengths, 2, 1, 64, 16)


@DTYPES
@pytest.mark.parametrize("sequences,longest", [(3, 2000), (90, 100), (90, 900)])
def test_replays_follow_lengths(abi, ctx, scope, dtype, sequences, longest):
    """One graph, lengths and rows of each replay its own; eager and timed launches between them."""
    rng = np.random.default_rng(21)
    counts = list(rng.integers(1, 5, sequences))
    cache = Cache(rng, dtype, counts, [longest] * sequences, 2, 64, 16)
    queries = rng.standard_normal((cache.rows, 4 * 64)).astype(dtype)
    output = scope.put(np.zeros((cache.rows, 4 * 64), dtype))
    op = abi.CacheAttentionOp(ctx, queries=scope.put(queries), output=output, heads=4, **cache.put(scope))
    graph = abi.Graph.capture(ctx, ctx.stream)
    with graph:
        op.enqueue(0, ctx.stream)
    start, end = abi.Event(ctx), abi.Event(ctx)
    for i in range(4):
        cache.lengths = rng.integers(4, longest + 1, sequences).astype(np.uint32)
        cache.counts = list(rng.permutation(cache.counts))
        cache.starts = np.concatenate([[0], np.cumsum(cache.counts)]).astype(np.uint32)
        cache.device["lengths"].upload(cache.lengths)
        cache.device["row_starts"].upload(cache.starts)
        output.upload(np.zeros((cache.rows, 4 * 64), dtype))
        ctx.synchronize()
        if i % 2:
            op.enqueue(0, start=start, end=end)
        else:
            graph.launch()
        ctx.synchronize()
        if i % 2:
            assert 0 < start.elapsed_ms(end) < 100
        check_attention(cache, output.download(), queries, 4)
    graph.release()
    op.release()


@DTYPES
@pytest.mark.parametrize("sequences,length", [(4, 60), (4, 3000), (70, 60), (70, 3000)])
def test_starts_that_decrease(abi, ctx, scope, dtype, sequences, length):
    """Rows that only the first sequence has are right, whatever those of several
    hold; to the bit they need not be, as too many rows in all are not split."""
    counts = [8] + [0] * (sequences - 1)
    lengths = [length] + [40] * (sequences - 1)

    def decrease(cache, queries):
        cache.starts[2:] = [2 if s % 2 == 0 else 6 for s in range(2, sequences + 1)]

    run = lambda **kw: run_attention(abi, ctx, scope, np.random.default_rng(3), dtype, counts, lengths, 4, 2, 64, 16, **kw)
    cache, want, queries = run()
    got = run(spoil=decrease, check=False)[1]
    got[2:6] = want[2:6]
    check_attention(cache, got, queries, 4)


@DTYPES
def test_offsets_past_32_bits(abi, ctx, scope, dtype):
    """Pages whose elements, and bytes, lie beyond 2^32."""
    rng, page, dim = np.random.default_rng(18), 16, 128
    stride = 2 ** 28 + 8
    pages, used = 17, [16, 0, 15]
    e = np.dtype(dtype).itemsize
    counts, lengths = [1], [40]
    cache = Cache(rng, dtype, counts, lengths, 1, dim, page)
    cache.table[0] = used
    size = (pages - 1) * stride + page * dim
    caches = [scope.empty(size, dtype) for _ in range(2)]
    small = [rng.standard_normal((3, page * dim)).astype(dtype) for _ in range(2)]
    for device, host in zip(caches, small):
        for number, part in zip(used, host):
            abi.check(abi.load().pk_upload(ctx.handle, device.ptr + number * stride * e, part.ctypes.data, part.nbytes, None))
    queries = rng.standard_normal((1, 2 * dim)).astype(dtype)
    output = scope.put(np.zeros((1, 2 * dim), dtype))
    kw = dict(rows=1, sequences=1, kv_heads=1, head_dim=dim, row_starts=scope.put(cache.starts),
              lengths=scope.put(cache.lengths), page_table=scope.put(cache.table), pages_per_sequence=3, pages=pages,
              page_size=page, page_stride=stride, key_cache=caches[0], value_cache=caches[1])
    rows = [rng.standard_normal((1, dim)).astype(dtype) for _ in range(2)]
    append = abi.CacheAppendOp(ctx, keys=scope.put(rows[0]), values=scope.put(rows[1]), **kw)
    op = abi.CacheAttentionOp(ctx, queries=scope.put(queries), output=output, heads=2, **kw)
    append.enqueue()
    op.enqueue()
    ctx.synchronize()
    append.release()
    op.release()
    for part, row in zip(small, rows):
        part[2].reshape(page, dim)[39 - 32] = row[0]
    cache.pages, cache.page_stride = 3, page * dim
    cache.table[0] = [0, 1, 2]
    cache.keys, cache.values = (x.reshape(-1) for x in small)
    check_attention(cache, output.download(), queries, 2)
