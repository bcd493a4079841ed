"""The cache and attention of a batch of sequences' new tokens
(cache_write_chunks, cache_read_chunks, attention_chunks) against plain forms
in 64 bits (tests/chunks.py)."""

import math

import numpy as np
import pytest
import torch

from drift_b200.ops import Attention, Chunks, CudaOps, KvCache, QuantizedKvCache
from tests import chunks as plain

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    return CudaOps()


# ---- the cache -----------------------------------------------------------------

# (type, dim, kv_heads, page size, new tokens, positions with them)
WRITES = [
    ("f32", 128, 8, 16, [1, 1, 1], [1, 17, 300]),         # a decoding step
    ("bf16", 128, 2, 16, [33, 1, 16], [33, 40, 16]),       # runs cut at either end
    ("f32", 64, 3, 48, [5, 0, 100], [95, 7, 100]),         # a sequence of no tokens
    ("bf16", 80, 1, 32, [70], [75]),
    ("f32", 256, 2, 64, [3, 65], [66, 129]),
]


def rows_of(rng, total, kv_heads, dim, dtype):
    """Rows of very different sizes, some with ties, zeros and subnormals."""
    x = rng.standard_normal((total, kv_heads, dim)) * np.exp(rng.uniform(-30, 30, (total, kv_heads, 1)))
    x[0, 0] = 0.0
    if total > 1:  # every quotient a half or a whole number
        x[1, 0] = rng.integers(-254, 255, dim) / 2
        x[1, 0, 0] = 127.0
    if total > 2:
        x[2, 0] = rng.integers(-300, 300, dim) * 2.0 ** -149
    return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
@pytest.mark.parametrize("case", WRITES, ids=str)
def test_write_and_read_back(ops, case, quantized):
    kind, dim, kv_heads, page_size, new, counts = case
    dtype = TYPES[kind]
    rng = np.random.default_rng(dim + sum(new))
    tables, pages = plain.tables_of(rng, len(new), -(-max(counts) // page_size) + 1)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    cache = plain.random_cache(rng, quantized, pages, page_size, kv_heads, dim)
    total = sum(new)
    k, v = (rows_of(rng, total + 2, kv_heads, dim, dtype) for _ in range(2))  # two rows behind the last
    before = [t.clone() for t in (cache.keys, cache.values)]
    expected = [t.cpu().numpy().copy() for t in before]
    scales = [t.cpu().numpy().copy() for t in (cache.key_scales, cache.value_scales)] if quantized else None
    ops.cache_write_chunks(k, v, cache, chunks)
    row = 0
    for z, (n, count) in enumerate(zip(new, counts)):
        for position in range(count - n, count):
            page, place = tables[z][position // page_size], position % page_size
            for side, x in enumerate((k, v)):
                x = x[row].float().cpu().numpy()
                if quantized:
                    held, scales[side][page, :, place] = plain.quantized(x)
                else:
                    with np.errstate(over="ignore"):
                        held = x.astype(np.float16)
                if side == 0:
                    expected[0][page, place] = held
                else:
                    expected[1][page, :, :, place] = held
            row += 1
    # the positions written, bit for bit; every other as it was
    for got, want in zip((cache.keys, cache.values), expected):
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    if quantized:
        for got, want in zip((cache.key_scales, cache.value_scales), scales):
            np.testing.assert_array_equal(got.cpu().numpy(), want)
    # and back
    for back_type in TYPES.values():
        back = [torch.full((total + 2, kv_heads, dim), 7.0, dtype=back_type, device="cuda") for _ in range(2)]
        ops.cache_read_chunks(cache, chunks, *back)
        row = 0
        for z, (n, count) in enumerate(zip(new, counts)):
            for got, want in zip(back, plain.sequence(cache, tables[z], count)):
                want = want[count - n:].float().to(back_type)  # one product of 24 + 8 bits: F32 rounds it once
                assert torch.equal(got[row:row + n], want)
            row += n
        assert all((got[total:] == 7.0).all() for got in back)
    assert ops.take_device_error() == 0


def test_codes_are_within_half_a_scale(ops):
    rng = np.random.default_rng(3)
    cache = QuantizedKvCache.allocate(4, 16, 2, 128)
    x = torch.from_numpy(rng.standard_normal((50, 2, 128)).astype(np.float32)).cuda()
    chunks = plain.chunks_of([50], [50], np.array([[3, 1, 0, 2]], np.int32), 16)
    ops.cache_write_chunks(x, x, cache, chunks)
    k, v = torch.empty_like(x), torch.empty_like(x)
    ops.cache_read_chunks(cache, chunks, k, v)
    assert torch.equal(k, v)
    step = x.abs().amax(-1, keepdim=True) / 127
    # half a scale, and the rounding of code x scale (24 bits of at most 127 scales)
    assert ((k - x).abs() <= step * (0.5 + 127 * 2.0 ** -23)).all()


def test_rows_with_nan_or_infinity_read_back_as_nans(ops):
    cache = QuantizedKvCache.allocate(1, 16, 1, 64)
    x = torch.ones(3, 1, 64, device="cuda")
    x[0, 0, 5], x[1, 0, 63] = math.nan, -math.inf
    chunks = plain.chunks_of([3], [3], np.zeros((1, 1), np.int32), 16)
    ops.cache_write_chunks(x, x, cache, chunks)
    k, v = torch.empty_like(x), torch.empty_like(x)
    ops.cache_read_chunks(cache, chunks, k, v)
    for got in (k, v):
        assert got[:2].isnan().all() and torch.equal(got[2], x[2])


# ---- attention ------------------------------------------------------------------

# (new tokens, positions with them, q heads, kv heads, dim, page size, window, first, softcap, sinks, causal)
ATTENTION = [
    ([1], [1], 32, 8, 128, 16, 0, 0, None, False, True),               # one key
    ([1, 1, 1, 1], [1, 17, 300, 1500], 32, 8, 128, 16, 0, 0, None, False, True),  # a decoding step
    ([1, 1], [130, 700], 16, 2, 256, 32, 0, 0, None, True, True),
    ([1, 1], [77, 513], 8, 8, 64, 48, 0, 0, 30.0, False, True),
    ([1, 1, 1], [3, 64, 333], 10, 2, 80, 16, 0, 0, None, True, True),
    ([1, 1], [900, 2000], 16, 1, 128, 64, 100, 4, None, False, True),   # a window and the first tokens
    ([1, 1], [900, 30], 4, 4, 64, 16, 1, 20, None, True, True),         # itself and the first ones
    ([5, 1, 3], [400, 9, 3], 32, 8, 128, 16, 0, 0, None, False, True),  # drafts
    ([3, 0, 4], [37, 5, 4], 8, 8, 64, 16, 0, 0, None, False, True),     # a sequence of no tokens
    ([33, 20], [33, 150], 8, 2, 128, 16, 0, 0, None, False, True),      # prompts
    ([130], [257], 10, 2, 80, 32, 50, 3, None, False, True),
    ([70, 9], [70, 70], 16, 2, 256, 16, 0, 0, 20.0, True, True),
    ([40], [200], 16, 1, 128, 48, 64, 16, None, False, True),
    ([20, 7], [100, 7], 8, 4, 64, 16, 0, 0, None, False, False),        # not causal
    ([20], [100], 8, 4, 128, 16, 30, 0, None, True, False),
    ([300], [700], 4, 1, 128, 16, 0, 0, None, False, True),
    ([600, 259], [601, 1300], 8, 2, 64, 64, 256, 130, None, False, True),
]


def attention_case(case, kind, quantized, seed=0):
    new, counts, q_heads, kv_heads, dim, page_size, window, first, softcap, sinks, causal = case
    rng = np.random.default_rng(sum(counts) + dim + seed)
    tables, pages = plain.tables_of(rng, len(new), -(-max(counts) // page_size) + 1)
    cache = plain.random_cache(rng, quantized, pages, page_size, kv_heads, dim)
    q = torch.from_numpy(rng.standard_normal((sum(new), q_heads, dim)).astype(np.float32)).to(TYPES[kind]).cuda()
    sink = torch.from_numpy(rng.standard_normal(q_heads).astype(np.float32)).cuda() if sinks else None
    spec = Attention(1 / math.sqrt(dim), causal, window or None, softcap, sink, first)
    return new, counts, tables, page_size, cache, q, spec


def held(got, expected, tolerance):
    off = (got.double() - expected).abs()
    worst = (off / tolerance).max().item()
    assert (off <= tolerance).all(), f"{worst:.3g} of the tolerance, largest error {off.max().item():.3g}"


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"{c[0]}of{c[1]}h{c[2]}/{c[3]}d{c[4]}w{c[6]}".replace(" ", ""))
def test_attention_is_the_formula(ops, case, kind, quantized):
    new, counts, tables, page_size, cache, q, spec = attention_case(case, kind, quantized)
    out = torch.full_like(q, 7.0)
    ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, page_size), spec, out)
    held(out, *plain.attention(q, cache, tables, new, counts, spec))
    assert ops.take_device_error() == 0


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_behind_the_last_sequence_stay(ops, kind):
    case = ([3, 40], [30, 90], 8, 2, 128, 16, 0, 0, None, False, True)
    new, counts, tables, page_size, cache, q, spec = attention_case(case, kind, True)
    padded = torch.cat((q, torch.full((9, 8, 128), math.nan, dtype=q.dtype, device="cuda")))
    out = torch.full_like(padded, 7.0)
    ops.attention_chunks(padded, cache, plain.chunks_of(new, counts, tables, page_size), spec, out)
    assert (out[43:] == 7.0).all()
    held(out[:43], *plain.attention(q, cache, tables, new, counts, spec))


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_what_no_token_sees_may_be_anything(ops, tokens, quantized):
    """NaNs and infinities past the last position, before the window and in
    other pages change nothing."""
    case = ([tokens], [205], 8, 2, 128, 16, 100, 4, None, False, True)
    new, counts, tables, page_size, cache, q, spec = attention_case(case, "f32", quantized)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    clean = torch.empty_like(q)
    ops.attention_chunks(q, cache, chunks, spec, clean)
    seen = set(range(4)) | set(range(205 - tokens - 99, 205))
    hidden = torch.ones(cache.pages, page_size, dtype=torch.bool, device="cuda")
    for position in seen:
        hidden[int(tables[0][position // page_size]), position % page_size] = False
    sides = (cache.key_scales, cache.value_scales) if quantized else (cache.keys, cache.values)
    page, place = hidden.nonzero(as_tuple=True)
    for bad in (math.nan, math.inf, -math.inf):
        if quantized:
            for side in sides:
                side[page, :, place] = bad
        else:
            cache.keys[page, place] = bad
            cache.values[page, :, :, place] = bad
        out = torch.empty_like(q)
        ops.attention_chunks(q, cache, chunks, spec, out)
        assert torch.equal(out, clean)


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_later_token_that_is_not_finite_does_not_reach_earlier_ones(ops, kind, quantized):
    case = ([40], [205], 8, 2, 128, 16, 0, 0, None, False, True)
    new, counts, tables, page_size, cache, q, spec = attention_case(case, kind, quantized)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    clean = torch.empty_like(q)
    ops.attention_chunks(q, cache, chunks, spec, clean)
    # position 190, which rows 25 and later see
    page, place = int(tables[0][190 // page_size]), 190 % page_size
    if quantized:
        cache.value_scales[page, 1, place] = math.nan
    else:
        cache.values[page, 1, 5, place] = math.inf
    out = torch.empty_like(q)
    ops.attention_chunks(q, cache, chunks, spec, out)
    assert torch.equal(out[:25], clean[:25])
    assert torch.equal(out[:, :4], clean[:, :4])  # the other key head's
    if quantized:
        assert out[25:, 4:].isnan().all()
    else:
        assert not out[25:, 4:, 5].isfinite().any()
        assert torch.equal(out[25:, 4:, :5], clean[25:, 4:, :5])


def test_a_row_that_sees_only_a_sink_or_small_scores(ops):
    """Scores far below a sink weigh nothing; equal scores of the lowest
    finite size are a mean."""
    cache = KvCache.allocate(1, 16, 1, 64)
    cache.keys[0, :4, 0] = -65504.0
    cache.values[0, 0, :, :4] = torch.arange(4.0, device="cuda")
    q = torch.full((1, 1, 64), 3e33, device="cuda")
    out = torch.empty_like(q)
    chunks = plain.chunks_of([1], [4], np.zeros((1, 1), np.int32), 16)
    ops.attention_chunks(q, cache, chunks, Attention(0.02), out)  # scores of -2.5e38
    assert torch.equal(out, torch.full_like(out, 1.5))
    ops.attention_chunks(q, cache, chunks, Attention(0.02, sinks=torch.zeros(1, device="cuda")), out)
    assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
def test_a_chunk_is_its_tokens_one_by_one(ops, quantized):
    """Drafted tokens at once, or one decoding step after another: equal within
    both calls' tolerances."""
    case = ([6], [300], 32, 8, 128, 16, 0, 0, None, False, True)
    new, counts, tables, page_size, cache, q, spec = attention_case(case, "f32", quantized)
    out, one = torch.empty_like(q), torch.empty_like(q)
    ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, page_size), spec, out)
    for i in range(6):
        ops.attention_chunks(q[i:i + 1], cache, plain.chunks_of([1], [295 + i], tables, page_size), spec, one[i:i + 1])
    _, tolerance = plain.attention(q, cache, tables, new, counts, spec)
    held(out, one.double(), 2 * tolerance)


def test_extreme_scales(ops):
    """Values' scales from the smallest normal size to 2^100 in one sequence:
    the weights' common unit follows the largest seen so far."""
    rng = np.random.default_rng(11)
    tables, pages = plain.tables_of(rng, 1, 40)
    cache = plain.random_cache(rng, True, pages, 16, 2, 128)
    cache.value_scales.copy_(torch.from_numpy(
        np.exp2(rng.uniform(-126, 100, (pages, 2, 16))).astype(np.float32)).cuda())
    cache.value_scales[int(tables[0][0])] = 0.0
    q = torch.from_numpy(rng.standard_normal((3, 8, 128)).astype(np.float32)).cuda()
    spec = Attention(1 / math.sqrt(128))
    for count in (20, 600):
        out = torch.empty_like(q)
        ops.attention_chunks(q, cache, plain.chunks_of([3], [count], tables, 16), spec, out)
        held(out, *plain.attention(q, cache, tables, [3], [count], spec))


# ---- the calls together, streams and graphs -----------------------------------------------

@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
def test_prompts_then_steps(ops, quantized):
    """Two sequences as a server runs them: their prompts written and attended
    in pieces, then decoding steps, each result that of the plain form over
    what was written."""
    rng = np.random.default_rng(5)
    q_heads, kv_heads, dim, page_size = 8, 2, 64, 16
    tables, pages = plain.tables_of(rng, 2, 8)
    cache = (QuantizedKvCache if quantized else KvCache).allocate(pages, page_size, kv_heads, dim)
    spec = Attention(1 / math.sqrt(dim), window=50, first=2)
    done = [0, 0]
    for new in ([30, 17], [33, 0], [1, 20], [1, 1], [1, 1], [3, 2]):
        counts = [d + n for d, n in zip(done, new)]
        chunks = plain.chunks_of(new, counts, tables, page_size)
        k, v = (torch.from_numpy(rng.standard_normal((sum(new), kv_heads, dim)).astype(np.float32)).cuda() for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((sum(new), q_heads, dim)).astype(np.float32)).cuda()
        out = torch.empty_like(q)
        ops.cache_write_chunks(k, v, cache, chunks)
        ops.attention_chunks(q, cache, chunks, spec, out)
        held(out, *plain.attention(q, cache, tables, new, counts, spec))
        done = counts
    assert ops.take_device_error() == 0


@pytest.mark.parametrize("tokens", [1, 70])
def test_captured_and_replayed_at_other_lengths(ops, tokens):
    """A captured write and attention replay at new starts and positions, and
    two graphs that overlap in time keep their partial results apart."""
    rng = np.random.default_rng(6)
    q_heads, kv_heads, dim, page_size = 8, 2, 128, 16
    graphs = []
    for which in range(2):
        tables, pages = plain.tables_of(rng, 2, 40)
        cache = QuantizedKvCache.allocate(pages, page_size, kv_heads, dim)
        chunks = plain.chunks_of([tokens, tokens], [tokens, tokens], tables, page_size, max_keys=640)
        rows = 2 * tokens
        q = torch.zeros(rows, q_heads, dim, device="cuda")
        k, v = (torch.zeros(rows, kv_heads, dim, device="cuda") for _ in range(2))
        out = torch.zeros_like(q)
        spec = Attention(1 / math.sqrt(dim))

        def step(k=k, v=v, q=q, cache=cache, chunks=chunks, spec=spec, out=out):
            ops.cache_write_chunks(k, v, cache, chunks)
            ops.attention_chunks(q, cache, chunks, spec, out)

        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        graphs.append((graph, stream, tables, cache, chunks, q, k, v, out, spec))
    for new, counts in (([tokens, max(1, tokens // 2)], [500, 640]), ([0, tokens], [3, 333])):
        for graph, stream, tables, cache, chunks, q, k, v, out, spec in graphs:
            for t in (q, k, v):
                t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
            fresh = plain.random_cache(rng, True, cache.pages, page_size, kv_heads, dim)
            for name in ("keys", "values", "key_scales", "value_scales"):
                getattr(cache, name).copy_(getattr(fresh, name))
            fresh = plain.chunks_of(new, counts, tables, page_size)
            chunks.starts.copy_(fresh.starts)
            chunks.positions.copy_(fresh.positions)
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for graph, stream, tables, cache, chunks, q, k, v, out, spec in graphs:
            n = sum(new)
            expected, tolerance = plain.attention(q[:n], cache, tables, new, counts, spec)
            held(out[:n], expected, tolerance)
    assert ops.take_device_error() == 0


# ---- refusals ----------------------------------------------------------------------------

def test_bad_chunks_are_left_out_and_flagged(ops):
    """Starts that fall, chunks past `longest`, the tokens, the table or
    max_key_count: that sequence's rows stay as they were, the others' are
    right, and the device error word is set."""
    rng = np.random.default_rng(8)
    tables, pages = plain.tables_of(rng, 3, 4)
    cache = plain.random_cache(rng, True, pages, 16, 2, 64)
    q = torch.from_numpy(rng.standard_normal((6, 4, 64)).astype(np.float32)).cuda()
    spec = Attention(0.125)
    expected, tolerance = plain.attention(q[4:6], cache, tables[2:], [2], [20], spec)
    kept = [t.clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales)]
    for starts, positions in (([0, 4, 2, 6], [0, 0, 18]),      # the second falls (and the third is long)
                              ([0, 2, 4, 6], [-1, 63, 18]),    # before the table, past it
                              ([-1, 1, 4, 6], [0, 62, 18]),    # a row before the first
                              ([0, 4, 4, 7], [0, 0, 18])):     # a row past the last
        chunks = Chunks(torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(positions, dtype=torch.int32).cuda(),
                        torch.from_numpy(tables).cuda(), 2, 64)
        good = [0 <= a <= b <= 6 and b - a <= 2 and 0 <= p <= 64 - (b - a)
                for a, b, p in zip(starts, starts[1:], positions)]
        out = torch.full_like(q, 7.0)
        ops.attention_chunks(q, cache, chunks, spec, out)
        assert ops.take_device_error() == 1
        for z, (a, b) in enumerate(zip(starts, starts[1:])):
            if not good[z]:
                rows = [r for r in range(max(a, 0), min(b, 6)) if not any(
                    good[y] and starts[y] <= r < starts[y + 1] for y in range(3))]
                assert (out[rows] == 7.0).all()
        if good[2]:
            held(out[4:6], expected, tolerance)
        k = torch.zeros(6, 2, 64, device="cuda")
        none = Chunks(chunks.starts[[0, 1]], chunks.positions[:1], chunks.page_tables[:1], 1, 64)
        ops.cache_write_chunks(k, k, cache, Chunks(none.starts * 0 + torch.tensor([3, 1], dtype=torch.int32).cuda(),
                                                   none.positions, none.page_tables, 1, 64))
        assert ops.take_device_error() == 1
        for t, was in zip((cache.keys, cache.values, cache.key_scales, cache.value_scales), kept):
            assert torch.equal(t, was)


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_pages_outside_the_cache_read_as_zeros(ops, tokens, quantized):
    rng = np.random.default_rng(9)
    tables, pages = plain.tables_of(rng, 1, 8)
    cache = plain.random_cache(rng, quantized, pages, 16, 2, 64)
    q = torch.from_numpy(rng.standard_normal((tokens, 8, 64)).astype(np.float32)).cuda()
    spec = Attention(0.125)
    for bad in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        broken = tables.copy()
        broken[0, 2] = bad
        out = torch.empty_like(q)
        chunks = plain.chunks_of([tokens], [100], broken, 16)
        ops.attention_chunks(q, cache, chunks, spec, out)
        assert ops.take_device_error() == 1
        zeroed = type(cache)(*[torch.cat((t, torch.zeros_like(t[:1]))) for t in
                               (cache.keys, cache.values) + ((cache.key_scales, cache.value_scales) if quantized else ())],
                             16)
        where = tables.copy()
        where[0, 2] = pages
        held(out, *plain.attention(q, zeroed, where, [tokens], [100], spec))
        kept = cache.keys.clone(), cache.values.clone()
        x = torch.ones(16, 2, 64, device="cuda")
        ops.cache_write_chunks(x, x, cache, plain.chunks_of([16], [48], broken, 16))
        assert ops.take_device_error() == 1
        assert torch.equal(cache.keys, kept[0]) and torch.equal(cache.values, kept[1])
        back = torch.full((16, 2, 64), 7.0, device="cuda")
        ops.cache_read_chunks(cache, plain.chunks_of([16], [48], broken, 16), back, torch.empty_like(back))
        assert ops.take_device_error() == 1 and (back == 0.0).all()


def test_refusals(ops):
    cache = QuantizedKvCache.allocate(4, 16, 2, 64)
    q = torch.zeros(3, 4, 64, device="cuda")
    k = torch.zeros(3, 2, 64, device="cuda")
    chunks = plain.chunks_of([3], [3], np.arange(4, dtype=np.int32)[None], 16)
    spec = Attention(0.125)
    with pytest.raises(ValueError, match="takes F32"):
        ops.attention_chunks(q.half(), cache, chunks, spec, q.half())
    with pytest.raises(ValueError, match="torch.float32 and torch.bfloat16"):
        ops.attention_chunks(q, cache, chunks, spec, q.bfloat16())
    with pytest.raises(ValueError, match="query heads over"):
        ops.attention_chunks(q[:, :3].contiguous(), cache, chunks, spec, q[:, :3].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        ops.attention_chunks(q[:, ::2], cache, chunks, spec, q[:, ::2])
    with pytest.raises(ValueError, match="for a cache of"):
        ops.attention_chunks(q[..., :32].contiguous(), cache, chunks, spec, q[..., :32].contiguous())
    with pytest.raises(ValueError, match="into a cache"):
        ops.cache_write_chunks(q, q, cache, chunks)
    with pytest.raises(ValueError, match="first keys without a window"):
        ops.attention_chunks(q, cache, chunks, Attention(0.125, first=4), q)
    with pytest.raises(ValueError, match="sinks"):
        ops.attention_chunks(q, cache, chunks, Attention(0.125, sinks=torch.zeros(3, device="cuda")), q)
    with pytest.raises(ValueError, match="keys in a page table"):
        ops.attention_chunks(q, cache, Chunks(chunks.starts, chunks.positions, chunks.page_tables, 3, 65), spec, q)
    with pytest.raises(ValueError, match="for 1 sequences"):
        ops.cache_write_chunks(k, k, cache, Chunks(chunks.starts[:1], chunks.positions, chunks.page_tables, 3, 3))
    with pytest.raises(ValueError, match="contiguous I32"):
        ops.cache_read_chunks(cache, Chunks(chunks.starts.long(), chunks.positions, chunks.page_tables, 3, 3), k, k)
    with pytest.raises(ValueError, match="scales"):
        ops.cache_write_chunks(k, k, QuantizedKvCache(cache.keys, cache.values, cache.key_scales[:1], cache.value_scales, 16), chunks)
    with pytest.raises(ValueError, match="16-byte boundary"):
        shifted = torch.zeros(3 * 2 * 64 + 1, device="cuda")[1:].view(3, 2, 64)
        ops.cache_write_chunks(shifted, k, cache, chunks)
    old = KvCache.allocate(4, 16, 2, 64)
    table = chunks.page_tables[0]
    with pytest.raises(ValueError, match="attention_chunks"):
        ops.attention(q, old, table, 0, 3, Attention(0.125, window=2, first=1), q)
    # nothing to do
    none = torch.zeros(0, 4, 64, device="cuda")
    ops.attention_chunks(none, cache, Chunks(chunks.starts * 0, chunks.positions, chunks.page_tables, 0, 3), spec, none)
