"""The chunk operators over their range: every kernel variant's first and last
sizes, page sizes, head groups, bounds above the lengths, shared pages, far
offsets, streams, in place -- against the plain forms in tests/chunks.py."""

import math

import numpy as np
import pytest
import torch

from drift_b200.ops import Attention, Chunks, CudaOps, KvCache, QuantizedKvCache
from tests import chunks as plain
from tests.test_gpu_chunks import TYPES, attention_case, held

pytestmark = pytest.mark.gpu

CACHES = pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
KINDS = pytest.mark.parametrize("kind", ["f32", "bf16"])


@pytest.fixture(scope="module")
def ops():
    return CudaOps()


def checked(ops, case, kind, quantized, **bounds):
    new, counts, tables, page_size, cache, q, spec = attention_case(case, kind, quantized)
    out = torch.full_like(q, 7.0)
    ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, page_size, **bounds), spec, out)
    held(out, *plain.attention(q, cache, tables, new, counts, spec))
    assert ops.take_device_error() == 0


@CACHES
@KINDS
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("tokens", [1, 2, 3, 6, 7, 8, 9, 10, 11, 32, 33, 64, 65])
def test_rows_around_each_kernels_limits(ops, tokens, dim, kind, quantized):
    """Four rows a token: 4 and 8 to a unit of the few-rows kernels, which end
    at 8, 24, 32 or 40 rows; row tiles of 128, by one and two."""
    new = [tokens, 1, max(tokens - 3, 0)]
    counts = [tokens + 277, 500, max(tokens - 3, 0) + 30]
    checked(ops, (new, counts, 8, 2, dim, 16, 0, 0, None, False, True), kind, quantized)


@CACHES
@KINDS
@pytest.mark.parametrize("tokens", [2, 40, 150])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_windows_and_sinks(ops, dim, tokens, kind, quantized):
    """Windows narrower and wider than a tile, so that some warps of a row tile
    see nothing of a tile that others do."""
    for window, first in ((5, 0), (70, 3), (200, 90)):
        checked(ops, ([tokens, tokens // 2], [tokens + 333, tokens // 2], 8, 2, dim, 32, window, first, None, True, True),
                kind, quantized)


@CACHES
@pytest.mark.parametrize("page_size", [16, 32, 48, 64, 80, 96, 128, 1024])
@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_page_sizes(ops, tokens, page_size, quantized):
    for dim in (80, 128):
        for kind in TYPES:
            checked(ops, ([tokens, 3], [tokens + 301, 45], 8, 2, dim, page_size, 0, 0, None, False, True), kind, quantized)


@CACHES
@KINDS
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (14, 2), (16, 1), (9, 9), (64, 4)], ids=str)
def test_head_groups(ops, heads, kind, quantized):
    for tokens in (1, 3, 17):
        checked(ops, ([tokens, tokens], [tokens + 130, tokens], *heads, 64, 16, 0, 0, None, False, True), kind, quantized)


@CACHES
@KINDS
@pytest.mark.parametrize("softcap", [0.5, 4.0, 50.0])
def test_softcaps_near_and_far_from_zero(ops, softcap, kind, quantized):
    """Scores of up to about four against caps from an eighth of that on."""
    for tokens in (1, 70):
        checked(ops, ([tokens], [tokens + 150], 8, 2, 128, 16, 0, 0, softcap, True, True), kind, quantized)


@CACHES
@KINDS
def test_bounds_above_the_lengths(ops, kind, quantized):
    """longest and max_key_count are bounds, as a captured launch has them."""
    for tokens in (1, 40):
        new, counts = [tokens, 1], [tokens + 60, 200]
        case = (new, counts, 8, 2, 64, 16, 0, 0, None, False, True)
        for longest, max_keys in ((tokens, 208), (tokens + 7, 224), (200, 224)):
            checked(ops, case, kind, quantized, longest=longest, max_keys=max_keys)


@CACHES
@pytest.mark.parametrize("tokens", [1, 40])
def test_scales_of_either_sign_and_zero(ops, tokens, quantized):
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens], [tokens + 99], 8, 2, 128, 16, 0, 0, None, False, True), "f32", quantized)
    for scale in (-0.05, 0.0, 1.0):
        spec = Attention(scale)
        out = torch.empty_like(q)
        ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, page_size), spec, out)
        held(out, *plain.attention(q, cache, tables, new, counts, spec))


@CACHES
@KINDS
@pytest.mark.parametrize("tokens", [1, 5, 40, 300])
def test_a_row_that_is_not_finite_stays_alone(ops, tokens, kind, quantized):
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens], [tokens + 99], 8, 2, 64, 16, 0, 0, None, False, True), kind, quantized)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    # Not bit for bit the call without the NaN: a row whose weights may not fit
    # (a NaN's never do) has all rows of its warp take a new base, and a weight
    # rounded over another base is off by as much, but by another amount. So
    # every other row is held to its own bound around the formula.
    expected, tolerance = plain.attention(q, cache, tables, new, counts, spec)
    out = torch.empty_like(q)
    q[tokens // 2, 3, 7] = math.nan
    ops.attention_chunks(q, cache, chunks, spec, out)
    assert out[tokens // 2, 3].isnan().all()
    out[tokens // 2, 3] = expected[tokens // 2, 3].to(out.dtype)
    held(out, expected, tolerance)


@CACHES
@KINDS
@pytest.mark.parametrize("tokens", [6, 300])
def test_hidden_positions_in_wide_chunks(ops, tokens, kind, quantized):
    """NaNs where no token looks: past the end and before the first window."""
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens], [tokens + 211], 8, 2, 64, 64, 60, 2, None, False, True), kind, quantized)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_chunks(q, cache, chunks, spec, clean)
    for position in list(range(2, 211 - 59)) + list(range(tokens + 211, tables.shape[1] * page_size)):
        page, place = int(tables[0][position // page_size]), position % page_size
        if quantized:
            cache.key_scales[page, :, place] = cache.value_scales[page, :, place] = math.nan
        else:
            cache.keys[page, place] = cache.values[page, :, :, place] = math.nan
    ops.attention_chunks(q, cache, chunks, spec, out)
    assert torch.equal(out, clean)


@KINDS
@pytest.mark.parametrize("size", [-110, -40, 90])
def test_small_and_large_scales(ops, size, kind):
    """All of a cache's scales around 2^size (the keys' smaller by as much as
    keeps scores ordinary), for few rows, tiles, and codes expanded first."""
    for tokens in (1, 6, 60, 500):
        new, counts, tables, page_size, cache, q, spec = attention_case(
            ([tokens], [tokens + 150], 8, 2, 64, 16, 100, 3, None, False, True), kind, True)
        cache.value_scales.mul_(2.0 ** size)
        if size < 0:
            cache.key_scales.mul_(2.0 ** size)
        out = torch.empty_like(q)
        ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, page_size), spec, out)
        held(out, *plain.attention(q, cache, tables, new, counts, spec))


@KINDS
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_expanded_codes(ops, dim, kind):
    """Many units of rows over an 8-bit cache: a window, tokens that are not
    finite for those that see them, bad pages, other bounds."""
    for new, counts, window, first, softcap in (([700, 5, 0, 333], [1100, 500, 40, 333], 0, 0, 20.0),
                                                ([700, 5, 0, 333], [1100, 500, 40, 333], 120, 6, None)):
        case = (new, counts, 8, 2, dim, 48, window, first, softcap, True, True)
        checked(ops, case, kind, True)
        checked(ops, case, kind, True, longest=1000, max_keys=1104)
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([900], [1400], 8, 2, dim, 16, 0, 0, None, False, True), kind, True)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_chunks(q, cache, chunks, spec, clean)
    cache.value_scales[int(tables[0][1000 // 16]), 1, 1000 % 16] = math.nan  # rows 500 and later see it
    ops.attention_chunks(q, cache, chunks, spec, out)
    assert torch.equal(out[:, :4], clean[:, :4]) and out[500:, 4:].isnan().all()
    expected, tolerance = plain.attention(q[:500], cache, tables, [500], [1000], spec)
    held(out[:500], expected, tolerance)
    broken = tables.copy()
    broken[0, 3] = cache.pages
    ops.attention_chunks(q, cache, plain.chunks_of(new, counts, broken, page_size), spec, out)
    assert ops.take_device_error() == 1
    zeroed = type(cache)(*[torch.cat((t, torch.zeros_like(t[:1]))) for t in
                           (cache.keys, cache.values, cache.key_scales, cache.value_scales)], page_size)
    expected, tolerance = plain.attention(q[:500], zeroed, broken, [500], [1000], spec)
    held(out[:500], expected, tolerance)


@CACHES
@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_shared_pages(ops, tokens, quantized):
    """Sequences with a common prefix in the same pages, one of them twice."""
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens] * 3, [tokens + 150] * 3, 8, 2, 128, 16, 0, 0, None, False, True), "f32", quantized)
    tables[1, :8], tables[2] = tables[0, :8], tables[1]
    out = torch.empty_like(q)
    ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, page_size), spec, out)
    held(out, *plain.attention(q, cache, tables, new, counts, spec))


@CACHES
@KINDS
@pytest.mark.parametrize("tokens", [1, 5, 40, 300])
def test_again(ops, tokens, kind, quantized):
    """A call repeats bit for bit, and is refused in place."""
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens, 1], [tokens + 700, 900], 8, 2, 128, 16, 0, 0, None, False, True), kind, quantized)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    out, again = torch.empty_like(q), torch.empty_like(q)
    ops.attention_chunks(q, cache, chunks, spec, out)
    ops.attention_chunks(q, cache, chunks, spec, again)
    assert torch.equal(out, again)
    with pytest.raises(ValueError, match="overlap"):
        ops.attention_chunks(q, cache, chunks, spec, q)


@CACHES
def test_no_tokens(ops, quantized):
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([2, 2], [50, 60], 8, 2, 64, 16, 0, 0, None, False, True), "f32", quantized)
    empty = plain.chunks_of([0, 0], [50, 60], tables, page_size, longest=2)
    out, k = torch.full_like(q, 7.0), torch.full((4, 2, 64), 7.0, device="cuda")
    kept = cache.keys.clone()
    ops.attention_chunks(q, cache, empty, spec, out)
    ops.cache_write_chunks(k, k, cache, empty)
    ops.cache_read_chunks(cache, empty, k, k.clone())
    assert (out == 7.0).all() and (k == 7.0).all() and torch.equal(cache.keys, kept)
    nothing = Chunks(empty.starts, empty.positions, empty.page_tables, 0, 0)
    ops.attention_chunks(q[:0], cache, nothing, spec, out[:0])
    ops.cache_write_chunks(k[:0], k[:0], cache, nothing)
    assert ops.take_device_error() == 0


@CACHES
def test_two_streams_at_once(ops, quantized):
    """Calls of every kernel under way together on two streams, each what it is
    alone."""
    cases = [attention_case(([n, 2], [n + 2000, 1500], 16, 4, 128, 16, 0, 0, None, False, True), kind, quantized, seed)
             for seed, (n, kind) in enumerate([(1, "f32"), (6, "bf16"), (60, "f32"), (200, "bf16")])]
    alone = []
    for new, counts, tables, page_size, cache, q, spec in cases:
        alone.append(torch.empty_like(q))
        ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, page_size), spec, alone[-1])
    prepared = [(plain.chunks_of(c[0], c[1], c[2], c[3]), [torch.empty_like(c[5]) for _ in range(6)]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        for n, (c, (chunks, outs)) in enumerate(zip(cases, prepared)):
            with torch.cuda.stream(streams[(n + i) % 2]):
                ops.attention_chunks(c[5], c[4], chunks, c[6], outs[i])
    torch.cuda.synchronize()
    for (chunks, outs), want in zip(prepared, alone):
        assert all(torch.equal(out, want) for out in outs)
    assert ops.take_device_error() == 0


@CACHES
def test_offsets_past_32_bits(ops, quantized):
    """A cache of more than 2^32 codes a side, and a sequence on its last pages."""
    kv_heads, dim, page_size, pages = 8, 128, 16, 262144 + 300
    rng = np.random.default_rng(21)
    make = lambda dtype, *s: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
    sides = (pages, page_size, kv_heads, dim), (pages, kv_heads, dim, page_size)
    if quantized:
        cache = QuantizedKvCache(*(make(torch.int8, *s) for s in sides),
                                 *(make(torch.float32, pages, kv_heads, page_size) for _ in range(2)), page_size)
    else:
        cache = KvCache(*(make(torch.float16, *s) for s in sides), page_size)
    tables = np.concatenate([pages - 1 - rng.permutation(12), [0, 131072]]).astype(np.int32)[None]
    counts, spec = [14 * page_size], Attention(1 / math.sqrt(dim))
    k, v = (torch.from_numpy(rng.standard_normal((counts[0], kv_heads, dim)).astype(np.float32)).cuda() for _ in range(2))
    whole = plain.chunks_of(counts, counts, tables, page_size)
    ops.cache_write_chunks(k, v, cache, whole)
    back = torch.empty_like(k), torch.empty_like(v)
    ops.cache_read_chunks(cache, whole, *back)
    for got, want in zip(back, plain.sequence(cache, tables[0], counts[0])):
        assert torch.equal(got, want.float())
    if quantized:
        assert torch.equal(cache.keys[int(tables[0][0])].cpu(),
                           torch.from_numpy(plain.quantized(k[:page_size].cpu().numpy())[0]))
    else:
        assert torch.equal(cache.keys[int(tables[0][0])], k[:page_size].half())
    for kind, dtype in TYPES.items():
        for tokens in (1, 40):
            q = torch.from_numpy(rng.standard_normal((tokens, 16, dim)).astype(np.float32)).to(dtype).cuda()
            out = torch.empty_like(q)
            ops.attention_chunks(q, cache, plain.chunks_of([tokens], counts, tables, page_size), spec, out)
            held(out, *plain.attention(q, cache, tables, [tokens], counts, spec))
    assert ops.take_device_error() == 0


def test_writes_of_one_position_at_every_place(ops):
    """A step's writes into each place of a page leave its neighbours alone."""
    for quantized in (True, False):
        cache = (QuantizedKvCache if quantized else KvCache).allocate(2, 32, 3, 80)
        tables = np.array([[1, 0]], np.int32)
        x = torch.from_numpy(np.random.default_rng(1).standard_normal((64, 3, 80)).astype(np.float32)).cuda()
        for position in range(64):
            ops.cache_write_chunks(x[position:position + 1], -x[position:position + 1], cache,
                                   plain.chunks_of([1], [position + 1], tables, 32))
        once = (QuantizedKvCache if quantized else KvCache).allocate(2, 32, 3, 80)
        ops.cache_write_chunks(x, -x, once, plain.chunks_of([64], [64], tables, 32))
        for name in ("keys", "values") + (("key_scales", "value_scales") if quantized else ()):
            assert torch.equal(getattr(cache, name), getattr(once, name))


@CACHES
@pytest.mark.parametrize("tokens", [2, 3, 9, 100, 515])
def test_f32_heads_of_256(ops, tokens, quantized):
    """A CTA for each half of a value, with and without splits, windows and
    values that are not finite."""
    checked(ops, ([tokens, 1], [tokens + 277, 300], 16, 2, 256, 16, 0, 0, 10.0, True, True), "f32", quantized)
    checked(ops, ([tokens] * 9, [tokens + 40] * 9, 16, 2, 256, 32, 90, 5, None, False, True), "f32", quantized)
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens], [tokens + 99], 16, 2, 256, 16, 0, 0, None, False, True), "f32", quantized)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ops.attention_chunks(q, cache, chunks, spec, clean)
    position = tokens + 97  # the last two tokens' and the last's
    page, place = int(tables[0][position // page_size]), position % page_size
    if quantized:
        cache.value_scales[page, 1, place] = math.nan
    else:
        cache.values[page, 1, 200, place] = math.inf
    ops.attention_chunks(q, cache, chunks, spec, out)
    assert torch.equal(out[:-2], clean[:-2]) and torch.equal(out[:, :8], clean[:, :8])
    if quantized:
        assert out[-2:, 8:].isnan().all()
    else:
        assert not out[-2:, 8:, 200].isfinite().any()
        assert torch.equal(out[-2:, 8:, :200], clean[-2:, 8:, :200])


@CACHES
@KINDS
def test_wide_chunks_captured_and_replayed(ops, kind, quantized):
    """Chunks of several units (an 8-bit cache's codes expanded in the launch)
    captured once and replayed at other lengths, positions and pages."""
    rng = np.random.default_rng(31)
    q_heads, kv_heads, dim, page_size = 8, 2, 128, 16
    tables, pages = plain.tables_of(rng, 2, 80)
    cache = plain.random_cache(rng, quantized, pages, page_size, kv_heads, dim)
    chunks = plain.chunks_of([500, 500], [500, 1200], tables, page_size, max_keys=1280)
    q = torch.from_numpy(rng.standard_normal((1000, q_heads, dim)).astype(np.float32)).to(TYPES[kind]).cuda()
    out = torch.empty_like(q)
    spec = Attention(1 / math.sqrt(dim), window=300, first=5)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.attention_chunks(q, cache, chunks, spec, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.attention_chunks(q, cache, chunks, spec, out)
    for new, counts in (([500, 130], [1280, 131]), ([0, 400], [3, 900]), ([1, 500], [700, 500])):
        tables = tables[::-1].copy()
        fresh = plain.chunks_of(new, counts, tables, page_size)
        for name in ("starts", "positions", "page_tables"):
            getattr(chunks, name).copy_(getattr(fresh, name))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(new)
        held(out[:n], *plain.attention(q[:n], cache, tables, new, counts, spec))
        assert (out[n:] == 7.0).all()
    assert ops.take_device_error() == 0
