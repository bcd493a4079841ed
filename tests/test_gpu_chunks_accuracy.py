"""attention_chunks held to what its kernels' roundings allow
(tests/chunk_accuracy.py): ordinary scores, a key that takes most of the weight
and has no value, scales far apart, scales that a row's mask hides, scores that
grow along the keys."""

import math

import numpy as np
import pytest
import torch

from drift_b200.ops import Attention, CudaOps, KvCache, QuantizedKvCache
from tests import chunk_accuracy
from tests import chunks as plain
from tests.test_gpu_chunks import TYPES, attention_case

pytestmark = pytest.mark.gpu

CACHES = pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
KINDS = pytest.mark.parametrize("kind", ["f32", "bf16"])


@pytest.fixture(scope="module")
def ops():
    return CudaOps()


def floats(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()


def holds(ops, q, cache, tables, new, counts, spec, **bounds):
    """Runs the call and holds it to the bound; the result."""
    out = torch.full_like(q, 7.0)
    ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, cache.page_size, **bounds), spec, out)
    expected, off = chunk_accuracy.attention(q, cache, tables, new, counts, spec, bounds.get("longest"))
    error = (out.double() - expected).abs()
    worst = (error / off).max().item()
    assert (error <= off).all(), f"{worst:.3g} of the bound, largest error {error.max().item():.3g}"
    assert ops.take_device_error() == 0
    return out


def written(ops, rng, quantized, k, v, page_size=16):
    """A cache with k, v [count, kv_heads, D] as one sequence, and its table."""
    count, kv_heads, dim = k.shape
    tables, pages = plain.tables_of(rng, 1, -(-count // page_size))
    cache = (QuantizedKvCache if quantized else KvCache).allocate(pages, page_size, kv_heads, dim)
    ops.cache_write_chunks(k, v, cache, plain.chunks_of([count], [count], tables, page_size))
    return cache, tables


# (new tokens, positions with them, q heads, kv heads, dim): four rows at most,
# eight, several units of eight
FEW = [
    ([1, 1], [4097, 700], 4, 1, 128),
    ([1, 1, 1], [2000, 16, 33], 16, 2, 256),
    ([2, 1], [3001, 5], 16, 4, 64),
    ([1, 1], [1500, 6000], 16, 1, 128),
    ([3, 1], [5000, 900], 10, 2, 80),
    ([5, 4], [2500, 2500], 8, 2, 128),
]


@pytest.mark.parametrize("window,softcap,sinks", [(0, None, False), (300, 20.0, True)], ids=["plain", "window-cap-sinks"])
@KINDS
@pytest.mark.parametrize("case", FEW, ids=lambda c: f"{c[0]}of{c[1]}h{c[2]}/{c[3]}d{c[4]}".replace(" ", ""))
def test_few_rows_over_8_bits(ops, case, kind, window, softcap, sinks):
    new, counts, tables, page_size, cache, q, spec = attention_case(
        (*case, 16, window, 4 if window else 0, softcap, sinks, True), kind, True)
    holds(ops, q, cache, tables, new, counts, spec)
    holds(ops, q * 4, cache, tables, new, counts, spec)  # scores of up to sixteen and more


def dominated(ops, rng, kind, quantized, tokens, count, q_heads, kv_heads, dim, rest, spread, value):
    """One early key that has 1 / `rest` times the weight of all others
    together, `value` times their values; theirs are of both signs."""
    group = q_heads // kv_heads
    along = floats(rng, kv_heads, 1, dim)
    along = along / along.norm(dim=2, keepdim=True)
    k, v = floats(rng, count, kv_heads, dim), floats(rng, count, kv_heads, dim)
    u = along[None, :, 0]
    k = k - (k * u).sum(2, keepdim=True) * u
    q = floats(rng, tokens, kv_heads, group, dim) * spread + math.sqrt(dim) * along
    k[3] = math.log(count * math.exp(spread ** 2 / 2) / rest) * u[0]
    v[3] *= value
    cache, tables = written(ops, rng, quantized, k, v)
    return q.reshape(tokens, q_heads, dim).to(TYPES[kind]), cache, tables


@pytest.mark.parametrize("rest,spread", [(0.1, 0.5), (0.5, 1.5)])
@pytest.mark.parametrize("value", [0.0, 1e-3])
@pytest.mark.parametrize("count", [500, 16384, 65536])
@KINDS
@pytest.mark.parametrize("tokens,heads", [(1, (4, 1)), (1, (16, 2)), (3, (16, 2))], ids=str)
def test_a_key_of_most_weight_and_no_value_over_8_bits(ops, tokens, heads, kind, count, value, rest, spread):
    """As an attention sink: what is left of the result is the other keys'
    small weights, which keep their own bits."""
    rng = np.random.default_rng(count + tokens)
    q, cache, tables = dominated(ops, rng, kind, True, tokens, count, *heads, 64, rest, spread, value)
    holds(ops, q, cache, tables, [tokens], [count], Attention(1 / math.sqrt(64)))


@pytest.mark.parametrize("power", [8, 20, 60, 100])
@KINDS
@pytest.mark.parametrize("heads", [(4, 2), (8, 2)], ids=str)
def test_hidden_scales_do_not_reach_earlier_rows_of_few(ops, heads, kind, power):
    """The last token's value scale is 2^power times the others': the rows
    before it are what they are without it, bit for bit."""
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([2], [258], *heads, 128, 16, 0, 0, None, False, True), kind, True)
    clean = holds(ops, q, cache, tables, new, counts, spec)
    page, place = int(tables[0][257 // 16]), 257 % 16
    cache.value_scales[page, :, place] *= 2.0 ** power
    out = holds(ops, q, cache, tables, new, counts, spec)
    assert torch.equal(out[:1], clean[:1])


@KINDS
def test_values_of_far_scales_in_one_tile_of_few_rows(ops, kind):
    """Scales from 2^-126 to 2^100, among them zeros: a tile's products are in
    steps of its own largest, whatever other tiles hold."""
    rng = np.random.default_rng(12)
    tables, pages = plain.tables_of(rng, 1, 40)
    cache = plain.random_cache(rng, True, pages, 16, 2, 128)
    for size in ([-126, -20], [-30, 100], [-110, -100], [95, 100]):
        spread = rng.uniform(*size, (pages, 2, 16)) if size[1] - size[0] < 50 else np.repeat(
            rng.uniform(*size, (pages, 2, 1)), 16, 2)
        cache.value_scales.copy_(torch.from_numpy(np.exp2(spread).astype(np.float32)).cuda())
        cache.value_scales[int(tables[0][0])] = 0.0
        q = floats(rng, 2, 8, 128).to(TYPES[kind])
        for count in (20, 600):
            holds(ops, q, cache, tables, [2], [count], Attention(1 / math.sqrt(128)))


# ---- many rows --------------------------------------------------------------------

@pytest.mark.parametrize("rest,spread", [(0.1, 0.5), (0.5, 1.5)])
@pytest.mark.parametrize("count", [500, 16384, 65536])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind,quantized", [("f32", True), ("f32", False), ("bf16", True), ("bf16", False)],
                         ids=["f32-i8", "f32-f16", "bf16-i8", "bf16-f16"])
def test_a_key_of_most_weight_and_no_value(ops, dim, count, kind, quantized, rest, spread):
    """The same for a chunk of 40 tokens and for a step over an F16 cache."""
    rng = np.random.default_rng(count + dim)
    for tokens in (40, 1):
        q, cache, tables = dominated(ops, rng, kind, quantized, tokens, count, 4, 2, dim, rest, spread, 0.0)
        holds(ops, q, cache, tables, [tokens], [count], Attention(1 / math.sqrt(dim)))


# (as FEW: units of 128 rows and of 256; codes converted tile by tile, or
# expanded first, which is where there are several units)
MANY = [
    ([12, 40], [3000, 700], 8, 2, 128),
    ([40, 1], [2000, 16], 16, 2, 256),
    ([70, 30], [1300, 30], 16, 4, 64),
    ([33], [1500], 10, 2, 80),
    ([150, 20], [4000, 2000], 8, 2, 128),
    ([700, 5], [1100, 500], 8, 2, 64),
    ([400], [400], 16, 2, 256),
    ([900], [1400], 8, 2, 128),
]


@pytest.mark.parametrize("window,softcap,sinks", [(0, None, False), (300, 20.0, True)], ids=["plain", "window-cap-sinks"])
@KINDS
@CACHES
@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{c[0]}of{c[1]}h{c[2]}/{c[3]}d{c[4]}".replace(" ", ""))
def test_many_rows(ops, case, quantized, kind, window, softcap, sinks):
    new, counts, tables, page_size, cache, q, spec = attention_case(
        (*case, 16, window, 4 if window else 0, softcap, sinks, True), kind, quantized)
    holds(ops, q, cache, tables, new, counts, spec)


@pytest.mark.parametrize("power", [8, 20, 40, 70])
@KINDS
@pytest.mark.parametrize("tokens", [48, 600])
def test_hidden_scales_do_not_reach_earlier_rows_of_many(ops, tokens, kind, power):
    """The last token's value scale, and its key's, is 2^power times the
    others', for converted codes and expanded ones: the rows before it keep
    their own bits."""
    for dim in (64, 128):
        new, counts, tables, page_size, cache, q, spec = attention_case(
            ([tokens], [tokens + 200], 8, 2, dim, 16, 0, 0, None, False, True), kind, True)
        page, place = int(tables[0][(tokens + 199) // 16]), (tokens + 199) % 16
        cache.value_scales[page, :, place] *= 2.0 ** power
        holds(ops, q, cache, tables, new, counts, spec)
        cache.key_scales[page, :, place] *= 2.0 ** power
        out = torch.empty_like(q)
        ops.attention_chunks(q, cache, plain.chunks_of(new, counts, tables, 16), spec, out)
        expected, off = chunk_accuracy.attention(q[:-1], cache, tables, [tokens - 1], [tokens + 199], spec, tokens)
        assert ((out[:-1].double() - expected).abs() <= off).all()


@KINDS
@pytest.mark.parametrize("tokens", [48, 600])
def test_values_of_far_scales_for_many_rows(ops, tokens, kind):
    """As for few rows; and scales that grow, or fall, from tile to tile."""
    rng = np.random.default_rng(13)
    count = tokens + 500
    tables, pages = plain.tables_of(rng, 1, -(-count // 16))
    cache = plain.random_cache(rng, True, pages, 16, 2, 128)
    position = np.zeros((pages, 1, 16))
    position[tables[0]] = np.arange(tables.size * 16).reshape(-1, 1, 16)
    grows = position / count * np.ones((1, 2, 1))
    q = floats(rng, tokens, 8, 128).to(TYPES[kind])
    for size in (rng.uniform(-40, 0, (pages, 2, 16)), rng.uniform(-110, -100, (pages, 2, 1)) * np.ones((1, 1, 16)),
                 rng.uniform(95, 100, (pages, 2, 1)) * np.ones((1, 1, 16)), 60 * grows, -60 * grows, 120 * grows - 100):
        cache.value_scales.copy_(torch.from_numpy(np.exp2(size).astype(np.float32)).cuda())
        cache.value_scales[int(tables[0][0])] = 0.0
        holds(ops, q, cache, tables, [tokens], [count], Attention(1 / math.sqrt(128)))


@pytest.mark.parametrize("power", [-70, -40, 40, 70])
@KINDS
@pytest.mark.parametrize("tokens", [1, 5, 48, 600])
def test_small_queries_of_large_keys(ops, tokens, kind, power):
    """q times 2^-power and keys' scales times 2^power: the same scores."""
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens], [tokens + 200], 8, 2, 64, 16, 0, 0, None, False, True), kind, True)
    cache.key_scales.mul_(2.0 ** power)
    holds(ops, q * 2.0 ** -power, cache, tables, new, counts, spec)
    none = Attention(0.0)
    holds(ops, q * 2.0 ** -power, cache, tables, new, counts, none)


# ---- scores and scales that change along the keys --------------------------------------

def ramped(ops, rng, kind, quantized, tokens, count, q_heads, kv_heads, dim, height, shape):
    """Scores that rise by `height` (in powers of e) along the keys, fall, or
    stand in steps of 200 keys, under noise of about one."""
    along = floats(rng, kv_heads, 1, dim)
    along = along / along.norm(dim=2, keepdim=True)
    at = torch.arange(count, device="cuda", dtype=torch.float32)[:, None, None] / count
    ramp = {"rises": at, "falls": 1 - at, "steps": torch.floor(at * count / 200) * 200 / count,
            "peaks": torch.exp(-((at - 0.5) * 8) ** 2)}[shape] * height
    q = floats(rng, tokens, kv_heads, q_heads // kv_heads, dim) + math.sqrt(dim) * along
    k = floats(rng, count, kv_heads, dim) + ramp * along[None, :, 0]
    cache, tables = written(ops, rng, quantized, k, floats(rng, count, kv_heads, dim))
    return q.reshape(tokens, q_heads, dim).to(TYPES[kind]), cache, tables


@pytest.mark.parametrize("shape", ["rises", "falls", "steps", "peaks"])
@pytest.mark.parametrize("height", [4.0, 15.0, 60.0])
@CACHES
@KINDS
def test_scores_that_grow_along_the_keys(ops, kind, quantized, height, shape):
    """Bases move in the middle of a chain of tiles, outputs with them: for few
    rows and many, whole and in splits, with a sink between the first score
    and the last."""
    rng = np.random.default_rng(int(height))
    for tokens, count, dim in ((1, 3000, 128), (5, 1500, 64), (40, 2500, 128), (300, 1700, 64), (130, 900, 256), (48, 20000, 80)):
        q, cache, tables = ramped(ops, rng, kind, quantized, tokens, count, 4, 2, dim, height, shape)
        for sinks in (None, torch.full((4,), height / 2, device="cuda")):
            holds(ops, q, cache, tables, [tokens], [count], Attention(1 / math.sqrt(dim), sinks=sinks))


@pytest.mark.parametrize("grows", [1.0, 3.0, -3.0])
@KINDS
def test_scales_that_grow_from_tile_to_tile(ops, kind, grows):
    """Key and value scales that double (or halve) every 64 positions once and
    thrice, under scores that rise."""
    rng = np.random.default_rng(17)
    for tokens, count, dim in ((1, 2000, 128), (5, 1500, 64), (40, 1500, 128), (300, 1400, 64), (130, 900, 256)):
        q, cache, tables = ramped(ops, rng, kind, True, tokens, count, 4, 2, dim, 10.0, "rises")
        position = np.zeros((cache.pages, 1, 16))
        position[tables[0]] = np.arange(tables.size * 16).reshape(-1, 1, 16)
        by = torch.from_numpy(np.exp2(position // 64 * grows).astype(np.float32)).cuda()
        cache.value_scales.mul_(by)
        holds(ops, q, cache, tables, [tokens], [count], Attention(1 / math.sqrt(dim)))
        cache.key_scales.mul_(by ** 0.1)
        holds(ops, q, cache, tables, [tokens], [count], Attention(1 / math.sqrt(dim)))


@CACHES
@KINDS
@pytest.mark.parametrize("tokens", [1, 2, 6, 48, 300])
def test_a_query_of_one_large_value(ops, tokens, kind, quantized):
    """A dimension in which q is 4000 times as large as elsewhere and the keys
    are nothing: the others' scores keep their bits."""
    rng = np.random.default_rng(tokens)
    for dim, heads in ((64, (4, 2)), (128, (4, 1)), (256, (16, 2))):
        k, v = floats(rng, 900, heads[1], dim), floats(rng, 900, heads[1], dim)
        k[..., 7] = 0.0
        cache, tables = written(ops, rng, quantized, k, v)
        q = floats(rng, tokens, heads[0], dim)
        q[..., 7] *= 4000.0
        holds(ops, q.to(TYPES[kind]), cache, tables, [tokens], [900], Attention(2 / math.sqrt(dim)))


@KINDS
def test_heads_and_sequences_of_far_scales_beside_others(ops, kind):
    """One head of one sequence has scales far apart and the others do not:
    each goes its own way (BF16 rows' expanded codes in two launches), with
    splits and without."""
    for new, counts in (([300, 250], [4000, 700]), ([1200, 700], [1300, 2400]), ([40, 48], [2000, 900])):
        new, counts, tables, page_size, cache, q, spec = attention_case(
            (new, counts, 8, 2, 128, 16, 0, 0, None, True, True), kind, True)
        cache.value_scales[int(tables[0][3]), 1, 5] *= 2.0 ** 30
        cache.key_scales[int(tables[1][20]), 0, 9] *= 2.0 ** -30
        holds(ops, q, cache, tables, new, counts, spec)
        windowed = Attention(spec.scale, window=200, first=3, sinks=spec.sinks)
        holds(ops, q, cache, tables, new, counts, windowed)


@KINDS
@pytest.mark.parametrize("tokens", [1, 5, 48, 600])
def test_keys_or_values_of_zeros(ops, tokens, kind):
    """Scales of zero in all that a head sees, or in all of its keys."""
    for dim in (64, 128, 256):
        new, counts, tables, page_size, cache, q, spec = attention_case(
            ([tokens, 1], [tokens + 90, 1], 8, 2, dim, 16, 0, 0, None, dim == 128, True), kind, True)
        cache.value_scales[:, 0] = 0.0
        cache.key_scales[:, 1] = 0.0
        bounds = dict(longest=tokens + 100, max_keys=tokens + 105)
        for b in ({}, bounds):
            out = holds(ops, q, cache, tables, new, counts, spec, **b)
            assert (out[:, :4] == 0.0).all()
        cache.value_scales.zero_()
        cache.key_scales.zero_()
        assert (holds(ops, q, cache, tables, new, counts, spec) == 0.0).all()
