"""What the chunk operators' 8-bit cache and its neighbours refuse, and the
accuracy that they keep where weights, scales and bounds are far apart."""

import math

import pytest
import torch

from drift_b200.ops import Attention, Chunks, CudaOps, KvCache, QuantizedKvCache, Rope
from tests import chunks as plain
from tests.test_gpu_chunks import attention_case, held

pytestmark = pytest.mark.gpu

CACHES = pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
KINDS = pytest.mark.parametrize("kind", ["f32", "bf16"])


@pytest.fixture(scope="module")
def ops():
    return CudaOps()


# ---- caches ---------------------------------------------------------------------

def test_the_f16_calls_refuse_an_8_bit_cache(ops):
    """cache_write, attention and the decode step's two calls read and write
    F16 values: an 8-bit cache's buffers are half as long."""
    zeros = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    codes = QuantizedKvCache.allocate(4, 16, 2, 64)
    halves = KvCache.allocate(4, 16, 2, 64)
    floats = KvCache(halves.keys.float(), halves.values.float(), 16)
    turned = KvCache(halves.keys, halves.keys, 16)
    k, q, norm = zeros(1, 2, 64), zeros(1, 4, 64), zeros(64)
    table, positions = zeros(4, dtype=torch.int32), zeros(1, dtype=torch.int32)
    spec, rope = Attention(0.125), Rope(10000.0, 64, 0)
    calls = [
        ("cacheWrite", lambda cache: ops.cache_write(k, k, cache, table, 0)),
        ("attention", lambda cache: ops.attention(q, cache, table, 0, 1, spec, q.clone())),
        ("attentionInputs", lambda cache: ops.attention_inputs_decode(
            q, k, k, norm, norm, 1e-6, positions, rope, q.clone(), cache, table[None])),
        ("attention", lambda cache: ops.attention_decode(q, cache, table[None], positions, 64, spec, q.clone())),
    ]
    for name, call in calls:
        for cache in (codes, floats):
            with pytest.raises(ValueError, match=f"{name}: the cache is contiguous device memory, torch.float16"):
                call(cache)
        with pytest.raises(ValueError, match=f"{name}: a cache of keys"):
            call(turned)
        call(halves)
    assert ops.take_device_error() == 0
    assert not codes.keys.any() and not codes.values.any()


# ---- bounds ---------------------------------------------------------------------

@CACHES
@KINDS
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("tokens", [1, 5, 60, 300])
def test_a_window_of_no_limit(ops, tokens, causal, kind, quantized):
    """The largest window that an int holds is no window, for few rows and
    many, and so is one of the positions that there are."""
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([tokens, 1], [tokens + 211, 130], 8, 2, 64, 16, 0, 0, None, False, causal), kind, quantized)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    for window in (2 ** 31 - 1, 2 ** 31 - 2 - tokens, tokens + 211):
        for first in (0, 7):
            out = torch.full_like(q, 7.0)
            wide = Attention(1 / math.sqrt(64), causal, window, first=first)
            ops.attention_chunks(q, cache, chunks, wide, out)
            held(out, *plain.attention(q, cache, tables, new, counts, spec))


def test_bounds_past_32_bits_are_refused(ops):
    """2^32 + 5 is not a window of 5."""
    new, counts, tables, page_size, cache, q, spec = attention_case(
        ([3], [30], 8, 2, 64, 16, 0, 0, None, False, True), "f32", True)
    chunks = plain.chunks_of(new, counts, tables, page_size)
    out = torch.full_like(q, 7.0)
    for changes in (dict(window=2 ** 32 + 5), dict(window=2 ** 31), dict(window=-1), dict(window=5, first=2 ** 32),
                    dict(window=5, first=-2 ** 32)):
        with pytest.raises(ValueError, match="a window of"):
            ops.attention_chunks(q, cache, chunks, Attention(0.125, **changes), out)
    for longest, max_keys in ((2 ** 32 + 3, 30), (3, 2 ** 32 + 30), (-1, 30), (3, -1)):
        with pytest.raises(ValueError, match="of one sequence"):
            Chunks(chunks.starts, chunks.positions, chunks.page_tables, longest, max_keys)
    assert (out == 7.0).all()
