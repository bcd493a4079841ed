"""The bound of tests/chunk_accuracy.py tells mistakes from roundings: a key left
out and a page taken from elsewhere are far outside it (on the CPU, planted in
the plain form)."""

import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from drift_b200.ops import Attention
from tests import chunk_accuracy

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def random_cache(rng, quantized, pages, page_size, kv_heads, dim):
    sides = (pages, page_size, kv_heads, dim), (pages, kv_heads, dim, page_size)
    if quantized:
        keys, values = (torch.from_numpy(rng.integers(-127, 128, s, dtype=np.int8)) for s in sides)
        scales = [torch.from_numpy(rng.uniform(0.005, 0.025, (pages, kv_heads, page_size)).astype(np.float32)) for _ in range(2)]
        return SimpleNamespace(keys=keys, values=values, key_scales=scales[0], value_scales=scales[1], page_size=page_size)
    keys, values = (torch.from_numpy(rng.standard_normal(s).astype(np.float16)) for s in sides)
    return SimpleNamespace(keys=keys, values=values, page_size=page_size)


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 2, 8, 40])
@pytest.mark.parametrize("count", [100, 1500, 4000])
def test_mistakes_are_outside_the_bound(count, tokens, kind, quantized):
    rng = np.random.default_rng(count + tokens)
    q_heads, kv_heads, dim, page_size = 4, 1, 128, 16
    stride = -(-count // page_size)
    cache = random_cache(rng, quantized, stride + 1, page_size, kv_heads, dim)
    tables = rng.permutation(stride + 1)[:stride].astype(np.int32)[None]
    q = torch.from_numpy(rng.standard_normal((tokens, q_heads, dim)).astype(np.float32)).to(TYPES[kind])
    spec = Attention(1 / math.sqrt(dim))
    expected, off = chunk_accuracy.attention(q, cache, tables, [tokens], [count], spec)
    assert (off > 0).all()

    def outside(other):
        return ((other - expected).abs() > off).any(2)

    spare = [p for p in range(stride + 1) if p not in tables[0]][0]
    # the last row's own key left out (it may weigh little for some head)
    last = expected.clone()
    last[-1:] = chunk_accuracy.attention(q[-1:], cache, tables, [1], [count - 1], spec)[0]
    assert outside(last)[-1].any()
    # a page of another sequence in the middle of the table
    swapped = tables.copy()
    swapped[0, stride // 2 if stride > 2 else 0] = spare
    assert outside(chunk_accuracy.attention(q, cache, swapped, [tokens], [count], spec)[0])[-1].any()
    # one value's scale, or value, doubled
    changed = cache.value_scales if quantized else cache.values
    page, place = tables[0][count // 2 // page_size], count // 2 % page_size
    before = changed.clone()
    changed[page, ..., place] *= 2
    other = chunk_accuracy.attention(q, cache, tables, [tokens], [count], spec)[0]
    changed.copy_(before)
    assert outside(other)[-1].any()
    # and its results rounded once to their type are inside
    assert not outside(expected.to(q.dtype).double()).any()


@pytest.mark.parametrize("quantized", [True, False], ids=["i8", "f16"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_a_missing_rescale_is_outside_the_bound(tokens, kind, quantized):
    """Scores that rise: a row's base moves, and the results so far with it. The
    last move left out of them is far outside, if keys before it count."""
    rng = np.random.default_rng(tokens)
    count, dim = 1500, 64
    cache = random_cache(rng, quantized, 94, 16, 1, dim)
    tables = np.arange(94, dtype=np.int32)[None]
    q = torch.from_numpy(rng.standard_normal((tokens, 1, dim)).astype(np.float32)).to(TYPES[kind])
    spec = Attention(1 / math.sqrt(dim))
    expected, off = chunk_accuracy.attention(q, cache, tables, [tokens], [count], spec)
    _, v, _ = chunk_accuracy.sequence(cache, tables[0], count)
    k = chunk_accuracy.sequence(cache, tables[0], count)[0]
    for i in range(tokens):
        score = k[:count - tokens + i + 1, 0] @ q[i, 0].double() * spec.scale
        p = torch.softmax(score, 0)
        for moved in (64, 640, 1216):  # keys before the move; it was by 2^3
            other = expected[i, 0] + 7 * (p[:moved] @ v[:moved, 0])
            assert ((other - expected[i, 0]).abs() > off[i, 0]).any()
