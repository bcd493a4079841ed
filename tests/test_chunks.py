"""What the chunk calls of the C ABI refuse, before any CUDA call."""

import ctypes

import pytest

from drift_b200 import _lib

F32, F16, Q8_0, I8, BF16 = 0, 1, 8, 24, 30
AT = 4096  # an aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(status, fragment):
    assert status == _lib.DRIFT_ERROR_INVALID_ARGUMENT
    message = _lib.load().drift_last_error_message().decode()
    assert fragment in message, message


GOOD = dict(x_dtype=F32, k=AT, v=AT, tokens=8, kv_heads=2, head_dim=128, cache_dtype=I8, keys=AT, values=AT,
            key_scales=AT, value_scales=AT, pages=4, page_size=16, tables=AT, stride=4, starts=AT, positions=AT,
            batch=2, longest=5)


def cache_call(lib, name, **changes):
    a = {**GOOD, **changes}
    return getattr(lib, name)(*(a[key] for key in GOOD), None)


SHARED = [
    (dict(x_dtype=F16), "takes F32 (or BF16), not F16"),
    (dict(cache_dtype=Q8_0), "a cache of Q8_0"),
    (dict(head_dim=96), "heads of 96"),
    (dict(page_size=24), "pages of 24 tokens: not a multiple of 16"),
    (dict(page_size=0), "pages of 0 tokens"),
    (dict(pages=0), "a cache of 0 pages"),
    (dict(kv_heads=0), "0 heads"),
    (dict(tokens=-1), "-1 tokens"),
    (dict(batch=-1), "of -1 sequences"),
    (dict(batch=65536), "of 65536 sequences"),
    (dict(longest=-1), "-1 of one at most"),
    (dict(longest=65), "a page table of 4 pages for 65 positions"),
    (dict(tables=None), "a page table"),
    (dict(stride=2 ** 27), "a page table"),  # 2^31 positions
    (dict(starts=None), "a null tensor"),
    (dict(positions=None), "a null tensor"),
    (dict(keys=None), "a null tensor"),
    (dict(key_scales=None), "an 8-bit cache without scales"),
    (dict(values=AT + 8), "16-byte boundary"),
]


@pytest.mark.parametrize("name", ["drift_cache_write_chunks", "drift_cache_read_chunks"])
@pytest.mark.parametrize("changes,fragment", SHARED + [(dict(k=None), "a null tensor"), (dict(v=AT + 4), "16-byte boundary")],
                         ids=str)
def test_cache_refusals(lib, name, changes, fragment):
    refused(cache_call(lib, name, **changes), fragment)


@pytest.mark.parametrize("name", ["drift_cache_write_chunks", "drift_cache_read_chunks"])
@pytest.mark.parametrize("changes", [dict(tokens=0), dict(batch=0), dict(longest=0)], ids=str)
def test_no_tokens_are_nothing_to_do(lib, name, changes):
    assert cache_call(lib, name, **changes) == 0


ATTENTION = dict(x_dtype=F32, q=AT, tokens=8, q_heads=8, kv_heads=2, head_dim=128, cache_dtype=I8, keys=AT, values=AT,
                 key_scales=AT, value_scales=AT, pages=4, page_size=16, tables=AT, stride=4, starts=AT, positions=AT,
                 batch=2, longest=5, max_keys=64, scale=0.1, causal=1, window=0, first=0, softcap=0.0, sinks=None,
                 out=AT, workspace=AT, workspace_bytes=1 << 40)


def attention_call(lib, **changes):
    a = {**ATTENTION, **changes}
    return lib.drift_attention_chunks(*(a[key] for key in ATTENTION), None)


@pytest.mark.parametrize("changes,fragment", SHARED + [
    (dict(q_heads=7), "7 query heads over 2"),
    (dict(q_heads=0), "0 query heads over 2"),
    (dict(q_heads=34), "17 query heads per key head"),
    (dict(max_keys=65), "65 keys in a page table of 4 pages"),
    (dict(max_keys=4), "4 keys in a page table of 4 pages, chunks of 5"),
    (dict(window=-1), "a window of -1"),
    (dict(window=3, first=-1), "with -1 first keys"),
    (dict(first=2), "first keys without a window"),
    (dict(q=None), "a null tensor"),
    (dict(out=AT + 8), "16-byte boundary"),
    (dict(stride=4096, max_keys=65536, longest=1, batch=1, workspace_bytes=0), "a workspace of 0 bytes"),
    (dict(stride=4096, max_keys=65536, longest=1, batch=1, workspace=None), "a workspace of"),
    (dict(stride=4096, max_keys=65536, longest=1, batch=1, workspace=AT + 4), "16-byte boundary"),
], ids=str)
def test_attention_refusals(lib, changes, fragment):
    refused(attention_call(lib, **changes), fragment)


def test_no_attention_is_nothing_to_do(lib):
    assert attention_call(lib, tokens=0) == 0
    assert attention_call(lib, batch=0) == 0


def test_workspace_bytes(lib):
    size = lambda **c: lib.drift_attention_chunks_workspace_bytes(*({**dict(  # noqa: E731
        x_dtype=F32, tokens=8, q_heads=32, kv_heads=8, head_dim=128, cache_dtype=I8, pages=64, page_size=16, batch=8,
        longest=1, max_keys=4096, causal=1,
        window=0, first=0), **c}.values()))
    assert size() > 0                       # few rows: split over the keys
    assert size(max_keys=16) == 0           # one split
    assert size(tokens=0) == 0
    assert size(window=16) < size()         # a window bounds the splits
    # a split's partial row: the output, the largest score and the sum
    assert size() % (8 * 32 * (128 + 2) * 4) == 0


def test_rows_past_32_bits_are_refused(lib):
    """`longest` bounds a launch's rows: sixteen heads of 2^27 - 1 tokens fit in
    31 bits, but not with the rest of their last unit."""
    for longest in (2 ** 27 - 1, 2 ** 27):
        for cache_dtype in (I8, F16):
            refused(attention_call(lib, longest=longest, max_keys=2 ** 27, stride=2 ** 23, q_heads=16, kv_heads=1, batch=1,
                                   cache_dtype=cache_dtype, out=AT + (1 << 20)), f"chunks of {longest} tokens of 16 heads")
