"""What the tests of the chunk operators share: random caches and chunks, and
plain forms in 64 bits with the error bounds that follow from the roundings."""

import math

import numpy as np
import torch

from drift_b200.ops import Chunks, KvCache, QuantizedKvCache

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def tables_of(rng, batch, stride, spare=3):
    """Page tables over a cache of a few pages more, in random order."""
    pages = batch * stride + spare
    return rng.permutation(pages)[:batch * stride].astype(np.int32).reshape(batch, stride), pages


def chunks_of(new, counts, tables, page_size, device="cuda", longest=None, max_keys=None):
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    positions = np.array([c - n for n, c in zip(new, counts)], dtype=np.int32)
    as_device = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(device)  # noqa: E731
    return Chunks(as_device(starts), as_device(positions), as_device(tables),
                  max(new) if longest is None else longest,
                  max(max(counts), max(new)) if max_keys is None else max_keys)


def random_cache(rng, quantized, pages, page_size, kv_heads, dim, scale_range=(0.005, 0.025)):
    """A cache full of random keys and values."""
    if quantized:
        codes = lambda *s: torch.from_numpy(rng.integers(-127, 128, s, dtype=np.int8)).cuda()  # noqa: E731
        scales = lambda: torch.from_numpy(  # noqa: E731
            rng.uniform(*scale_range, (pages, kv_heads, page_size)).astype(np.float32)).cuda()
        return QuantizedKvCache(codes(pages, page_size, kv_heads, dim),
                                codes(pages, kv_heads, dim, page_size), scales(), scales(), page_size)
    halves = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float16)).cuda()  # noqa: E731
    return KvCache(halves(pages, page_size, kv_heads, dim), halves(pages, kv_heads, dim, page_size),
                   page_size)


def sequence(cache, table, count):
    """Keys and values of positions 0 .. count - 1 in 64 bits, [count, kv_heads, D]."""
    at = torch.arange(count, device="cuda")
    page = torch.as_tensor(np.asarray(table), device="cuda")[at // cache.page_size].long()
    place = at % cache.page_size
    k, v = cache.keys[page, place].double(), cache.values[page, :, :, place].double()
    if isinstance(cache, QuantizedKvCache):
        k = k * cache.key_scales[page, :, place].double()[..., None]
        v = v * cache.value_scales[page, :, place].double()[..., None]
    return k, v


def attention(q, cache, tables, new, counts, spec):
    """(out, tolerance) of attention_chunks in 64 bits.

    The tolerance, per value, from the kernels' roundings. A score is a sum of
    q_i k_i: q in two F16 terms is off by 2^-21 of its row's largest value at
    most (one term holds BF16 exactly), and each of the D / 16 accumulations a
    term drops at most 2^-22 of the sum of magnitudes; the scale, the
    softcap's functions and the base-2 factor are a few F32 roundings of the
    score. A weight's relative error is the score's absolute one, twice over
    (its row's largest is off too), exp2's 2^-22, its rounding (2^-21 in two
    terms, 2^-11 in one, and 2^-38 of the largest at least), and its sums'
    accumulations, 2^-22 of the magnitudes each over a chain of keys / 16
    steps. The result is rounded to its type."""
    tokens, q_heads, dim = q.shape
    group = q_heads // cache.kv_heads
    out = torch.zeros(tokens, q_heads, dim, dtype=torch.float64, device="cuda")
    tolerance = torch.zeros_like(out)
    row = 0
    for z, (n, count) in enumerate(zip(new, counts)):
        if n == 0:
            continue
        k, v = sequence(cache, tables[z], count)
        scales = None
        if isinstance(cache, QuantizedKvCache):
            at = torch.arange(count, device="cuda")
            page = torch.as_tensor(np.asarray(tables[z]), device="cuda")[at // cache.page_size].long()
            scales = cache.value_scales[page, :, at % cache.page_size].double()
            key_scales = cache.key_scales[page, :, at % cache.page_size].double()
        key = torch.arange(count, device="cuda")[None]
        position = torch.arange(count - n, count, device="cuda")[:, None]
        seen = key <= position if spec.causal else torch.ones(n, count, dtype=torch.bool, device="cuda")
        if spec.window:
            seen = seen & ((key > position - spec.window) | (key < spec.first))
        for h in range(q_heads):
            x, kh, vh = q[row:row + n, h].double(), k[:, h // group], v[:, h // group]
            # (what no row sees may be a NaN)
            kh = torch.where(seen.any(0)[:, None], kh, 0.0)
            vh = torch.where(seen.any(0)[:, None], vh, 0.0)
            score = (x @ kh.T) * spec.scale
            magnitude = (x.abs() @ kh.abs().T) * abs(spec.scale)
            # (few BF16 rows over an 8-bit cache: q in steps of 2^-13 of its
            # leading bit's worth, and weights in steps of 2^-18)
            steps = 2.0 ** -14 if cache.keys.dtype == torch.int8 and q.dtype == torch.bfloat16 else 2.0 ** -21
            lost = (x.abs().amax(1, keepdim=True) * kh.abs().sum(1)[None]) * abs(spec.scale) * steps
            if spec.softcap:
                score = spec.softcap * torch.tanh(score / spec.softcap)
            rounded = coded = 0.0
            if scales is not None and q.dtype == torch.bfloat16:
                # BF16 rows may meet keys and values rounded to F16 over a power
                # of two under twice the largest scale: 2^-11 for the scale's
                # rounding and 2^-11 for the product's, of each key and value,
                # and 2^-25 of the power at least.
                rounded = magnitude * 2 * 2.0 ** -11 + x.abs().sum(1, keepdim=True) * abs(spec.scale) * (
                    2.0 ** -25 * 2 * key_scales[seen.any(0), h // group].max())
                coded = 2 * 2.0 ** -11
            delta = rounded + lost + magnitude * (2 * dim / 16 * 2.0 ** -22) + score.abs() * 2.0 ** -20
            score = score.masked_fill(~seen, -math.inf)
            delta = delta.masked_fill(~seen, 0.0).amax(1, keepdim=True)
            largest = score.amax(1, keepdim=True)
            if spec.sinks is not None:
                largest = torch.maximum(largest, spec.sinks[h].double())
            none = largest == -math.inf
            weight = torch.exp(score - torch.where(none, 0.0, largest))
            total = weight.sum(1, keepdim=True)
            if spec.sinks is not None:
                total = total + torch.exp(spec.sinks[h].double() - largest)
            safe = torch.where(total > 0, total, 1.0)
            out[row:row + n, h] = (weight @ vh) / safe
            mass = (weight @ vh.abs()) / safe
            rounding = 2.0 ** -21 if q.dtype == torch.float32 else 2.0 ** -11
            chain = 2 * (count / 16 + 16) * 2.0 ** -22
            # An 8-bit cache's weight is rounded with its value's scale in it,
            # in units of a power of two under twice the largest scale seen:
            # off by 2^-38 of that, times a code of at most 127.
            reach = 254 * scales[seen.any(0), h // group].max() if scales is not None else vh.abs().amax(0, keepdim=True)
            # (and a value so rounded is off by 2^-25 of the power at least; the weights sum to one)
            if scales is not None and q.dtype == torch.bfloat16:
                coded_floor = 2.0 ** -25 * 2 * scales[seen.any(0), h // group].max()
            else:
                coded_floor = 0.0
            # a weight in whole steps is off by 2^-27 of one (F32, and up to four
            # rows) or 2^-19, in F16 terms by 2^-38
            step = (2.0 ** -27 if q.dtype == torch.float32 else 2.0 ** -19) if scales is not None else 2.0 ** -38
            floor = coded_floor + seen.sum(1, keepdim=True) * step * reach / torch.where(
                total > 0, torch.minimum(safe, torch.ones_like(safe)), 1.0)
            tolerance[row:row + n, h] = (mass * (2 * delta + 2.0 ** -21 + rounding + coded + chain) + floor
                                         + out[row:row + n, h].abs() * UNIT[q.dtype] + 1e-30)
        row += n
    return out, tolerance


def quantized(x):
    """(codes, scales) of rows in 64 bits: numpy's rounding of an exact-enough
    quotient (53 bits decide where 24-bit operands fall to a half)."""
    x = x.astype(np.float32)
    scale = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
    step = np.where(scale > 0, scale, np.float32(1)).astype(np.float64)
    codes = np.clip(np.rint(x.astype(np.float64) / step[..., None]), -127, 127).astype(np.int8)
    return np.where(scale[..., None] > 0, codes, 0).astype(np.int8), scale
