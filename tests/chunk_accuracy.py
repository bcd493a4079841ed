"""attention_chunks in 64 bits with the error to expect of each kernel, tight
enough to tell a key left out or taken from another page.

A result is o = sum_k p_k v_k over the keys that a row sees. If key k's score
is off by e_k, o is off by sum_k p_k e_k (v_k - o): the sum of the weights is off
with them. A weight's rounding for the product with its value is not in that
sum: there o is off by sum_k p_k e_k v_k (a row of one key, whose weight over
the sum is one: by all of a half step). Roundings of different keys are
independent, so their squares add, and a result may be off by SIGMAS times the root; a uniform
error of a half step h has a deviation of h / sqrt(3). What repeats from key to
key (F32 and tensor-core sums of a score, the functions of one score) is added
in the open. The result's own rounding is half a step of its type."""

import math

import numpy as np
import torch

from drift_b200.ops import QuantizedKvCache

SIGMAS = 7.0
UNIFORM = 1 / math.sqrt(3)
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative
FEW_ROWS = {torch.float32: {64: 40, 80: 40, 128: 40, 256: 64}, torch.bfloat16: {64: 32, 80: 32, 128: 32, 256: 24}}


def sequence(cache, table, count):
    """Positions 0 .. count - 1: keys, values in 64 bits [count, kv_heads, D]
    and the values' scales [count, kv_heads] (None for an F16 cache)."""
    device = cache.keys.device
    at = torch.arange(count, device=device)
    page = torch.as_tensor(np.asarray(table), device=device)[at // cache.page_size].long()
    place = at % cache.page_size
    k, v = cache.keys[page, place].double(), cache.values[page, :, :, place].double()
    if not hasattr(cache, "key_scales"):
        return k, v, None
    scales = cache.value_scales[page, :, place].double()
    return k * cache.key_scales[page, :, place].double()[..., None], v * scales[..., None], scales


def roundings(dtype, quantized, rows, dim):
    """(q's step over its largest value, a weight's relative half step, its
    absolute half step over the row's largest, the step of a tile's products of
    weight and scale over the largest of 32 keys, a key's and value's relative
    half step) of the kernel that a chunk of `rows` rows of a key head goes to."""
    f32 = dtype == torch.float32
    if not quantized:
        # two F16 terms, or one; the largest weight is 2^12 or more (BF16: 2^8)
        if f32:
            return 2.0 ** -21, 2.0 ** -22, 2.0 ** -37, 0.0, 0.0
        return 0.0, 2.0 ** -11, 2.0 ** -33, 0.0, 0.0
    if rows <= FEW_ROWS[dtype][dim]:
        # whole numbers, of 29 bits or (BF16, more than four rows) 21
        step = 2.0 ** -29 if f32 or rows <= 4 else 2.0 ** -21
        return step, 0.0, 0.0, step, 0.0
    if f32:
        return 2.0 ** -21, 2.0 ** -22, 2.0 ** -36, 0.0, 0.0
    # (codes expanded first: with their scales, in F16)
    return 0.0, 2.0 ** -11, 2.0 ** -31, 0.0, 2.0 ** -11


def attention(q, cache, tables, new, counts, spec, longest=None):
    """(results, how far off they may be), both [tokens, q_heads, D] in 64 bits."""
    tokens, q_heads, dim = q.shape
    group = q_heads // cache.keys.shape[2]
    quantized = isinstance(cache, QuantizedKvCache) or hasattr(cache, "key_scales")
    rows = (longest or max(new)) * group
    q_step, relative, absolute, product, coded = roundings(q.dtype, quantized, rows, dim)
    # (many BF16 rows: all keys of a split are one chain; else a tile's are)
    in_place = q.dtype == torch.bfloat16 and rows > (FEW_ROWS[q.dtype][dim] if quantized else 8)
    out = torch.zeros(tokens, q_heads, dim, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    row = 0
    for z, (n, count) in enumerate(zip(new, counts)):
        if n == 0:
            continue
        k, v, scales = sequence(cache, tables[z], count)
        key = torch.arange(count, device=q.device)[None]
        position = torch.arange(count - n, count, device=q.device)[:, None]
        seen = key <= position if spec.causal else torch.ones(n, count, dtype=torch.bool, device=q.device)
        if spec.window:
            seen = seen & ((key > position - spec.window) | (key < spec.first))
        any_row = seen.any(0)
        for h in range(q_heads):
            x = q[row:row + n, h].double()
            kh = torch.where(any_row[:, None], k[:, h // group], 0.0)  # (what no row sees may be a NaN)
            vh = torch.where(any_row[:, None], v[:, h // group], 0.0)
            score = (x @ kh.T) * spec.scale
            magnitude = (x.abs() @ kh.abs().T) * abs(spec.scale)
            if spec.softcap:
                score = spec.softcap * torch.tanh(score / spec.softcap)
            hidden = score.masked_fill(~seen, -math.inf)
            largest = hidden.amax(1, keepdim=True)
            if spec.sinks is not None:
                largest = torch.maximum(largest, spec.sinks[h].double())
            weight = torch.exp(hidden - largest)
            total = weight.sum(1, keepdim=True)
            if spec.sinks is not None:
                total = total + torch.exp(spec.sinks[h].double() - largest)
            p = weight / total
            o = p @ vh
            # one key's own: q's steps in its score
            step = q_step * x.abs().amax(1, keepdim=True) / 2 * UNIFORM * abs(spec.scale)
            own = (step * kh.norm(dim=1)[None]) ** 2
            if coded:
                own = own + (coded * UNIFORM * spec.scale) ** 2 * ((x * x) @ (kh * kh).T)
            mass = p * p * own
            square = mass @ (vh * vh) - 2 * o * (mass @ vh) + o * o * mass.sum(1, keepdim=True)
            # its weight's rounding, and its value's
            square = square + (relative ** 2 + coded ** 2) * UNIFORM ** 2 * ((p * p) @ (vh * vh))
            # rounded with its value's scale in it, of which the largest counts; where
            # scales are in the values (BF16 rows' expanded codes) of the largest weight
            if absolute:
                reach = p if scales is None else p * scales[None, :, h // group].nan_to_num(0.0)
                reach = torch.where(seen, reach, 0.0).amax(1, keepdim=True)
                size = vh if scales is None else torch.where(scales[:, h // group, None] > 0,
                                                             vh / scales[:, h // group, None], 0.0)
                square = square + (absolute * UNIFORM * reach) ** 2 * (seen.double() @ (size * size))
                if coded:
                    square = square + (absolute * UNIFORM * p.amax(1, keepdim=True)) ** 2 * (seen.double() @ (vh * vh))
            if product:
                s = torch.where(any_row, scales[:, h // group], 0.0)
                tiles = torch.nn.functional.pad(torch.where(seen, p * s, 0.0), (0, -count % 32)).view(n, -1, 32)
                tile = tiles.amax(2, keepdim=True).expand_as(tiles).reshape(n, -1)[:, :count]
                code = torch.where(s[:, None] > 0, vh / torch.where(s > 0, s, 1.0)[:, None], 0.0)
                square = square + (product / 2 * UNIFORM) ** 2 * ((tile * seen) ** 2 @ (code * code))
            # sums of a score (D / 16 steps of one or two terms) and the functions of it
            common = p * (magnitude * (dim / 8) * 2.0 ** -24 + score.abs() * 2.0 ** -22 + 2.0 ** -21)
            shared = common @ vh.abs() + o.abs() * common.sum(1, keepdim=True)
            # the results' sums: a chain's steps drop bits of the largest that they add
            largest = torch.stack([(p[i, :, None] * vh.abs()).amax(0) for i in range(n)])
            largest = torch.maximum(largest, o.abs() + 4 * ((p * p) @ (vh * vh)).sqrt())
            chain = (16 + count / (16 if in_place else 128)) * 2.0 ** -24 * largest
            out[row:row + n, h] = o
            off[row:row + n, h] = SIGMAS * square.clamp(min=0).sqrt() + shared + chain + o.abs() * ROUND[q.dtype] + 1e-37
        row += n
    return out, off
