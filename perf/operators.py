"""The paged cache in 8 bits and the attention of new tokens over it: the cases
measured, their plain form and their definition in 64 bits.

Four operators of `drift_b200.ops.CudaOps`, over a batch of sequences whose new
tokens ("chunks": a prompt or a piece of one, drafted tokens, one token each)
are rows of one array:

- write: `cache_write_chunks` rounds the new keys and values to 8-bit codes
  with one scale per position and head, into each sequence's pages, and
  `cache_read_chunks` reads them back;
- read: `cache_read_chunks` alone, over whole sequences;
- step: `attention_chunks` of one token per sequence;
- chunk: `attention_chunks` of several tokens per sequence.

A cache is F16 or 8-bit ("i8"), pages of `page` positions; q, k, v and the
results are F32 or BF16.
"""

import math

import torch

own = False

BF16, F32 = "bf16", "f32"
TYPES = {BF16: torch.bfloat16, F32: torch.float32}


def listed():
    return [
        # One decoding step's keys and values of 16 sequences (the dense decoder's
        # 8 key heads of 128): the smallest call, where latency counts.
        dict(name="write_step", op="write", type=F32, batch=16, tokens=1, keys=4096, kv=8, dim=128, page=16),
        # Prompts of four users, of different lengths, written in one call.
        dict(name="write_prompts", op="write", type=BF16, batch=4, tokens=4099, keys=8192, kv=8, dim=128, page=16),
        # One short conversation read back whole (the hybrid decoder's 2 key heads
        # of 256), as to hand it to another machine.
        dict(name="read_one", op="read", type=F32, batch=1, tokens=501, keys=501, kv=2, dim=256, page=16),
        # Sixteen conversations of the dense decoder's full context read back.
        dict(name="read_batch", op="read", type=BF16, batch=16, tokens=4096, keys=4096, kv=8, dim=128, page=16),
        # A decoding step of one sequence at the dense decoder's context.
        dict(name="step_one", op="step", cache="i8", type=F32, batch=1, tokens=1, keys=4096, q=32, kv=8, dim=128,
             page=16, window=0, first=0, softcap=0.0, sinks=False),
        # A decoding step of 16 sequences of long contexts.
        dict(name="step_batch", op="step", cache="i8", type=F32, batch=16, tokens=1, keys=16384, q=32, kv=8, dim=128,
             page=16, window=0, first=0, softcap=0.0, sinks=False),
        # The hybrid decoder's heads, F16 cache, a window with the first tokens kept.
        dict(name="step_window", op="step", cache="f16", type=BF16, batch=13, tokens=1, keys=9001, q=16, kv=2, dim=256,
             page=32, window=1024, first=4, softcap=0.0, sinks=False),
        # Up to five drafted tokens of each of eight sequences checked at once.
        dict(name="chunk_drafts", op="chunk", cache="i8", type=F32, batch=8, tokens=5, keys=4096, q=32, kv=8, dim=128,
             page=16, window=0, first=0, softcap=0.0, sinks=False),
        # A piece of a long prompt, the largest case: 2048 tokens after 6144 others.
        dict(name="chunk_long", op="chunk", cache="f16", type=BF16, batch=1, tokens=2048, keys=8192, q=32, kv=8, dim=128,
             page=16, window=0, first=0, softcap=0.0, sinks=False),
        # Pieces of three prompts of different lengths over the 8-bit cache.
        dict(name="chunk_ragged", op="chunk", cache="i8", type=BF16, batch=3, tokens=1001, keys=5003, q=32, kv=8, dim=128,
             page=64, window=0, first=0, softcap=0.0, sinks=False),
        # A whole prompt of narrow heads under a window with the first tokens kept.
        dict(name="chunk_window", op="chunk", cache="f16", type=BF16, batch=1, tokens=6000, keys=6000, q=8, kv=8, dim=64,
             page=32, window=1024, first=4, softcap=0.0, sinks=False),
        # A whole prompt in the runner's own F32, with a softcap and sink logits.
        dict(name="chunk_f32", op="chunk", cache="f16", type=F32, batch=1, tokens=1500, keys=1500, q=16, kv=4, dim=128,
             page=16, window=0, first=0, softcap=30.0, sinks=True),
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "read", "step", "step", "chunk", "chunk"))
    kv, group, dim = rng.choice(((8, 4, 128), (2, 8, 256), (8, 1, 64), (2, 5, 80), (4, 4, 128), (1, 16, 128)))
    case = dict(op=op, type=rng.choice((BF16, F32)), kv=kv, dim=dim, page=rng.choice((16, 32, 48, 64, 128)))
    if op == "write":
        batch = _between(rng, 1, 32)
        tokens = _between(rng, 1, max(1, 8192 // batch))
        return dict(case, batch=batch, tokens=tokens, keys=tokens + _between(rng, 1, 4096))
    if op == "read":
        batch = _between(rng, 1, 16)
        keys = _between(rng, 1, 4096)
        return dict(case, batch=batch, tokens=keys, keys=keys)
    case.update(cache=rng.choice(("i8", "f16")), q=kv * group, softcap=rng.choice((0.0, 0.0, 30.0)),
                sinks=rng.random() < 0.3)
    if op == "step":
        batch = _between(rng, 1, 32)
        keys, tokens = _between(rng, 1, max(64, 65536 // batch)), 1
    else:
        batch = _between(rng, 1, 8)
        tokens = _between(rng, 2, 2048 // batch)
        keys = tokens + _between(rng, 1, 4096)
    windowed = rng.random() < 0.4
    return dict(case, batch=batch, tokens=tokens, keys=keys, window=_between(rng, 1, keys) if windowed else 0,
                first=rng.choice((0, 1, 4, 20)) if windowed else 0)


def _lengths(case):
    """Each sequence's new tokens and its positions with them: the case's in the
    first sequence, from half of them upwards in the others."""
    batch, tokens, keys = case["batch"], case["tokens"], case["keys"]
    part = [1.0 - 0.5 * z / batch for z in range(batch)]
    new = [max(1, round(tokens * p)) for p in part]
    counts = [max(n, round(keys * p)) for n, p in zip(new, part)]
    return (counts, counts) if case["op"] == "read" else (new, counts)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    new, counts = _lengths(case)
    batch, page, kv, dim = case["batch"], case["page"], case["kv"], case["dim"]
    stride = -(-max(counts) // page)
    pages = batch * stride

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # sequences' pages are anywhere in the cache
    tables = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(batch, stride)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = dict(case=case, tables=tables, longest=max(new), keys=max(counts),
                 starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 positions=torch.tensor([c - n for c, n in zip(counts, new)], dtype=torch.int32, device="cuda"))
    total, dtype = starts[-1], TYPES[case["type"]]
    quantized = case.get("cache", "i8") == "i8"
    if case["op"] == "write":
        # keys of a model have a few dimensions much larger than the rest
        wide = 1 + 7 * (torch.rand(dim, generator=g, device="cuda") > 0.95)
        state.update(k=(normal(total, kv, dim) * wide).to(dtype), v=normal(total, kv, dim).to(dtype))
    if quantized:
        blank = case["op"] == "write"

        def codes(*shape):
            return torch.zeros(shape, dtype=torch.int8, device="cuda") if blank else torch.randint(
                -127, 128, shape, generator=g, device="cuda", dtype=torch.int8)

        def scales():
            size = (pages, kv, page)
            return torch.zeros(size, device="cuda") if blank else torch.rand(size, generator=g, device="cuda") * 0.02 + 0.005

        state.update(keys8=codes(pages, page, kv, dim), values8=codes(pages, kv, dim, page), key_scales=scales(),
                     value_scales=scales())
    else:
        state.update(keys16=normal(pages, page, kv, dim).half(), values16=normal(pages, kv, dim, page).half())
    if case["op"] in ("write", "read"):
        state["k_back"] = torch.zeros(total, kv, dim, dtype=dtype, device="cuda")
        state["v_back"] = torch.zeros(total, kv, dim, dtype=dtype, device="cuda")
    else:
        state["q"] = normal(total, case["q"], dim).to(dtype)
        state["out"] = torch.zeros(total, case["q"], dim, dtype=dtype, device="cuda")
        state["sinks"] = normal(case["q"]) if case["sinks"] else None
    if own:
        from drift_b200 import ops

        state["ops"] = ops.CudaOps()
        state["chunks"] = ops.Chunks(state["starts"], state["positions"], tables, state["longest"], state["keys"])
        if quantized:
            state["cache"] = ops.QuantizedKvCache(state["keys8"], state["values8"], state["key_scales"],
                                                  state["value_scales"], page)
        else:
            state["cache"] = ops.KvCache(state["keys16"], state["values16"], page)
        if "q" in state:
            state["attention"] = ops.Attention(1 / math.sqrt(dim), window=case["window"] or None,
                                               softcap=case["softcap"] or None, sinks=state["sinks"],
                                               first=case["first"])
    return state


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "write":
        _plain_write(state)
    if op in ("write", "read"):
        return _plain_read(state)
    return _plain_attention(state)


def _run_own(state):
    calls, op = state["ops"], state["case"]["op"]
    if op in ("write", "read"):
        if op == "write":
            calls.cache_write_chunks(state["k"], state["v"], state["cache"], state["chunks"])
        calls.cache_read_chunks(state["cache"], state["chunks"], state["k_back"], state["v_back"])
        return state["k_back"], state["v_back"]
    calls.attention_chunks(state["q"], state["cache"], state["chunks"], state["attention"], state["out"])
    return state["out"]


# ---- the plain form -------------------------------------------------------------


def _rows(state, total):
    """Each row's sequence and token, and its page and place in the page."""
    row = torch.arange(total, device="cuda")
    starts = state["starts"].long()
    sequence = torch.searchsorted(starts[1:], row, right=True)
    token = row - starts[sequence]
    position = state["positions"].long()[sequence] + token
    page = state["case"]["page"]
    return sequence, token, state["tables"][sequence, position // page].long(), position % page


def _quantized(x):
    """Codes and scales of rows: the scale is the F32 nearest to the largest
    magnitude / 127, a code the whole number nearest to value / scale, halves to
    the even one. In 64 bits, where no quotient is rounded onto a half."""
    x = x.float()
    scale = x.abs().amax(-1) / 127
    quotient = x.double() / torch.where(scale > 0, scale, 1).double()[..., None]
    return quotient.round().clamp(-127, 127).to(torch.int8), scale


def _plain_write(state):
    _, _, page, place = _rows(state, state["k"].shape[0])
    codes, scale = _quantized(state["k"])
    state["keys8"][page, place] = codes
    state["key_scales"][page, :, place] = scale
    codes, scale = _quantized(state["v"])
    state["values8"][page, :, :, place] = codes
    state["value_scales"][page, :, place] = scale


def _plain_read(state):
    k, v = state["k_back"], state["v_back"]
    _, _, page, place = _rows(state, k.shape[0])
    k.copy_(state["keys8"][page, place].float() * state["key_scales"][page, :, place][..., None])
    v.copy_(state["values8"][page, :, :, place].float() * state["value_scales"][page, :, place][..., None])
    return k, v


def _plain_attention(state):
    case, q = state["case"], state["q"]
    kv, dim = case["kv"], case["dim"]
    group, longest, keys = case["q"] // kv, state["longest"], state["keys"]
    # every sequence's keys and values in order, in 32 bits: [batch][kv][keys][dim]
    key = torch.arange(keys, device="cuda")
    page, place = state["tables"][:, key // case["page"]].long(), key % case["page"]
    if "keys8" in state:
        k = state["keys8"][page, place].float() * state["key_scales"][page, :, place][..., None]
        v = state["values8"][page, :, :, place].float() * state["value_scales"][page, :, place][..., None]
    else:
        k, v = state["keys16"][page, place].float(), state["values16"][page, :, :, place].float()
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    # the chunks side by side: [batch][kv][group x longest][dim]
    starts, positions = state["starts"].long(), state["positions"].long()
    token = torch.arange(longest, device="cuda")
    row = (starts[:-1, None] + token).clamp(max=q.shape[0] - 1)
    padded = q[row].float().view(-1, longest, kv, group, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(padded.reshape(-1, kv, group * longest, dim), k.transpose(2, 3)) / math.sqrt(dim)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    position = (positions[:, None] + token)[:, :, None]
    visible = key <= position
    if case["window"]:
        visible &= (key > position - case["window"]) | (key < case["first"])
    scores = scores.view(-1, kv, group, longest, keys).masked_fill_(~visible[:, None, None], -math.inf)
    largest = scores.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(kv, group, 1, 1)
        largest = torch.maximum(largest, sink)
    weights = torch.exp(scores - largest)
    total = weights.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sink - largest)
    out = torch.matmul(weights.view(-1, kv, group * longest, keys), v).view(-1, kv, group, longest, dim) / total
    sequence, token, _, _ = _rows(state, q.shape[0])
    state["out"].copy_(out.permute(0, 3, 1, 2, 4)[sequence, token].reshape(q.shape))
    return state["out"]


# ---- what an operator cannot do without ---------------------------------------------


def _seen(case):
    """Keys that some token of a sequence sees, and pairs of a token and a key it sees, over the batch."""
    keys = pairs = 0
    for n, count in zip(*_lengths(case)):
        window, first = case["window"] or count, case["first"] if case["window"] else 0
        lowest = max(0, count - n + 1 - window)
        keys += count - lowest + min(first, lowest)
        for position in range(count - n, count):
            low = max(0, position + 1 - window)
            pairs += position + 1 - low + min(first, low)
    return keys, pairs


def work(case):
    size = 4 if case["type"] == F32 else 2
    new, _ = _lengths(case)
    if case["op"] in ("write", "read"):
        values = 2 * sum(new) * case["kv"] * case["dim"]
        scales = 2 * sum(new) * case["kv"] * 4
        once = values * (size + 1) + scales
        return dict(bytes=once * (2 if case["op"] == "write" else 1), flops=values)
    keys, pairs = _seen(case)
    held = 2 * keys * case["kv"] * (case["dim"] + 4 if case["cache"] == "i8" else 2 * case["dim"])
    return dict(bytes=held + 2 * sum(new) * case["q"] * case["dim"] * size, flops=4 * pairs * case["q"] * case["dim"])


# ---- the definition, in 64 bits -------------------------------------------------------


def exact(case, seed):
    """One position, one key head at a time, over the positions that it sees."""
    state = prepare(case, seed)
    tables, page_size = state["tables"].tolist(), case["page"]
    new, counts = _lengths(case)
    start, parts_k, parts_v, outs = 0, [], [], []
    for z, (n, count) in enumerate(zip(new, counts)):
        at = torch.arange(count)
        page = torch.tensor(tables[z])[at // page_size].cuda()
        place = (at % page_size).cuda()
        if case["op"] == "write":
            for name, parts in (("k", parts_k), ("v", parts_v)):
                x = state[name][start:start + n].double()
                step = (x.float().abs().max(dim=2, keepdim=True).values.double() / 127).float().double()
                near = torch.round(x / step)
                parts.append(torch.where(step > 0, near * step, torch.zeros_like(x)))
        else:
            if "keys8" in state:
                k = state["keys8"][page, place].double() * state["key_scales"][page, :, place].double().unsqueeze(2)
                v = state["values8"][page, :, :, place].double() * state["value_scales"][page, :, place].double().unsqueeze(2)
            else:
                k, v = state["keys16"][page, place].double(), state["values16"][page, :, :, place].double()
            if case["op"] == "read":
                parts_k.append(k)
                parts_v.append(v)
            else:
                outs.append(_exact_sequence(case, state, start, n, count, k, v))
        start += n
    if case["op"] in ("write", "read"):
        return torch.cat(parts_k), torch.cat(parts_v)
    return torch.cat(outs)


def _exact_sequence(case, state, start, n, count, k, v):
    group = case["q"] // case["kv"]
    out = torch.zeros(n, case["q"], case["dim"], dtype=torch.float64, device="cuda")
    key = torch.arange(count, device="cuda")[None, :]
    position = torch.arange(count - n, count, device="cuda")[:, None]
    hidden = key > position
    if case["window"]:
        hidden |= (position - key >= case["window"]) & (key >= case["first"])
    for head in range(case["q"]):
        q = state["q"][start:start + n, head].double()
        score = (q @ k[:, head // group].T) * case["dim"] ** -0.5
        if case["softcap"]:
            score = case["softcap"] * torch.tanh(score / case["softcap"])
        score[hidden] = -math.inf
        if state["sinks"] is not None:
            sink = state["sinks"][head].double().expand(n, 1)
            share = torch.softmax(torch.cat((score, sink), 1), 1)[:, :count]
        else:
            share = torch.softmax(score, 1)
        out[:, head] = share @ v[:, head // group]
    return out
