"""Operators of a serving loop on a 4-bit paged cache, as measured cases.

Four kinds of call, each through the package's public entry points when ``own`` is true and in elementary torch operations
otherwise:

* ``prompt``: ``prompt_attention``, the causal attention of whole prompts of different lengths that lie one behind the
  other in packed tensors;
* ``store``: ``PagedInt4Cache.write`` of the tokens of a step (whole prompts, or one token of every sequence), and
  ``read`` of what the cache now holds for them;
* ``attend``: ``PagedInt4Cache.attend``, one query token of every sequence against its pages;
* ``copy``: ``PagedInt4Cache.copy_pages``, the copies behind forking sequences and compacting the pool.

Heads are 128 wide.  The cache keeps a token's vector of one head as codes of 4 bits in two groups of 64 coordinates, each
with a scale and an offset in the model's type: offset = min, scale = (max - min) / 15 rounded to the type, code =
round((x - offset) / scale) to the nearest, ties to even, at most 15; a group whose scale is 0 has codes 0.  Its value is
offset + scale * code.  Sizes are those of this repository's benchmark and tests (32 query / 8 KV heads, contexts around
8192, batch 1 to 32) and odd ones around them.
"""

from __future__ import annotations

import math

import torch

own = False  # False: plain form; True: the package's operators

_PAGE = 64          # tokens of a page
_GROUP = 64         # coordinates that share a scale
_SIDE_BYTES = 72    # of a token and head: 64 of codes, two scales, two offsets
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

_MOST_PROMPT = 32 * 8192 * 8193 // 2      # (query head, query, key) triples of the largest listed prompt case
_MOST_STORE = 8 * 8 * 4000                # (token, KV head) pairs of the largest listed store case
_MOST_ATTEND = 32 * 8 * 8128              # (token, KV head) pairs of the largest listed attend case
_MOST_COPY = 32 * 8 * 192                 # (layer, KV head, page) triples of the largest listed copy case


def listed():
    return [
        # -- attention over prompts -----------------------------------------------------------------------------------
        # a few short chat turns, one of them a single token, that arrive together
        _prompt("prompt 5 short fp16", [1, 17, 128, 300, 64]),
        # an ordinary packed batch of documents, every length odd, eight query heads per KV head
        _prompt("prompt 7 ragged bf16 r8", [1333, 257, 2049, 640, 91, 1801, 777], kv_heads=4, ratio=8, kind="bf16"),
        # one long prompt: the benchmark's context
        _prompt("prompt 1x8192 fp16", [8192]),
        # -- the cache takes tokens -----------------------------------------------------------------------------------
        # a decode step of a batch: one token each, somewhere inside a page
        _store("store step b32 fp16", [1] * 32, list(range(100, 100 + 32 * 37, 37))),
        # prompts of different lengths go into fresh pages
        _store("store 6 prompts bf16", [1200, 333, 64, 1, 2047, 901], [0] * 6, kind="bf16"),
        # a batch of prompts, on contexts that they continue
        _store("store 8x4000 fp16", [4000] * 8, [0, 5, 64, 100, 0, 31, 0, 63]),
        # -- one token against the pages ------------------------------------------------------------------------------
        # the smallest call: one user, a short conversation
        _attend("attend b1 t300 fp16", [300]),
        # one user at 8K
        _attend("attend b1 t8128 fp16", [8128]),
        # a ragged batch, eight query heads per KV head, one sequence just begun
        _attend("attend b9 ragged bf16 r8", [4870, 77, 1, 9001, 640, 2999, 130, 6016, 63], ratio=8, kind="bf16"),
        # the benchmark's batch at 8K
        _attend("attend b32 t8128 fp16", [8128] * 32),
        # -- pages ----------------------------------------------------------------------------------------------------
        # four samples of one prompt: a partly filled page each, all layers of the benchmark's model
        _copy("copy 4 pages x 32 layers", 32, 8, 64, 4),
        # the pool is compacted after a busy hour
        _copy("copy 192 pages x 32 layers", 32, 8, 512, 192),
    ]


def _text(numbers):
    return " ".join(str(n) for n in numbers)


def _numbers(text):
    return [int(w) for w in text.split()]


def _prompt(name, lengths, *, kv_heads=8, ratio=4, kind="fp16"):
    return dict(name=name, op="prompt", lengths=_text(lengths), kv_heads=kv_heads, ratio=ratio, kind=kind)


def _store(name, counts, starts, *, kv_heads=8, kind="fp16"):
    return dict(name=name, op="store", counts=_text(counts), starts=_text(starts), kv_heads=kv_heads, kind=kind)


def _attend(name, lengths, *, kv_heads=8, ratio=4, kind="fp16"):
    return dict(name=name, op="attend", lengths=_text(lengths), kv_heads=kv_heads, ratio=ratio, kind=kind)


def _copy(name, layers, kv_heads, pages, copies):
    return dict(name=name, op="copy", layers=layers, kv_heads=kv_heads, pages=pages, copies=copies)


def _between(rng, low, high):
    """A whole number, spread evenly over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "store", "attend", "attend", "copy"))
    kv_heads, ratio, kind = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 7, 8)), rng.choice(tuple(_TYPES))
    if op == "prompt":
        lengths = [_between(rng, 1, 6000) for _ in range(_between(rng, 1, 12))]
        while kv_heads * ratio * sum(t * (t + 1) // 2 for t in lengths) > _MOST_PROMPT:
            lengths = [max(1, t * 3 // 4) for t in lengths]
        case = _prompt("", lengths, kv_heads=kv_heads, ratio=ratio, kind=kind)
    elif op == "store":
        step = rng.random() < 0.5
        n = _between(rng, 1, 64) if step else _between(rng, 1, 10)
        counts = [1 if step else _between(rng, 1, 5000) for _ in range(n)]
        while kv_heads * sum(counts) > _MOST_STORE:
            counts = [max(1, t * 3 // 4) for t in counts]
        case = _store("", counts, [rng.choice((0, _between(rng, 1, 3000))) for _ in counts], kv_heads=kv_heads, kind=kind)
    elif op == "attend":
        lengths = [_between(rng, 1, 20000) for _ in range(_between(rng, 1, 40))]
        while kv_heads * sum(lengths) > _MOST_ATTEND:
            lengths = [max(1, t * 3 // 4) for t in lengths]
        case = _attend("", lengths, kv_heads=kv_heads, ratio=ratio, kind=kind)
    else:
        layers, copies = _between(rng, 1, 32), _between(rng, 1, 192)
        case = _copy("", layers, kv_heads, 2 * copies + _between(rng, 1, 128), copies)
    del case["name"]
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _normal(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _vectors(seed, tokens, heads, dtype, outliers):
    """[tokens, heads, 128]; ``outliers``: as keys have them, a few channels of every head are several times larger and off
    centre."""
    x = _normal(seed, tokens, heads, 128)
    if outliers:
        channel = _normal(seed + 1, heads, 128)
        x = x * torch.where(channel > 1.6, 4.0, 1.0) + channel
    return x.to(dtype)


def _prompt_inputs(case, seed):
    """Views of one projection's output [tokens, (query heads + 2 KV heads) * 128], as a model has them."""
    h, r, lengths, dtype = case["kv_heads"], case["ratio"], _numbers(case["lengths"]), _TYPES[case["kind"]]
    total = sum(lengths)
    fused = _normal(seed, total, h * (r + 2), 128)
    fused[:, :h * r] *= 1.5
    fused = fused.to(dtype)
    return fused[:, :h * r], fused[:, h * r:h * (r + 1)], fused[:, h * (r + 1):], lengths


def _cached_inputs(case, seed):
    lengths, dtype = _numbers(case["lengths"]), _TYPES[case["kind"]]
    total, h = sum(lengths), case["kv_heads"]
    k = _vectors(seed * 10 + 1, total, h, dtype, True)
    v = _vectors(seed * 10 + 5, total, h, dtype, False)
    q = _normal(seed * 10 + 7, len(lengths), h * case["ratio"], 128).to(dtype)
    return q, k, v, lengths


def _store_inputs(case, seed):
    counts, dtype = _numbers(case["counts"]), _TYPES[case["kind"]]
    total, h = sum(counts), case["kv_heads"]
    return (_vectors(seed * 10 + 1, total, h, dtype, True), _vectors(seed * 10 + 5, total, h, dtype, False), counts,
            _numbers(case["starts"]))


def _copy_inputs(case, seed):
    """Bytes of a pool [layers, pages, bytes of a page] and two disjoint lists of page numbers."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (case["layers"], case["pages"], case["kv_heads"] * _PAGE * 2 * _SIDE_BYTES)
    words = torch.randint(-2**62, 2**62, (*shape[:2], shape[2] // 8), generator=g, device="cuda")
    order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed)).tolist()
    return words.view(torch.uint8), order[:case["copies"]], order[case["copies"]:2 * case["copies"]]


def _ends(lengths):
    out = [0]
    for t in lengths:
        out.append(out[-1] + t)
    return out


def prepare(case, seed):
    op = case["op"]
    if op == "prompt":
        q, k, v, lengths = _prompt_inputs(case, seed)
        ends = _ends(lengths)
        return dict(op=op, q=q, k=k, v=v, ends=ends, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device="cuda"))
    if op == "copy":
        pool, src, dst = _copy_inputs(case, seed)
        state = dict(op=op, src=src, dst=dst)
        if own:
            cache = _cache(case["layers"], case["kv_heads"], case["pages"], torch.float16)
            cache.pages.view(pool.shape).copy_(pool)
            return dict(state, cache=cache)
        return dict(state, pool=pool, src_index=torch.tensor(src, device="cuda"), dst_index=torch.tensor(dst, device="cuda"))
    if op == "store":
        k, v, counts, starts = _store_inputs(case, seed)
        state = dict(op=op, k=k, v=v)
        if own:
            cache = _cache(1, case["kv_heads"], _pages([c + s for c, s in zip(counts, starts)]), k.dtype)
            sequences = cache.add(len(counts))
            cache.extend(sequences, starts)
            return dict(state, cache=cache, step=cache.extend(sequences, counts))
        return state
    q, k, v, lengths = _cached_inputs(case, seed)
    state = dict(op=op, q=q)
    if own:
        cache = _cache(1, case["kv_heads"], _pages(lengths), k.dtype)
        step = cache.extend(cache.add(len(lengths)), lengths)
        cache.write(0, step, k, v)
        return dict(state, cache=cache, step=step)
    return dict(state, ends=_ends(lengths), k=_codes(k), v=_codes(v))


def _cache(layers, kv_heads, pages, dtype):
    from reskv_b200 import PagedInt4Cache

    return PagedInt4Cache(layers, kv_heads, pages, dtype=dtype, device="cuda")


def _pages(lengths):
    return sum(-(-t // _PAGE) for t in lengths)


# ---- the plain form -------------------------------------------------------------------------------------------------------
def _codes(x):
    """(codes, scale, offset) of [tokens, heads, 128] as [tokens, heads, 2, 64] and [tokens, heads, 2, 1]."""
    g = x.unflatten(-1, (2, _GROUP)).float()
    low = g.amin(-1, keepdim=True)
    scale = ((g.amax(-1, keepdim=True) - low) / 15).to(x.dtype).float()
    code = torch.where(scale > 0, ((g - low) / torch.where(scale > 0, scale, 1.0)).round().clamp(0, 15), 0.0)
    return code.to(torch.uint8), scale, low


def _values(codes, part=slice(None)):
    code, scale, low = codes
    return (low[part] + scale[part] * code[part].float()).flatten(-2)


def _attention(q, k, v, causal):
    """q [queries, heads, 128], k and v [keys, KV heads, 128], FP32 -> [queries, heads, 128]."""
    n, heads, _ = q.shape
    t, h, _ = k.shape
    out = torch.empty_like(q)
    for i in range(h):  # a KV head at a time: the scores of one fit
        part = slice(i * (heads // h), (i + 1) * (heads // h))
        s = torch.matmul(q[:, part].transpose(0, 1), k[:, i].t()) * 128**-0.5  # [group, queries, keys]
        if causal:
            s = s.masked_fill(torch.ones(n, t, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[:, part] = (torch.matmul(p, v[:, i]) / p.sum(-1, keepdim=True)).transpose(0, 1)
    return out


def _plain(state):
    if state["op"] == "prompt":
        q, k, v = state["q"], state["k"], state["v"]
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        for a, b in zip(state["ends"], state["ends"][1:]):
            out[a:b] = _attention(q[a:b].float(), k[a:b].float(), v[a:b].float(), True).to(q.dtype)
        return out
    if state["op"] == "store":
        return [_values(_codes(x)).to(x.dtype) for x in (state["k"], state["v"])]
    if state["op"] == "attend":
        q = state["q"]
        out = torch.empty_like(q)
        for i, (a, b) in enumerate(zip(state["ends"], state["ends"][1:])):
            k, v = _values(state["k"], slice(a, b)), _values(state["v"], slice(a, b))
            out[i] = _attention(q[i:i + 1].float(), k, v, False)[0].to(q.dtype)
        return out
    state["pool"][:, state["dst_index"]] = state["pool"][:, state["src_index"]]
    return state["pool"]


# ---- a pass ---------------------------------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    if state["op"] == "prompt":
        from reskv_b200 import prompt_attention

        return prompt_attention(state["q"], state["k"], state["v"], state["cu_seqlens"])
    cache = state["cache"]
    if state["op"] == "store":
        cache.write(0, state["step"], state["k"], state["v"])
        return list(cache.read(0, state["step"]))
    if state["op"] == "attend":
        return cache.attend(0, state["step"], state["q"])
    cache.copy_pages(state["src"], state["dst"])
    return cache.pages.view(cache.layers, cache.capacity, -1)


def work(case):
    if case["op"] == "prompt":
        lengths, heads = _numbers(case["lengths"]), case["kv_heads"] * case["ratio"]
        return {"bytes": sum(lengths) * (2 * heads + 2 * case["kv_heads"]) * 256,
                "flops": 4 * 128 * heads * sum(t * (t + 1) // 2 for t in lengths)}
    if case["op"] == "store":  # the tokens, their place in the cache, and the values read back
        rows = sum(_numbers(case["counts"])) * case["kv_heads"]
        return {"bytes": rows * 2 * (256 + _SIDE_BYTES + 256), "flops": rows * 2 * 128 * 8}
    if case["op"] == "attend":
        lengths, heads = _numbers(case["lengths"]), case["kv_heads"] * case["ratio"]
        return {"bytes": sum(lengths) * case["kv_heads"] * 2 * _SIDE_BYTES + len(lengths) * heads * 512,
                "flops": 4 * 128 * heads * sum(lengths)}
    moved = case["layers"] * case["copies"] * case["kv_heads"] * _PAGE * 2 * _SIDE_BYTES
    return {"bytes": 2 * moved, "flops": 0}


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------------
def _exact_value(x):
    """What the cache holds for x, in 64 bits: the scale is rounded to the type of x, as stored."""
    y = x.double().reshape(*x.shape[:-1], 128 // _GROUP, _GROUP)
    least, most = y.min(dim=-1, keepdim=True)[0], y.max(dim=-1, keepdim=True)[0]
    step = ((most - least) / 15).to(x.dtype).double()
    number = torch.round((y - least) / step.masked_fill(step == 0, math.inf)).clamp(max=15)
    return (least + number * step).reshape(x.shape)


def _exact_softmax_rows(q, k, v, first):
    """q [rows, 128], k and v [keys, 128], 64 bits; row i sees the keys up to first + i, or all where first is None."""
    weights = (q @ k.mT) / math.sqrt(128.0)
    if first is not None:
        seen = torch.arange(k.shape[0], device=q.device)[None, :] <= first + torch.arange(q.shape[0], device=q.device)[:, None]
        weights = torch.where(seen, weights, -math.inf)
    return torch.softmax(weights, dim=1) @ v


def exact(case, seed):
    if case["op"] == "copy":
        return None
    if case["op"] == "store":
        k, v, _, _ = _store_inputs(case, seed)
        return [_exact_value(k), _exact_value(v)]
    ratio = case["ratio"]
    if case["op"] == "prompt":
        q, k, v, lengths = _prompt_inputs(case, seed)
        out, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
        for t in lengths:
            for head in range(q.shape[1]):
                kk, vv = k[at:at + t, head // ratio].double(), v[at:at + t, head // ratio].double()
                for i in range(0, t, 2048):
                    j = min(t, i + 2048)
                    out[at + i:at + j, head] = _exact_softmax_rows(q[at + i:at + j, head].double(), kk[:j], vv[:j], i)
            at += t
        return out
    q, k, v, lengths = _cached_inputs(case, seed)
    out, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
    for n, t in enumerate(lengths):
        kk, vv = _exact_value(k[at:at + t]), _exact_value(v[at:at + t])
        for head in range(kk.shape[1]):
            rows = slice(head * ratio, (head + 1) * ratio)
            out[n, rows] = _exact_softmax_rows(q[n, rows].double(), kk[:, head], vv[:, head], None)
        at += t
    return out
