"""``ResKVLlama(cache="int4")``: prompts of different lengths in one batch, the 4-bit paged cache, rows that fork and go."""

import pytest
import torch

TINY = dict(hidden=256, layers=2, heads=8, kv_heads=2, ffn=512, vocab=320)
# logits of the FP16 model against an FP32 one: the bound that the other model tests use for a reordered FP16 sum
CLOSE = dict(atol=3e-2, rtol=3e-2)


def make(seed=5, **kw):
    from reskv_b200.models import LlamaShape, ResKVLlama

    return ResKVLlama(LlamaShape(**TINY), cache="int4", seed=seed, **kw)


def prompts(*lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 320, (t,), generator=g).cuda() for t in lengths]


def plain(model, ids, row=None):
    """Logits behind ``ids`` in FP32: of a prompt, or (``row``) of that row's newest token against what its cache holds.  (A key that
    FP32 and FP16 round to different codes would move the logits by far more than rounding does; what the cache holds is tested
    where it is written.)"""
    m, s = model, model.shape
    step = None if row is None else m.paged.extend([m.sequences[row]], 0)
    past = 0 if row is None else step.lengths[0] - 1
    ang = torch.arange(past, past + len(ids), device="cuda").float()[:, None] * m.inv_freq
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def norm(x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + s.rms_eps) * w.float()

    def rope(x):
        a, b = x[..., :64], x[..., 64:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    x = m.embed[ids].float()
    for i, layer in enumerate(m.layers):
        q, k, v = (norm(x, layer["norm1"]) @ layer["wqkv"].float().T).split((m.h_q * 128, m.h_kv * 128, m.h_kv * 128), -1)
        q, k, v = rope(q.unflatten(-1, (-1, 128))), rope(k.unflatten(-1, (-1, 128))), v.unflatten(-1, (-1, 128))
        if row is not None:
            k, v = (y.float() for y in m.paged.read(i, step, everything=True))
        k, v = (y.repeat_interleave(m.h_q // m.h_kv, 1) for y in (k, v))
        w = torch.einsum("ihd,jhd->hij", q, k) * 128**-0.5
        if row is None:
            w = w.masked_fill(torch.ones(len(ids), len(ids), device="cuda").triu(1).bool(), -torch.inf)
        x = x + torch.einsum("hij,jhd->ihd", w.softmax(-1), v).flatten(1) @ layer["wo"].float().T
        gate, up = (norm(x, layer["norm2"]) @ layer["w_gate_up"].float().T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ layer["w_down"].float().T
    return norm(x[-1], m.final_norm) @ m.lm_head.float().T


def plain_rows(model, tokens):
    return torch.stack([plain(model, t[None], row) for row, t in enumerate(tokens)])


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [65536, 100])
def test_ragged_prompts_and_steps_against_fp32(chunk):
    model, ids = make(prefill_chunk=chunk), prompts(70, 1, 130, 64)
    logits = model.prefill(ids, reserve=8)
    torch.testing.assert_close(logits, torch.stack([plain(model, x) for x in ids]), **CLOSE)
    for step in range(6):
        tok = logits.argmax(-1)
        logits = model.decode(tok)
        torch.testing.assert_close(logits, plain_rows(model, tok), **CLOSE)
    model.paged.check()
    assert [model.paged.length(s) for s in model.sequences] == [76, 7, 136, 70]


@pytest.mark.gpu
def test_equal_lengths_as_a_tensor_are_the_same_batch():
    ids = torch.stack(prompts(40, 40))
    a, b = make(), make()
    assert torch.equal(a.prefill(ids, reserve=4), b.prefill(list(ids), reserve=4))
    assert make().generate(ids, 5).shape == (2, 5) and make().generate(prompts(3, 90), 5).shape == (2, 5)


@pytest.mark.gpu
def test_graph_decode_matches_eager_decode():
    """One capture serves all steps, over page boundaries; a table that becomes too narrow brings another one."""
    eager, graph = make(), make()
    ids = prompts(60, 7)
    tok = eager.prefill(ids, reserve=80).argmax(-1)
    assert torch.equal(tok, graph.prefill(ids, reserve=80).argmax(-1))
    graph.begin_graph_decode(2)
    for step in range(80):
        le, lg = eager.decode(tok), graph.decode_graph(tok).clone()
        torch.testing.assert_close(lg, le, atol=2e-2, rtol=2e-2)
        tok = le.argmax(-1)
        if step == 0:
            captured = graph._graph
    assert graph._graph is captured, "the step was captured again"
    graph._raise_on_status()


@pytest.mark.gpu
def test_tables_grow_under_graph_decode():
    eager, graph = make(pages=20), make(pages=20)
    ids = prompts(10, 30)
    tok = eager.prefill(ids).argmax(-1)
    graph.prefill(ids)
    graph.begin_graph_decode(2)
    for _ in range(150):  # past the width that the first table has
        le, lg = eager.decode(tok), graph.decode_graph(tok).clone()
        torch.testing.assert_close(lg, le, atol=2e-2, rtol=2e-2)
        tok = le.argmax(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_select_forks_drops_and_reorders(graph):
    model, ids = make(pages=30), prompts(70, 20, 64)
    model.prefill(ids)
    if graph:
        model.begin_graph_decode(3)
    decode = model.decode_graph if graph else model.decode
    decode(torch.tensor([1, 2, 3], device="cuda"))
    before = [model.paged.read(1, model.paged.extend([s], 0), everything=True)[0] for s in model.sequences]
    model.select([2, 0, 0, 2])
    assert len(set(model.sequences)) == 4 and len(model.paged._book.sequences) == 4
    for s, was in zip(model.sequences, (2, 0, 0, 2)):
        assert torch.equal(model.paged.read(1, model.paged.extend([s], 0), everything=True)[0], before[was])
    if graph:
        model.begin_graph_decode(4)
    for turn in range(3):
        tok = torch.tensor([5, 6, 7, 8], device="cuda") + turn
        got = decode(tok).clone()
        torch.testing.assert_close(got, plain_rows(model, tok), **CLOSE)
    assert not torch.equal(got[1], got[2])  # the two samples of row 0 went their own ways
    model.select([1])
    assert model.paged.compact() == 2  # 74 tokens
    torch.testing.assert_close(decode(tok[:1]), plain_rows(model, tok[:1]), **CLOSE)
    model.select([])
    assert model.paged.free_pages == 30


@pytest.mark.gpu
def test_refusals():
    model = make(pages=3)
    for bad in ([], [torch.zeros(0, dtype=torch.long, device="cuda")], [torch.zeros((2, 2), dtype=torch.long, device="cuda")]):
        with pytest.raises(ValueError):
            model.prefill(bad)
    with pytest.raises(ValueError):
        model.prefill(prompts(4), reserve=-1)
    with pytest.raises(RuntimeError, match="out of pages"):
        model.prefill(prompts(65, 65))
    model.prefill(prompts(5, 6))
    with pytest.raises(ValueError):
        model.decode(torch.zeros(3, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        model.begin_graph_decode(3)
    for rows in ([2], [-1], [0.0]):
        with pytest.raises(ValueError):
            model.select(rows)


@pytest.mark.gpu
def test_a_reused_step_keeps_its_tensors():
    from reskv_b200 import PagedInt4Cache

    cache = PagedInt4Cache(1, 1, 8)
    seqs = cache.add(2)
    first = cache.extend(seqs, 1, width=3)
    assert first.table.shape == (2, 3)
    second = cache.extend(seqs, [64, 2], reuse=first)
    torch.cuda.synchronize()
    assert second.table.data_ptr() == first.table.data_ptr() and second.cu_seqlens.tolist() == [0, 64, 66]
    assert second.starts.tolist() == [1, 1] and second.device_lengths.tolist() == [65, 3]
    assert second.table.tolist() == [[0, 2, 0], [1, 0, 0]]
    with pytest.raises(ValueError):
        cache.attend(0, first, torch.zeros(2, 1, 128, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError, match="do not fit"):
        cache.extend(seqs, [200, 0], reuse=second)
    assert cache.length(seqs[0]) == 65 and cache.free_pages == 5
    for bad in (dict(reuse=0), dict(width=-1), dict(width=1.5)):
        with pytest.raises(ValueError):
            cache.extend(seqs, 0, **bad)
    with pytest.raises(ValueError):
        cache.extend(seqs[:1], 0, reuse=second)


def test_constructor_checks():
    from reskv_b200.models import LlamaShape, ResKVLlama

    for kw in (dict(cache="dense", pages=4), dict(cache="int4", pages=0), dict(cache="int4", pages=2.0)):
        with pytest.raises(ValueError, match="pages"):
            ResKVLlama(LlamaShape(**TINY), device="cpu", **kw)
    with pytest.raises(RuntimeError, match="select"):
        ResKVLlama(LlamaShape(**TINY), cache="dense", device="cpu").select([0])


@pytest.mark.gpu
def test_reused_tables_belong_to_the_last_step_of_this_cache():
    from reskv_b200 import PagedInt4Cache

    cache, other = (PagedInt4Cache(1, 1, 16) for _ in range(2))
    a, b = cache.add(2), cache.add(2)
    first = cache.extend(a, [3, 4])
    second = cache.extend(a, [1, 1], reuse=first)
    third = cache.extend(b, [2, 2], reuse=first)  # other sequences, over the same tensors
    x = torch.ones(2, 1, 128, dtype=torch.float16, device="cuda")
    for stale in (first, second):
        with pytest.raises(ValueError, match="the step belongs"):
            cache.write(0, stale, x, x)
        with pytest.raises(ValueError, match="the step belongs"):
            cache.attend(0, stale, x)
    assert third.table.data_ptr() == first.table.data_ptr()
    k = torch.ones(4, 1, 128, dtype=torch.float16, device="cuda")
    cache.write(0, third, k, k)
    assert torch.equal(cache.attend(0, third, x), x)
    with pytest.raises(ValueError, match="reuse must be a step of this cache"):
        other.extend(other.add(2), 1, reuse=third)
    cache.attend(0, third, x)  # and nothing changed
    cache.check()


@pytest.mark.gpu
def test_a_prompt_whose_wait_ran_out_raises(monkeypatch):
    """The word is set by the host, no wait runs out here: what the attention of a prompt reports is the cache's to tell, and the model
    asks for it."""
    import reskv_b200.models.llama as llama

    model, real = make(), llama.prompt_attention
    assert model.prefill(prompts(5, 6)).isfinite().all()

    def lost(*args, status=None, **kw):
        out = real(*args, status=status, **kw)
        if status is not None:
            status.fill_(1)
        return out

    monkeypatch.setattr(llama, "prompt_attention", lost)
    with pytest.raises(RuntimeError, match="device status"):
        model.prefill(prompts(5, 6))


@pytest.mark.gpu
def test_a_prompt_that_fails_leaves_no_batch():
    """Two slices of prompts, of which the second finds no pages: nothing may attend to the tokens that were never written."""
    model = make(pages=3, prefill_chunk=100)
    model.prefill(prompts(5, 6))
    with pytest.raises(RuntimeError, match="out of pages"):
        model.prefill(prompts(65, 65))
    for call in (lambda: model.decode(torch.zeros(2, dtype=torch.long, device="cuda")), lambda: model.select([0]),
                 lambda: model.begin_graph_decode(2)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    assert model.sequences == [] and model.cache_bytes() == 0
    ids = prompts(64, 65)
    assert torch.equal(model.prefill(ids), make().prefill(ids))
    model.layers[1] = None  # a layer that fails in the middle of a prompt
    with pytest.raises(TypeError):
        model.prefill(ids)
    with pytest.raises((RuntimeError, ValueError)):
        model.decode(torch.zeros(2, dtype=torch.long, device="cuda"))


@pytest.mark.gpu
def test_bad_prompts_leave_the_batch_as_it_is():
    model, ids = make(), prompts(5, 6)
    logits = model.prefill(ids, reserve=4)
    for bad in ([], [torch.zeros(0, dtype=torch.long, device="cuda")], [3]):
        with pytest.raises((ValueError, TypeError)):
            model.prefill(bad)
    with pytest.raises(ValueError):
        model.prefill(ids, reserve=1.5)
    assert model.decode(logits.argmax(-1)).isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_a_step_that_fails_does_not_count(graph):
    """Some layers have written the token, others not: nobody attends to it, and the step can be made again."""
    model, other, ids = make(pages=8), make(pages=8), prompts(64, 6)
    tok = model.prefill(ids).argmax(-1)
    other.prefill(ids)
    if graph:
        model.begin_graph_decode(2), other.begin_graph_decode(2)
    step, want = (model.decode_graph, other.decode_graph) if graph else (model.decode, other.decode)
    layer, model.layers[1] = model.layers[1], None
    with pytest.raises(TypeError):
        step(tok)
    model.layers[1] = layer
    assert [model.paged.length(s) for s in model.sequences] == [64, 6] and model.paged.free_pages == 6
    for _ in range(3):
        assert torch.equal(step(tok), want(tok))
    with pytest.raises(ValueError):
        step(tok[:1])
    assert [model.paged.length(s) for s in model.sequences] == [67, 9]


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_a_beam_replaces_another_in_a_full_pool(graph):
    """The pool that a prompt brings has room for its rows and no more: the dropped row's pages serve the forked one."""
    model, ids = make(), prompts(70, 80)
    tok = model.prefill(ids, reserve=2).argmax(-1)
    assert model.paged.free_pages == 0
    if graph:
        model.begin_graph_decode(2)
    decode = model.decode_graph if graph else model.decode
    decode(tok)
    before = model.paged.read(1, model.paged.extend([model.sequences[1]], 0), everything=True)
    with pytest.raises(RuntimeError, match="out of pages"):
        model.select([0, 1, 1])
    model.select([1, 1])
    for s in model.sequences:
        got = model.paged.read(1, model.paged.extend([s], 0), everything=True)
        assert torch.equal(got[0], before[0]) and torch.equal(got[1], before[1])
    tok = torch.tensor([5, 6], device="cuda")
    torch.testing.assert_close(decode(tok).clone(), plain_rows(model, tok), **CLOSE)


@pytest.mark.gpu
def test_a_batch_without_rows():
    """select([]) ends all rows; there is nothing to decode then, said in words, until the next prompt."""
    model, ids = make(pages=8), prompts(5, 6)
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    for call in (lambda: model.decode(none), lambda: model.begin_graph_decode(0)):
        with pytest.raises((RuntimeError, ValueError), match="prefill"):
            call()
    model.prefill(ids)
    with pytest.raises(RuntimeError, match="begin_graph_decode"):
        model.decode_graph(torch.tensor([1, 2], device="cuda"))
    assert [model.paged.length(s) for s in model.sequences] == [5, 6]
    model.begin_graph_decode(2)
    model.decode_graph(torch.tensor([1, 2], device="cuda"))
    model.select([])
    assert model.paged.free_pages == 8
    for call in (lambda: model.decode(none), lambda: model.decode_graph(none), lambda: model.begin_graph_decode(0)):
        with pytest.raises(ValueError, match="no rows"):
            call()
    assert model.generate(ids, 3).shape == (2, 3)


def test_more_query_heads_than_the_cache_takes_are_refused_at_the_start():
    """The prompt's attention takes more, so that the first token behind a prompt would have been the first refusal."""
    from reskv_b200.models import LlamaShape, ResKVLlama

    with pytest.raises(ValueError, match="8 query heads per KV head"):
        ResKVLlama(LlamaShape(**TINY | dict(heads=9, kv_heads=1)), cache="int4", device="cpu")
    for heads in (8, 16):
        ResKVLlama(LlamaShape(**TINY | dict(heads=heads)), cache="int4", device="cpu")
    ResKVLlama(LlamaShape(**TINY | dict(heads=9, kv_heads=1)), cache="dense", device="cpu")
