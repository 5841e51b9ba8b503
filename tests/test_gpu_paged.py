"""``PagedInt4Cache``: what it stores, and attention over it, against their definitions."""

import numpy as np
import pytest
import torch

from reskv_b200 import PagedInt4Cache, prompt_attention

DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def stored(x):
    """(value, scale, offset, code) per group of 64, FP32 from the definition: the quotient is rounded to FP32, then to the
    nearest whole number."""
    g = x.float().cpu().unflatten(-1, (2, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = torch.from_numpy((high - low).numpy() / np.float32(15)).to(x.dtype).float()
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.rint((g - low).numpy() / scale.numpy())
    code = torch.from_numpy(np.where(scale.numpy() > 0, np.minimum(code, 15), 0).astype(np.float32))
    return low + scale * code, scale, low, code


def values_of(x):
    return stored(x)[0].flatten(-2).to(x.dtype).to(x.device)


def vectors(tokens, heads, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(tokens, heads, 128, generator=g, device=DEV)
    return (x * torch.where(torch.rand(heads, 128, generator=g, device=DEV) > 0.95, 5.0, 1.0) + 0.3).to(dtype)


def fill(cache, lengths, seed=0, pieces=1):
    """Sequences of these lengths, written in ``pieces`` steps -> (last step's sequences, keys and values of each)."""
    seqs = cache.add(len(lengths))
    k = [vectors(t, cache.kv_heads, cache.dtype, seed + 2 * i) for i, t in enumerate(lengths)]
    v = [vectors(t, cache.kv_heads, cache.dtype, seed + 2 * i + 1) for i, t in enumerate(lengths)]
    for piece in range(pieces):
        cuts = [(t * piece // pieces, t * (piece + 1) // pieces) for t in lengths]
        step = cache.extend(seqs, [b - a for a, b in cuts])
        for layer in range(cache.layers):
            cache.write(layer, step, *(torch.cat([x[a:b] for x, (a, b) in zip(side, cuts)]) for side in (k, v)))
    return seqs, k, v


def formula(q, k, v, scaling=128**-0.5):
    """(out, lse, bound) in 64 bits for one query row [H, 128] and the stored keys and values of its sequence.

    The weights times their token's scale are rounded to FP16 (half a step: 2^-11) in front of their product with the codes,
    whose absolute sum is S = sum_j p_j (v_j - offset_j); those below FP16's normal numbers are off by 2^-25 where the largest
    scale counts 2^14, so all together by less than 2^-38 T max(v - offset).  The result is rounded once (u).  A score is off by
    at most ds: 128 products and their scaling in FP32, 130 * 2^-23 sum |q| (|offset| + 15 scale); that and 2^-20 for the
    exponential and the sums of T weights (T 2^-24) count twice (numerator, sum) with A = sum_j p_j (|offset_j| + v_j - offset_j)."""
    u = torch.finfo(q.dtype).eps / 2
    heads, ratio = q.shape[0], q.shape[0] // k.shape[1]
    q = q.double()
    (kv, ks, kl, _), (vv, vs, vl, vc) = stored(k), stored(v)
    to = lambda x: x.double().to(DEV)  # noqa: E731
    key, value = to(kv).flatten(-2), to(vv).flatten(-2)
    big = (to(kl).abs() + 15 * to(ks)).expand(-1, -1, 2, 64).flatten(-2)
    above, below = (to(vs) * to(vc)).flatten(-2), to(vl).abs().expand(-1, -1, 2, 64).flatten(-2)
    out, bound, lse = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(heads, dtype=torch.float64, device=DEV)
    t = key.shape[0]
    for h in range(heads):
        g = h // ratio
        s = key[:, g] @ q[h] * scaling
        p = torch.softmax(s, 0)
        lse[h] = torch.logsumexp(s, 0)
        out[h] = p @ value[:, g]
        ds = 130 * 2.0**-23 * scaling * (big[:, g] @ q[h].abs()).max()
        bound[h] = (2.0**-11 * (p @ above[:, g]) + u * out[h].abs() + 2 * (ds + 2.0**-20 + t * 2.0**-24) * (p @ (above + below)[:, g])
                    + 2.0**-38 * t * above[:, g].amax(0) + 2.0**-25)
    return out, lse, bound


def assert_attends(cache, seqs, k, v, ratio, seed=50, layer=0, **kw):
    step = cache.extend(seqs, 0)
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(len(seqs), cache.kv_heads * ratio, 128, generator=g, device=DEV).to(cache.dtype)
    got, lse = cache.attend(layer, step, q, return_lse=True, **kw)
    assert got.dtype == cache.dtype and got.shape == q.shape
    for i in range(len(seqs)):
        if len(k[i]) == 0:
            assert not got[i].any() and (lse[i] == -torch.inf).all()
            continue
        want, want_lse, bound = formula(q[i], k[i], v[i], **kw)
        undefined = want.isnan()  # values beyond the type's range were infinite before they were stored
        assert torch.equal(got[i].isnan(), undefined)
        err, bound = (got[i].double() - want).abs()[~undefined], bound[~undefined]
        assert (err <= bound).all(), f"sequence {i}: off by {err.max():.3e}, {(err - bound).max():.3e} too much"
        assert (lse[i].double() - want_lse).abs().max() < 1e-3
    return got


# ---- storing ------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv_heads", [1, 3, 8])
def test_what_is_written_is_read(dtype, kv_heads):
    lengths = [1, 64, 65, 200, 0, 129]
    cache = PagedInt4Cache(2, kv_heads, 16, dtype=dtype)
    seqs, k, v = fill(cache, lengths, seed=3, pieces=3)
    got = cache.read(1, cache.extend(seqs, 0), everything=True)
    for x, side in zip(got, (k, v)):
        assert x.dtype == dtype and torch.equal(x, torch.cat([values_of(y) for y in side]))
    cache.check()


@pytest.mark.gpu
def test_read_gives_the_tokens_of_the_step():
    cache = PagedInt4Cache(1, 2, 8)
    seqs, k, v = fill(cache, [70, 10], seed=1)
    step = cache.extend(seqs, [3, 60])
    nk, nv = vectors(63, 2, torch.float16, 90), vectors(63, 2, torch.float16, 91)
    cache.write(0, step, nk, nv)
    got = cache.read(0, step)
    assert torch.equal(got[0], values_of(nk)) and torch.equal(got[1], values_of(nv))
    whole = cache.read(0, step, everything=True)[0]
    assert torch.equal(whole, torch.cat([values_of(x) for x in (k[0], nk[:3], k[1], nk[3:])]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_at_the_edges(dtype):
    """Constant rows, the largest and smallest numbers of the type, quotients on a half, signed zeros; NaN and infinities make
    their group of 64 NaN and no other."""
    info = torch.finfo(dtype)
    x = torch.zeros(12, 1, 128)
    x[1] = 3.5
    x[2, 0, :64], x[2, 0, 64:] = info.max / 2, -info.max / 2
    x[2, 0, ::2] *= -0.5
    x[3, 0, 1] = info.smallest_normal * info.eps  # the smallest subnormal
    x[4] = torch.linspace(0, 15, 128)
    x[5, 0, :64] = torch.arange(64) / 4  # with 15.75 as the largest: a scale of 1.05
    x[6, 0, :64] = (torch.arange(64) / 2).clamp(max=15)  # scale 1: halves go to the even code
    x[7, 0, 64:] = -0.0
    x[8, 0, 0] = torch.nan
    x[9, 0, 100] = torch.inf
    x[10, 0, 3] = -torch.inf
    x[11] = torch.randn(128, generator=torch.Generator().manual_seed(0)) * 1e-4
    x = x.to(dtype).to(DEV)
    cache = PagedInt4Cache(1, 1, 1, dtype=dtype)
    step = cache.extend(cache.add(1), 12)
    cache.write(0, step, x, x.flip(0))
    k, v = cache.read(0, step)
    assert torch.equal(k[:8], values_of(x[:8])) and torch.equal(k[11], values_of(x[11:])[0])
    assert torch.equal(v[4:], values_of(x[:8].flip(0))) and torch.equal(v[0], k[11])
    for row, group in ((8, 0), (9, 1), (10, 0)):
        bad, good = (k[row, 0, 64 * i:64 * i + 64] for i in (group, 1 - group))
        assert bad.isnan().all() and not good.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_codes_at_ties_and_at_every_magnitude(dtype):
    """Quotients that are halves, or next to one, and scales from the subnormal numbers to the largest: the codes of the division."""
    info = torch.finfo(dtype)
    g = torch.Generator(device=DEV).manual_seed(3)
    halves = torch.arange(31, device=DEV) / 2  # 0, 0.5, .. 15: with 15 and 0 among them the scale is 1
    rows = []
    for i in range(400):
        x = halves[torch.randint(31, (128,), generator=g, device=DEV)]
        x[[0, 64]], x[[1, 65]] = 0.0, 15.0
        if i % 4 == 1:  # a step of the type beside them
            x = x * (1 + info.eps * (torch.randint(3, (128,), generator=g, device=DEV) - 1))
        elif i % 4 == 2:
            x = torch.rand(128, generator=g, device=DEV) * 15
        elif i % 4 == 3:
            x = x - 7.5
        least, most = (-132, 123) if dtype == torch.bfloat16 else (-24, 11)
        rows.append((x.double() * 2.0 ** (least + i * (most - least) // 399)).to(dtype))
    x = torch.stack(rows)[:, None]
    cache = PagedInt4Cache(1, 1, 8, dtype=dtype)
    step = cache.extend(cache.add(1), [400])
    cache.write(0, step, x, x.flip(0))
    k, v = cache.read(0, step)
    assert torch.equal(k, values_of(x)) and torch.equal(v, values_of(x.flip(0)))


@pytest.mark.gpu
def test_layouts_in_memory():
    """Views of a fused projection, head-major and misaligned tensors are stored alike."""
    cache = PagedInt4Cache(1, 2, 4)
    fused = torch.randn(100, 8, 128, device=DEV).half()
    k, v = fused[:, 4:6], fused[:, 6:]
    step = cache.extend(cache.add(1), 100)

    def after(key, value):
        cache.pages.zero_()
        cache.write(0, step, key, value)
        return cache.pages.clone()

    want = after(k.contiguous(), v.contiguous())
    assert torch.equal(after(k, v), want)
    assert torch.equal(after(k.transpose(0, 1).contiguous().transpose(0, 1), v), want)
    odd = torch.empty(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape).copy_(k)
    assert torch.equal(after(odd, v), want)
    one = k[:, :1].contiguous()
    assert torch.equal(after(one.expand(-1, 2, -1), v), after(one.repeat(1, 2, 1), v))


@pytest.mark.gpu
def test_rows_behind_the_step_and_other_pages_stay():
    cache = PagedInt4Cache(1, 2, 6)
    cache.pages.fill_(17)
    seqs = cache.add(2)
    step = cache.extend(seqs, [5, 70])
    more = vectors(90, 2, torch.float16, 5)
    from reskv_b200._extension import host

    # tensors longer than the step (a padded batch): the tokens behind the last sequence are ignored
    host().paged_write(cache.pages, 0, cache._status, more, more, step.cu_seqlens, step.starts, step.table)
    assert torch.equal(cache.read(0, step)[0], values_of(more[:75]))
    assert (cache.pages[0, 3:] == 17).all()
    assert (cache.pages[0, 0, :, 1:] == 17).all()  # the blocks of the first page behind its five tokens
    k, v = host().paged_read(cache.pages, 0, cache._status, False, step.cu_seqlens, step.starts, step.table, 75)
    assert torch.equal(k, cache.read(0, step)[0])
    cache.check()


# ---- attention ----------------------------------------------------------------------------------------------------------------
LENGTHS = [[1], [15, 16, 17], [63, 64, 65], [128, 0, 129], [300], [1000, 3, 777], [5000, 1, 130, 64, 2222]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(lengths, dtype):
    cache = PagedInt4Cache(1, 2, sum(-(-t // 64) for t in lengths), dtype=dtype)
    assert_attends(cache, *fill(cache, lengths, seed=7), 4)
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,ratio", [(1, 1), (3, 2), (2, 3), (1, 5), (2, 7), (8, 8)])
def test_head_layouts(kv_heads, ratio):
    cache = PagedInt4Cache(2, kv_heads, 40)
    assert_attends(cache, *fill(cache, [600, 77, 1], seed=11), ratio, layer=1)


@pytest.mark.gpu
def test_many_short_sequences():
    """More units than there are CTAs: shares that hold several units, or parts of two."""
    lengths = [(37 * i) % 190 for i in range(120)]
    cache = PagedInt4Cache(1, 4, sum(-(-t // 64) for t in lengths))
    assert_attends(cache, *fill(cache, lengths, seed=13), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("key_size,value_size,scaling", [(1.0, 1e-4, 0.1), (1.0, 2000.0, 0.1), (100.0, 1.0, 0.01), (1e-3, 1.0, 30.0)])
def test_magnitudes(dtype, key_size, value_size, scaling):
    cache = PagedInt4Cache(1, 1, 20, dtype=dtype)
    seqs = cache.add(2)
    k = [vectors(t, 1, torch.float32, i).mul(key_size).to(dtype) for i, t in enumerate((500, 90))]
    v = [vectors(t, 1, torch.float32, 5 + i).mul(value_size).to(dtype) for i, t in enumerate((500, 90))]
    v[0][100:] *= 16  # scales that grow along the sequence
    cache.write(0, cache.extend(seqs, [500, 90]), torch.cat(k), torch.cat(v))
    assert_attends(cache, seqs, k, v, 4, scaling=scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,ratio", [(4, 1), (2, 3), (2, 4), (1, 5), (2, 8)])
def test_an_fp16_result_is_as_good_as_its_rounding(kv_heads, ratio):
    """Besides the result's rounding (2^-11 at most, about 2e-4 in the mean square) there are FP32 errors of scores, exponentials and
    sums: below 2e-5 of a result that is a fiftieth of its terms, a tenth of the rounding, sqrt(1 + 0.1^2) = 1.005 together."""
    cache = PagedInt4Cache(1, kv_heads, 40)
    seqs, k, v = fill(cache, [2000, 300], seed=11)
    got = assert_attends(cache, seqs, k, v, ratio, seed=4)
    q = torch.randn(2, kv_heads * ratio, 128, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).half()
    for i in range(2):
        want = formula(q[i], k[i], v[i])[0]
        off, rounding = (got[i].double() - want).norm(), (want.half().double() - want).norm()
        assert off < 1.05 * rounding, f"sequence {i}: {off / rounding:.3f}"


@pytest.mark.gpu
def test_a_maximum_that_grows_along_the_sequence():
    cache = PagedInt4Cache(1, 1, 40)
    seqs = cache.add(1)
    k = vectors(2000, 1, torch.float16, 1) * 0.1 + torch.linspace(0, 4, 2000, device=DEV)[:, None, None].half()
    v = vectors(2000, 1, torch.float16, 2)
    cache.write(0, cache.extend(seqs, 2000), k, v)
    step = cache.extend(seqs, 0)
    q = torch.full((1, 4, 128), 0.5, dtype=torch.float16, device=DEV)
    want, _, bound = formula(q[0], k, v)
    assert ((cache.attend(0, step, q)[0].double() - want).abs() <= bound).all()


@pytest.mark.gpu
def test_what_lies_behind_a_sequence_counts_for_nothing():
    """Uninitialised parts of pages hold whatever was there: NaN scales, infinities."""
    cache = PagedInt4Cache(1, 2, 8)
    cache.pages.view(torch.int16).fill_(0x7E01)  # FP16 NaN in every parameter
    seqs, k, v = fill(cache, [100, 7, 130], seed=17)
    assert_attends(cache, seqs, k, v, 4)


@pytest.mark.gpu
def test_a_nan_reaches_its_sequence_and_head_only():
    cache = PagedInt4Cache(1, 2, 8)
    seqs, k, v = fill(cache, [100, 130], seed=19)
    q = torch.randn(2, 8, 128, device=DEV).half()
    clean = cache.attend(0, cache.extend(seqs, 0), q)
    step = cache.extend(seqs, [1, 1])
    nk, nv = vectors(2, 2, torch.float16, 1), vectors(2, 2, torch.float16, 2)
    nk[0, 1, 3] = torch.nan
    cache.write(0, step, nk, nv)
    got = cache.attend(0, step, q)
    assert got[0, 4:].isnan().all() and got[0, :4].isfinite().all() and got[1].isfinite().all()
    assert clean.isfinite().all()
    step = cache.extend(seqs, [1, 1])
    nk[0, 1, 3], nv[1, 0, 100] = 0, torch.inf
    cache.write(0, step, nk, nv)
    got = cache.attend(0, step, q)
    assert got[1, :4, 64:].isnan().all() and got[1, :4, :64].isfinite().all() and got[1, 4:].isfinite().all()


@pytest.mark.gpu
def test_query_layouts_streams_and_a_captured_call():
    cache = PagedInt4Cache(1, 2, 40)
    seqs, k, v = fill(cache, [1500, 20], seed=23)
    step = cache.extend(seqs, 0)
    fused = torch.randn(2, 12, 128, device=DEV).half()
    q = fused[:, :8]
    want = cache.attend(0, step, q.contiguous())
    assert torch.equal(cache.attend(0, step, q), want)
    assert torch.equal(cache.attend(0, step, q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    for _ in range(10):
        assert torch.equal(cache.attend(0, step, q), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        here = cache.attend(0, step, q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            there = cache.attend(0, step, q)
    torch.cuda.synchronize()
    assert torch.equal(here, want)
    fused.copy_(torch.randn_like(fused))
    graph.replay()
    assert torch.equal(there, cache.attend(0, step, q))


@pytest.mark.gpu
def test_pages_outside_the_pool_set_the_status_and_touch_nothing():
    from reskv_b200._extension import host

    cache = PagedInt4Cache(1, 1, 2)
    cache.pages.fill_(3)
    seqs = cache.add(1)
    step = cache.extend(seqs, 70)
    x = vectors(70, 1, torch.float16, 1)
    for table in ([[0, 2]], [[0, -1]]):
        bad = torch.tensor(table, dtype=torch.int32, device=DEV)
        with pytest.raises(RuntimeError, match="status 0x2"):
            host().paged_write(cache.pages, 0, cache._status, x, x, step.cu_seqlens, step.starts, bad)
            cache.check()
        assert (cache.pages[0, 1] == 3).all()
        cache._status.zero_()
        with pytest.raises(RuntimeError, match="status 0x2"):
            host().paged_attention(cache.pages, 0, cache._status, x[:1], step.device_lengths, bad, None, False)
            cache.check()
        cache._status.zero_()
    far = torch.tensor([200], dtype=torch.int32, device=DEV)  # tokens behind the table
    with pytest.raises(RuntimeError, match="status 0x2"):
        host().paged_read(cache.pages, 0, cache._status, False, step.cu_seqlens, far, step.table, 70)
        cache.check()
    cache._status.zero_()


# ---- pages ------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("layers,kv_heads,pages,pairs", [(1, 1, 2, 1), (3, 2, 40, 17), (2, 1, 1200, 600)])
def test_copy_pages(layers, kv_heads, pages, pairs):
    cache = PagedInt4Cache(layers, kv_heads, pages)
    cache.pages.copy_(torch.randint(0, 256, cache.pages.shape, device=DEV, dtype=torch.uint8))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    src, dst = order[:pairs], order[pairs:2 * pairs]
    src[-1] = src[0]  # a source may serve several destinations
    want = cache.pages.clone()
    want[:, dst] = want[:, src]
    cache.copy_pages(src, dst)
    assert torch.equal(cache.pages, want)
    cache.copy_pages([], [])


@pytest.mark.gpu
def test_forked_sequences_go_their_own_ways_and_survive_a_compaction():
    cache = PagedInt4Cache(2, 2, 30)
    seqs, k, v = fill(cache, [130, 64, 300], seed=29)
    children = cache.fork([seqs[0], seqs[0], seqs[1]])
    everyone = [seqs[0], seqs[2], *children]
    ks, vs = [k[0], k[2], k[0], k[0], k[1]], [v[0], v[2], v[0], v[0], v[1]]
    cache.free([seqs[1]])
    for turn in range(3):
        step = cache.extend(everyone, [1, 60, 2, 1, 3])
        nk, nv = vectors(67, 2, torch.float16, 100 + turn), vectors(67, 2, torch.float16, 200 + turn)
        for layer in range(2):
            cache.write(layer, step, nk, nv)
        at = np.concatenate(([0], np.cumsum(step.counts)))
        ks = [torch.cat((x, nk[a:b])) for x, a, b in zip(ks, at, at[1:])]
        vs = [torch.cat((x, nv[a:b])) for x, a, b in zip(vs, at, at[1:])]
        if turn == 1:
            before = cache.attend(1, step, torch.ones(5, 4, 128, dtype=torch.float16, device=DEV))
            used = cache.compact()
            assert used == cache.capacity - cache.free_pages
            assert max(max(e.pages) for e in cache._book.sequences.values()) == used - 1
            with pytest.raises(ValueError, match="moved"):
                cache.attend(1, step, torch.ones(5, 4, 128, dtype=torch.float16, device=DEV))
            again = cache.attend(1, cache.extend(everyone, 0), torch.ones(5, 4, 128, dtype=torch.float16, device=DEV))
            assert (again - before).abs().max() < 2e-3  # other shares, another order of the sums
    for layer in range(2):
        assert_attends(cache, everyone, ks, vs, 4, layer=layer)
    cache.free(everyone)
    assert cache.free_pages == cache.capacity
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_prompts_then_tokens(dtype):
    """A batch as a server has it: packed prompts are attended to and stored, then every sequence takes tokens; each step's
    attention is that over the stored values."""
    cache = PagedInt4Cache(1, 2, 20, dtype=dtype)
    seqs, lengths = cache.add(3), [200, 33, 64]
    step = cache.extend(seqs, lengths)
    q, k, v = vectors(297, 8, dtype, 1), vectors(297, 2, dtype, 2), vectors(297, 2, dtype, 3)
    cache.write(0, step, k, v)
    stored_k, stored_v = cache.read(0, step)
    full = prompt_attention(q, stored_k, stored_v, step.cu_seqlens)
    last = [t - 1 for t in step.cu_seqlens[1:].tolist()]
    one = cache.attend(0, step, q[last])
    u = torch.finfo(dtype).eps
    # the prompt's attention reads the stored values rounded to the type and rounds its weights to it: a few steps of the type
    assert (one.double() - full[last].double()).abs().max() <= 8 * u * stored_v.abs().max().double()
    ks, vs = [list(x.split(lengths)) for x in (k, v)]
    for turn in range(3):
        step = cache.extend(seqs, 1)
        nk, nv = vectors(3, 2, dtype, 10 + turn), vectors(3, 2, dtype, 20 + turn)
        cache.write(0, step, nk, nv)
        ks, vs = [torch.cat((x, y[None])) for x, y in zip(ks, nk)], [torch.cat((x, y[None])) for x, y in zip(vs, nv)]
        assert_attends(cache, seqs, ks, vs, 4, seed=60 + turn)


@pytest.mark.gpu
def test_refusals():
    for args in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, True, 1), (1.0, 1, 1)):
        with pytest.raises(ValueError):
            PagedInt4Cache(*args)
    with pytest.raises(ValueError):
        PagedInt4Cache(1, 1, 1, dtype=torch.float32)
    with pytest.raises(ValueError):
        PagedInt4Cache(1, 1, 1, device="cpu")
    cache = PagedInt4Cache(1, 2, 4)
    seqs = cache.add(2)
    step = cache.extend(seqs, [3, 4])
    x, q = vectors(7, 2, torch.float16, 1), vectors(2, 8, torch.float16, 2)
    for key, value in ((x[:6], x[:6]), (x.bfloat16(), x.bfloat16()), (x, x[:6]), (x, x.float()), (x[:, :1], x[:, :1]), (x[..., :64], x[..., :64]),
                       (x.cpu(), x.cpu()), (x.clone().requires_grad_(), x)):
        with pytest.raises(ValueError):
            cache.write(0, step, key, value)
    for layer in (-1, 1):
        with pytest.raises(ValueError):
            cache.write(layer, step, x, x)
    for bad in (q[:1], q.float(), q[:, :3], q[..., :64], vectors(2, 18, torch.float16, 2), q.cpu(), q.clone().requires_grad_()):
        with pytest.raises(ValueError):
            cache.attend(0, step, bad)
    for scaling in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            cache.attend(0, step, q, scaling=scaling)
    with pytest.raises(TypeError):
        cache.attend(0, None, q)
    other = PagedInt4Cache(1, 2, 4)
    with pytest.raises(ValueError, match="another cache"):
        other.attend(0, step, q)
    for src, dst in (([0], [4]), ([0], []), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0.0], [1])):
        with pytest.raises(ValueError):
            cache.copy_pages(src, dst)
    cache.extend([seqs[0]], 1)  # the older step is out of date now
    with pytest.raises(ValueError, match="extended"):
        cache.write(0, step, x, x)
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.extend([seqs[0]], 1000)
    step = cache.extend(seqs, 1)
    cache.fork([seqs[0]])
    with pytest.raises(ValueError):
        cache.write(0, step, x[:2], x[:2])


@pytest.mark.gpu
def test_attention_on_two_streams_at_once():
    """Every call has scratch of its own: calls that overlap give the bits of calls in turn."""
    from concurrent.futures import ThreadPoolExecutor

    cache = PagedInt4Cache(1, 2, 200)
    seqs, _, _ = fill(cache, [3000, 20, 1500, 64], seed=31)
    steps = [cache.extend(seqs[:2], 0), cache.extend(seqs[2:], 0)]
    queries = [torch.randn(2, 8, 128, device=DEV).half() for _ in range(2)]
    want = [cache.attend(0, s, q) for s, q in zip(steps, queries)]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [cache.attend(0, steps[i], queries[i]) for _ in range(50)]
        torch.cuda.synchronize()
        return all(torch.equal(g, want[i]) for g in got)

    with ThreadPoolExecutor(2) as pool:
        assert list(pool.map(work, (0, 1))) == [True, True]


@pytest.mark.gpu
def test_steps_without_sequences_or_tokens():
    cache = PagedInt4Cache(1, 2, 2)
    none = cache.extend([], [])
    empty = torch.zeros(0, 2, 128, dtype=torch.float16, device=DEV)
    cache.write(0, none, empty, empty)
    assert cache.attend(0, none, torch.zeros(0, 4, 128, dtype=torch.float16, device=DEV)).shape == (0, 4, 128)
    assert cache.read(0, none, everything=True)[0].shape == (0, 2, 128)
    step = cache.extend(cache.add(2), 0)  # sequences that have no tokens: no pages
    out, lse = cache.attend(0, step, torch.ones(2, 4, 128, dtype=torch.float16, device=DEV), return_lse=True)
    assert not out.any() and (lse == -torch.inf).all()
    assert cache.fork([]) == [] and cache.compact() == 0
    cache.free([])


@pytest.mark.gpu
def test_long_sequences_and_a_pool_beyond_four_gigabytes():
    """Byte offsets that pass 32 bits."""
    cache = PagedInt4Cache(1, 8, 62000)  # 4.57 GB
    filler, target = cache.add(2)
    cache.extend([filler], 61000 * 64)
    seqs = [target]
    k, v = vectors(40000, 8, torch.float16, 41), vectors(40000, 8, torch.float16, 42)
    step = cache.extend(seqs, 40000)
    assert min(cache._book.of(target).pages) * 8 * 9216 > 2**32
    cache.write(0, step, k, v)
    got = cache.read(0, step)
    assert torch.equal(got[0], values_of(k)) and torch.equal(got[1], values_of(v))
    assert_attends(cache, seqs, [k], [v], 2)
    cache.copy_pages([cache._book.of(target).pages[0]], [0])
    assert torch.equal(cache.pages[0, 0], cache.pages[0, cache._book.of(target).pages[0]])


@pytest.mark.gpu
def test_tables_are_not_made_in_a_capture():
    """A captured copy would read host memory that belongs to somebody else by the time of a replay."""
    cache = PagedInt4Cache(1, 1, 4)
    seqs, _, _ = fill(cache, [5, 70])
    step = cache.extend(seqs, 1)
    x = torch.zeros(2, 1, 128, dtype=torch.float16, device=DEV)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    cache.write(0, step, x, x)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="outside of the capture"):
                cache.extend(seqs, 1)
            with pytest.raises(RuntimeError, match="outside of the capture"):
                cache.read(0, step, everything=True)
            out = cache.attend(0, step, x)
        finally:
            graph.capture_end()
    assert cache.length(seqs[0]) == 6
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, cache.attend(0, step, x))


@pytest.mark.gpu
def test_what_is_no_tensor_is_refused():
    cache = PagedInt4Cache(1, 1, 4)
    step = cache.extend(cache.add(1), 1)
    x = torch.zeros(1, 1, 128, dtype=torch.float16, device=DEV)
    for call in (lambda: cache.write(0, step, None, x), lambda: cache.write(0, step, x, 1.0), lambda: cache.attend(0, step, [1])):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        cache.write(0, step, x[0, 0, 0], x)


@pytest.mark.gpu
def test_a_workspace_for_more_is_enough_for_less():
    from reskv_b200._extension import library

    need = library().reskv_paged_attention_workspace_bytes
    for sequences in (1, 2, 7, 40):
        for heads in (1, 2, 8):
            sizes = [need(sequences, width, heads) for width in range(0, 300)]
            assert sizes == sorted(sizes) and sizes[-1] <= need(sequences + 1, 299, heads) <= need(sequences + 1, 299, heads + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_shares_of_several_segments_have_the_same_bits_every_time(dtype):
    """Shares that hold several units, each one or two pages long: every lane of a warp has to see the segment that the
    warp has gone on to.  Against the formula, and the same bits in every call."""
    lengths = [1 + (53 * i) % 128 for i in range(250)]
    cache = PagedInt4Cache(1, 3, sum(-(-t // 64) for t in lengths), dtype=dtype)
    seqs, k, v = fill(cache, lengths, seed=43)
    first = assert_attends(cache, seqs, k, v, 3, seed=44)
    step = cache.extend(seqs, 0)
    q = torch.randn(250, 9, 128, generator=torch.Generator(device=DEV).manual_seed(44), device=DEV).to(dtype)
    for _ in range(30):
        assert torch.equal(cache.attend(0, step, q), first)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[40, 90], [600, 33], [5000]], ids=str)
def test_keys_whose_scores_overflow_to_minus_infinity(lengths):
    """BF16 keys so large that their products leave FP32: where these are the first ones of a warp or of a share, the later ones have
    the weights that they have alone."""
    cache = PagedInt4Cache(1, 2, 100, dtype=torch.bfloat16)
    seqs = cache.add(len(lengths))
    k = [vectors(t, 2, torch.bfloat16, 80 + i) for i, t in enumerate(lengths)]
    v = [vectors(t, 2, torch.bfloat16, 90 + i) for i, t in enumerate(lengths)]
    for x in k:
        x[:len(x) - 7, 1] = -1e38
    cache.write(0, cache.extend(seqs, lengths), torch.cat(k), torch.cat(v))
    q = vectors(len(lengths), 8, torch.bfloat16, 99).abs() + 1
    got, lse = cache.attend(0, cache.extend(seqs, 0), q, return_lse=True)
    for i in range(len(lengths)):
        for heads, keys in ((slice(0, 4), slice(None)), (slice(4, 8), slice(-7, None))):
            g = slice(heads.start // 4, heads.start // 4 + 1)
            want, want_lse, bound = formula(q[i, heads], k[i][keys, g], v[i][keys, g])
            assert ((got[i, heads].double() - want).abs() <= bound).all()
            assert (lse[i, heads].double() - want_lse).abs().max() < 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scaling", [1e-12, 1e-20, 1e-37])
def test_queries_of_zeros_with_a_tiny_scaling(dtype, scaling):
    """All scores are 0: the mean of the values, whatever factor the scores are brought to."""
    cache = PagedInt4Cache(1, 2, 20, dtype=dtype)
    seqs, k, v = fill(cache, [40, 300], seed=47)
    q = torch.zeros(2, 8, 128, dtype=dtype, device=DEV)
    q[:, 4:] = vectors(2, 4, dtype, 48)  # scores that are as good as 0
    got, lse = cache.attend(0, cache.extend(seqs, 0), q, scaling=scaling, return_lse=True)
    for i in range(2):
        want, want_lse, bound = formula(q[i], k[i], v[i], scaling)
        assert ((got[i].double() - want).abs() <= bound).all()
        assert (lse[i].double() - want_lse).abs().max() < 1e-3


class Tagged(torch.Tensor):
    pass


@pytest.mark.gpu
def test_what_would_be_lost_without_a_word_is_refused():
    from torch.autograd import forward_ad

    cache = PagedInt4Cache(1, 2, 4)
    step = cache.extend(cache.add(2), [1, 1])
    x, q = vectors(2, 2, torch.float16, 1), vectors(2, 8, torch.float16, 2)
    cache.write(0, step, x, x)
    want, pages = cache.attend(0, step, q), cache.pages[0, :2, :, 0].clone()
    with forward_ad.dual_level():
        dual = lambda y: forward_ad.make_dual(y, torch.ones_like(y))  # noqa: E731
        for call in (lambda: cache.write(0, step, dual(x), x), lambda: cache.write(0, step, x, dual(x)), lambda: cache.attend(0, step, dual(q))):
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
    tag = lambda y: y.as_subclass(Tagged)  # noqa: E731
    for call in (lambda: cache.write(0, step, tag(x), x), lambda: cache.write(0, step, x, tag(x)), lambda: cache.attend(0, step, tag(q)),
                 lambda: torch.vmap(lambda y: cache.attend(0, step, y))(q[None]),
                 lambda: torch.jit.trace(lambda y: cache.attend(0, step, y), (q,), check_trace=False)):
        with pytest.raises(ValueError, match="plain tensors"):
            call()
    cache.write(0, step, torch._neg_view(-x), torch._neg_view(-x))
    assert torch.equal(cache.pages[0, :2, :, 0, :64], pages[..., :64]) and torch.equal(cache.attend(0, step, torch._neg_view(-q)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("reuse", [False, True])
def test_what_fails_in_front_of_the_device_leaves_the_cache_as_it_is(monkeypatch, reuse):
    """No memory for a step's tables, a page copy that is not launched: no tokens counted, no sequences, no pages moved, and the step in
    front is still the one."""
    import reskv_b200.paged as paged

    cache = PagedInt4Cache(1, 2, 12)
    seqs, k, v = fill(cache, [100, 64, 130], seed=61)
    cache.free([seqs.pop(1)])
    k.pop(1), v.pop(1)
    step = cache.extend(seqs, 0, width=8)
    q = vectors(2, 8, torch.float16, 62)
    want, free = cache.attend(0, step, q), cache.free_pages

    def fails(*args):
        raise MemoryError

    with monkeypatch.context() as m:
        m.setattr(paged, "_pinned", fails)
        with pytest.raises(MemoryError):
            cache.extend(seqs, [200, 1], reuse=step if reuse else None)
        m.setattr(PagedInt4Cache, "_copy", fails)
        for call in (lambda: cache.fork([seqs[0], seqs[1]]), cache.compact):
            with pytest.raises(MemoryError):
                call()
    assert [cache.length(s) for s in seqs] == [100, 130] and cache.free_pages == free and len(cache._book.sequences) == 2
    assert torch.equal(cache.attend(0, step, q), want)
    assert_attends(cache, seqs, k, v, 4)
    step = cache.extend(seqs, 0, reuse=step if reuse else None)
    twins = cache.fork(seqs)
    assert cache.compact() == 7
    assert torch.equal(cache.attend(0, cache.extend(twins, 0, width=8), q), want)


@pytest.mark.gpu
def test_pages_are_not_forked_or_moved_in_a_capture():
    """The book would change once and the captured copies run at every replay, the first time behind whoever reads the pages."""
    cache = PagedInt4Cache(1, 1, 8)
    seqs, k, v = fill(cache, [70, 5, 70])
    cache.free([seqs.pop(1)])
    step, q = cache.extend(seqs, 0), vectors(2, 2, torch.float16, 3)
    want = cache.attend(0, step, q)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            for call in (lambda: cache.fork(seqs), cache.compact):
                with pytest.raises(RuntimeError, match="outside of the capture"):
                    call()
            out = cache.attend(0, step, q)
        finally:
            graph.capture_end()
    assert len(cache._book.sequences) == 2 and cache.free_pages == 4
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    twins = cache.fork(seqs)
    assert cache.compact() == 6
    assert torch.equal(cache.attend(0, cache.extend(twins, 0), q), want)


def test_a_capture_is_looked_for_on_the_cache_s_device(monkeypatch):
    """The stream that counts is the current one of the cache's device, whichever device is current."""
    import reskv_b200.paged as paged

    seen = []

    class On:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            seen.append(self.device)

        def __exit__(self, *args):
            seen.append(None)

    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(seen) and seen[-1] == torch.device("cuda", 1))
    with pytest.raises(RuntimeError, match="outside of the capture"):
        paged._refuse_capture(torch.device("cuda", 1))
    paged._refuse_capture(torch.device("cuda", 0))
    assert seen == [torch.device("cuda", 1), None, torch.device("cuda", 0), None]


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [2.0**-10, 128**-0.5, 1.0])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 32000.0), (torch.bfloat16, 32000.0), (torch.bfloat16, 2.0**60)])
@pytest.mark.parametrize("ratio", [3, 6])
def test_scores_so_large_that_one_key_takes_all(ratio, dtype, size, scaling):
    """Scores up to 2^30, 2^120: the largest one's weight is 1 (of several that are alike an equal share), the others' are 0, however
    large the step of FP32 is there.  Value groups with scales far apart bring other units to the weights."""
    cache = PagedInt4Cache(1, 1, 200, dtype=dtype)
    seqs, lengths = cache.add(3), [40, 700, 3000]
    places = torch.randperm(250, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) - 125
    k = torch.zeros(3740, 1, 128, dtype=dtype, device=DEV)
    k[:, 0, 3] = places.repeat(15)[:3740].double().mul(size / 128).to(dtype)
    v = vectors(3740, 1, dtype, 5) * torch.where(torch.arange(3740, device=DEV) % 7 == 0, 100.0, 0.01).to(dtype)[:, None, None]
    step = cache.extend(seqs, lengths)
    cache.write(0, step, k, v)
    key = stored(k)[0].double().flatten(-2).to(DEV)
    q = torch.zeros(3, ratio, 128, dtype=dtype, device=DEV)
    q[..., 3] = size * torch.tensor([1.0, -1.0] * 4, device=DEV)[:ratio].to(dtype)
    got, lse = cache.attend(0, step, q, scaling=scaling, return_lse=True)
    u = torch.finfo(dtype).eps / 2
    for i, (a, b) in enumerate(((0, 40), (40, 740), (740, 3740))):
        low, scale, code = (x[a:b] for x in (stored(v)[2], stored(v)[1], stored(v)[3]))
        value = (low.double() + scale.double() * code.double()).flatten(-2)[:, 0].to(DEV)
        size_of = (low.double().abs() + scale.double() * code.double()).flatten(-2)[:, 0].to(DEV)
        for h in range(ratio):
            s = key[a:b, 0].double() @ q[i, h].double() * scaling
            share = (s == s.max()).double() / (s == s.max()).sum()
            want, terms = share @ value, share @ size_of
            # as in `formula`, without an error of the scores
            bound = u * want.abs() + (2.0**-11 + 2.0**-19) * terms + 2.0**-38 * (b - a) * terms.amax() + 2.0**-25
            off = (got[i, h].double() - want).abs()
            assert (off <= bound).all(), f"sequence {i}, head {h}: off by {off.max():.3e}, {(off - bound).max():.3e} too much"
            assert (lse[i, h].double() - s.max()).abs() <= 2.0**-20 * s.max().abs() + 8


@pytest.mark.gpu
@pytest.mark.parametrize("key_power,value_power", [(0, -57), (0, 98), (108, 0), (108, 98), (-100, 0)])
def test_bf16_at_the_ends_of_its_range(key_power, value_power):
    """The largest keys (2^111) and values (2^101) and the finest scales (2^-60) that are promised."""
    dtype = torch.bfloat16
    cache = PagedInt4Cache(1, 1, 20, dtype=dtype)
    seqs, lengths = cache.add(2), [500, 90]
    k = [vectors(t, 1, torch.float32, i).clamp(-8, 8).double().mul(2.0**key_power).to(dtype) for i, t in enumerate(lengths)]
    v = [vectors(t, 1, torch.float32, 5 + i).clamp(-8, 8).double().mul(2.0**value_power).to(dtype) for i, t in enumerate(lengths)]
    cache.write(0, cache.extend(seqs, lengths), torch.cat(k), torch.cat(v))
    q = vectors(2, 4, dtype, 6)
    scaling = 0.1 * 2.0**-key_power
    got = cache.attend(0, cache.extend(seqs, 0), q, scaling=scaling)
    for i in range(2):
        want, _, bound = formula(q[i], k[i], v[i], scaling)
        assert ((got[i].double() - want).abs() <= bound - 2.0**-25).all()  # without the part that is not relative to the values
