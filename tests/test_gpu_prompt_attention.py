"""``prompt_attention`` against the formula in 64 bits."""

import pytest
import torch

from reskv_b200 import prompt_attention

DEV = "cuda"


def formula(q, k, v, ends, scaling=128**-0.5, causal=True):
    """(out, lse, bound) in 64 bits; ``bound``: how far a kernel may be off that rounds weights and results once to the type.

    With u half a step of the type and A = sum_j p_j |v_j|: the weights' rounding moves a result by at most u A, its own
    rounding by u |o|.  An error e of a weight's exponential moves it by at most 2 e A (numerator and sum); e is at most 2^-13
    for the exponential itself and |ds| for a score that is off by ds, where 128 products are added in FP32 with an error of
    at most 128 * 2^-23 sum|q k|.  FP16 weights below 2^-14 are off by up to 2^-25 of the largest weight, in all 2^-25 sum|v|."""
    u = torch.finfo(q.dtype).eps / 2
    q, k, v = q.double(), k.double(), v.double()
    heads, ratio = q.shape[1], q.shape[1] // k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for a, b in zip(ends, ends[1:]):
        if a == b:
            continue
        for h in range(heads):
            qq, kk, vv = q[a:b, h], k[a:b, h // ratio], v[a:b, h // ratio]
            s = qq @ kk.T * scaling
            if causal:
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -torch.inf)
            p = torch.softmax(s, -1)
            ds = 128 * 2.0**-23 * scaling * (qq.abs() @ kk.abs().T).amax(-1, keepdim=True)
            out[a:b, h], spread = p @ vv, p @ vv.abs()
            lse[a:b, h] = torch.logsumexp(s, -1)
            bound[a:b, h] = u * (spread + out[a:b, h].abs()) + 2 * spread * (2.0**-13 + ds) + 2.0**-25 * vv.abs().sum(0)
    return out, lse, bound


def inputs(lengths, kv_heads, ratio, dtype, seed=0, spread=1.5, behind=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    total = sum(lengths) + behind
    x = torch.randn(total, kv_heads * (ratio + 2), 128, generator=g, device=DEV)
    x[:, :kv_heads * ratio] *= spread
    x = x.to(dtype)
    ends = [0]
    for t in lengths:
        ends.append(ends[-1] + t)
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    h = kv_heads
    return x[:, :h * ratio], x[:, h * ratio:h * (ratio + 1)], x[:, h * (ratio + 1):], ends, cu


def assert_within(got, want, bound):
    excess = ((got.double() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert excess <= 0, f"off by {(got.double() - want).abs().max().item():.3e}, {excess:.3e} too much"


LENGTHS = [[1], [2, 1, 3], [127], [128], [129], [64, 65], [255, 256, 257], [300, 0, 17, 0], [1000], [31, 513, 128, 1, 700]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(lengths, dtype):
    q, k, v, ends, cu = inputs(lengths, 2, 4, dtype)
    got, lse = prompt_attention(q, k, v, cu, return_lse=True)
    want, want_lse, bound = formula(q, k, v, ends)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    assert_within(got, want, bound)
    # the sum of exponentials: relative 2^-13 at most, scores off by 128 * 2^-23 * sum|q k| * scaling (< 2^-10 here)
    assert (lse.double() - want_lse).abs().max().item() < 2e-3


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kv_heads,ratio", [(1, 1), (3, 1), (2, 2), (1, 3), (2, 5), (1, 7), (1, 8), (1, 12), (1, 40), (1, 128)])
def test_head_layouts(kv_heads, ratio, causal):
    q, k, v, ends, cu = inputs([45, 200, 1], kv_heads, ratio, torch.float16, seed=1)
    assert_within(prompt_attention(q, k, v, cu, causal=causal), *formula(q, k, v, ends, causal=causal)[::2])


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [0.01, 1.0])
def test_scaling(scaling):
    q, k, v, ends, cu = inputs([400], 1, 4, torch.bfloat16, seed=2)
    assert_within(prompt_attention(q, k, v, cu, scaling=scaling), *formula(q, k, v, ends, scaling=scaling)[::2])


@pytest.mark.gpu
def test_a_maximum_that_grows_with_every_key_tile():
    """Scores rise along the keys, so that the running maximum and the output so far are rescaled again and again."""
    q, k, v, ends, cu = inputs([900, 700], 1, 4, torch.float16, seed=3, spread=1.0)
    rise = torch.linspace(0, 60, q.shape[0], device=DEV)[:, None]
    k[:, 0, :] = (k[:, 0, :].float() * 0.1 + rise / 128).half()
    q[:, :, :] = (q.float() * 0.05 + 10).half()
    assert_within(prompt_attention(q, k, v, cu), *formula(q, k, v, ends)[::2])


@pytest.mark.gpu
def test_layouts_in_memory():
    """Views, token-major and head-major, copies where rows cannot be read in place: the same numbers."""
    q, k, v, ends, cu = inputs([77, 130], 2, 4, torch.float16, seed=4)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert torch.equal(prompt_attention(q, k, v, cu), want)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*heads_first, cu), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(prompt_attention(odd, k, v, cu), want)
    strided = torch.empty((*k.shape[:2], 256), dtype=k.dtype, device=DEV)[..., ::2].copy_(k)
    assert torch.equal(prompt_attention(q, strided, v, cu), want)
    one = k[:, :1].contiguous()
    assert torch.equal(prompt_attention(q, one.expand(-1, 2, -1), one.expand(-1, 2, -1), cu),
                       prompt_attention(q, one.repeat(1, 2, 1), one.repeat(1, 2, 1), cu))


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_stay_and_do_not_count():
    q, k, v, ends, cu = inputs([70, 33], 2, 4, torch.float16, seed=5, behind=40)
    want = prompt_attention(q[:103], k[:103], v[:103], cu)
    for x in (q, k, v):
        x[103:] = float("nan")
    v[110] = float("inf")
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    got = prompt_attention(q, k, v, cu, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(got[:103], want) and (got[103:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ratio", [1, 4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("side", ["key", "value"])
def test_what_is_not_finite_counts_only_where_it_is_attended_to(dtype, ratio, bad, side):
    """A later token's infinities and NaN do not reach the rows before it; the rows that see them have what the formula has."""
    q, k, v, ends, cu = inputs([200, 150], 2, ratio, dtype, seed=6)
    clean = prompt_attention(q, k, v, cu)
    at = 131  # inside a key tile, seen by part of a row tile
    (k if side == "key" else v)[at, 1, 5:9] = bad
    got = prompt_attention(q, k, v, cu)
    own = slice(ratio, 2 * ratio)  # the query heads of KV head 1
    assert torch.equal(got[:at], clean[:at]) and torch.equal(got[200:], clean[200:]) and torch.equal(got[:, :ratio], clean[:, :ratio])
    if side == "value":
        seen = got[at:200, own]
        assert torch.equal(seen[..., :5], clean[at:200, own, :5]) and torch.equal(seen[..., 9:], clean[at:200, own, 9:])
        assert (seen[..., 5:9].isnan() if bad != bad else seen[..., 5:9] == bad).all()
    else:
        # a score of NaN or +inf: NaN.  -inf: a weight of 0
        score = (q[at:200, own].double()[..., 5:9] * bad).sum(-1)
        assert got[at:200, own][(score != score) | (score > 0)].isnan().all()
        rest = score == -torch.inf
        assert got[at:200, own][rest].isfinite().all()


@pytest.mark.gpu
def test_no_tokens_and_no_sequences():
    q, k, v, _, cu = inputs([4], 1, 1, torch.float16)
    assert prompt_attention(q[:0], k[:0], v[:0], cu[:1]).shape == (0, 1, 128)
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    assert not prompt_attention(q, k, v, cu[:1], out=out).any()
    assert not prompt_attention(q, k, v, torch.zeros(5, dtype=torch.int32, device=DEV), out=out).any()


@pytest.mark.gpu
def test_bounds_are_clamped():
    q, k, v, ends, cu = inputs([40, 60], 1, 4, torch.float16, seed=7)
    wild = torch.tensor([-5, 40, 2**31 - 1], dtype=torch.int32, device=DEV)
    assert torch.equal(prompt_attention(q, k, v, wild), prompt_attention(q, k, v, cu))
    back = torch.tensor([0, 100, 30], dtype=torch.int32, device=DEV)  # the second sequence has a negative length: none
    assert torch.equal(prompt_attention(q, k, v, back), prompt_attention(q, k, v, cu[[0, 2]]))


@pytest.mark.gpu
def test_many_sequences_and_calls_in_a_row():
    lengths = [(7 * i) % 90 for i in range(150)]
    q, k, v, ends, cu = inputs(lengths, 2, 2, torch.float16, seed=8)
    want = formula(q, k, v, ends)[::2]
    first = prompt_attention(q, k, v, cu)
    assert_within(first, *want)
    for _ in range(20):
        assert torch.equal(prompt_attention(q, k, v, cu), first)


@pytest.mark.gpu
def test_streams_and_a_captured_call():
    q, k, v, ends, cu = inputs([500, 123], 2, 4, torch.float16, seed=9)
    want = prompt_attention(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        here = prompt_attention(q, k, v, cu)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            there = prompt_attention(q, k, v, cu)
    torch.cuda.synchronize()
    assert torch.equal(here, want)
    other, _, _, _, _ = inputs([500, 123], 2, 4, torch.float16, seed=10)
    q.copy_(other)
    graph.replay()
    assert torch.equal(there, prompt_attention(q, k, v, cu))


@pytest.mark.gpu
def test_refusals():
    q, k, v, _, cu = inputs([8], 2, 4, torch.float16)
    bad = [
        dict(query=q.float()), dict(query=q[..., :64]), dict(key=k[:7]), dict(value=v.bfloat16()), dict(key=k[:, :1]),
        dict(query=q[:, :7]), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[None]), dict(cu_seqlens=cu[:0]), dict(cu_seqlens=cu.cpu()),
        dict(scaling=0.0), dict(scaling=-1.0), dict(scaling=float("nan")), dict(scaling=float("inf")),
        dict(out=torch.empty(8, 8, 64, device=DEV)), dict(out=torch.empty(8, 8, 128, device=DEV)),
        dict(out=torch.empty(8, 8, 256, dtype=torch.float16, device=DEV)[..., :128]), dict(key=k.cpu()),
        dict(query=q.clone().requires_grad_()),
    ]
    for change in bad:
        args = dict(query=q, key=k, value=v, cu_seqlens=cu) | change
        with pytest.raises(ValueError):
            prompt_attention(args.pop("query"), args.pop("key"), args.pop("value"), args.pop("cu_seqlens"), **args)
    with pytest.raises(TypeError):
        prompt_attention(q, k, None, cu)


def test_the_library_refuses_bad_arguments_before_any_launch():
    import numpy as np

    from reskv_b200._extension import ERR_INVALID, ERR_LIMIT, library

    lib = library()
    x = np.zeros((4, 2, 128), np.float16)
    cu = np.array([0, 4], np.int32)
    assert x.ctypes.data % 16 == 0

    def call(q=x.ctypes.data, kh=2, nh=2, step=256, scaling=0.1, total=4, sequences=1):
        return lib.reskv_prompt_attention(q, x.ctypes.data, x.ctypes.data, cu.ctypes.data, sequences, total, kh, nh, 0, step, 128,
                                          256, 128, 256, 128, scaling, 1, x.ctypes.data, None, None)

    assert call(q=None) == ERR_INVALID and b"null" in lib.reskv_last_error()
    assert call(nh=3) == ERR_INVALID and call(kh=0) == ERR_INVALID and call(sequences=-1) == ERR_INVALID
    assert call(kh=1, nh=129) == ERR_LIMIT
    assert call(scaling=0.0) == ERR_INVALID and call(scaling=float("nan")) == ERR_INVALID
    assert call(step=129) == ERR_INVALID and call(q=x.ctypes.data + 2) == ERR_INVALID
    assert call() == ERR_INVALID and b"prompt_attention: q" in lib.reskv_last_error()  # host memory
    assert call(total=0) == 0 and call(sequences=0) == 0


@pytest.mark.gpu
def test_a_thousand_sequences():
    """More sequences than a warp looks at at once, of very different lengths."""
    lengths = [(i * 7919) % 61 for i in range(1000)] + [700, 1, 333]
    q, k, v, ends, cu = inputs(lengths, 1, 2, torch.bfloat16, seed=11)
    assert_within(prompt_attention(q, k, v, cu), *formula(q, k, v, ends)[::2])


@pytest.mark.gpu
def test_two_calls_at_once():
    """Calls of two threads on two streams give the bits of calls in turn."""
    from concurrent.futures import ThreadPoolExecutor

    cases = [inputs(lengths, 2, 4, torch.float16, seed=i) for i, lengths in enumerate(([500, 40], [1, 2, 1200]))]
    want = [prompt_attention(q, k, v, cu) for q, k, v, _, cu in cases]
    torch.cuda.synchronize()

    def work(i):
        q, k, v, _, cu = cases[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [prompt_attention(q, k, v, cu) for _ in range(20)]
        torch.cuda.synchronize()
        return all(torch.equal(g, want[i]) for g in got)

    with ThreadPoolExecutor(2) as pool:
        assert list(pool.map(work, (0, 1))) == [True, True]


# Short calls give every row tile an item of its own; with 150 further sequences there are too many for that, and items hold two.
CROWD = [1] * 150


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", [*LENGTHS, [500, 123]], ids=str)
def test_one_and_two_row_tiles_per_item(lengths, dtype, causal):
    q, k, v, ends, cu = inputs(lengths + CROWD, 2, 4, dtype, seed=12)
    got, lse = prompt_attention(q, k, v, cu, causal=causal, return_lse=True)
    want, want_lse, bound = formula(q, k, v, ends, causal=causal)
    assert_within(got, want, bound)
    assert (lse.double() - want_lse).abs().max().item() < 2e-3
    few = slice(0, ends[len(lengths)])  # a row's arithmetic does not depend on what shares its item
    alone, alone_lse = prompt_attention(q[few], k[few], v[few], cu[:len(lengths) + 1], causal=causal, return_lse=True)
    assert torch.equal(alone, got[few]) and torch.equal(alone_lse, lse[few])


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,ratio", [(3, 1), (1, 3), (2, 5), (1, 12), (1, 40), (1, 128)])
def test_head_layouts_with_two_row_tiles_per_item(kv_heads, ratio):
    q, k, v, ends, cu = inputs([45, 200, 1] + CROWD, kv_heads, ratio, torch.float16, seed=13)
    assert_within(prompt_attention(q, k, v, cu), *formula(q, k, v, ends)[::2])


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [1, 4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_value_that_is_not_finite_with_two_row_tiles_per_item(ratio, bad):
    q, k, v, ends, cu = inputs([200, 150] + CROWD, 2, ratio, torch.float16, seed=14)
    clean = prompt_attention(q, k, v, cu)
    at = 131
    v[at, 1, 5:9] = bad
    got = prompt_attention(q, k, v, cu)
    own = slice(ratio, 2 * ratio)
    seen = torch.zeros_like(got, dtype=torch.bool)
    seen[at:200, own, 5:9] = True
    assert torch.equal(got[~seen], clean[~seen])
    assert (got[seen].isnan() if bad != bad else got[seen] == bad).all()


@pytest.mark.gpu
def test_the_number_of_items_decides_at_its_limit():
    """As many items of one row tile as there are SMs, one less and one more: 32 tokens each."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for n in (sms - 1, sms, sms + 1):
        q, k, v, ends, cu = inputs([32 * 4] * (n // 4) + [32] * (n % 4), 1, 4, torch.float16, seed=n)
        assert_within(prompt_attention(q, k, v, cu), *formula(q, k, v, ends)[::2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bad", [(torch.float16, "infinite"), (torch.bfloat16, "infinite"), (torch.bfloat16, "overflow")])
@pytest.mark.parametrize("crowd", [[], CROWD], ids=["few", "many"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("scaling", [128**-0.5, 4.0])
@pytest.mark.parametrize("at", [79, 80, 160, 230])
def test_leading_keys_whose_scores_are_minus_infinity(at, scaling, dtype, causal, crowd, bad):
    """The first ``at`` keys of a sequence have scores of -inf for all of its queries: their weights are 0, and every row that sees a
    later key has what the sequence without them has.  A row that sees nothing else: no weights, NaN and a sum of 0."""
    q, k, v, ends, cu = inputs([33, 2 * at] + crowd, 2, 4, dtype, seed=15)
    clean = prompt_attention(q, k, v, cu, scaling=scaling, causal=causal)
    a, b = ends[1], ends[2]
    q[a:b, 4:, 7] = 2 + q[a:b, 4:, 7].abs()
    k[a:a + at, 1, 7] = -torch.inf if bad == "infinite" else -torch.finfo(dtype).max
    got, lse = prompt_attention(q, k, v, cu, scaling=scaling, causal=causal, return_lse=True)
    assert torch.equal(got[:, :4], clean[:, :4]) and torch.equal(got[:a], clean[:a]) and torch.equal(got[b:], clean[b:])
    for first in (a, a + at):  # two halves of as many rows
        rows = slice(first, first + at)
        if first == a and causal:
            if bad == "infinite":
                assert got[rows, 4:].isnan().all() and (lse[rows, 4:] == -torch.inf).all()
            continue
        want, want_lse, bound = formula(q[rows, 4:], k[a + at:b, 1:], v[a + at:b, 1:], [0, at], scaling=scaling, causal=causal)
        assert_within(got[rows, 4:], want, bound)
        # a score is off by less than 128 * 2^-23 * sum|q k| * scaling (sum|q k| < 600), the sum of exponentials by 2^-13
        assert (lse[rows, 4:].double() - want_lse).abs().max().item() < 2e-3 + 0.01 * scaling


@pytest.mark.gpu
def test_what_a_call_met_is_its_own():
    """The words are set by the host, no wait runs out here: a call reports to the word that it is given, and calls without one do not
    speak of others."""
    q, k, v, ends, cu = inputs([50, 70], 2, 4, torch.float16, seed=16)
    want = prompt_attention(q, k, v, cu)
    clean, marked = torch.zeros(1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="prompt_attention: device status 0x1"):  # RESKV_CHECK_STATUS=1
        prompt_attention(q, k, v, cu, status=marked)
    assert torch.equal(prompt_attention(q, k, v, cu, status=clean), want) and clean.item() == 0
    assert torch.equal(prompt_attention(q, k, v, cu), want)
    for bad in (clean.float(), clean[:0], clean.cpu()):
        with pytest.raises(ValueError):
            prompt_attention(q, k, v, cu, status=bad)


def test_the_library_refuses_a_status_word_of_the_host():
    import numpy as np

    from reskv_b200._extension import ERR_INVALID, library

    x, cu = np.zeros((4, 2, 128), np.float16), np.array([0, 4], np.int32)
    assert x.ctypes.data % 16 == 0
    call = library().reskv_prompt_attention_reporting
    assert call(*[x.ctypes.data] * 3, cu.ctypes.data, 1, 4, 2, 3, 0, *[256, 128] * 3, 0.1, 1, x.ctypes.data, None, cu.ctypes.data, None) == ERR_INVALID
    assert call(*[x.ctypes.data] * 3, cu.ctypes.data, 0, 4, 2, 2, 0, *[256, 128] * 3, 0.1, 1, x.ctypes.data, None, cu.ctypes.data, None) == 0


class Tagged(torch.Tensor):
    pass


@pytest.mark.gpu
def test_what_would_be_lost_without_a_word_is_refused():
    """Tangents, subclasses, vmap and traces; a negated view is read as what it stands for."""
    from torch.autograd import forward_ad

    q, k, v, ends, cu = inputs([30, 20], 1, 2, torch.float16, seed=17)
    want = prompt_attention(q, k, v, cu)
    with forward_ad.dual_level():
        for i in range(3):
            args = [forward_ad.make_dual(x, torch.ones_like(x)) if i == j else x for j, x in enumerate((q, k, v))]
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                prompt_attention(*args, cu)
    for i in range(4):
        args = [x.as_subclass(Tagged) if i == j else x for j, x in enumerate((q, k, v, cu))]
        with pytest.raises(ValueError, match="plain tensors"):
            prompt_attention(*args)
    with pytest.raises(ValueError, match="plain tensors"):
        torch.vmap(lambda x: prompt_attention(x, k, v, cu))(q[None])
    with pytest.raises(ValueError, match="plain tensors"):
        torch.jit.trace(lambda x: prompt_attention(x, k, v, cu), (q,), check_trace=False)
    with torch.no_grad():
        assert torch.equal(prompt_attention(torch.nn.Parameter(q), k, v, cu), want)
    with torch.inference_mode():
        assert torch.equal(prompt_attention(q.clone(), k, v, cu), want)
    assert torch.equal(prompt_attention(torch._neg_view(-q), torch._neg_view(-k.contiguous()), v, cu), want)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [2.0**-10, 128**-0.5, 1.0])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 32000.0), (torch.bfloat16, 32000.0), (torch.bfloat16, 2.0**60)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_so_large_that_one_key_takes_all(sign, dtype, size, scaling):
    """Scores up to 2^30, 2^120: the largest one's distance to the next is thousands at least, so its weight is 1 (of two that are alike
    a half each) and the others' are 0, however large the step of FP32 is there.  Weights and results are rounded once, an exponential
    is off by 2^-13 at most (see ``formula``)."""
    q, k, v, ends, cu = inputs([50, 300], 1, 4, dtype, seed=18)
    q[..., :], k[..., :] = 0, 0
    q[..., 3] = sign * size
    places = torch.randperm(250, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) - 125  # exact in either type
    k[:, 0, 3] = torch.cat((places, places))[:350].double().mul(size / 128).to(dtype)
    got, lse = prompt_attention(q, k, v, cu, scaling=scaling, return_lse=True)
    for a, b in zip(ends, ends[1:]):
        s = q[a:b, 0].double() @ k[a:b, 0].double().T * scaling
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -torch.inf)
        best = s.amax(-1, keepdim=True)
        share = (s == best).double() / (s == best).sum(-1, keepdim=True)
        want, spread = share @ v[a:b, 0].double(), share @ v[a:b, 0].double().abs()
        u = torch.finfo(dtype).eps / 2
        for h in range(4):
            assert_within(got[a:b, h], want, u * (spread + want.abs()) + 2 * spread * 2.0**-13)
            assert ((lse[a:b, h].double() - best[:, 0]).abs() <= 2.0**-21 * best[:, 0].abs() + 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [3, 5, 7, 12, 40])
def test_what_an_earlier_call_left_on_the_chip_does_not_matter(ratio):
    """128 rows are no multiple of these groups; the rows beyond them hold what was there."""
    q, k, v, ends, cu = inputs([300, 90], 2, ratio, torch.float16, seed=19)
    want = prompt_attention(q, k, v, cu)
    assert_within(want, *formula(q, k, v, ends)[::2])
    for left in (float("nan"), float("inf"), 60000.0):
        y = torch.full((3000, 8, 128), left, dtype=torch.float16, device=DEV)
        prompt_attention(y, y, y, torch.arange(0, 3001, 20, dtype=torch.int32, device=DEV))  # a block or more on every SM
        assert torch.equal(prompt_attention(q, k, v, cu), want)
