"""Attention of whole prompts (psx_b200_prompt_attention) against the formula in double precision.

Tolerance: a score is a sum of head_dim products in float, off by sqrt(head_dim) * 2^-23 or so of the sum of its terms' sizes
(fp32 operands: the dropped products of parts add 2^-23 of it), and twice a factor's rounding; a weight is off by that, by 2^-22 of the
exponential and by its rounding to the operands' type (half a step; fp32: 2^-24); a context by twice its weights' error and
its sums', times the largest value, plus half a step of its own."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx

pytestmark = pytest.mark.gpu
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _attention(q, k, v, q_at, k_at, scale, causal, window):
    """(context, nan where no sequence is; per element the slack that its sequence's sizes give)"""
    heads, kv_heads = q.shape[1], k.shape[1]
    out, most, value = np.full(q.shape, np.nan), np.zeros(q.shape[0]), np.zeros(q.shape[0])
    for b in range(len(q_at) - 1):
        n, m = q_at[b + 1] - q_at[b], k_at[b + 1] - k_at[b]
        if n <= 0:
            continue
        rows = slice(q_at[b], q_at[b + 1])
        out[rows] = 0
        if m <= 0:
            continue
        place, j = m - n + np.arange(n)[:, None], np.arange(m)[None, :]
        seen = j <= place if causal else np.ones((n, m), dtype=bool)
        if causal and window:
            seen &= j > place - window
        for h in range(heads):
            kk, vv = k[k_at[b]:k_at[b + 1], h // (heads // kv_heads)], v[k_at[b]:k_at[b + 1], h // (heads // kv_heads)]
            s = np.where(seen, q[rows, h] @ kk.T * scale, -np.inf)
            w = np.exp(s - np.where(seen.any(1), s.max(1), 0)[:, None])
            total = w.sum(1, keepdims=True)
            out[rows, h] = (w / np.where(total > 0, total, 1)) @ vv
            most[rows] = np.maximum(most[rows], (np.abs(q[rows, h]) @ np.abs(kk).T).max(1) * abs(scale))
            value[rows] = np.maximum(value[rows], np.abs(vv).max())
    return out, most, value


def _slack(dtype, most, value, head_dim, keys):
    score = most * (2 * np.sqrt(head_dim) + 4) * 2.0 ** -23
    weight = 2 * score + 2.0 ** -21 + 2 * HALF_STEP[dtype] + (np.sqrt(keys) + 8) * 2.0 ** -23
    return (weight * value)[:, None, None]


def _tensor(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, dtype)).cuda()


def _check(dtype, q_lens, k_lens, heads, kv_heads, head_dim, causal=True, window=0, scale=None, seed=0, lead=0, behind=0, ctx=None, size=1.0):
    """lead, behind: positions before the first sequence and behind the last one, that belong to none."""
    import torch
    rng = np.random.RandomState(seed + head_dim + sum(q_lens))
    q_at, k_at = (lead + np.concatenate([[0], np.cumsum(n)]).astype(np.int64) for n in (q_lens, k_lens))
    q, k, v = (_tensor(rng.randn(n[-1] + behind, h, head_dim) * s, dtype) for n, h, s in ((q_at, heads, size), (k_at, kv_heads, size), (k_at, kv_heads, 1.0)))
    clean = [x.double().cpu().numpy() for x in (q, k, v)]
    for x, n in ((q, q_at), (k, k_at), (v, k_at)):  # what belongs to no sequence
        x[:lead] = float("nan")
        x[n[-1]:] = float("inf")
    out = torch.full_like(q, 7.0)
    got, status = (ctx or gh.ctx()).prompt_attention(q, k, v, torch.from_numpy(q_at).cuda(), torch.from_numpy(k_at).cuda(), causal=causal, window=window,
                                                     scale=scale, out=out)
    torch.cuda.synchronize()
    assert int(status[0]) == 0
    want, most, value = _attention(*clean, q_at, k_at, head_dim ** -0.5 if scale is None else scale, causal, window)
    got = got.double().cpu().numpy()
    none = np.isnan(want)
    assert (got[none] == 7.0).all()
    slack = _slack(dtype, most, value, head_dim, max(k_lens)) + HALF_STEP[dtype] * np.abs(want)
    bad = ~(np.abs(got - want) <= slack) & ~none
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want)[bad][:5], slack[bad][:5])
    return got


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("head_dim", [64, 128, 96, 80, 8, 72])
def test_one_block(dtype, head_dim):
    _check(dtype, [100], [100], 2, 1, head_dim)
    _check(dtype, [128], [64], 1, 1, head_dim, causal=False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("head_dim", [64, 128, 88])
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 700])
def test_every_length(dtype, head_dim, length):
    _check(dtype, [length], [length], 2, 2, head_dim)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (8, 1), (5, 5)])
def test_packed_sequences_and_head_layouts(dtype, heads, kv_heads):
    _check(dtype, [130, 1, 0, 300, 17, 256, 64], [130, 1, 0, 300, 17, 256, 64], heads, kv_heads, 64, lead=3, behind=70)
    _check(dtype, [5, 200, 33], [205, 200, 600], heads, kv_heads, 128, behind=200)     # prompts that continue a prefix
    _check(dtype, [300, 140, 9], [100, 0, 8], heads, kv_heads, 64)                       # queries before the first key see nothing


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("causal,window", [(False, 0), (False, 9), (True, 1), (True, 50), (True, 128), (True, 129), (True, 300), (True, 2 ** 50)])
def test_masks(dtype, causal, window):
    _check(dtype, [500, 77, 260], [500, 300, 260], 2, 1, 64, causal=causal, window=window, seed=window % 100)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_scales_and_scores_of_every_size(dtype):
    for scale in (0.0, -0.125, 1e-30, 2.0):
        _check(dtype, [200], [200], 2, 1, 64, scale=scale, seed=3)
    _check(dtype, [300], [300], 1, 1, 128, size=6.0)   # scores of some hundred: maxima that grow from block to block


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_long_prompts(dtype):
    _check(dtype, [2500, 1111], [2500, 1500], 2, 1, 128)


def test_many_short_sequences():
    rng = np.random.RandomState(8)
    lens = rng.randint(0, 40, 700).tolist()
    _check("bfloat16", lens, lens, 3, 1, 64)
    _check("float32", lens[:300], lens[:300], 2, 2, 64)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_as_many_sequences_as_there_may_be(dtype):
    lens = np.random.RandomState(14).randint(0, 4, 4096).tolist()
    _check(dtype, lens, lens, 1, 1, 128)


def test_slices_of_one_projection():
    import torch
    rng = np.random.RandomState(9)
    for dtype in ("bfloat16", "float32"):
        wide = _tensor(rng.randn(333, 4 + 2 + 2, 64), dtype)
        q, k, v = wide[:, :4], wide[:, 4:6], wide[:, 6:]
        at = torch.tensor([0, 33, 333], device="cuda")
        a, _ = gh.ctx().prompt_attention(q, k, v, at)
        b, _ = gh.ctx().prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), at)
        assert (a == b).all()


def test_a_nan_stays_in_its_sequence():
    import torch
    rng = np.random.RandomState(10)
    for dtype in ("bfloat16", "float32"):
        q, k, v = (_tensor(rng.randn(300, 2, 64), dtype) for _ in range(3))
        at = torch.tensor([0, 100, 200, 300], device="cuda")
        want, _ = gh.ctx().prompt_attention(q, k, v, at)
        for x in (q, k, v):
            x[150:200] = float("nan")
        got, _ = gh.ctx().prompt_attention(q, k, v, at)
        assert (got[:100] == want[:100]).all() and (got[200:] == want[200:]).all() and got[150:200].isnan().all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_a_key_that_is_not_finite_reaches_every_query_that_sees_it(dtype):
    import torch
    rng = np.random.RandomState(12)
    q, k, v = (_tensor(rng.rand(400, 1, 64) + 0.1, dtype) for _ in range(3))
    at = torch.tensor([0, 400], device="cuda")
    want, _ = gh.ctx().prompt_attention(q, k, v, at)
    for j in range(0, 400, 7):
        for what in (float("nan"), float("inf")):
            bad = k.clone()
            bad[j] = what
            got, _ = gh.ctx().prompt_attention(q, bad, v, at)
            assert got[j:].isnan().all() and (got[:j] == want[:j]).all(), (j, what)


def test_the_same_call_gives_the_same_bits_and_graphs_replay():
    import torch
    rng = np.random.RandomState(11)
    for dtype in ("bfloat16", "float32"):
        ctx = psx.Context(0)
        q, k, v = (_tensor(rng.randn(900, h, 64), dtype) for h in (4, 2, 2))
        at = torch.tensor([0, 300, 900], device="cuda")
        first = ctx.prompt_attention(q, k, v, at)[0].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, status = ctx.prompt_attention(q, k, v, at)
        big = _tensor(rng.randn(3000, 4, 64), dtype)
        ctx.prompt_attention(big, big, big, torch.tensor([0, 3000], device="cuda"))  # (the scratch grows)
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert (out == first).all() and int(status) == 0
        at.copy_(torch.tensor([0, 10, 800]))
        want = ctx.prompt_attention(q, k, v, at)[0]
        graph.replay()
        torch.cuda.synchronize()
        assert (out[:800] == want[:800]).all()


def test_another_stream_and_the_device_stays():
    import torch
    s = torch.cuda.Stream()
    q = torch.randn(200, 2, 64, device="cuda").bfloat16()
    at = torch.tensor([0, 200], device="cuda")
    want = gh.ctx().prompt_attention(q, q, q, at)[0]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = gh.ctx().prompt_attention(q, q, q, at)[0]
    s.synchronize()
    assert (got == want).all()


def test_a_wait_that_runs_out_is_reported():
    import torch
    for dtype in ("bfloat16", "float32"):
        ctx = psx.Context(0)
        q = torch.randn(1000, 2, 64, device="cuda").to(getattr(torch, dtype))
        at = torch.tensor([0, 1000], device="cuda")
        want = ctx.prompt_attention(q, q, q, at)[0]
        ctx.set_wait_limit(20_000_000)
        ctx.test_short_copy(True)
        assert int(ctx.prompt_attention(q, q, q, at)[1].cpu()) == 1
        ctx.test_short_copy(False)
        got, status = ctx.prompt_attention(q, q, q, at)
        assert int(status.cpu()) == 0 and (got == want).all()


def test_refusals():
    import torch
    ctx = gh.ctx()
    at = torch.tensor([0, 4], device="cuda")

    def call(heads=2, kv_heads=1, head_dim=64, dtype=torch.bfloat16, offsets=at, **kw):
        q, k = torch.zeros(4, heads, head_dim, dtype=dtype, device="cuda"), torch.zeros(4, kv_heads, head_dim, dtype=dtype, device="cuda")
        return ctx.prompt_attention(q, k, k, offsets, **kw)

    for status, kw in ((psx.ERR_BAD_ARGUMENT, dict(heads=3, kv_heads=2)), (psx.ERR_UNSUPPORTED, dict(head_dim=136)), (psx.ERR_UNSUPPORTED, dict(head_dim=20, dtype=torch.float32)),
                       (psx.ERR_BAD_ARGUMENT, dict(scale=float("inf"))), (psx.ERR_BAD_ARGUMENT, dict(window=-1)),
                       (psx.ERR_UNSUPPORTED, dict(offsets=torch.zeros(4098, dtype=torch.int64, device="cuda")))):
        with pytest.raises(psx.PsxError) as e:
            call(**kw)
        assert e.value.status == status
    with pytest.raises(TypeError):
        call(dtype=torch.float64)
    for kw in (dict(offsets=at.int()), dict(k_offsets=at[:1]), dict(out=torch.zeros(4, 2, 64, device="cuda"))):
        with pytest.raises(ValueError):
            call(**kw)
    flat = torch.zeros(4 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(psx.PsxError) as e:  # a base that is not on a 16-byte boundary
        x = flat[1:1 + 4 * 128].view(4, 2, 64)
        ctx.prompt_attention(x, x, x, at)
    assert e.value.status == psx.ERR_BAD_ARGUMENT
    q = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert ctx.prompt_attention(q, q, q, torch.tensor([0, 0], device="cuda"))[0].shape == (0, 2, 64)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    out, _ = ctx.prompt_attention(x, q, q, torch.tensor([0, 3], device="cuda"), torch.tensor([0, 0], device="cuda"))  # no keys at all
    assert (out == 0).all()


def test_a_stride_that_no_tensor_map_has_is_refused():
    import torch
    ctx, x, at = gh.ctx(), torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda"), torch.tensor([0, 1], device="cuda")
    for strides in ((2 ** 40, 64, 64), (64, 2 ** 36, 64), (64, 64, 2 ** 62)):
        assert ctx._lib.psx_b200_prompt_attention(ctx._ctx, None, 1, x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), 1, 1, *strides, at.data_ptr(),
                                                  at.data_ptr(), 1, 1, 1, 64, 1.0, 1, 0, None) == psx.ERR_UNSUPPORTED


# Few groups of rows: clusters of CTAs share their keys.  (A piece's factor is one more exponential, 2^-22, and its sums one more rounding:
# within the 2^-21 and the eight roundings of the slack.)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,head_dim", [([16], [16000], 4, 2, 64), ([1], [5000], 1, 1, 128), ([300, 7], [4000, 900], 3, 1, 96),
                                                                   ([1], [640], 1, 1, 8), ([1], [641], 2, 1, 128), ([2000], [500], 1, 1, 64)])
def test_keys_shared_out(dtype, q_lens, k_lens, heads, kv_heads, head_dim):
    _check(dtype, q_lens, k_lens, heads, kv_heads, head_dim, lead=2, behind=90)
    _check(dtype, q_lens, k_lens, heads, kv_heads, head_dim, causal=False, scale=-0.2)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads", [18, 21, 24, 29, 37, 49, 74, 75])
def test_every_number_of_pieces(dtype, heads):
    _check(dtype, [40], [1500], heads, 1, 64)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [1, 64, 700, 1300])
def test_windows_of_keys_shared_out(dtype, window):
    _check(dtype, [600, 130], [3000, 1700], 2, 1, 64, window=window)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_prompts_whose_keys_are_not_shared_out(dtype):
    _check(dtype, [1500, 700], [1500, 1100], 16, 4, 128)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_nan_among_keys_shared_out(dtype):
    import torch
    q, k = (torch.randn(n, 2, 64, device="cuda").to(getattr(torch, dtype)) for n in (300, 2000))
    q_at, k_at = torch.tensor([0, 300], device="cuda"), torch.tensor([0, 2000], device="cuda")
    want = gh.ctx().prompt_attention(q, k, k, q_at, k_at)[0]
    bad = k.clone()
    bad[1850] = float("nan")   # query 150 and those behind it see the key
    got, status = gh.ctx().prompt_attention(q, bad, k, q_at, k_at)
    assert int(status) == 0 and got[150:].isnan().all() and (got[:150] == want[:150]).all()


def test_a_captured_call_whose_keys_are_shared_out():
    import torch
    ctx = psx.Context(0)
    q, k = (torch.randn(n, 2, 128, device="cuda").bfloat16() for n in (200, 4000))
    q_at, k_at = torch.tensor([0, 200], device="cuda"), torch.tensor([0, 4000], device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):   # (no scratch: nothing has to be called before)
        got, status = ctx.prompt_attention(q, k, k, q_at, k_at)
    for lens in ((200, 4000), (200, 700), (130, 130), (0, 0)):
        q_at[1], k_at[1] = lens
        q.normal_()
        graph.replay()
        want = ctx.prompt_attention(q, k, k, q_at, k_at)[0]
        torch.cuda.synchronize()
        assert int(status) == 0 and (got[:lens[0]] == want[:lens[0]]).all() and not want[:lens[0]].isnan().any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_limit_of_a_wait_is_that_of_a_block(dtype):
    import torch
    ctx = psx.Context(0)
    q, k = (torch.randn(n, 1, 64, device="cuda").to(getattr(torch, dtype)) for n in (1, 400_001))
    at = torch.tensor([0, 1], device="cuda"), torch.tensor([0, 400_001], device="cuda")
    want = ctx.prompt_attention(q, k, k, *at)[0]
    torch.cuda.synchronize()
    ctx.set_wait_limit(150_000)   # the keys' last block comes some 400 microseconds after the first
    got, status = ctx.prompt_attention(q, k, k, *at)
    assert int(status) == 0 and (got == want).all()


# Many groups of rows: a tile takes the heads that share a kv head together, a divisor of them up to 16.
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("heads,kv_heads", [(16, 4), (24, 8), (10, 2), (14, 2), (64, 2), (34, 2), (48, 2), (16, 1)])
def test_heads_of_a_tile(dtype, heads, kv_heads):
    lens = [1, 130, 33, 0, 7, 64, 65, 16, 12, 129] * 3
    longer = [n + (37 * i) % 200 for i, n in enumerate(lens)]
    _check(dtype, lens, lens, heads, kv_heads, 64, lead=1, behind=30)
    _check(dtype, lens, longer, heads, kv_heads, 72, window=50)
    _check(dtype, lens, longer[::-1], heads, kv_heads, 128, causal=False, behind=5)


# Keys 18 nats above the rest whose values are 0: what the rest weigh, 2^-26 each, is all that there is.  fp16 weights are 2^7 at the row's reference
# point: those of e^-18.5 of it are multiples of 2^-24, off by 2^-25, which is 0.026 of them (as 1 at the reference point they would be 0).
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("queries,keys,every,heads", [(3, 8192, 8192, 1), (300, 3000, 60, 1), (200, 1000, 1000, 40)])
def test_weights_far_below_the_largest_count(dtype, queries, keys, every, heads):
    import torch
    rng = np.random.RandomState(keys)
    q, k, v = np.zeros((queries, heads, 64)), np.zeros((keys, 1, 64)), rng.uniform(0.5, 2.0, (keys, 1, 64))
    q[:, :, :2] = 1.0
    k[:, 0, 1] = rng.randint(-4, 5, keys) / 8
    k[::every, 0, 0], v[::every] = 18.0, 0.0
    q, k, v = (_tensor(x, dtype) for x in (q, k, v))
    at, to = torch.tensor([0, queries], device="cuda"), torch.tensor([0, keys], device="cuda")
    got, status = gh.ctx().prompt_attention(q, k, v, at, to, scale=1.0, causal=False)
    want, most, _ = _attention(*(x.double().cpu().numpy() for x in (q, k, v)), at.tolist(), to.tolist(), 1.0, False, 0)
    # (relative to the context, whose terms all have one sign)
    slack = _slack(dtype, most, 1.0, 64, keys) + (2.0 ** -25 / (2.0 ** 7 * np.exp(-18.5)) if dtype == "float16" else 0.0)
    context = got.double().cpu().numpy()
    step = np.maximum(HALF_STEP[dtype] * want, 2.0 ** -25 if dtype == "float16" else 0.0)  # (fp16 below 2^-14: multiples of 2^-24)
    assert int(status) == 0 and (np.abs(context - want) <= slack * want + step).all(), (np.abs(context - want) / want).max()


# Visible scores of -inf.  A softmax over nothing else is NaN, beside finite ones they weigh nothing; a query that sees no key has the context 0.
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("scale", [0.125, -0.125])
@pytest.mark.parametrize("heads,kv_heads,sequences,keys", [(1, 1, 1, 60), (2, 1, 1, 3000), (4, 1, 200, 60)])
def test_scores_of_minus_infinity(dtype, scale, heads, kv_heads, sequences, keys):
    import torch
    far = float("inf") if dtype == "float16" else 2.0 ** 100   # (2^100 has one bf16 part; times 2^100 it is beyond a float)
    q, v = torch.zeros(4 * sequences, heads, 64, device="cuda"), torch.randn(keys * sequences, kv_heads, 64, device="cuda")
    k = torch.zeros_like(v)
    first = torch.arange(sequences, device="cuda") * keys
    k[:, :, :3] = (-1.0 if scale > 0 else 1.0) * min(far, 1e4 if dtype == "float16" else far)
    k[first, :, 1] = k[first + keys - 1, :, 2] = 0.0
    q[1::4, :, 0] = far             # every key
    if dtype != "float16":
        q[2::4, :, 1] = q[3::4, :, 2] = far  # every key but the first, but the last
    q, k, v = (x.to(getattr(torch, dtype)) for x in (q, k, v))
    at, to = torch.arange(sequences + 1, device="cuda") * 4, torch.arange(sequences + 1, device="cuda") * keys
    got, status = gh.ctx().prompt_attention(q, k, v, at, to, scale=scale, causal=False)
    assert int(status) == 0 and got[1::4].isnan().all() and got[0::4].isfinite().all()
    if dtype != "float16":
        for i, of in ((2, first), (3, first + keys - 1)):
            want = v[of].repeat_interleave(heads // kv_heads, 1)
            assert ((got[i::4] - want).abs() <= 2.0 ** -20 * want.abs()).all()
    got = gh.ctx().prompt_attention(q, k, v, at, torch.zeros_like(to), scale=scale, causal=False)[0]
    assert (got == 0).all()


def _plan(dtype, q_lens, heads, kv_heads, head_dim, total_k):
    """(heads of a tile, pieces) by the kernel's rule: as few heads as keep the CTAs to one for an SM, clusters where half of the SMs were idle."""
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles, block = (1, 64) if dtype == "float32" else (2, 128)
    groups = lambda packed: (sum(q_lens) // (tiles * (128 // packed)) + len(q_lens)) * (heads // packed)  # noqa: E731
    packed = 1
    for d in range(1, min(heads // kv_heads, 16) + 1):
        if heads // kv_heads % d == 0:
            packed = d
            if groups(d) <= sms:
                break
    return packed, max(1, min(sms // groups(packed), total_k // block + 1, 8))


# Few groups of rows, each of several heads of a kv head: the CTAs of a cluster share their keys.
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,head_dim", [([1, 20, 7, 13, 3, 18], [3000, 2000, 70, 900, 128, 1], 28, 4, 128),
                                                                   ([1, 20, 7, 13, 3, 18], [90, 20, 57, 13, 83, 18], 28, 4, 64),
                                                                   ([1] * 16, [17 * i for i in range(16)], 10, 2, 72), ([2, 1] * 8, [700, 40] * 8, 20, 2, 64),
                                                                   ([5] * 3 + [0, 130], [1000, 0, 65, 30, 640], 33, 3, 96), ([40, 3], [41, 1500], 91, 7, 128)])
def test_heads_of_a_tile_whose_keys_are_shared_out(dtype, q_lens, k_lens, heads, kv_heads, head_dim):
    import torch
    packed, pieces = _plan(dtype, q_lens, heads, kv_heads, head_dim, sum(k_lens))
    assert packed > 1 and pieces > 1
    _check(dtype, q_lens, k_lens, heads, kv_heads, head_dim, lead=2, behind=9)
    _check(dtype, q_lens, k_lens, heads, kv_heads, head_dim, causal=False, scale=-0.2, behind=80)
    for window in (1, 60, 700):
        _check(dtype, q_lens, k_lens, heads, kv_heads, head_dim, window=window)
    # a key that is not finite reaches the queries of its sequence that see it and their heads, no other
    rng = np.random.RandomState(len(q_lens))
    q_at, k_at = (np.concatenate([[0], np.cumsum(n)]).astype(np.int64) for n in (q_lens, k_lens))
    q, k, v = (_tensor(rng.rand(n[-1], h, head_dim) + 0.1, dtype) for n, h in ((q_at, heads), (k_at, kv_heads), (k_at, kv_heads)))
    at, to = torch.from_numpy(q_at).cuda(), torch.from_numpy(k_at).cuda()
    want = gh.ctx().prompt_attention(q, k, v, at, to)[0]
    longest = int(np.argmax(k_lens))
    for j in (0, k_lens[longest] // 2, k_lens[longest] - 1):
        bad = k.clone()
        bad[k_at[longest] + j, kv_heads - 1] = float("nan")
        got, status = gh.ctx().prompt_attention(q, bad, v, at, to)
        hit = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
        sees = max(j - (k_lens[longest] - q_lens[longest]), 0)
        hit[q_at[longest] + sees:q_at[longest + 1], heads - heads // kv_heads:] = True
        assert int(status) == 0 and got[hit].isnan().all() and (got[~hit] == want[~hit]).all()


def test_scratch_is_as_much_as_the_call_needs_where_more_is_not_free():
    import torch
    # fp32 keys and values take scratch of 1.5 times their bytes; the quarter on top gives way when the device is nearly full
    ctx, positions = psx.Context(0), 400_000
    q, k = torch.randn(2, 8, 128, device="cuda"), torch.randn(positions, 8, 128, device="cuda")
    at, to = torch.tensor([0, 2], device="cuda"), torch.tensor([0, positions], device="cuda")
    other = psx.Context(0)
    want = other.prompt_attention(q, k, k, at, to)[0]
    torch.cuda.synchronize()
    other.close()
    need = 12 * 128 * positions * 8
    few = torch.tensor([0, 40], device="cuda")
    ctx.prompt_attention(q, k[:40], k[:40], at, few)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held = torch.empty(torch.cuda.mem_get_info()[0] - need - need // 8, dtype=torch.uint8, device="cuda")
    got, status = ctx.prompt_attention(q, k, k, at, to)
    assert int(status) == 0 and (got == want).all()
    ctx.close()
    del held
    torch.cuda.empty_cache()
    # not even that: the call says so, and the context stays usable
    ctx = psx.Context(0)
    ctx.prompt_attention(q, k[:40], k[:40], at, few)
    held = torch.empty(torch.cuda.mem_get_info()[0] - need // 8, dtype=torch.uint8, device="cuda")
    with pytest.raises(psx.PsxError) as e:
        ctx.prompt_attention(q, k, k, at, to)
    assert e.value.status == psx.ERR_CUDA
    del held
    torch.cuda.empty_cache()
    got, status = ctx.prompt_attention(q, k, k, at, to)
    assert int(status) == 0 and (got == want).all()


def test_scratch_that_no_capture_has_used_goes_when_it_is_outgrown():
    import torch
    ctx, most = psx.Context(0), 120_000
    q, k = torch.randn(2, 8, 128, device="cuda"), torch.randn(most, 8, 128, device="cuda")
    at = torch.tensor([0, 2], device="cuda")
    ctx.prompt_attention(q, k[:2], k[:2], at, at)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    for positions in range(20_000, most + 1, 10_000):   # a conversation that goes on
        ctx.prompt_attention(q, k[:positions], k[:positions], at, at * (positions // 2))
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] <= 1.25 * 12 * 128 * most * 8 + (64 << 20)   # (and what torch holds of its own)
