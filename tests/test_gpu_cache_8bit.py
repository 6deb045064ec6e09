"""The cache in 8 bits: its writer (psx_b200_store_cache_8bit) bit for bit against a restatement of the format, and attention over
it (psx_b200_decode_attention_8bit) against the formula in double precision.

Tolerance of the attention: a score is off by the rounding of the query (to halves of its power of two: 2^-11 of an element for
fp32's high half, what is left again 2^-11 of that, so 2^-22; bf16 and fp16 queries are exact to 2^-25 of the row's largest),
by the sums of a product of head_dim terms in float and by two factors; the weights by that times the score's size, by 2^-22 of the
exponential and, for bf16 and fp16 contexts, by their rounding to halves, 2^-11 each.  With |s| <= S the context is off by at most
(2 * dS + 2^-11 or 2^-22 + n terms of 2^-24 each in sums that grow like their square root) times the largest value, plus its own
rounding, half a step of its type.  `_tolerance` adds these up."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx

pytestmark = pytest.mark.gpu
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _codes(x):
    """Nearest e4m3 code (ties to even) of numbers within +-448, as its value."""
    x = np.asarray(x, dtype=np.float64)
    size = np.abs(x)
    with np.errstate(all="ignore"):
        exponent = np.maximum(np.floor(np.log2(np.where(size > 0, size, 1))), -6)
    step = 2.0 ** (exponent - 3)
    return np.clip(np.rint(x / step) * step, -448, 448)  # (rint: ties to even; nan stays nan)


def _scale(largest):
    if largest == 0:
        return 2.0 ** -100
    m, e = np.frexp(np.float64(largest))
    return 2.0 ** max(e - 9 + (m > 0.875), -100)


def _store(values, scales, new, offsets, cached, block):
    """values: what the codes stand for / scale, float64 (batch, kv, max_len, d)."""
    values, scales = values.copy(), scales.copy()
    batch, kv_heads, max_len, _ = values.shape
    for b in range(batch):
        n, at = offsets[b + 1] - offsets[b], cached[b]
        if n <= 0 or at < 0 or at + n > max_len:
            continue
        for h in range(kv_heads):
            for i in range(at // block, (at + n - 1) // block + 1):
                low, high = max(at, i * block), min(at + n, (i + 1) * block)
                x = new[offsets[b] + low - at:offsets[b] + high - at, h].astype(np.float64)
                finite = np.abs(x[np.isfinite(x)])
                scale = _scale(finite.max() if finite.size else 0)
                if low > i * block:
                    old = scales[b, h, i]
                    scale = max(scale, old)
                    values[b, h, i * block:low] = _codes(values[b, h, i * block:low] * (old / scale))
                values[b, h, low:high] = _codes(np.clip(x / scale, -448, 448))
                scales[b, h, i] = scale
    return values, scales


def _tensor(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, dtype)).cuda()


def _parts(cache):
    return [x.float().double().cpu().numpy() for x in (cache.key_codes, cache.value_codes)], [x.double().cpu().numpy() for x in (cache.key_scales, cache.value_scales)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("kv_heads,head_dim", [(1, 16), (3, 80), (2, 128), (1, 256)])
def test_what_is_stored(dtype, block, kv_heads, head_dim):
    import torch
    rng = np.random.RandomState(block + head_dim)
    max_len = 150
    cache = psx.Cache8bit.empty(6, kv_heads, max_len, head_dim, block)
    cached = np.zeros(6, dtype=np.int64)
    state = [(np.zeros((6, kv_heads, max_len, head_dim)), np.zeros((6, kv_heads, -(-max_len // block)))) for _ in range(2)]
    # prompts of several lengths, then one position at a time with magnitudes that make scales grow, then rows that do not fit
    for step, counts in enumerate([[0, 1, 15, 64, 100, 150], [1, 1, 1, 1, 1, 0], [3, 17, 1, 0, 33, 0], [1, 1, 1, 1, 17, 1]]):
        offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
        total = int(offsets[-1])
        new = [(rng.randn(total, kv_heads, head_dim) * 2.0 ** rng.randint(-6, 7, (total, 1, 1)) * 4.0 ** step) for _ in range(2)]
        new = [_tensor(x, dtype) for x in new]
        status = gh.ctx().store_cache_8bit(cache, *new, torch.from_numpy(offsets).cuda(), torch.from_numpy(cached).cuda())
        fits = cached + counts <= max_len
        assert status.cpu().tolist() == [0 if f else psx.ROW_CACHE_FULL for f in fits]
        state = [_store(v, s, x.double().cpu().numpy(), offsets, cached, block) for (v, s), x in zip(state, new)]
        codes, scales = _parts(cache)
        for i in range(2):
            assert (scales[i] == state[i][1]).all()
            assert (codes[i] == state[i][0]).all()
        cached = cached + np.where(fits, counts, 0)


def test_one_position_at_a_time_is_as_all_at_once():
    import torch
    rng = np.random.RandomState(5)
    new = [_tensor(rng.uniform(0.5, 8, (40, 2, 32)) * rng.choice([-1, 1], (40, 2, 32)), "float32") for _ in range(2)]  # (no code becomes subnormal)
    one, all_ = (psx.Cache8bit.empty(1, 2, 64, 32, 16) for _ in range(2))
    for i in range(40):
        gh.ctx().store_cache_8bit(one, new[0][i:i + 1], new[1][i:i + 1], torch.tensor([0, 1], device="cuda"), torch.tensor([i], device="cuda"))
    gh.ctx().store_cache_8bit(all_, *new, torch.tensor([0, 40], device="cuda"), torch.tensor([0], device="cuda"))
    for a, b in zip(_parts(one), _parts(all_)):
        assert (a[1] == b[1]).all()
        # codes were rounded at a finer scale first: a second rounding may move a tie, by one step of the coarser scale
        assert (np.abs(a[0] - b[0]) <= 2.0 ** -3 * np.maximum(np.abs(b[0]), 2.0 ** -6)).all()


def test_numbers_that_are_not_finite_zeros_and_extremes():
    import torch
    x = np.zeros((64, 1, 16), dtype=np.float32)
    x[0, 0, :4] = [np.nan, np.inf, -np.inf, 100.0]     # the scale is that of 100
    x[16, 0, :3] = [3.4e38, -3.4e38, 1e38]
    x[32, 0, :3] = [1e-45, 1e-38, 0]
    x[48, 0, :2] = [448.0, 449.0]                      # 448 * 2^0 does not reach 449
    cache = psx.Cache8bit.empty(1, 1, 64, 16, 16)
    gh.ctx().store_cache_8bit(cache, _tensor(x, "float32"), _tensor(x, "float32"), torch.tensor([0, 64], device="cuda"), torch.tensor([0], device="cuda"))
    codes, scales = _parts(cache)
    assert scales[0][0, 0].tolist() == [2.0 ** -2, _scale(np.float32(3.4e38)), 2.0 ** -100, 2.0]
    got = codes[0][0, 0] * scales[0][0, 0].repeat(16)[:, None]
    assert np.isnan(got[0, 0]) and got[0, 1:4].tolist() == [112.0, -112.0, 96.0]  # (400 lies between 384 and 416: to even)
    want = _codes(x[:, 0].astype(np.float64)[1:] / scales[0][0, 0].repeat(16)[1:, None])
    assert (codes[0][0, 0][1:] == want).all()


@pytest.mark.parametrize("offsets,cached,status", [([0, 4, 2, 9], [0, 0, 0], [0, 65, 0]), ([-1, 2, 4, 10], [0, 0, 0], [65, 0, 65]), ([0, 2, 4, 6], [-1, 30, 31], [65, 0, 64]),
                                                   ([0, 9, 9, 9], [33, 32, 2 ** 62], [64, 0, 64])])
def test_rows_whose_numbers_make_no_sense_are_left_alone(offsets, cached, status):
    import torch
    rng = np.random.RandomState(1)
    new = [_tensor(rng.randn(9, 1, 16), "float32") for _ in range(2)]
    cache = psx.Cache8bit.empty(3, 1, 32, 16, 16)
    got = gh.ctx().store_cache_8bit(cache, *new, torch.tensor(offsets, device="cuda"), torch.tensor(cached, device="cuda"))
    assert got.cpu().tolist() == status
    fine = [c if s == 0 else 33 for c, s in zip(cached, status)]
    values, scales = _store(np.zeros((3, 1, 32, 16)), np.zeros((3, 1, 2)), new[0].double().cpu().numpy(), offsets, fine, 16)
    codes, found = _parts(cache)
    assert (codes[0] == values).all() and (found[0] == scales).all()


def test_slices_of_a_wider_projection():
    import torch
    rng = np.random.RandomState(2)
    wide = _tensor(rng.randn(20, 7, 32), "bfloat16")
    keys, values = wide[:, 3:5], wide[:, 5:7]
    a, b = (psx.Cache8bit.empty(2, 2, 32, 32, 16) for _ in range(2))
    offsets, cached = torch.tensor([0, 9, 20], device="cuda"), torch.tensor([1, 2], device="cuda")
    gh.ctx().store_cache_8bit(a, keys, values, offsets, cached)
    gh.ctx().store_cache_8bit(b, keys.contiguous(), values.contiguous(), offsets, cached)
    for x, y in zip(_parts(a), _parts(b)):
        assert all((u == v).all() for u, v in zip(x, y))


# ---- attention ------------------------------------------------------------------------------------------------------------
def _cache(rng, batch, kv_heads, max_len, head_dim, block, lengths, spread=2):
    """Random codes and scales; NaN codes where no position is."""
    import torch
    parts = []
    for _ in range(2):
        codes = _codes(np.clip(rng.randn(batch, kv_heads, max_len, head_dim) * 100, -448, 448))
        for b, n in enumerate(lengths):
            codes[b, :, max(n, 0):] = np.nan
        scales = 2.0 ** rng.randint(-7 - spread, -7 + spread + 1, (batch, kv_heads, -(-max_len // block))) * rng.choice([1.0, 1.25], (batch, kv_heads, -(-max_len // block)))
        parts += [torch.from_numpy(codes.astype(np.float32)).cuda().to(torch.float8_e4m3fn), torch.from_numpy(scales.astype(np.float32)).cuda()]
    return psx.Cache8bit(*parts, block=block)


def _attention(q, cache, lengths, scale, causal, window):
    """(context, largest |score|, largest value), double precision."""
    codes, scales = _parts(cache)
    keys, values = (c * s.repeat(cache.block, 2)[:, :, :cache.max_len, None] for c, s in zip(codes, scales))
    batch, heads, q_len, head_dim = q.shape
    group = heads // cache.kv_heads
    out, most, value = np.zeros(q.shape), 0.0, 0.0
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), cache.max_len)
        for i in range(q_len):
            p = n - q_len + i
            last = p if causal else n - 1
            first = max(p - window + 1, 0) if causal and window else 0
            if last < first:
                continue
            for h in range(heads):
                k, v = keys[b, h // group, first:last + 1], values[b, h // group, first:last + 1]
                s = (k @ q[b, h, i]) * scale
                w = np.exp(s - s.max())
                out[b, h, i] = (w / w.sum()) @ v
                most, value = max(most, np.abs(k).max() * np.abs(q[b, h, i]).sum() * scale, np.abs(s).max()), max(value, np.abs(v).max())
    return out, most, value


def _tolerance(dtype, most, value, head_dim, n):
    """most: the largest sum of a score's terms' sizes."""
    score = most * ((2.0 ** -22 if dtype == "float32" else 2.0 ** -24) + (np.sqrt(head_dim) + 4) * 2.0 ** -23)
    weight = 2 * score + 2.0 ** -21 + (2.0 ** -11 if dtype != "float32" else 2.0 ** -21) + (np.sqrt(n) + 8) * 2.0 ** -23
    return weight * value, HALF_STEP[dtype]


def _check(dtype, batch, heads, kv_heads, q_len, head_dim, max_len, lengths, block=32, causal=True, window=0, seed=0, scale=None, ctx=None):
    import torch
    rng = np.random.RandomState(seed + head_dim + max_len)
    cache = _cache(rng, batch, kv_heads, max_len, head_dim, block, lengths)
    q = _tensor(rng.randn(batch, heads, q_len, head_dim), dtype)
    got = (ctx or gh.ctx()).decode_attention_8bit(q, cache, torch.tensor(lengths, device="cuda"), scale=scale, causal=causal, window=window)
    torch.cuda.synchronize()
    for codes in (cache.key_codes, cache.value_codes):  # (for the restatement)
        codes.copy_(codes.float().nan_to_num(0.0).to(torch.float8_e4m3fn))
    scale = head_dim ** -0.5 if scale is None else scale
    want, most, value = _attention(q.double().cpu().numpy(), cache, lengths, scale, causal, window)
    slack, step = _tolerance(dtype, most, value, head_dim, max_len)
    error = np.abs(got.double().cpu().numpy() - want)
    assert np.isfinite(error).all()
    assert (error <= slack + step * np.abs(want)).all(), (error.max(), slack)
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("heads,kv_heads,q_len,head_dim", [(1, 1, 1, 16), (8, 2, 1, 64), (4, 4, 1, 128), (16, 2, 1, 128), (16, 1, 1, 96), (6, 2, 3, 80), (5, 1, 2, 48),
                                                           (2, 2, 8, 64), (8, 1, 2, 128), (8, 1, 1, 256), (4, 2, 4, 160)])
def test_head_layouts_and_lengths(dtype, heads, kv_heads, q_len, head_dim):
    lengths = [300, 1, 16, 33, 0, 64, 257, 5]
    _check(dtype, 8, heads, kv_heads, q_len, head_dim, 301, lengths, block=16 << (heads % 3))


@pytest.mark.parametrize("length", [1, 31, 32, 33, 255, 256, 257, 1000, 4097])
@pytest.mark.parametrize("block", [16, 32, 64])
def test_one_row_of_every_length(length, block):
    _check("bfloat16", 1, 8, 2, 1, 128, length + 3, [length], block=block, seed=length)


@pytest.mark.parametrize("causal,window,q_len", [(False, 0, 4), (False, 7, 2), (True, 1, 1), (True, 7, 4), (True, 100, 2), (True, 33, 1), (True, 2 ** 40, 2)])
def test_masks(causal, window, q_len):
    _check("float32", 5, 4, 2, q_len, 64, 400, [400, 399, 130, 2, 0], causal=causal, window=window, seed=window % 97)


def test_lengths_beyond_the_cache_count_as_the_nearer_end():
    _check("float32", 3, 2, 1, 2, 64, 96, [2 ** 50, -4, 97])


def test_few_rows_share_the_gpu_and_many_rows_fill_it():
    _check("bfloat16", 1, 8, 8, 1, 128, 30000, [29999], seed=1, block=64)        # pieces of one row over all blocks
    _check("bfloat16", 40, 16, 8, 1, 64, 700, list(np.random.RandomState(0).randint(0, 701, 40)), seed=2)
    _check("float32", 3, 2, 2, 1, 64, 5000, [5000, 3, 4000], seed=3)
    _check("float16", 1, 16, 1, 1, 64, 160000, [160000], seed=4)                         # as many pieces as a pair can have


def test_scores_and_scales_of_every_size():
    import torch
    # block scales from 2^-100 to 2^20 side by side, scores of +-1000: the weights of the small blocks are not lost where the large
    # ones' scores are low
    rng = np.random.RandomState(4)
    cache = _cache(rng, 1, 1, 128, 64, 16, [128])
    cache.key_scales[:] = 1.0 / 64
    cache.value_scales[0, 0] = torch.tensor([2.0 ** e for e in (20, -100, 0, -20, 10, -3, 0, -60)])
    q = _tensor(rng.randn(1, 1, 1, 64) * 3, "float32")
    got = gh.ctx().decode_attention_8bit(q, cache, torch.tensor([128], device="cuda"), scale=0.5).double().cpu().numpy()
    want, most, _ = _attention(q.double().cpu().numpy(), cache, [128], 0.5, True, 0)
    codes, scales = _parts(cache)
    s = (codes[0][0, 0] / 64) @ q.double().cpu().numpy()[0, 0, 0] * 0.5
    w = np.exp(s - s.max())
    size = (w / w.sum()) @ np.abs(codes[1][0, 0] * scales[1][0, 0].repeat(16)[:, None])  # what the terms add up to without their signs
    slack, step = _tolerance("float32", most, 1.0, 64, 128)
    assert (np.abs(got[0, 0, 0] - want[0, 0, 0]) <= slack * size + step * np.abs(want[0, 0, 0])).all()
    cache.value_scales.zero_()
    assert (gh.ctx().decode_attention_8bit(q, cache, torch.tensor([128], device="cuda")) == 0).all()


def test_the_same_call_gives_the_same_bits_and_graphs_replay():
    import torch
    ctx = psx.Context(0)
    rng = np.random.RandomState(6)
    cache = _cache(rng, 2, 2, 3000, 64, 32, [3000, 1777])
    q, lengths = _tensor(rng.randn(2, 8, 1, 64), "bfloat16"), torch.tensor([3000, 1777], device="cuda")
    first = ctx.decode_attention_8bit(q, cache, lengths).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ctx.decode_attention_8bit(q, cache, lengths)
    wide = _cache(rng, 70, 4, 64, 64, 32, [64] * 70)
    ctx.decode_attention_8bit(_tensor(rng.randn(70, 4, 1, 64), "bfloat16"), wide, torch.full((70,), 64, device="cuda"))  # (more pairs: the scratch grows)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (out == first).all()
    lengths.copy_(torch.tensor([5, 1200]))
    graph.replay()
    torch.cuda.synchronize()
    assert (out == psx.Context(0).decode_attention_8bit(q, cache, lengths)).all()


def test_as_many_rows_as_there_may_be():
    import torch
    batch = 4096
    rng = np.random.RandomState(13)
    cache = psx.Cache8bit.empty(batch, 1, 48, 16, 16)
    counts = rng.randint(0, 9, batch)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    new = [_tensor(rng.randn(int(offsets[-1]), 1, 16), "float16") for _ in range(2)]
    cached = np.zeros(batch, dtype=np.int64)
    status = gh.ctx().store_cache_8bit(cache, *new, torch.from_numpy(offsets).cuda(), torch.from_numpy(cached).cuda())
    assert (status == 0).all()
    codes, scales = _parts(cache)
    for i in range(2):
        want = _store(np.zeros((batch, 1, 48, 16)), np.zeros((batch, 1, 3)), new[i].double().cpu().numpy(), offsets, cached, 16)
        assert (codes[i] == want[0]).all() and (scales[i] == want[1]).all()
    q = _tensor(rng.randn(batch, 2, 1, 16), "float16")
    got = gh.ctx().decode_attention_8bit(q, cache, torch.from_numpy(counts.astype(np.int64)).cuda()).double().cpu().numpy()
    want, most, value = _attention(q.double().cpu().numpy(), cache, counts, 0.25, True, 0)
    slack, step = _tolerance("float16", most, value, 16, 9)
    assert (np.abs(got - want) <= slack + step * np.abs(want)).all()


def test_refusals():
    import torch
    ctx = gh.ctx()
    cache = psx.Cache8bit.empty(2, 2, 64, 64, 32)
    lengths = torch.tensor([4, 4], device="cuda")

    def decode(heads, q_len, cache=cache, dtype="float32", **kw):
        return ctx.decode_attention_8bit(_tensor(np.zeros((2, heads, q_len, cache.head_dim)), dtype), cache, lengths, **kw)

    for status, call in ((psx.ERR_BAD_ARGUMENT, lambda: decode(3, 1)), (psx.ERR_UNSUPPORTED, lambda: decode(34, 1)), (psx.ERR_UNSUPPORTED, lambda: decode(4, 9)),
                         (psx.ERR_BAD_ARGUMENT, lambda: decode(4, 1, window=-1)), (psx.ERR_UNSUPPORTED, lambda: decode(34, 1, psx.Cache8bit.empty(2, 2, 64, 144, 32))),
                         (psx.ERR_UNSUPPORTED, lambda: decode(2, 1, psx.Cache8bit.empty(2, 2, 64, 40, 32))), (psx.ERR_UNSUPPORTED, lambda: decode(2, 1, psx.Cache8bit.empty(2, 2, 64, 64, 8))),
                         (psx.ERR_UNSUPPORTED, lambda: decode(2, 1, psx.Cache8bit.empty(2, 2, 64, 272, 32)))):
        with pytest.raises(psx.PsxError) as e:
            call()
        assert e.value.status == status
    with pytest.raises(TypeError):
        ctx.decode_attention_8bit(torch.zeros(2, 2, 1, 64, dtype=torch.float64, device="cuda"), cache, lengths)
    with pytest.raises(ValueError):
        ctx.decode_attention_8bit(torch.zeros(2, 2, 1, 64, device="cuda"), cache, lengths.int())
    with pytest.raises(ValueError):
        psx.Cache8bit(cache.key_codes, cache.key_scales, cache.value_codes[:, :, :32], cache.value_scales)
    new, offsets = torch.zeros(3, 2, 64, device="cuda"), torch.tensor([0, 1, 3], device="cuda")
    with pytest.raises(ValueError):
        ctx.store_cache_8bit(cache, new[:, :1], new[:, :1], offsets, lengths)
    with pytest.raises(ValueError):
        ctx.store_cache_8bit(cache, new, new, offsets[:2], lengths)
    with pytest.raises(psx.PsxError) as e:  # a base that is not on a boundary of four elements
        flat = torch.zeros(3 * 128 + 4, device="cuda")[1:3 * 128 + 1].view(3, 2, 64)
        ctx.store_cache_8bit(cache, flat, flat, offsets, lengths)
    assert e.value.status == psx.ERR_BAD_ARGUMENT
    too_many = psx.Cache8bit.empty(4097, 1, 16, 16, 16)
    with pytest.raises(psx.PsxError) as e:
        ctx.decode_attention_8bit(torch.zeros(4097, 1, 1, 16, device="cuda"), too_many, torch.ones(4097, dtype=torch.int64, device="cuda"))
    assert e.value.status == psx.ERR_UNSUPPORTED


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("heads,kv_heads,q_len,head_dim", [(16, 2, 2, 256), (9, 1, 1, 144), (16, 1, 1, 256), (2, 2, 11, 208), (6, 2, 5, 176)])
def test_more_than_eight_query_rows_beyond_128_dimensions(dtype, heads, kv_heads, q_len, head_dim):
    _check(dtype, 7, heads, kv_heads, q_len, head_dim, 1500, [1500, 1, 16, 33, 0, 640, 5], block=32)
    _check(dtype, 2, heads, kv_heads, q_len, head_dim, 90, [90, 70], block=16, window=9, causal=True)
    _check(dtype, 100, heads, kv_heads, q_len, head_dim, 40, [40 - i % 37 for i in range(100)], block=64, causal=False)


# Positions that no query of a row sees are not read: neither their codes nor their scales, ahead of a window or behind the length.
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("head_dim,heads,q_len,window", [(64, 2, 1, 7), (128, 4, 2, 40), (96, 2, 1, 1), (256, 2, 3, 17)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_scales_and_codes_that_no_query_sees_are_not_read(dtype, block, head_dim, heads, q_len, window, what):
    import torch
    rng = np.random.RandomState(block + head_dim)
    lengths = [130, 113, 200, 48, 3, 161, 0]
    cache = _cache(rng, len(lengths), 2, 210, head_dim, block, lengths)
    q, seen_to = _tensor(rng.randn(len(lengths), heads, q_len, head_dim), dtype), torch.tensor(lengths, device="cuda")
    want = gh.ctx().decode_attention_8bit(q, cache, seen_to, window=window)
    assert want.isfinite().all()
    for row, n in enumerate(lengths):
        seen = max(n - q_len - window + 1, 0)  # the first position that a query sees
        for codes, scales in ((cache.key_codes, cache.key_scales), (cache.value_codes, cache.value_scales)):
            codes[row, :, :seen].copy_(torch.full_like(codes[row, :, :seen].float(), float("nan")).to(codes.dtype))
            scales[row, :, :seen // block] = what
            scales[row, :, -(-n // block):] = what
    got = gh.ctx().decode_attention_8bit(q, cache, seen_to, window=window)
    assert (got == want).all()


def _check_by_size(got, q, cache, lengths, scale, dtype):
    """Relative to what a context's terms add up to without their signs, not to the largest value."""
    want, most, _ = _attention(q.double().cpu().numpy(), cache, lengths, scale, True, 0)
    bare = psx.Cache8bit(cache.key_codes, cache.key_scales, cache.value_codes.float().abs().to(cache.value_codes.dtype), cache.value_scales, block=cache.block)
    size, _, _ = _attention(q.double().cpu().numpy(), bare, lengths, scale, True, 0)
    slack, step = _tolerance(dtype, most, 1.0, cache.head_dim, max(lengths))
    error = np.abs(got.double().cpu().numpy() - want)
    assert (error <= slack * size + step * np.abs(want)).all(), (error / size).max()


# A first position far above the rest whose value is 0: what the rest weigh, 2^-26 each, is all that there is.  Weights are halves of at
# most 2^15 with 11 bits down to 2^-14, 2^-29 of the largest.
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,length,every", [(1, 8192, 8192), (1, 4000, 32), (40, 1000, 32), (300, 500, 500)])
def test_weights_far_below_the_largest_count(dtype, rows, length, every):
    import torch
    rng = np.random.RandomState(length)
    keys, values = np.zeros((rows, 1, length, 64)), _codes(rng.uniform(-300, 300, (rows, 1, length, 64)))
    keys[:, :, :, 1] = _codes(rng.randn(rows, 1, length) * 0.5)
    keys[:, :, ::every, 0] = 18.0                      # 18 nats above the others
    values[:, :, ::every] = 0.0
    blocks = -(-length // 32)
    parts = [t for x in (keys, values) for t in (torch.from_numpy(x.astype(np.float32)).cuda().to(torch.float8_e4m3fn), torch.ones(rows, 1, blocks, device="cuda"))]
    cache = psx.Cache8bit(*parts, block=32)
    q = torch.zeros(rows, 2, 1, 64, device="cuda", dtype=getattr(torch, dtype))
    q[..., :2] = 1.0
    got = gh.ctx().decode_attention_8bit(q, cache, torch.full((rows,), length, device="cuda"), scale=1.0)
    _check_by_size(got, q, cache, [length] * rows, 1.0, dtype)


def test_values_of_zero_and_of_every_scale():
    import torch
    # blocks of zeros have the scale 2^-100, whose weights are the largest floats; blocks of 1e36 the smallest
    rng = np.random.RandomState(2)
    cache = _cache(rng, 2, 1, 40000, 16, 16, [40000, 40000])
    cache.key_scales.fill_(2.0 ** -8)
    cache.value_scales.fill_(2.0 ** -100)
    cache.value_codes[0].copy_(torch.zeros_like(cache.value_codes[0].float()).to(cache.value_codes.dtype))
    q = _tensor(rng.randn(2, 1, 1, 16), "float32")
    n = torch.tensor([40000, 40000], device="cuda")
    got = gh.ctx().decode_attention_8bit(q, cache, n)
    assert (got[0] == 0).all()
    # (the context has some 2^-95: values of a scale below 2^-82 have weights below 2^15, by 2^18 here, so 2^-3 at most and halves of 2^-25)
    want, most, _ = _attention(q.double().cpu().numpy(), cache, [40000, 40000], 0.25, True, 0)
    slack, step = _tolerance("float32", most, 448 * 2.0 ** -100, 16, 40000)
    assert (np.abs(got[1].double().cpu().numpy() - want[1]) <= slack + 448 * 2.0 ** -122 + step * np.abs(want[1])).all()
    cache.value_scales.fill_(2.0 ** 110)
    got = gh.ctx().decode_attention_8bit(q, cache, n)
    want, most, value = _attention(q.double().cpu().numpy(), cache, [40000, 40000], 0.25, True, 0)
    slack, step = _tolerance("float32", most, value, 16, 40000)
    assert (np.abs(got.double().cpu().numpy() - want) <= slack + step * np.abs(want)).all()


# Elements of a query far below its largest: the keys are 0 where that is.  Queries are brought to 2^14, so that what is left of an
# element of 2^-17 of the largest has 22 bits in two halves, and one of 2^-28 has 11 in one.
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 14, 2.0 ** 17])
@pytest.mark.parametrize("head_dim", [64, 256])
def test_elements_of_a_query_far_below_its_largest_count(dtype, ratio, head_dim):
    import torch
    rng = np.random.RandomState(head_dim)
    cache = _cache(rng, 2, 1, 300, head_dim, 32, [300, 299])
    cache.key_scales.fill_(1.0 / 64)
    cache.key_codes.view(torch.uint8)[..., 5] = 0
    x = np.where(rng.rand(2, 2, 1, head_dim) < 0.5, -1.0, 1.0) * rng.uniform(1, 2, (2, 2, 1, head_dim))
    x[..., 5] = ratio
    q, n = _tensor(x, dtype), torch.tensor([300, 299], device="cuda")
    got = gh.ctx().decode_attention_8bit(q, cache, n, scale=1.0)
    plain = q.clone()
    plain[..., 5] = 0
    cache.value_codes.copy_(cache.value_codes.float().nan_to_num(0.0).to(cache.value_codes.dtype))
    cache.key_codes.copy_(cache.key_codes.float().nan_to_num(0.0).to(cache.key_codes.dtype))
    want, _, value = _attention(plain.double().cpu().numpy(), cache, [300, 299], 1.0, True, 0)
    codes, scales = _parts(cache)
    most = max((np.abs(codes[0][b, 0]) / 64 @ np.abs(plain.double().cpu().numpy()[b].reshape(2, -1).T)).max() for b in range(2))
    slack, step = _tolerance(dtype, most, value, head_dim, 300)
    error = np.abs(got.double().cpu().numpy() - want)
    assert (error <= slack + step * np.abs(want)).all(), (error.max(), slack)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("exponent", [100, 115, 119, 125])
def test_large_queries_over_small_keys(dtype, exponent):
    import torch
    rng = np.random.RandomState(exponent)
    cache = _cache(rng, 2, 1, 200, 64, 32, [200, 200])
    cache.key_scales.fill_(2.0 ** -100)
    q, scale = _tensor(np.clip(rng.randn(2, 2, 1, 64), -3.9, 3.9) * 2.0 ** exponent, dtype), 2.0 ** (92 - exponent)
    got = gh.ctx().decode_attention_8bit(q, cache, torch.tensor([200, 200], device="cuda"), scale=scale)
    want, most, value = _attention(q.double().cpu().numpy(), cache, [200, 200], scale, True, 0)
    slack, step = _tolerance(dtype, most, value, 64, 200)
    assert (np.abs(got.double().cpu().numpy() - want) <= slack + step * np.abs(want)).all()


@pytest.mark.parametrize("length", [1, 40, 3000])
def test_scores_that_are_all_minus_infinity_are_not_an_empty_row(length):
    import torch
    # an infinite query against keys of the other sign: softmax of nothing but -inf is NaN; a query that sees nothing has the context 0
    rng = np.random.RandomState(length)
    cache = _cache(rng, 3, 1, length, 64, 16, [length] * 3)
    cache.key_codes[..., 3] = cache.key_codes[..., 3].float().abs().clamp(min=1.0).neg().to(cache.key_codes.dtype)
    q = torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    q[1, 0, 1, 3] = float("inf")
    got = gh.ctx().decode_attention_8bit(q, cache, torch.tensor([length, length, 0], device="cuda"))
    assert got[1, 0, 1].isnan().all() and got[0].isfinite().all() and (got[2] == 0).all()
    assert got[1, 0, 0].isfinite().all() and (length > 1 or (got[1, 0, 0] == 0).all())
