"""Attention over a cache in pages (psx_b200_decode_attention_pages) against the formula in double precision.

Tolerance.  Scores: bf16 and fp16 products are exact, fp32's are off by 2^-21 of a term (what each factor's two numbers leave, 2^-23 and
2^-23, and the product of the smaller parts, 2^-22); a sum over head_dim / 8 instructions and the factor by 2^-23 of the sum of the terms' sizes
for each of them, four more for the scale and the difference to the maximum.  Weights: twice that, 2^-21 of the exponential, and what their two numbers leave: bf16 2^-18, fp16
2^-22 and 2^-38 of the largest, fp32 as above.  Sums over n positions: n / 64 instructions of one warp after the other and the joins, 2^-23 each.  The sum of
these times the largest value, and half a step of the context's type."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx

pytestmark = pytest.mark.gpu
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _numbers(t):
    return t.double().cpu().numpy()


def _tensor(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, dtype)).cuda()


def _cache(rng, dtype, lengths, kv_heads, head_dim, size, max_pages=None, spare=3):
    """Pages scattered over a pool that holds NaN wherever no position is."""
    import torch
    counts = [-(-max(n, 0) // size) for n in lengths]
    max_pages = max_pages or max(1, max(counts))
    num_pages = sum(counts) + spare
    order = rng.permutation(num_pages)
    table = np.full((len(lengths), max_pages), -7, dtype=np.int32)
    references = np.zeros(num_pages, dtype=np.int32)
    pools = [np.full((num_pages, kv_heads, size, head_dim), np.nan, dtype=np.float32) for _ in range(2)]
    at = 0
    for b, n in enumerate(lengths):
        for i in range(counts[b]):
            page = order[at]
            at += 1
            table[b, i], references[page] = page, 1
            filled = min(size, n - i * size)
            for pool in pools:
                pool[page, :, :filled] = rng.randn(kv_heads, filled, head_dim)
    cuda = lambda x: torch.from_numpy(x).cuda()
    book = psx.PageTable(cuda(table), torch.tensor(lengths, device="cuda"), cuda(references), size)
    return psx.PagedCache(book, *[_tensor(p, dtype) for p in pools])


def _attention(q, cache, q_len, scale, causal, window):
    """(context, largest sum of a score's terms' sizes, largest value), double precision."""
    table, size = cache.table.pages.cpu().numpy(), cache.table.page_size
    keys, values = _numbers(cache.key_pages), _numbers(cache.value_pages)
    heads = q.shape[1]
    group = heads // cache.kv_heads
    out, most, value = np.zeros(q.shape), 0.0, 0.0
    for b, n in enumerate(cache.table.lengths.tolist()):
        n = min(max(n, 0), cache.table.max_pages * size)
        pages = table[b, :-(-n // size)]
        for h in range(heads):
            for i in range(q_len):
                p = n - q_len + i
                last = p if causal else n - 1
                first = max(p - window + 1, 0) if causal and window else 0
                if last < first:
                    continue
                k, v = (np.concatenate([x[page, h // group] for page in pages])[first:last + 1] for x in (keys, values))
                one = q[b * q_len + i, h]
                s = (k @ one) * scale
                w = np.exp(s - s.max())
                out[b * q_len + i, h] = (w / w.sum()) @ v
                most, value = max(most, (np.abs(k) @ np.abs(one)).max() * abs(scale)), max(value, np.abs(v).max())
    return out, most, value


def _slack(dtype, most, value, head_dim, n):
    score = most * ((2.0 ** -21 if dtype == "float32" else 0.0) + (head_dim / 8 + 4) * 2.0 ** -23)
    left = {"float32": 2.0 ** -21, "bfloat16": 2.0 ** -18, "float16": 2.0 ** -22 + n * 2.0 ** -38}[dtype]
    return (2 * score + 2.0 ** -21 + left + (n / 64 + 16) * 2.0 ** -23) * value


def _near(got, want, dtype, slack):
    error = np.abs(_numbers(got) - want)
    assert np.isfinite(error).all()
    assert (error <= slack + HALF_STEP[dtype] * np.abs(want)).all(), (error.max(), slack)


def _check(dtype, heads, kv_heads, q_len, head_dim, lengths, size, causal=True, window=0, seed=0, scale=None, ctx=None, max_pages=None):
    rng = np.random.RandomState(seed + head_dim + len(lengths))
    cache = _cache(rng, dtype, lengths, kv_heads, head_dim, size, max_pages)
    q = _tensor(rng.randn(len(lengths) * q_len, heads, head_dim), dtype)
    got = (ctx or gh.ctx()).decode_attention_pages(q, cache, q_len=q_len, scale=scale, causal=causal, window=window)
    want, most, value = _attention(_numbers(q), cache, q_len, head_dim ** -0.5 if scale is None else scale, causal, window)
    _near(got, want, dtype, _slack(dtype, most, value, head_dim, max(lengths)))
    return got, q, cache


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("heads,kv_heads,q_len,head_dim", [(1, 1, 1, 8), (8, 2, 1, 64), (4, 4, 1, 128), (16, 2, 1, 128), (16, 1, 1, 96), (6, 2, 3, 80), (5, 1, 2, 48),
                                                           (2, 2, 8, 64), (8, 1, 2, 128), (8, 1, 1, 256), (4, 2, 4, 160), (16, 1, 1, 200), (3, 3, 5, 72)])
@pytest.mark.parametrize("size", [16, 32, 64, 128])
def test_head_layouts_and_lengths(dtype, heads, kv_heads, q_len, head_dim, size):
    _check(dtype, heads, kv_heads, q_len, head_dim, [300, 1, 16, 33, 0, 64, 257, 5], size)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 63, 64, 65, 255, 256, 1000, 4097])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_one_row_of_every_length(length, dtype):
    _check(dtype, 8, 2, 1, 128, [length], 32, seed=length)
    _check(dtype, 8, 2, 1, 128, [length], 16, seed=length, max_pages=1 << 14)  # (a table for far more)


@pytest.mark.parametrize("causal,window,q_len", [(False, 0, 4), (False, 7, 2), (True, 1, 1), (True, 7, 4), (True, 100, 2), (True, 33, 1), (True, 2 ** 40, 2), (True, 16, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_masks(causal, window, q_len, dtype):
    _check(dtype, 4, 2, q_len, 64, [400, 399, 130, 2, 0, 1, 17], 16, causal=causal, window=window, seed=window % 97)


def test_few_rows_share_the_gpu_and_many_rows_fill_it():
    _check("bfloat16", 8, 8, 1, 128, [29999], 64, seed=1)
    _check("bfloat16", 16, 8, 1, 64, np.random.RandomState(0).randint(0, 701, 40).tolist(), 16, seed=2)
    _check("float32", 2, 2, 1, 64, [5000, 3, 4000], 128, seed=3)
    _check("float16", 16, 1, 1, 64, [160000], 64, seed=4)
    _check("bfloat16", 4, 4, 1, 64, [9000] + [10] * 300, 32, seed=5)
    _check("float32", 8, 1, 2, 256, [3000, 20000], 32, seed=6)


def test_lengths_beyond_the_table_count_as_the_nearer_end():
    import torch
    rng = np.random.RandomState(7)
    cache = _cache(rng, "float32", [96, 96, 96], 1, 64, 32)
    q = _tensor(rng.randn(6, 2, 64), "float32")
    whole = gh.ctx().decode_attention_pages(q, cache, q_len=2)
    cache.table.lengths.copy_(torch.tensor([2 ** 50, -4, 97]))
    got = gh.ctx().decode_attention_pages(q, cache, q_len=2)
    assert (got[:2] == whole[:2]).all() and (got[4:] == whole[4:]).all() and (got[2:4] == 0).all()


def test_rows_that_share_pages():
    import torch
    rng = np.random.RandomState(8)
    ctx = gh.ctx()
    table = psx.PageTable.empty(6, 12, 40, 16)
    cache = psx.PagedCache(table, *[torch.full((40, 2, 16, 64), float("nan"), device="cuda") for _ in range(2)])
    offsets, first = torch.tensor([0, 100, 100, 100, 170, 170, 170], device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    counts = offsets.diff()
    k, v = (_tensor(rng.randn(170, 2, 64), "float32") for _ in range(2))
    assert not ctx.extend_pages(table, counts, cache.pools()).any()
    ctx.rotate_heads(k, k, v, offsets=offsets, first=first, cache=cache)
    ctx.fork_pages(table, torch.tensor([[0, 0, 0], [0, 0, 0]], device="cuda"))
    one = torch.ones(6, dtype=torch.int64, device="cuda")
    for step in range(20):
        before = table.lengths.clone()
        assert not ctx.extend_pages(table, one, cache.pools()).any()
        k1, v1 = (_tensor(rng.randn(6, 2, 64), "float32") for _ in range(2))
        ctx.rotate_heads(k1, k1, v1, offsets=torch.arange(7, device="cuda"), first=before, cache=cache)
        k, v = torch.cat([k, k1]), torch.cat([v, v1])
    q = _tensor(rng.randn(6, 8, 64), "float32")
    got = _numbers(ctx.decode_attention_pages(q, cache))
    want, most, value = _attention(_numbers(q), cache, 1, 0.125, True, 0)
    _near(torch.from_numpy(got), want, "float32", _slack("float32", most, value, 64, 120))
    # and from the positions that went in, without any page
    keys, values = _numbers(k), _numbers(v)
    for b in range(6):
        mine = list(range(0, 100) if b < 3 else range(100, 170)) + [170 + 6 * s + b for s in range(20)]
        for h in range(8):
            s = keys[mine, h // 4] @ _numbers(q)[b, h] * 0.125
            w = np.exp(s - s.max())
            assert np.abs((w / w.sum()) @ values[mine, h // 4] - got[b, h]).max() <= _slack("float32", most, value, 64, 120) + 2.0 ** -24 * value


def test_pages_that_are_none():
    import torch
    rng = np.random.RandomState(9)
    for dtype in ("float32", "bfloat16", "float16"):
        cache = _cache(rng, dtype, [70, 40, 20], 2, 64, 16)
        q = _tensor(rng.randn(3, 4, 64), dtype)
        whole = gh.ctx().decode_attention_pages(q, cache)
        for bad in (-1, cache.table.num_pages, 2 ** 31 - 1, -2 ** 31):
            cache.table.pages[1, 1] = bad
            cache.table.pages[2, 0] = cache.table.pages[2, 1] = bad
            got = gh.ctx().decode_attention_pages(q, cache)
            assert (got[0] == whole[0]).all() and torch.isnan(got[2]).all()  # (scores of -inf alone)
            keys, values = _numbers(cache.key_pages), _numbers(cache.value_pages)
            pages = cache.table.pages[1].tolist()
            k, v = (np.concatenate([x[pages[0]], x[pages[2], :, :8]], 1) for x in (keys, values))
            for h in range(4):
                s = k[h // 2] @ _numbers(q)[1, h] * 0.125
                w = np.exp(s - s.max())
                want = (w / w.sum()) @ v[h // 2]
                size = (np.abs(k[h // 2]) @ np.abs(_numbers(q)[1, h])).max() * 0.125
                _near(got[1, h], want, dtype, _slack(dtype, size, np.abs(v).max(), 64, 40))


def test_numbers_that_are_not_finite():
    import torch
    rng = np.random.RandomState(10)
    for dtype in ("float32", "bfloat16", "float16"):
        cache = _cache(rng, dtype, [40, 40], 1, 64, 16)
        q = _tensor(np.abs(rng.randn(2, 2, 64)) + 0.1, dtype)
        before = gh.ctx().decode_attention_pages(q, cache)
        cache.value_pages[int(cache.table.pages[0, 1]), 0, 3, 5] = float("nan")
        got = gh.ctx().decode_attention_pages(q, cache)
        assert torch.isnan(got[0, :, 5]).all() and (got[1] == before[1]).all()
        # a window that no longer holds the position
        window = gh.ctx().decode_attention_pages(q, cache, window=20)
        assert torch.isfinite(window).all()
        if dtype == "float32":
            continue
        cache.key_pages[int(cache.table.pages[1, 0]), 0, :] = -float("inf")  # scores of -inf weigh nothing
        got = gh.ctx().decode_attention_pages(q, cache)
        want, most, value = _attention_of_the_rest(q, cache)
        _near(got[1], want, dtype, _slack(dtype, most, value, 64, 40))
        cache.key_pages.fill_(-float("inf"))
        assert torch.isnan(gh.ctx().decode_attention_pages(q, cache)[1]).all()


def _attention_of_the_rest(q, cache):
    pages = cache.table.pages[1].tolist()
    k, v = (np.concatenate([_numbers(x)[pages[1], 0], _numbers(x)[pages[2], 0, :8]]) for x in (cache.key_pages, cache.value_pages))
    out, most = [], 0.0
    for h in range(2):
        s = k @ _numbers(q)[1, h] * 0.125
        w = np.exp(s - s.max())
        out.append((w / w.sum()) @ v)
        most = max(most, (np.abs(k) @ np.abs(_numbers(q)[1, h])).max() * 0.125)
    return np.array(out), most, np.abs(v).max()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_small_weights_count(dtype):
    """One position leads by some nats and has the value 0: the context is the sum of the others' small weights."""
    import torch
    for lead in (5.0, 12.0, 18.0, 24.0):
        n = 600
        keys, values = torch.zeros(n, 64), torch.full((n, 64), 3.0)
        keys[100, 0], values[100] = lead * 8, 0.0
        cache = _cache(np.random.RandomState(0), dtype, [n], 1, 64, 32)
        pages = cache.table.pages[0].tolist()
        for i, page in enumerate(pages):
            for pool, x in zip(cache.pools(), (keys, values)):
                part = x[i * 32:(i + 1) * 32]
                pool[page, 0, :len(part)] = part.to(pool.dtype)
        q = torch.zeros(1, 1, 64, device="cuda", dtype=cache.key_pages.dtype)
        q[0, 0, 0] = 1.0
        got = _numbers(gh.ctx().decode_attention_pages(q, cache))
        small = np.exp(-lead)
        want = 3.0 * (n - 1) * small / (1 + (n - 1) * small)
        left = {"float32": 2.0 ** -21, "bfloat16": 2.0 ** -18, "float16": 2.0 ** -22 + 2.0 ** -39 / small}[dtype]
        # (halves below 2^-14 are 2^-24 apart, so a context there is off by up to 2^-25 by its rounding alone: at 24 nats it is 6.8e-8, between
        # 2^-24 = 6.0e-8 and 2^-23)
        step = 2.0 ** -25 if dtype == "float16" and want < 2.0 ** -14 else 0.0
        assert (np.abs(got - want) <= want * (2.0 ** -19 + left + lead * 2.0 ** -22 + HALF_STEP[dtype]) + step).all(), (lead, got[0, 0, 0], want)


def test_scores_of_every_size():
    for scale in (0.0, 1e-3, 4.0, -1.0):
        for dtype in ("float32", "bfloat16", "float16"):
            _check(dtype, 4, 2, 1, 64, [200, 77], 16, scale=scale, seed=int(abs(scale)))


def test_the_same_call_gives_the_same_bits_and_graphs_replay():
    import torch
    ctx = psx.Context(0)
    rng = np.random.RandomState(11)
    cache = _cache(rng, "bfloat16", [3000, 1777], 2, 64, 32)
    q = _tensor(rng.randn(2, 8, 64), "bfloat16")
    first = ctx.decode_attention_pages(q, cache).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ctx.decode_attention_pages(q, cache)
    _check("bfloat16", 4, 4, 1, 64, [64] * 70, 16, ctx=ctx)  # (more pairs: the scratch grows)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (out == first).all()
    cache.table.lengths.copy_(torch.tensor([5, 1200]))
    graph.replay()
    torch.cuda.synchronize()
    assert (out == psx.Context(0).decode_attention_pages(q, cache)).all()


def test_scratch_does_not_grow_inside_a_capture():
    import torch
    ctx = psx.Context(0)
    rng = np.random.RandomState(12)
    cache = _cache(rng, "bfloat16", [3000, 1777], 2, 64, 32)
    q = _tensor(rng.randn(2, 8, 64), "bfloat16")
    graph = torch.cuda.CUDAGraph()
    refused = None
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = torch.zeros(1, device="cuda")
        try:
            ctx.decode_attention_pages(q, cache)
        except psx.PsxError as e:
            refused = e.status
    assert refused == psx.ERR_UNSUPPORTED
    ctx.decode_attention_pages(q, cache)


def test_two_contexts_on_two_streams():
    import torch
    rng = np.random.RandomState(13)
    caches = [_cache(rng, "float16", [5000, 100, 2000], 4, 128, 64) for _ in range(2)]
    qs = [_tensor(rng.randn(3, 16, 128), "float16") for _ in range(2)]
    ctxs, streams = [psx.Context(0) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    alone = [gh.ctx().decode_attention_pages(q, c).clone() for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [ctx.decode_attention_pages(q, c, stream=s.cuda_stream) for ctx, q, c, s in zip(ctxs, qs, caches, streams)]
        torch.cuda.synchronize()
        assert all((a == b).all() for a, b in zip(got, alone))


def test_many_rows():
    rng = np.random.RandomState(14)
    _check("float16", 2, 1, 1, 16, rng.randint(0, 40, 4096).tolist(), 16, seed=3)
    cache = psx.PagedCache(psx.PageTable.empty(0, 1, 1, 16), *[_tensor(np.zeros((1, 1, 16, 16)), "float32") for _ in range(2)])
    assert gh.ctx().decode_attention_pages(_tensor(np.zeros((0, 2, 16)), "float32"), cache).shape == (0, 2, 16)


def test_refusals():
    import torch
    ctx = gh.ctx()
    rng = np.random.RandomState(15)
    cache = _cache(rng, "float32", [4, 4], 2, 64, 16)

    def decode(heads, q_len, cache=cache, dtype="float32", **kw):
        return ctx.decode_attention_pages(_tensor(np.zeros((2 * q_len, heads, cache.head_dim)), dtype), cache, q_len=q_len, **kw)

    wide = psx.PagedCache(psx.PageTable.empty(2, 4, 8, 16), *[torch.zeros(8, 2, 16, 264, device="cuda") for _ in range(2)])
    odd = psx.PagedCache(psx.PageTable.empty(2, 4, 8, 16), *[torch.zeros(8, 2, 16, 20, device="cuda") for _ in range(2)])
    for status, call in ((psx.ERR_BAD_ARGUMENT, lambda: decode(3, 1)), (psx.ERR_UNSUPPORTED, lambda: decode(34, 1)), (psx.ERR_UNSUPPORTED, lambda: decode(4, 9)),
                         (psx.ERR_BAD_ARGUMENT, lambda: decode(4, 1, window=-1)), (psx.ERR_BAD_ARGUMENT, lambda: decode(4, 1, scale=float("nan"))),
                         (psx.ERR_UNSUPPORTED, lambda: decode(4, 1, wide)), (psx.ERR_UNSUPPORTED, lambda: decode(4, 1, odd))):
        with pytest.raises(psx.PsxError) as e:
            call()
        assert e.value.status == status
    q = torch.zeros(2, 4, 64, device="cuda")
    for bad in (q.half(), q[:1], q.cpu(), q[:, :, :32].contiguous(), torch.zeros(2, 64, 4, device="cuda").transpose(1, 2)):
        with pytest.raises(ValueError):
            ctx.decode_attention_pages(bad, cache)
    pool = torch.zeros(8, 2, 16, 64, device="cuda")
    table = psx.PageTable.empty(2, 4, 8, 16)
    for keys, values in ((pool[:7], pool[:7]), (pool, pool.half()), (pool, pool[:, :1]), (pool.transpose(1, 2), pool), (pool.cpu(), pool), (pool[0], pool[0])):
        with pytest.raises(ValueError):
            psx.PagedCache(table, keys, values)
    with pytest.raises(TypeError):
        psx.PagedCache(table, pool.double(), pool.double())
