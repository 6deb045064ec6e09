"""Norm per head, rotation by the position and the way into a cache in pages (psx_b200_rotate_heads) against the formula in double precision.

Tolerance, in units of 2^-24 of |x| + |y|, the normed elements of a pair: a square and its sum over a lane's eight and five steps between lanes
are off by at most 15, the root of it by half of that; mean, eps, root, quotient and the two products by one each: 13.5.  Cosine and sine: the angle
is off by 2^-26 quarter turns (0.4), the functions by 2 (two roundings of numbers up to 1, and 2.2e-9); product and sum 2.  Together less than 20.  The result is
rounded to its type: half a step of it, 2^-25 at least in fp16's subnormal range."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx

pytestmark = pytest.mark.gpu
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _numbers(t):
    return t.double().cpu().numpy()


def _formula(x, weight, eps, position, frequencies, interleaved):
    """(total, heads, dims): the result, and |x| + |y| of each element's pair."""
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    out, size = x.copy(), np.abs(x)
    pairs = len(frequencies)
    i = np.arange(pairs)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    angle = (position[:, None] * frequencies)[:, None]
    u, v = x[..., a], x[..., b]
    out[..., a], out[..., b] = u * np.cos(angle) - v * np.sin(angle), v * np.cos(angle) + u * np.sin(angle)
    size[..., a] = size[..., b] = np.abs(u) + np.abs(v)
    return out, size


def _near(got, want, size, dtype):
    slack = 20 * 2.0 ** -24 * size + HALF_STEP[dtype] * np.abs(want) * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype == "float16" else 0.0)
    return (np.abs(got - want) <= slack).all()


def _case(dtype, heads, kv_heads, dims, rotated, counts, first, size, seed, norm=True, max_pages=None):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = getattr(torch, dtype)
    total = sum(counts)
    qkv = torch.randn(total, heads + 2 * kv_heads, dims, generator=gen, device="cuda").mul(2).to(kind)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    weights = [torch.randn(dims, generator=gen, device="cuda").to(kind) for _ in range(2)] if norm else [None, None]
    frequencies = 10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device="cuda") / rotated) if rotated else None
    lengths = [n + f for n, f in zip(counts, first)]
    max_pages = max_pages or max(1, max(-(-n // size) for n in lengths))
    table = psx.PageTable.empty(len(counts), max_pages, sum(-(-n // size) for n in lengths) + 2, size)
    gh.ctx().extend_pages(table, torch.tensor(lengths, device="cuda"))
    cache = psx.PagedCache(table, *[torch.full((table.num_pages, kv_heads, size, dims), 7.0, device="cuda", dtype=kind) for _ in range(2)])
    return q, k, v, weights, frequencies, cache, torch.tensor([0] + list(np.cumsum(counts)), device="cuda"), torch.tensor(first, device="cuda")


def _paged(pages, table, rows, positions):
    """What the table's pages hold at these (row, position)."""
    entries = table.pages.cpu().numpy()
    at = entries[rows, positions // table.page_size]
    return _numbers(pages)[at, :, positions % table.page_size]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("dims,rotated", [(8, 8), (64, 64), (80, 32), (96, 96), (128, 128), (128, 64), (256, 256), (200, 0), (40, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv_heads,counts,first,size", [(4, 2, [1, 1, 1], [0, 16, 1000], 16), (3, 1, [5, 0, 33, 1], [0, 3, 15, 64], 32),
                                                              (16, 8, [130, 2], [0, 127], 64)])
def test_packed_rows(dtype, dims, rotated, interleaved, heads, kv_heads, counts, first, size):
    q, k, v, weights, frequencies, cache, offsets, start = _case(dtype, heads, kv_heads, dims, rotated, counts, first, size, dims + heads)
    got_q, got_k, status = gh.ctx().rotate_heads(q, k, v, offsets=offsets, first=start, frequencies=frequencies, q_weight=weights[0], k_weight=weights[1],
                                                 eps=1e-5, interleaved=interleaved, cache=cache, keys_too=True)
    assert status.tolist() == [0] * len(counts)
    rows = np.repeat(np.arange(len(counts)), counts)
    position = np.concatenate([np.arange(f, f + n) for f, n in zip(first, counts)]).astype(np.int64)
    turns = np.array([]) if frequencies is None else frequencies.cpu().numpy()
    for x, weight, got in ((q, weights[0], got_q), (k, weights[1], got_k)):
        want, size_of = _formula(_numbers(x), _numbers(weight), 1e-5, position, turns, interleaved)
        assert _near(_numbers(got), want, size_of, dtype)
    assert (_paged(cache.key_pages, cache.table, rows, position) == _numbers(got_k)).all()  # (the same bits)
    assert (_paged(cache.value_pages, cache.table, rows, position) == _numbers(v)).all()
    for pages in cache.pools():  # nothing else was written
        assert int((pages == 7.0).all(-1).sum()) >= pages.shape[0] * pages.shape[1] * pages.shape[2] - sum(counts) * kv_heads
    # without the cache, and without norms
    same_q, same_k, _ = gh.ctx().rotate_heads(q, k, offsets=offsets, first=start, frequencies=frequencies, q_weight=weights[0], k_weight=weights[1], eps=1e-5,
                                              interleaved=interleaved)
    assert (same_q == got_q).all() and (same_k == got_k).all()
    plain_q, _, _ = gh.ctx().rotate_heads(q, k, offsets=offsets, first=start, frequencies=frequencies, interleaved=interleaved, k_weight=weights[1])
    want, size_of = _formula(_numbers(q), None, 0, position, turns, interleaved)
    assert _near(_numbers(plain_q), want, size_of, dtype)
    if frequencies is None:
        assert (plain_q == q).all()


@pytest.mark.parametrize("position", [0, 1, 2 ** 17 + 1, 10 ** 6 + 7, 2 ** 29 - 1])
def test_far_positions(position):
    import torch
    x = torch.randn(1, 2, 128, device="cuda")
    frequencies = 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64, device="cuda") / 128)
    got, _, _ = gh.ctx().rotate_heads(x, x, offsets=torch.tensor([0, 1], device="cuda"), first=torch.tensor([position], device="cuda"), frequencies=frequencies)
    # (the angle in double precision: 3 units of 2^-53 of it)
    want, size = _formula(_numbers(x), None, 0, np.array([position]), frequencies.cpu().numpy(), False)
    assert (np.abs(_numbers(got) - want) <= (20 * 2.0 ** -24 + 3 * 2.0 ** -53 * position) * size).all()


def test_quarter_turns_are_exact_enough():
    # frequencies of quarter turns: cosine and sine are 0, 1 or -1 but for the rounding of pi / 2
    import torch
    x = torch.randn(9, 1, 8, device="cuda")
    frequencies = torch.full((4,), np.pi / 2, dtype=torch.float64, device="cuda")
    got, _, _ = gh.ctx().rotate_heads(x, x, offsets=torch.tensor([0, 9], device="cuda"), first=torch.tensor([3], device="cuda"), frequencies=frequencies)
    want, size = _formula(_numbers(x), None, 0, np.arange(3, 12), frequencies.cpu().numpy(), False)
    assert _near(_numbers(got), want, size, "float32")


def test_many_rows_and_positions_of_none():
    import torch
    rng = np.random.RandomState(0)
    for batch in (31, 32, 33, 1000, 4096):
        counts = rng.randint(0, 3, batch)
        gap, behind = 5, 7
        total = int(counts.sum()) + gap + behind
        q = torch.randn(total, 1, 8, device="cuda")
        offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]) + gap).cuda()
        first = torch.from_numpy(rng.randint(0, 1000, batch)).cuda()
        frequencies = torch.tensor([1.0, 0.5, 0.25, 0.125], dtype=torch.float64, device="cuda")
        out = torch.full_like(q, 3.0)
        status = torch.full((batch,), 9, dtype=torch.int32, device="cuda")
        ctx = gh.ctx()
        assert ctx._lib.psx_b200_rotate_heads(ctx._ctx, None, 0, q.data_ptr(), q.data_ptr(), None, out.data_ptr(), torch.empty_like(q).data_ptr(), total, 8, 8, 8,
                                              offsets.data_ptr(), first.data_ptr(), batch, 1, 1, 8, None, None, 0.0, frequencies.data_ptr(), 8, 0, None,
                                              status.data_ptr()) == 0
        torch.cuda.synchronize()
        position = np.concatenate([np.arange(f, f + n) for f, n in zip(first.tolist(), counts)])
        want, size = _formula(_numbers(q)[gap:total - behind], None, 0, position, frequencies.cpu().numpy(), False)
        assert _near(_numbers(out)[gap:total - behind], want, size, "float32")
        assert (out[:gap] == 3.0).all() and (out[total - behind:] == 3.0).all() and not status.any()


def test_rows_that_do_not_fit_and_bad_pages():
    import torch
    q, k, v, _, frequencies, cache, offsets, start = _case("float32", 2, 1, 16, 16, [4, 4, 4, 4], [0, 20, 5, 1], 16, 3, norm=False)
    cache.table.lengths.copy_(torch.tensor([4, 23, 9, 5]))  # row 1 lacks one position
    cache.table.pages[2, 0], cache.table.pages[3, 0] = cache.table.num_pages, -2
    got_q, _, status = gh.ctx().rotate_heads(q, k, v, offsets=offsets, first=start, frequencies=frequencies, cache=cache)
    assert status.tolist() == [0, psx.ROW_CACHE_FULL, 0, 0]
    written = (cache.value_pages != 7.0).any(-1).nonzero().tolist()
    page = int(cache.table.pages[0, 0])
    assert written == [[page, 0, i] for i in range(4)]
    want, size = _formula(_numbers(q), None, 0, np.concatenate([np.arange(f, f + 4) for f in (0, 20, 5, 1)]), frequencies.cpu().numpy(), False)
    assert _near(_numbers(got_q), want, size, "float32")
    start = torch.tensor([-1, 2 ** 62, 0, 0], device="cuda")
    _, _, status = gh.ctx().rotate_heads(q, k, v, offsets=torch.tensor([0, 4, 8, 7, 20], device="cuda"), first=start, frequencies=frequencies, cache=cache)
    assert status.tolist() == [65, 64, 65, 65]
    assert (cache.value_pages != 7.0).any(-1).nonzero().tolist() == written


def test_numbers_that_are_not_finite_stay_in_their_head():
    import torch
    x = torch.ones(3, 2, 16, device="cuda")
    x[0, 0, 3], x[1, 1, 0], x[2, 0, 15] = float("nan"), float("inf"), float("-inf")
    offsets, first = torch.tensor([0, 3], device="cuda"), torch.tensor([1], device="cuda")
    weight = torch.ones(16, device="cuda")
    got, _, _ = gh.ctx().rotate_heads(x, x, offsets=offsets, first=first, frequencies=torch.ones(4, dtype=torch.float64, device="cuda"))
    bad = ~torch.isfinite(got)
    assert sorted(map(tuple, bad.nonzero().tolist())) == [(0, 0, 3), (0, 0, 7), (1, 1, 0), (1, 1, 4), (2, 0, 15)]
    got, _, _ = gh.ctx().rotate_heads(x, x, offsets=offsets, first=first, q_weight=weight, k_weight=weight)
    assert torch.isfinite(got[[0, 1, 2], [1, 0, 1]]).all() and torch.isnan(got[0, 0]).all() and torch.isnan(got[1, 1, 0])
    zero, _, _ = gh.ctx().rotate_heads(torch.zeros_like(x), x, offsets=offsets, first=first, q_weight=weight)
    assert (zero == 0).all()


def test_in_place_captured_and_on_another_stream():
    import torch
    ctx = psx.Context(0)
    q, k, v, weights, frequencies, cache, offsets, start = _case("bfloat16", 4, 2, 64, 64, [7, 9], [3, 30], 16, 5)
    call = lambda **more: ctx.rotate_heads(q, k, v, offsets=offsets, first=start, frequencies=frequencies, q_weight=weights[0], k_weight=weights[1], cache=cache,
                                           keys_too=True, **more)
    want_q, want_k, _ = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    other_q, other_k, _ = call(stream=stream.cuda_stream)
    stream.synchronize()
    assert (other_q == want_q).all() and (other_k == want_k).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graph_q, graph_k, _ = call()
    start.add_(1)
    cache.table.lengths.add_(1)
    cache.table.pages.clamp_(min=0)
    graph.replay()
    torch.cuda.synchronize()
    again_q, again_k, _ = call()
    assert (graph_q == again_q).all() and (graph_k == again_k).all() and not (graph_q == want_q).all()
    # in place
    whole_q, whole_k = q.contiguous(), k.contiguous()
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert ctx._lib.psx_b200_rotate_heads(ctx._ctx, None, 1, whole_q.data_ptr(), whole_k.data_ptr(), None, whole_q.data_ptr(), whole_k.data_ptr(), 16, 256, 128, 128,
                                          offsets.data_ptr(), start.data_ptr(), 2, 4, 2, 64, weights[0].data_ptr(), weights[1].data_ptr(), 1e-6,
                                          frequencies.data_ptr(), 64, 0, None, status.data_ptr()) == 0
    torch.cuda.synchronize()
    assert (whole_q == again_q).all() and (whole_k == again_k).all()


def test_nothing_to_do():
    import torch
    empty = torch.empty(0, 2, 16, device="cuda")
    q, k, status = gh.ctx().rotate_heads(empty, empty, offsets=torch.zeros(3, dtype=torch.int64, device="cuda"), first=torch.zeros(2, dtype=torch.int64, device="cuda"))
    assert q.shape == (0, 2, 16) and status.tolist() == [0, 0]
    q, k, status = gh.ctx().rotate_heads(empty, empty, offsets=torch.zeros(1, dtype=torch.int64, device="cuda"), first=torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert status.tolist() == []


def test_refusals():
    import torch
    q, k, v, weights, frequencies, cache, offsets, start = _case("bfloat16", 4, 2, 64, 64, [7, 9], [3, 30], 16, 5)
    ctx = gh.ctx()

    def call(q=q, k=k, v=v, offsets=offsets, first=start, frequencies=frequencies, q_weight=weights[0], k_weight=weights[1], cache=cache, **more):
        return ctx.rotate_heads(q, k, v, offsets=offsets, first=first, frequencies=frequencies, q_weight=q_weight, k_weight=k_weight, cache=cache, **more)

    other = psx.PagedCache(cache.table, *[x.half() for x in cache.pools()])
    for bad in (dict(k=k[1:]), dict(k=k.float()), dict(v=None), dict(v=v[:, :1]), dict(offsets=offsets[:2]), dict(offsets=offsets.int()), dict(first=start[:1]),
                dict(frequencies=frequencies.float()), dict(q_weight=weights[0].float()), dict(k_weight=weights[1][:8]), dict(q=q.cpu()), dict(cache=other),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(frequencies=frequencies.cpu()), dict(offsets=offsets.cpu())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad, status in ((dict(frequencies=frequencies[:30]), psx.ERR_UNSUPPORTED), (dict(frequencies=torch.ones(33, dtype=torch.float64, device="cuda")), psx.ERR_BAD_ARGUMENT),
                        (dict(eps=-1.0), psx.ERR_BAD_ARGUMENT), (dict(eps=float("nan")), psx.ERR_BAD_ARGUMENT),
                        (dict(cache=psx.PagedCache(psx.PageTable.empty(3, 4, cache.table.num_pages, 16), *cache.pools())), psx.ERR_BAD_ARGUMENT),
                        (dict(offsets=offsets[:2], first=start[:1]), psx.ERR_BAD_ARGUMENT)):
        with pytest.raises(psx.PsxError) as e:
            call(**bad)
        assert e.value.status == status
    odd = torch.zeros(16, 4, 68, device="cuda", dtype=torch.bfloat16)[:, :, :64]
    with pytest.raises(ValueError):
        call(q=odd)
    shifted = torch.zeros(16 * 256 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(16, 4, 64)
    with pytest.raises(psx.PsxError) as e:
        call(q=shifted)
    assert e.value.status == psx.ERR_BAD_ARGUMENT
    with pytest.raises(TypeError):
        ctx.rotate_heads(q.double(), k.double(), offsets=offsets, first=start)
    with pytest.raises(psx.PsxError) as e:
        ctx.rotate_heads(q[:, :, :60].contiguous(), k[:, :, :60].contiguous(), offsets=offsets, first=start)
    assert e.value.status == psx.ERR_UNSUPPORTED
    args = lambda k_out: (ctx._ctx, None, 1, q.data_ptr(), k.data_ptr(), None, q.data_ptr(), k_out, 16, 512, 512, 512, offsets.data_ptr(), start.data_ptr(), 2, 4, 2, 64,
                          None, None, 0.0, None, 0, 0, None, None)
    assert ctx._lib.psx_b200_rotate_heads(*args(None)) == psx.ERR_BAD_ARGUMENT
