"""Log-probabilities of given tokens, entropy and alternatives (psx_b200_token_log_probs) against the formula in double precision.

Tolerance, in units u = 2^-24.  With r the sum of exp(x - m) over all logits but the largest, m: a term at the distance d from m is off by 2 d for its
exponent (a difference and a product) and 4 for its exponential; those that matter have d < 18 + g, g being the distance of the second largest (all of
r lies that far below where the largest leads); a thread adds at most 128 pairs, one unit each, and takes at most eight factors for a new largest, two
each; ten joins.  Together less than 200 + 2 g of r, and log(1 + r) by that times r / (1 + r).  The entropy's second sum is off by as much again and is divided by 1 +
r: 400 + 4 g of the entropy.  A term below 2^-126 is no float and counts nothing: vocab * 2^-126 of r, and times its logarithm, 90 nats, of the entropy.
Results are rounded once: half a step.  Tokens are exact."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = ["float32", "bfloat16", "float16"]


def _tensor(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(getattr(torch, dtype)).cuda()


def _formula(x, top):
    """x: float64 (rows, vocab), finite or -inf, one finite at least: log-probabilities, r, entropies, the alternatives' tokens."""
    m = x.max(1, keepdims=True)
    gap = x - m
    e = np.exp(gap)
    first = gap.argmax(1)
    e[np.arange(len(x)), first] = 0.0
    r = e.sum(1)
    finite = np.where(np.isinf(gap), 0.0, gap)
    log_p = gap - np.log1p(r)[:, None]
    entropy = np.log1p(r) - (e * finite).sum(1) / (1 + r)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return log_p, r, entropy, order


def _check(logits, tokens, top, ctx=None, view=None):
    """logits: a tensor; view: what the call gets instead (the same numbers)."""
    import torch
    rows = logits.shape[0]
    out = (ctx or gh.ctx()).token_log_probs(logits if view is None else view, None if tokens is None else torch.from_numpy(tokens).cuda(), top=top, entropy=True)
    x = logits.double().cpu().numpy()
    log_p, r, entropy, order = _formula(x, top)
    assert out["status"].tolist() == [0] * rows
    two = np.sort(np.where(np.isinf(x), np.finfo(np.float64).min, x), axis=1)[:, -2:]
    g = np.where(x.shape[1] > 1, np.minimum(two[:, -1] - two[:, 0], 104.0), 0.0)  # (beyond that r is no float)
    lost = x.shape[1] * 2.0 ** -126
    slack = ((200 + 2 * g) * U * r + lost) / (1 + r)
    if tokens is None:
        assert out["log_probs"] is None
    else:
        got, want = out["log_probs"].double().cpu().numpy(), log_p[np.arange(rows), tokens]
        gone = want < -np.finfo(np.float32).max  # (-inf, or no float: the lowest logit 2^129 below the largest)
        assert (got[gone] == -np.inf).all()
        assert (np.abs(got[~gone] - want[~gone]) <= (slack + U * np.abs(want))[~gone] * (1 + 1e-9) + 1e-45).all()
    got = out["entropy"].double().cpu().numpy()
    assert (np.abs(got - entropy) <= (401 + 4 * g) * U * entropy + 91 * lost + 1e-45).all()
    if top == 0:
        assert out["top_tokens"] is None
        return out
    got, tokens = out["top_log_probs"].double().cpu().numpy(), out["top_tokens"].cpu().numpy()
    filled = order.shape[1]
    want = np.take_along_axis(log_p, order, 1)
    there = want >= -np.finfo(np.float32).max
    assert (tokens[:, :filled] == np.where(np.isinf(want), -1, order)).all()
    assert (tokens[:, filled:] == -1).all() and (got[:, filled:] == -np.inf).all() and (got[:, :filled][~there] == -np.inf).all()
    error = np.abs(np.where(there, got[:, :filled], 0) - np.where(there, want, 0))
    assert (error <= slack[:, None] + U * np.abs(np.where(there, want, 0)) * (1 + 1e-9) + 1e-45).all()
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 1000, 1024, 4096, 4097, 50257])
@pytest.mark.parametrize("rows,top", [(1, 5), (3, 0), (2, 128), (200, 1)])
def test_rows_of_every_length(dtype, vocab, rows, top):
    rng = np.random.RandomState(vocab + rows)
    _check(_tensor(rng.randn(rows, vocab) * 3, dtype), rng.randint(0, vocab, rows), top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(64, 151936, 20), (1, 262144, 64), (1, 151936, 128), (700, 32000, 8), (5, 1000003, 16)])
def test_large_rows(dtype, rows, vocab, top):
    rng = np.random.RandomState(rows)
    x = rng.randn(rows, vocab).astype(np.float32) * 3
    x[rng.rand(rows, vocab) < 0.1] = -np.inf
    x[:, 0] = 1.0
    tokens = np.where(rng.rand(rows) < 0.5, x.argmax(1), rng.randint(0, vocab, rows))
    _check(_tensor(x, dtype), tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,pad,shift", [(1000, 1, 0), (1001, 0, 1), (50257, 0, 3), (4096, 5, 7), (9, 0, 5), (3, 2, 1), (151936, 8, 2)])
def test_rows_that_start_anywhere(dtype, vocab, pad, shift):
    import torch
    rng = np.random.RandomState(vocab)
    rows, stride = 5, vocab + pad
    flat = torch.full((rows * stride + shift,), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    view = flat[shift:].view(rows, stride)[:, :vocab]
    logits = _tensor(rng.randn(rows, vocab) * 4, dtype)
    view.copy_(logits)
    _check(logits, rng.randint(0, vocab, rows), 6, view=view)
    # a shorter vocabulary than the row has columns
    whole = flat[shift:].view(rows, stride)
    if vocab > 4:
        out = gh.ctx().token_log_probs(whole, top=3, vocab=vocab - 3)
        assert (out["top_tokens"].cpu().numpy() == _formula(logits[:, :vocab - 3].double().cpu().numpy(), 3)[3]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [2.0, 8.0, 16.0, 24.0, 60.0])
@pytest.mark.parametrize("vocab", [11, 5000, 60000])
def test_a_token_that_is_nearly_certain(dtype, gap, vocab):
    rng = np.random.RandomState(int(gap))
    x = rng.randn(6, vocab) * 0.5
    at = rng.randint(0, vocab, 6)
    at[:2] = [0, vocab - 1]
    x[np.arange(6), at] = gap
    _check(_tensor(x, dtype), at, 4)
    # two of them
    x[np.arange(6), (at + 1 + rng.randint(0, vocab - 1, 6)) % vocab] = gap
    _check(_tensor(x, dtype), at, 4)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits(dtype):
    for vocab in (5, 3000, 50257, 140000):
        _check(_tensor(np.full((3, vocab), -1.5), dtype), np.array([0, vocab - 1, vocab // 2]), 20)
        x = np.full((2, vocab), -np.inf)
        x[:, ::2] = 0.0
        x[1, ::2] = -0.0 * np.arange(x[1, ::2].size)
        _check(_tensor(x, dtype), np.array([0, 2]), 100)
    # thousands at the bound among others
    rng = np.random.RandomState(0)
    _check(_tensor(np.clip(rng.randn(4, 100000), -9, 1.0), dtype), np.arange(4), 100)


@pytest.mark.parametrize("dtype", TYPES)
def test_logits_of_every_size(dtype):
    import torch
    largest = float(torch.finfo(getattr(torch, dtype)).max)
    x = np.zeros((5, 3000))
    x[0, [5, 77]] = [largest, -largest]
    x[1] = -largest
    x[2] = largest
    x[3, 10:] = -np.inf
    x[4, :] = np.linspace(-largest, -largest * 0.5, 3000)
    _check(_tensor(x, dtype), np.array([77, 2999, 0, 2999, 0]), 7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [9, 20000])
def test_what_a_row_reports(dtype, vocab):
    import torch
    rng = np.random.RandomState(vocab)
    x = rng.randn(8, vocab)
    x[1] = -np.inf
    x[2, vocab // 2], x[3, 0], x[4, vocab - 1] = np.nan, np.inf, np.nan
    x[4, 1] = np.inf
    tokens = np.array([3, 3, 3, 0, 3, -1, vocab, 2 ** 62])
    out = gh.ctx().token_log_probs(_tensor(x, dtype), torch.from_numpy(tokens).cuda(), top=4, entropy=True)
    assert out["status"].tolist() == [0, psx.ROW_ALL_REMOVED] + [psx.ROW_NON_FINITE] * 3 + [psx.ROW_BAD_TOKEN] * 3
    log_p, got, entropy = (out[k].cpu().numpy() for k in ("log_probs", "top_log_probs", "entropy"))
    assert np.isnan(log_p[1:]).all() and np.isfinite(log_p[0]) and np.isnan(entropy[1:5]).all() and np.isfinite(entropy[[0, 5, 6, 7]]).all()
    assert (out["top_tokens"][1:5] == -1).all() and (got[1] == -np.inf).all() and np.isnan(got[2:5]).all() and np.isfinite(got[5:]).all()
    assert (out["top_tokens"][5:].cpu().numpy() == _formula(_tensor(x[5:], dtype).double().cpu().numpy(), 4)[3]).all()
    negative = torch.full((1, vocab), float("nan"), device="cuda", dtype=getattr(torch, dtype))
    assert int(gh.ctx().token_log_probs(-negative)["status"]) == psx.ROW_NON_FINITE


def test_the_log_probability_of_a_sampled_token():
    import torch
    ctx = gh.ctx()
    logits = torch.randn(16, 50257, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 3
    drawn = ctx.sample_rows(logits, None, None, psx.SamplingConfig.make(do_sample=False), None)
    scored = ctx.token_log_probs(logits, drawn["tokens"], top=1)
    assert (scored["top_tokens"][:, 0] == drawn["tokens"]).all()
    assert torch.allclose(scored["log_probs"], drawn["log_probs"], rtol=1e-5, atol=0)
    assert (scored["top_log_probs"][:, 0] == scored["log_probs"]).all()


def test_the_same_bits_captured_replayed_and_on_another_stream():
    import torch
    ctx = psx.Context(0)
    rng = np.random.RandomState(3)
    logits, tokens = _tensor(rng.randn(5, 50257), "bfloat16"), torch.from_numpy(rng.randint(0, 50257, 5)).cuda()
    call = lambda **more: ctx.token_log_probs(logits, tokens, top=9, entropy=True, **more)
    want = {k: v.clone() for k, v in call().items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    other = call(stream=stream.cuda_stream)
    stream.synchronize()
    assert all((other[k] == want[k]).all() for k in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all((out[k] == want[k]).all() for k in want)
    logits.copy_(logits.flip(0))
    tokens.copy_(tokens.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert (out["top_tokens"] == want["top_tokens"].flip(0)).all()
    # a context's first call may be captured, and its calls may overlap: there is no scratch
    fresh, graph, other = psx.Context(0), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = fresh.token_log_probs(logits, tokens, top=9)
    for _ in range(10):
        graph.replay()
        beside = fresh.token_log_probs(logits, tokens, top=9, stream=other.cuda_stream)
        torch.cuda.synchronize()
        assert (out["log_probs"] == beside["log_probs"]).all() and (out["top_tokens"] == beside["top_tokens"]).all()


def test_many_rows_and_none():
    rng = np.random.RandomState(4)
    _check(_tensor(rng.randn(20000, 40), "float16"), rng.randint(0, 40, 20000), 3)
    out = gh.ctx().token_log_probs(_tensor(np.zeros((0, 40)), "float16"), top=3, entropy=True)
    assert out["top_tokens"].shape == (0, 3) and out["status"].shape == (0,)


def test_refusals():
    import torch
    ctx = gh.ctx()
    x, tokens = torch.zeros(4, 100, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (dict(tokens=tokens[:3]), dict(tokens=tokens.int()), dict(tokens=tokens.cpu()), dict(vocab=0), dict(vocab=101)):
        with pytest.raises(ValueError):
            ctx.token_log_probs(x, **bad)
    for bad in (x.cpu(), x.t()):
        with pytest.raises(ValueError):
            ctx.token_log_probs(bad)
    with pytest.raises(TypeError):
        ctx.token_log_probs(x.double())
    for bad, status in ((dict(top=129), psx.ERR_UNSUPPORTED), (dict(top=-1), psx.ERR_BAD_ARGUMENT)):
        with pytest.raises(psx.PsxError) as e:
            ctx.token_log_probs(x, **bad)
        assert e.value.status == status
    call = lambda vocab, stride, logits=x.data_ptr(), log_probs=None, toks=None, top=0: ctx._lib.psx_b200_token_log_probs(
        ctx._ctx, None, 0, logits, 4, vocab, stride, toks, log_probs, None, top, None, None, None)
    assert call(100, 99) == psx.ERR_BAD_ARGUMENT and call((1 << 30) + 1, 1 << 31) == psx.ERR_UNSUPPORTED
    assert call(100, 100, logits=None) == psx.ERR_BAD_ARGUMENT and call(100, 100, toks=tokens.data_ptr()) == psx.ERR_BAD_ARGUMENT
    assert call(100, 100, top=1) == psx.ERR_BAD_ARGUMENT and call(100, 100, logits=x.data_ptr() + 2) == psx.ERR_BAD_ARGUMENT
    assert ctx._lib.psx_b200_token_log_probs(ctx._ctx, None, 3, x.data_ptr(), 4, 100, 100, None, None, None, 0, None, None, None) == psx.ERR_BAD_ARGUMENT
