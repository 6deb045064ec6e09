"""Log-probabilities of given tokens (psx_b200_token_log_probs) for rows that a thread takes in many steps: stretches that are masked ahead of low logits, rows of
millions of logits, and rows so long that a thread keeps one maximum for several steps.  Against the formula in double precision.

Tolerance, in units u = 2^-24, as in test_gpu_token_log_probs.py but for what grows with the row: a term is off by 2 d + 4, d < 18 + g, and by ten joins and the sum of
a pair.  A thread adds a pair for every 512 logits of its part, one unit each, and takes a factor for every 4096, two each; both rounded up to whole steps,
18: less than 100 + vocab / 400 + 2 g together.  After at most 294,912 logits of a part its sums are handed on to sums in double precision (2^-53 each): 576 additions, 72
factors, 800 + 2 g at most.  The entropy's second sum is off by as much again."""
import numpy as np
import pytest

import gpu_harness as gh
import test_gpu_token_log_probs as score_test

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = score_test.TYPES


def _units(vocab):
    return min(100 + vocab / 400, 800)


def _check(logits, tokens, top):
    """score_test._check, on the device, a row at a time."""
    import torch
    out = gh.ctx().token_log_probs(logits, tokens, top=top, entropy=True)
    assert not out["status"].any()
    for row in range(logits.shape[0]):
        x = logits[row].double() + 0.0
        (high, second), at = torch.topk(x, 2)[0].tolist(), int(x.argmax())
        weight = torch.exp(x - high)
        weight[at] = 0.0
        r = float(weight.sum())
        gap = (x - high).masked_fill_(x == -np.inf, 0.0)
        entropy = np.log1p(r) - float((weight * gap).sum()) / (1 + r)
        g, lost = min(high - second, 104.0), len(x) * 2.0 ** -126
        slack = ((_units(len(x)) + 2 * g) * U * r + lost) / (1 + r)
        want = float(x[tokens[row]]) - high - np.log1p(r)
        assert abs(float(out["log_probs"][row]) - want) <= (slack + U * abs(want)) * (1 + 1e-9) + 1e-45 or want == float(out["log_probs"][row])
        assert abs(float(out["entropy"][row]) - entropy) <= (2 * _units(len(x)) + 1 + 4 * g) * U * entropy + 91 * lost + 1e-45
        if top:
            values, best = torch.sort(x, descending=True, stable=True)
            values, best = values[:top], best[:top].masked_fill(values[:top] == -np.inf, -1)
            assert (out["top_tokens"][row] == best).all()
            want = (values - high - np.log1p(r)).cpu().numpy()
            got = out["top_log_probs"][row].double().cpu().numpy()
            finite = np.isfinite(want)
            assert (got[~finite] == want[~finite]).all()
            assert (np.abs(got[finite] - want[finite]) <= (slack + U * np.abs(want[finite])) * (1 + 1e-9) + 1e-45).all()


def _plan(rows, vocab, dtype):
    """Chunks of a part and parts of a row, restated for 148 SMs: what the cases below are to reach."""
    elements, least = 4 if dtype == "float32" else 8, None
    for vectors in (4, 1):
        chunk, chain, further = (0.375, 4.3, 1.2) if vectors == 1 else (0.79, 5.2, 1.7)
        steps = -(-(vocab + elements - 1) // (256 * vectors * elements))
        for parts in (1, 2, 4, 8, 16):
            each, beside = -(-steps // parts), max(1.0, rows * parts / 148)
            if vectors == 1 and each > (8 if beside > 8.0 else 32) or parts > 1 and (each * (parts - 1) >= steps or (parts == 16 and beside > 1.0)):
                continue
            cost = each * chunk + chain + (parts > 1) + (beside - 1.0) * (further + 0.09 * vectors * each)
            if least is None or cost < least[0]:
                least = cost, each, parts
    return least[1:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(300, 50257), (600, 40000), (40, 100000), (1, 262144)])
@pytest.mark.parametrize("low", [-89.0, -100.0, -1000.0, -60000.0])
def test_masked_stretches_ahead_of_low_logits(dtype, rows, vocab, low):
    # every thread's first steps hold nothing but masked logits, and what comes then lies far below 0; with an ordinary largest one elsewhere, and without
    import torch
    steps, parts = _plan(rows, vocab, dtype)
    assert steps > 1
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = (low * (1 + 0.05 * torch.rand(rows, vocab, generator=gen, device="cuda"))).to(getattr(torch, dtype))
    begin = -(-vocab // parts) // 2
    for part in range(parts):
        at = part * (-(-vocab // parts))
        x[:, at:at + begin + 5000] = -np.inf
    x[:, vocab - 3:] = low
    x[rows // 2:, vocab // 2] = 1.0 if rows > 1 else low
    tokens = torch.randint(vocab - 3, vocab, (rows,), generator=gen, device="cuda")
    some = torch.tensor(sorted({0, rows // 2, rows - 1}), device="cuda")
    out = gh.ctx().token_log_probs(x, tokens, top=5, entropy=True)
    assert not out["status"].any() and not any(bool(torch.isnan(out[k]).any()) for k in ("log_probs", "entropy", "top_log_probs"))
    _check(x[some].contiguous(), tokens[some], 5)
    _check(x, tokens, 0) if rows == 1 else None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 200])
def test_a_few_tokens_that_a_grammar_allows(dtype, rows):
    import torch
    rng, vocab = np.random.RandomState(rows), 128256
    x = np.full((rows, vocab), -np.inf, np.float32)
    for row in range(rows):
        allowed = rng.choice(vocab, 50, replace=False)
        x[row, allowed] = rng.uniform(-400, -90, 50)
    logits = score_test._tensor(x, dtype)
    tokens = torch.from_numpy(x.argmax(1)).cuda()
    _check(logits, tokens, 60)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(300, 600000), (1000, 270000), (1200, 320000), (1, 8400001), (5, 4200000)])
@pytest.mark.parametrize("top", [1, 20, 128])
def test_more_steps_than_a_thread_keeps_maxima_of(dtype, rows, vocab, top):
    import torch
    steps, parts = _plan(rows, vocab, dtype)
    assert steps > 32
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=gen, device="cuda") * 3).to(getattr(torch, dtype))
    x[::3, -7:] = 30.0    # (the best ones in the last group, which may be a part of one)
    x[1::3] = x[1::3].clamp(max=1.0)  # thousands that are equal: the list overflows
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    some = torch.tensor(sorted({0, min(1, rows - 1), min(2, rows - 1), rows - 1}), device="cuda")
    out = gh.ctx().token_log_probs(x, tokens, top=top, entropy=True)
    few = gh.ctx().token_log_probs(x[some].contiguous(), tokens[some], top=top, entropy=True)  # (other plans, the same row)
    assert (out["top_tokens"][some] == few["top_tokens"]).all()
    for row in some.tolist():
        best = torch.sort(x[row].float() + 0.0, descending=True, stable=True)[1][:top]
        assert (out["top_tokens"][row] == best).all()
    _check(x[some].contiguous(), tokens[some], top)
    if rows > 100:  # every row's sums
        lse = torch.cat([torch.logsumexp(part.double(), 1) for part in x.split(30)])
        want = x.gather(1, tokens[:, None])[:, 0].double() - lse
        assert ((out["log_probs"].double() - want).abs() <= (_units(vocab) + 6) * U + U * want.abs()).all()  # (r / (1 + r) < 1, g < 3)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "small"])
def test_rows_of_tens_of_millions(dtype, kind):
    # (sums of floats alone lose hundreds of units in a row of equal terms)
    import torch
    vocab = 1 << 26
    if kind == "equal":
        x = torch.full((1, vocab), -1.0, device="cuda")
        x[0, 12345] = 0.0
    elif kind == "small":  # all others at one distance
        x = torch.full((1, vocab), -0.7, device="cuda")
        x[0, vocab - 1] = 0.0
    else:
        x = torch.linspace(0.0, 3.0, vocab, device="cuda")[None]
        if kind == "falling":
            x = x.flip(1)
    x = x.contiguous().to(getattr(torch, dtype))
    _check(x, torch.tensor([vocab // 2], device="cuda"), 3 if kind == "small" else 0)
