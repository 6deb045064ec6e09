"""Beam search's selection (psx_b200_beam_select) and the states that follow the beams (psx_b200_reorder_states) against plain
restatements: the selection in double precision, the states by indexing, bit for bit.

Tolerance of a score, in units of 2^-24 of the sum of exponentials: a term's exponent is off by at most 3 |x| (difference, factor,
its own rounding) and x e^x adds up to at most 0.37 of its weight, 1.1; its exponential by 4; a chunk of 16 terms is summed in
four sums of four, 5 roundings with their join; a thread's running sum takes eight chunks, 8 roundings, and at most seven factors for a
new maximum, each off by 5 and rounded; threads, warps and parts are joined by three more such factors.  Together 1.1 + 4 + 5 +
8 + 7 * 6 + 3 * 6 < 80 units, 4.8e-6 in the logarithm; the logarithm of the sum's fraction is within 2 units; the score itself is
rounded once, 2^-24 of its size."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx

pytestmark = pytest.mark.gpu
LOG_SUM = 82 * 2.0 ** -24


def _values(logits, scores, beams, finished=None, finished_token=0):
    """(groups, beams, vocab): every candidate's value in double precision, -inf: none."""
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        log_sum = np.where(np.isfinite(top), top, 0) + np.log(np.exp(x - np.where(np.isfinite(top), top, 0)).sum(1, keepdims=True))
        value = (scores.astype(np.float64)[:, None] - log_sum) + x
    value = np.where(np.isneginf(x) | np.isneginf(scores)[:, None], -np.inf, value)
    if finished is not None:
        value[finished] = -np.inf
        value[finished, finished_token] = scores[finished]
    return value.reshape(-1, beams, logits.shape[1])


def _run(logits, scores, beams, keep, finished=None, finished_token=0, shift=0, pad=0, ctx=None):
    import torch
    rows, vocab = logits.shape
    flat = torch.full((rows * (vocab + pad) + shift + 8,), float("nan"), device="cuda")
    view = flat[shift:shift + rows * (vocab + pad)].view(rows, vocab + pad)
    view[:, :vocab] = torch.from_numpy(logits).cuda()
    out = (ctx or gh.ctx()).beam_select(view, torch.from_numpy(scores).cuda(), beams, keep, vocab=vocab, finished_token=finished_token,
                                        finished=None if finished is None else torch.from_numpy(finished).cuda())
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in out.items()}


def _check(out, value, keep):
    groups, beams, vocab = value.shape
    for g in range(groups):
        flat = value[g].ravel()
        order = np.argsort(-flat, kind="stable")[:keep]
        want = flat[order]
        real = np.isfinite(want)
        count = int(real.sum())
        assert out["status"][g] == (0 if count else 5)
        assert (out["parents"][g, count:] == -1).all() and (out["tokens"][g, count:] == -1).all() and np.isneginf(out["scores"][g, count:]).all()
        at = out["parents"][g, :count] * vocab + out["tokens"][g, :count]
        assert len(set(at.tolist())) == count and (at >= 0).all() and (at < beams * vocab).all()
        slack = LOG_SUM + 2.0 ** -24 * np.abs(want[real])
        given = np.maximum(want[real], -np.finfo(np.float32).max)  # (what is below the lowest float is given as that)
        assert (np.abs(out["scores"][g, :count] - given) <= slack).all()
        # a candidate is the one of its place, or as good as it is to within what both normalisers may be off
        assert (np.abs(flat[at] - want[real]) <= 2 * LOG_SUM).all()
        clear = np.abs(np.diff(np.concatenate([[np.inf], want[real], [-np.inf]]))) > 2 * LOG_SUM
        alone = clear[:-1] & clear[1:]
        alone[-1:] &= count < keep or np.isinf(flat[order[-1]]) or len(flat) == keep
        assert (at[alone] == order[real][alone]).all()


@pytest.mark.parametrize("groups,beams,vocab,keep", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 21), (1, 4, 2048, 8), (3, 2, 2049, 4), (1, 4, 50257, 8),
                                                     (2, 5, 151936, 10), (7, 1, 8193, 1), (1, 64, 1000, 128), (40, 8, 8192, 16), (30, 6, 8191, 12)])
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 3)])
def test_the_best_candidates(groups, beams, vocab, keep, shift, pad):
    rng = np.random.RandomState(groups * 1000 + vocab)
    logits = (rng.randn(groups * beams, vocab) * 3).astype(np.float32)
    scores = -(rng.rand(groups * beams) * 20).astype(np.float32)
    out = _run(logits, scores, beams, keep, shift=shift, pad=pad)
    _check(out, _values(logits, scores, beams), keep)


@pytest.mark.parametrize("vocab", [37, 3000, 50257])
def test_masked_tokens_dead_and_finished_beams(vocab):
    rng = np.random.RandomState(vocab)
    groups, beams, keep = 6, 4, 8
    logits = (rng.randn(groups * beams, vocab) * 4).astype(np.float32)
    logits[rng.rand(*logits.shape) < 0.5] = -np.inf
    scores = -(rng.rand(groups * beams) * 10).astype(np.float32)
    finished = rng.rand(groups * beams) < 0.3
    scores[4:8] = [-np.inf, -1, -np.inf, -np.inf]    # one beam alive, as before the first step
    finished[4:8] = False
    logits[8:12] = -np.inf                           # a group that nothing is left of
    finished[8:12] = False
    logits[12:16] = -np.inf                          # a group with three candidates
    logits[13, [1, vocab - 1]] = [2.0, 2.0]
    finished[12:16] = [False, False, True, False]
    logits[16, :] = np.nan                           # (a finished beam's logits are not looked at)
    finished[16:20] = [True, False, False, False]
    out = _run(logits, scores, beams, keep, finished=finished, finished_token=vocab - 2)
    _check(out, _values(logits, scores, beams, finished, vocab - 2), keep)
    assert out["status"][2] == psx.ROW_ALL_REMOVED


def test_a_group_with_a_number_that_is_not_finite_says_so():
    rng = np.random.RandomState(3)
    for where, what in (("logits", np.nan), ("logits", np.inf), ("scores", np.nan), ("scores", np.inf)):
        logits, scores = rng.randn(6, 9000).astype(np.float32), np.zeros(6, dtype=np.float32)
        if where == "logits":
            logits[3, 8500] = what
        else:
            scores[3] = what
        out = _run(logits, scores, 2, 4)
        assert out["status"].tolist() == [0, psx.ROW_NON_FINITE, 0]
        assert (out["tokens"][1] == -1).all() and (out["parents"][1] == -1).all() and np.isneginf(out["scores"][1]).all()
        good = [0, 2]
        value = _values(np.nan_to_num(logits, posinf=0), np.nan_to_num(scores, posinf=0), 2)[good]
        _check({k: v[good] for k, v in out.items()}, value, 4)


@pytest.mark.parametrize("vocab", [10, 2049, 9001, 50257])
@pytest.mark.parametrize("shift", [0, 1])
def test_ties_go_to_the_lowest_beam_then_the_lowest_token(vocab, shift):
    # equal rows: every beam offers the same values, whatever the alignment of its row
    rng = np.random.RandomState(vocab)
    row = rng.randint(0, 6, vocab).astype(np.float32)  # few values: long lists of ties
    for logits in (np.tile(row, (4, 1)), np.zeros((4, vocab), dtype=np.float32), np.tile(np.where(np.arange(vocab) % 2, 0.0, -0.0), (4, 1)).astype(np.float32)):
        keep = 12
        out = _run(logits, np.zeros(4, dtype=np.float32), 4, keep, shift=shift, pad=1)
        order = np.argsort(-np.tile(logits[0] + 0.0, 4).reshape(4, -1).ravel(), kind="stable")[:keep]
        assert (out["parents"][0] * vocab + out["tokens"][0]).tolist() == order.tolist()
        out = _run(np.tile(logits, (60, 1)), np.zeros(240, dtype=np.float32), 4, keep, shift=shift)  # (the longer parts)
        assert ((out["parents"] * vocab + out["tokens"]) == order).all()


def test_logits_of_every_size():
    logits = np.array([[3e38, -3e38, 0, 1e-40, -np.inf, 88.0], [-3e38, -3.2e38, -3.4e38, -np.inf, -np.inf, -np.inf]], dtype=np.float32)
    scores = np.array([-1.0, -3e38], dtype=np.float32)
    _check(_run(logits, scores, 1, 6), _values(logits, scores, 1), 6)


def test_a_captured_selection_follows_its_inputs():
    import torch
    ctx = psx.Context(0)
    x, s = torch.randn(8, 5000, device="cuda"), torch.zeros(8, device="cuda")
    ctx.beam_select(x, s, 4, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ctx.beam_select(x, s, 4, 8)
    ctx.beam_select(torch.randn(64, 50000, device="cuda"), torch.zeros(64, device="cuda"), 4, 8)  # (the scratch grows; the graph keeps its own)
    for _ in range(2):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        _check({k: v.cpu().numpy() for k, v in out.items()}, _values(x.cpu().numpy(), s.cpu().numpy(), 4), 8)


def test_scratch_does_not_grow_inside_a_capture():
    import torch
    ctx = psx.Context(0)
    x, s = torch.randn(4, 5000, device="cuda"), torch.zeros(4, device="cuda")
    graph, refused = torch.cuda.CUDAGraph(), []
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        try:
            ctx.beam_select(x, s, 4, 8)
        except psx.PsxError as e:
            refused.append(e.status)
        x + 1  # (the capture goes on)
    assert refused == [psx.ERR_UNSUPPORTED]


def test_refusals_of_the_selection():
    import torch
    ctx, x, s = gh.ctx(), torch.zeros(4, 100, device="cuda"), torch.zeros(4, device="cuda")
    for kw in (dict(beams=3, keep=2), dict(beams=0, keep=2), dict(beams=2, keep=2, finished=torch.zeros(3, dtype=torch.bool, device="cuda")),
               dict(beams=2, keep=2, vocab=101)):
        with pytest.raises(ValueError):
            ctx.beam_select(x, s, **kw)
    with pytest.raises(ValueError):
        ctx.beam_select(x.double(), s, 2, 2)
    with pytest.raises(ValueError):
        ctx.beam_select(x.cpu(), s, 2, 2)
    for status, kw in ((psx.ERR_BAD_ARGUMENT, dict(beams=2, keep=0)), (psx.ERR_UNSUPPORTED, dict(beams=2, keep=129)),
                       (psx.ERR_BAD_ARGUMENT, dict(beams=2, keep=2, finished=torch.zeros(4, dtype=torch.bool, device="cuda"), finished_token=100))):
        with pytest.raises(psx.PsxError) as e:
            ctx.beam_select(x, s, **kw)
        assert e.value.status == status
    with pytest.raises(psx.PsxError):
        ctx.beam_select(torch.zeros(65, 4, device="cuda"), torch.zeros(65, device="cuda"), 65, 2)
    assert ctx.beam_select(x[:0], s[:0], 2, 2)["tokens"].shape == (0, 2)


def test_more_pairs_of_a_group_than_there_may_be_are_refused():
    import torch
    ctx, x = gh.ctx(), torch.zeros(64, device="cuda")  # (refused ahead of any launch: the logits do not exist)
    for beams, vocab in ((64, 2 ** 25 + 1), (3, 2 ** 30), (1, 2 ** 30 + 1)):
        assert ctx._lib.psx_b200_beam_select(ctx._ctx, None, x.data_ptr(), 1, beams, vocab, vocab, x.data_ptr(), None, 0, 4, x.data_ptr(),
                                             x.data_ptr(), x.data_ptr(), None) == psx.ERR_UNSUPPORTED


# ---- states ---------------------------------------------------------------------------------------------------------------
def _moved(x, parents, lengths, per):
    groups, beams = parents.shape
    y = x.copy()
    for g in range(groups):
        for j in range(beams):
            p = int(parents[g, j])
            if 0 <= p < beams:
                n = x.shape[2] if lengths is None else min(x.shape[2], -(-max(int(lengths[g * beams + p]), 0) // per))
                y[g * beams + j, :, :n] = x[g * beams + p, :, :n]
    return y


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 13, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("with_lengths", [False, True])
def test_states_follow_their_beams(beams, with_lengths):
    import torch
    rng = np.random.RandomState(beams)
    groups, positions = 3, 45
    # widths of 16, 8, 4 and 1 bytes, a base that is only 4-byte aligned, a scale for every 16 tokens
    shapes = [((2, positions, 16), np.uint8, 1, 0), ((1, positions, 8), np.uint8, 1, 0), ((3, 3), np.float32, 16, 0), ((1, positions, 3), np.uint8, 1, 0),
              ((2, positions, 12), np.float32, 1, 1), ((2, 700, 64), np.float32, 1, 0)]
    parents = rng.randint(0, beams, (groups, beams)).astype(np.int64)
    parents[0] = np.arange(beams)[::-1]      # a permutation: every row is read and written
    parents[2, 0] = [-1, beams, 2 ** 40][beams % 3]   # not a beam: the row stays
    lengths = rng.choice([-3, 0, 1, 16, 17, positions, positions + 9, 2 ** 60], groups * beams).astype(np.int64) if with_lengths else None
    states, want = [], []
    for shape, kind, per, shift in shapes:
        x = rng.randint(0, 255, (groups * beams,) + shape).astype(kind)
        flat = torch.zeros(x.size + 16, dtype=torch.from_numpy(x).dtype, device="cuda")
        t = flat[shift:shift + x.size].view(x.shape)
        t.copy_(torch.from_numpy(x))
        states.append((t, per))
        want.append(_moved(x, parents, lengths, per))
    gh.ctx().reorder_states(torch.from_numpy(parents).cuda(), states, None if lengths is None else torch.from_numpy(lengths).cuda())
    torch.cuda.synchronize()
    for (t, _), w in zip(states, want):
        assert (t.cpu().numpy() == w).all()


def test_many_states_and_states_of_nothing():
    import torch
    parents = torch.tensor([[1, 0]], device="cuda")
    states = [torch.full((2, 1, 4, 3), float(i), device="cuda") for i in range(130)]
    for i, s in enumerate(states):
        s[1] = -i
    gh.ctx().reorder_states(parents, states + [torch.zeros(2, 0, 4, 3, device="cuda"), torch.zeros(2, 3, 0, 3, device="cuda"), torch.zeros(2, 3, 4, 0, device="cuda")])
    torch.cuda.synchronize()
    for i, s in enumerate(states):
        assert (s[0] == -i).all() and (s[1] == i).all()
    gh.ctx().reorder_states(parents, [])
    gh.ctx().reorder_states(parents[:0], [torch.zeros(0, 1, 4, 3, device="cuda")])


def test_captured_states_follow_the_parents_of_the_replay():
    import torch
    ctx = psx.Context(0)
    parents, x = torch.tensor([[1, 2, 0]], device="cuda"), torch.arange(3 * 40, device="cuda", dtype=torch.float32).view(3, 1, 40, 1)
    first = x.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ctx.reorder_states(parents, [x])
    graph.replay()
    torch.cuda.synchronize()
    assert (x == first[[1, 2, 0]]).all()
    parents.copy_(torch.tensor([[0, 0, 0]]))
    graph.replay()
    torch.cuda.synchronize()
    assert (x == first[[1, 1, 1]]).all()


def test_refusals_of_the_states():
    import torch
    ctx, parents, x = gh.ctx(), torch.zeros((2, 2), dtype=torch.int64, device="cuda"), torch.zeros(4, 2, 8, 4, device="cuda")
    for bad in (x[:3], x.transpose(1, 2), x[0], x.cpu()):
        with pytest.raises(ValueError):
            ctx.reorder_states(parents, [bad])
    with pytest.raises(ValueError):
        ctx.reorder_states(parents.int(), [x])
    lengths = torch.zeros(4, dtype=torch.int64, device="cuda")
    both = torch.zeros(4 * 64 + 8, device="cuda")
    for states, given in (([x, x], None), ([both[:256].view(4, 2, 8, 4), both[8:264].view(4, 2, 8, 4)], None), ([lengths.view(4, 1, 1)], lengths),
                          ([parents.view(4, 1, 1)], None), ([(x, 0)], None)):
        with pytest.raises(psx.PsxError) as e:
            ctx.reorder_states(parents, states, lengths=given)
        assert e.value.status == psx.ERR_BAD_ARGUMENT
    with pytest.raises(psx.PsxError) as e:
        ctx.reorder_states(torch.zeros((1, 65), dtype=torch.int64, device="cuda"), [torch.zeros(65, 1, 1, device="cuda")])
    assert e.value.status == psx.ERR_UNSUPPORTED


def test_a_refused_call_moves_no_state():
    import torch
    ctx, parents = gh.ctx(), torch.tensor([[1, 0], [1, 0]], device="cuda")
    states = [torch.arange(4.0, device="cuda").view(4, 1, 1) for _ in range(64)]
    described = (psx.binding.BeamState * 65)(*[psx.binding.BeamState(s.data_ptr(), 1, 1, 4, 1) for s in states])
    described[64] = psx.binding.BeamState(1 << 46, 1 << 30, 1, 1, 1)  # (does not exist; groups x heads of all is beyond 2^31)
    call = lambda count: ctx._lib.psx_b200_reorder_states(ctx._ctx, None, described, count, 2, 2, parents.data_ptr(), None)
    assert call(65) == psx.ERR_UNSUPPORTED and call(65537) == psx.ERR_UNSUPPORTED and call(2 ** 62) == psx.ERR_UNSUPPORTED
    torch.cuda.synchronize()
    assert all((s.flatten() == torch.arange(4.0, device="cuda")).all() for s in states)


# Strongly peaked rows: the largest logit's term is 1 and what the others add, r, is small.  In units of 2^-24 of the sum: the terms of r are off by 80 r
# as above; the thread that holds the 1 rounds what it adds to it, four times in that chunk and three in its joins, then once for each of eight chunks, a
# unit each: 15.  Joins and the logarithm are in double precision.  Together 80 r + 16.
@pytest.mark.parametrize("gap", [5.0, 12.0, 14.0, 17.0, 20.0, 40.0])
@pytest.mark.parametrize("groups,vocab", [(1, 50257), (40, 8192), (3, 151936), (1, 1000)])
def test_peaked_rows(gap, groups, vocab):
    rng = np.random.RandomState(int(gap))
    beams = 4
    logits = (rng.randn(groups * beams, vocab) * 0.5).astype(np.float32)
    logits[np.arange(groups * beams), rng.randint(0, vocab, groups * beams)] = np.float32(gap + 3)
    out = _run(logits, np.zeros(groups * beams, dtype=np.float32), beams, beams)
    value = _values(logits, np.zeros(groups * beams, dtype=np.float32), beams)
    for g in range(groups):
        best = value[g].max(1)
        rest = np.expm1(-best)                       # r of each beam
        slack = (80 * rest + 16) * 2.0 ** -24
        at, tokens = out["parents"][g], out["tokens"][g]
        assert (np.abs(out["scores"][g] - value[g, at, tokens]) <= slack[at] + 2.0 ** -24 * np.abs(value[g, at, tokens])).all()
        if rest.max() < 0.3:                          # every beam's best is ahead of every other candidate
            assert sorted(at.tolist()) == [0, 1, 2, 3] and (tokens == value[g].argmax(1)[at]).all()
            assert (np.diff(best[at]) <= 2 * slack.max()).all()


def test_a_token_that_is_nearly_certain_has_its_own_logarithm():
    # beams whose best token leaves 2^-26 and less to the others: the values differ by less than a float's step at 1, and are in order
    rest = -18.0 - np.arange(8) * 0.5
    logits = np.full((8, 5000), -200.0, dtype=np.float32)
    logits[:, 2500] = rest
    logits[:, 10] = 0.0
    scores = np.zeros(8, dtype=np.float32)
    for rows in (np.arange(8), np.arange(8)[::-1], np.array([3, 7, 0, 5, 1, 6, 2, 4])):
        out = _run(logits[rows], scores, 8, 8)
        assert (out["tokens"] == 10).all()
        assert (rows[out["parents"][0]] == np.arange(8)[::-1]).all()
        want = -np.log1p(np.exp(np.float64(rest[::-1])))
        assert (np.abs(out["scores"][0] - want) <= 100 * 2.0 ** -24 * np.abs(want)).all()
