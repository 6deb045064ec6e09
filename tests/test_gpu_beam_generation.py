"""Generation with beams over a cache in 8 bits, as a program runs it: packed prompts through prompt_attention, their keys and values
into the cache (store_cache_8bit), then step after step the LM head (lm_head_logits), the choice (beam_select), the states that
follow the beams (reorder_states: the cache, its scales and the token histories) and one new position per beam (store_cache_8bit,
decode_attention_8bit).  Every call is held to its restatement on the inputs that the run gives it."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx
import test_gpu_beams as beams_test
import test_gpu_cache_8bit as cache_test
import test_gpu_prompt_attention as prompt_test

pytestmark = pytest.mark.gpu
GROUPS, BEAMS, HEADS, KV_HEADS, DIM, VOCAB, MOST, BLOCK, EOS = 3, 4, 4, 2, 32, 2003, 128, 16, 7
ROWS, WIDTH = GROUPS * BEAMS, HEADS * DIM


class _Model:
    """One attention layer between an embedding and its transpose as the head."""

    def __init__(self, dtype, seed):
        import torch
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.embed = torch.randn(VOCAB, WIDTH, generator=gen, device="cuda")
        self.qkv = torch.randn(WIDTH, (HEADS + 2 * KV_HEADS) * DIM, generator=gen, device="cuda") * WIDTH ** -0.5
        self.dtype = getattr(torch, dtype)

    def project(self, tokens):
        x = (self.embed[tokens] @ self.qkv).to(self.dtype).view(len(tokens), HEADS + 2 * KV_HEADS, DIM)
        return x[:, :HEADS], x[:, HEADS:HEADS + KV_HEADS], x[:, HEADS + KV_HEADS:]

    def hidden(self, tokens, context):
        return (self.embed[tokens] + context.float().reshape(len(tokens), WIDTH)).contiguous()


def _numbers(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_generation_with_beams(dtype):
    import torch
    ctx, model = psx.Context(0), _Model(dtype, 1)
    rng = np.random.RandomState(2)
    lengths = [5, 37, 70]
    at = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    prompt = torch.from_numpy(rng.randint(0, VOCAB, at[-1])).cuda()
    q, k, v = model.project(prompt)
    context, status = ctx.prompt_attention(q, k, v, torch.from_numpy(at).cuda())
    want, most, value = prompt_test._attention(_numbers(q), _numbers(k), _numbers(v), at, at, DIM ** -0.5, True, 0)
    assert int(status) == 0
    assert (np.abs(_numbers(context) - want) <= prompt_test._slack(dtype, most, value, DIM, max(lengths)) + prompt_test.HALF_STEP[dtype] * np.abs(want)).all()

    # The prompt of a group goes into its first row; the beams take it over with the first choice.
    cache = psx.Cache8bit.empty(ROWS, KV_HEADS, MOST, DIM, BLOCK)
    counts = np.zeros(ROWS, dtype=np.int64)
    counts[::BEAMS] = lengths
    offsets, cached = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64), np.zeros(ROWS, dtype=np.int64)
    state = [(np.zeros((ROWS, KV_HEADS, MOST, DIM)), np.zeros((ROWS, KV_HEADS, MOST // BLOCK))) for _ in range(2)]

    def store(keys, values, offsets, cached):
        status = ctx.store_cache_8bit(cache, keys, values, torch.from_numpy(offsets).cuda(), torch.from_numpy(cached).cuda())
        assert (status == 0).all()
        for i, x in enumerate((keys, values)):
            state[i] = cache_test._store(*state[i], _numbers(x), offsets, cached, BLOCK)

    def check_cache():
        codes, scales = cache_test._parts(cache)
        for i in range(2):
            assert (codes[i] == state[i][0]).all() and (scales[i] == state[i][1]).all()

    store(k, v, offsets, cached)
    check_cache()
    held = torch.from_numpy(counts).cuda()                      # positions that each row holds
    history = torch.full((ROWS, 1, MOST), -1, dtype=torch.int64, device="cuda")
    for g in range(GROUPS):
        history[g * BEAMS, 0, :lengths[g]] = prompt[at[g]:at[g + 1]]
    last = torch.from_numpy(at[1:] - 1).cuda()
    hidden = model.hidden(prompt[last], context[last]).repeat_interleave(BEAMS, 0)
    scores = torch.full((GROUPS, BEAMS), -np.inf, device="cuda")
    scores[:, 0] = 0.0
    finished = torch.zeros(ROWS, dtype=torch.bool, device="cuda")

    for step in range(8):
        logits = ctx.lm_head_logits(hidden, model.embed)
        if step < 3:  # (no end before the fourth token)
            logits[:, EOS] = -np.inf
        else:         # (every group's best beam may end)
            logits[::BEAMS, EOS] = logits[::BEAMS].amax(1) + 0.5
        chosen = ctx.beam_select(logits, scores.view(-1), BEAMS, BEAMS, finished=finished, finished_token=EOS)
        values = beams_test._values(logits.cpu().numpy(), scores.view(-1).cpu().numpy(), BEAMS, finished.cpu().numpy(), EOS)
        beams_test._check({name: x.cpu().numpy() for name, x in chosen.items()}, values, BEAMS)

        parents, tokens = chosen["parents"], chosen["tokens"].view(-1)
        source = (parents + torch.arange(GROUPS, device="cuda")[:, None] * BEAMS).view(-1)
        moved = [beams_test._moved(x, parents.cpu().numpy(), held.cpu().numpy(), per) for x, per in
                 ((state[0][0], 1), (state[0][1], BLOCK), (state[1][0], 1), (state[1][1], BLOCK), (history.cpu().numpy(), 1))]
        ctx.reorder_states(parents, cache.states() + [history], lengths=held)
        state[:] = [(moved[0], moved[1]), (moved[2], moved[3])]
        check_cache()
        assert (history.cpu().numpy() == moved[4]).all()
        held = held[source]
        finished = finished[source] | (tokens == EOS)
        scores = chosen["scores"].contiguous()

        history[torch.arange(ROWS), 0, held] = tokens
        q, k, v = model.project(tokens)
        store(k, v, np.arange(ROWS + 1, dtype=np.int64), held.cpu().numpy())
        check_cache()
        held = held + 1
        context = ctx.decode_attention_8bit(q.reshape(ROWS, HEADS, 1, DIM).contiguous(), cache, held)
        want, most, value = cache_test._attention(_numbers(q).reshape(ROWS, HEADS, 1, DIM), cache, held.cpu().numpy(), DIM ** -0.5, True, 0)
        slack, half_step = cache_test._tolerance(dtype, most, value, DIM, MOST)
        assert (np.abs(_numbers(context) - want) <= slack + half_step * np.abs(want)).all()
        hidden = model.hidden(tokens, context)
    assert finished.any() and (history[:, 0, :5] >= 0).all()


def test_a_step_is_captured_as_a_whole():
    import torch
    ctx, model = psx.Context(0), _Model("bfloat16", 3)
    gen = torch.Generator(device="cuda").manual_seed(4)

    def new_state():
        cache = psx.Cache8bit.empty(ROWS, KV_HEADS, MOST, DIM, BLOCK)
        length = 40
        k, v = (torch.randn(ROWS * length, KV_HEADS, DIM, generator=gen, device="cuda").bfloat16() for _ in range(2))
        ctx.store_cache_8bit(cache, k, v, torch.arange(ROWS + 1, device="cuda") * length, torch.zeros(ROWS, dtype=torch.int64, device="cuda"))
        return dict(cache=cache, held=torch.full((ROWS,), length, dtype=torch.int64, device="cuda"), scores=-torch.rand(ROWS, generator=gen, device="cuda"),
                    tokens=torch.randint(0, VOCAB, (ROWS,), generator=gen, device="cuda"), offsets=torch.arange(ROWS + 1, device="cuda"))

    def step(s):
        q, k, v = model.project(s["tokens"])
        ctx.store_cache_8bit(s["cache"], k, v, s["offsets"], s["held"])
        s["held"] += 1
        context = ctx.decode_attention_8bit(q.reshape(ROWS, HEADS, 1, DIM).contiguous(), s["cache"], s["held"])
        logits = ctx.lm_head_logits(model.hidden(s["tokens"], context), model.embed)
        chosen = ctx.beam_select(logits, s["scores"], BEAMS, BEAMS)
        ctx.reorder_states(chosen["parents"], s["cache"].states(), lengths=s["held"])
        s["scores"].copy_(chosen["scores"].view(-1))
        s["tokens"].copy_(chosen["tokens"].view(-1))

    eager = new_state()
    copied = dict(cache=psx.Cache8bit(*[t.clone() for t, _ in eager["cache"].states()], block=BLOCK), **{n: eager[n].clone() for n in ("held", "scores", "tokens", "offsets")})
    start = {n: copied[n].clone() for n in ("held", "scores", "tokens")}
    first = [t.clone() for t, _ in copied["cache"].states()]
    step(copied)  # (every buffer has its size)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(copied)
    for name, x in start.items():
        copied[name].copy_(x)
    for (t, _), x in zip(copied["cache"].states(), first):
        t.copy_(x)
    for _ in range(5):
        step(eager)
        graph.replay()
    torch.cuda.synchronize()
    for name in ("held", "scores", "tokens"):
        assert (eager[name] == copied[name]).all()
    for (a, _), (b, _) in zip(eager["cache"].states(), copied["cache"].states()):
        assert (a.view(torch.uint8) == b.view(torch.uint8)).all()
