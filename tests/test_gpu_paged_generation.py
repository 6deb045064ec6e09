"""Generation with beams over a cache in pages, as a program runs it: prompts through rotate_heads (norm, rotation, pages) and prompt_attention, beams that
share their prompt's pages (fork_pages), then step after step the LM head (lm_head_logits), the choice (beam_select) and its log-probabilities
(token_log_probs), the rows that follow their beams (fork_pages), room for the new position (extend_pages), the new queries and keys (rotate_heads) and their
attention over the pages (decode_attention_pages); at the end drafts that are taken back (release_pages) and the pools brought together
(compact_pages).  Attention and log-probabilities are held to their formulas on what went in, kept by this program row by row without any page."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx
import test_gpu_decode_attention_pages as pages_test
import test_gpu_prompt_attention as prompt_test
import test_gpu_token_log_probs as score_test

pytestmark = pytest.mark.gpu
GROUPS, BEAMS, HEADS, KV_HEADS, DIM, VOCAB, SIZE, LAYERS = 3, 4, 4, 2, 32, 2003, 16, 2
ROWS, WIDTH = GROUPS * BEAMS, HEADS * DIM


def _numbers(t):
    return t.double().cpu().numpy()


class _Model:
    """Attention layers between an embedding and its transpose as the head."""

    def __init__(self, dtype, seed):
        import torch
        gen = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
        self.dtype = getattr(torch, dtype)
        self.embed = normal(VOCAB, WIDTH)
        self.qkv = [normal(WIDTH, (HEADS + 2 * KV_HEADS) * DIM) * WIDTH ** -0.5 for _ in range(LAYERS)]
        self.weights = [[(1 + 0.1 * normal(DIM)).to(self.dtype) for _ in range(2)] for _ in range(LAYERS)]
        self.frequencies = 10000.0 ** (-torch.arange(0, DIM, 2, dtype=torch.float64, device="cuda") / DIM)

    def project(self, layer, hidden):
        x = (hidden @ self.qkv[layer]).to(self.dtype).view(len(hidden), HEADS + 2 * KV_HEADS, DIM)
        return x[:, :HEADS], x[:, HEADS:HEADS + KV_HEADS], x[:, HEADS + KV_HEADS:]


class _Run:
    def __init__(self, ctx, model, num_pages, max_pages):
        import torch
        self.ctx, self.model = ctx, model
        self.table = psx.PageTable.empty(ROWS, max_pages, num_pages, SIZE)
        self.caches = [psx.PagedCache(self.table, *[torch.full((num_pages, KV_HEADS, SIZE, DIM), float("nan"), device="cuda", dtype=model.dtype) for _ in range(2)])
                       for _ in range(LAYERS)]
        self.pools = [p for c in self.caches for p in c.pools()]
        self.one_each = torch.arange(ROWS + 1, device="cuda")
        self.one = torch.ones(ROWS, dtype=torch.int64, device="cuda")

    def step(self, tokens, first):
        """One new position of every row: its logits, and what every layer's attention saw."""
        ctx, model = self.ctx, self.model
        status = ctx.extend_pages(self.table, self.one, self.pools)
        hidden, seen = model.embed[tokens], []
        for layer, cache in enumerate(self.caches):
            q, k, v = model.project(layer, hidden)
            q, k, stored = ctx.rotate_heads(q, k, v, offsets=self.one_each, first=first, frequencies=model.frequencies, q_weight=model.weights[layer][0],
                                            k_weight=model.weights[layer][1], cache=cache, keys_too=True)
            context = ctx.decode_attention_pages(q, cache)
            seen.append((q, k, v, context))
            hidden = hidden + context.float().view(ROWS, WIDTH)
        return ctx.lm_head_logits(hidden.contiguous(), model.embed), seen, status, stored


@pytest.mark.parametrize("dtype", ["bfloat16", "float32", "float16"])
def test_generation_with_beams(dtype):
    import torch
    ctx, model = psx.Context(0), _Model(dtype, 1)
    run = _Run(ctx, model, 64, 9)
    rng = np.random.RandomState(2)
    lengths = [5, 37, 64]
    counts = np.zeros(ROWS, dtype=np.int64)
    counts[::BEAMS] = lengths
    at = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda()
    prompt = torch.from_numpy(rng.randint(0, VOCAB, sum(lengths))).cuda()
    nothing = torch.zeros(ROWS, dtype=torch.int64, device="cuda")
    assert not ctx.extend_pages(run.table, torch.from_numpy(counts).cuda(), run.pools).any()
    kept = [[[np.zeros((0, KV_HEADS, DIM))] * 2 for _ in range(ROWS)] for _ in range(LAYERS)]  # a row's keys and values, by layer
    hidden = model.embed[prompt]
    ends = np.concatenate([[0], np.cumsum(counts)])
    for layer, cache in enumerate(run.caches):
        q, k, v = model.project(layer, hidden)
        q, k, status = ctx.rotate_heads(q, k, v, offsets=at, first=nothing, frequencies=model.frequencies, q_weight=model.weights[layer][0],
                                        k_weight=model.weights[layer][1], cache=cache, keys_too=True)
        assert not status.any()
        context, late = ctx.prompt_attention(q, k, v, at)
        assert int(late) == 0
        want, most, value = prompt_test._attention(_numbers(q), _numbers(k), _numbers(v), ends, ends, DIM ** -0.5, True, 0)
        assert (np.abs(_numbers(context) - want) <= prompt_test._slack(dtype, most, value, DIM, max(lengths)) + prompt_test.HALF_STEP[dtype] * np.abs(want)).all()
        hidden = hidden + context.float().view(-1, WIDTH)
        for b in range(ROWS):
            kept[layer][b] = [_numbers(x)[ends[b]:ends[b + 1]] for x in (k, v)]
    # every beam goes on from its group's prompt, in the same pages
    parents = torch.zeros((GROUPS, BEAMS), dtype=torch.int64, device="cuda")
    ctx.fork_pages(run.table, parents)
    kept = [[one[b // BEAMS * BEAMS] for b in range(ROWS)] for one in kept]
    assert int(run.table.references.sum()) == BEAMS * sum(-(-n // SIZE) for n in lengths) and int((run.table.references > 0).sum()) == sum(-(-n // SIZE) for n in lengths)
    last = torch.from_numpy(ends[1::BEAMS] - 1).cuda()
    logits = ctx.lm_head_logits(hidden[last].contiguous(), model.embed).repeat_interleave(BEAMS, 0)
    scores = torch.full((GROUPS, BEAMS), -np.inf, device="cuda")
    scores[:, 0] = 0.0
    for step in range(20):
        chosen = ctx.beam_select(logits, scores.view(-1), BEAMS, BEAMS)
        parents, tokens = chosen["parents"], chosen["tokens"].view(-1)
        source = (parents + torch.arange(GROUPS, device="cuda")[:, None] * BEAMS).view(-1)
        # the same choice, scored: a beam's score is its parent's and the token's log-probability
        scored = score_test._check(logits[source], tokens.cpu().numpy(), 3)
        before = scores.view(-1)[source].double()
        assert (chosen["scores"].view(-1).double() - (before + scored["log_probs"].double())).abs().max() <= 2.0 ** -22 * (1 + before.abs().max())
        scores = chosen["scores"].contiguous()
        ctx.fork_pages(run.table, parents)
        kept = [[one[b] for b in source.tolist()] for one in kept]
        first = run.table.lengths.clone()
        logits, seen, status, stored = run.step(tokens, first)
        assert not status.any() and not stored.any()
        for layer, (q, k, v, context) in enumerate(seen):
            for b in range(ROWS):
                kept[layer][b] = [np.concatenate([x, _numbers(new)[b:b + 1]]) for x, new in zip(kept[layer][b], (k, v))]
                keys, values = kept[layer][b]
                assert len(keys) == int(run.table.lengths[b])
                for h in range(HEADS):
                    one, group = _numbers(q)[b, h], h // (HEADS // KV_HEADS)
                    s = keys[:, group] @ one * DIM ** -0.5
                    w = np.exp(s - s.max())
                    want = (w / w.sum()) @ values[:, group]
                    most = (np.abs(keys[:, group]) @ np.abs(one)).max() * DIM ** -0.5
                    pages_test._near(context[b, h], want, dtype, pages_test._slack(dtype, most, np.abs(values[:, group]).max(), DIM, len(keys)))
    assert int((run.table.references > 1).sum()) > 0  # (prompts are still shared)
    # half of the groups are done; the others take back two positions; what is left fills the beginning of the pools, and goes on
    keep = run.table.lengths - 2
    keep[:BEAMS] = 0
    ctx.release_pages(run.table, keep)
    used = int(ctx.compact_pages(run.table, run.pools))
    assert used == int((run.table.references > 0).sum()) and (run.table.references[used:] == 0).all()
    for layer, cache in enumerate(run.caches):
        for b in range(BEAMS, ROWS):
            n = int(run.table.lengths[b])
            pages = run.table.pages[b, :-(-n // SIZE)].long()
            for x, want in zip(cache.pools(), kept[layer][b]):
                assert (_numbers(x[pages].transpose(1, 2).reshape(-1, KV_HEADS, DIM))[:n] == want[:n]).all()
    ctx.release_pages(run.table)
    assert not run.table.references.any()


def test_a_step_is_captured_as_a_whole():
    import torch
    ctx, model = psx.Context(0), _Model("bfloat16", 3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    one = _Run(ctx, model, 100, 9)
    ctx.extend_pages(one.table, torch.full((ROWS,), 40, dtype=torch.int64, device="cuda"), one.pools)
    for p in one.pools:
        p.copy_(torch.randn(p.shape, generator=gen, device="cuda"))
    tokens, scores = torch.randint(0, VOCAB, (ROWS,), generator=gen, device="cuda"), -torch.rand(ROWS, generator=gen, device="cuda")
    first = one.table.lengths.clone()

    def step():
        first.copy_(one.table.lengths)
        logits, _, _, _ = one.step(tokens, first)
        chosen = ctx.beam_select(logits, scores, BEAMS, BEAMS)
        source = (chosen["parents"] + torch.arange(GROUPS, device="cuda")[:, None] * BEAMS).view(-1)
        log_probs = ctx.token_log_probs(logits[source], chosen["tokens"].view(-1), top=2, entropy=True)
        ctx.fork_pages(one.table, chosen["parents"])
        scores.copy_(chosen["scores"].view(-1))
        tokens.copy_(chosen["tokens"].view(-1))
        return log_probs

    buffers = [one.table.pages, one.table.lengths, one.table.references, tokens, scores] + one.pools
    start = [x.clone() for x in buffers]
    want = []
    for _ in range(6):
        scored = step()
        want.append([x.clone() for x in buffers] + [scored["log_probs"].clone(), scored["entropy"].clone()])
    for x, y in zip(buffers, start):
        x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scored = step()
    for x, y in zip(buffers, start):
        x.copy_(y)
    for expected in want:
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(buffers + [scored["log_probs"], scored["entropy"]], expected):
            assert (x == y).all()


def test_pools_of_more_than_two_to_the_31_elements():
    """The same pages at the end of a pool of 4.4 GB and in a small one: every call leaves the same in both."""
    import torch
    ctx, gen = gh.ctx(), torch.Generator(device="cuda").manual_seed(6)
    size, kv_heads, dim, heads, many, few = 128, 8, 256, 16, 8400, 12
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda").bfloat16()
    lengths = torch.tensor([300, 300, 130, 1], device="cuda")
    small = torch.tensor([[9, 4, 11, 0], [9, 4, 11, 0], [7, 5, 0, 0], [10, 0, 0, 0]], dtype=torch.int32, device="cuda")  # (rows 0 and 1 share theirs)
    caches = []
    for pages, shift in ((few, 0), (many, many - few)):
        table = psx.PageTable(small + shift, lengths.clone(), torch.zeros(pages, dtype=torch.int32, device="cuda"), size)
        used = [9, 9, 4, 4, 11, 11, 7, 5, 10]
        table.references.index_add_(0, torch.tensor(used, device="cuda") + shift, torch.ones(len(used), dtype=torch.int32, device="cuda"))
        table.references[:shift] = 1  # (what lies below is taken)
        caches.append(psx.PagedCache(table, *[torch.empty(pages, kv_heads, size, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]))
    assert caches[1].key_pages.numel() > 2 ** 31
    for p in range(few):
        page = [normal(kv_heads, size, dim) for _ in range(2)]
        for cache in caches:
            cache.key_pages[p - few], cache.value_pages[p - few] = page[0], page[1]

    def same():
        torch.cuda.synchronize()
        a, b = caches
        assert (a.table.lengths == b.table.lengths).all() and (a.table.references == b.table.references[many - few:]).all()
        assert ((a.table.pages + (many - few) == b.table.pages)[:, :3] | (a.table.lengths[:, None] <= torch.arange(3, device="cuda") * size)).all()
        assert (a.key_pages == b.key_pages[many - few:]).all() and (a.value_pages == b.value_pages[many - few:]).all()

    one, qkv = torch.ones(4, dtype=torch.int64, device="cuda"), normal(4, heads + 2 * kv_heads, dim)
    results = []
    for cache in caches:
        first = cache.table.lengths.clone()
        status = ctx.extend_pages(cache.table, one, cache.pools())  # (row 0 gets a page of its own)
        q, _, stored = ctx.rotate_heads(qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], offsets=torch.arange(5, device="cuda"), first=first,
                                        frequencies=torch.rand(dim // 2, generator=torch.Generator().manual_seed(1), dtype=torch.float64).cuda(), cache=cache)
        results.append((status, stored, ctx.decode_attention_pages(q, cache)))
    assert not results[0][0].any() and not results[0][1].any() and torch.isfinite(results[0][2]).all()
    assert all((x == y).all() for x, y in zip(*results))
    same()
    big = caches[1]
    big.table.references[:many - few] = 0
    kept = [(big.key_pages[p.long()].clone(), big.value_pages[p.long()].clone()) for p in big.table.pages[:, :2]]
    assert int(ctx.compact_pages(big.table, big.pools())) == 7
    again = ctx.decode_attention_pages(q, big)
    assert (again == results[0][2]).all()
    for b in range(3):
        now = big.table.pages[b, :2].long()
        assert (now < 7).all() and (big.key_pages[now] == kept[b][0]).all() and (big.value_pages[now] == kept[b][1]).all()
