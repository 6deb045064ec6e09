"""The operators of generation over a cache in pages, as a program calls them, and the same in plain torch: bookkeeping of pages in a
step of beams (`branch`: what a draft got wrong is taken back, rows follow their beams, the next tokens get room) and when a pool is to
shrink (`compact`), queries and keys on their way from a projection into the cache (`rotate`: norm per head, rotation, store), attention of
new positions over pages (`pages`), and log-probabilities of given tokens with entropy and the top alternatives (`score`).  `own` says
which of the two `run` computes."""
import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
VOCABULARIES = (49152, 50257, 128256, 151936, 262144)  # those of the benchmark's workloads, and an odd one
EPS = 1e-6


def listed():
    return [
        # one request's token, what a single user waits for: the odd vocabulary, five alternatives
        dict(name="score-1", op="score", rows=1, vocab=50257, top=5, dtype="float32", masked=False),
        # a server's step: the sampled tokens of 64 rows, twenty alternatives, a tenth of the vocabulary masked
        dict(name="score-64", op="score", rows=64, vocab=151936, top=20, dtype="bfloat16", masked=True),
        # prompts that are scored: every position's next token
        dict(name="score-2048", op="score", rows=2048, vocab=151936, top=1, dtype="bfloat16", masked=False),
        # one new position of one request, grouped heads
        dict(name="rotate-1", op="rotate", batch=1, heads=32, kv_heads=8, head_dim=128, rotated=128, interleaved=False, norm=True, longest_new=1,
             cached=776, page_size=16, keys_too=False, dtype="bfloat16"),
        # prompts of different lengths: keys into the pages, and packed for the attention of prompts
        dict(name="rotate-12", op="rotate", batch=12, heads=32, kv_heads=8, head_dim=128, rotated=128, interleaved=False, norm=True, longest_new=2111,
             cached=0, page_size=32, keys_too=True, dtype="bfloat16"),
        # one request, grouped heads, a short cache
        dict(name="pages-1", op="pages", batch=1, heads=32, kv_heads=8, head_dim=128, q_len=1, longest=777, page_size=16, window=0, dtype="bfloat16"),
        # four new positions at a time (a draft being checked), every head with keys of its own, fp32
        dict(name="pages-12-draft", op="pages", batch=12, heads=16, kv_heads=16, head_dim=64, q_len=4, longest=1999, page_size=16, window=0, dtype="float32"),
        # a server's batch over long caches of different lengths, eight heads to a kv head
        dict(name="pages-64-long", op="pages", batch=64, heads=64, kv_heads=8, head_dim=128, q_len=1, longest=8191, page_size=64, window=0, dtype="bfloat16"),
        # one request of four beams, one layer
        dict(name="branch-1x4", op="branch", groups=1, beams=4, kv_heads=8, head_dim=128, page_size=16, longest=200, draft=1, layers=1, dtype="bfloat16"),
        # 16 requests of eight beams over long prompts, two layers
        dict(name="branch-16x8", op="branch", groups=16, beams=8, kv_heads=8, head_dim=128, page_size=64, longest=8000, draft=3, layers=2, dtype="bfloat16"),
        # a small pool from which half of the rows are gone
        dict(name="compact-256", op="compact", rows=8, num_pages=256, kv_heads=4, head_dim=64, page_size=16, layers=1, dtype="float32"),
        # a server's pool after a peak: two layers of 4096 pages, scattered
        dict(name="compact-4096", op="compact", rows=96, num_pages=4096, kv_heads=8, head_dim=128, page_size=32, layers=2, dtype="bfloat16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("score", "rotate", "pages", "branch", "compact"))
    dtype = rng.choice(sorted(TYPES))
    width = 4 if dtype == "float32" else 2
    if op == "score":
        vocab = rng.choice(VOCABULARIES + (_spread(rng, 1000, 200000),))
        rows = _spread(rng, 1, max(1, min(2048, 600_000_000 // (vocab * width))))
        return dict(op=op, rows=rows, vocab=vocab, top=rng.choice((0, 1, 5, 8, 20, 64)), dtype=dtype, masked=rng.random() < 0.5)
    if op == "rotate":
        kv_heads, group, head_dim = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 96, 128, 256))
        longest_new = rng.choice((1, 1, _spread(rng, 2, 4000)))
        batch = _spread(rng, 1, max(1, min(96, 60_000_000 // (kv_heads * (group + 2) * head_dim * longest_new))))
        cached = rng.choice((0, _spread(rng, 1, max(2, min(100000, 100_000_000 // (batch * kv_heads * head_dim))))))
        return dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, rotated=rng.choice((head_dim, head_dim, head_dim // 2)),
                    interleaved=rng.random() < 0.25, norm=rng.random() < 0.7, longest_new=longest_new, cached=cached,
                    page_size=rng.choice((16, 32, 64, 128)), keys_too=rng.random() < 0.5, dtype=dtype)
    if op == "pages":
        kv_heads, group, q_len = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 1, 2))
        head_dim, longest = rng.choice((64, 80, 96, 128, 256)), max(q_len, _spread(rng, 1, 16384))
        batch = _spread(rng, 1, max(1, min(96, 800_000_000 // (kv_heads * head_dim * (longest + 64) * width))))
        return dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, q_len=q_len, longest=longest,
                    page_size=rng.choice((16, 32, 64, 128)), window=rng.choice((0, 0, 0, _spread(rng, 1, 4096))), dtype=dtype)
    kv_heads, head_dim, page_size = rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 128)), rng.choice((16, 32, 64, 128))
    page = kv_heads * head_dim * page_size * width
    layers = rng.choice((1, 2, 4))
    if op == "branch":
        beams, longest = rng.choice((2, 3, 4, 5, 8, 16)), _spread(rng, 1, 8000)
        groups = _spread(rng, 1, max(1, min(64, 1_500_000_000 // (2 * layers * page * (longest // page_size + 2 * beams)))))
        return dict(op=op, groups=groups, beams=beams, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, longest=longest, draft=rng.choice((1, 1, 3, 5)),
                    layers=layers, dtype=dtype)
    return dict(op=op, rows=_spread(rng, 1, 256), num_pages=_spread(rng, 64, max(65, min(8192, 1_000_000_000 // (2 * layers * page)))), kv_heads=kv_heads,
                head_dim=head_dim, page_size=page_size, layers=layers, dtype=dtype)


def _lengths(count, longest, word):
    """`count` lengths up to `longest`, which is the first; the same ones for the same numbers."""
    rng = random.Random("%s %d %d" % (word, count, longest))
    return [longest] + [rng.randint(1 + longest // 2 if rng.random() < 0.8 else 1, max(1, longest)) for _ in range(count - 1)]


def _offsets(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return total


def _page_counts(lengths, page_size):
    return [-(-n // page_size) for n in lengths]


def _scattered(counts, num_pages, rng):
    """A page table whose rows use `counts` pages of their own, anywhere in the pool, and the pages' references."""
    pages = rng.sample(range(num_pages), sum(counts))
    table, references, at = [], [0] * num_pages, 0
    for n in counts:
        table.append(pages[at:at + n])
        at += n
    for p in pages:
        references[p] = 1
    return table, references


def _compact_rows(case):
    """Rows that hold half of a pool."""
    rng = random.Random("compact %d %d" % (case["rows"], case["num_pages"]))
    half, rows = case["num_pages"] // 2, case["rows"]
    cuts = sorted(rng.randint(0, half) for _ in range(rows - 1))
    counts = [b - a for a, b in zip([0] + cuts, cuts + [half])]
    return [max(0, n * case["page_size"] - rng.randrange(case["page_size"])) for n in counts]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op = case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    def whole(values, kind=torch.int64):
        return torch.tensor(values, dtype=kind, device="cuda")

    kind = TYPES[case["dtype"]]
    state = dict(case=case, seed=seed)
    if op == "score":
        logits = torch.empty((case["rows"], case["vocab"]), dtype=kind, device="cuda")
        for rows in logits.split(256):
            x = normal(*rows.shape).mul_(3.0)
            if case["masked"]:  # tokens that a grammar or a filter took out
                x.masked_fill_(torch.rand(x.shape, generator=gen, device="cuda") < 0.1, -math.inf)
            rows.copy_(x)
        tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda")
        likely = torch.rand(case["rows"], generator=gen, device="cuda") < 0.7  # (most are likely ones, as a model's own are)
        tokens = torch.where(likely, logits.argmax(1), tokens)
        return dict(state, logits=logits, tokens=tokens)

    def pool(num_pages, filled=True):
        shape = (num_pages, case["kv_heads"], case["page_size"], case["head_dim"])
        if not filled:
            return torch.zeros(shape, dtype=kind, device="cuda")
        pages = torch.empty(shape, dtype=kind, device="cuda")
        for some in pages.split(max(1, (1 << 26) // pages[0].numel())):
            some.copy_(normal(*some.shape))
        return pages

    def book(lengths, table, references):
        most = max(1, max(len(row) for row in table))
        return dict(table=whole([row + [-1] * (most - len(row)) for row in table], torch.int32), lengths=whole(lengths),
                    references=whole(references, torch.int32))

    if op == "rotate":
        new = _lengths(case["batch"], case["longest_new"], "rotate")
        first = _lengths(case["batch"], case["cached"], "cached") if case["cached"] else [0] * case["batch"]
        lengths = [a + b for a, b in zip(first, new)]
        counts = _page_counts(lengths, case["page_size"])
        num_pages = sum(counts) + 3
        heads, kv_heads, dims = case["heads"], case["kv_heads"], case["head_dim"]
        total = sum(new)
        qkv = normal(total, heads + 2 * kv_heads, dims).to(kind)  # one projection
        weights = [(1 + 0.2 * normal(dims)).to(kind) for _ in range(2)] if case["norm"] else [None, None]
        frequencies = 10000.0 ** (-torch.arange(0, case["rotated"], 2, dtype=torch.float64, device="cuda") / case["rotated"])
        return dict(state, q=qkv[:, :heads], k=qkv[:, heads:heads + kv_heads], v=qkv[:, heads + kv_heads:], q_weight=weights[0], k_weight=weights[1],
                    frequencies=frequencies, offsets=whole(_offsets(new)), first=whole(first), keys=pool(num_pages, False), values=pool(num_pages, False),
                    **book(lengths, *_scattered(counts, num_pages, rng)))
    if op == "pages":
        lengths = [max(n, case["q_len"]) for n in _lengths(case["batch"], case["longest"], "pages")]
        counts = _page_counts(lengths, case["page_size"])
        num_pages = sum(counts) + 3
        q = normal(case["batch"] * case["q_len"], case["heads"], case["head_dim"]).to(kind)
        return dict(state, q=q, keys=pool(num_pages), values=pool(num_pages), **book(lengths, *_scattered(counts, num_pages, rng)))
    if op == "branch":
        # a group's beams share their prompt's whole pages and hold what they wrote themselves: a draft, part of which is kept
        beams, size, draft = case["beams"], case["page_size"], case["draft"]
        keep = [n for n in _lengths(case["groups"], case["longest"], "branch") for _ in range(beams)]
        lengths = [n + draft for n in keep]
        most = -(-(case["longest"] + draft) // size)
        num_pages = sum(n // size + beams * (2 + draft // size + 1) for n in keep[::beams]) + 8
        pages = iter(rng.sample(range(num_pages), num_pages))
        references, table = [0] * num_pages, []
        for g in range(case["groups"]):
            shared = [next(pages) for _ in range(keep[g * beams] // size)]
            for b in range(beams):
                row = shared + [next(pages) for _ in range(-(-lengths[g * beams] // size) - len(shared))]
                table.append(row + [-1] * (most - len(row)))
                for p in row:
                    references[p] += 1
        parents = torch.randint(0, beams, (case["groups"], beams), generator=gen, device="cuda")
        stays = torch.rand(parents.shape, generator=gen, device="cuda") < 0.3
        parents = torch.where(stays, torch.arange(beams, device="cuda"), parents)
        return dict(state, parents=parents, keep=whole(keep), new=whole([draft] * len(keep)), pools=[pool(num_pages) for _ in range(2 * case["layers"])],
                    table=whole(table, torch.int32), lengths=whole(lengths), references=whole(references, torch.int32))
    lengths = _compact_rows(case)
    held = book(lengths, *_scattered(_page_counts(lengths, case["page_size"]), case["num_pages"], rng))
    return dict(state, pools=[pool(case["num_pages"]) for _ in range(2 * case["layers"])], before=(held["table"].clone(), held["references"].clone()), **held)


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _score(s):
    c = s["case"]
    out = dict(log_probs=[], entropy=[], top_log_probs=[], top_tokens=[])
    for logits, tokens in zip(s["logits"].split(512), s["tokens"].split(512)):
        x = logits.double()
        top = x.amax(1, keepdim=True)
        gap = x - top
        weight = torch.exp(gap)
        total = weight.sum(1, keepdim=True)
        lse = torch.log(total)
        out["log_probs"].append((gap.gather(1, tokens[:, None]) - lse)[:, 0].float())
        gap.masked_fill_(gap == -math.inf, 0.0)
        out["entropy"].append((lse - (weight * gap).sum(1, keepdim=True) / total)[:, 0].float())
        if c["top"]:
            values, at = logits.float().sort(dim=1, descending=True, stable=True)
            values, at = values[:, :c["top"]].double(), at[:, :c["top"]]
            out["top_log_probs"].append(((values - top) - lse).float())
            out["top_tokens"].append(torch.where(values == -math.inf, -1, at))
    return {name: torch.cat(parts) for name, parts in out.items() if parts}


def _positions(offsets, first, total):
    """Row and position of every token of a packed batch."""
    row = torch.repeat_interleave(torch.arange(first.shape[0], device=first.device), offsets[1:] - offsets[:-1], output_size=total)
    return row, first[row] + torch.arange(total, device=first.device) - offsets[row]


def _rotated(x, weight, angle, c):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turned, rest = x[..., :c["rotated"]], x[..., c["rotated"]:]
    if c["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _rotate(s):
    c = s["case"]
    total = s["q"].shape[0]
    row, position = _positions(s["offsets"], s["first"], total)
    angle = position[:, None].double() * s["frequencies"]
    q = _rotated(s["q"], s["q_weight"], angle, c).to(s["q"].dtype)
    k = _rotated(s["k"], s["k_weight"], angle, c).to(s["q"].dtype)
    page, inside = s["table"][row, position // c["page_size"]].long(), position % c["page_size"]
    s["keys"][page, :, inside] = k
    s["values"][page, :, inside] = s["v"]
    return [q, s["keys"], s["values"]] + ([k] if c["keys_too"] else [])


def _pages(s):
    c = s["case"]
    batch, q_len, kv_heads, dims, size = c["batch"], c["q_len"], c["kv_heads"], c["head_dim"], c["page_size"]
    group = c["heads"] // kv_heads
    used = s["table"].clamp(min=0).long()
    span = used.shape[1] * size
    rows = max(1, (1 << 30) // (span * kv_heads * dims))
    out = []
    position = torch.arange(span, device="cuda")
    for b in range(0, batch, rows):
        take = used[b:b + rows]
        keys, values = (x[take].float().transpose(1, 2).reshape(take.shape[0], kv_heads, span, dims) for x in (s["keys"], s["values"]))
        q = s["q"].view(batch, q_len, kv_heads, group, dims)[b:b + rows].float().permute(0, 2, 1, 3, 4).reshape(-1, kv_heads, q_len * group, dims)
        score = torch.matmul(q, keys.transpose(2, 3)).view(-1, kv_heads, q_len, group, span) * dims ** -0.5
        place = s["lengths"][b:b + rows, None] - q_len + torch.arange(q_len, device="cuda")
        hidden = position > place[:, :, None]
        if c["window"]:
            hidden |= position + c["window"] <= place[:, :, None]
        score = score.masked_fill(hidden[:, None, :, None], -math.inf)
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        weight = (weight / weight.sum(-1, keepdim=True)).view(-1, kv_heads, q_len * group, span)
        context = torch.matmul(weight, values).view(-1, kv_heads, q_len, group, dims).permute(0, 2, 1, 3, 4)
        out.append(context.reshape(-1, c["heads"], dims).to(s["q"].dtype))
    return torch.cat(out)


def _used(lengths, most, size):
    return torch.arange(most, device=lengths.device) * size < lengths[:, None]


def _count(table, used, num_pages):
    """How many entries in use name each page."""
    return torch.zeros(num_pages, dtype=torch.int32, device=table.device).index_add_(0, table[used].long(), torch.ones_like(table[used]))


def _branch(s):
    size, table, lengths, references = s["case"]["page_size"], s["table"], s["lengths"], s["references"]
    rows, most = table.shape
    num_pages = references.shape[0]
    # what the draft got wrong
    lengths.copy_(torch.minimum(lengths, s["keep"]))
    # rows that follow their beams
    beams = s["parents"].shape[1]
    source = (s["parents"] + torch.arange(s["parents"].shape[0], device="cuda")[:, None] * beams).reshape(-1)
    taken, held = table[source], lengths[source]
    lengths.copy_(held)
    used = _used(lengths, most, size)
    table.copy_(torch.where(used, taken, table))
    references.copy_(_count(table, used, num_pages))
    # room for the next tokens; a shared last page is copied, but by the last row that goes on from it where nobody else holds it
    row = torch.arange(rows, device="cuda")
    partly = (lengths % size != 0) & (s["new"] > 0)
    last = torch.where(partly, table[row, (lengths // size).clamp(max=most - 1)].long(), 0)
    writers = torch.zeros(num_pages, dtype=torch.int64, device="cuda").index_add_(0, last[partly], torch.ones_like(last[partly]))
    final = torch.full((num_pages,), -1, dtype=torch.int64, device="cuda").scatter_reduce_(0, last[partly], row[partly], "amax")
    copies = partly & (references[last] > 1) & ~((writers[last] == references[last]) & (final[last] == row))
    fits = (s["new"] >= 0) & (lengths + s["new"] <= most * size)
    after = lengths + s["new"]
    need = torch.where(fits, (after + size - 1) // size - (lengths + size - 1) // size + copies.long(), 0)
    end = need.cumsum(0)
    free = (references == 0).nonzero()[:, 0]
    fits &= (need == 0) | (end <= free.shape[0])
    need, copies = torch.where(fits, need, 0), copies & fits
    who = torch.repeat_interleave(row, need)
    slot = torch.arange(who.shape[0], device="cuda") - (end - need)[who]
    given = free[:who.shape[0]]
    old, new = last[copies], given[(end - need)[copies]]
    part = torch.arange(size, device="cuda")[None] < (lengths % size)[copies][:, None]
    which, position = part.nonzero(as_tuple=True)
    for pool in s["pools"]:
        pool[new[which], :, position] = pool[old[which], :, position]
    at = (lengths[who] + size - 1) // size - copies[who].long() + slot
    table[who, at] = given.int()
    lengths.copy_(torch.where(fits, after, lengths))
    references.copy_(_count(table, _used(lengths, most, size), num_pages))
    return [table, lengths, references, torch.where(fits, 0, 64).int()] + s["pools"]


def _compact(s):
    table, references = s["table"], s["references"]
    table.copy_(s["before"][0])  # (a pass begins where the first one did; the pages that it moved are still there)
    references.copy_(s["before"][1])
    in_use = references > 0
    count = in_use.sum()
    page = torch.arange(references.shape[0], device="cuda")
    old, new = page[in_use & (page >= count)], page[~in_use & (page < count)]
    for pool in s["pools"]:
        pool[new] = pool[old]
    moved_to = page.clone()
    moved_to[old] = new
    used = _used(s["lengths"], table.shape[1], s["case"]["page_size"])
    table.copy_(torch.where(used, moved_to[table.clamp(min=0).long()].int(), table))
    references[new] = references[old]
    references[old] = 0
    return [table, references, count.reshape(1)] + s["pools"]


# ---- the framework's calls ------------------------------------------------------------------------------------------------
_held = {}


def _context():
    """The handle that a program makes once."""
    if "context" not in _held:
        import pulsatrix_b200 as psx
        _held["context"] = psx.Context(0)
        _held["table"], _held["cache"] = psx.PageTable, psx.PagedCache
    return _held["context"]


def _run_own(s):
    c, context = s["case"], _context()
    if c["op"] == "score":
        scored = context.token_log_probs(s["logits"], s["tokens"], top=c["top"], entropy=True)
        return {name: scored[name] for name in ("log_probs", "entropy", "top_log_probs", "top_tokens") if scored[name] is not None}
    table = _held["table"](s["table"], s["lengths"], s["references"], c["page_size"])
    if c["op"] == "rotate":
        cache = _held["cache"](table, s["keys"], s["values"])
        q, k, _ = context.rotate_heads(s["q"], s["k"], s["v"], offsets=s["offsets"], first=s["first"], frequencies=s["frequencies"], q_weight=s["q_weight"],
                                       k_weight=s["k_weight"], eps=EPS, interleaved=c["interleaved"], cache=cache, keys_too=c["keys_too"])
        return [q, s["keys"], s["values"]] + ([k] if c["keys_too"] else [])
    if c["op"] == "pages":
        return context.decode_attention_pages(s["q"], _held["cache"](table, s["keys"], s["values"]), q_len=c["q_len"], window=c["window"])
    if c["op"] == "branch":
        context.release_pages(table, s["keep"])
        context.fork_pages(table, s["parents"])
        status = context.extend_pages(table, s["new"], s["pools"])
        return [s["table"], s["lengths"], s["references"], status] + s["pools"]
    s["table"].copy_(s["before"][0])
    s["references"].copy_(s["before"][1])
    used = context.compact_pages(table, s["pools"])
    return [s["table"], s["references"], used] + s["pools"]


def run(state):
    if own:
        return _run_own(state)
    return {"score": _score, "rotate": _rotate, "pages": _pages, "branch": _branch, "compact": _compact}[state["case"]["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    op, width = case["op"], 4 if case["dtype"] == "float32" else 2
    if op == "score":
        logits = case["rows"] * case["vocab"]
        return {"bytes": width * logits + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * logits}
    row = case["kv_heads"] * case["head_dim"] * width  # of a position's keys, or values
    if op == "rotate":
        total = sum(_lengths(case["batch"], case["longest_new"], "rotate"))
        queries = case["heads"] * case["head_dim"] * width
        return {"bytes": total * (2 * queries + (5 if case["keys_too"] else 4) * row), "flops": 10 * total * (case["heads"] + case["kv_heads"]) * case["head_dim"]}
    if op == "pages":
        lengths = [max(n, case["q_len"]) for n in _lengths(case["batch"], case["longest"], "pages")]
        seen = [min(n, case["window"] + case["q_len"] - 1) if case["window"] else n for n in lengths]
        return {"bytes": 2 * sum(seen) * row + 2 * case["batch"] * case["heads"] * case["q_len"] * case["head_dim"] * width,
                "flops": 4 * sum(seen) * case["heads"] * case["q_len"] * case["head_dim"]}
    if op == "branch":  # table entries are read and some written; some 70 % of the rows come from another one, whose last page they copy
        keep = _lengths(case["groups"], case["longest"], "branch")
        entries = sum(-(-n // case["page_size"]) for n in keep) * case["beams"]
        copied = sum(n % case["page_size"] for n in keep) * 0.6 * case["beams"]
        return {"bytes": 8 * entries + 2 * copied * row * 2 * case["layers"], "flops": 0}
    moved = sum(_page_counts(_compact_rows(case), case["page_size"])) // 2  # half of the pages in use lie behind the middle
    return {"bytes": 2 * moved * case["page_size"] * row * 2 * case["layers"] + 8 * case["num_pages"], "flops": 0}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------------
def _exact_score(s):
    c, out = s["case"], dict(log_probs=[], entropy=[], top_log_probs=[], top_tokens=[])
    for x, token in zip(s["logits"].split(64), s["tokens"].split(64)):
        log_p = torch.log_softmax(x.double(), 1)
        out["log_probs"].append(log_p.gather(1, token[:, None])[:, 0])
        out["entropy"].append(torch.special.entr(torch.exp(log_p)).sum(1))
        if c["top"]:
            bits = (x.float() + 0.0).view(torch.int32).long()
            rank = torch.where(bits < 0, -(bits & 0x7fffffff) - 1, bits) * 2 ** 30 - torch.arange(x.shape[1], device=x.device)
            at = torch.topk(rank, c["top"]).indices
            out["top_log_probs"].append(log_p.gather(1, at))
            out["top_tokens"].append(torch.where(torch.isinf(log_p.gather(1, at)), -1, at))
    return {name: torch.cat(parts) for name, parts in out.items() if parts}


def _exact_rotate(s):
    c = s["case"]
    dims, size, half = c["head_dim"], c["page_size"], c["rotated"] // 2
    keys, values = s["keys"].double(), s["values"].double()
    offsets, first, table = s["offsets"].tolist(), s["first"].tolist(), s["table"].long()

    def turned(x, weight, position):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / dims + EPS) * weight.double()
        pair = torch.arange(half, device="cuda")
        i, j = (2 * pair, 2 * pair + 1) if c["interleaved"] else (pair, pair + half)
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), position[:, None] * s["frequencies"][None])[:, None]
        z = torch.complex(x[..., i], x[..., j]) * turn
        x = x.clone()
        x[..., i], x[..., j] = z.real, z.imag
        return x

    q, k = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), torch.empty(s["k"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        own_tokens = slice(offsets[b], offsets[b + 1])
        position = torch.arange(first[b], first[b] + offsets[b + 1] - offsets[b], device="cuda")
        q[own_tokens] = turned(s["q"][own_tokens], s["q_weight"], position.double())
        k[own_tokens] = turned(s["k"][own_tokens], s["k_weight"], position.double())
        page = table[b][torch.div(position, size, rounding_mode="floor")]
        keys[page, :, position % size] = k[own_tokens]
        values[page, :, position % size] = s["v"][own_tokens].double()
    return [q, keys, values] + ([k] if c["keys_too"] else [])


def _exact_pages(s):
    c = s["case"]
    size, kv_heads, q_len, dims = c["page_size"], c["kv_heads"], c["q_len"], c["head_dim"]
    group = c["heads"] // kv_heads
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][b, :-(-n // size)].long()
        for h in range(kv_heads):
            keys, values = (x[pages, h].reshape(-1, dims)[:n].double() for x in (s["keys"], s["values"]))
            for i in range(q_len):
                end = n - q_len + i + 1
                begin = max(0, end - c["window"]) if c["window"] else 0
                q = s["q"][b * q_len + i, h * group:(h + 1) * group].double()
                out[b * q_len + i, h * group:(h + 1) * group] = torch.softmax(q @ keys[begin:end].T / math.sqrt(dims), 1) @ values[begin:end]
    return out


def _exact_branch(s):
    size = s["case"]["page_size"]
    table, lengths, references = s["table"].tolist(), s["lengths"].tolist(), s["references"].tolist()
    beams, most = s["parents"].shape[1], len(table[0])
    pools = [p.clone() for p in s["pools"]]

    def pages(b):
        return table[b][:-(-lengths[b] // size)]

    for b, keep in enumerate(s["keep"].tolist()):
        held = pages(b)
        lengths[b] = min(lengths[b], keep)
        for p in held[len(pages(b)):]:
            references[p] -= 1
    for g, chosen in enumerate(s["parents"].tolist()):
        before = [(pages(g * beams + p), lengths[g * beams + p]) for p in chosen]
        for j in range(beams):
            for p in pages(g * beams + j):
                references[p] -= 1
        for j, (held, n) in enumerate(before):
            table[g * beams + j][:len(held)] = held
            lengths[g * beams + j] = n
            for p in held:
                references[p] += 1
    new = s["new"].tolist()
    shared, free = list(references), [p for p, n in enumerate(references) if n == 0]
    going = {}
    for b in range(len(table)):
        if lengths[b] % size and new[b] > 0:
            going.setdefault(table[b][lengths[b] // size], []).append(b)
    status, asked, available = [], 0, len(free)
    for b in range(len(table)):
        filled, n = lengths[b] % size, lengths[b] + new[b]
        if n > most * size:
            status.append(64)
            continue
        wanted = list(range(-(-lengths[b] // size), -(-n // size)))
        last = table[b][lengths[b] // size] if filled and new[b] > 0 else None
        copied = last is not None and shared[last] > 1 and not (len(going[last]) == shared[last] and going[last][-1] == b)
        if copied:
            wanted.insert(0, lengths[b] // size)
        asked += len(wanted)
        if wanted and asked > available:
            status.append(64)
            continue
        for at in wanted:
            page = free.pop(0)
            references[page] += 1
            if copied and at == lengths[b] // size:
                references[last] -= 1
                for pool in pools:
                    pool[page, :, :filled] = pool[last, :, :filled]
            table[b][at] = page
        lengths[b] = n
        status.append(0)
    return [torch.tensor(table, dtype=torch.int32), torch.tensor(lengths), torch.tensor(references, dtype=torch.int32),
            torch.tensor(status, dtype=torch.int32)] + [p.double() for p in pools]


def _exact_compact(s):
    table, references, size = s["table"].tolist(), s["references"].tolist(), s["case"]["page_size"]
    count = sum(1 for n in references if n)
    movers = [p for p in range(count, len(references)) if references[p]]
    goals = [p for p in range(count) if not references[p]]
    goal = dict(zip(movers, goals))
    pools = [p.double() for p in s["pools"]]
    for a, b in goal.items():
        references[b], references[a] = references[a], 0
        for pool in pools:
            pool[b] = pool[a]
    for row, n in zip(table, s["lengths"].tolist()):
        for i in range(-(-n // size)):
            row[i] = goal.get(row[i], row[i])
    return [torch.tensor(table, dtype=torch.int32), torch.tensor(references, dtype=torch.int32), torch.tensor([count])] + pools


def exact(case, seed):
    width = 4 if case["dtype"] == "float32" else 2
    if case["op"] in ("branch", "compact"):  # (in pools of gigabytes the copies alone would take their time)
        s = prepare(case, seed)
        if sum(p.numel() for p in s["pools"]) * width > 2_000_000_000:
            return None
        return (_exact_branch if case["op"] == "branch" else _exact_compact)(s)
    return {"score": _exact_score, "rotate": _exact_rotate, "pages": _exact_pages}[case["op"]](prepare(case, seed))
