"""The operators of a generation loop over beams, an 8-bit cache and packed prompts, as a program calls them, and the same in
plain torch: the candidates of a beam search (`beam_select`), the states that follow the beams (`reorder`), new keys and values on
their way into a cache held in 8 bits (`store`), attention of new positions over that cache (`decode`), and attention of whole
prompts, packed one behind the other (`prompt`).  `own` says which of the two `run` computes."""
import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CODES = torch.float8_e4m3fn
VOCABULARIES = (49152, 50257, 128256, 151936, 262144)  # those of the benchmark's workloads, and an odd one


def listed():
    return [
        # one request, four beams, the odd vocabulary: what a single user waits for
        dict(name="beams-1x4", op="beam_select", groups=1, beams=4, vocab=50257, keep=8, masked=False, finished=False),
        # a server's batch: 64 requests of eight beams, a tenth of the vocabulary masked, some beams finished
        dict(name="beams-64x8", op="beam_select", groups=64, beams=8, vocab=151936, keep=16, masked=True, finished=True),
        # one request's 8-bit cache of one layer, early in the generation
        dict(name="reorder-1x4", op="reorder", groups=1, beams=4, kv_heads=8, head_dim=128, max_len=256, longest=200, layers=1, dtype="8bit", block=32),
        # 16 requests of four beams, two layers of an 8-bit cache
        dict(name="reorder-16x4", op="reorder", groups=16, beams=4, kv_heads=8, head_dim=128, max_len=2304, longest=2111, layers=2, dtype="8bit", block=32),
        # a decoding step: one new position for each of 64 rows, blocks half filled
        dict(name="store-step-64", op="store", batch=64, kv_heads=8, head_dim=128, max_len=2304, block=32, longest_new=1, cached=2048, dtype="bfloat16"),
        # prompts of different lengths on their way into the cache
        dict(name="store-prompt-24", op="store", batch=24, kv_heads=8, head_dim=128, max_len=4096, block=32, longest_new=3999, cached=0, dtype="float32"),
        # one request, grouped heads, a short cache
        dict(name="decode-1", op="decode", batch=1, heads=32, kv_heads=8, head_dim=128, q_len=1, max_len=1024, longest=777, block=32, window=0, dtype="bfloat16"),
        # four new positions at a time (a draft being checked), every head with keys of its own, fp32
        dict(name="decode-12-draft", op="decode", batch=12, heads=16, kv_heads=16, head_dim=64, q_len=4, max_len=2048, longest=1999, block=16, window=0, dtype="float32"),
        # a server's batch over long caches of different lengths, eight heads to a kv head
        dict(name="decode-64-long", op="decode", batch=64, heads=64, kv_heads=8, head_dim=128, q_len=1, max_len=8192, longest=8191, block=64, window=0, dtype="bfloat16"),
        # one short prompt
        dict(name="prompt-1-short", op="prompt", batch=1, heads=8, kv_heads=2, head_dim=64, longest=100, prefix=0, window=0, dtype="float16"),
        # fp32 prompts that continue a cached prefix, a head dimension that is no power of two
        dict(name="prompt-5-fp32", op="prompt", batch=5, heads=16, kv_heads=4, head_dim=96, longest=1501, prefix=300, window=0, dtype="float32"),
        # long packed prompts: the sizes at which a server spends its time
        dict(name="prompt-2-long", op="prompt", batch=2, heads=32, kv_heads=8, head_dim=128, longest=8192, prefix=0, window=0, dtype="bfloat16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("beam_select", "reorder", "store", "decode", "prompt"))
    if op == "beam_select":
        beams, vocab = rng.choice((1, 2, 3, 4, 5, 8, 12, 16)), rng.choice(VOCABULARIES + (_spread(rng, 1000, 200000),))
        groups = _spread(rng, 1, max(1, min(256, 75_000_000 // (beams * vocab))))
        return dict(op=op, groups=groups, beams=beams, vocab=vocab, keep=min(vocab, beams * rng.choice((1, 2))), masked=rng.random() < 0.5,
                    finished=rng.random() < 0.5)
    if op == "reorder":
        beams, kv_heads, head_dim = rng.choice((2, 3, 4, 5, 8, 16)), rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 128))
        longest, dtype = _spread(rng, 1, 2048), rng.choice(("8bit", "float32", "bfloat16"))
        width = {"8bit": 1, "float32": 4, "bfloat16": 2}[dtype]
        groups = _spread(rng, 1, max(1, min(64, 160_000_000 // (beams * kv_heads * head_dim * (longest + 64) * width))))
        return dict(op=op, groups=groups, beams=beams, kv_heads=kv_heads, head_dim=head_dim, max_len=longest + rng.randrange(0, 64), longest=longest,
                    layers=rng.choice((1, 2)), dtype=dtype, block=rng.choice((16, 32, 64)))
    if op == "store":
        kv_heads, head_dim, longest_new = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 80, 128)), rng.choice((1, 1, _spread(rng, 2, 4000)))
        cached = rng.choice((0, _spread(rng, 1, 2048)))
        batch = _spread(rng, 1, max(1, min(96, 98_000_000 // (kv_heads * head_dim * (longest_new + 64)))))
        return dict(op=op, batch=batch, kv_heads=kv_heads, head_dim=head_dim, max_len=cached + longest_new + rng.randrange(0, 70), block=rng.choice((16, 32, 64)),
                    longest_new=longest_new, cached=cached, dtype=rng.choice(sorted(TYPES)))
    if op == "decode":
        kv_heads, group, q_len = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 1, 2))
        head_dim, longest = rng.choice((64, 80, 96, 128, 256)), max(q_len, _spread(rng, 1, 16384))
        batch = _spread(rng, 1, max(1, min(96, 500_000_000 // (kv_heads * head_dim * (longest + 64)))))
        return dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, q_len=q_len, max_len=longest + rng.randrange(0, 70),
                    longest=longest, block=rng.choice((16, 32, 64)), window=rng.choice((0, 0, 0, _spread(rng, 1, 4096))), dtype=rng.choice(sorted(TYPES)))
    kv_heads, group, dtype = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 8)), rng.choice(sorted(TYPES))
    longest = _spread(rng, 1, 4096)
    most = 32 * 8192 * 8192 // 4 // (3 if dtype == "float32" else 1)
    batch = _spread(rng, 1, max(1, min(32, most // (kv_heads * group * longest * longest))))
    return dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, head_dim=rng.choice((64, 80, 96, 128)), longest=longest,
                prefix=rng.choice((0, 0, _spread(rng, 1, 500))), window=rng.choice((0, 0, 0, _spread(rng, 1, 2048))), dtype=dtype)


def _lengths(count, longest, word):
    """`count` lengths up to `longest`, which is the first; the same ones for the same numbers."""
    rng = random.Random("%s %d %d" % (word, count, longest))
    return [longest] + [rng.randint(1 + longest // 2 if rng.random() < 0.8 else 1, max(1, longest)) for _ in range(count - 1)]


def _offsets(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return total


def _prompt_lengths(case):
    q = _lengths(case["batch"], case["longest"], "prompt")
    p = _lengths(case["batch"], case["prefix"], "prefix") if case["prefix"] else [0] * case["batch"]
    return q, [a + b for a, b in zip(q, p)]


def _cache(case, rows, gen, filled=True):
    """Codes and scales of a cache as earlier steps left them."""
    blocks = -(-case["max_len"] // case["block"])
    shape = (rows, case["kv_heads"], case["max_len"], case["head_dim"])

    def codes():
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * 110).clamp(-448, 448).to(CODES)

    def scales():
        return torch.exp2(torch.randint(-9, -6, shape[:2] + (blocks,), generator=gen, device="cuda").float())

    if not filled:
        empty = [torch.zeros(shape, device="cuda").to(CODES), torch.zeros(shape[:2] + (blocks,), device="cuda")]
        return empty + [x.clone() for x in empty]
    return [codes(), scales(), codes(), scales()]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    def whole(values):
        return torch.tensor(values, dtype=torch.int64, device="cuda")

    state = dict(case=case, seed=seed)
    if op == "beam_select":
        rows = case["groups"] * case["beams"]
        logits = normal(rows, case["vocab"]).mul_(3.0)
        if case["masked"]:  # tokens that a grammar or a filter took out
            logits.masked_fill_(torch.rand(logits.shape, generator=gen, device="cuda") < 0.1, -math.inf)
        scores = -torch.rand(rows, generator=gen, device="cuda") * 20
        finished = None
        if case["finished"]:
            finished = torch.rand(rows, generator=gen, device="cuda") < 0.15
            scores = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.05, torch.full_like(scores, -math.inf), scores)
            scores.view(case["groups"], -1)[:, 0] = -3.0  # (one beam at least is alive)
        return dict(state, logits=logits, scores=scores, finished=finished)
    if op == "reorder":
        rows = case["groups"] * case["beams"]
        parents = torch.randint(0, case["beams"], (case["groups"], case["beams"]), generator=gen, device="cuda")
        stays = torch.rand(parents.shape, generator=gen, device="cuda") < 0.3
        parents = torch.where(stays, torch.arange(case["beams"], device="cuda"), parents)
        lengths = whole(_lengths(case["groups"], case["longest"], "reorder")).repeat_interleave(case["beams"])
        if case["dtype"] == "8bit":
            states = [s for _ in range(case["layers"]) for s in _cache(case, rows, gen)]
            per = [1, case["block"]] * (2 * case["layers"])
        else:
            states = [normal(rows, case["kv_heads"], case["max_len"], case["head_dim"]).to(TYPES[case["dtype"]]) for _ in range(2 * case["layers"])]
            per = [1] * len(states)
        return dict(state, parents=parents, lengths=lengths, states=states, per=per)
    if op == "store":
        new = _lengths(case["batch"], case["longest_new"], "store")
        cached = [min(n, case["max_len"] - m) for n, m in zip(_lengths(case["batch"], case["cached"], "cached"), new)] if case["cached"] else [0] * case["batch"]
        total = sum(new)
        keys, values = (normal(total, case["kv_heads"], case["head_dim"]).to(TYPES[case["dtype"]]) for _ in range(2))
        return dict(state, cache=_cache(case, case["batch"], gen, filled=case["cached"] > 0), keys=keys, values=values, offsets=whole(_offsets(new)),
                    cached=whole(cached))
    if op == "decode":
        lengths = [max(n, case["q_len"]) for n in _lengths(case["batch"], case["longest"], "decode")]
        q = normal(case["batch"], case["heads"], case["q_len"], case["head_dim"]).to(TYPES[case["dtype"]])
        return dict(state, q=q, cache=_cache(case, case["batch"], gen), lengths=whole([min(n, case["max_len"]) for n in lengths]))
    q_lens, k_lens = _prompt_lengths(case)
    kind = TYPES[case["dtype"]]
    return dict(state, q=normal(sum(q_lens), case["heads"], case["head_dim"]).to(kind), k=normal(sum(k_lens), case["kv_heads"], case["head_dim"]).to(kind),
                v=normal(sum(k_lens), case["kv_heads"], case["head_dim"]).to(kind), q_offsets=whole(_offsets(q_lens)), k_offsets=whole(_offsets(k_lens)))


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _beam_select(s):
    c = s["case"]
    groups, beams, vocab, keep = c["groups"], c["beams"], c["vocab"], c["keep"]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    value = (s["scores"].double()[:, None] - lse) + x
    if s["finished"] is not None:
        ended = s["finished"][:, None]
        value = torch.where(ended, -math.inf, value)
        value[:, 0] = torch.where(ended[:, 0], s["scores"].double(), value[:, 0])  # (the token that a finished beam repeats is 0)
    value, at = value.view(groups, beams * vocab).sort(dim=1, descending=True, stable=True)
    value, at = value[:, :keep], at[:, :keep]
    gone = value == -math.inf
    status = torch.where(gone.all(1), 5, 0).to(torch.int32)
    return dict(scores=value.float(), parents=torch.where(gone, -1, at // vocab), tokens=torch.where(gone, -1, at % vocab), status=status)


def _reorder_one(x, per, source, lengths):
    taken = x[source]
    positions = torch.arange(x.shape[2], device=x.device)
    valid = positions[None, :] * per < lengths[source][:, None]
    valid = valid[:, None, :].expand(x.shape[:3])
    x[valid] = taken[valid]
    return x


def _reorder(s):
    parents, beams = s["parents"], s["case"]["beams"]
    source = (parents + torch.arange(parents.shape[0], device=parents.device)[:, None] * beams).reshape(-1)
    raw = [x.view(torch.uint8) if x.dtype == CODES else x for x in s["states"]]
    return [_reorder_one(x, per, source, s["lengths"]).view(y.dtype) for x, y, per in zip(raw, s["states"], s["per"])]


def _store_one(codes, scales, new, offsets, cached, block, longest_new):
    """The blocks that the new tokens touch: their scale, the codes that stay brought to it, and the new ones."""
    batch, kv_heads, max_len, head_dim = codes.shape
    counts = offsets[1:] - offsets[:-1]
    window = -(-(longest_new + block - 1) // block)  # blocks that one row's new tokens can touch
    blocks = (cached // block)[:, None] + torch.arange(window, device=codes.device)
    position = (blocks * block)[:, :, None] + torch.arange(block, device=codes.device)  # (batch, window, block)
    ends = (cached + counts)[:, None, None]
    old = position < cached[:, None, None]
    fresh = (position >= cached[:, None, None]) & (position < ends)
    touched = fresh.any(2)
    rows = torch.arange(batch, device=codes.device)
    at = position.clamp(max=max_len - 1)
    held = codes.view(torch.uint8)[rows[:, None, None], :, at].view(CODES).float()  # (batch, window, block, kv, dim)
    token = (offsets[:-1, None, None] + position - cached[:, None, None]).clamp(0, max(new.shape[0] - 1, 0))
    given = new[token].float()
    size = torch.where(fresh[..., None, None], given.abs(), 0.0).amax((2, 4))  # (batch, window, kv)
    size = size.nan_to_num(0.0)
    mantissa, exponent = torch.frexp(size)
    exponent = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-100)  # 448 = 0.875 * 2^9
    scale = torch.where(size > 0, torch.exp2(exponent.float()), 2.0 ** -100)
    index = blocks.clamp(max=scales.shape[2] - 1)
    before = scales[rows[:, None], :, index]
    scale = torch.where(old.any(2)[..., None], torch.maximum(scale, before), scale)
    rate = (before / scale)[:, :, None, :, None]
    kept = (held * rate).to(CODES)
    made = (given / scale[:, :, None, :, None]).clamp(-448, 448).to(CODES)
    result = torch.where(fresh[..., None, None], made.view(torch.uint8), kept.view(torch.uint8))
    write = (old | fresh) & touched[..., None]
    r, w, p = write.nonzero(as_tuple=True)
    codes.view(torch.uint8)[r, :, position[r, w, p]] = result[r, w, p]
    r, w = touched.nonzero(as_tuple=True)
    scales[r, :, blocks[r, w]] = scale[r, w]
    return codes, scales


def _store(s):
    c = s["case"]
    kc, ks, vc, vs = s["cache"]
    out = _store_one(kc, ks, s["keys"], s["offsets"], s["cached"], c["block"], c["longest_new"])
    out += _store_one(vc, vs, s["values"], s["offsets"], s["cached"], c["block"], c["longest_new"])
    return list(out)


def _decode(s):
    c = s["case"]
    kc, ks, vc, vs = s["cache"]
    batch, kv_heads, max_len, head_dim = kc.shape
    group, q_len = c["heads"] // kv_heads, c["q_len"]
    spread = lambda x: x.repeat_interleave(c["block"], 2)[:, :, :max_len, None]  # noqa: E731
    keys, values = kc.float() * spread(ks), vc.float() * spread(vs)
    q = s["q"].float().view(batch, kv_heads, group * q_len, head_dim)
    score = torch.matmul(q, keys.transpose(2, 3)).view(batch, kv_heads, group, q_len, max_len) * head_dim ** -0.5
    position = torch.arange(max_len, device=q.device)
    own_position = s["lengths"][:, None] - q_len + torch.arange(q_len, device=q.device)  # (batch, q_len)
    hidden = position[None, None, :] > own_position[:, :, None]
    if c["window"]:
        hidden |= position[None, None, :] + c["window"] <= own_position[:, :, None]
    score = score.masked_fill(hidden[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    weight = (weight / weight.sum(-1, keepdim=True)).view(batch, kv_heads, group * q_len, max_len)
    return torch.matmul(weight, values).view(s["q"].shape).to(s["q"].dtype)


def _padded(x, offsets, longest):
    """(batch, longest, ...) of packed rows; what lies behind a sequence holds some other row."""
    at = offsets[:-1, None] + torch.arange(longest, device=x.device)
    return x[at.clamp(max=x.shape[0] - 1)]


def _prompt(s):
    c = s["case"]
    q_lens, k_lens = _prompt_lengths(c)
    most_q, most_k = max(q_lens), max(k_lens)
    group = c["heads"] // c["kv_heads"]
    q = _padded(s["q"], s["q_offsets"], most_q).float().view(c["batch"], most_q, c["kv_heads"], group, c["head_dim"]).permute(0, 2, 3, 1, 4)
    k = _padded(s["k"], s["k_offsets"], most_k).float().permute(0, 2, 3, 1)[:, :, None]
    v = _padded(s["v"], s["k_offsets"], most_k).float().permute(0, 2, 1, 3)[:, :, None]
    q_count, k_count = (o[1:] - o[:-1] for o in (s["q_offsets"], s["k_offsets"]))
    place = torch.arange(most_q, device=q.device)[None, :] + (k_count - q_count)[:, None]  # a query's position among the keys
    position = torch.arange(most_k, device=q.device)
    hidden = position[None, None, :] > place[:, :, None]
    if c["window"]:
        hidden |= position[None, None, :] + c["window"] <= place[:, :, None]
    score = torch.matmul(q, k).mul_(c["head_dim"] ** -0.5)
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score, v).div_(total)
    real = torch.arange(most_q, device=q.device)[None, :] < q_count[:, None]
    return out.permute(0, 3, 1, 2, 4).reshape(c["batch"], most_q, c["heads"], c["head_dim"])[real].to(s["q"].dtype)


# ---- the framework's calls ------------------------------------------------------------------------------------------------
_held = {}


def _context():
    """The handle that a program makes once."""
    if "context" not in _held:
        import pulsatrix_b200 as psx
        _held["context"] = psx.Context(0)
        _held["cache"] = psx.Cache8bit
    return _held["context"]


def _run_own(s):
    c, context = s["case"], _context()
    if c["op"] == "beam_select":
        return context.beam_select(s["logits"], s["scores"], c["beams"], c["keep"], finished=s["finished"], finished_token=0)
    if c["op"] == "reorder":
        context.reorder_states(s["parents"], list(zip(s["states"], s["per"])), lengths=s["lengths"])
        return s["states"]
    if c["op"] == "store":
        context.store_cache_8bit(_held["cache"](*s["cache"], block=c["block"]), s["keys"], s["values"], s["offsets"], s["cached"])
        return s["cache"]
    if c["op"] == "decode":
        return context.decode_attention_8bit(s["q"], _held["cache"](*s["cache"], block=c["block"]), s["lengths"], window=c["window"])
    return context.prompt_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], window=c["window"])[0]


def run(state):
    if own:
        return _run_own(state)
    return {"beam_select": _beam_select, "reorder": _reorder, "store": _store, "decode": _decode, "prompt": _prompt}[state["case"]["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def _visible(q_lens, k_lens, window):
    """Pairs of a query and a key that it sees."""
    pairs = 0
    for q, k in zip(q_lens, k_lens):
        first = k - q + 1  # keys that the first query sees
        if window == 0 or window >= k:
            pairs += q * first + q * (q - 1) // 2
        else:
            pairs += sum(min(window, first + i) for i in range(q))
    return pairs


def _width(case):
    return {"float32": 4, "8bit": 1}.get(case["dtype"], 2)


def work(case):
    op = case["op"]
    if op == "beam_select":
        logits = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": 4 * logits + 20 * case["groups"] * case["keep"], "flops": 5 * logits}
    if op == "reorder":  # some 70 % of the rows change; what they come from is about 70 % of the rows too
        lengths = _lengths(case["groups"], case["longest"], "reorder")
        row = case["kv_heads"] * case["head_dim"] * _width(case) * 2 * case["layers"]
        return {"bytes": sum(1.2 * case["beams"] * n * row for n in lengths), "flops": 0}
    if op == "store":
        tokens = sum(_lengths(case["batch"], case["longest_new"], "store")) * case["kv_heads"] * case["head_dim"] * 2
        return {"bytes": tokens * (_width(case) + 1), "flops": 3 * tokens}
    if op == "decode":
        lengths = _lengths(case["batch"], case["longest"], "decode")
        seen = [min(n, case["window"] + case["q_len"] - 1) if case["window"] else n for n in lengths]
        cache = sum(seen) * case["kv_heads"] * (2 * case["head_dim"] + 8 / case["block"])
        return {"bytes": cache + 2 * case["batch"] * case["heads"] * case["q_len"] * case["head_dim"] * _width(case),
                "flops": 4 * sum(seen) * case["heads"] * case["q_len"] * case["head_dim"]}
    q_lens, k_lens = _prompt_lengths(case)
    values = 2 * sum(q_lens) * case["heads"] + 2 * sum(k_lens) * case["kv_heads"]
    return {"bytes": values * case["head_dim"] * _width(case), "flops": 4 * case["head_dim"] * case["heads"] * _visible(q_lens, k_lens, case["window"])}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------------
def _exact_beams(s):
    c = s["case"]
    out = dict(scores=[], parents=[], tokens=[], status=[])
    for g in range(c["groups"]):
        rows = slice(g * c["beams"], (g + 1) * c["beams"])
        log_p = torch.log_softmax(s["logits"][rows].double(), 1)
        total = s["scores"][rows].double()[:, None] + log_p
        if s["finished"] is not None:
            for b in s["finished"][rows].nonzero().flatten().tolist():
                total[b] = -math.inf
                total[b, 0] = s["scores"][g * c["beams"] + b].double()
        flat = total.flatten()
        order = torch.topk(flat, c["keep"]).indices
        values = flat[order]
        none = torch.isinf(values)
        out["scores"].append(values)
        out["parents"].append(torch.where(none, -1, order // c["vocab"]))
        out["tokens"].append(torch.where(none, -1, order % c["vocab"]))
        out["status"].append(5 if bool(none.all()) else 0)
    return dict(scores=torch.stack(out["scores"]), parents=torch.stack(out["parents"]), tokens=torch.stack(out["tokens"]),
                status=torch.tensor(out["status"], dtype=torch.int32))


def _exact_heads(q, keys, values, first, window):
    """One sequence: q (heads, n, d), keys and values (kv heads, m, d) in 64 bits; `first`: the first query's position."""
    heads, n, d = q.shape
    group = heads // keys.shape[0]
    place = first + torch.arange(n, device=q.device)
    position = torch.arange(keys.shape[1], device=q.device)
    seen = position[None, :] <= place[:, None]
    if window:
        seen &= position[None, :] > place[:, None] - window
    bias = torch.zeros(seen.shape, dtype=torch.float64, device=q.device).masked_fill(~seen, -math.inf)
    out = torch.empty_like(q)
    for h in range(heads):
        out[h] = torch.softmax(q[h] @ keys[h // group].T / math.sqrt(d) + bias, 1) @ values[h // group]
    return out


def _exact_decode(s):
    c = s["case"]
    kc, ks, vc, vs = s["cache"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        block = torch.arange(n, device="cuda") // c["block"]
        keys = kc[b, :, :n].double() * ks[b][:, block, None].double()
        values = vc[b, :, :n].double() * vs[b][:, block, None].double()
        out[b] = _exact_heads(s["q"][b].double(), keys, values, n - c["q_len"], c["window"])
    return out


def _exact_prompt(s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at, to = s["q_offsets"].tolist(), s["k_offsets"].tolist()
    for b in range(len(at) - 1):
        q, k, v = s["q"][at[b]:at[b + 1]], s["k"][to[b]:to[b + 1]], s["v"][to[b]:to[b + 1]]
        first = (to[b + 1] - to[b]) - (at[b + 1] - at[b])
        out[at[b]:at[b + 1]] = _exact_heads(*(x.double().transpose(0, 1) for x in (q, k, v)), first, s["case"]["window"]).transpose(0, 1)
    return out


def _exact_reorder(s):
    c, out = s["case"], []
    lengths, parents = s["lengths"].tolist(), s["parents"].tolist()
    for x, per in zip(s["states"], s["per"]):
        x = x.float()
        y = x.clone()
        for g in range(c["groups"]):
            for j, p in enumerate(parents[g]):
                n = -(-lengths[g * c["beams"] + p] // per)
                y[g * c["beams"] + j, :, :n] = x[g * c["beams"] + p, :, :n]
        out.append(y)
    return out


def _exact_store(s):
    c = s["case"]
    offsets, cached = s["offsets"].tolist(), s["cached"].tolist()
    out = []
    for new, codes, scales in ((s["keys"], *s["cache"][:2]), (s["values"], *s["cache"][2:])):
        codes, scales = codes.double(), scales.double()
        for b in range(c["batch"]):
            for start in range(cached[b] // c["block"] * c["block"], cached[b] + offsets[b + 1] - offsets[b], c["block"]):
                low, high = max(start, cached[b]), min(start + c["block"], cached[b] + offsets[b + 1] - offsets[b])
                x = new[offsets[b] + low - cached[b]:offsets[b] + high - cached[b]].double().transpose(0, 1)  # (kv, tokens, dim)
                need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448)))
                if start < cached[b]:
                    before = scales[b, :, start // c["block"]]
                    need = torch.maximum(need, before)
                    part = codes[b, :, start:low] * (before / need)[:, None, None]
                    codes[b, :, start:low] = part.float().to(CODES).double()
                codes[b, :, low:high] = (x / need[:, None, None]).float().to(CODES).double()
                scales[b, :, start // c["block"]] = need
        out += [codes, scales]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store" and case["batch"] * case["longest_new"] > 200_000:
        return None
    return {"beam_select": _exact_beams, "reorder": _exact_reorder, "store": _exact_store, "decode": _exact_decode, "prompt": _exact_prompt}[case["op"]](s)
