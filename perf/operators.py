"""The operators of a decode step for requests of unequal lengths, as cases to be timed and compared.

  plan    page_plan_hip: the pages that new tokens need, block tables, and the slot and position of every token, from request lengths
  store   rope_store_paged_hip: the prompts' queries rotated, their keys (rotated) and values stored to pages by the slot map
  attend  attention_paged_hip: one new token per request over the paged cache, its own key and value appended
  sample  sample_hip: the next tokens from logits with temperature, top-k, top-p and min-p, from given random numbers

Requests are rows of a batch; a row without a request is idle.  Pages are dealt in shuffled order, as a pool in use leaves them.
"""
import math

import torch

own = False
DEVICE = "cuda"
ROPE_THETA = 500000.0


# ------------------------------------------------------------------------------------------------- cases
def _plan(rows, page, max_pages, new_lo, new_hi, held_hi, pad=0):
    return {"op": "plan", "rows": rows, "page": page, "max_pages": max_pages, "new_lo": new_lo, "new_hi": new_hi, "held_hi": held_hi, "pad": pad}


def _store(heads, kv_heads, dim, page, rows, new_hi):
    return {"op": "store", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "rows": rows, "new_hi": new_hi}


def _attend(heads, kv_heads, dim, page, rows, len_lo, len_hi):
    return {"op": "attend", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "rows": rows, "len_lo": len_lo, "len_hi": len_hi}


def _sample(rows, vocab, kind):
    return {"op": "sample", "rows": rows, "vocab": vocab, "kind": kind}


def listed():
    cases = [
        # every step of a serving loop: one token for each of 48 requests, a few of them finished
        ("plan_step", _plan(48, 16, 512, 1, 1, 8000)),
        # ragged prompts come in beside requests that go on, in a batch padded to a fixed row count
        ("plan_prompts", _plan(100, 32, 256, 1, 2000, 0, pad=777)),
        # one short prompt of an 8B-shape model
        ("store_short", _store(32, 8, 128, 16, 1, 131)),
        # many ragged prompts of a 70B-shape model
        ("store_prompts", _store(64, 8, 128, 64, 9, 2048)),
        # one request, early in its answer: what counts is the chain of latencies
        ("attend_one_short", _attend(32, 8, 128, 16, 1, 385, 385)),
        # a batch of requests of very unequal lengths, 8B shape
        ("attend_ragged", _attend(32, 8, 128, 16, 48, 1, 4096)),
        # two long documents, 70B shape
        ("attend_long", _attend(64, 8, 128, 256, 2, 60001, 99991)),
        # small heads, as many key heads as query heads, a large batch
        ("attend_small_heads", _attend(16, 16, 64, 32, 200, 100, 1500)),
        # one request, a small vocabulary, all of the usual settings together
        ("sample_one", _sample(1, 32000, "nucleus")),
        # a batch of requests, each with settings of its own, large vocabulary
        ("sample_mixed", _sample(48, 128256, "mixed")),
        # temperature alone, a vocabulary of odd size, a large batch
        ("sample_plain", _sample(200, 50257, "plain")),
    ]
    return [dict(case, name=name) for name, case in cases]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    pick = rng.random()
    page = rng.choice((16, 32, 64, 128, 256))
    if pick < 0.2:
        rows = _log_int(rng, 1, 300)
        if rng.random() < 0.5:
            return _plan(rows, page, rng.randint(80, 600), 1, 1, _log_int(rng, 100, 1200))
        return _plan(rows, page, rng.randint(130, 300), rng.randint(0, 3), _log_int(rng, 10, min(2000, max(11, 100000 // rows))), 0, pad=rng.randint(0, 1000))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 10, 16))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8))
    dim = rng.choice((64, 128, 128))
    if pick < 0.35:
        rows = _log_int(rng, 1, 40)
        most = min(2048, 9000 * 80 * 128 // ((heads + 2 * kv_heads) * dim * rows))
        return _store(heads, kv_heads, dim, page, rows, _log_int(rng, 1, max(2, most)))
    if pick < 0.7:
        rows = _log_int(rng, 1, 256)
        most = min(60000, 90000 * 8 * 128 // (rows * kv_heads * dim), 60000 * 64 * 2 // (rows * heads))
        hi = _log_int(rng, 2, max(3, most))
        return _attend(heads, kv_heads, dim, page, rows, rng.choice((0, 1, hi, (hi + 1) // 2)), hi)
    vocab = _log_int(rng, 1000, 128256)
    return _sample(_log_int(rng, 1, min(256, 200 * 50257 // vocab)), vocab, rng.choice(("nucleus", "mixed", "plain", "top_k", "top_p", "min_p", "greedy")))


# ------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randint(lo, hi, size, gen, dtype=torch.int32):
    """Whole numbers of lo .. hi, both among them."""
    return torch.randint(lo, hi + 1, size, device=DEVICE, generator=gen, dtype=dtype)


def _pages(n, page):
    return (n + page - 1) // page


def _spread(lo, hi, rows, gen, dtype=torch.int32):
    """Whole numbers from lo to hi at equal steps, in shuffled order: the same sum for every seed."""
    steps = torch.linspace(lo, hi, rows, device=DEVICE, dtype=torch.float64).round() if rows > 1 else torch.full((1,), hi, device=DEVICE)
    return steps.to(dtype)[torch.randperm(rows, device=DEVICE, generator=gen)]


def _tables(lengths, max_pages, page, pool, gen):
    """(block table [rows, max_pages], the pages that no row holds): shuffled pages of the pool, each row as many as its length takes."""
    held = _pages(lengths.long(), page)
    ends = held.cumsum(0)
    order = torch.randperm(pool, device=DEVICE, generator=gen).int()
    index = (ends - held)[:, None] + torch.arange(max_pages, device=DEVICE)
    table = torch.zeros(lengths.numel(), max_pages, dtype=torch.int32, device=DEVICE)
    inside = torch.arange(max_pages, device=DEVICE) < held[:, None]
    table[inside] = order[index[inside]]
    return table, order[int(ends[-1]):]


def _rope_tables(positions, dim):
    inv = 1.0 / (ROPE_THETA ** (torch.arange(0, dim, 2, device=DEVICE, dtype=torch.float64) / dim))
    angles = torch.arange(positions, device=DEVICE, dtype=torch.float64)[:, None] * inv
    return angles.cos().half(), angles.sin().half()


def _prepare_plan(c, gen):
    rows, page, max_pages = c["rows"], c["page"], c["max_pages"]
    most = max_pages * page
    if c["held_hi"]:                                                      # every row goes on with one token
        going = torch.ones(rows, dtype=torch.bool, device=DEVICE)
        new = _spread(c["new_lo"], c["new_hi"], rows, gen)
        held = _randint(1, min(c["held_hi"], most - 1), (rows,), gen)
    else:                                                                 # prompts come in, a third of the rows go on with one token
        new = torch.cat([torch.ones(rows // 3, dtype=torch.int32, device=DEVICE), _spread(c["new_lo"], min(c["new_hi"], most), rows - rows // 3, gen)])
        going = torch.arange(rows, device=DEVICE) < rows // 3
        shuffle = torch.randperm(rows, device=DEVICE, generator=gen)
        new, going = new[shuffle], going[shuffle]
        held = torch.where(going, _randint(1, most - 1, (rows,), gen), 0)
    tokens = int(new.sum()) + c["pad"]
    released = going & (torch.rand(rows, device=DEVICE, generator=gen) < 0.06)
    new[released] = 0
    pool = rows * (max_pages + 1)
    table, free = _tables(held, max_pages, page, pool, gen)
    need = int((_pages(held.long() + new, page) - _pages(held.long(), page)).sum())
    free = free[:need + rows // 2]
    ring = torch.zeros(pool, dtype=torch.int32, device=DEVICE)
    head = pool - free.numel() // 2                                       # the ring's free part goes over its end
    ring[(head + torch.arange(free.numel(), device=DEVICE)) % pool] = free
    return {"held": held, "new": new, "released": released, "table": table, "ring": ring, "page": page,
            "state": torch.tensor([head % pool, free.numel()], dtype=torch.int32, device=DEVICE), "tokens": tokens}


def _prepare_store(c, gen):
    rows, page, dim = c["rows"], c["page"], c["dim"]
    new = _spread((c["new_hi"] + 1) // 2, c["new_hi"], rows, gen)
    held = _randint(0, 40, (rows,), gen) * (torch.rand(rows, device=DEVICE, generator=gen) < 0.3)       # some go on behind a cached prefix
    max_pages = _pages(c["new_hi"] + 40, page)
    pool = rows * max_pages + 1
    table, _ = _tables(held + new, max_pages, page, pool, gen)
    tokens = int(new.sum())
    ends = new.long().cumsum(0)
    row = torch.searchsorted(ends, torch.arange(tokens, device=DEVICE), right=True)
    positions = (held[row] + torch.arange(tokens, device=DEVICE) - (ends - new)[row]).int()
    slots = table[row, positions.long() // page].long() * page + positions % page
    slots[torch.rand(tokens, device=DEVICE, generator=gen) < 0.01] = -1   # tokens that were given no slot
    heads, kv_heads = c["heads"], c["kv_heads"]
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * dim, device=DEVICE, generator=gen).half()
    cos, sin = _rope_tables(c["new_hi"] + 40, dim)
    pages = torch.randn(2, pool, kv_heads, page, dim, device=DEVICE, generator=gen, dtype=torch.float16)
    return {"qkv": qkv, "cos": cos, "sin": sin, "kpages": pages[0], "vpages": pages[1], "positions": positions, "slots": slots,
            "heads": heads, "kv_heads": kv_heads, "dim": dim}


def _prepare_attend(c, gen):
    rows, page, dim = c["rows"], c["page"], c["dim"]
    lengths = _spread(c["len_lo"], c["len_hi"], rows, gen)
    max_pages = _pages(c["len_hi"], page)
    pool = int(_pages(lengths.long(), page).sum()) + 4
    table, _ = _tables(lengths, max_pages, page, pool, gen)
    heads, kv_heads = c["heads"], c["kv_heads"]
    qkv = torch.randn(rows, (heads + 2 * kv_heads) * dim, device=DEVICE, generator=gen)
    qkv[:, :heads * dim] *= 1.5                                           # scores of a few units, as trained heads have them
    last = (lengths.long() - 1).clamp(min=0)
    slots = table.gather(1, last[:, None] // page)[:, 0].long() * page + last % page
    slots = torch.where(lengths > 0, slots, -1)
    cos, sin = _rope_tables(c["len_hi"], dim)
    pages = torch.randn(2, pool, kv_heads, page, dim, device=DEVICE, generator=gen, dtype=torch.float16)
    return {"qkv": qkv.half(), "kpages": pages[0], "vpages": pages[1], "cos": cos, "sin": sin, "table": table, "lengths": lengths,
            "slots": slots, "heads": heads, "kv_heads": kv_heads, "dim": dim}


def _prepare_sample(c, gen):
    rows, vocab, kind = c["rows"], c["vocab"], c["kind"]
    # from rows that are sure of a few tokens to rows that spread over thousands
    logits = torch.randn(rows, vocab, device=DEVICE, generator=gen) * (1.5 + 1.5 * torch.rand(rows, 1, device=DEVICE, generator=gen))
    sure = torch.randint(0, vocab, (rows, 8), device=DEVICE, generator=gen)
    logits.scatter_add_(1, sure, 8.0 * torch.rand(rows, 8, device=DEVICE, generator=gen))
    rand = lambda: torch.rand(rows, device=DEVICE, generator=gen)         # noqa: E731
    temperature = 0.5 + 0.8 * rand()
    top_k = _randint(1, 100, (rows,), gen)
    top_p = 0.8 + 0.2 * rand()
    min_p = 0.1 * rand()
    if kind == "mixed":                                                   # every request has settings of its own, many leave some of them out
        temperature *= rand() < 0.85
        top_k *= rand() < 0.5
        top_p = torch.where(rand() < 0.6, top_p, 1.0)
        min_p *= rand() < 0.3
    state = {"logits": logits.half(), "uniform": rand(), "temperature": None if kind == "greedy" else temperature, "top_k": None, "top_p": None, "min_p": None}
    if kind == "greedy":
        state["temperature"] = torch.zeros(rows, device=DEVICE)
    for name, values in (("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        if kind == "mixed" or kind == name or (kind == "nucleus" and name != "min_p"):
            state[name] = values
    return state


def prepare(case, seed):
    return dict({"plan": _prepare_plan, "store": _prepare_store, "attend": _prepare_attend, "sample": _prepare_sample}[case["op"]](case, _gen(seed)), op=case["op"])


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_plan(s):
    page, table, ring = s["page"], s["table"], s["ring"]
    rows, max_pages = table.shape
    pool, new = ring.numel(), s["new"].long()
    before = s["held"].long()
    given = torch.where(s["released"], _pages(before, page), 0)
    held = torch.where(s["released"], 0, before)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    possible = (_pages(held + new, page) <= max_pages) & (starts[1:] <= s["tokens"])
    need = torch.where(possible, _pages(held + new, page) - _pages(held, page), 0)
    head, count = s["state"].long()
    upto = need.cumsum(0)
    ok = possible & ((need == 0) | (upto <= count))
    need, granted = torch.where(ok, need, 0), torch.where(ok, new, 0)
    first = need.cumsum(0) - need
    column = torch.arange(max_pages, device=table.device)
    # pages that come back go behind the ring's last
    back = (column < given[:, None])
    to = (head + count + (given.cumsum(0) - given)[:, None] + column) % pool
    returned = torch.where(back, to, pool)
    longer = torch.cat([ring, ring[:1]]).scatter_(0, returned.flatten(), table.flatten())
    # pages that are taken come from its front
    place = column - _pages(held, page)[:, None]
    take = (place >= 0) & (place < need[:, None])
    taken = ring[(head + first[:, None] + place.clamp(min=0)) % pool]
    table.copy_(torch.where(take, taken, table))
    ring.copy_(longer[:pool])
    lengths = held + granted
    token = torch.arange(s["tokens"], device=table.device)
    row = torch.searchsorted(starts[1:].contiguous(), token, right=True).clamp(max=rows - 1)
    at = token - starts[row]
    valid = (token < starts[-1]) & (at < granted[row])
    position = torch.where(valid, held[row] + at, 0)
    slot = table[row, position // page].long() * page + position % page
    return {"table": table, "ring": ring, "lengths": lengths.int(), "state": torch.stack([(head + need.sum()) % pool, count - need.sum() + given.sum()]).int(),
            "granted": granted.int(), "starts": starts.int(), "positions": torch.where(valid, position, -1).int(), "slots": torch.where(valid, slot, -1)}


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_store(s):
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    qkv, slots = s["qkv"], s["slots"]
    tokens, page = qkv.shape[0], s["kpages"].shape[2]
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), 1))
    at = s["positions"].long()
    cos, sin = s["cos"][at].float()[:, None], s["sin"][at].float()[:, None]
    there = (slots >= 0)[:, None, None]
    rotated = torch.where(there, _rotate(q.float(), cos, sin).half(), q)
    k = _rotate(k.float(), cos, sin).half()
    # a token without a slot writes what its place holds already: that of the first token that has one
    first = there[:, 0, 0].int().argmax()
    slot = torch.where(slots >= 0, slots, slots[first])
    same = torch.where(slots >= 0, torch.arange(tokens, device=slots.device), first)
    s["kpages"][slot // page, :, slot % page] = k[same]
    s["vpages"][slot // page, :, slot % page] = v[same]
    return {"q": rotated.flatten(1), "kpages": s["kpages"], "vpages": s["vpages"]}


def _plain_attend(s):
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    qkv, table, lengths, slots = s["qkv"].float(), s["table"].long(), s["lengths"].long(), s["slots"]
    rows, page = qkv.shape[0], s["kpages"].shape[2]
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), 1))
    last = (lengths - 1).clamp(min=0)
    cos, sin = s["cos"][last].float()[:, None], s["sin"][last].float()[:, None]
    q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    # idle rows write what their place holds already
    live = (slots >= 0)[:, None, None]
    for pages, x in ((s["kpages"], k), (s["vpages"], v)):
        x = x.half()
        kept = torch.where(slots >= 0, slots, slots.max())
        who = torch.where(slots >= 0, torch.arange(rows, device=slots.device), slots.argmax())
        pages[kept // page, :, kept % page] = torch.where(live.any(), x[who], pages[kept // page, :, kept % page])
    group = heads // kv_heads
    keys = s["kpages"][table].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, -1, dim).float()
    scores = torch.matmul(q.view(rows, kv_heads, group, dim), keys.transpose(2, 3).contiguous()) / math.sqrt(dim)
    del keys
    scores.masked_fill_(torch.arange(scores.shape[-1], device=scores.device) >= lengths[:, None, None, None], float("-inf"))
    weights = (scores - scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    values = s["vpages"][table].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, -1, dim).float()
    out = torch.matmul(weights, values) / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.where(live[..., None], out, 0.0)
    return {"out": out.reshape(rows, heads * dim).half(), "kpages": s["kpages"], "vpages": s["vpages"]}


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    temperature = s["temperature"].double()[:, None]
    weight = ((x - x.amax(1, keepdim=True)) / torch.where(temperature > 0, temperature, 1.0)).exp()
    order = x.sort(dim=1, descending=True, stable=True).indices
    sorted_weight = weight.gather(1, order)
    if s["top_k"] is not None:
        top_k = s["top_k"][:, None]
        sorted_weight = torch.where((top_k <= 0) | (torch.arange(vocab, device=x.device) < top_k), sorted_weight, 0.0)
    keep = sorted_weight > 0
    if s["top_p"] is not None:
        top_p = s["top_p"].double()[:, None]
        total = sorted_weight.cumsum(1)
        before = torch.cat([total.new_zeros(rows, 1), total[:, :-1]], 1)
        keep &= (top_p >= 1) | (before < top_p * total[:, -1:])
    if s["min_p"] is not None:
        keep &= sorted_weight >= s["min_p"].double()[:, None]
    kept = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, sorted_weight, 0.0)).cumsum(1)
    drawn = (kept <= s["uniform"].double()[:, None] * kept[:, -1:]).sum(1)
    return torch.where(temperature[:, 0] > 0, drawn, order[:, 0])


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, op = state, state["op"]
    if not own:
        return {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend, "sample": _plain_sample}[op](s)
    from bitstack_amd.utils import inference_utils as ops
    if op == "plan":
        plan = ops.page_plan_hip(s["held"], s["new"], s["table"], s["ring"], s["state"], s["page"], s["tokens"], released=s["released"])
        return {"table": s["table"], "ring": s["ring"], "lengths": plan.lengths, "state": plan.state, "granted": plan.granted, "starts": plan.starts,
                "positions": plan.positions, "slots": plan.slots}
    if op == "store":
        wide = s["heads"] * s["dim"], s["kv_heads"] * s["dim"], s["kv_heads"] * s["dim"]
        q, k, v = s["qkv"].split(wide, 1)
        q = ops.rope_store_paged_hip(q, k, v, s["cos"], s["sin"], s["kpages"], s["vpages"], s["positions"], s["slots"], out=torch.empty(q.shape, dtype=q.dtype, device=q.device))
        return {"q": q, "kpages": s["kpages"], "vpages": s["vpages"]}
    if op == "attend":
        out = ops.attention_paged_hip(s["qkv"], s["kpages"], s["vpages"], s["cos"], s["sin"], s["table"], s["lengths"], s["slots"], s["heads"], s["kv_heads"])
        return {"out": out, "kpages": s["kpages"], "vpages": s["vpages"]}
    return ops.sample_hip(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


# ------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    c = case
    mean = lambda lo, hi: (lo + hi) / 2                                   # noqa: E731
    if c["op"] == "plan":
        prompts = 0 if c["held_hi"] else c["rows"] - c["rows"] // 3
        tokens = c["rows"] - prompts + prompts * mean(c["new_lo"], min(c["new_hi"], c["max_pages"] * c["page"])) + c["pad"]
        return {"bytes": int(12 * tokens + 8 * tokens / c["page"] + 21 * c["rows"]), "flops": int(8 * tokens)}
    if c["op"] == "store":
        tokens = c["rows"] * mean((c["new_hi"] + 1) // 2, c["new_hi"])
        values = tokens * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": int(4 * values + 12 * tokens + 2 * c["dim"] * c["new_hi"]), "flops": int(3 * values)}
    if c["op"] == "attend":
        positions = c["rows"] * mean(c["len_lo"], c["len_hi"])
        row = c["rows"] * c["dim"] * 2
        return {"bytes": int(4 * positions * c["kv_heads"] * c["dim"] + row * (2 * c["heads"] + 4 * c["kv_heads"]) + 4 * positions / c["page"]),
                "flops": int(4 * positions * c["heads"] * c["dim"])}
    return {"bytes": 2 * c["rows"] * c["vocab"], "flops": 4 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _turn(x, cos, sin):
    """x [tokens, heads, dim], the two halves of a head as a complex number times cos + i sin."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(cos, sin)[:, None]
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    """The outputs in 64 bits from the definition; whole numbers (plans, tokens) are compared as they are."""
    if case["op"] in ("plan", "sample"):
        return None
    s = prepare(case, seed)
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    x = s["qkv"].double().view(s["qkv"].shape[0], -1, dim)
    kpages, vpages = s["kpages"].double(), s["vpages"].double()
    pool, page = kpages.shape[0], kpages.shape[2]
    at = (s["positions"] if case["op"] == "store" else s["lengths"] - 1).long().clamp(min=0)
    turned = _turn(x[:, :heads + kv_heads], s["cos"][at].double(), s["sin"][at].double())
    q, k, v = turned[:, :heads], turned[:, heads:], x[:, heads + kv_heads:]
    live = s["slots"] >= 0
    place = s["slots"][live]
    kpages.view(pool, kv_heads, page, dim)[place // page, :, place % page] = k[live]
    vpages.view(pool, kv_heads, page, dim)[place // page, :, place % page] = v[live]
    if case["op"] == "store":
        return {"q": torch.where(live[:, None, None], q, x[:, :heads]).reshape(x.shape[0], -1), "kpages": kpages, "vpages": vpages}
    out = torch.zeros(x.shape[0], heads, dim, dtype=torch.float64, device=x.device)
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, :_pages(n, page)].long()
        keys = kpages[pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :n]
        values = vpages[pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :n]
        score = torch.matmul(q[b].view(kv_heads, -1, dim), keys.transpose(1, 2).contiguous()) * dim ** -0.5
        out[b] = torch.matmul(torch.softmax(score, -1), values).view(heads, dim)
    return {"out": out.view(x.shape[0], -1), "kpages": kpages, "vpages": vpages}
