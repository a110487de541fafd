"""The operators of drafted and forked requests over a cache in pages, as cases to be timed and compared.

  plan    tree_plan_hip: the positions of drafted tokens, and which of them each one attends to, from the parents of a tree per request
  attend  attention_tree_hip: the drafted tokens' rotated queries over the paged cache and over their own ancestors
  accept  tree_accept_hip: the path that the model agrees with, its keys and values moved together in every layer, pages behind them given back
  fork    page_fork_hip: rows become copies of other rows: whole pages shared, the last one copied, pages that nobody holds any more given back
  adjust  logits_adjust_hip: penalties for repeated tokens, biases and grammar masks on logits

Requests are rows of a batch.  A request's drafted tokens are the nodes of a tree, node 0 (the token that it goes on with) its root, parents before their
children; token rows lie side by side, request after request.  Pages are dealt in shuffled order, as a pool in use leaves them.
"""
import math

import torch

own = False
DEVICE = "cuda"
NODES = 64                                                                # of one request, at most: a mask is 64 bits


# ------------------------------------------------------------------------------------------------- cases
def _plan(rows, nodes_lo, nodes_hi, pad=0):
    return {"op": "plan", "rows": rows, "nodes_lo": nodes_lo, "nodes_hi": nodes_hi, "pad": pad}


def _attend(heads, kv_heads, dim, page, rows, held_lo, held_hi, nodes_lo, nodes_hi):
    return {"op": "attend", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "rows": rows, "held_lo": held_lo, "held_hi": held_hi,
            "nodes_lo": nodes_lo, "nodes_hi": nodes_hi}


def _accept(layers, kv_heads, dim, page, rows, held_hi, nodes_lo, nodes_hi):
    return {"op": "accept", "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page, "rows": rows, "held_hi": held_hi, "nodes_lo": nodes_lo, "nodes_hi": nodes_hi}


def _fork(layers, kv_heads, dim, page, rows, held_lo, held_hi, kind):
    return {"op": "fork", "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page, "rows": rows, "held_lo": held_lo, "held_hi": held_hi, "kind": kind}


def _adjust(rows, nodes, vocab, history, kind):
    return {"op": "adjust", "rows": rows, "nodes": nodes, "vocab": vocab, "history": history, "kind": kind}


def listed():
    cases = [
        # one request with a small tree, in front of every step
        ("plan_one", _plan(1, 24, 24)),
        # many requests with trees of all sizes, in a batch padded to a fixed row count
        ("plan_batch", _plan(300, 1, 64, pad=100)),
        # one request, early in its answer, with a few drafted tokens: what counts is the chain of latencies
        ("attend_one_short", _attend(32, 8, 128, 16, 1, 385, 385, 8, 8)),
        # a batch of requests of very unequal lengths and trees, 8B shape
        ("attend_ragged", _attend(32, 8, 128, 16, 48, 0, 4096, 1, 16)),
        # two long documents with the largest trees, 70B shape
        ("attend_long", _attend(64, 8, 128, 256, 2, 60001, 99991, 64, 64)),
        # small heads, as many key heads as query heads, a large batch with a few drafted tokens each
        ("attend_small_heads", _attend(16, 16, 64, 32, 200, 100, 1500, 1, 5)),
        # one request of an 8B-shape model, its small tree checked
        ("accept_one", _accept(32, 8, 128, 16, 1, 200, 8, 8)),
        # a batch of requests, trees of up to 32 nodes, 8B shape
        ("accept_batch", _accept(32, 8, 128, 16, 48, 200, 1, 32)),
        # four beams of one request change places after a step
        ("fork_beams", _fork(32, 8, 128, 16, 4, 300, 300, "beams")),
        # prompts that get several continuations each, in place of requests that have ended
        ("fork_samples", _fork(32, 8, 128, 64, 64, 1, 500, "samples")),
        # one request, a small vocabulary, penalties for what it has said
        ("adjust_one", _adjust(1, 1, 32000, 700, "penalties")),
        # a batch of requests with drafted tokens, large vocabulary, everything together
        ("adjust_batch", _adjust(48, 8, 128256, 3000, "all")),
    ]
    return [dict(case, name=name) for name, case in cases]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    pick = rng.random()
    page = rng.choice((16, 32, 64, 128, 256))
    if pick < 0.1:
        return _plan(_log_int(rng, 1, 300), rng.randint(0, 3), _log_int(rng, 3, NODES), pad=rng.randint(0, 300))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 10, 16))
    dim = rng.choice((64, 128, 128))
    if pick < 0.5:
        heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8))
        rows = _log_int(rng, 1, 256)
        nodes = _log_int(rng, 1, NODES)
        most = min(60000, 90000 * 8 * 128 // (rows * kv_heads * dim), 160000 * 64 * 64 // (rows * heads * nodes))
        held = _log_int(rng, 2, max(3, most))
        return _attend(heads, kv_heads, dim, page, rows, rng.choice((0, 1, held, (held + 1) // 2)), held, rng.randint(1, nodes), nodes)
    layers = rng.choice((1, 2, 16, 28, 32))
    if pick < 0.65:
        nodes, held = _log_int(rng, 1, NODES), rng.randint(1, 200)
        rows = _log_int(rng, 1, min(200, max(1, 10 ** 9 // ((held + nodes + page) * kv_heads * dim * layers))))
        return _accept(layers, kv_heads, dim, page, rows, held, rng.randint(1, nodes), nodes)
    if pick < 0.8:
        held = _log_int(rng, 1, 500)
        rows = _log_int(rng, 2, min(256, max(2, 10 ** 9 // ((held + 4 * page) * kv_heads * dim * layers))))
        return _fork(layers, kv_heads, dim, page, rows, rng.choice((0, 1, held)), held, rng.choice(("beams", "samples")))
    vocab = _log_int(rng, 1000, 128256)
    nodes = _log_int(rng, 1, 16)
    rows = _log_int(rng, 1, min(128, max(1, 384 * 128256 // (vocab * nodes))))
    return _adjust(rows, nodes, vocab, _log_int(rng, 1, 3000), rng.choice(("penalties", "bias", "grammar", "all")))


# ------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _rand(gen, *size):
    return torch.rand(*size, device=DEVICE, generator=gen)


def _randint(lo, hi, size, gen, dtype=torch.int32):
    """Whole numbers of lo .. hi, both among them."""
    return torch.randint(lo, hi + 1, size, device=DEVICE, generator=gen, dtype=dtype)


def _pages(n, page):
    return (n + page - 1) // page


def _spread(lo, hi, rows, gen):
    """Whole numbers from lo to hi at equal steps, in shuffled order: the same sum for every seed."""
    steps = torch.linspace(lo, hi, rows, device=DEVICE, dtype=torch.float64).round() if rows > 1 else torch.full((1,), hi, device=DEVICE)
    return steps.int()[torch.randperm(rows, device=DEVICE, generator=gen)]


def _starts(counts):
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()


def _rows_of(starts, tokens):
    """(request, node) of every token row; the rows behind the last token belong to the last request."""
    token = torch.arange(tokens, device=starts.device)
    row = torch.searchsorted(starts[1:].contiguous(), token, right=True).clamp(max=starts.numel() - 2)
    return row, token - starts[row]


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


def _ring(free, pool):
    """(ring, its {first, count}): the free part goes over the ring's end."""
    ring = torch.zeros(pool, dtype=torch.int32, device=DEVICE)
    head = pool - free.numel() // 2
    ring[(head + torch.arange(free.numel(), device=DEVICE)) % pool] = free
    return ring, torch.tensor([head % pool, free.numel()], dtype=torch.int32, device=DEVICE)


def _parents(starts, tokens, gen):
    """Trees in which a node continues one of the few in front of it, as drafts with several choices per place do; -1 for roots."""
    row, node = _rows_of(starts, tokens)
    back = (1 + 6 * _rand(gen, tokens).square()).long()
    return torch.where(node > 0, (node - back).clamp(min=0), -1).int()


def _prepare_plan(c, gen):
    counts = _spread(c["nodes_lo"], c["nodes_hi"], c["rows"], gen)
    starts = _starts(counts)
    tokens = int(starts[-1]) + c["pad"]
    refused = (_rand(gen, c["rows"]) < 0.05) & (c["rows"] > 1)            # requests whose pages were not there
    granted = torch.where(refused, 0, counts)
    held = _randint(0, 8000, (c["rows"],), gen)
    return {"parents": _parents(starts, tokens, gen), "starts": starts, "granted": granted, "lengths": held + granted}


def _prepare_attend(c, gen):
    rows, page, dim, heads, kv_heads = c["rows"], c["page"], c["dim"], c["heads"], c["kv_heads"]
    counts = _spread(c["nodes_lo"], c["nodes_hi"], rows, gen)
    held = _spread(c["held_lo"], c["held_hi"], rows, gen)
    starts = _starts(counts)
    tokens = int(starts[-1])
    lengths = held + counts
    max_pages = _pages(c["held_hi"] + c["nodes_hi"], page)
    pool = int(_pages(lengths.long(), page).sum()) + 4
    table, _ = _tables(lengths, max_pages, page, pool, gen)
    q = 1.5 * torch.randn(tokens, heads * dim, device=DEVICE, generator=gen)       # scores of a few units, as trained heads have them
    pages = torch.randn(2, pool, kv_heads, page, dim, device=DEVICE, generator=gen, dtype=torch.float16)
    masks = _plain_plan({"parents": _parents(starts, tokens, gen), "starts": starts, "granted": counts, "lengths": lengths})["masks"]
    return {"q": q.half(), "kpages": pages[0], "vpages": pages[1], "table": table, "lengths": lengths, "granted": counts, "starts": starts, "masks": masks,
            "nodes": c["nodes_hi"], "dim": dim}


def _prepare_accept(c, gen):
    rows, page, nodes = c["rows"], c["page"], c["nodes_hi"]
    counts = _spread(c["nodes_lo"], nodes, rows, gen)
    held = _randint(0, c["held_hi"], (rows,), gen)
    starts = _starts(counts)
    tokens = int(starts[-1])
    refused = (_rand(gen, rows) < 0.04) & (rows > 1)
    granted = torch.where(refused, 0, counts)
    lengths = held + granted
    max_pages = _pages(c["held_hi"] + nodes, page)
    pool = rows * max_pages + 5
    table, free = _tables(lengths, max_pages, page, pool, gen)
    ring, state = _ring(free[:pool // 3], pool)
    row, node = _rows_of(starts, tokens)
    at = held[row].long() + node
    slots = torch.where(granted[row] > 0, table[row, at // page].long() * page + at % page, -1)
    parents = _parents(starts, tokens, gen)
    drafted = _randint(0, 31999, (tokens,), gen, torch.int64)
    # the model agrees with a child of four nodes in five: that of the last one that names them
    targets = _randint(0, 31999, (tokens,), gen, torch.int64)
    child = torch.zeros(tokens + 1, dtype=torch.int64, device=DEVICE).scatter_reduce_(
        0, torch.where(parents >= 0, starts[row] + parents, tokens).long(), torch.arange(tokens, device=DEVICE), "amax")[:tokens]
    agrees = (child > 0) & (_rand(gen, tokens) < 0.8)
    targets = torch.where(agrees, drafted[child], targets)
    pages = torch.randn(2, c["layers"], pool, c["kv_heads"], page, c["dim"], device=DEVICE, generator=gen, dtype=torch.float16)
    return {"tokens": drafted, "parents": parents, "targets": targets, "slots": slots, "lengths": lengths, "granted": granted, "starts": starts, "table": table,
            "ring": ring, "state": state, "kpages": pages[0], "vpages": pages[1], "nodes": nodes}


def _prepare_fork(c, gen):
    rows, page = c["rows"], c["page"]
    lengths = _spread(c["held_lo"], c["held_hi"], rows, gen)
    if c["kind"] == "beams":                                              # the better ones take the places of the worse
        source = torch.minimum(_randint(0, rows - 1, (rows,), gen), _randint(0, rows - 1, (rows,), gen))
    else:                                                                 # three rows in four go on as continuations of the others, some end
        source = torch.where(torch.arange(rows, device=DEVICE) % 4 == 0, torch.arange(rows, device=DEVICE), torch.arange(rows, device=DEVICE) // 4 * 4).int()
        source = torch.where(_rand(gen, rows) < 0.1, -1, source)
    max_pages = _pages(c["held_hi"], page) + 2
    pool = rows * max_pages + rows + 2
    table, free = _tables(lengths, max_pages, page, pool, gen)
    shares = torch.zeros(pool, dtype=torch.int32, device=DEVICE)
    if rows > 1:                                                          # rows that were one request's before share their first pages already
        common = min(int(lengths.min()) // page, max_pages // 2)
        pair = torch.arange(rows // 2, device=DEVICE) * 2
        shares[table[pair, :common].flatten().long()] += 1
        free = torch.cat([free, table[pair + 1, :common].flatten()])
        table[pair + 1, :common] = table[pair, :common]
    ring, state = _ring(free, pool)
    pages = torch.randn(2, c["layers"], pool, c["kv_heads"], page, c["dim"], device=DEVICE, generator=gen, dtype=torch.float16)
    return {"source": source.int(), "lengths": lengths, "table": table, "ring": ring, "state": state, "shares": shares, "kpages": pages[0], "vpages": pages[1]}


def _prepare_adjust(c, gen):
    rows, nodes, vocab, kind, most = c["rows"], c["nodes"], c["vocab"], c["kind"], c["history"]
    logits = (torch.randn(rows * nodes, vocab, device=DEVICE, generator=gen) * 2.5).half()
    request = torch.arange(rows, device=DEVICE, dtype=torch.int32).repeat_interleave(nodes)
    s = {"logits": logits, "requests": request, "history": None, "history_lengths": None, "prompt_lengths": None, "repetition": None, "frequency": None, "presence": None,
         "drafted": None, "bias_tokens": None, "bias": None, "allowed": None, "allowed_rows": None}
    if kind in ("penalties", "all"):
        # tokens as texts repeat them: a few very often, most of them seldom
        s["history"] = (vocab * _rand(gen, rows, most).pow(4)).int().clamp(max=vocab - 1)
        s["history_lengths"] = _spread((most + 1) // 2, most, rows, gen)
        s["prompt_lengths"] = (s["history_lengths"] * _rand(gen, rows)).int()
        s["repetition"] = torch.where(_rand(gen, rows) < 0.8, 1.0 + 0.5 * _rand(gen, rows), 1.0)
        s["frequency"], s["presence"] = 0.7 * _rand(gen, rows), _rand(gen, rows) - 0.3
        if nodes > 1:                                                     # what a drafted token has in front of it on its own path, -1 where there is nothing
            depth = torch.arange(nodes, device=DEVICE).repeat(rows)
            s["drafted"] = torch.where(torch.arange(nodes - 1, device=DEVICE) < depth[:, None], _randint(0, vocab - 1, (rows * nodes, nodes - 1), gen), -1)
    if kind in ("bias", "all"):
        s["bias_tokens"] = torch.rand(rows, vocab, device=DEVICE, generator=gen).topk(min(50, vocab), 1).indices.int()
        s["bias_tokens"][:, 30:] = torch.where(_rand(gen, rows, 1) < 0.5, -1, s["bias_tokens"][:, 30:])
        s["bias"] = 8.0 * torch.randn(s["bias_tokens"].shape, device=DEVICE, generator=gen)
    if kind in ("grammar", "all"):                                        # a few grammars, each with states that allow little or nearly everything
        states = 2 * rows
        dense = _rand(gen, states, 1).square()
        bits = (_rand(gen, states, _pages(vocab, 32), 32) < dense[:, None]).long() << torch.arange(32, device=DEVICE)
        s["allowed"] = torch.where(bits.sum(-1) >= 1 << 31, bits.sum(-1) - (1 << 32), bits.sum(-1)).int()
        s["allowed_rows"] = _randint(0, states - 1, (rows * nodes,), gen)
        s["allowed_rows"] = torch.where(_rand(gen, rows * nodes) < 0.2, -1, s["allowed_rows"])
    return s


def prepare(case, seed):
    make = {"plan": _prepare_plan, "attend": _prepare_attend, "accept": _prepare_accept, "fork": _prepare_fork, "adjust": _prepare_adjust}[case["op"]]
    return dict(make(case, _gen(seed)), op=case["op"])


# ------------------------------------------------------------------------------------------------- plain forms
def _ancestors(parents, starts, rows, nodes):
    """[rows, nodes, nodes]: whether the second node is the first one or an ancestor of it, from the powers of the parents' matrix."""
    node = torch.arange(nodes, device=parents.device)
    index = (starts[:-1, None] + node).clamp(max=parents.numel() - 1).long()
    there = node < (starts[1:] - starts[:-1])[:, None]
    parent = torch.where(there, parents[index], -1)
    step = (parent[..., None] == node) | torch.eye(nodes, dtype=torch.bool, device=parents.device)
    return (torch.matrix_power(step.double(), NODES) > 0) & there[..., None] & there[:, None]


def _plain_plan(s):
    parents, starts, granted = s["parents"], s["starts"], s["granted"].long()
    tokens, rows = parents.numel(), granted.numel()
    above = _ancestors(parents, starts, rows, NODES)
    row, node = _rows_of(starts, tokens)
    live = node < granted[row]
    above = above[row, node.clamp(max=NODES - 1)]
    bits = (above.long() << torch.arange(NODES, device=parents.device)).sum(1)
    place = s["lengths"][row] - granted[row] + above.sum(1) - 1
    return {"positions": torch.where(live, place, -1).int(), "masks": torch.where(live, bits, 0)}


def _plain_attend(s):
    q, table, lengths, starts, dim, nodes = s["q"].float(), s["table"].long(), s["lengths"].long(), s["starts"].long(), s["dim"], s["nodes"]
    rows, (pool, kv_heads, page, _) = lengths.numel(), s["kpages"].shape
    heads, tokens = q.shape[1] // dim, q.shape[0]
    held = lengths - s["granted"]
    node = torch.arange(nodes, device=q.device)
    index = (starts[:-1, None] + node).clamp(max=tokens - 1)
    q = q[index].view(rows, nodes, kv_heads, heads // kv_heads, dim).transpose(1, 2).reshape(rows, kv_heads, -1, dim)
    keys = s["kpages"][table].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, -1, dim).float()
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()) / math.sqrt(dim)
    del keys
    at = torch.arange(scores.shape[-1], device=q.device) - held[:, None]
    named = (s["masks"][index][:, :, None] >> at.clamp(0, 63)[:, None]) & 1
    seen = (at < 0)[:, None] | ((at < nodes) & (at < s["granted"][:, None]))[:, None] & (named == 1)      # [rows, nodes, positions]
    scores = scores.view(rows, kv_heads, nodes, heads // kv_heads, -1)
    scores.masked_fill_(~seen[:, None, :, None], float("-inf"))
    weights = (scores - scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp().flatten(2, 3)
    values = s["vpages"][table].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, -1, dim).float()
    out = torch.matmul(weights, values) / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.view(rows, kv_heads, nodes, -1, dim).transpose(1, 2).reshape(rows, nodes, heads * dim)
    row, node = _rows_of(starts, tokens)
    return {"out": out[row, node].half()}


def _plain_accept(s):
    parents, starts, granted, nodes, page = s["parents"], s["starts"], s["granted"].long(), s["nodes"], s["kpages"].shape[3]
    rows, tokens = granted.numel(), parents.numel()
    node = torch.arange(nodes, device=parents.device)
    index = (starts[:-1, None] + node).clamp(max=tokens - 1).long()
    there = node < granted[:, None]
    parent = torch.where(there, parents[index].long(), -1)
    drafted, target = s["tokens"][index], s["targets"][index]
    agreed = (parent >= 0) & (drafted == target.gather(1, parent.clamp(min=0)))
    # of children with the same token the first one counts
    same = agreed[:, None] & (parent[:, :, None] == parent[:, None]) & (drafted[:, :, None] == drafted[:, None]) & (node < node[:, None])
    agreed = (agreed & ~same.any(2)) | (node == 0)
    above = _ancestors(parents, starts, rows, nodes)
    kept = there & ~(above & ~agreed[:, None]).any(2) & above[:, :, 0]
    accepted = kept.sum(1)
    path = torch.where(kept, node, nodes).sort(1).values
    path = torch.where(path < nodes, path, -1)
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])
    token = torch.where(accepted > 0, target.gather(1, last.clamp(min=0))[:, 0], -1)
    slots = s["slots"][index]
    moved = path >= 0
    to, source = slots[moved], slots.gather(1, path.clamp(min=0))[moved]
    for_all = torch.arange(s["kpages"].shape[0], device=parents.device)[:, None]
    kmoved, vmoved = s["kpages"][for_all, source // page, :, source % page], s["vpages"][for_all, source // page, :, source % page]
    s["kpages"][for_all, to // page, :, to % page] = kmoved
    s["vpages"][for_all, to // page, :, to % page] = vmoved
    before = s["lengths"].long()
    lengths = before - granted + accepted
    first, back = _pages(lengths, page), _pages(before, page) - _pages(lengths, page)
    ring, table = s["ring"], s["table"]
    pool, column = ring.numel(), torch.arange(table.shape[1], device=table.device)
    place = column - first[:, None]
    goes = (place >= 0) & (place < back[:, None])
    head, count = s["state"].long()
    to = torch.where(goes, (head + count + (back.cumsum(0) - back)[:, None] + place) % pool, pool)
    ring.copy_(torch.cat([ring, ring[:1]]).scatter_(0, to.flatten(), table.flatten())[:pool])
    return {"lengths": lengths.int(), "state": torch.stack([head, count + back.sum()]).int(), "accepted": accepted.int(), "path": path.int(), "token": token,
            "ring": ring, "kpages": s["kpages"], "vpages": s["vpages"]}


def _plain_fork(s):
    table, ring, shares, before, page = s["table"], s["ring"], s["shares"], s["lengths"].long(), s["kpages"].shape[3]
    (rows, max_pages), pool = table.shape, ring.numel()
    me, column = torch.arange(rows, device=table.device), torch.arange(max_pages, device=table.device)
    source = s["source"].long()
    lengths = torch.where(source >= 0, before[source.clamp(min=0)], 0)
    whole, rest = lengths // page, lengths % page
    need = ((source >= 0) & (source != me) & (rest > 0)).long()
    head, count = s["state"].long()
    granted = (need == 0) | (need.cumsum(0) <= count)
    source = torch.where(granted, source, me)
    lengths = torch.where(granted, lengths, before)
    need = torch.where(granted, need, 0)
    moves = source != me
    fresh = ring[(head + need.cumsum(0) - need) % pool]
    old = table.long().clone()
    # who holds which page afterwards
    gives = moves[:, None] & (column < _pages(before, page)[:, None])
    takes = (moves & (source >= 0))[:, None] & (column < whole[:, None])
    mine = old[source.clamp(min=0)]
    one = torch.ones((), dtype=torch.int32, device=table.device)
    spare = torch.cat([shares, shares[:1]])
    spare.index_add_(0, torch.where(takes, mine, pool).flatten(), one.expand(rows * max_pages))
    spare.index_add_(0, torch.where(gives, old, pool).flatten(), -one.expand(rows * max_pages))
    left = spare[:pool]
    # a page that nobody holds any more goes back at the place of the first row that gave it
    entry = torch.arange(rows * max_pages, device=table.device)
    first = torch.full((pool + 1,), rows * max_pages, device=table.device).scatter_reduce_(0, torch.where(gives, old, pool).flatten(), entry, "amin")
    back = gives.flatten() & (first[old.flatten()] == entry) & (left[old.flatten()] < 0)
    to = torch.where(back, (head + count + back.cumsum(0) - 1) % pool, pool)
    copied = (need > 0).nonzero()[:, 0]
    ring_after = torch.cat([ring, ring[:1]]).scatter_(0, to, old.flatten().int())[:pool]
    shares.copy_(left.clamp(min=0))
    table.copy_(torch.where(takes, mine, torch.where((need > 0)[:, None] & (column == whole[:, None]), fresh[:, None].long(), old)))
    ring.copy_(ring_after)
    # the positions of the last page
    position = torch.arange(page, device=table.device)
    there = (position < rest[copied][:, None])[None, :, None, :, None]
    of, new = mine[copied, whole[copied]], fresh[copied].long()
    s["kpages"][:, new] = torch.where(there, s["kpages"][:, of], s["kpages"][:, new])
    s["vpages"][:, new] = torch.where(there, s["vpages"][:, of], s["vpages"][:, new])
    s["lengths"].copy_(lengths)
    s["state"].copy_(torch.stack([(head + need.sum()) % pool, count - need.sum() + back.sum()]))
    return {"table": table, "ring": ring, "lengths": s["lengths"], "state": s["state"], "granted": granted.int(), "shares": shares,
            "kpages": s["kpages"], "vpages": s["vpages"]}


def _counts(s, tokens, there):
    """How often each token of the vocabulary is among tokens [n, m], where `there`; fp32 [n, vocab]."""
    vocab = s["logits"].shape[1]
    counts = torch.zeros(tokens.shape[0], vocab + 1, device=tokens.device)
    counts.scatter_add_(1, torch.where(there, tokens.long(), vocab), torch.ones((), device=tokens.device).expand(tokens.shape))
    return counts[:, :vocab]


def _plain_adjust(s):
    logits, request = s["logits"], s["requests"].long()
    x, vocab = logits.float(), logits.shape[1]
    if s["history"] is not None:
        at = torch.arange(s["history"].shape[1], device=x.device)
        seen = _counts(s, s["history"], at < s["history_lengths"][:, None])[request]
        said = _counts(s, s["history"], (at < s["history_lengths"][:, None]) & (at >= s["prompt_lengths"][:, None]))[request]
        if s["drafted"] is not None:
            more = _counts(s, s["drafted"], s["drafted"] >= 0)
            seen, said = seen + more, said + more
        r = s["repetition"][request][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][request][:, None] * said
        x = x - torch.where(said > 0, s["presence"][request][:, None], 0.0)
    if s["bias"] is not None:
        bias = torch.zeros(s["bias"].shape[0], vocab + 1, device=x.device)
        bias.scatter_(1, torch.where(s["bias_tokens"] >= 0, s["bias_tokens"].long(), vocab), s["bias"])
        x = x + bias[request, :vocab]
    x = x.clamp(-65504, 65504)
    if s["allowed"] is not None:
        bits = (s["allowed"][s["allowed_rows"].clamp(min=0).long()][..., None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where((bits.flatten(1)[:, :vocab] == 1) | (s["allowed_rows"] < 0)[:, None], x, float("-inf"))
    return x.half()


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, op = state, state["op"]
    if not own:
        return {"plan": _plain_plan, "attend": _plain_attend, "accept": _plain_accept, "fork": _plain_fork, "adjust": _plain_adjust}[op](s)
    from bitstack_amd.utils import inference_utils as ops
    if op == "plan":
        plan = ops.tree_plan_hip(s["parents"], s["lengths"], s["granted"], s["starts"])
        return {"positions": plan.positions, "masks": plan.masks}
    if op == "attend":
        return {"out": ops.attention_tree_hip(s["q"], s["kpages"], s["vpages"], s["table"], s["lengths"], s["granted"], s["starts"], s["masks"], s["nodes"])}
    if op == "accept":
        done = ops.tree_accept_hip(s["tokens"], s["parents"], s["targets"], s["slots"], s["lengths"], s["granted"], s["starts"], s["table"], s["ring"], s["state"],
                                   s["kpages"], s["vpages"], s["nodes"])
        return {"lengths": done.lengths, "state": done.state, "accepted": done.accepted, "path": done.path, "token": done.token, "ring": s["ring"],
                "kpages": s["kpages"], "vpages": s["vpages"]}
    if op == "fork":
        done = ops.page_fork_hip(s["source"], s["lengths"], s["table"], s["ring"], s["state"], s["shares"], s["kpages"], s["vpages"], inplace=True)
        return {"table": s["table"], "ring": s["ring"], "lengths": done.lengths, "state": done.state, "granted": done.granted, "shares": s["shares"],
                "kpages": s["kpages"], "vpages": s["vpages"]}
    settings = {name: s[name] for name in ("history", "history_lengths", "prompt_lengths", "repetition", "frequency", "presence", "drafted", "requests", "bias_tokens", "bias",
                                           "allowed", "allowed_rows")}
    return ops.logits_adjust_hip(s["logits"], out=torch.empty_like(s["logits"]), **settings)


# ------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    c = case
    if c["op"] == "adjust":
        logits = c["rows"] * c["nodes"] * c["vocab"]
        given = 3 * c["rows"] * c["history"] if c["kind"] in ("penalties", "all") else 0
        masks = logits // 10 if c["kind"] in ("grammar", "all") else 0
        return {"bytes": 4 * logits + given + masks, "flops": 4 * logits}
    if c["op"] == "fork":
        copied = c["rows"] * (0.5 if c["kind"] == "beams" else 0.68) * min(c["page"] / 2, (c["held_lo"] + c["held_hi"]) / 4 + 0.5)
        return {"bytes": int(8 * copied * c["layers"] * c["kv_heads"] * c["dim"] + 4 * c["rows"] * c["held_hi"] / c["page"] + 40 * c["rows"]), "flops": 0}
    nodes = c["rows"] * (c["nodes_lo"] + c["nodes_hi"]) / 2
    if c["op"] == "plan":
        return {"bytes": int(16 * (nodes + c["pad"]) + 12 * c["rows"]), "flops": int(20 * nodes)}
    if c["op"] == "accept":
        moved = c["rows"] * min(1.5, 0.1 * (c["nodes_lo"] + c["nodes_hi"]) / 2)
        return {"bytes": int(8 * moved * c["layers"] * c["kv_heads"] * c["dim"] + 32 * nodes + 40 * c["rows"]), "flops": int(20 * nodes)}
    held = c["rows"] * (c["held_lo"] + c["held_hi"]) / 2
    each = nodes / c["rows"]
    return {"bytes": int(4 * (held + nodes) * c["kv_heads"] * c["dim"] + 4 * nodes * c["heads"] * c["dim"] + 4 * held / c["page"] + 8 * nodes),
            "flops": int(4 * c["heads"] * c["dim"] * each * (held + nodes / 4))}


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The outputs in 64 bits from the definition; whole numbers, and keys and values that are moved as they are, are compared as they are."""
    if case["op"] in ("plan", "accept", "fork"):
        return None
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    return _exact_adjust(s)


def _exact_attend(s):
    q, dim, page, kv_heads = s["q"].double(), s["dim"], s["kpages"].shape[2], s["kpages"].shape[1]
    out = torch.zeros_like(q)
    starts, lengths, masks = s["starts"].tolist(), s["lengths"].tolist(), s["masks"].tolist()
    for b, n in enumerate(lengths):
        count = starts[b + 1] - starts[b]
        pages = s["table"][b, :_pages(n, page)].long()
        keys = s["kpages"][pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :n].double()
        values = s["vpages"][pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :n].double()
        back = keys.transpose(1, 2).contiguous()
        for j in range(count):
            t = starts[b] + j
            score = torch.matmul(q[t].view(kv_heads, -1, dim), back) * dim ** -0.5
            hidden = [n - count + i for i in range(count) if not masks[t] >> i & 1]
            score[:, :, hidden] = float("-inf")
            out[t] = torch.matmul(torch.softmax(score, -1), values).flatten()
    return {"out": out}


def _exact_adjust(s):
    x = s["logits"].double()
    vocab = x.shape[1]
    value = lambda name, b: float(s[name][b])                             # noqa: E731
    for t, b in enumerate(s["requests"].tolist()):
        row = x[t]
        if s["history"] is not None:
            n, own_from = int(s["history_lengths"][b]), int(s["prompt_lengths"][b])
            path = s["drafted"][t][s["drafted"][t] >= 0].long() if s["drafted"] is not None else s["history"][b, :0].long()
            text = s["history"][b, :n].long()
            seen, said = torch.cat([text, path]), torch.bincount(torch.cat([text[own_from:], path]), minlength=vocab).double()
            index = seen.unique()
            row[index] = torch.where(row[index] > 0, row[index] / value("repetition", b), row[index] * value("repetition", b))
            row -= value("frequency", b) * said + value("presence", b) * (said > 0)
        if s["bias"] is not None:
            named = s["bias_tokens"][b] >= 0
            row[s["bias_tokens"][b][named].long()] += s["bias"][b][named].double()
        if s["allowed"] is not None and int(s["allowed_rows"][t]) >= 0:
            words = s["allowed"][s["allowed_rows"][t].long()].long() & 0xFFFFFFFF
            row[torch.arange(vocab, device=x.device)[(words[:, None] // (1 << torch.arange(32, device=x.device)) % 2 == 0).flatten()[:vocab]]] = float("-inf")
    return x
