"""Plain 64-bit forms of the operators for requests of unequal lengths, one request, one token, one page at a time."""
import numpy as np
import torch


def pages_of(n, page):
    return -(-n // page)


def plan(lengths, new, table, ring, state, page, tokens, released=None):
    """(table, ring, lengths, state, granted, starts, positions, slots) afterwards, as lists and arrays of their own."""
    table, ring, lengths = [list(r) for r in table], list(ring), list(lengths)
    B, pool, max_pages = len(lengths), len(ring), len(table[0]) if table else 0
    head, count = state
    free = [ring[(head + j) % pool] for j in range(count)]
    granted, starts, positions, slots = [0] * B, [0], [-1] * tokens, [-1] * tokens
    back, short, used = [], False, 0
    for b in range(B):
        starts.append(starts[-1] + new[b])
        if released is not None and released[b]:
            back += table[b][:pages_of(lengths[b], page)]
            lengths[b] = 0
    for b in range(B):
        have = pages_of(lengths[b], page)
        need = pages_of(lengths[b] + new[b], page) - have
        if have + need > max_pages or starts[b + 1] > tokens:
            continue
        if need and (short or used + need > count):
            short = True
            continue
        table[b][have:have + need] = free[used:used + need]
        used += need
        for i in range(new[b]):
            p = lengths[b] + i
            positions[starts[b] + i] = p
            slots[starts[b] + i] = table[b][p // page] * page + p % page
        lengths[b] += new[b]
        granted[b] = new[b]
    for j, p in enumerate(back):
        ring[(head + count + j) % pool] = p
    return table, ring, lengths, ((head + used) % pool, count - used + len(back)), granted, starts, positions, slots


def rotate(x, cos, sin):
    """x [.., d] in 64 bits, cos and sin [.., d / 2]."""
    a, b = x.double().chunk(2, -1)
    cos, sin = cos.double(), sin.double()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def attend(q, keys, values, kv_heads):
    """(out, sum of weights times |v|, largest sum of |q k| / sqrt(d), what weights below 2^-25 of the largest add) of one request: q [heads, d],
    keys and values [n, kv_heads, d], 64 bits."""
    heads, d = q.shape
    q = q.double().view(kv_heads, -1, d)
    k, v = keys.double().transpose(0, 1), values.double().transpose(0, 1)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) / d ** 0.5
    size = (torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()) / d ** 0.5).amax(-1)
    e = (s - s.amax(-1, keepdim=True)).exp()
    total = e.sum(-1, keepdim=True)
    out, spread = torch.matmul(e / total, v), torch.matmul(e / total, v.abs())
    lost = 2.0 ** -25 * v.abs().sum(1, keepdim=True) / total
    return out.reshape(heads, d), spread.reshape(heads, d), size.reshape(heads, 1), lost.reshape(heads, d)


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row of logits (any float array) -> index."""
    x = np.array(x, dtype=np.float64)
    x[np.isnan(x)] = -np.inf
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return 0
    if not temperature > 0:
        return int(order[0])
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(np.float32(temperature))))
    w[(x == -np.inf) | (w < 1e-300)] = 0.0
    if top == np.inf:
        w[x != top] = 0.0
    keep = np.zeros(len(x), bool)
    kept = order[:top_k] if 0 < top_k < len(x) else order
    if top_p < 1.0:
        s = w[kept]
        before = np.concatenate([[0.0], np.cumsum(s)[:-1]])
        stay = before < np.float64(np.float32(top_p)) * s.sum()
        stay[0] = True
        kept = kept[stay]
    keep[kept] = True
    if min_p > 0:
        keep &= w >= min(np.float64(np.float32(min_p)), 1.0)
    c = np.cumsum(np.where(keep, w, 0.0))
    u = min(max(float(np.float32(u)), 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    return int(np.argmax(c > u * c[-1]))
