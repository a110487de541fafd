"""Plain forms of the operators for drafted trees, forked rows and settings on logits: one request, one node, one page, one token at a time."""
import numpy as np
import torch

from paged_oracle import pages_of


def trees(granted, starts, T, most=64):
    """[(first token row, nodes)] of every request: no nodes where there are more than `most`, or than token rows."""
    found = []
    for b, n in enumerate(granted):
        start, end = starts[b], min(starts[b + 1], T)
        found.append((start, n if 0 < n <= most and n <= end - start else 0))
    return found


def ancestors(parents):
    """The node itself and its ancestors, for every node of one tree."""
    found = []
    for j, p in enumerate(parents):
        found.append({j} | (found[p] if 0 <= p < j else set()))
    return found


def plan(parents, lengths, granted, starts):
    """(positions, masks as signed 64-bit numbers)"""
    T = len(parents)
    positions, masks = [-1] * T, [0] * T
    for b, (start, n) in enumerate(trees(granted, starts, T)):
        for j, above in enumerate(ancestors(parents[start:start + n])):
            positions[start + j] = lengths[b] - granted[b] + len(above) - 1
            mask = sum(1 << i for i in above)
            masks[start + j] = mask - (1 << 64) if mask >> 63 else mask
    return positions, masks


def accept(tokens, parents, targets, lengths, granted, starts, table, ring, state, page, nodes):
    """(lengths, state, accepted, path, token, ring)"""
    ring, lengths = list(ring), list(lengths)
    pool, (head, count) = len(ring), state
    accepted, path, token = [], [], []
    for b, (start, n) in enumerate(trees(granted, starts, len(parents), nodes)):
        way = [0] if n else []
        while n:
            at = way[-1]
            child = [j for j in range(at + 1, n) if parents[start + j] == at and tokens[start + j] == targets[start + at]]
            if not child:
                break
            way.append(child[0])
        before, lengths[b] = lengths[b], lengths[b] - granted[b] + len(way)
        for p in table[b][pages_of(lengths[b], page):pages_of(before, page)]:
            ring[(head + count) % pool] = p
            count += 1
        accepted.append(len(way))
        path.append(way + [-1] * (nodes - len(way)))
        token.append(targets[start + way[-1]] if way else -1)
    return lengths, (head, count), accepted, path, token, ring


def moved(pages, slots, starts, path, page):
    """The pages [layers, pool, kv, page, d] after the accepted nodes' rows have moved."""
    pages = pages.clone()
    for b, way in enumerate(path):
        rows = [slots[starts[b] + j] for j in way if j >= 0]
        old = [pages[:, s // page, :, s % page].clone() for s in rows]
        for i, row in enumerate(old):
            to = slots[starts[b] + i]
            pages[:, to // page, :, to % page] = row
    return pages


def fork(source, lengths, table, ring, state, shares, page):
    """(table, ring, lengths, state, shares, granted, [(new page, the page it is a copy of, positions)])"""
    old, before, ring, shares = [list(r) for r in table], list(lengths), list(ring), list(shares)
    table, lengths = [list(r) for r in table], list(lengths)
    pool, (head, count) = len(ring), state
    B, used, short, granted, copies, moving = len(source), 0, False, [], [], []
    for b, s in enumerate(source):
        moves = s != b and -1 <= s < B
        n = before[s] if moves and s >= 0 else 0
        need = n % page != 0
        if need and (short or used == count):
            short, moves = True, False
            granted.append(0)
            continue
        granted.append(1)
        if not moves:
            continue
        moving.append(b)
        lengths[b] = n
        if n:
            table[b][:n // page] = old[s][:n // page]
        if need:
            table[b][n // page] = ring[(head + used) % pool]
            copies.append((table[b][n // page], old[s][n // page], n % page))
            used += 1
        for p in table[b][:n // page]:
            shares[p] += 1
    gone = []
    for b in moving:
        for p in old[b][:pages_of(before[b], page)]:
            shares[p] -= 1
            gone.append(p)
    back = []
    for p in gone:
        if shares[p] < 0:
            shares[p] = 0
            back.append(p)
    for j, p in enumerate(back):
        ring[(head + count + j) % pool] = p
    return table, ring, lengths, ((head + used) % pool, count - used + len(back)), shares, granted, copies


def adjust(x, seen=(), said=(), repetition=1.0, frequency=0.0, presence=0.0, bias=(), allowed=None):
    """One row of logits in 64 bits (before it is rounded, and whether it is held to fp16's largest numbers).  seen: tokens of the text; said: those
    behind the prompt; bias: (token, value) in order; allowed: truth values."""
    x = np.array(x, dtype=np.float64)
    V = len(x)
    finite = np.isfinite(x)
    r = repetition if repetition > 0 else 1.0
    for t in {t for t in list(seen) + list(said) if 0 <= t < V}:
        x[t] = x[t] / r if x[t] > 0 else x[t] * r
    for t in {t for t in said if 0 <= t < V}:
        x[t] -= frequency * list(said).count(t) + presence
    with np.errstate(invalid="ignore"):
        for t, w in {t: w for t, w in bias if 0 <= t < V}.items():
            x[t] += w
            finite[t] &= np.isfinite(w)
    x = np.where(finite, np.clip(x, -65504, 65504), x)
    return x if allowed is None else np.where(allowed, x, -np.inf)


def attend(q, keys, values, seen):
    """One token row: q [heads, d], keys and values [n, kv, d], seen [n]: (out, sum of weights times |v|, largest sum of |q k| / sqrt(d), sum of |v| over the sum of
    weights, the largest being 1), 64 bits."""
    heads, d = q.shape
    kv = keys.shape[1]
    if not bool(seen.any()):
        zero = torch.zeros(heads, d, dtype=torch.float64, device=q.device)
        return zero, zero, zero[:, :1], zero
    q = q.double().view(kv, -1, d)
    k, v = keys[seen].double().transpose(0, 1), values[seen].double().transpose(0, 1)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) / d ** 0.5
    size = (torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()) / d ** 0.5).amax(-1)
    e = (s - s.amax(-1, keepdim=True)).exp()
    total = e.sum(-1, keepdim=True)
    out, spread = torch.matmul(e / total, v), torch.matmul(e / total, v.abs())
    return out.reshape(heads, d), spread.reshape(heads, d), size.reshape(heads, 1), (v.abs().sum(1, keepdim=True) / total).expand(-1, q.shape[1], -1).reshape(heads, d)
