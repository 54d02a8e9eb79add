"""Trees of drafted tokens, attention with the weights that its keys get, and caches that keep some
of their rows, by their definitions in float64, one sequence at a time (tests only).

The reference has none of them; positions, tables and lengths mean what they do in its attention
(needle/layers/attention.py:120-154).
"""
import math

import torch

from . import fp8_ref


def parent_of(parents, t):
    """The node that node t of one sequence follows, or None."""
    p = int(parents[t])
    return p if 0 <= p < t else None


def sees(parents):
    """[n, n] truth values: node b is t itself or one of its ancestors."""
    n = len(parents)
    see = torch.zeros(n, n, dtype=torch.bool)
    for t in range(n):
        at = t
        while at is not None:
            see[t, at] = True
            at = parent_of(parents, at)
    return see


def mask_words(see, words):
    """[n, words] int64 of truth values [n, m]: bit b % 64 of word b // 64; none past the words."""
    out = torch.zeros(see.shape[0], words, dtype=torch.int64)
    for t, b in see.nonzero().tolist():
        if b // 64 < words:
            bit = 1 << (b % 64)
            out[t, b // 64] |= bit - (1 << 64) if bit >> 63 else bit
    return out


def pool_values(kv_cache):
    """Values of a 16-bit pool, or of (codes, scales), as a function of (blocks, rows):
    [keys, 2, Hkv, D] in float64."""
    if torch.is_tensor(kv_cache):
        return lambda blk, row: kv_cache[:, blk, :, row].double()
    codes, scales = kv_cache
    return lambda blk, row: fp8_ref.values(codes[:, blk, :, row], scales[:, blk, :, row])


class Attended:
    """out, weight [T, H, D]: the attention and sum_t p_t |v_t|; big [T, H]: the largest
    scale * sum_d |q_d k_d|; lens [T]: attended tokens; rows outside cu are NaN.  probs[i]:
    [n, H, keys] and at[i]: the keys' (position, block, row), of the sequences that have any."""


def attention(q, kv_cache, table, cu, context_lens, scale, see=None):
    """see(i): [n, n] which of the chunk's tokens token t attends (None: up to itself)."""
    _, nb, hkv, bs, d = (kv_cache if torch.is_tensor(kv_cache) else kv_cache[0]).shape
    values = pool_values(kv_cache)
    t, h, _ = q.shape
    g, w = h // hkv, table.shape[1]
    r = Attended()
    r.out = torch.full((t, h, d), math.nan, dtype=torch.float64)
    r.weight, r.big = r.out.clone(), torch.zeros(t, h, dtype=torch.float64)
    r.lens = torch.zeros(t, dtype=torch.long)
    r.probs, r.at = {}, {}
    for i in range(table.shape[0]):
        a, n = int(cu[i]), int(cu[i + 1]) - int(cu[i])
        ctx = int(context_lens[i])
        if n == 0:
            continue
        r.out[a:a + n], r.weight[a:a + n] = 0.0, 0.0
        if ctx < 0:
            continue
        at = [(p, fp8_ref.slot(table[i], p, bs, nb)) for p in range(min(ctx + n, w * bs))]
        at = [(p, *s) for p, s in at if s is not None]
        if not at:
            continue
        pos, blk, row = (torch.tensor(x) for x in zip(*at))
        kv = values(blk, row)
        tree = torch.ones(n, n, dtype=torch.bool).tril() if see is None else see(i)
        seen = (pos < ctx)[None] | tree[:, (pos - ctx).clamp(min=0)]
        r.lens[a:a + n] = seen.sum(1)
        some = seen.any(1)
        r.at[i], r.probs[i] = (pos, blk, row), torch.zeros(n, h, len(pos), dtype=torch.float64)
        for head in range(h):
            k, v = kv[:, 0, head // g], kv[:, 1, head // g]
            qr = q[a:a + n, head].double()
            s = (qr @ k.T * scale).masked_fill(~seen, -math.inf)
            p = torch.where(some[:, None] & seen, torch.softmax(s, dim=1), 0.0)
            r.probs[i][:, head] = p
            r.big[a:a + n, head] = torch.where(
                seen, qr.abs() @ k.abs().T, 0.0).nan_to_num(0.0).amax(1) * abs(scale)
            # what is not finite reaches the rows that attend it, and not as 0 * inf
            hits = [seen.double() @ x.double() > 0
                    for x in (v.isnan(), v == math.inf, v == -math.inf)]
            v = torch.where(v.isfinite(), v, 0.0)
            o = p @ v
            o = torch.where(hits[1], o + math.inf, o)      # (a NaN weight's stays)
            o = torch.where(hits[2], o - math.inf, o)
            r.out[a:a + n, head] = torch.where(hits[0] | (hits[1] & hits[2]), math.nan, o)
            r.weight[a:a + n, head] = p @ v.abs()
    return r


def mass(r, before, cu, context_lens, num_heads, decay=1.0):
    """The weights [NB, Hkv, bs] after an attention r: of cached tokens decay times what they were
    and what they got now, of the new ones what they got."""
    out = before.double().clone()
    hkv = before.shape[1]
    for i, (pos, blk, row) in r.at.items():
        p = r.probs[i]
        got = p.view(p.shape[0], hkv, num_heads // hkv, -1).sum((0, 2))       # [Hkv, keys]
        for x in range(len(pos)):
            b, y = int(blk[x]), int(row[x])
            old = out[b, :, y] * decay if int(pos[x]) < int(context_lens[i]) and decay else 0.0
            out[b, :, y] = old + got[:, x]
    return out


def verify(logits, ids, parents, cu, uniforms, temperature=None):
    """(tokens, accepted, path)."""
    t, v = logits.shape
    n = len(cu) - 1
    tokens, accepted, path = [-1] * t, [0] * n, [-1] * t

    def target(i, r):
        row = logits[r].double()
        temp = 1.0 if temperature is None else float(temperature[i])
        if not temp > 0 or not math.isfinite(float(row.max())):
            p = torch.zeros(v, dtype=torch.float64)
            p[fp8_ref.point(logits[r])] = 1.0
            return p
        return torch.softmax((row - row.max()) / temp, dim=0)

    for i in range(n):
        a, b = int(cu[i]), int(cu[i + 1])
        up = [parent_of(parents[a:b], x) for x in range(b - a)]
        at, k = 0, 0
        path[a] = 0
        while True:
            p = target(i, a + at)
            kids = [x for x in range(b - a) if up[x] == at]
            upto, seen, to = 0.0, set(), None
            for x in kids:
                token = int(ids[a + x])
                if token in seen or not 0 <= token < v:
                    continue
                seen.add(token)
                upto += float(p[token])
                if float(uniforms[a + at]) < upto:
                    to = x
                    break
            if to is None:
                break
            tokens[a + k] = int(ids[a + to])
            k += 1
            path[a + k] = at = to
        accepted[i] = k
        weights = p.clone()
        for x in kids:
            if 0 <= int(ids[a + x]) < v:
                weights[int(ids[a + x])] = 0.0
        if not float(weights.sum()) > 0:
            tokens[a + k] = fp8_ref.point(logits[a + at])
            continue
        u = float(uniforms[b - 1])
        u = min(max(u, 0.0), 1.0) if u == u else 0.0
        # sums of whole numbers: a border that u falls on exactly is kept
        w = [int(math.ldexp(x, 200)) for x in weights.tolist()]
        num, den = u.as_integer_ratio()
        goal, upto, last = num * sum(w), 0, 0
        for x, y in enumerate(w):
            upto += y
            if y > 0:
                last = x
                if upto * den > goal:
                    break
        tokens[a + k] = last
    return tokens, accepted, path


def select(mass, table, lens, budget, sinks=0, recent=0):
    """(keep [B, Hkv, budget], kept [B]): of every kv head the positions that stay, ascending.  A NaN
    counts as the largest weight; rows without a block as the smallest."""
    nb, hkv, bs = mass.shape
    n, w = table.shape
    keep = torch.full((n, hkv, budget), -1, dtype=torch.int32)
    kept = torch.zeros(n, dtype=torch.int32)
    for i in range(n):
        length = max(0, min(int(lens[i]), w * bs))
        k = kept[i] = min(length, budget)
        for head in range(hkv):
            def rank(p):
                at = fp8_ref.slot(table[i], p, bs, nb)
                x = -math.inf if at is None else float(mass[at[0], head, at[1]])
                always = p < sinks or p >= length - recent
                return (not always, x == x, -x if x == x else 0.0, p)
            best = sorted(range(length), key=rank)[:int(k)]
            keep[i, head, :int(k)] = torch.tensor(sorted(best), dtype=torch.int32)
    return keep, kept


def compact(tensors, table, keep, counts, first=None, cu=None, dst_table=None):
    """Rows moved in place in tensors [.., NB, Hkv, bs, ..] given as (tensor, dim of NB)."""
    to = table if dst_table is None else dst_table
    for x, dim in tensors:
        y = x.movedim(dim, 0).movedim(dim + 1, 1).movedim(dim + 2, 2)     # [NB, Hkv, bs, ..] view
        nb, hkv, bs = y.shape[:3]
        old = y.clone()
        for i in range(table.shape[0]):
            base = 0 if first is None else int(first[i])
            if base < 0:
                continue
            for head in range(hkv):
                rows = keep[int(cu[i]):int(cu[i + 1])] if cu is not None else keep[i, head]
                for j in range(min(int(counts[i]), len(rows))):
                    a, b = base + int(rows[j]), base + j
                    if int(rows[j]) < 0 or a >= table.shape[1] * bs or b >= to.shape[1] * bs:
                        continue
                    s, t = (fp8_ref.slot(tb[i], p, bs, nb) for tb, p in ((table, a), (to, b)))
                    if s is not None and t is not None:
                        y[t[0], head, t[1]] = old[s[0], head, s[1]]
