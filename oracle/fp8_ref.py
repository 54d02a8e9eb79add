"""The 8-bit pool and draft verification from their definitions, in float64 on the CPU (tests
only)."""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def code_values() -> torch.Tensor:
    """The value of each e4m3 byte (NaN at 0x7f and 0xff)."""
    out = []
    for b in range(256):
        m, e = b & 7, (b >> 3) & 15
        v = (1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6
        v = math.nan if b & 127 == 127 else v
        out.append(-v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def quantise_row(x):
    """(codes, byte) of one row of floats: the nearest code of x * 2^-e, ties to the even code."""
    table = code_values()[:127]
    finite = [abs(v) for v in x if math.isfinite(v)]
    a, e = max(finite, default=0.0), -126
    while a > E4M3_MAX * 2.0 ** e:
        e += 1
    codes = []
    for v in x:
        if not math.isfinite(v):
            codes.append(0x7F)
            continue
        y = abs(v) * 2.0 ** -e
        d = (table - y).abs()
        near = (d == d.min()).nonzero()[:, 0].tolist()
        c = near[0] if len(near) == 1 else next(i for i in near if i % 2 == 0)
        codes.append(c | (0x80 if math.copysign(1.0, v) < 0 else 0))
    return codes, e + 127


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of codes [.., D] (bytes) under scales [..]."""
    two = torch.tensor([2.0 ** (b - 127) for b in range(256)], dtype=torch.float64)
    return code_values()[codes.view(torch.uint8).long()] * two[scales.long()].unsqueeze(-1)


def slot(table_row, p, block_size, num_blocks):
    """(block, row) of position p, or None."""
    if p < 0:
        return None
    b = int(table_row[min(p // block_size, len(table_row) - 1)])
    return (b, p % block_size) if 0 <= b < num_blocks else None


def append(k, v, codes, scales, block_table, cu, context_lens):
    """Rows of k and v into the pool's bytes, in place."""
    for i in range(block_table.shape[0]):
        for t in range(int(cu[i]), int(cu[i + 1])):
            at = slot(block_table[i], int(context_lens[i]) + t - int(cu[i]), codes.shape[3],
                      codes.shape[1])
            for plane, x in enumerate((k, v)):
                for head in range(x.shape[1] if at is not None else 0):
                    c, byte = quantise_row(x[t, head].double().tolist())
                    codes[plane, at[0], head, at[1]] = torch.tensor(c, dtype=torch.uint8)
                    scales[plane, at[0], head, at[1]] = byte


def attention(q, codes, scales, block_table, cu, context_lens, scale):
    """(out, weight) [T, H, D] in float64: the attention, and sum_t p_t |v_t|, what a rounding of
    the probabilities is relative to; rows outside cu are NaN.  Also the largest
    scale * sum_d |q_d k_d| of every row [T, H] and the attended lengths [T]."""
    _, nb, hkv, bs, d = codes.shape
    t, h, _ = q.shape
    g = h // hkv
    out = torch.full((t, h, d), math.nan, dtype=torch.float64)
    weight, big = out.clone(), torch.zeros(t, h, dtype=torch.float64)
    lens = torch.zeros(t, dtype=torch.long)
    w = block_table.shape[1]
    for i in range(block_table.shape[0]):
        a, n = int(cu[i]), int(cu[i + 1]) - int(cu[i])
        ctx = int(context_lens[i])
        if n == 0:
            continue
        out[a:a + n], weight[a:a + n] = 0.0, 0.0
        if ctx < 0:
            continue
        at = [(p, slot(block_table[i], p, bs, nb)) for p in range(min(ctx + n, w * bs))]
        at = [(p, s) for p, s in at if s is not None]
        if not at:
            continue
        pos = torch.tensor([p for p, _ in at])
        blk, row = (torch.tensor(x) for x in zip(*(s for _, s in at)))
        kv = values(codes[:, blk, :, row], scales[:, blk, :, row])         # [keys, 2, Hkv, D]
        seen = pos[None, :] <= ctx + torch.arange(n)[:, None]              # [n, keys]
        lens[a:a + n] = seen.sum(1)
        some = seen.any(1)
        for head in range(h):
            k, v = kv[:, 0, head // g], kv[:, 1, head // g]
            qr = q[a:a + n, head].double()
            s = (qr @ k.T * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, dim=1)
            p = torch.where(some[:, None] & seen, p, 0.0)
            # a NaN reaches the rows that attend it, and not as 0 * NaN
            nan = (seen.double() @ v.isnan().double() > 0)
            big[a:a + n, head] = torch.where(
                seen, qr.abs() @ k.abs().T, 0.0).nan_to_num(0.0).amax(1) * abs(scale)
            o = p @ v.nan_to_num(0.0)
            out[a:a + n, head] = torch.where(nan, math.nan, o)
            weight[a:a + n, head] = p @ v.nan_to_num(0.0).abs()
    return out, weight, big, lens


def point(row: torch.Tensor) -> int:
    """torch's argmax: the first NaN, or the first of the largest."""
    return int(row.argmax())


def verify(logits, ids, cu, uniforms, temperature=None, draft_probs=None):
    """(tokens, accepted) by the definition, one sequence at a time."""
    t, v = logits.shape
    n = len(cu) - 1
    tokens, accepted = [-1] * t, [0] * n

    def target(i, r):
        row = logits[r].double()
        temp = 1.0 if temperature is None else float(temperature[i])
        if not temp > 0 or not math.isfinite(float(row.max())):
            p = torch.zeros(v, dtype=torch.float64)
            p[point(logits[r])] = 1.0
            return p
        return torch.softmax((row - row.max()) / temp, dim=0)

    for i in range(n):
        a, b = int(cu[i]), int(cu[i + 1])
        k = 0
        for r in range(a, b - 1):
            x = int(ids[r + 1])
            p = target(i, r)
            q = torch.zeros(v, dtype=torch.float64)
            if draft_probs is not None:
                q = draft_probs[r - i].double()
            elif 0 <= x < v:
                q[x] = 1.0
            if not (0 <= x < v and float(uniforms[r]) * float(q[x]) < float(p[x])):
                break
            tokens[a + k] = x
            k += 1
        accepted[i] = k
        p = target(i, a + k)
        weights = p
        if a + k < b - 1:
            weights = (p - torch.where(q > 0, q, 0.0)).clamp(min=0.0)
            if not float(weights.sum()) > 0:
                weights = p
        u = float(uniforms[b - 1])
        u = min(max(u, 0.0), 1.0) if u == u else 0.0
        c = weights.cumsum(0)
        hit = ((c > u * c[-1]) & (weights > 0)).nonzero()[:, 0]
        some = (weights > 0).nonzero()[:, 0]
        tokens[a + k] = int(hit[0]) if len(hit) else int(some[-1])
    return tokens, accepted
