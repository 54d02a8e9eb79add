"""The measured work of speculation by trees and of bounded caches, over the paged pools.

Kinds of case (field "kind"):
  plan    a batch of drafted trees, given by each node's parent, as the words that say which nodes
          a node sees, and every node's depth (ops.tree_mask); once a step, for all layers.
  tree    attention of the trees' nodes over the paged pool that holds the cached tokens and the
          nodes: a node sees what is cached, its ancestors and itself (ops.tree_attention).
  verify  the trees against the target's logits (ops.verify_tree).
  commit  the accepted path's rows move to the front of their sequence's nodes, in every layer's
          pool (ops.kv_compact, in place).
  weigh   attention whose weights are added up for every cached token and kv head: a decode step,
          or a window of a prompt's last tokens (ops.attention_mass).
  evict   of every kv head the tokens with the largest weights stay, beside the first and the latest
          (ops.kv_select), and move to other blocks with their weights (ops.kv_compact).

A pool in 8 bits stores a row of K or V (one token, one head) as e4m3 codes and one byte s: the
values are code * 2^(s - 127), with the smallest power of two that keeps the row's largest within
448.  Weights are float32 [num_blocks, num_kv_heads, block_size], a number for each row of K.

Lengths and (but for a plan) trees belong to the case (field "lens"), values and block tables to
the seed.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0

# heads, kv heads, head_dim
QWEN_05B = (14, 2, 64)
QWEN_7B = (28, 4, 128)
LLAMA_8B = (32, 8, 128)

SHAPES = (QWEN_05B, QWEN_7B, LLAMA_8B, (32, 32, 128), (4, 1, 128), (7, 1, 64), (12, 4, 64))
VOCABS = (151936, 128256, 32000, 50257, 4099)


def _case(name, kind, shape=LLAMA_8B, **more):
    h, hkv, d = shape
    c = {"name": name, "kind": kind, "heads": h, "kv_heads": hkv, "head_dim": d, "dtype": "bf16",
         "page": 16, "lens": 3, "new_lo": 1, "new_hi": 1, "layers": 1, "fp8": False}
    c.update(more)
    return c


def listed():
    return [
        # the trees of a small batch: latency
        _case("plan-step", "plan", seqs=8, new_lo=16, new_hi=26),
        # many and large trees
        _case("plan-batch", "plan", seqs=64, new_lo=60, new_hi=400, lens=5),
        # a step of a small model and batch: latency
        _case("tree-small", "tree", QWEN_05B, seqs=4, lo=64, hi=800, new_lo=16, new_hi=16),
        # an ordinary step: trees of uneven sizes after contexts of uneven lengths
        _case("tree-batch", "tree", LLAMA_8B, seqs=64, lo=512, hi=4096, new_lo=16, new_hi=64,
              lens=4),
        # few long contexts in an 8-bit pool, an fp16 model with larger pages
        _case("tree-long-fp8", "tree", QWEN_7B, seqs=8, lo=4096, hi=32768, new_lo=40, new_hi=60,
              dtype="fp16", page=64, fp8=True, lens=9),
        # one tree: latency
        _case("verify-one", "verify", seqs=1, new_lo=60, new_hi=60, vocab=151936, greedy=0, lens=1),
        # a batch, some sequences greedy
        _case("verify-batch", "verify", seqs=32, new_lo=16, new_hi=64, vocab=128256, greedy=4,
              lens=2),
        # what was accepted of a batch's trees, in all layers of a model
        _case("commit-layers", "commit", LLAMA_8B, seqs=32, lo=16, hi=200, new_lo=16, new_hi=64,
              layers=32, lens=6),
        # an ordinary decode step
        _case("weigh-step", "weigh", LLAMA_8B, seqs=64, lo=512, hi=4096, lens=4),
        # the last tokens of prompts that were prefilled before, an fp16 model, larger pages
        _case("weigh-window-fp16", "weigh", QWEN_7B, seqs=8, lo=2000, hi=16000, new_lo=32,
              new_hi=32, dtype="fp16", page=64, lens=11),
        # a small batch whose caches have just passed their bound: latency
        _case("evict-step", "evict", QWEN_05B, seqs=8, lo=530, hi=640, budget=512, sinks=4,
              recent=64, lens=7),
        # long prompts cut to their bound after the prefill
        _case("evict-prompts-fp16", "evict", LLAMA_8B, seqs=16, lo=4096, hi=16384, budget=2048,
              sinks=4, recent=256, dtype="fp16", page=32, lens=8),
    ]


def _between(rng, lo, hi):
    """Spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "tree", "tree", "verify", "commit", "weigh", "weigh", "evict"))
    shape = rng.choice(SHAPES)
    h, hkv, d = shape
    more = {"dtype": rng.choice(("bf16", "fp16")), "page": rng.choice((16, 16, 32, 64, 256)),
            "lens": rng.randrange(1 << 20)}
    if kind == "plan":
        seqs = _between(rng, 1, 64)
        hi = _between(rng, 12, 400)
        more.update(seqs=seqs, new_lo=rng.randint(12, hi), new_hi=hi)
    elif kind == "verify":
        vocab = rng.choice(VOCABS)
        hi = _between(rng, 1, 64)
        more.update(seqs=min(_between(rng, 1, 100), max(1, 1200 // hi)), new_lo=rng.randint(1, hi),
                    new_hi=hi, vocab=vocab, greedy=rng.choice((0, 0, 3)),
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    elif kind == "tree":
        hi_new = _between(rng, 1, 130)
        seqs = _between(rng, 1, 64)
        hi = max(1, min(_between(rng, 32, 32768), 1000000 // (hkv * seqs),
                        16000000 // (h * hi_new * seqs)))
        more.update(seqs=seqs, lo=rng.choice((0, hi // 8)), hi=hi, new_lo=rng.randint(1, hi_new),
                    new_hi=hi_new, fp8=rng.random() < 0.35)
    elif kind == "commit":
        hi_new = _between(rng, 2, 64)
        seqs = _between(rng, 1, 32)
        more.update(seqs=seqs, lo=0, hi=_between(rng, 2, 200), new_lo=rng.randint(1, hi_new),
                    new_hi=hi_new, layers=rng.randint(1, 12), fp8=rng.random() < 0.35)
    elif kind == "weigh":
        new_hi = rng.choice((1, 1, _between(rng, 2, 64)))
        seqs = _between(rng, 1, 64)
        hi = max(1, min(_between(rng, 32, 16384), 1000000 // (hkv * seqs),
                        16000000 // (h * new_hi * seqs)))
        more.update(seqs=seqs, lo=rng.choice((0, hi // 8)), hi=hi,
                    new_lo=1 if new_hi == 1 else rng.randint(1, new_hi), new_hi=new_hi)
    else:
        seqs = _between(rng, 1, 32)
        hi = max(20, min(_between(rng, 40, 16384), 700000 // (hkv * seqs)))
        budget = max(8, int(hi * rng.uniform(0.1, 0.9)))
        more.update(seqs=seqs, lo=hi // 4, hi=hi, budget=budget, sinks=rng.choice((0, 4)),
                    recent=rng.choice((0, budget // 8, budget // 2)))
    c = _case("", kind, shape, **more)
    if "lo" in c:
        c["lo"] = min(c["lo"], c["hi"])
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs

def _lengths(case):
    """(cached tokens, new tokens) of every sequence."""
    r = np.random.default_rng(case["lens"])
    n = r.integers(case["new_lo"], case["new_hi"], size=case["seqs"], endpoint=True).tolist()
    if "lo" not in case:
        return [0] * len(n), n
    lo, hi = case["lo"], case["hi"]
    c = np.exp(r.uniform(math.log(lo + 1), math.log(hi + 2), case["seqs"])).astype(np.int64) - 1
    return np.clip(c, lo, hi).tolist(), n


def _trees(case, seed=0):
    """Every sequence's parents (node 0 is its newest token, parents come before their children),
    the nodes in the order in which a drafter takes them: a few long branches, many short ones."""
    r = np.random.default_rng((case["lens"], seed))
    out = []
    for n in _lengths(case)[1]:
        j = np.arange(n)
        p = np.floor(j * r.uniform(0, 1, n) ** r.uniform(0.4, 2.0)).astype(np.int64)
        p = np.minimum(p, j - 1)
        # no more than eight children of a node
        kids = np.zeros(n + 1, dtype=np.int64)
        for x in range(1, n):
            while kids[p[x]] >= 8:
                p[x] = (p[x] + 1) % x
            kids[p[x]] += 1
        out.append(p)
    return out


def _sees(p):
    """[n, n] truth values: node b is t itself or an ancestor of it."""
    n = len(p)
    see = np.zeros((n, n), dtype=bool)
    for t in range(n):
        if t > 0 and p[t] >= 0:
            see[t] = see[p[t]]
        see[t, t] = True
    return see


def _power(byte):
    """2^(byte - 127) in float32, exactly; byte from 1 to 254."""
    return (byte.int() << 23).view(torch.float32)


def _quantise(x):
    """Codes and scale bytes of the rows of x (finite), in torch operations."""
    m, ex = torch.frexp(x.float().abs().amax(-1))
    byte = (ex + 118 + (m > E4M3_MAX / 512)).clamp_(min=1)
    codes = (x.float() * _power(254 - byte).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes, byte.to(torch.uint8)


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEVICE)


def _bytes_of(pool):
    """The pool's tensors whose rows move: of an 8-bit one the codes as bytes, and the scales."""
    return [pool] if torch.is_tensor(pool) else [pool[0].view(torch.uint8), pool[1]]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    host = np.random.default_rng(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    ctx, new = _lengths(case)
    total, n = sum(new), len(new)
    cu = np.concatenate([[0], np.cumsum(new)])
    s = {"case": case, "max_new": max(new), "total": total, "cu": _i32(cu)}

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)

    if kind in ("plan", "tree", "verify"):
        trees = _trees(case, seed if kind == "plan" else 0)   # the trees are a plan's inputs
        s["parents"] = _i32(np.concatenate(trees))
        s["depth"] = max(int(_sees(p).sum(1).max()) for p in trees)
    if kind == "plan":
        return s
    if kind == "verify":
        v = case["vocab"]
        s["uniforms"] = torch.rand(total, generator=gen, device=DEVICE)
        temp = torch.rand(n, generator=gen, device=DEVICE).mul_(0.7).add_(0.5)
        if case["greedy"]:
            temp[::case["greedy"]] = 0.0
        s["temperature"] = temp
        # a peaked distribution over a long tail, and a drafter near it: a node's children are
        # its best tokens, the first the best
        s["logits"] = torch.empty(total, v, dtype=dtype, device=DEVICE)
        best = torch.empty(total, 8, dtype=torch.long, device=DEVICE)
        for a in range(0, total, 512):
            x = randn(min(512, total - a), v).mul_(2.2)
            s["logits"][a:a + 512] = x.to(dtype)
            best[a:a + 512] = x.add_(randn(*x.shape).mul_(0.3)).topk(8, -1).indices
        row, rank = np.zeros(total, dtype=np.int64), np.zeros(total, dtype=np.int64)
        for i, p in enumerate(trees):
            seen = {}
            for x in range(1, len(p)):
                row[cu[i] + x] = cu[i] + p[x]
                rank[cu[i] + x] = seen.get(p[x], 0)
                seen[p[x]] = rank[cu[i] + x] + 1
        s["ids"] = best[torch.from_numpy(row).to(DEVICE), torch.from_numpy(rank).to(DEVICE)]
        return s

    h, hkv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if kind == "evict":
        new = [0] * n
    blocks = [-(-(c + m) // page) for c, m in zip(ctx, new)]
    kept = [-(-min(c, case["budget"]) // page) if kind == "evict" else 0 for c in ctx]
    held = sum(blocks)
    num_blocks = held + sum(kept) + 2
    perm = host.permutation(held)
    table = np.full((n, max(max(blocks), 1)), num_blocks - 1, dtype=np.int32)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = perm[at:at + b]
        at += b
    s.update(table=_i32(table), lens=_i32(ctx), max_ctx=max(ctx), scale=1.0 / math.sqrt(d))
    # what the pool holds: keys with a few channels far larger than the rest
    gain = torch.ones(d, device=DEVICE)
    gain[3::29] = 4.0

    def pool():
        shape = (2, num_blocks, hkv, page)
        if case["fp8"]:
            out = (torch.empty(*shape, d, dtype=torch.float8_e4m3fn, device=DEVICE),
                   torch.empty(*shape, dtype=torch.uint8, device=DEVICE))
        else:
            out = torch.empty(*shape, d, dtype=dtype, device=DEVICE)
        step = max(1, (1 << 26) // (hkv * page * d))
        for b in range(0, num_blocks, step):
            e = min(num_blocks, b + step)
            for p, g in ((0, gain), (1, 1.0)):
                x = (randn(e - b, hkv, page, d) * g).to(dtype)
                if case["fp8"]:
                    out[0][p, b:e], out[1][p, b:e] = _quantise(x)
                else:
                    out[p, b:e] = x
        return out

    s["pools"] = [pool() for _ in range(case["layers"])]
    if kind in ("tree", "weigh"):
        # the projection's output: a view of a fused q/k/v row per token
        qkv = randn(total, (h + 2 * hkv) * d).to(dtype)
        s["q"] = qkv[:, :h * d].view(total, h, d)
    if kind == "tree":
        words = (max(new) + 63) // 64
        see = np.zeros((total, words * 64), dtype=bool)
        for i, p in enumerate(trees):
            see[cu[i]:cu[i + 1], :len(p)] = _sees(p)
        bits = np.packbits(see, axis=1, bitorder="little").view(np.int64)
        s["mask"] = torch.from_numpy(bits.copy()).to(DEVICE)
    elif kind == "commit":
        # paths: a node's best child comes next to it in the first few, which stay where they are
        path = np.full(total, -1, dtype=np.int64)
        count = np.zeros(n, dtype=np.int64)
        for i, m in enumerate(new):
            c = int(host.integers(1, min(m, 8), endpoint=True))
            stay = int(host.integers(1, c, endpoint=True))
            far = np.sort(host.permutation(np.arange(c, m))[:c - stay])
            c = stay + len(far)
            path[cu[i]:cu[i] + c] = np.concatenate([np.arange(stay), far])
            count[i] = c
        s["path"], s["count"] = _i32(path), _i32(count)
    elif kind == "weigh":
        # the weights so far: a few tokens have most of them
        s["before"] = randn(num_blocks, hkv, page).mul_(2.5).exp_().mul_(0.01)
        s["mass"] = s["before"].clone()
    elif kind == "evict":
        s["mass"] = randn(num_blocks, hkv, page).mul_(2.5).exp_().mul_(0.01)
        # equal ones among them: tokens that nothing has attended
        s["mass"][s["mass"] < 0.002] = 0.0
        to = np.full((n, max(kept)), num_blocks - 1, dtype=np.int32)
        fresh = held + host.permutation(sum(kept))
        at = 0
        for i, b in enumerate(kept):
            to[i, :b] = fresh[at:at + b]
            at += b
        s["to"] = _i32(to)
        s["fresh"] = (held, held + sum(kept))
    return s


# ---------------------------------------------------------------------------- plain forms

def _owner(cu, total):
    """(sequence, offset in it) of each of `total` packed tokens."""
    t = torch.arange(total, device=DEVICE)
    i = torch.searchsorted(cu[1:].long(), t, right=True)
    return i, t - cu.long()[i]


def _words(see):
    """[T, 64 W] truth values as int64 [T, W], bit b of word w for place 64 w + b."""
    w = see.view(see.shape[0], -1, 64).long() << torch.arange(64, device=DEVICE)
    return w.sum(-1)


def _plain_plan(s):
    total, most = s["total"], s["max_new"]
    i, j = _owner(s["cu"], total)
    base = s["cu"].long()[i]
    up = s["parents"].long()
    at = j
    see = torch.zeros(total, (most + 63) // 64 * 64, dtype=torch.bool, device=DEVICE)
    for _ in range(s["depth"]):
        see |= (torch.arange(see.shape[1], device=DEVICE) == at[:, None])
        p = up[base + at.clamp(min=0)]
        at = torch.where((at >= 0) & (p >= 0) & (p < at), p, -1)
    return _words(see), (see.sum(-1) - 1).int()


def _plane(s, p):
    """K or V of the sequences' table rows, in float32: [B, Hkv, W * page, D]."""
    pool, t = s["pools"][0], s["table"].long()
    if torch.is_tensor(pool):
        x = pool[p][t].float()
    else:
        x = pool[0].view(torch.uint8)[p][t].view(torch.float8_e4m3fn).float()
        x = x * _power(pool[1][p][t]).unsqueeze(-1)
    b, w, hkv, page, d = x.shape
    return x.transpose(1, 2).reshape(b, hkv, w * page, d)


def _padded(s):
    """(sequence, offset) of the packed tokens and q as [B, N, H, D] in float32."""
    i, j = _owner(s["cu"], s["total"])
    q = torch.zeros(s["lens"].shape[0], s["max_new"], *s["q"].shape[1:], device=DEVICE)
    q[i, j] = s["q"].float()
    return i, j, q


def _plain_attention(s, q, show):
    """q [B, N, H, D], show [B, N, keys]: outputs and, per kv head, weights [B, Hkv, g, N, keys]."""
    b, n, h, d = q.shape
    k = _plane(s, 0)
    hkv = k.shape[1]
    qg = q.view(b, n, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    w = torch.matmul(qg, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    del k
    w = w.view(b, hkv, h // hkv, n, -1).masked_fill_(~show[:, None, None], -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    w = w.div_(w.sum(-1, keepdim=True).clamp(min=1e-30))
    o = torch.matmul(w.view(b, hkv, -1, w.shape[-1]), _plane(s, 1))
    return o.view(b, hkv, h // hkv, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d), w


def _key_index(s):
    """Position of each key of a table row less the sequence's cached tokens: [B, keys]."""
    page = _bytes_of(s["pools"][0])[0].shape[3]
    return torch.arange(s["table"].shape[1] * page, device=DEVICE) - s["lens"].long()[:, None]


def _plain_tree(s):
    i, j, q = _padded(s)
    at, most = _key_index(s), s["max_new"]
    see = (s["mask"][:, :, None] >> torch.arange(64, device=DEVICE)) & 1
    seen = torch.zeros(q.shape[0], most, most, dtype=torch.bool, device=DEVICE)
    seen[i, j] = see.view(s["total"], -1)[:, :most] > 0
    node = at.clamp(0, most - 1)[:, None].expand(-1, most, -1)
    show = torch.where(at[:, None] < 0, True, seen.gather(2, node))
    show &= (at < s["cu"].diff().long()[:, None])[:, None]
    return _plain_attention(s, q, show)[0][i, j].to(s["q"].dtype)


def _plain_verify(s):
    cu, ids, u, logits = s["cu"].long(), s["ids"], s["uniforms"].double(), s["logits"]
    total, v = logits.shape
    n, most = cu.shape[0] - 1, s["max_new"]
    i, j = _owner(cu, total)
    temp = s["temperature"].double()[i]
    top, best = logits.double().max(-1)
    p = logits.double().sub_(top[:, None]).div_(torch.where(temp > 0, temp, 1.0)[:, None]).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    point = (torch.arange(v, device=DEVICE) == best[:, None]).double()
    p = torch.where((temp > 0)[:, None], p, point)
    # each node's probability where it hangs, and with those of its earlier siblings
    grid = lambda x, fill: torch.full((n, most), fill, dtype=x.dtype,  # noqa: E731
                                      device=DEVICE).index_put_((i, j), x)
    up = s["parents"].long()
    px = p[cu[:-1][i] + up.clamp(min=0), ids]
    up, tok, px, us = grid(up, -1), grid(ids, -1), grid(px, 0.0), grid(u, 0.0)
    earlier = (up[:, :, None] == up[:, None]) & (torch.arange(most, device=DEVICE)[:, None]
                                                 > torch.arange(most, device=DEVICE))
    again = (earlier & (tok[:, :, None] == tok[:, None])).any(-1)
    px = torch.where(again, 0.0, px)
    upto = px + (earlier * px[:, None]).sum(-1)
    hangs = up >= 0
    taken = hangs & (us.gather(1, up.clamp(min=0)) < upto)
    # the path: from a node to the first of its children that is taken
    at = torch.zeros(n, dtype=torch.long, device=DEVICE)
    path = torch.full((n, most), -1, dtype=torch.long, device=DEVICE)
    path[:, 0] = 0
    accepted = torch.zeros(n, dtype=torch.long, device=DEVICE)
    going = torch.ones(n, dtype=torch.bool, device=DEVICE)
    for step in range(1, s["depth"]):
        kid = taken & (up == at[:, None]) & going[:, None]
        going = kid.any(-1)
        at = torch.where(going, kid.long().argmax(-1), at)
        path[:, step] = torch.where(going, at, -1)
        accepted += going
    # the token after it: none of the children that were not taken
    w = p[cu[:-1] + at]
    kids = (up == at[:, None]) & hangs
    left = torch.cat([w, w[:, :1]], dim=1)
    left = left.scatter_(1, torch.where(kids, tok, v), 0.0)[:, :v]
    c = left.cumsum(-1)
    goal = u[cu[1:] - 1] * left.sum(-1)
    pick = (c <= goal[:, None]).sum(-1)
    pick = torch.minimum(pick, (torch.arange(v, device=DEVICE) * (left > 0)).amax(-1))
    pick = torch.where(left.sum(-1) > 0, pick, w.argmax(-1))
    after = path.roll(-1, 1)
    after[:, -1] = -1
    out = torch.where(after >= 0, tok.gather(1, after.clamp(min=0)), -1)
    out = torch.where(torch.arange(most, device=DEVICE) == accepted[:, None], pick[:, None], out)
    return out[i, j], accepted.int(), path[i, j].int()


def _plain_move(pools, src, dst, page, table, to, heads=None):
    """Rows `src` [K] of sequences `seq` [K] to `dst`; heads [K]: of one kv head each."""
    (seq, a), b = src, dst
    from_b, from_r = table.long()[seq, a // page], a % page
    to_b, to_r = to.long()[seq, b // page], b % page
    for pool in pools:
        for x in _bytes_of(pool):
            for p in (0, 1):
                if heads is None:
                    x[p][to_b, :, to_r] = x[p][from_b, :, from_r]
                else:
                    x[p][to_b, heads, to_r] = x[p][from_b, heads, from_r]


def _plain_commit(s):
    i, j = _owner(s["cu"], s["total"])
    live = (j < s["count"].long()[i]).nonzero()[:, 0]
    i, j = i[live], j[live]
    first = s["lens"].long()[i]
    _plain_move(s["pools"], (i, first + s["path"].long()[live]), first + j, s["case"]["page"],
                s["table"], s["table"])
    return [x for pool in s["pools"] for x in _bytes_of(pool)]


def _plain_weigh(s):
    i, j, q = _padded(s)
    at, most, count = _key_index(s), s["max_new"], s["cu"].diff().long()
    node = torch.arange(most, device=DEVICE)[None, :, None]
    show = (at[:, None] <= node) & (at < count[:, None])[:, None]
    o, w = _plain_attention(s, q, show)
    w = w.mul_((node[:, :, 0] < count[:, None])[:, None, None, :, None]).sum((2, 3))
    s["mass"].copy_(s["before"])
    b, hkv, keys = w.shape
    page = s["mass"].shape[2]
    live = (at < count[:, None]).nonzero()
    seq, key = live[:, 0], live[:, 1]
    blk, row = s["table"].long()[seq, key // page], key % page
    old = torch.where((at[seq, key] < 0)[:, None], s["mass"][blk, :, row], 0.0)
    s["mass"][blk, :, row] = old + w[seq, :, key]
    return o[i, j].to(s["q"].dtype), s["mass"]


def _plain_evict(s):
    case, lens, page = s["case"], s["lens"].long(), s["mass"].shape[2]
    budget, n = case["budget"], s["lens"].shape[0]
    m = s["mass"][s["table"].long()].transpose(1, 2).reshape(n, case["kv_heads"], -1)
    key = torch.arange(m.shape[-1], device=DEVICE)
    inside = key < lens[:, None]
    always = (key < case["sinks"]) | (key >= (lens - case["recent"])[:, None])
    m = torch.where(always[:, None], math.inf, m)
    m = torch.where(inside[:, None], m, -math.inf)
    # of equal ones the lowest; then in the order in which they are cached
    k = min(budget, m.shape[-1])
    best = m.sort(dim=-1, descending=True, stable=True).indices[:, :, :k]
    best = torch.where(inside.gather(1, best.flatten(1)).view(best.shape), best, 1 << 30)
    best = best.sort(-1).values
    keep = torch.full((n, case["kv_heads"], budget), -1, dtype=torch.int32, device=DEVICE)
    keep[:, :, :k] = torch.where(best < (1 << 30), best, -1).int()
    kept = lens.clamp(max=budget)
    seq, head, at = (keep >= 0).nonzero().unbind(1)
    src = keep.long()[seq, head, at]
    _plain_move(s["pools"], (seq, src), at, page, s["table"], s["to"], head)
    s["mass"][s["to"].long()[seq, at // page], head, at % page] = (
        s["mass"][s["table"].long()[seq, src // page], head, src % page])
    return keep, kept.int(), *_evicted(s)


def _evicted(s):
    a, b = s["fresh"]
    return [x[:, a:b] for x in _bytes_of(s["pools"][0])] + [s["mass"][a:b]]


def _pool(pool):
    from needle_amd import ops
    return pool if torch.is_tensor(pool) else ops.Fp8KVCache(*pool)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"plan": _plain_plan, "tree": _plain_tree, "verify": _plain_verify,
                "commit": _plain_commit, "weigh": _plain_weigh, "evict": _plain_evict}[kind](s)
    from needle_amd import ops
    heads = (case["heads"], case["kv_heads"], case["head_dim"])
    if kind == "plan":
        return ops.tree_mask(s["parents"], s["cu"], s["max_new"])
    if kind == "tree":
        return ops.tree_attention(s["q"], _pool(s["pools"][0]), s["table"], s["cu"], s["lens"],
                                  s["mask"], s["max_new"], s["scale"], *heads,
                                  max_context_len=s["max_ctx"])
    if kind == "verify":
        return ops.verify_tree(s["logits"], s["ids"], s["parents"], s["cu"], s["uniforms"],
                               temperature=s["temperature"])
    if kind == "commit":
        ops.kv_compact([_pool(p) for p in s["pools"]], s["table"], s["path"], s["count"],
                       first=s["lens"], cu_seqlens=s["cu"])
        return [x for pool in s["pools"] for x in _bytes_of(pool)]
    if kind == "weigh":
        s["mass"].copy_(s["before"])
        cu = None if s["max_new"] == 1 else s["cu"]
        out = ops.attention_mass(s["q"], s["pools"][0], s["table"], s["lens"], s["mass"],
                                 s["scale"], *heads, cu_seqlens=cu, max_seqlen=s["max_new"],
                                 max_context_len=s["max_ctx"])
        return out, s["mass"]
    keep, kept = ops.kv_select(s["mass"], s["table"], s["lens"], case["budget"],
                               sinks=case["sinks"], recent=case["recent"])
    ops.kv_compact([_pool(p) for p in s["pools"]], s["table"], keep, kept, dst_table=s["to"],
                   mass=s["mass"])
    return keep, kept, *_evicted(s)


# ---------------------------------------------------------------------------- exact values

def _two(e):
    """2^e in float64, exactly, of whole numbers e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rows(pool, p, head, blk, row):
    """K or V of one kv head at (block, row), in float64."""
    if torch.is_tensor(pool):
        return pool[p, blk, head, row].double()
    b = pool[0].view(torch.uint8)[p, blk, head, row].long()
    m, ex = (b & 7).double(), (b >> 3) & 15
    mag = torch.where(ex > 0, (8 + m) * _two(ex - 10), m * 2.0 ** -9)
    mag = torch.where(b & 128 > 0, -mag, mag)
    return mag * _two(pool[1][p, blk, head, row].long() - 127).unsqueeze(-1)


def _exact_commit(s):
    lens, cu, count = s["lens"].tolist(), s["cu"].tolist(), s["count"].tolist()
    for pool in s["pools"]:
        for x in _bytes_of(pool):
            for i, (c, k) in enumerate(zip(lens, count)):
                t = s["table"][i].tolist()
                page = x.shape[3]
                src = [c + a for a in s["path"][cu[i]:cu[i] + k].tolist()]
                at = lambda p: (t[p // page], slice(None), p % page)  # noqa: E731
                rows = [x[(slice(None), *at(a))].clone() for a in src]
                for j, row in enumerate(rows):
                    if src[j] != c + j:
                        x[(slice(None), *at(c + j))] = row
    return [x.double() for x in s["pools"]]


def _exact_evict(s):
    case, page = s["case"], s["mass"].shape[2]
    mass = s["mass"].cpu().numpy()
    parts = [s["pools"][0], s["mass"]] if torch.is_tensor(s["pools"][0]) else [s["mass"]]
    out = [x.double() for x in parts]
    for i, n in enumerate(s["lens"].tolist()):
        t, to = s["table"][i].tolist(), s["to"][i].tolist()
        at = np.arange(n)
        blk, row = np.array(t)[at // page], at % page
        for head in range(case["kv_heads"]):
            src = at
            if n > case["budget"]:
                m = mass[blk, head, row].astype(np.float64)
                m[:case["sinks"]] = np.inf
                m[n - case["recent"]:] = np.inf
                src = np.sort(np.lexsort((at, -m))[:case["budget"]])
            dst = np.arange(len(src))
            move = [torch.from_numpy(x).to(DEVICE) for x in
                    (blk[src], row[src], np.array(to)[dst // page], dst % page)]
            for x, y in zip(parts, out):
                if x.dim() == 5:
                    y[:, move[2], head, move[3]] = x[:, move[0], head, move[1]].double()
                else:
                    y[move[2], head, move[3]] = x[move[0], head, move[1]].double()
    a, b = s["fresh"]
    if len(out) == 1:
        return None, None, None, None, out[0][a:b]
    return None, None, out[0][:, a:b], out[1][a:b]


@torch.no_grad()
def exact(case, seed):
    if case["kind"] in ("plan", "verify") or (case["kind"] == "commit" and case["fp8"]):
        return None   # whole numbers (codes and scale bytes too)
    s = prepare(case, seed)
    if case["kind"] == "commit":
        return _exact_commit(s)
    if case["kind"] == "evict":
        return _exact_evict(s)
    ctx, new = _lengths(case)
    page, table = case["page"], s["table"].long()
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    g = h // hkv
    trees = _trees(case) if case["kind"] == "tree" else None
    out = torch.empty(sum(new), h, d, dtype=torch.float64, device=DEVICE)
    mass = s["before"].double() if case["kind"] == "weigh" else None
    at = 0
    for i, (c, n) in enumerate(zip(ctx, new)):
        pos = torch.arange(c + n, device=DEVICE)
        blk, row = table[i][pos // page], pos % page
        hide = torch.ones(n, c + n, dtype=torch.bool, device=DEVICE)
        hide[:, :c] = False
        if trees:
            hide[:, c:] = ~torch.from_numpy(_sees(trees[i])).to(DEVICE)
        else:
            hide[:, c:] = torch.ones(n, n, dtype=torch.bool, device=DEVICE).triu(1)
        for kv in range(hkv):
            keys = _exact_rows(s["pools"][0], 0, kv, blk, row)
            values = _exact_rows(s["pools"][0], 1, kv, blk, row)
            q = s["q"][at:at + n, kv * g:(kv + 1) * g].double().reshape(n * g, d)
            w = torch.mm(q, keys.t().contiguous()) / math.sqrt(d)
            w = w.masked_fill(hide.repeat_interleave(g, 0), -math.inf)
            w = torch.softmax(w, dim=-1)
            out[at:at + n, kv * g:(kv + 1) * g] = torch.mm(w, values).view(n, g, d)
            if mass is not None:
                mass[blk[c:], kv, row[c:]] = 0.0
                mass[blk, kv, row] += w.sum(0)
        at += n
    return out if mass is None else (out, mass)


# ---------------------------------------------------------------------------- work

def work(case):
    ctx, new = _lengths(case)
    kind, total, n = case["kind"], sum(new), len(new)
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "plan":
        words = (max(new) + 63) // 64
        # a word with a node's own bit and its parent's word
        return {"bytes": total * (4 + 8 * words + 4), "flops": total * words}
    if kind == "verify":
        e = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": total * (case["vocab"] * e + 8 + 4 + 4 + 8 + 4),
                "flops": 4 * total * case["vocab"]}
    row = 2 * hkv * (d + 1 if case["fp8"] else 2 * d)       # the cache's bytes per token
    if kind == "commit":
        # about half of a path of half the most moves
        moved = sum(min(m, 8) for m in new) * 0.25
        return {"bytes": case["layers"] * moved * 2 * row + 4 * total, "flops": 0}
    if kind == "evict":
        kept = sum(min(c, case["budget"]) for c in ctx)
        return {"bytes": 4 * hkv * sum(ctx) + kept * (2 * row + 4 * hkv + 8 * hkv),
                "flops": hkv * sum(ctx)}
    if kind == "tree":
        pairs = sum(c * m + int(_sees(p).sum()) for c, m, p in zip(ctx, new, _trees(case)))
        extra = 8 * total * ((max(new) + 63) // 64)
    else:
        pairs = sum(c * m + m * (m + 1) // 2 for c, m in zip(ctx, new))
        extra = 8 * hkv * sum(c + m for c, m in zip(ctx, new))
    pages = sum(-(-(c + m) // case["page"]) for c, m in zip(ctx, new))
    return {"bytes": sum(c + m for c, m in zip(ctx, new)) * row + total * h * d * 4 + 4 * pages
            + extra, "flops": 4 * h * d * pairs}
