"""The measured work of the 8-bit KV cache and of speculative verification.

Kinds of case (field "kind"):
  cache   new tokens are rotated, quantised and written into the paged pool of e4m3 codes
          (ops.kv_append_fp8), and the sequences are read back in the model's format
          (ops.kv_read_fp8): every token, or the `tail` last ones of each sequence.
  decode  attention of one token per sequence over the 8-bit pool (ops.paged_decode_fp8).
  chunk   attention of a chunk of new tokens per sequence, causal, over the 8-bit pool that
          holds the cached tokens and the chunk's (ops.varlen_prefill_fp8).
  verify  drafted tokens against the target's logits (ops.verify_drafts).

A row of K or V (one token, one head) is stored as e4m3 codes and one byte s: the values are
code * 2^(s - 127), with the smallest power of two that keeps the row's largest within 448.

Lengths belong to the case (field "lens"), values and block tables to the seed.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROPE_THETA = 1000000.0
E4M3_MAX = 448.0

# heads, kv heads, head_dim
QWEN_05B = (14, 2, 64)
QWEN_7B = (28, 4, 128)
LLAMA_8B = (32, 8, 128)

SHAPES = (QWEN_05B, QWEN_7B, LLAMA_8B, (32, 32, 128), (4, 1, 128), (7, 1, 64), (12, 4, 64))
VOCABS = (151936, 128256, 32000, 50257, 4099)


def _attn(name, kind, shape, **more):
    h, hkv, d = shape
    c = {"name": name, "kind": kind, "heads": h, "kv_heads": hkv, "head_dim": d, "dtype": "bf16",
         "page": 16, "lens": 3, "new_lo": 1, "new_hi": 1}
    c.update(more)
    return c


def listed():
    return [
        # a decode step of a small batch: one token per sequence, the last page read back
        _attn("cache-step", "cache", QWEN_05B, seqs=8, lo=32, hi=512, tail=16),
        # the prompts of a prefill, written whole and read back for attention in 16 bits
        _attn("cache-prompts", "cache", QWEN_7B, seqs=16, lo=0, hi=0, new_lo=128, new_hi=2048,
              tail=0, lens=5),
        # chunks after cached prefixes, larger pages, an fp16 model: prefixes and chunks read back
        _attn("cache-prefix-fp16", "cache", LLAMA_8B, seqs=24, lo=256, hi=4096, new_lo=1,
              new_hi=301, tail=0, dtype="fp16", page=64, lens=7),
        # a decode step of a small model and batch: latency
        _attn("decode-small", "decode", QWEN_05B, seqs=8, lo=32, hi=512),
        # an ordinary decode step
        _attn("decode-batch", "decode", LLAMA_8B, seqs=64, lo=512, hi=4096, lens=4),
        # few long contexts, an fp16 model with larger pages
        _attn("decode-long-fp16", "decode", QWEN_7B, seqs=24, lo=4096, hi=32768, dtype="fp16",
              page=64, lens=9),
        # a verification step of a small batch: four drafts and the last token
        _attn("chunk-small", "chunk", QWEN_05B, seqs=4, lo=64, hi=800, new_lo=5, new_hi=5),
        # a verification step of a batch, drafts of uneven lengths
        _attn("chunk-drafts", "chunk", LLAMA_8B, seqs=64, lo=512, hi=4096, new_lo=1, new_hi=8,
              lens=6),
        # prompts continued after cached prefixes
        _attn("chunk-prompts", "chunk", QWEN_7B, seqs=4, lo=2048, hi=8192, new_lo=500,
              new_hi=1100, lens=11),
        # one sequence, four drafts of a lookup (no draft distribution): latency
        {"name": "verify-one", "kind": "verify", "seqs": 1, "new_lo": 5, "new_hi": 5,
         "vocab": 151936, "dtype": "bf16", "probs": False, "greedy": 0, "lens": 1},
        # a batch with a draft model's distributions, some sequences greedy
        {"name": "verify-batch", "kind": "verify", "seqs": 64, "new_lo": 1, "new_hi": 8,
         "vocab": 151936, "dtype": "bf16", "probs": True, "greedy": 4, "lens": 2},
        # float32 logits of an odd vocabulary
        {"name": "verify-fp32-odd", "kind": "verify", "seqs": 96, "new_lo": 2, "new_hi": 6,
         "vocab": 50257, "dtype": "fp32", "probs": True, "greedy": 0, "lens": 8},
    ]


def _between(rng, lo, hi):
    """Spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("cache", "decode", "chunk", "verify"))
    lens = rng.randrange(1 << 20)
    if kind == "verify":
        most = rng.randint(2, 8)
        vocab = rng.choice(VOCABS)
        return {"kind": kind, "seqs": min(_between(rng, 1, 200), 500 // most),
                "new_lo": rng.randint(1, most),
                "new_hi": most, "vocab": vocab, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                "probs": rng.random() < 0.6, "greedy": rng.choice((0, 0, 3)), "lens": lens}
    shape = rng.choice(SHAPES)
    more = {"dtype": rng.choice(("bf16", "fp16")), "page": rng.choice((16, 16, 32, 64, 256)),
            "lens": lens}
    if kind == "cache":
        seqs, hi = _between(rng, 1, 64), _between(rng, 20, 4096)
        new_hi = max(1, min(_between(rng, 1, 2048), 60000 // (shape[1] * seqs)))
        more.update(seqs=seqs, lo=rng.choice((0, hi // 8)), hi=min(hi, 360000 // (shape[1] * seqs)),
                    new_lo=rng.randint(1, new_hi),
                    new_hi=new_hi, tail=rng.choice((0, 0, 16)))
    elif kind == "decode":
        seqs = _between(rng, 1, 128)
        hi = max(1, min(_between(rng, 32, 32768), 1200000 // (shape[1] * seqs)))
        more.update(seqs=seqs, lo=max(1, hi // rng.choice((2, 8))), hi=hi)
    elif rng.random() < 0.6:   # drafts
        seqs = _between(rng, 1, 96)
        hi = max(1, min(_between(rng, 32, 16384), 1000000 // (shape[1] * seqs)))
        more.update(seqs=seqs, lo=max(1, hi // 8), hi=hi, new_lo=rng.randint(1, 4),
                    new_hi=rng.randint(4, 16))
    else:                      # prompts after a prefix
        seqs = rng.randint(1, 4)
        new_hi = _between(rng, 24, 600)
        more.update(seqs=seqs, lo=rng.choice((0, 100)), hi=_between(rng, 200, 5000),
                    new_lo=max(1, new_hi // 3), new_hi=new_hi)
    c = _attn("", kind, shape, **more)
    c["lo"] = min(c["lo"], c["hi"])
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs

def _lengths(case):
    """(cached tokens, new tokens) of every sequence."""
    r = np.random.default_rng(case["lens"])
    n = r.integers(case["new_lo"], case["new_hi"], size=case["seqs"], endpoint=True).tolist()
    if case["kind"] == "verify":
        return [0] * len(n), n
    lo, hi = case["lo"], case["hi"]
    c = np.exp(r.uniform(math.log(lo + 1), math.log(hi + 2), case["seqs"])).astype(np.int64) - 1
    return np.clip(c, lo, hi).tolist(), n


def _power(byte):
    """2^(byte - 127) in float32, exactly; byte from 1 to 254."""
    return (byte.int() << 23).view(torch.float32)


def _quantise(x):
    """Codes and scale bytes of the rows of x (finite), in torch operations."""
    m, ex = torch.frexp(x.float().abs().amax(-1))
    byte = (ex + 118 + (m > E4M3_MAX / 512)).clamp_(min=1)
    codes = (x.float() * _power(254 - byte).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes, byte.to(torch.uint8)


def _values(codes, scales):
    """What codes [.., D] and scales [..] stand for, in float32."""
    return codes.float() * _power(scales).unsqueeze(-1)


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    ctx, new = _lengths(case)
    total, n = sum(new), len(new)
    cu = np.concatenate([[0], np.cumsum(new)])
    s = {"case": case, "max_new": max(new), "cu": _i32(cu)}

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)

    if case["kind"] == "verify":
        v = case["vocab"]
        # a peaked distribution over a long tail; the draft model's is near the target's
        logits = randn(total, v).mul_(2.2)
        s["logits"] = logits.to(dtype)
        temp = torch.rand(n, generator=gen, device=DEVICE).mul_(0.7).add_(0.5)
        if case["greedy"]:
            temp[::case["greedy"]] = 0.0
        s["temperature"] = temp
        rows = torch.tensor([r for i in range(n) for r in range(cu[i], cu[i + 1] - 1)],
                            dtype=torch.long, device=DEVICE)
        seq = torch.repeat_interleave(torch.arange(n, device=DEVICE), s["cu"].diff().long())
        s["ids"] = torch.randint(0, v, (total,), generator=gen, device=DEVICE)
        s["probs"] = None
        if rows.numel():
            near = logits[rows].add_(randn(rows.numel(), v).mul_(0.4))
            near.div_(temp[seq[rows]].clamp(min=0.2).unsqueeze(1))
            draft = torch.softmax(near, dim=-1)
            del near
            x = torch.multinomial(draft, 1, generator=gen)[:, 0]
            best = s["logits"][rows].float().argmax(-1)
            if not case["probs"]:   # a lookup's drafts: often what the target would say
                x = torch.where(torch.rand(rows.numel(), generator=gen, device=DEVICE) < 0.8,
                                best, x)
            x = torch.where(temp[seq[rows]] == 0, torch.where(x % 5 == 0, x, best), x)
            s["ids"][rows + 1] = x
            if case["probs"]:
                s["probs"] = draft
        elif case["probs"]:
            s["probs"] = torch.empty(0, v, device=DEVICE)
        s["uniforms"] = torch.rand(total, generator=gen, device=DEVICE)
        return s

    h, hkv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    blocks = [-(-(c + m) // page) for c, m in zip(ctx, new)]
    num_blocks = sum(blocks) + 2
    perm = np.random.default_rng(seed).permutation(num_blocks - 1)
    table = np.full((n, max(blocks)), num_blocks - 1, dtype=np.int32)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = perm[at:at + b]
        at += b
    s.update(table=_i32(table), lens=_i32(ctx), max_ctx=max(ctx), scale=1.0 / math.sqrt(d))
    # what the pool holds: keys with a few channels far larger than the rest
    codes = torch.empty(2, num_blocks, hkv, page, d, dtype=torch.float8_e4m3fn, device=DEVICE)
    scales = torch.empty(2, num_blocks, hkv, page, dtype=torch.uint8, device=DEVICE)
    gain = torch.ones(d, device=DEVICE)
    gain[3::29] = 4.0
    step = max(1, (1 << 26) // (hkv * page * d))
    for b in range(0, num_blocks, step):
        e = min(num_blocks, b + step)
        for p, g in ((0, gain), (1, 1.0)):
            codes[p, b:e], scales[p, b:e] = _quantise(
                (randn(e - b, hkv, page, d) * g).to(dtype))
    s["codes"], s["scales"] = codes, scales
    # the projections' outputs: views of one fused q/k/v row per token
    qkv = randn(total, (h + 2 * hkv) * d).to(dtype)
    q, k, v = qkv.split([h * d, hkv * d, hkv * d], dim=-1)
    s["q"], s["k"], s["v"] = q.view(total, h, d), k.view(total, hkv, d), v.view(total, hkv, d)
    if case["kind"] == "cache":
        pos = torch.tensor(np.concatenate([np.arange(c, c + m) for c, m in zip(ctx, new)]),
                           device=DEVICE)
        inv = 1.0 / (ROPE_THETA ** (torch.arange(0, d, 2, device=DEVICE).double() / d))
        angle = torch.outer(pos.double(), inv)
        angle = torch.cat([angle, angle], dim=-1)
        s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
        first, count = _read_range(case)
        s["first"], s["read"] = _i32(first), sum(count)
        s["read_cu"] = _i32(np.concatenate([[0], np.cumsum(count)]))
    return s


def _read_range(case):
    """(first position, tokens) read back of every sequence."""
    ctx, new = _lengths(case)
    count = [min(c + m, case["tail"] or c + m) for c, m in zip(ctx, new)]
    return [c + m - k for c, m, k in zip(ctx, new, count)], count


# ---------------------------------------------------------------------------- plain forms

def _owner(cu, total):
    """(sequence, offset in it) of each of `total` packed tokens."""
    t = torch.arange(total, device=DEVICE)
    i = torch.searchsorted(cu[1:].long(), t, right=True)
    return i, t - cu.long()[i]


def _slots(s, i, p):
    """(block, row) of position p of sequence i."""
    page, width = s["codes"].shape[3], s["table"].shape[1]
    return s["table"].long()[i, (p // page).clamp(max=width - 1)], p % page


def _rotate(x, cos, sin):
    """The model's rotary embedding: each product and the sum rounded to the model's format."""
    dt, half = x.dtype, x.shape[-1] // 2
    r = torch.cat([-x[..., half:], x[..., :half]], dim=-1)
    a = (x.float() * cos.float().unsqueeze(1)).to(dt)
    b = (r.float() * sin.float().unsqueeze(1)).to(dt)
    return (a.float() + b.float()).to(dt)


def _plain_cache(s):
    q, k = _rotate(s["q"], s["cos"], s["sin"]), _rotate(s["k"], s["cos"], s["sin"])
    i, j = _owner(s["cu"], k.shape[0])
    blk, row = _slots(s, i, s["lens"].long()[i] + j)
    kc, ks = _quantise(k)
    vc, vs = _quantise(s["v"])
    codes = s["codes"].view(torch.uint8)
    codes[0, blk, :, row], codes[1, blk, :, row] = kc.view(torch.uint8), vc.view(torch.uint8)
    s["scales"][0, blk, :, row], s["scales"][1, blk, :, row] = ks, vs
    i, j = _owner(s["read_cu"], s["read"])
    blk, row = _slots(s, i, s["first"].long()[i] + j)
    got = _values(codes[:, blk, :, row].view(torch.float8_e4m3fn), s["scales"][:, blk, :, row])
    got = got.to(s["k"].dtype)   # [R, 2, Hkv, D]
    return q, got[:, 0].contiguous(), got[:, 1].contiguous()


def _plain_attention(s, q, last):
    """q [B, N, H, D] in float32, token (b, n) over positions up to last[b, n]."""
    b, n, h, d = q.shape
    page, width, hkv = s["codes"].shape[3], s["table"].shape[1], s["codes"].shape[2]
    t = s["table"].long()
    keys = torch.arange(width * page, device=DEVICE)
    # [B, W, Hkv, page, D] -> [B, Hkv, W * page, D]
    def plane(p):
        x = _values(s["codes"].view(torch.uint8)[p][t].view(torch.float8_e4m3fn),
                    s["scales"][p][t])
        return x.transpose(1, 2).reshape(b, hkv, width * page, d)
    k = plane(0)
    qg = q.view(b, n, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    w = torch.matmul(qg, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    del k
    hide = keys > last[:, None, None, :, None]                   # [B, 1, 1, N, keys]
    w = w.view(b, hkv, h // hkv, n, -1).masked_fill_(hide, -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True)).exp_()
    w = w.div_(w.sum(-1, keepdim=True))
    v = plane(1).masked_fill_((keys > last.amax(1)[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(w.view(b, hkv, -1, width * page), v)
    return o.view(b, hkv, h // hkv, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)


def _plain_chunk(s):
    q, most = s["q"], s["max_new"]
    i, j = _owner(s["cu"], q.shape[0])
    padded = torch.zeros(s["lens"].shape[0], most, *q.shape[1:], device=DEVICE)
    padded[i, j] = q.float()
    last = s["lens"].long()[:, None] + torch.arange(most, device=DEVICE)
    last = torch.minimum(last, s["lens"].long()[:, None] + s["cu"].diff().long()[:, None] - 1)
    return _plain_attention(s, padded, last)[i, j].to(q.dtype)


def _plain_verify(s):
    cu, ids, u, logits = s["cu"].long(), s["ids"], s["uniforms"].double(), s["logits"]
    total, v = logits.shape
    n = cu.shape[0] - 1
    i, j = _owner(cu, total)
    count = cu.diff()
    # the target's distributions
    temp = s["temperature"].double()[i]
    z = logits.double()
    top, best = z.max(-1)
    p = z.sub_(top[:, None]).div_(torch.where(temp > 0, temp, 1.0)[:, None]).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    point = (torch.arange(v, device=DEVICE) == best[:, None]).double()
    p = torch.where((temp > 0)[:, None], p, point)
    # drafts that are accepted: those before a sequence's first rejected one
    drafted = j + 1 < count[i]
    x = torch.where(drafted, ids.roll(-1), 0)
    at = torch.where(drafted, torch.arange(total, device=DEVICE) - i, 0)   # draft row
    qx = s["probs"].double()[at, x] if s["probs"] is not None and s["probs"].shape[0] else 1.0
    ok = drafted & (u * qx < p.gather(1, x[:, None])[:, 0])
    most = s["max_new"]
    grid = torch.zeros(n, most, dtype=torch.long, device=DEVICE)
    grid[i, j] = ok.long()
    accepted = grid.cumprod(1).sum(1)
    # the token after them
    row = cu[:-1] + accepted
    w, rejected = p[row], accepted + 1 < count
    xr = torch.where(rejected, ids[(row + 1).clamp(max=total - 1)], 0)
    if s["probs"] is not None and s["probs"].shape[0]:
        q = s["probs"].double()[torch.where(rejected, row - torch.arange(n, device=DEVICE), 0)]
    else:
        q = (torch.arange(v, device=DEVICE) == xr[:, None]).double()
    left = torch.where(rejected[:, None], (w - q).clamp_(min=0.0), w)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
    c = left.cumsum(-1)
    goal = u[cu[1:] - 1] * left.sum(-1)
    pick = (c <= goal[:, None]).sum(-1)
    last = (torch.arange(v, device=DEVICE) * (left > 0)).amax(-1)
    pick = torch.minimum(pick, last)
    tokens = torch.where(j < accepted[i], ids.roll(-1), -1)
    tokens = torch.where(j == accepted[i], pick[i], tokens)
    return tokens, accepted.int()


def run(s):
    kind = s["case"]["kind"]
    if own:
        from needle_amd import ops
        case = s["case"]
        if kind == "verify":
            return ops.verify_drafts(s["logits"], s["ids"], s["cu"], s["uniforms"],
                                     temperature=s["temperature"], draft_probs=s["probs"])
        if kind == "cache":
            q = ops.kv_append_fp8(s["k"], s["v"], s["codes"], s["scales"], s["table"], s["lens"],
                                  s["cu"], q=s["q"], cos=s["cos"], sin=s["sin"])
            k, v = ops.kv_read_fp8(s["codes"], s["scales"], s["table"], s["first"],
                                   s["read_cu"], s["read"], dtype=s["k"].dtype)
            return q, k, v
        heads = (s["scale"], case["heads"], case["kv_heads"], case["head_dim"])
        if kind == "decode":
            return ops.paged_decode_fp8(s["q"], s["codes"], s["scales"], s["table"], s["lens"],
                                        *heads)
        return ops.varlen_prefill_fp8(s["q"], s["codes"], s["scales"], s["table"], s["cu"],
                                      s["lens"], s["max_new"], *heads,
                                      max_context_len=s["max_ctx"])
    if kind == "verify":
        return _plain_verify(s)
    if kind == "cache":
        return _plain_cache(s)
    if kind == "decode":
        last = s["lens"].long()[:, None]
        return _plain_attention(s, s["q"].float().unsqueeze(1), last)[:, 0].to(s["q"].dtype)
    return _plain_chunk(s)


# ---------------------------------------------------------------------------- exact values

def _two(e):
    """2^e in float64, exactly, of whole numbers e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rows(x):
    """The values that quantised rows of x (float64) stand for."""
    a = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(a.clamp(min=2.0 ** -126) / E4M3_MAX))
    e = torch.where(a <= E4M3_MAX * _two(e - 1), e - 1, e)
    e = torch.where(a > E4M3_MAX * _two(e), e + 1, e).clamp(min=-126.0)
    y = x / _two(e)
    # three bits after the leading one, steps of 2^-9 below 2^-6
    size = y.abs().clamp(min=2.0 ** -6)
    lead = torch.floor(torch.log2(size))
    lead = torch.where(_two(lead) > size, lead - 1, lead)
    lead = torch.where(_two(lead + 1) <= size, lead + 1, lead)
    return torch.round(y / _two(lead - 3)) * _two(lead - 3) * _two(e)


def _exact_values(codes, scales):
    b = codes.view(torch.uint8).long()
    m, ex = (b & 7).double(), (b >> 3) & 15
    mag = torch.where(ex > 0, (8 + m) * _two(ex - 10), m * 2.0 ** -9)
    mag = torch.where(b & 128 > 0, -mag, mag)
    return mag * _two(scales.long() - 127).unsqueeze(-1)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    if case["kind"] == "verify":
        return None   # whole numbers
    page, table = case["page"], s["table"].long()
    dt = s["q"].dtype

    def rows(i, first, count):
        p = torch.arange(first, first + count, device=DEVICE)
        return table[i][p // page], p % page

    if case["kind"] == "cache":
        # the rotation's roundings are part of its definition
        def rope(x):
            half = x.shape[-1] // 2
            turned = torch.cat([x[..., half:].neg(), x[..., :half]], dim=-1).double()
            a = x.double() * s["cos"].double()[:, None]
            b = turned * s["sin"].double()[:, None]
            return (a.to(dt).double() + b.to(dt).double()).to(dt).double()
        k, v = _exact_rows(rope(s["k"])), _exact_rows(s["v"].double())
        first, count = _read_range(case)
        out, at = [], 0
        for i, (c, n) in enumerate(zip(ctx, new)):
            blk, row = rows(i, first[i], max(0, c - first[i]))
            old = _exact_values(s["codes"].view(torch.uint8)[:, blk, :, row],
                                s["scales"][:, blk, :, row])
            fresh = torch.stack([k[at:at + n], v[at:at + n]], dim=1)
            out.append(torch.cat([old, fresh[max(0, first[i] - c):]]))
            at += n
        out = torch.cat(out)
        return rope(s["q"]), out[:, 0].contiguous(), out[:, 1].contiguous()
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.empty(sum(new), h, d, dtype=torch.float64, device=DEVICE)
    at = 0
    for i, (c, n) in enumerate(zip(ctx, new)):
        blk, row = rows(i, 0, c + n)
        kv = _exact_values(s["codes"].view(torch.uint8)[:, blk, :, row],
                           s["scales"][:, blk, :, row])
        far = torch.arange(c + n, device=DEVICE) - torch.arange(c, c + n, device=DEVICE)[:, None]
        for head in range(h):
            keys = kv[:, 0, head // (h // hkv)].contiguous()
            values = kv[:, 1, head // (h // hkv)].contiguous()
            w = torch.mm(s["q"][at:at + n, head].double(), keys.t()) / math.sqrt(d)
            w = torch.softmax(w.masked_fill(far > 0, -math.inf), dim=-1)
            out[at:at + n, head] = torch.mm(w, values)
        at += n
    return out


# ---------------------------------------------------------------------------- work

def work(case):
    ctx, new = _lengths(case)
    total = sum(new)
    if case["kind"] == "verify":
        e = 4 if case["dtype"] == "fp32" else 2
        # every logit, and of the drafts' distributions the rejected row and the drafts' own
        return {"bytes": total * case["vocab"] * e
                + (case["seqs"] * case["vocab"] * 4 if case["probs"] else 0) + 20 * total,
                "flops": 4 * total * case["vocab"]}
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    row = 2 * hkv * (d + 1)                      # the cache's bytes per token
    if case["kind"] == "cache":
        read = sum(_read_range(case)[1])
        return {"bytes": total * (2 * (h + 2 * hkv) * d + 4 * d + 2 * h * d + row)
                + read * (row + 4 * hkv * d), "flops": total * (3 * (h + hkv) + 2 * hkv) * d}
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    pages = sum(-(-(c + n) // case["page"]) for c, n in zip(ctx, new))
    return {"bytes": sum(c + n for c, n in zip(ctx, new)) * row + total * h * d * 4 + 4 * pages,
            "flops": 4 * h * d * pairs}
