"""The 8-bit pool under the layer, the runner and the engine, and its operators together as a
speculative decoder uses them: the bytes of every pool and every verified token as defined, the
attention within the bound of test_gpu_fp8_attention."""
import numpy as np
import pytest
import torch

from needle_amd import ops
from needle_amd.backend.engine import LLMEngine
from needle_amd.backend.request import SamplingParams, SeqState
from needle_amd.layers.attention import Attention
from needle_amd.layers.rope import RotaryEmbedding
from needle_amd.model.config import ModelConfig
from needle_amd.model.qwen2 import build_model, random_init_
from needle_amd.model.runner import ModelRunner
from oracle import fp8_ref, paged_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

TOY = dict(model_type="qwen2", hidden_size=256, num_hidden_layers=3, num_attention_heads=4,
           num_key_value_heads=2, intermediate_size=512, vocab_size=1000,
           max_position_embeddings=2048, rms_norm_eps=1e-6, rope_theta=1e6)


def _close(got, attended, dtype, d):
    """Within the attention's bound (the module docstring of test_gpu_fp8_attention)."""
    out, weight, big, n = attended
    got = got.double().cpu().view(out.shape)
    rel = 2 * (d + 8) * 2.0 ** -24 * big[..., None] + 2.0 ** -20 + n[:, None, None] * 2.0 ** -23
    bound = torch.finfo(dtype).eps / 2 * (weight + out.abs()) + rel * weight
    if dtype == torch.float16:
        # a probability below 2^-14 is off by 2^-25 where the largest is at least 1
        bound = bound + n[:, None, None] * 2.0 ** -25 * 32
    assert ((got - out).abs() <= bound).all()


@pytest.mark.parametrize("fuse_rope", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,d,bs", [(14, 2, 64, 16), (8, 2, 128, 32)])
@torch.no_grad()
def test_layer(h, hkv, d, bs, dtype, fuse_rope):
    """A prefill, a chunk after it and two decode steps of one layer."""
    torch.manual_seed(1)
    cfg = ModelConfig(hidden_size=h * d, num_attention_heads=h, num_key_value_heads=hkv,
                      max_position_embeddings=512)
    layer = Attention(cfg, 0, qkv_bias=True)
    for p in layer.parameters():
        torch.nn.init.normal_(p, std=0.05)
    layer = layer.to(dtype).to(DEV)
    layer.fuse_rope = fuse_rope
    seen = {}
    for name in ("q_proj", "k_proj", "v_proj"):
        getattr(layer, name).register_forward_hook(
            lambda _m, _i, out, name=name: seen.__setitem__(name, out.clone()))
    layer.o_proj.register_forward_pre_hook(lambda _m, i: seen.__setitem__("attended", i[0].clone()))
    rope = RotaryEmbedding(d, 512, 1e4).to(dtype)

    nb = 20
    table = torch.randperm(nb, generator=torch.Generator().manual_seed(2))[:18]
    table = table.to(torch.int32).view(3, 6)
    pool = ops.fp8_kv_pool(nb, hkv, bs, d, device=DEV)
    codes, scales = pool.codes.view(torch.uint8).cpu(), pool.scales.cpu()
    assert not codes.any() and not fp8_ref.values(codes, scales).any()
    cur = [0, 0, 0]
    for counts, prefill in (([37, 5, 18], True), ([3, 9, 1], True), ([1] * 3, False),
                            ([1] * 3, False)):
        x = torch.randn(sum(counts), h * d).to(dtype).to(DEV)
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cur, counts)])
        cos, sin = rope.get_cos_sin(pos)
        cu = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32)
        ctx = torch.tensor(cur, dtype=torch.int32)
        got = layer(x, pos.to(DEV), pool, table.to(DEV), cu.to(DEV), ctx.to(DEV), max(counts),
                    prefill, cos.to(DEV), sin.to(DEV))
        q, k, v = (seen[n].cpu().view(len(pos), -1, d) for n in ("q_proj", "k_proj", "v_proj"))
        q, k = paged_ref.apply_rope(q, k, cos, sin)
        fp8_ref.append(k, v, codes, scales, table, cu, ctx)
        assert torch.equal(pool.codes.view(torch.uint8).cpu(), codes)
        assert torch.equal(pool.scales.cpu(), scales)
        _close(seen["attended"], fp8_ref.attention(q, codes, scales, table, cu, ctx, layer.scale),
               dtype, d)
        assert torch.equal(got, layer.o_proj(seen["attended"]))
        cur = [c + n for c, n in zip(cur, counts)]


@torch.no_grad()
def test_a_swapped_sequence_decodes_exactly_as_an_unswapped_one():
    cfg = ModelConfig(**TOY)
    base = random_init_(build_model(cfg), seed=21)
    runners = []
    for n_cpu in (0, 32):
        model = build_model(cfg)
        model.load_state_dict(base.state_dict())
        r = ModelRunner(cfg, device=DEV, model=model, kv_cache_dtype="fp8")
        r.init_kv_cache(64, n_cpu)
        runners.append(r)
    a, b = runners
    prompt = np.random.default_rng(2).integers(0, cfg.vocab_size, 50).tolist()
    sa, sb = (SeqState(1, n, prompt, SamplingParams(temperature=0.0)) for n in "ab")
    sa.blocks, sb.blocks = [0, 1, 2, 3, 4], [10, 11, 12, 13, 14]

    def step(prefill):
        la = a.forward(a.prepare_inputs([sa], is_prefill=prefill))
        lb = b.forward(b.prepare_inputs([sb], is_prefill=prefill))
        assert torch.equal(la.view(torch.int16), lb.view(torch.int16))
        tok = int(la.argmax(-1)[0])
        sa.tokens.append(tok)
        sb.tokens.append(tok)

    step(True)
    for _ in range(3):
        step(False)
    cpu_ids, new_ids = [5, 9, 6, 30, 0], [40, 17, 33, 63, 2]
    b.swap(dict(zip(sb.blocks, cpu_ids)), to_cpu=True)
    for codes, scales in b.kv_caches:                  # the GPU copies are gone
        codes.view(torch.uint8)[:, sb.blocks] = 0x55
        scales[:, sb.blocks] = 0x55
    before = [(c.view(torch.uint8).clone(), s.clone()) for c, s in b.kv_caches]
    b.swap(dict(zip(cpu_ids, new_ids)), to_cpu=False)
    torch.cuda.synchronize()
    others = [i for i in range(64) if i not in new_ids]
    for pa, pb, old in zip(a.kv_caches, b.kv_caches, before):
        for x, y, z in zip(pa, pb, old):
            x, y = x.view(torch.uint8), y.view(torch.uint8)
            assert torch.equal(x[:, sa.blocks], y[:, new_ids])
            assert torch.equal(y[:, others], z[:, others])
    sb.blocks = new_ids
    for _ in range(4):
        step(False)


def test_pools_of_both_kinds_are_not_copied():
    a = [ops.fp8_kv_pool(4, 2, 16, 64, device=DEV)]
    b = [torch.zeros(2, 4, 2, 16, 64, dtype=torch.bfloat16, device=DEV)]
    ids = torch.zeros(1, dtype=torch.int32, device=DEV)
    for x, y in ((a, b), (b, a)):
        with pytest.raises(TypeError, match="8-bit pool copies to"):
            ops.kv_block_copy(x, y, ids, ids)


@pytest.mark.parametrize("bs,dtype", [(16, "bfloat16"), (32, "float16")])
@torch.no_grad()
def test_engine(bs, dtype):
    """Requests through graph-replayed decode steps, and with a GPU pool so small that sequences
    are swapped out and in."""
    cfg = ModelConfig(**TOY)
    base = random_init_(build_model(cfg), seed=5).state_dict()
    rng = np.random.default_rng(1)
    reqs = [(f"q{i}", rng.integers(0, cfg.vocab_size, int(rng.integers(1, 90))).tolist(),
             int(rng.integers(1, 40))) for i in range(8)]
    per_block = cfg.num_hidden_layers * 2 * cfg.num_key_value_heads * bs * (cfg.head_dim + 1)

    def run(blocks, graphs, swap=0):
        model = build_model(cfg)
        model.load_state_dict(base)
        eng = LLMEngine(cfg, block_size=bs, max_gpu_blocks=blocks, model=model,
                        decode_graphs=graphs, max_model_len=512, max_num_seqs=8, dtype=dtype,
                        cpu_swap_bytes=swap * per_block, kv_cache_dtype="fp8")
        assert eng.runner.bytes_per_block() == per_block
        assert eng.allocator.num_free_cpu_blocks == swap
        swaps, real = [], eng.runner.swap
        eng.runner.swap = lambda mapping, to_cpu: (swaps.append(len(mapping)),
                                                   real(mapping, to_cpu))
        for name, prompt, n in reqs:
            eng.add_request(name, prompt, SamplingParams(temperature=0.0, max_new_tokens=n))
        got, steps = {}, 0
        while eng.has_unfinished_requests() and steps < 2000:
            got.update(eng.step())
            steps += 1
        assert {k: len(v) for k, v in got.items()} == {name: n for name, _, n in reqs}
        assert eng.allocator.num_free_gpu_blocks == blocks - (1 if graphs else 0)
        assert eng.allocator.num_free_cpu_blocks == swap
        return eng, sum(swaps)

    eng, _ = run(256, True)
    a, b = (eng.generate([5, 6, 7] * 20, SamplingParams(temperature=0.0, max_new_tokens=8), n)
            for n in "ab")
    assert a == b and len(a) == 8
    assert run(320 // bs, False, swap=40)[1] > 0


@torch.no_grad()
def test_graph_replays_are_the_eager_step():
    cfg = ModelConfig(**TOY)
    eng = LLMEngine(cfg, max_gpu_blocks=200, seed=6, decode_graphs=True, max_model_len=512,
                    max_num_seqs=8, kv_cache_dtype="fp8")
    r = eng.runner
    checked = []

    def wrap(bucket, graph, logits):
        class Replay:
            def replay(self):
                rows = r._rows
                n = len(rows.rows)
                ids = torch.tensor([s.last_token for s in rows.rows] + [0] * (bucket - n))
                ctx = torch.tensor([s.length - 1 for s in rows.rows] + [0] * (bucket - n),
                                   dtype=torch.int32, device=DEV)
                table = np.full((bucket, rows.width), rows.scratch, dtype=np.int32)
                for i, s in enumerate(rows.rows):
                    table[i, :len(s.blocks)] = s.blocks
                eager = r.model(ids.to(DEV), ctx.long(), r.kv_caches,
                                torch.from_numpy(table).to(DEV),
                                torch.arange(bucket + 1, dtype=torch.int32, device=DEV), ctx, 1,
                                False)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(eager[:n], logits[:n])
                checked.append(bucket)
        return Replay()

    for bucket, (graph, logits) in list(r._graphs.items()):
        r._graphs[bucket] = (wrap(bucket, graph, logits), logits)
    rng = np.random.default_rng(7)
    for i in range(5):
        eng.add_request(f"r{i}", rng.integers(0, cfg.vocab_size, 30 + 50 * i).tolist(),
                        SamplingParams(temperature=0.0, max_new_tokens=4 + 5 * i))
    while eng.has_unfinished_requests():
        eng.step()
    assert len(checked) > 20 and len(set(checked)) > 1


@pytest.mark.parametrize("temps", [[0.0, 0.0, 0.0], [0.8, 0.0, 1.3]])
@pytest.mark.parametrize("dtype,h,hkv,d", [(torch.bfloat16, 8, 2, 64), (torch.float16, 7, 1, 128)])
def test_speculative_decoding(dtype, h, hkv, d, temps):
    """Drafts decoded on a copy of the pool (some replaced by others), appended, attended as a
    chunk and verified, step after step; what is rejected is overwritten by the next step.  Every
    step's pool, attention and tokens are the definition's.  Then the accepted tokens are decoded
    one by one into another pool, which ends with the same bytes."""
    gen = torch.Generator().manual_seed(3)
    vocab, nb, bs, n = 300, 40, 16, 3
    table = torch.randperm(nb, generator=gen)[:36].to(torch.int32).view(n, 12)
    emb = torch.randn(vocab, (h + 2 * hkv) * d, generator=gen).to(dtype)
    head = (torch.randn(h * d, vocab, generator=gen) * 4 * (h * d) ** -0.5).to(DEV)
    rope = RotaryEmbedding(d, 256, 1e4).to(dtype)
    scale = 2.0 / d ** 0.5
    temperature = torch.tensor(temps)
    pool = ops.fp8_kv_pool(nb, hkv, bs, d, device=DEV)
    codes, scales = pool.codes.view(torch.uint8).cpu(), pool.scales.cpu()
    one_each = torch.arange(n + 1, dtype=torch.int32)

    def attend(pool, ids, pos, cu, ctx, most):
        """The attention's output, the logits, and q, k and v as they are attended."""
        q, k, v = (x.view(len(ids), -1, d) for x in
                   emb[ids].split([h * d, hkv * d, hkv * d], dim=-1))
        cos, sin = rope.get_cos_sin(pos)
        rot = paged_ref.apply_rope(q, k, cos, sin)
        gcu, gctx, gtable = cu.to(DEV), ctx.to(DEV), table.to(DEV)
        gq = ops.kv_append_fp8(k.to(DEV), v.to(DEV), *pool, gtable, gctx,
                               None if most == 1 else gcu, q=q.to(DEV), cos=cos.to(DEV),
                               sin=sin.to(DEV))
        if most == 1:
            out = ops.paged_decode_fp8(gq, *pool, gtable, gctx, scale, h, hkv, d)
        else:
            out = ops.varlen_prefill_fp8(gq, *pool, gtable, gcu, gctx, most, scale, h, hkv, d)
        return out, out.flatten(1).float() @ head, rot[0], rot[1], v

    def draft(ends, at, counts):
        """counts[i] tokens after ends[i], the last token, which is at position at[i]."""
        copy = ops.Fp8KVCache(*(x.clone() for x in pool))
        ids, found = torch.tensor(ends), [[] for _ in range(n)]
        for step in range(max(counts)):
            pos = torch.tensor(at) + step
            _, logits, *_ = attend(copy, ids, pos, one_each, pos.to(torch.int32), 1)
            ids = logits.argmax(-1).cpu()
            swap = torch.rand(n, generator=gen) < 0.25
            ids = torch.where(swap, torch.randint(0, vocab, (n,), generator=gen), ids)
            for i in range(n):
                if step < counts[i]:
                    found[i].append(int(ids[i]))
        return found

    text = [torch.randint(0, vocab, (m,), generator=gen).tolist() for m in (20, 3, 41)]
    done, taken, steps = [0, 0, 0], 0, 0                # done: tokens in the pool
    while min(len(t) for t in text) < 40 and steps < 60:
        steps += 1
        counts = [0] * n if not steps > 1 else torch.randint(0, 5, (n,), generator=gen).tolist()
        drafts = draft([t[-1] for t in text], done, counts) if max(counts) else [[]] * n
        new = [t[c:] + x for t, c, x in zip(text, done, drafts)]
        counts = [len(x) for x in new]
        cu = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32)
        ctx = torch.tensor(done, dtype=torch.int32)
        ids = torch.tensor(sum(new, []))
        pos = torch.cat([torch.arange(c, c + m) for c, m in zip(done, counts)])
        out, logits, q, k, v = attend(pool, ids, pos, cu, ctx, max(counts))
        fp8_ref.append(k, v, codes, scales, table, cu, ctx)
        assert torch.equal(pool.codes.view(torch.uint8).cpu(), codes)
        assert torch.equal(pool.scales.cpu(), scales)
        _close(out, fp8_ref.attention(q, codes, scales, table, cu, ctx, scale), dtype, d)
        # the rows of each sequence's last token and of its drafts
        rows = torch.cat([torch.arange(int(cu[i + 1]) - len(drafts[i]) - 1, int(cu[i + 1]))
                          for i in range(n)])
        vcu = torch.tensor([0] + np.cumsum([len(x) + 1 for x in drafts]).tolist(),
                           dtype=torch.int32)
        vl, u = logits[rows.to(DEV)], torch.rand(len(rows), generator=gen)
        tokens, accepted = ops.verify_drafts(vl, ids[rows].to(DEV), vcu.to(DEV), u.to(DEV),
                                             temperature=temperature.to(DEV))
        assert (tokens.tolist(), accepted.tolist()) == fp8_ref.verify(vl.cpu(), ids[rows], vcu, u,
                                                                      temperature, None)
        for i in range(n):
            keep = int(accepted[i])
            done[i] = len(text[i]) + keep               # the last token is not in the pool yet
            text[i] += tokens[int(vcu[i]):int(vcu[i]) + keep + 1].tolist()
            taken += keep
    assert taken > 10

    other = ops.fp8_kv_pool(nb, hkv, bs, d, device=DEV)
    for p in range(max(done)):
        # a sequence that has ended decodes its last token again, at its own place
        at = [min(p, c - 1) for c in done]
        attend(other, torch.tensor([t[a] for t, a in zip(text, at)]), torch.tensor(at), one_each,
               torch.tensor(at, dtype=torch.int32), 1)
    for i in range(n):
        p = torch.arange(done[i])
        blk, row = table[i][p // bs].long(), p % bs
        for x, y in zip(pool, other):
            x, y = x.view(torch.uint8).cpu(), y.view(torch.uint8).cpu()
            assert torch.equal(x[:, blk, :, row], y[:, blk, :, row])
