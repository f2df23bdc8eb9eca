"""The 4-bit cache as a model uses it: an attention layer with normed and turned heads over prompts, portions and single tokens, whole
engines that hold their cache in 4 bits, and the calls of a decode step recorded together and replayed."""
import numpy as np
import pytest
import torch

import burn_transformers_b200 as bt
import plain_cache4 as plain
from burn_transformers_b200 import kernels
from burn_transformers_b200.cache import CacheBank, CacheConfig, CacheNeed, KvSpec
from burn_transformers_b200.engine import StepBuilder, StepEntry
from burn_transformers_b200.parts import CausalSelfAttention, HalfSplitRotary, InterleavedRotary
from burn_transformers_b200.weights import MATRIX, random_tensors
from burn_transformers_b200.weights.spec import WeightPlan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def host(t):
    return t.detach().double().cpu().numpy()


def bound(part, dtype):
    plan = WeightPlan(dict(part.specs()))
    tensors = random_tensors(plan, 3, storage="bfloat16" if dtype == torch.bfloat16 else "float32", loud=True)
    keep = {n: (t.to(dtype) if plan.tensors[n].kind == MATRIX else t.float()).to(DEV) for n, t in tensors.items()}
    part.bind(keep)
    return {n: host(t) for n, t in keep.items()}


# of the layer's result, against 64 bits from the layer's own inputs and the keys and values that its cache holds
TOL = {torch.float32: 1e-5, torch.bfloat16: 1.5e-2}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads, kv, dim, rotary, window, keep", [
    (4, 2, 64, HalfSplitRotary(64, 10000.0), None, 0), (8, 1, 32, InterleavedRotary(16, 500.0), 90, 3),
    (2, 2, 128, HalfSplitRotary(64, 10000.0, yarn=(4.0, 64.0, 8.0, 1.0)), 150, 0), (3, 3, 96, None, None, 0)])
def test_a_layer_over_prompts_portions_and_single_tokens(dtype, heads, kv, dim, rotary, window, keep):
    width = 192
    part = CausalSelfAttention(width, heads, kv, dim, dim ** -0.5, positions=rotary, qk_norm_eps=1e-5, cache_bits=4, window=window, keep_first=keep)
    w = bound(part, dtype)
    cache = CacheBank([part.cache_need()], CacheConfig(64 * 40, 8, 640), dtype, DEV)
    builder = StepBuilder(cache, dtype, DEV)
    slots = [cache.acquire() for _ in range(3)]
    gen = torch.Generator(device=DEV).manual_seed(1)
    for news in ([200, 1, 70], [1, 1, 1], [33, 150, 2], [1, 1, 1]):
        pasts = [cache.length(s) for s in slots]
        cache.reserve([(s, p + n) for s, p, n in zip(slots, pasts, news)])
        ctx = builder.build([StepEntry(s, [0] * n, []) for s, n in zip(slots, news)])
        x = torch.randn(sum(news), width, generator=gen, device=DEV).to(dtype)
        residual = torch.randn(sum(news), width, generator=gen, device=DEV)
        before = host(residual)
        builder.ws.reset()
        part.forward(ctx, x, residual, 0)
        kernels.check_status(torch.device(DEV))
        proj = host(x) @ w["qkv.weight"] + w["qkv.bias"]
        pool, _, group, g = cache.layer_pools(0)
        row = 0
        for i, (past, new) in enumerate(zip(pasts, news)):
            total = past + new
            at = torch.arange(total, dtype=torch.int32, device=DEV)
            got_k, got_v = (torch.empty(total, kv, dim, device=DEV) for _ in range(2))
            kernels.cache4_gather(pool, at, torch.full_like(at, i), ctx.tables[g], group.table_len, got_k, got_v, n_tokens=total)
            q, k, v = np.split(proj[row:row + new], [heads * dim, (heads + kv) * dim], axis=1)
            freq = np.zeros(1) if rotary is None else np.array(rotary.frequencies())
            rot, near, size = (0, False, 1.0) if rotary is None else (rotary.dims, rotary.neighbours, rotary.size)
            turn = lambda t, n, name: plain.norm_rotary(t.reshape(new, n, dim), past + np.arange(new), freq[:rot // 2], rot,      # noqa: E731
                                                        w[name], 1e-5, near, size)[0]
            q, k = turn(q, heads, "q_norm.weight"), turn(k, kv, "k_norm.weight")
            # what the cache holds is within half a step of what went there, and a step is at most 9/8 of a group's largest number over 7
            for held, want in ((host(got_k)[past:], k), (host(got_v)[past:], v.reshape(new, kv, dim))):
                top = np.abs(want.reshape(new, kv, -1, 32)).max(-1, keepdims=True)
                off = np.abs(held - want).reshape(new, kv, -1, 32) / top
                assert off.max() < 9 / 8 / 7 / 2 + 2.0 ** -6
            y = plain.attention(q, host(got_k), host(got_v), past, dim ** -0.5, window or 0, keep)[0].reshape(new, -1)
            want = before[row:row + new] + y @ w["out.weight"] + w["out.bias"]
            got = host(residual[row:row + new])
            assert np.abs(got - want).max() / np.abs(want).max() < TOL[dtype], (news, i)
            row += new
        for s, p, n in zip(slots, pasts, news):
            cache.commit(s, p + n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rotary", [HalfSplitRotary(48, 10000.0), InterleavedRotary(32, 10000.0, yarn=(4.0, 64.0, 8.0, 1.0))])
def test_rotations_of_a_step_without_norms(dtype, rotary):
    heads, kv, dim, n = 3, 1, 64, 70
    part = CausalSelfAttention(64, heads, kv, dim, 0.125, positions=rotary)
    bound(part, dtype)
    cache = CacheBank([part.cache_need()], CacheConfig(64 * 8, 2, 256), dtype, DEV)
    slot = cache.acquire()
    cache.reserve([(slot, n)])
    ctx = StepBuilder(cache, dtype, DEV).build([StepEntry(slot, [0] * n, [])])
    proj = torch.randn(n, (heads + 2 * kv) * dim, device=DEV).to(dtype)
    x = host(proj)[:, :(heads + kv) * dim].reshape(n, heads + kv, dim)
    rotary.rotate(ctx, proj, heads, kv, dim)
    y, mass = plain.norm_rotary(x, np.arange(n), host(rotary.inv_freq(DEV)), rotary.dims, interleaved=rotary.neighbours, size=rotary.size)
    got = host(proj)[:, :(heads + kv) * dim].reshape(x.shape)
    assert (np.abs(got - y) <= 64 * 2.0 ** -24 * mass + torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -7) * np.abs(y)).all()


def folder(tmp_path, heads):
    return bt.write_random_model(str(tmp_path / "m"), dict(model_type="gpt2", n_layer=3, n_embd=128, n_head=heads, vocab_size=257, n_positions=512),
                                 seed=5, storage="bfloat16", loud=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads", [2, 4])
def test_an_engine_that_holds_its_cache_in_4_bits(tmp_path, dtype, heads):
    path = folder(tmp_path, heads)
    prompts = [list(range(1, 90)), [5, 6, 7], list(range(40, 170))]
    seen = []
    for graphs in (True, False):
        engine = bt.Engine.from_folder(path, dtype, max_tokens=64 * 24, cache_bits=4)
        assert all(g.k.dtype == torch.uint8 for g in engine.cache.groups)
        engine.use_graphs = graphs
        slots = [engine.new_sequence() for _ in prompts]
        logits = [engine.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)]).clone()]
        for step in range(70):                                   # (across the end of a page)
            logits.append(engine.step([StepEntry(s, [(7 * step + s) % 257], [0]) for s in slots]).clone())
        for _ in range(3):                                       # (a shape that comes again is recorded and replayed)
            logits.append(engine.step([StepEntry(s, [3, 1, 4, 1, 5], [4]) for s in slots]).clone())
        engine.check_kernels()
        seen.append(torch.stack(logits))
    assert bool(torch.isfinite(seen[0]).all())
    assert torch.equal(seen[0], seen[1])


def test_generation_with_a_cache_in_4_bits(tmp_path):
    path = folder(tmp_path, 2)
    loaded = bt.AutoCausalLm.load_local(path, bt.AutoLoadOptions(dtype="bfloat16", max_tokens=64 * 8, cache_bits=4))
    request = bt.CausalGenerationRequest([[1, 2, 3], [4, 5]], bt.GenerationConfig(max_new_tokens=80))
    first = [s.token_ids for s in bt.generate_causal(loaded.model, request).sequences]
    assert [len(t) for t in first] == [80, 80]
    assert first == [s.token_ids for s in bt.generate_causal(loaded.model, request).sequences]
    with pytest.raises(bt.CacheError, match="not of 16"):
        bt.Engine.from_folder(folder(tmp_path / "narrow", 8) if (tmp_path / "narrow").mkdir() is None else "", "bfloat16", cache_bits=4)


@pytest.mark.parametrize("heads, kv, dim", [(4, 4, 64), (16, 2, 128)])
def test_the_calls_of_a_step_recorded_together_and_replayed(heads, kv, dim):
    """Two recordings with scratch of their own, replayed in turn on two streams, against the same calls one by one."""
    seqs, width, dtype = 3, 40, torch.bfloat16
    rng = np.random.default_rng(2)
    freq = torch.tensor(10000.0 ** (-2.0 * np.arange(dim // 2) / dim), dtype=torch.float32, device=DEV)
    weight = torch.tensor(1 + 0.1 * rng.standard_normal(dim), dtype=torch.float32, device=DEV)
    sizes = dict(n_tokens=seqs, n_seqs=seqs, max_new=1, max_ctx=width * 64, n_heads=heads, n_kv_heads=kv, head_dim=dim)
    start = [700, 63, 2000]

    def one(lane):
        s = dict(proj=torch.empty(seqs, (heads + 2 * kv) * dim, dtype=dtype, device=DEV), out=torch.empty(seqs, heads * dim, dtype=dtype, device=DEV),
                 table=torch.tensor(np.random.default_rng(lane).permutation(seqs * width).reshape(seqs, width), dtype=torch.int32, device=DEV),
                 past=torch.tensor(start, dtype=torch.int32, device=DEV), starts=torch.arange(seqs + 1, dtype=torch.int32, device=DEV),
                 which=torch.arange(seqs, dtype=torch.int32, device=DEV),
                 scratch=torch.empty(kernels.cache4_attention_scratch_floats(**sizes), device=DEV))
        gen = torch.Generator(device=DEV).manual_seed(lane)
        pool = torch.randint(0, 256, (seqs * width, kv, 68 * dim), dtype=torch.uint8, generator=gen, device=DEV)
        pool[:, :, 64 * dim:].clamp_(100, 160)                   # scales of ordinary size
        s["pool"] = pool
        s["inputs"] = [torch.randn(s["proj"].shape, generator=gen, device=DEV).to(dtype) for _ in range(6)]
        return s

    def calls(s):
        kernels.qk_norm_rotary(s["proj"], s["past"], freq, n_tokens=seqs, n_heads=heads, n_kv_heads=kv, head_dim=dim, rot_dims=dim, q_weight=weight,
                               k_weight=weight, eps=1e-6)
        k = s["proj"][:, heads * dim:(heads + kv) * dim].view(seqs, kv, dim)
        v = s["proj"][:, (heads + kv) * dim:].view(seqs, kv, dim)
        length = s["past"] + 1
        kernels.cache4_append(k, v, s["pool"], s["past"], s["which"], length, s["table"], width, n_tokens=seqs)
        kernels.cache4_attention(s["proj"], s["out"], s["pool"], s["table"], width, s["starts"], s["past"], scale=dim ** -0.5, scratch=s["scratch"], **sizes)
        s["past"] += 1

    def run(s, step):
        results = []
        for x in s["inputs"]:
            s["proj"].copy_(x)
            step(s)
            results.append(s["out"].clone())
        return torch.stack(results)

    want = [run(one(lane), calls) for lane in (1, 2)]
    lanes = [one(lane) for lane in (1, 2)]
    graphs = []
    for s in lanes:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            calls(s)
        graphs.append(graph)
        s["past"].copy_(torch.tensor(start, dtype=torch.int32))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lanes]
    got = [[], []]
    for i in range(6):
        for s, graph, stream, results in zip(lanes, graphs, streams, got):
            with torch.cuda.stream(stream):
                s["proj"].copy_(s["inputs"][i])
                graph.replay()
                results.append(s["out"].clone())
    torch.cuda.synchronize()
    kernels.check_status(torch.device(DEV))
    for lane in range(2):
        assert torch.equal(torch.stack(got[lane]), want[lane])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads, kv, dim, window", [(4, 2, 64, 100), (2, 2, 128, 150), (8, 1, 32, 64), (3, 3, 96, 1)])
def test_a_layer_over_a_ring_and_over_every_position(dtype, heads, kv, dim, window):
    """Prompts longer than the ring, single tokens across its turns, and the longest portions that it takes: the same bits as over a cache
    that keeps every position."""
    width, longest = 96, 64 * 40
    part = CausalSelfAttention(width, heads, kv, dim, dim ** -0.5, cache_bits=4, window=window)
    bound(part, dtype)
    caches = [CacheBank([need], CacheConfig(64 * 100, 4, longest), dtype, DEV) for need in (part.cache_need(), CacheNeed(kv=KvSpec(kv, dim, bits=4)))]
    ring = caches[0].groups[0]
    assert ring.is_ring and not caches[1].groups[0].is_ring
    run = caches[0].max_continued_run
    builders = [StepBuilder(cache, dtype, DEV) for cache in caches]
    slots = [[cache.acquire() for _ in range(3)] for cache in caches]
    gen = torch.Generator(device=DEV).manual_seed(1)
    for news in [[400, 1, 200]] + [[1, 1, 1]] * 3 + [[run, 1, min(run, 2)]] * 4 + [[1, 1, 1]] * 70 + [[min(run, 5), run, run]] * 3:
        x = torch.randn(sum(news), width, generator=gen, device=DEV).to(dtype)
        residual = torch.randn(sum(news), width, generator=gen, device=DEV)
        results = []
        for cache, builder, ids in zip(caches, builders, slots):
            cache.reserve([(s, cache.length(s) + n) for s, n in zip(ids, news)])
            ctx = builder.build([StepEntry(s, [0] * n, []) for s, n in zip(ids, news)])
            out = residual.clone()
            builder.ws.reset()
            part.forward(ctx, x, out, 0)
            results.append(out)
            for s, n in zip(ids, news):
                cache.commit(s, cache.length(s) + n)
        kernels.check_status(torch.device(DEV))
        assert bool(torch.isfinite(results[0]).all()) and torch.equal(*results), news
