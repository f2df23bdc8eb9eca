"""What holds its keys and values in 4 bits, and what refuses to, without a device."""
import random

import pytest
import torch

import gokezen_configs
from burn_transformers_b200.cache import CacheBank, CacheConfig, CacheNeed, KvSpec
from burn_transformers_b200.config import Gpt2Config
from burn_transformers_b200.config.gokezen import GokezenConfig
from burn_transformers_b200.engine import StepBuilder, StepEntry
from burn_transformers_b200.errors import CacheError, ShapeError
from burn_transformers_b200.models.gokezen import build_gokezen
from burn_transformers_b200.models.gpt2 import build_gpt2
from burn_transformers_b200.parts import CausalSelfAttention, attention


def test_a_group_in_4_bits_is_one_pool_of_bytes():
    needs = [CacheNeed(kv=KvSpec(2, 64)), CacheNeed(kv=KvSpec(2, 64, bits=4)), CacheNeed(kv=KvSpec(2, 64, bits=4))]
    bank = CacheBank(needs, CacheConfig(64 * 6, 3, 64 * 5), torch.bfloat16, "cpu")
    plain, packed = bank.groups
    assert plain.k.dtype == torch.bfloat16 and packed.k.dtype == torch.uint8
    assert list(packed.k.shape) == [2, 6, 2, 68 * 64] and packed.v.numel() == 0
    assert packed.k[0].nbytes * 256 == (plain.k[0].nbytes + plain.v[0].nbytes) * 68
    slot = bank.acquire()
    bank.reserve([(slot, 130)])
    assert len(bank.table_row(1, slot)) == 3
    bank.check()


@pytest.mark.parametrize("spec", [dict(head_dim=48, bits=4), dict(head_dim=288, bits=4), dict(head_dim=64, bits=8),
                                  dict(head_dim=64, bits=4, has_values=False)])
def test_specs_that_are_refused(spec):
    with pytest.raises(ValueError):
        KvSpec(2, **spec)


def test_a_plan_holds_its_softmax_attention_in_4_bits():
    config = dict(model_type="gpt2", n_layer=3, n_embd=128, n_head=2, vocab_size=64, n_positions=128)
    plan = build_gpt2(Gpt2Config.from_dict(config))
    assert all(need.kv.bits is None for need in plan.cache_needs())
    plan.hold_cache_in(4)
    assert [need.kv for need in plan.cache_needs()] == [KvSpec(2, 64, bits=4)] * 3
    with pytest.raises(CacheError, match="not in 8"):
        plan.hold_cache_in(8)
    odd = build_gpt2(Gpt2Config.from_dict(dict(config, n_head=8)))
    with pytest.raises(CacheError, match="multiple of 32 channels, not of 16"):
        odd.hold_cache_in(4)


def test_a_model_without_softmax_attention_refuses(monkeypatch):
    plan = build_gpt2(Gpt2Config.from_dict(dict(model_type="gpt2", n_layer=1, n_embd=128, n_head=2, vocab_size=64, n_positions=128)))
    monkeypatch.setattr(plan, "all_parts", lambda: [plan.embedding, plan.final_norm])
    with pytest.raises(CacheError, match="fewer bits"):
        plan.hold_cache_in(4)


@pytest.mark.parametrize("kw, words", [(dict(keep_first=2), "kept positions"), (dict(keep_first=2, window=8), "kept positions"),
                                       (dict(keep_first=-1), "kept positions"), (dict(cache_bits=3), "not in 3"),
                                       (dict(cache_bits=4, causal=False), "causal")])
def test_an_attention_that_is_refused(kw, words):
    with pytest.raises(ShapeError, match=words):
        CausalSelfAttention(128, 2, 2, 64, 0.125, **kw)


def test_norms_of_heads_are_tensors_of_the_part():
    part = CausalSelfAttention(128, 4, 2, 32, 0.125, qk_norm_eps=1e-6, cache_bits=4, window=100, keep_first=4)
    assert part.specs()["q_norm.weight"].shape == (32,) and part.specs()["k_norm.weight"].shape == (32,)
    assert part.cache_need().kv == KvSpec(2, 32, bits=4)


def gokezen_plan(config):
    return build_gokezen(GokezenConfig.from_dict(config))


@pytest.mark.parametrize("config", [gokezen_configs.ONLY_LEFT, gokezen_configs.ODD])
def test_mixers_side_by_side_hold_their_cache_in_4_bits(config):
    plan = gokezen_plan(config)
    before = plan.cache_needs()
    plan.hold_cache_in(4)
    for need, was in zip(plan.cache_needs(), before):
        assert need.kv.bits == 4 and (need.kv.n_kv_heads, need.kv.head_dim) == (was.kv.n_kv_heads, was.kv.head_dim)
        assert need.states == was.states
    bank = CacheBank(plan.cache_needs(), CacheConfig(64 * 8, 2, 200), torch.bfloat16, "cpu")
    assert all(g.k.dtype == torch.uint8 for g in bank.groups)


@pytest.mark.parametrize("bits, config, words", [(4, gokezen_configs.MIXED, "not of 16"), (8, gokezen_configs.ONLY_LEFT, "not in 8")])
def test_a_plan_that_is_refused_stays_as_it_was(bits, config, words):
    plan = gokezen_plan(config)
    before = plan.cache_needs()
    with pytest.raises(CacheError, match=words):
        plan.hold_cache_in(bits)
    assert plan.cache_needs() == before


@pytest.fixture
def asked(monkeypatch):
    """The sizes that a layer hands to the attention over its 4-bit cache; nothing is computed."""
    calls = []
    monkeypatch.setattr(attention.kernels, "cache4_append", lambda *args, **kw: None)
    monkeypatch.setattr(attention.kernels, "cache4_attention_scratch_floats", lambda **kw: 0)
    monkeypatch.setattr(attention.kernels, "cache4_attention", lambda *args, **kw: calls.append(kw))
    monkeypatch.setattr(attention, "linear", lambda *args, **kw: None)
    return calls


def steps_of(part, runs, max_context=640, max_tokens=64 * 20):
    """Has `part` take steps of new tokens a sequence, (3, 1) for two sequences, one after another."""
    part.t_qkv_weight = part.t_qkv_bias = part.t_out_weight = part.t_out_bias = None
    part.nk_qkv_weight = part.nk_out_weight = False
    cache = CacheBank([part.cache_need()], CacheConfig(max_tokens, 4, max_context), torch.bfloat16, "cpu")
    builder = StepBuilder(cache, torch.bfloat16, "cpu")
    slots = [cache.acquire() for _ in runs[0]]
    for news in runs:
        cache.reserve([(s, cache.length(s) + n) for s, n in zip(slots, news)])
        ctx = builder.build([StepEntry(s, [0] * n, []) for s, n in zip(slots, news)])
        builder.ws.reset()
        part.forward(ctx, torch.zeros(sum(news), part.width), torch.zeros(sum(news), part.width), 0)
        for s, n in zip(slots, news):
            cache.commit(s, cache.length(s) + n)
    return cache


def test_prompts_without_a_past_are_planned_as_such(asked):
    """Steps whose sequences all begin are bounded by their own tokens; others by the cache's longest sequence, as recorded ones are."""
    steps_of(CausalSelfAttention(128, 2, 2, 64, 0.125, cache_bits=4), [(200, 33), (1, 1), (7, 2)])
    assert [(kw["max_new"], kw["max_ctx"]) for kw in asked] == [(200, 200), (1, 640), (7, 640)]


def windowed(window, keep=0, dim=64):
    return CausalSelfAttention(128, 2, 2, dim, 0.125, cache_bits=4, window=window, keep_first=keep)


def nbytes(bank):
    return sum(g.k.nbytes + g.v.nbytes for g in bank.groups)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window, context", [(1, 64), (50, 400), (64, 4096), (130, 640), (512, 1900), (512, 4096), (512, 16_384), (5000, 4096)])
@pytest.mark.parametrize("slots, tokens", [(1, 64), (3, 1000), (8, 4096), (64, 4096), (7, 100_000)])
def test_a_window_in_4_bits_takes_no_more_than_in_the_model_type(dtype, window, context, slots, tokens):
    """Neither bytes nor, for any lengths of the sequences, room."""
    config = CacheConfig(tokens, slots, context)
    part = windowed(window)
    assert part.cache_need().kv.window == window
    plain = CacheBank([CacheNeed(kv=KvSpec(2, 64, window))], config, dtype, "cpu")
    packed = CacheBank([part.cache_need()], config, dtype, "cpu")
    assert nbytes(packed) <= nbytes(plain)
    assert packed.groups[0].k.dtype == torch.uint8 and (packed.groups[0].is_ring or packed.groups[0].whole)
    if packed.groups[0].is_ring:
        assert packed.max_continued_run == plain.max_continued_run and nbytes(packed) * 2 * plain.groups[0].k.element_size() * 64 == nbytes(plain) * 68
    rng = random.Random(window + slots)
    for _ in range(20):
        wanted = [rng.choice((1, 64, rng.randint(1, context), context)) for _ in range(slots)]
        held = []
        for bank in (plain, packed):
            slot_ids, room = [bank.acquire() for _ in wanted], 0
            for slot, length in zip(slot_ids, wanted):
                try:
                    bank.reserve([(slot, length)])
                    room += 1
                except CacheError:
                    break
            bank.check()
            for slot in slot_ids:
                bank.release(slot)
            held.append(room)
        assert held[1] >= held[0]


def test_kept_positions_need_every_page():
    bank = CacheBank([windowed(50, 4).cache_need()], CacheConfig(4096, 2, 4096), torch.bfloat16, "cpu")
    assert not bank.groups[0].is_ring and bank.max_continued_run is None


def test_a_prompt_longer_than_the_ring_attends_over_pages_of_its_step(asked, monkeypatch):
    filed, read = [], []
    monkeypatch.setattr(attention.kernels, "cache4_append", lambda k, v, pool, *args, **kw: filed.append((pool, args[3], args[4])))
    monkeypatch.setattr(attention.kernels, "cache4_attention",
                        lambda q, out, pool, table, table_len, *args, **kw: read.append((pool, table.clone(), table_len, kw["max_ctx"])))
    news = (200, 1, 65, 64)
    cache = steps_of(windowed(100), [news, (1, 1, 1, 1), (29, 2, 1, 3)], max_context=4096)
    ring = cache.groups[0]
    assert ring.is_ring and ring.table_len == 2 and cache.max_continued_run == 29
    # the prompts: filed in the ring and in the step's own pages, read from those
    assert len(filed) == 4 and [f[0].data_ptr() == ring.k[0].data_ptr() for f in filed] == [True, False, True, True]
    pool, table, table_len, bound = read[0]
    assert pool.data_ptr() == filed[1][0].data_ptr() and (table_len, bound) == (4, 200) and pool.shape[1:] == (2, 68 * 64)
    pages = [table[i, :-(-n // 64)].tolist() for i, n in enumerate(news)]
    flat = sum(pages, [])
    assert len(set(flat)) == len(flat) and min(flat) >= 0 and max(flat) < pool.shape[0]
    # and later steps from the ring
    assert [(r[0].data_ptr() == ring.k[0].data_ptr(), r[2], r[3]) for r in read[1:]] == [(True, 2, 4096)] * 2


@pytest.mark.parametrize("seed", range(4))
def test_pages_of_a_step_for_any_lengths(asked, monkeypatch, seed):
    read = []
    monkeypatch.setattr(attention.kernels, "cache4_attention", lambda q, out, pool, table, *args, **kw: read.append((pool, table.clone())))
    rng = random.Random(seed)
    for _ in range(20):
        news = tuple(rng.choice((1, 63, 64, 65, 128, rng.randint(1, 500))) for _ in range(4)) [:rng.randint(1, 4)] + (200,)
        steps_of(windowed(100), [news[-4:]], max_context=4096)
        pool, table = read.pop()
        flat = sum((table[i, :-(-n // 64)].tolist() for i, n in enumerate(news[-4:])), [])
        assert len(set(flat)) == len(flat) and min(flat) >= 0 and max(flat) < pool.shape[0]


def test_a_run_that_the_ring_does_not_hold_is_refused(asked):
    with pytest.raises(CacheError, match="ring"):
        steps_of(windowed(100), [(5, 200), (30, 1)], max_context=4096)
