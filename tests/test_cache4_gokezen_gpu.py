"""Gokezen, whose windowed attention sits beside a matrix memory, with its keys and values held in 4 bits: engines against the plain
implementation with keys and values taken to what the cache would hold."""
import numpy as np
import pytest
import torch

import engine_replay as replay
import gokezen_configs as gc
import plain_cache4
import plain_gokezen as plain
from burn_transformers_b200 import Engine, StepEntry
from burn_transformers_b200.models.gokezen import attention_head_size

LENGTHS = [1, 5, 50, 51, 64, 140, 333]
# the library's keys and values are off by some 10^-6 of a group's largest number, which is 7 codes: nearer to the border between two codes, or two
# scales, than this it may take the other
SURE = 3e-5
TOL = 1e-4          # of a position's largest logit, 32-bit, as in test_gokezen_gpu.py


def held_with_margin(x, size):
    """[T, heads, dim] as heads of `size` channels (the rest zeros) hold it, and per token the distance in codes to the nearest border."""
    wide = np.zeros((*x.shape[:2], size))
    wide[..., :x.shape[2]] = x
    y = plain_cache4.held(wide)
    groups = wide.reshape(*wide.shape[:2], -1, plain_cache4.GROUP)
    top = np.abs(groups).max(-1)
    s = plain_cache4.SCALES[np.searchsorted(7.0 * plain_cache4.SCALES, top)]
    between = np.abs(np.abs(groups / s[..., None]) % 1.0 - 0.5).min((1, 2, 3))
    scales = np.where(top[..., None] > 0, np.abs(top[..., None] / (7.0 * plain_cache4.SCALES) - 1.0), 1.0)
    return y[..., :x.shape[2]], np.minimum(between, 7.0 * scales.min((1, 2, 3)))


def reference(config, weights, seqs, monkeypatch):
    """Logits per sequence, and per position whether no code before it lies next to a border."""
    margins = []

    def attention(h, w, prefix, c):
        T = h.shape[0]
        H, G, dim, vdim = c["heads"], c["kv_heads"], c["dim"], c["vdim"]
        size = attention_head_size(dim, vdim)
        q = (h @ w[prefix + "q"].T).reshape(T, H, dim)
        k, near_k = held_with_margin((h @ w[prefix + "k"].T).reshape(T, G, dim), size)
        v, near_v = held_with_margin((h @ w[prefix + "v"].T).reshape(T, G, vdim), size)
        margins[-1] = np.minimum(margins[-1], np.minimum(near_k, near_v))
        wide = np.zeros((T, H, size)), np.zeros((T, G, size)), np.zeros((T, G, size))
        wide[0][..., :dim], wide[1][..., :dim], wide[2][..., :vdim] = q, k, v
        y = plain_cache4.attention(*wide, 0, c["scale"], c["mask"]["size"])[0][..., :vdim]
        return y.reshape(T, H * vdim) @ w[prefix + "o"].T

    logits = []
    with monkeypatch.context() as patch:
        patch.setattr(plain, "window_attention", attention)
        for seq in seqs:
            margins.append(np.full(len(seq), np.inf))
            logits.append(plain.forward(config, weights, seq))
    return logits, [np.minimum.accumulate(m) >= SURE for m in margins]


def in_portions(engine, seqs, size):
    got = {}
    for r, seq in enumerate(seqs):
        slot = engine.new_sequence()
        for lo in range(0, len(seq), size):
            piece = seq[lo:lo + size]
            for i, row in enumerate(engine.step([StepEntry(slot, piece, list(range(len(piece))))]).detach().cpu().double().numpy()):
                got[(r, lo + i)] = row
        engine.release(slot)
    return got


def case(tmp_path, config, seed=21):
    folder = gc.make_folder(tmp_path, config, seed=seed)
    return folder, *gc.load_plain(folder), gc.prompts(config, LENGTHS, seed=2)


@pytest.mark.gpu
@pytest.mark.parametrize("positions, ring", [(400, False), (900, True)])
@pytest.mark.parametrize("schedule", ["whole", "tail", "portions"])
def test_an_engine_in_32_bits(tmp_path, monkeypatch, schedule, positions, ring):
    folder, config, weights, seqs = case(tmp_path, dict(gc.ONLY_LEFT, max_positions=positions))
    ref, sure = reference(config, weights, seqs, monkeypatch)
    engine = Engine.from_folder(folder, "float32", max_tokens=64 * 16, max_context=positions, cache_bits=4)
    assert [(g.k.dtype, g.is_ring) for g in engine.cache.groups] == [(torch.uint8, ring)]
    # (15 tokens: what any cache of a window of 50 takes behind others)
    got = {"whole": lambda: replay.whole(engine, seqs), "tail": lambda: replay.tail_one_by_one(engine, seqs, tail=70),
           "portions": lambda: in_portions(engine, seqs, 15)}[schedule]()
    engine.check_kernels()
    engine.cache.check()
    assert len(got) == sum(LENGTHS)
    for (r, p), row in got.items():
        assert np.isfinite(row).all()
        if sure[r][p]:
            assert np.abs(row - ref[r][p]).max() / np.abs(ref[r]).max() < TOL, (r, p)


def test_most_positions_are_looked_at(tmp_path, monkeypatch):
    _, config, weights, seqs = case(tmp_path, gc.ONLY_LEFT)
    _, sure = reference(config, weights, seqs, monkeypatch)
    assert sum(s.sum() for s in sure) > 0.6 * sum(LENGTHS)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("config", [gc.ONLY_LEFT, gc.ODD], ids=["one layer", "two windows"])
def test_recorded_steps_are_the_same(tmp_path, dtype, config):
    folder, _, _, _ = case(tmp_path, config)
    seqs = gc.prompts(config, [3, 70, 140], seed=5)
    seen = []
    for graphs in (True, False):
        engine = Engine.from_folder(folder, dtype, max_tokens=64 * 16, cache_bits=4)
        engine.use_graphs = graphs
        logits = []
        for _ in range(3):                       # (a shape that comes again is recorded)
            slots = [engine.new_sequence() for _ in seqs]
            logits.append(engine.step([StepEntry(s, t, [len(t) - 1]) for s, t in zip(slots, seqs)]).clone())
            for step in range(20):
                logits.append(engine.step([StepEntry(s, [(11 * step + i) % config["vocab"]], [0]) for i, s in enumerate(slots)]).clone())
            for s in slots:
                engine.release(s)
        engine.check_kernels()
        seen.append(torch.stack(logits))
    assert bool(torch.isfinite(seen[0]).all())
    assert torch.equal(seen[0], seen[1])
    assert torch.equal(seen[0][:21], seen[0][21:42]) and torch.equal(seen[0][:21], seen[0][42:])
