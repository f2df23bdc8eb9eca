"""The norms of query and key heads with the rotation in the same pass, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import plain_cache4 as plain
from burn_transformers_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def host(t):
    return t.detach().double().cpu().numpy()


def check(got, x, positions, freq, rot, weights, heads, eps, interleaved, size, dtype):
    dim = x.shape[-1]
    for part, weight in ((slice(0, heads), weights[0]), (slice(heads, None), weights[1])):
        if x[:, part].size == 0:
            continue
        y, mass = plain.norm_rotary(x[:, part], positions, freq, rot, weight, eps, interleaved, size)
        # 32-bit arithmetic (a sum of `dim` squares, a root, an angle within half a turn, four products) and one rounding to the type
        allowed = mass * 2.0 ** -24 * (32 + dim / 2) + torch.finfo(dtype).eps / 2 * np.abs(y) * (1 + 2.0 ** -7) + 1e-40
        far = np.abs(got[:, part] - y) / allowed
        assert far.max() <= 1.0, float(far.max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim, rot", [(128, 128), (64, 32), (80, 80), (80, 48), (256, 256), (16, 16), (48, 0), (7, 4), (100, 50), (192, 64), (250, 250)])
@pytest.mark.parametrize("tokens, heads, kv", [(1, 1, 1), (9, 12, 12), (37, 32, 8), (300, 5, 1)])
def test_against_the_definition(dtype, interleaved, dim, rot, tokens, heads, kv):
    rng = np.random.default_rng(dim * 7 + rot + tokens)
    width = (heads + 2 * kv) * dim
    proj = torch.tensor(2.0 * rng.standard_normal((tokens + 2, width)) * np.exp(2 * rng.standard_normal((tokens + 2, 1)))).to(dtype).to(DEV)
    positions = torch.tensor(rng.choice([0, 1, 63, 1023, 100_003, 2 ** 24 - 1, 2 ** 31 - 1], tokens + 2), dtype=torch.int32, device=DEV)
    freq = torch.tensor(10000.0 ** (-2.0 * np.arange(max(1, rot // 2)) / max(1, rot)), dtype=torch.float32, device=DEV)
    weights = [torch.tensor(1 + 0.3 * rng.standard_normal(dim), dtype=torch.float32, device=DEV) for _ in range(2)]
    x = host(proj)[:tokens, :(heads + kv) * dim].reshape(tokens, heads + kv, dim)
    args = dict(n_tokens=tokens, n_heads=heads, n_kv_heads=kv, head_dim=dim, rot_dims=rot, q_weight=weights[0], k_weight=weights[1], eps=1e-5,
                interleaved=interleaved)
    out = torch.full((tokens + 1, (heads + kv) * dim + 8), 3.0, dtype=dtype, device=DEV)
    kernels.qk_norm_rotary(proj, positions, freq, out=out, **args)
    got = host(out)[:tokens, :(heads + kv) * dim].reshape(x.shape)
    check(got, x, host(positions)[:tokens], host(freq)[:rot // 2], rot, [host(w) for w in weights], heads, 1e-5, interleaved, 1.0, dtype)
    assert bool((out[tokens:] == 3).all()) and bool((out[:, (heads + kv) * dim:] == 3).all())
    before = proj.clone()
    kernels.qk_norm_rotary(proj, positions, freq, **args)
    assert torch.equal(proj[:tokens, :(heads + kv) * dim], out[:tokens, :(heads + kv) * dim])
    assert torch.equal(proj[tokens:], before[tokens:]) and torch.equal(proj[:, (heads + kv) * dim:], before[:, (heads + kv) * dim:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_no_norm_a_sized_turn_and_rows_off_the_16_byte_boundary(dtype, shift):
    rng, tokens, heads, kv, dim = np.random.default_rng(4), 33, 6, 2, 64
    proj = torch.tensor(rng.standard_normal((tokens, 10 * dim + shift))).to(dtype).to(DEV)[:, shift:]
    positions = torch.arange(tokens, dtype=torch.int32, device=DEV) * 31
    freq = torch.tensor(500.0 ** (-np.arange(32) / 32.0), dtype=torch.float32, device=DEV)
    x = host(proj)[:, :8 * dim].reshape(tokens, 8, dim)
    kernels.qk_norm_rotary(proj, positions, freq, n_tokens=tokens, n_heads=heads, n_kv_heads=kv, head_dim=dim, rot_dims=64, size=1.25)
    check(host(proj)[:, :8 * dim].reshape(x.shape), x, host(positions), host(freq), 64, [None, None], heads, 0.0, False, 1.25, dtype)


def test_rows_of_zeros_infinities_and_nan():
    dim = 64
    proj = torch.zeros(4, 2 * dim, device=DEV)
    proj[1, 3], proj[2, 5] = float("inf"), float("nan")
    w = torch.ones(dim, device=DEV)
    positions = torch.zeros(4, dtype=torch.int32, device=DEV)
    kernels.qk_norm_rotary(proj, positions, torch.ones(32, device=DEV), n_tokens=4, n_heads=1, n_kv_heads=1, head_dim=dim, rot_dims=64, q_weight=w,
                           k_weight=w, eps=1e-6)
    assert bool((proj[[0, 3]] == 0).all()) and bool((proj[:, dim:] == 0).all())      # (other heads and rows are not touched)
    assert bool(torch.isnan(proj[1, 3])) and bool(torch.isnan(proj[2, :dim]).all())
