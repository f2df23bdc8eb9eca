"""The 4-bit cache on the device: what it holds after a step, bit for bit, and the attention over it, against the definitions in
64 bits."""
import numpy as np
import pytest
import torch

import plain_cache4 as plain
from burn_transformers_b200 import kernels
from burn_transformers_b200.errors import KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def host(t):
    return t.detach().double().cpu().numpy()


class Step:
    """The integers of a step; pages handed out in a scrambled order, two pages of the pool in nobody's list."""

    def __init__(self, pasts, news, ring=None, seed=7):
        self.pasts, self.news, self.lens = pasts, news, [p + n for p, n in zip(pasts, news)]
        self.width = ring or max(1, -(-max(self.lens) // PAGE))
        self.pages = len(news) * self.width + 2
        order = np.random.default_rng(seed).permutation(self.pages)
        self.lists = order[:len(news) * self.width].reshape(len(news), self.width)
        self.n, self.n_seqs = sum(news), len(news)
        self.starts = np.concatenate([[0], np.cumsum(news)])
        self.seq_start, self.past, self.ctx, self.table = ints(self.starts), ints(pasts), ints(self.lens), ints(self.lists)
        self.positions = ints(np.concatenate([np.arange(p, p + n) for p, n in zip(pasts, news)]))
        self.token_seq = ints(np.concatenate([np.full(n, s) for s, n in enumerate(news)]))

    def sizes(self, heads, kv, dim, window=0, keep=0):
        return dict(n_tokens=self.n, n_seqs=self.n_seqs, max_new=max(self.news), max_ctx=max(self.lens), n_heads=heads, n_kv_heads=kv,
                    head_dim=dim, window=window, keep_first=keep)


def awkward_rows(rng, n, kv, dim, dtype):
    """Rows whose groups end where a rule could slip: ties between codes, a largest number at and beside a scale's seventh multiple,
    zeros, subnormals, numbers past the format, infinities and NaN."""
    x = rng.standard_normal((n, kv, dim)) * np.exp(3 * rng.standard_normal((n, kv, 1)))
    g = x.reshape(-1, 32)
    b = rng.integers(0, 255, len(g))
    s = plain.SCALES[b]
    for i in range(len(g)):
        kind = i % 11
        if kind == 0:
            g[i] = s[i] * (rng.integers(-7, 7, 32) + 0.5)
            g[i, 0] = 7 * s[i]
        elif kind == 1:
            g[i] = np.clip(g[i], -1, 1) * s[i]
            g[i, 5] = 7 * s[i] * (1 + 2.0 ** -7)
        elif kind == 2:
            g[i] = np.clip(g[i], -1, 1) * s[i]
            g[i, 31] = -7 * s[i]
        elif kind == 3:
            g[i] = 0.0
        elif kind == 4:
            g[i] *= 1e-30 if i % 2 else 1e-41
        elif kind == 5:
            g[i] *= 1e6
        elif kind == 6 and i % 2:
            g[i, 7] = [np.nan, np.inf, -np.inf][i % 3]
        elif kind == 7:
            g[i] = s[i] * (rng.integers(-7, 7, 32) + 0.5) * (1 + 2.0 ** -23 * rng.integers(-2, 3, 32))
            g[i, 3] = 7 * s[i]
    return torch.tensor(g.reshape(n, kv, dim)).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv, dim", [(1, 32), (3, 64), (2, 96), (8, 128), (5, 256)])
@pytest.mark.parametrize("pasts, news", [([0], [1]), ([63, 64, 0], [2, 1, 130]), ([5, 700], [600, 1])])
def test_what_the_pages_hold_is_the_definition_bit_for_bit(dtype, kv, dim, pasts, news):
    step, rng = Step(pasts, news), np.random.default_rng(dim + len(news))
    rows = awkward_rows(rng, step.n + 3, 2 * kv, dim, dtype)
    k, v = rows[:, :kv], rows[:, kv:]
    before = torch.randint(0, 256, (step.pages, kv, kernels.cache4_record_bytes(dim)), dtype=torch.uint8, device=DEV)
    pool = before.clone()
    kernels.cache4_append(k, v, pool, step.positions, step.token_seq, step.ctx, step.table, step.width, n_tokens=step.n)
    want = before.cpu().numpy().copy()
    xk, xv = host(k), host(v)
    hk, hv = plain.held(xk), plain.held(xv)
    for t in range(step.n):
        seq, pos = int(step.token_seq[t]), int(step.positions[t])
        page, r, at = step.lists[seq, pos // PAGE], pos % PAGE, dim // 2
        for h in range(kv):
            one = plain.record(np.repeat(xk[t, h][None], PAGE, 0), np.repeat(xv[t, h][None], PAGE, 0))
            for first, size in ((0, at), (32 * dim, at), (64 * dim, dim // 32), (66 * dim, dim // 32)):
                want[page, h, first + r * size:first + (r + 1) * size] = one[first:first + size]
    assert np.array_equal(pool.cpu().numpy(), want)
    got_k = torch.full((step.n + 2, kv, dim), 9.0, dtype=dtype, device=DEV)
    got_v = torch.full_like(got_k, 9.0)
    kernels.cache4_gather(pool, step.positions, step.token_seq, step.table, step.width, got_k, got_v, n_tokens=step.n)
    assert np.array_equal(host(got_k[:step.n]), hk[:step.n], equal_nan=True)
    assert np.array_equal(host(got_v[:step.n]), hv[:step.n], equal_nan=True)
    assert bool((got_k[step.n:] == 9).all()) and bool((got_v[step.n:] == 9).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_of_any_stride_and_alignment(dtype, shift):
    kv, dim, step = 2, 64, Step([10, 0], [1, 70])
    gen = torch.Generator(device=DEV).manual_seed(3)
    proj = torch.randn(step.n, 5 * kv * dim + 7 + shift, generator=gen, device=DEV).to(dtype)[:, shift:]
    k = proj[:, 3:3 + 2 * kv * dim].view(step.n, kv, 2 * dim)[..., :dim]      # heads two heads apart
    v = proj[:, 300:300 + kv * dim].view(step.n, kv, dim)
    pool = torch.zeros(step.pages, kv, kernels.cache4_record_bytes(dim), dtype=torch.uint8, device=DEV)
    kernels.cache4_append(k, v, pool, step.positions, step.token_seq, step.ctx, step.table, step.width, n_tokens=step.n)
    rows = torch.zeros(step.n, 3 * kv * dim + shift, dtype=dtype, device=DEV)[:, shift:]
    got_k, got_v = rows[:, :kv * dim].view(step.n, kv, dim), rows[:, 2 * kv * dim:].view(step.n, kv, dim)
    kernels.cache4_gather(pool, step.positions, step.token_seq, step.table, step.width, got_k, got_v, n_tokens=step.n)
    assert np.array_equal(host(got_k), plain.held(host(k))) and np.array_equal(host(got_v), plain.held(host(v)))
    assert bool((rows[:, kv * dim:2 * kv * dim] == 0).all())


def test_a_ring_keeps_its_newest_positions():
    kv, dim, step = 1, 32, Step([100, 0], [300, 10], ring=3)
    gen = torch.Generator(device=DEV).manual_seed(5)
    k, v = (torch.randn(step.n, kv, dim, generator=gen, device=DEV).bfloat16() for _ in range(2))
    pool = torch.zeros(step.pages, kv, kernels.cache4_record_bytes(dim), dtype=torch.uint8, device=DEV)
    kernels.cache4_append(k, v, pool, step.positions, step.token_seq, step.ctx, step.table, step.width, n_tokens=step.n)
    got_k, got_v = torch.empty_like(k), torch.empty_like(v)
    kernels.cache4_gather(pool, step.positions, step.token_seq, step.table, step.width, got_k, got_v, n_tokens=step.n)
    kept = [t for t in range(step.n) if int(step.positions[t]) >= step.lens[int(step.token_seq[t])] - 3 * PAGE]
    assert len(kept) == 3 * PAGE + 10
    assert np.array_equal(host(got_k)[kept], plain.held(host(k))[kept]) and np.array_equal(host(got_v)[kept], plain.held(host(v))[kept])


def filled(step, kv, dim, rng, spread=1.0):
    """A pool whose records hold every sequence's keys and values; everything else in it (rows past a sequence's end, pages of nobody)
    stands for NaN.  Returns the pool and the held values, [positions, kv, dim] a sequence."""
    pool = np.full((step.pages, kv, kernels.cache4_record_bytes(dim)), 255, dtype=np.uint8)
    keys, values = [], []
    for s, length in enumerate(step.lens):
        gain = np.exp(0.5 * rng.standard_normal((kv, dim)))
        k = rng.standard_normal((length, kv, dim)) * gain * spread
        v = rng.standard_normal((length, kv, dim)) * np.exp(rng.standard_normal((length, kv, 1)))
        keys.append(plain.held(k))
        values.append(plain.held(v))
        lost = max(0, -(-length // PAGE) - step.width)       # pages of a ring that have come round
        for page in range(lost, -(-length // PAGE)):
            for h in range(kv):
                rows = [np.full((PAGE, dim), np.nan) for _ in range(2)]
                n = min(PAGE, length - page * PAGE)
                rows[0][:n], rows[1][:n] = k[page * PAGE:page * PAGE + n, h], v[page * PAGE:page * PAGE + n, h]
                pool[step.lists[s, page % step.width], h] = plain.record(*rows)
    return torch.tensor(pool, device=DEV), keys, values


def attend(step, q, pool, heads, kv, dim, window, keep, scale, rows=2, **kw):
    sizes = step.sizes(heads, kv, dim, window, keep)
    out = torch.full((step.n + rows, heads * dim), 7.0, dtype=q.dtype, device=DEV)
    scratch = torch.full((max(1, kernels.cache4_attention_scratch_floats(**sizes)),), float("nan"), device=DEV)
    kernels.cache4_attention(q, out, pool, step.table, step.width, step.seq_start, step.past, scale=scale, scratch=scratch, **sizes, **kw)
    kernels.check_status(torch.device(DEV))
    assert bool((out[step.n:] == 7).all())
    return out[:step.n]


def compare(step, got, q, keys, values, heads, kv, dim, window, keep, scale):
    bits = 8 if got.dtype == torch.bfloat16 else 24
    for s in range(step.n_seqs):
        a, b = step.starts[s], step.starts[s + 1]
        if a == b:
            continue
        x = host(q[a:b, :heads * dim]).reshape(-1, heads, dim)
        y, size, reach, count = plain.attention(x, keys[s], values[s], step.pasts[s], scale, window, keep)
        far = np.abs(host(got[a:b]).reshape(y.shape) - y) / (plain.allowed(bits, y, size, reach, count, dim) + 1e-300)      # (a channel of zeros allows nothing)
        assert far.max() <= 1.0, (s, float(far.max()), np.unravel_index(far.argmax(), far.shape))


STEPS = [([0], [1]), ([62, 63, 64, 900], [1, 1, 1, 1]), ([0, 0, 0], [1, 65, 200]), ([3, 0, 300, 129], [70, 1, 129, 0]),
         ([1000, 2], [16, 3])]
SEES = [(0, 0), (1, 0), (50, 3), (64, 64), (100, 130)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv, dim", [(1, 1, 32), (4, 4, 64), (8, 1, 128), (6, 2, 96), (2, 1, 256), (15, 3, 64), (16, 2, 128)])
@pytest.mark.parametrize("pasts, news", STEPS)
@pytest.mark.parametrize("window, keep", SEES)
def test_attention(dtype, heads, kv, dim, pasts, news, window, keep):
    step, rng = Step(pasts, news), np.random.default_rng(heads * dim + window)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim + 24))).to(dtype).to(DEV)
    scale = dim ** -0.5
    got = attend(step, q, pool, heads, kv, dim, window, keep, scale)
    compare(step, got, q, keys, values, heads, kv, dim, window, keep, scale)
    assert torch.equal(got, attend(step, q, pool, heads, kv, dim, window, keep, scale))


@pytest.mark.parametrize("heads, kv, dim", [(2, 2, 64), (5, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize("pasts, news", [([9001], [1]), ([5000, 17, 0], [1, 1, 1]), ([4500, 60], [3, 1]), ([6000, 300], [50, 41]), ([4000], [257])])
@pytest.mark.parametrize("window, keep", [(0, 0), (2100, 70), (3000, 0)])
def test_long_runs_in_pieces(heads, kv, dim, pasts, news, window, keep):
    step, rng = Step(pasts, news), np.random.default_rng(heads + window)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    got = attend(step, q, pool, heads, kv, dim, window, keep, -0.2)
    compare(step, got, q, keys, values, heads, kv, dim, window, keep, -0.2)
    assert torch.equal(got, attend(step, q, pool, heads, kv, dim, window, keep, -0.2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv, dim", [(4, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("pasts, news", [([70, 300], [3, 2]), ([0, 100], [140, 1])])
@pytest.mark.parametrize("window, keep", [(0, 0), (40, 3)])
def test_a_key_or_value_of_nan_reaches_the_queries_that_see_it_and_no_other(dtype, heads, kv, dim, pasts, news, window, keep):
    step, rng = Step(pasts, news), np.random.default_rng(dim)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).to(dtype).to(DEV)
    clean = attend(step, q, pool, heads, kv, dim, window, keep, dim ** -0.5)
    for where, which in ((1, 1), (60, 1), (71, 1), (71, 0), (99, 1), (2, 0)):
        bad, group, h = pool.clone(), rng.integers(dim // 32), rng.integers(kv)
        s = 0 if where < step.lens[0] else 1
        at = (66 if which else 64) * dim + where % PAGE * (dim // 32) + group
        bad[int(step.lists[s, where // PAGE]), h, at] = 255
        got = attend(step, q, bad, heads, kv, dim, window, keep, dim ** -0.5).view(step.n, heads, dim)
        hit = torch.zeros(step.n, heads, dim, dtype=torch.bool, device=DEV)
        for t in range(step.starts[s], step.starts[s + 1]):
            p = int(step.positions[t])
            if where <= p and (not window or where > p - window or where < keep):
                channels = slice(32 * group, 32 * group + 32) if which else slice(0, dim)
                hit[t, h * (heads // kv):(h + 1) * (heads // kv), channels] = True
        assert torch.equal(torch.isnan(got), hit), (where, which)
        assert torch.equal(got[~hit], clean.view(got.shape)[~hit])


@pytest.mark.parametrize("heads, kv, dim, news", [(4, 4, 64, [1, 1]), (4, 4, 64, [40, 3]), (2, 2, 32, [2, 1]), (64, 1, 128, [1, 1])])
def test_a_page_outside_the_pool_is_reported(heads, kv, dim, news):
    step, rng = Step([100, 70], news), np.random.default_rng(1)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    k, v = (torch.zeros(step.n, kv, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for wrong in (-1, step.pages, 2 ** 31 - 1):
        table = step.table.clone()
        table[1, 0] = wrong
        table[1, 1] = wrong
        args = step.sizes(heads, kv, dim)
        out = torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device=DEV)
        scratch = torch.empty(kernels.cache4_attention_scratch_floats(**args), device=DEV)
        before = pool.clone()
        calls = [lambda: kernels.cache4_attention(q, out, pool, table, step.width, step.seq_start, step.past, scale=1.0, scratch=scratch, **args),
                 lambda: kernels.cache4_append(k, v, pool, step.positions, step.token_seq, step.ctx, table, step.width, n_tokens=step.n),
                 lambda: kernels.cache4_gather(pool, step.positions, step.token_seq, table, step.width, k, v, n_tokens=step.n)]
        for call in calls:
            call()
            with pytest.raises(KernelError, match="outside its table or pool"):
                kernels.check_status(torch.device(DEV))
        first = step.starts[1]
        assert bool(torch.isnan(k[first:]).all()) and not bool(torch.isnan(k[:first]).any())
        pages = [int(p) for p in step.lists[0]]
        others = [p for p in range(step.pages) if p not in pages]
        assert torch.equal(pool[others], before[others])          # (nothing of the second sequence went anywhere)
        pool.copy_(before)
        k.zero_()
        v.zero_()


def test_tokens_of_a_sequence_or_position_outside_the_table_are_reported():
    kv, dim = 2, 64
    pool = torch.zeros(3, kv, 68 * dim, dtype=torch.uint8, device=DEV)
    k = torch.ones(4, kv, dim, dtype=torch.bfloat16, device=DEV)
    table = ints([[0, 1]])
    for seq, pos in (([0, 0, 0, 1], [0, 1, 2, 3]), ([0, 0, -1, 0], [0, 1, 2, 3]), ([0, 0, 0, 0], [0, 1, -5, 3])):
        pool.zero_()
        kernels.cache4_append(k, k, pool, ints(pos), ints(seq), ints([4]), table, 2, n_tokens=4)
        with pytest.raises(KernelError, match="outside its table or pool"):
            kernels.check_status(torch.device(DEV))
        assert int((pool[0, 0, 64 * dim:66 * dim] != 0).sum()) == 3 * dim // 32      # (the three others are filed)


@pytest.mark.parametrize("heads, kv, dim", [(4, 4, 64), (32, 4, 128), (3, 1, 96)])
def test_what_a_step_may_leave_out(heads, kv, dim):
    """No tokens, no sequences, sequences without tokens, starts that lie behind the step's tokens."""
    step, rng = Step([30, 5, 64, 7], [0, 3, 0, 1]), np.random.default_rng(4)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n + 3, heads * dim))).bfloat16().to(DEV)
    got = attend(step, q, pool, heads, kv, dim, 0, 0, 0.1)
    compare(step, got, q, keys, values, heads, kv, dim, 0, 0, 0.1)
    out = torch.full((step.n, heads * dim), 5.0, dtype=torch.bfloat16, device=DEV)
    args = step.sizes(heads, kv, dim)
    scratch = torch.empty(kernels.cache4_attention_scratch_floats(**args), device=DEV)
    for change in (dict(n_tokens=0), dict(n_seqs=0), dict(max_new=0)):
        kernels.cache4_attention(q, out, pool, step.table, step.width, step.seq_start, step.past, scale=0.1, scratch=scratch, **{**args, **change})
    assert bool((out == 5).all())
    # the last sequence's tokens are not the step's: its rows stay as they are
    kernels.cache4_attention(q[:3], out, pool, step.table, step.width, step.seq_start, step.past, scale=0.1, scratch=scratch, **{**args, "n_tokens": 3})
    assert bool((out[3:] == 5).all()) and torch.equal(out[:3], got[:3])
    empty = torch.empty(0, kv, dim, dtype=torch.bfloat16, device=DEV)
    kernels.cache4_append(empty, empty, pool, ints([]), ints([]), step.ctx, step.table, step.width, n_tokens=0)
    kernels.cache4_gather(pool, ints([]), ints([]), step.table, step.width, empty, empty, n_tokens=0)
    kernels.check_status(torch.device(DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv, dim", [(2, 2, 64), (64, 1, 128), (24, 1, 64)])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("news", [[1, 2], [90, 1]])
def test_scales_rows_of_any_alignment_and_windows_of_any_length(dtype, heads, kv, dim, scale, news):
    step, rng = Step([150, 10], news), np.random.default_rng(heads)
    pool, keys, values = filled(step, kv, dim, rng)
    for shift, window in ((0, 1 << 40), (1, 33)):
        q = torch.tensor(rng.standard_normal((step.n, heads * dim + 9))).to(dtype).to(DEV)[:, shift:]
        got = attend(step, q, pool, heads, kv, dim, window, 5, scale)
        compare(step, got, q, keys, values, heads, kv, dim, window, 5, scale)


@pytest.mark.parametrize("heads, kv, dim, news", [(2, 2, 64, [1, 1]), (4, 1, 128, [60, 1]), (2, 1, 96, [5, 1])])
def test_queries_that_are_no_numbers(heads, kv, dim, news):
    """A row of NaN or infinities is NaN, and no other row notices."""
    step, rng = Step([500, 70], news), np.random.default_rng(3)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    clean = attend(step, q, pool, heads, kv, dim, 0, 0, 0.1).view(step.n, heads, dim)
    for value in (float("nan"), float("inf"), float("-inf")):
        bad = q.clone()
        bad[-1, 3] = value
        got = attend(step, bad, pool, heads, kv, dim, 0, 0, 0.1).view(step.n, heads, dim)
        assert bool(torch.isnan(got[-1, 0]).all())
        assert torch.equal(got[:-1], clean[:-1]) and torch.equal(got[-1, 1:], clean[-1, 1:])


def test_a_window_over_pages_that_come_round():
    """Pages of a ring hold the newest positions only; rows that have been overwritten are never looked at."""
    for heads, kv, dim in ((2, 2, 64), (8, 1, 128), (2, 1, 96)):
        for window, pasts, news in ((100, [1000, 130], [1, 1]), (60, [777, 64], [5, 30]), (20, [500, 3], [100, 2])):
            step, rng = Step(pasts, news, ring=3), np.random.default_rng(window)
            pool, keys, values = filled(step, kv, dim, rng)
            q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
            got = attend(step, q, pool, heads, kv, dim, window, 0, 0.1)
            compare(step, got, q, keys, values, heads, kv, dim, window, 0, 0.1)


def test_every_bfloat16_as_the_largest_of_a_group():
    """Each finite magnitude once: its scale is the smallest that reaches it, with ties and near ties of that scale beside it."""
    bits = np.arange(0x7f80, dtype=np.uint32)
    top = (bits << 16).view(np.float32).astype(np.float64)
    s = plain.SCALES[np.minimum(np.searchsorted(7.0 * plain.SCALES, top), 254)]
    rng = np.random.default_rng(11)
    x = s[:, None] * (rng.integers(-7, 7, (len(top), 32)) + 0.5) * (1 + rng.integers(-1, 2, (len(top), 32)) * 2.0 ** -7)
    x = np.clip(x, -top[:, None], top[:, None])
    x[np.arange(len(top)), rng.integers(0, 32, len(top))] = top * rng.choice([-1, 1], len(top))
    kv, dim = 2, 128
    rows = x.reshape(-1, kv, dim)
    step = Step([0], [len(rows)])
    for shift in (0, 1):                                 # in 16-byte pieces, and one by one
        wide = torch.zeros(len(rows), kv * dim + 8, dtype=torch.bfloat16, device=DEV)
        k = wide.as_strided((len(rows), kv, dim), (kv * dim + 8, dim, 1), shift)
        k.copy_(torch.tensor(rows).bfloat16())
        v = torch.flip(k, (0,))
        pool = torch.zeros(step.pages, kv, kernels.cache4_record_bytes(dim), dtype=torch.uint8, device=DEV)
        kernels.cache4_append(k, v, pool, step.positions, step.token_seq, step.ctx, step.table, step.width, n_tokens=step.n)
        got_k, got_v = (torch.empty(len(rows), kv, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        kernels.cache4_gather(pool, step.positions, step.token_seq, step.table, step.width, got_k, got_v, n_tokens=step.n)
        assert np.array_equal(host(got_k), plain.held(host(k))) and np.array_equal(host(got_v), plain.held(host(v)))


@pytest.mark.parametrize("heads, kv, dim, pasts, news", [
    (4, 4, 64, [1900], [201]), (4, 4, 128, [1900], [201]), (64, 8, 128, [1206, 33], [14, 9]), (3, 1, 128, [4439], [204]),
    (8, 8, 64, [3500, 0, 700], [40, 17, 1]), (16, 2, 128, [5825, 100, 2000], [31, 30, 1]), (10, 2, 64, [2500], [700]), (32, 4, 128, [4000, 9], [250, 1])])
@pytest.mark.parametrize("window, keep", [(0, 0), (900, 5)])
def test_rows_of_both_kinds_in_pieces(heads, kv, dim, pasts, news, window, keep):
    step, rng = Step(pasts, news), np.random.default_rng(heads + dim + window)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    got = attend(step, q, pool, heads, kv, dim, window, keep, 0.15)
    compare(step, got, q, keys, values, heads, kv, dim, window, keep, 0.15)
    assert torch.equal(got, attend(step, q, pool, heads, kv, dim, window, keep, 0.15))
    if kernels._sm_count() == 148:
        kind, _, pieces, *_ = kernels._cache4_plan(148, len(pasts), max(news), max(step.lens), heads, kv, dim, window, keep, True)
        assert kind == "many" and (pieces > 1 or window)


@pytest.mark.parametrize("heads, kv, dim, pasts, news", [(4, 4, 64, [1500, 300], [90, 2]), (4, 1, 128, [1500, 3000], [40, 64])])
@pytest.mark.parametrize("window, keep", [(0, 0), (700, 3)])
def test_values_of_nan_in_pieces(heads, kv, dim, pasts, news, window, keep):
    test_a_key_or_value_of_nan_reaches_the_queries_that_see_it_and_no_other(torch.bfloat16, heads, kv, dim, pasts, news, window, keep)


@pytest.mark.parametrize("seqs, new", [(50, 1), (112, 2), (128, 1), (131, 1)])
@pytest.mark.parametrize("heads, kv, dim", [(8, 8, 64), (16, 4, 128)])
@pytest.mark.parametrize("window, keep", [(0, 0), (100, 3)])
def test_more_sequences_than_run_at_once(seqs, new, heads, kv, dim, window, keep):
    """Lengths in any order, many of them alike, sequences without tokens among them: the blocks are not begun in their order."""
    rng = np.random.default_rng(seqs + dim)
    pasts = [int(p) for p in rng.choice([0, 5, 63, 64, 200, 200, 391], seqs)]
    news = [int(n) for n in rng.integers(0, new + 1, seqs)]
    news[3] = new
    step = Step(pasts, news)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    got = attend(step, q, pool, heads, kv, dim, window, keep, 0.2)
    compare(step, got, q, keys, values, heads, kv, dim, window, keep, 0.2)
    # the same sequences the other way round: every one's result to the bit
    back = Step(pasts[::-1], news[::-1])
    order = torch.cat([torch.arange(step.starts[s], step.starts[s + 1]) for s in reversed(range(seqs))]).to(DEV)
    back.table = torch.flip(step.table, (0,)).contiguous()
    assert torch.equal(attend(back, q[order], pool, heads, kv, dim, window, keep, 0.2), got[order])


@pytest.mark.parametrize("seqs, new, longest", [(9, 70, 300), (12, 33, 200), (40, 20, 100)])
@pytest.mark.parametrize("heads, kv, dim", [(64, 8, 128), (32, 16, 64)])
@pytest.mark.parametrize("window, keep", [(0, 0), (150, 3)])
def test_more_portions_than_run_at_once(seqs, new, longest, heads, kv, dim, window, keep):
    """Pasts in any order, sequences without tokens among them: the blocks are not begun in their order, and the results do not show it."""
    rng = np.random.default_rng(seqs + dim)
    pasts = [int(p) for p in rng.choice([0, 7, 64, 190, 190, longest], seqs)]
    news = [int(n) for n in rng.integers(0, new + 1, seqs)]
    news[2] = new
    step = Step(pasts, news)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    got = attend(step, q, pool, heads, kv, dim, window, keep, 0.2)
    compare(step, got, q, keys, values, heads, kv, dim, window, keep, 0.2)
    back = Step(pasts[::-1], news[::-1])
    order = torch.cat([torch.arange(step.starts[s], step.starts[s + 1]) for s in reversed(range(seqs))]).to(DEV)
    back.table = torch.flip(step.table, (0,)).contiguous()
    assert torch.equal(attend(back, q[order], pool, heads, kv, dim, window, keep, 0.2), got[order])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv, dim", [(4, 4, 64), (16, 4, 128)])
@pytest.mark.parametrize("seqs, new", [(2, 1), (2, 90), (70, 1), (30, 60)])
@pytest.mark.parametrize("window, keep", [(0, 0), (90, 3)])
def test_a_past_that_no_sequence_has_is_reported(dtype, heads, kv, dim, seqs, new, window, keep):
    """It counts as none; the other sequences do not notice."""
    step, rng = Step([150 + 2 * s for s in range(seqs)], [new] * seqs), np.random.default_rng(1)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).to(dtype).to(DEV)
    clean, past = attend(step, q, pool, heads, kv, dim, window, keep, 0.1), step.past
    step.past = past.clone()
    step.past[1] = 0
    none = attend(step, q, pool, heads, kv, dim, window, keep, 0.1)[new:2 * new]
    for wrong in (-1, -64, -2 ** 31, 2 ** 31 - 1):
        step.past[1] = wrong
        args = step.sizes(heads, kv, dim, window, keep)
        out = torch.empty(step.n, heads * dim, dtype=dtype, device=DEV)
        scratch = torch.empty(kernels.cache4_attention_scratch_floats(**args), device=DEV)
        kernels.cache4_attention(q, out, pool, step.table, step.width, step.seq_start, step.past, scale=0.1, scratch=scratch, **args)
        with pytest.raises(KernelError, match="outside its table or pool"):
            kernels.check_status(torch.device(DEV))
        assert torch.equal(out[new:2 * new], none)
        assert torch.equal(out[:new], clean[:new]) and torch.equal(out[2 * new:], clean[2 * new:])


@pytest.mark.parametrize("heads, kv, dim, pasts, news", [(4, 2, 64, [70, 300, 0], [3, 1, 2]), (8, 1, 128, [900, 3000], [1, 1]), (6, 3, 64, [0, 65], [140, 90])])
@pytest.mark.parametrize("window, keep", [(0, 0), (100, 3)])
def test_the_kernel_for_every_case_when_it_is_asked_for(heads, kv, dim, pasts, news, window, keep):
    step, rng = Step(pasts, news), np.random.default_rng(dim)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    got = attend(step, q, pool, heads, kv, dim, window, keep, dim ** -0.5, impl="any")
    compare(step, got, q, keys, values, heads, kv, dim, window, keep, dim ** -0.5)


@pytest.mark.parametrize("heads, kv, dim", [(1, 1, 128), (2, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("past, new, window, keep", [(967, 56, 415, 0), (3013, 12, 467, 0), (5000, 25, 334, 1), (2000, 17, 512, 70)])
def test_few_rows_behind_a_window(heads, kv, dim, past, new, window, keep):
    step, rng = Step([past], [new]), np.random.default_rng(new)
    pool, keys, values = filled(step, kv, dim, rng)
    q = torch.tensor(rng.standard_normal((step.n, heads * dim))).bfloat16().to(DEV)
    got = attend(step, q, pool, heads, kv, dim, window, keep, dim ** -0.5)
    compare(step, got, q, keys, values, heads, kv, dim, window, keep, dim ** -0.5)
