"""What the calls of the 4-bit cache and of the norm with rotation refuse, and how a step is cut into pieces: no device is needed (a
tensor that says it lies on one, and a library that must not be reached)."""
import math
import random
import re
from pathlib import Path

import pytest
import torch

from burn_transformers_b200 import kernels
from burn_transformers_b200.errors import KernelError, ShapeError


class OnDevice(torch.Tensor):
    """A host tensor that says it lies on the current device."""
    place = 0

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return self.place


class OnAnother(OnDevice):
    place = 1


def dev(*shape, dtype=torch.bfloat16, kind=OnDevice):
    return torch.zeros(*shape, dtype=dtype).as_subclass(kind)


def ints(*shape, kind=OnDevice):
    return dev(*shape, dtype=torch.int32, kind=kind)


class Reached(Exception):
    pass


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    def reached():
        raise Reached
    monkeypatch.setattr(kernels, "library", reached)
    monkeypatch.setattr(kernels.torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(kernels, "_sm_count", lambda device=None: 148)
    monkeypatch.setattr(kernels, "_status_address", lambda device: 0)
    monkeypatch.setattr(kernels, "_raw_stream", lambda device: 0)


def rotary(**kw):
    args = dict(proj=dev(5, 512), positions=ints(5), inv_freq=dev(32, dtype=torch.float32), n_tokens=5, n_heads=4, n_kv_heads=2, head_dim=64,
                rot_dims=64, q_weight=dev(64, dtype=torch.float32), k_weight=dev(64, dtype=torch.float32), eps=1e-6)
    args.update(kw)
    return kernels.qk_norm_rotary(args.pop("proj"), args.pop("positions"), args.pop("inv_freq"), **args)


def append(**kw):
    args = dict(k=dev(5, 2, 64), v=dev(5, 2, 64), pool=dev(9, 2, 4352, dtype=torch.uint8), positions=ints(5), token_seq=ints(5), ctx_len=ints(3),
                table=ints(3, 4), table_len=4, n_tokens=5)
    args.update(kw)
    n = args.pop("n_tokens")
    return kernels.cache4_append(**args, n_tokens=n)


def gather(**kw):
    args = dict(pool=dev(9, 2, 4352, dtype=torch.uint8), positions=ints(5), token_seq=ints(5), table=ints(3, 4), table_len=4, k=dev(5, 2, 64),
                v=dev(5, 2, 64), n_tokens=5)
    args.update(kw)
    return kernels.cache4_gather(**args)


def attend(**kw):
    args = dict(q=dev(5, 256), out=dev(5, 256), pool=dev(9, 2, 4352, dtype=torch.uint8), table=ints(3, 4), table_len=4, seq_start=ints(4),
                past_len=ints(3), n_tokens=5, n_seqs=3, max_new=3, max_ctx=200, n_heads=4, n_kv_heads=2, head_dim=64, scale=0.125,
                scratch=dev(1 << 16, dtype=torch.float32))
    args.update(kw)
    return kernels.cache4_attention(**args)


CASES = [
    (rotary, dict(proj=torch.zeros(5, 512, dtype=torch.bfloat16)), KernelError, "cpu"),
    (rotary, dict(proj=dev(5, 512, kind=OnAnother)), KernelError, "cuda:1"),
    (rotary, dict(positions=ints(5, kind=OnAnother)), KernelError, "cuda:1"),
    (rotary, dict(proj=dev(5, 512, dtype=torch.float16)), ShapeError, "bfloat16 or 32-bit"),
    (rotary, dict(proj=dev(4, 512)), ShapeError, "proj"),
    (rotary, dict(proj=dev(5, 383)), ShapeError, "proj"),
    (rotary, dict(proj=dev(512, 5).t()), ShapeError, "proj"),
    (rotary, dict(proj=dev(1, 512).expand(5, 512)), ShapeError, "proj"),
    (rotary, dict(out=dev(5, 384, dtype=torch.float32)), ShapeError, "out"),
    (rotary, dict(out=dev(4, 384)), ShapeError, "out"),
    (rotary, dict(out=dev(1, 384).expand(5, 384)), ShapeError, "out"),
    (rotary, dict(positions=ints(4)), ShapeError, "positions"),
    (rotary, dict(positions=dev(5, dtype=torch.int64)), ShapeError, "positions"),
    (rotary, dict(positions=None), ShapeError, "positions"),
    (rotary, dict(inv_freq=dev(31, dtype=torch.float32)), ShapeError, "inv_freq"),
    (rotary, dict(q_weight=None), ShapeError, "both weights"),
    (rotary, dict(k_weight=dev(63, dtype=torch.float32)), ShapeError, "k_weight"),
    (rotary, dict(rot_dims=63), ShapeError, "pairs"),
    (rotary, dict(rot_dims=66), ShapeError, "pairs"),
    (rotary, dict(head_dim=257), ShapeError, "257"),
    (rotary, dict(n_heads=0, n_kv_heads=0), ShapeError, "heads"),
    (rotary, dict(n_tokens=-1), ShapeError, "-1"),
    (append, dict(k=torch.zeros(5, 2, 64, dtype=torch.bfloat16)), KernelError, "cpu"),
    (append, dict(v=dev(5, 2, 64, kind=OnAnother)), KernelError, "cuda:1"),
    (append, dict(v=dev(5, 2, 64, dtype=torch.float32)), ShapeError, "v"),
    (append, dict(v=dev(5, 2, 32)), ShapeError, "v"),
    (append, dict(k=dev(5, 64, 2).transpose(1, 2)), ShapeError, "k"),
    (append, dict(k=dev(5, 128)), ShapeError, "key heads"),
    (append, dict(k=dev(4, 2, 64)), ShapeError, "k"),
    (append, dict(k=dev(5, 2, 48), v=dev(5, 2, 48)), ShapeError, "multiples of 32"),
    (append, dict(k=dev(5, 2, 288), v=dev(5, 2, 288)), ShapeError, "up to 256"),
    (append, dict(pool=dev(9, 2, 4351, dtype=torch.uint8)), ShapeError, "pool"),
    (append, dict(pool=dev(0, 2, 4352, dtype=torch.uint8)), ShapeError, "pool"),
    (append, dict(pool=dev(9, 3, 4352, dtype=torch.uint8)[:, :2]), ShapeError, "pool"),
    (append, dict(table=ints(4, 3).t()), ShapeError, "table"),
    (append, dict(table_len=5), ShapeError, "list of 5"),
    (append, dict(table_len=0), ShapeError, "list of 0"),
    (append, dict(token_seq=ints(4)), ShapeError, "token_seq"),
    (append, dict(ctx_len=None), ShapeError, "ctx_len"),
    (gather, dict(k=dev(1, 2, 64).expand(5, 2, 64)), ShapeError, "k"),
    (gather, dict(v=dev(5, 1, 64).expand(5, 2, 64)), ShapeError, "v"),
    (gather, dict(positions=ints(4)), ShapeError, "positions"),
    (gather, dict(n_tokens=-2), ShapeError, "-2"),
    (attend, dict(q=torch.zeros(5, 256, dtype=torch.bfloat16)), KernelError, "cpu"),
    (attend, dict(out=dev(5, 256, kind=OnAnother)), KernelError, "cuda:1"),
    (attend, dict(scratch=dev(1 << 16, dtype=torch.float32, kind=OnAnother), max_new=1, max_ctx=250 * 64, table_len=250, table=ints(3, 250)),
     KernelError, "cuda:1"),
    (attend, dict(n_heads=3), ShapeError, "cannot share"),
    (attend, dict(n_kv_heads=0), ShapeError, "cannot share"),
    (attend, dict(out=dev(5, 256, dtype=torch.float32)), ShapeError, "out"),
    (attend, dict(out=dev(5, 264)[:, :256]), ShapeError, "out"),
    (attend, dict(out=dev(4, 256)), ShapeError, "out"),
    (attend, dict(q=dev(5, 255)), ShapeError, "q"),
    (attend, dict(q=dev(5, 256, dtype=torch.float64)), ShapeError, "q"),
    (attend, dict(table=ints(2, 4)), ShapeError, "table"),
    (attend, dict(seq_start=ints(3)), ShapeError, "seq_start"),
    (attend, dict(past_len=ints(2)), ShapeError, "past_len"),
    (attend, dict(window=-1), ShapeError, "negative"),
    (attend, dict(keep_first=-1), ShapeError, "negative"),
    (attend, dict(max_ctx=257), ShapeError, "come round"),
    (attend, dict(max_ctx=300, window=100, keep_first=1), ShapeError, "come round"),
    (attend, dict(max_ctx=300, window=255, max_new=3), ShapeError, "come round"),
    (attend, dict(impl="fast"), ShapeError, "unknown kernel"),
    (attend, dict(max_new=1, max_ctx=250 * 64, table_len=250, table=ints(3, 250), scratch=None), ShapeError, "floats of scratch"),
    (attend, dict(max_new=1, max_ctx=250 * 64, table_len=250, table=ints(3, 250), scratch=dev(100, dtype=torch.float32)), ShapeError, "scratch"),
    (attend, dict(max_new=1, max_ctx=250 * 64, table_len=250, table=ints(3, 250), scratch=dev(1 << 20, dtype=torch.float32)[1:]), ShapeError,
     "16-byte"),
    (attend, dict(q=dev(40, 256), out=dev(40, 256), n_tokens=40, n_seqs=1, max_new=40, max_ctx=250 * 64, table_len=250, table=ints(3, 250),
                  scratch=dev(1 << 22, dtype=torch.float32)[3:]), ShapeError, "16-byte"),
]


@pytest.mark.parametrize("call, change, error, words", CASES, ids=[f"{c[0].__name__}-{'-'.join(c[1])}-{i}" for i, c in enumerate(CASES)])
def test_refusals(call, change, error, words):
    with pytest.raises(error, match=words):
        call(**change)


@pytest.mark.parametrize("call, change", [
    (rotary, {}), (rotary, dict(out=dev(6, 400))), (rotary, dict(q_weight=None, k_weight=None, rot_dims=0, inv_freq=None)), (append, {}),
    (rotary, dict(n_tokens=0)), (gather, {}), (gather, dict(k=dev(2, 5, 64).transpose(0, 1))), (attend, {}), (attend, dict(impl="any")),
    (attend, dict(max_ctx=300, window=254)), (attend, dict(q=dev(5, 300))), (append, dict(k=dev(1, 2, 64).expand(5, 2, 64)))])
def test_what_is_allowed_reaches_the_library(call, change):
    with pytest.raises(Reached):
        call(**change)


@pytest.mark.parametrize("heads, kv, dim", [(32, 8, 128), (12, 12, 64), (8, 1, 64), (6, 3, 96)])
@pytest.mark.parametrize("new", [1, 3, 40, 700])
@pytest.mark.parametrize("window, keep", [(0, 0), (100, 0), (1000, 4)])
def test_the_scratch_that_is_asked_for_covers_every_smaller_step(heads, kv, dim, new, window, keep):
    """A program keeps the scratch of its bounds: fewer or shorter sequences never need more, whichever kernel takes them."""
    sizes = [(seqs, ctx) for seqs in (1, 2, 5, 64, 300) for ctx in (new, new + 63, new + 1000, new + 30_000, 1 << 17)]
    asked = {s: kernels.cache4_attention_scratch_floats(s[0] * new, s[0], new, s[1], heads, kv, dim, window, keep) for s in sizes}
    for seqs, ctx in sizes:
        needs = [kernels._cache4_plan(148, fewer, new, shorter, heads, kv, dim, window, keep, fast)[3]
                 for fewer in {1, 2, 3, 5, 17, 64, 300} if fewer <= seqs for shorter in {new, new + 63, new + 200, new + 1000, new + 9_000, ctx}
                 if shorter <= ctx for fast in (True, False)]
        assert max(needs) <= asked[seqs, ctx], (seqs, ctx)


def test_records_are_laid_out_as_the_library_reads_them():
    api = (Path(kernels.__file__).parent / "csrc" / "api.h").read_text()
    letters = {"long long": "q", "int": "i", "float": "f", "cudaStream_t": "Q"}
    for name, record in kernels._RECORDS.items():
        parameters = re.search(rf"int {name.removesuffix('_packed')}\(([^)]*)\);", api).group(1).split(",")
        kinds = ["Q" if "*" in p else letters[p.rsplit(" ", 1)[0].strip()] for p in parameters]
        assert record.format == "=" + "".join(kinds), name


@pytest.mark.parametrize("call, change", [(rotary, dict(eps=1e300)), (rotary, dict(size=-1e39)), (attend, dict(scale=1e300))])
def test_arguments_that_fit_no_record(call, change):
    with pytest.raises(ShapeError, match="does not fit"):
        call(**change)


# heads, key heads, new tokens, longest sequence, window, kept positions: few rows behind a window of a few pages, one or two blocks
FEW_ROWS_IN_A_WINDOW = [(1, 1, 56, 1023, 415, 0), (2, 2, 56, 3301, 448, 0), (4, 2, 16, 23_538, 482, 0), (2, 1, 12, 3025, 467, 0), (1, 1, 25, 12_292, 334, 1),
                        (2, 2, 40, 10_764, 433, 0)]


@pytest.mark.parametrize("heads, kv, new, ctx, window, keep", FEW_ROWS_IN_A_WINDOW)
@pytest.mark.parametrize("dim", [64, 128])
def test_the_scratch_that_is_asked_for_is_taken(heads, kv, new, ctx, window, keep, dim):
    sizes = dict(n_tokens=new, n_seqs=1, max_new=new, max_ctx=ctx, n_heads=heads, n_kv_heads=kv, head_dim=dim, window=window, keep_first=keep)
    floats = kernels.cache4_attention_scratch_floats(**sizes)
    width = -(-ctx // 64)
    with pytest.raises(Reached):
        attend(q=dev(new, heads * dim), out=dev(new, heads * dim), pool=dev(2, kv, 68 * dim, dtype=torch.uint8), table=ints(1, width), table_len=width,
               seq_start=ints(2), past_len=ints(1), scratch=dev(floats, dtype=torch.float32), **sizes)


def test_scratch_over_random_sizes():
    """What is asked for covers the step itself and any of fewer or shorter sequences, over sizes of every order."""
    rng = random.Random(4)

    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    for _ in range(3000):
        kv, group, dim = rng.choice((1, 1, 2, 3, 8)), rng.choice((1, 1, 2, 4, 8)), rng.choice((32, 64, 128, 128))
        seqs, new = spread(1, 40), spread(1, 400)
        ctx = new + rng.choice((0, spread(1, 40_000)))
        window, keep = rng.choice(((0, 0), (spread(1, 3000), rng.choice((0, 1, 4, 70, 500))), (rng.randint(300, 520), 0)))
        sms = rng.choice((148, 148, 16, 132))
        plan = lambda n, c, fast: kernels._cache4_plan(sms, n, new, c, kv * group, kv, dim, window, keep, fast)      # noqa: E731
        asked = max(plan(seqs, ctx, fast)[4] for fast in (True, False))
        for fewer in {1, max(1, seqs // 2), seqs}:
            for shorter in {new, new + (ctx - new) // 3, new + (ctx - new) * 2 // 3, ctx}:
                needs = max(plan(fewer, shorter, fast)[3] for fast in (True, False))
                assert needs <= asked, (sms, seqs, new, ctx, kv, group, dim, window, keep, fewer, shorter)
