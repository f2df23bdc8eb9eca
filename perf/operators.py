"""Operators of a serving path over a cache held in 4 bits, as cases that can be timed and checked one by one.

Three kinds of case:

* `rotary`: the norm of every query and key head of a step's projections and their rotation by position, in one pass.
* `cache`: a step's keys and values filed in 4-bit pages, and the values that the pages then hold read back.
* `attend`: attention of a step's queries over the 4-bit pages, causal, or with a window and a few first positions that stay
  visible; one new token a sequence, or prompts.

The plain forms are torch in 32 bits (angles in 64), without this library.  A page holds 64 positions of one key head:
`64 x dim / 2` bytes of key codes, as many of value codes, then `64 x dim / 32` bytes of key scales and of value scales.  Channel
c of a row has nibble c % 2 (0: the lower) of byte c / 2: a code n stands for (n - 8) s.  Every 32 channels share the scale s =
2^((b >> 3) - 20) (1 + (b & 7) / 8) of a byte b; 255 stands for NaN.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64
GROUP = 32


# ---- the cases ---------------------------------------------------------------------------------------------------

def _rotary(tokens, heads, kv_heads, dim, rot, far=0, interleaved=False, dtype="bfloat16", name=None):
    case = {"kind": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "far": far,
            "interleaved": interleaved, "dtype": dtype}
    return dict(case, name=name) if name else case


def _cache(seqs, past_lo, past_hi, new_lo, new_hi, kv_heads, dim, dtype="bfloat16", name=None):
    case = {"kind": "cache", "seqs": seqs, "past_lo": past_lo, "past_hi": past_hi, "new_lo": new_lo, "new_hi": new_hi,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    return dict(case, name=name) if name else case


def _attend(seqs, past_lo, past_hi, new_lo, new_hi, heads, kv_heads, dim, window=0, keep=0, name=None):
    case = {"kind": "attend", "seqs": seqs, "past_lo": past_lo, "past_hi": past_hi, "new_lo": new_lo, "new_hi": new_hi,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "keep": keep}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a decode step of a handful of conversations: the smallest call, all latency
        _rotary(8, 12, 12, 64, 64, name="rotary_decode_8"),
        # a full batch of long prompts with shared key heads: the most bytes
        _rotary(16 * 1024, 32, 8, 128, 128, name="rotary_prompts_16x1024"),
        # the 32-bit path: an odd number of rows, neighbouring channels turned, half of a head's channels, far positions
        _rotary(804, 25, 25, 64, 32, far=900_000, interleaved=True, dtype="float32", name="rotary_f32_far"),
        # one token for each of 64 sequences goes into the pages
        _cache(64, 250, 4100, 1, 1, 8, 128, name="cache_decode_64"),
        # prompts of unequal lengths go into the pages
        _cache(8, 0, 0, 101, 2047, 8, 128, name="cache_prompts_ragged"),
        # one user with a long document
        _attend(1, 32_766, 32_766, 1, 1, 32, 8, 128, name="decode_1_long"),
        # a handful of conversations of a small model, every head with keys of its own
        _attend(8, 202, 900, 1, 1, 12, 12, 64, name="decode_8_small"),
        # a serving batch with unequal histories: the most cache bytes
        _attend(64, 1_000, 8_000, 1, 1, 32, 8, 128, name="decode_64"),
        # long conversations that see a window and their first positions
        _attend(16, 4_001, 30_000, 1, 1, 32, 8, 128, window=1000, keep=4, name="decode_16_window"),
        # two prompts of a small model
        _attend(2, 0, 0, 1024, 1024, 12, 12, 64, name="prompts_2x1024_small"),
        # long prompts, shared key heads: the most operations
        _attend(2, 0, 0, 4095, 4096, 32, 8, 128, name="prompts_2x4096"),
        # prompts brought in portions behind unequal beginnings, with a window and kept first positions
        _attend(8, 17, 3771, 257, 257, 32, 8, 128, window=1024, keep=4, name="portions_8x257_window"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    what = rng.choice(("rotary", "cache", "decode", "decode", "prompts", "portions"))
    dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    if what == "rotary":
        dim = rng.choice((64, 80, 128))
        rot = rng.choice((dim, dim // 2))
        return _rotary(spread(1, 16 * 1024) * 32 // max(32, heads), heads, kv_heads, dim, rot, far=rng.choice((0, spread(10, 1_000_000))),
                       interleaved=rng.random() < 0.4, dtype=rng.choice(("bfloat16", "bfloat16", "float32"))) if heads <= 32 else \
            _rotary(spread(1, 8_000), heads, kv_heads, dim, rot)
    if what == "cache":
        new = spread(1, 2000)
        past = rng.choice((0, spread(1, 4000)))
        return _cache(rng.randint(1, 8) if new > 1 else spread(1, 64), past // 2, past, (new + 1) // 2, new, kv_heads, dim,
                      dtype=rng.choice(("bfloat16", "bfloat16", "float32")))
    window, keep = rng.choice(((0, 0), (0, 0), (spread(16, 4000), rng.choice((0, 1, 4, 70)))))
    if what == "decode":
        seqs = spread(1, 64)
        past = spread(1, min(32_000, 256_000 // seqs))
        return _attend(seqs, spread(1, past), past, 1, 1, heads, kv_heads, dim, window, keep)
    if what == "prompts":
        seqs = rng.randint(1, 6)
        new = spread(2, 3000 // seqs)
        return _attend(seqs, 0, 0, spread(1, new), new, min(heads, 32) // kv_heads * kv_heads, kv_heads, dim, window, keep)
    seqs = spread(1, 12)
    past, new = spread(1, 4000), spread(2, 300)
    return _attend(seqs, spread(1, past), past, spread(1, new), new, min(heads, 32) // kv_heads * kv_heads, kv_heads, dim, window, keep)


def _between(lo, hi, count):
    """`count` lengths from lo to hi, the longest first."""
    return [hi - (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _lengths(case):
    pasts = _between(case["past_lo"], case["past_hi"], case["seqs"])
    news = _between(case["new_lo"], case["new_hi"], case["seqs"])[::-1]      # (the longest run is not behind the longest past)
    return pasts, news


# ---- inputs ------------------------------------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _keys_and_values(rows, kv_heads, dim, gen, dtype):
    """Keys with a few loud channels, as trained models have them, and values of every size."""
    gain = torch.exp(0.6 * torch.randn(kv_heads, dim, generator=gen, device="cuda"))
    k = (torch.randn(rows, kv_heads, dim, generator=gen, device="cuda") * gain).to(dtype)
    v = torch.randn(rows, kv_heads, dim, generator=gen, device="cuda")
    v.mul_(torch.exp(torch.randn(rows, kv_heads, 1, generator=gen, device="cuda")))
    return k, v.to(dtype)


def _step(case, gen):
    """The integers of a step: where each new token belongs, and a table of pages in no order."""
    pasts, news = _lengths(case)
    starts = [0]
    starts += [sum(news[:i + 1]) for i in range(len(news))]
    lens = [p + n for p, n in zip(pasts, news)]
    width = -(-max(lens) // PAGE)
    held = [-(-n // PAGE) for n in lens]
    order = torch.randperm(sum(held), generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    first = 0
    for i, n in enumerate(held):
        table[i, :n] = order[first:first + n]
        first += n
    return {"seq_start": _ints(starts), "past": _ints(pasts), "ctx": _ints(lens), "table": table.cuda(),
            "token_seq": _ints([i for i, n in enumerate(news) for _ in range(n)]),
            "positions": _ints([p + j for p, n in zip(pasts, news) for j in range(n)]),
            "n_tokens": starts[-1], "max_new": max(news), "max_ctx": max(lens), "width": width, "pages": sum(held)}


def _filled_pages(pages, kv_heads, dim, gen):
    """Pages full of keys and values, filed by the rule."""
    pool = torch.empty(pages, kv_heads, 68 * dim, dtype=torch.uint8, device="cuda")
    for first in range(0, pages, 256):       # (in pieces: what is made on the way stays small)
        n = min(256, pages - first)
        k, v = _keys_and_values(n * PAGE, kv_heads, dim, gen, torch.bfloat16)
        shape = (n, PAGE, kv_heads, dim)
        kc, ks = _codes(k.view(shape).transpose(1, 2))
        vc, vs = _codes(v.view(shape).transpose(1, 2))
        flat = [t.reshape(n, kv_heads, -1) for t in (kc, vc, ks, vs)]
        pool[first:first + n] = torch.cat(flat, dim=-1)
    return pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "rotary":
        n, heads, kv, dim, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], getattr(torch, case["dtype"])
        proj = (1.5 * torch.randn(n, (heads + 2 * kv) * dim, generator=gen, device="cuda")).to(dtype)
        first = case["far"]
        positions = (first + torch.arange(n, device="cuda") % 1024).to(torch.int32)
        freq = (10000.0 ** (-2.0 * torch.arange(case["rot"] // 2, dtype=torch.float64) / case["rot"])).float().cuda()
        weights = [1.0 + 0.2 * torch.randn(dim, generator=gen, device="cuda") for _ in range(2)]
        return {"case": case, "proj": proj, "positions": positions, "freq": freq, "q_weight": weights[0], "k_weight": weights[1],
                "eps": 1e-6, "out": torch.empty(n, (heads + kv) * dim, dtype=dtype, device="cuda")}
    state = dict(_step(case, gen), case=case)
    n, kv, dim = state["n_tokens"], case["kv_heads"], case["dim"]
    if case["kind"] == "cache":
        dtype = getattr(torch, case["dtype"])
        k, v = _keys_and_values(n, kv, dim, gen, dtype)
        rows = torch.cat([k.reshape(n, -1), v.reshape(n, -1)], dim=1)      # as they lie in a step's projections
        state.update(k=rows[:, :kv * dim].view(n, kv, dim), v=rows[:, kv * dim:].view(n, kv, dim),
                     pool=torch.zeros(state["pages"], kv, 68 * dim, dtype=torch.uint8, device="cuda"),
                     k_out=torch.empty(n, kv, dim, dtype=dtype, device="cuda"), v_out=torch.empty(n, kv, dim, dtype=dtype, device="cuda"))
        return state
    heads = case["heads"]
    gain = torch.exp(0.5 * torch.randn(heads, 1, generator=gen, device="cuda"))
    q = (torch.randn(n, heads, dim, generator=gen, device="cuda") * gain).to(torch.bfloat16).reshape(n, heads * dim)
    state.update(q=q, out=torch.empty_like(q), pool=_filled_pages(state["pages"], kv, dim, gen), scale=dim ** -0.5)
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _scale_of(byte):
    """The scale that a byte stands for, in 32 bits (exact)."""
    b = byte.to(torch.int32)
    s = torch.ldexp(1.0 + (b & 7).float() / 8.0, (b >> 3) - 20)
    return torch.where(b == 255, torch.full_like(s, math.nan), s)


def _codes(x):
    """[..., dim] -> ([..., dim / 2] bytes of codes, [..., dim / 32] bytes of scales)."""
    g = x.to(torch.float64).unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    fine = torch.isfinite(top)
    part, power = torch.frexp(torch.where(fine, top, torch.zeros_like(top)) / 7.0)
    # top / 7 = 2 part 2^(power - 1): the next of eight steps of its power of two, not below it
    byte = (power.to(torch.int32) - 1 + 20) * 8 + torch.ceil((2.0 * part - 1.0) * 8.0).to(torch.int32)
    byte = torch.where(top > 0, byte, torch.zeros_like(byte)).clamp(0, 254)
    code = torch.round(g / _scale_of(byte).to(torch.float64)[..., None]).clamp(-7, 7)
    code = (torch.where(fine[..., None], code, torch.zeros_like(code)) + 8).to(torch.uint8).flatten(-2)
    byte = torch.where(fine, byte, torch.full_like(byte, 255)).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def _values(codes, scales):
    """The values of rows of codes, 32-bit: [..., dim / 2], [..., dim / 32] -> [..., dim]."""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float() - 8.0
    return code * _scale_of(scales).repeat_interleave(GROUP, dim=-1)


def _pages_of(pool, table, dim):
    """Keys and values of whole page lists: [seqs, kv_heads, width * 64, dim] each, 32-bit."""
    rec = pool[table.long()].transpose(1, 2)                     # [seqs, kv_heads, width, bytes]
    seqs, kv, width = rec.shape[:3]
    kc, vc, ks, vs = rec.split([32 * dim, 32 * dim, 2 * dim, 2 * dim], dim=-1)
    shape = lambda t: t.reshape(seqs, kv, width * PAGE, -1)      # noqa: E731
    return _values(shape(kc), shape(ks)), _values(shape(vc), shape(vs))


def _plain_rotary(s):
    case, proj = s["case"], s["proj"]
    n, heads, kv, dim, rot = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rot"]
    x = proj[:, :(heads + kv) * dim].float().view(n, heads + kv, dim)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
    x = torch.cat((x[:, :heads] * s["q_weight"], x[:, heads:] * s["k_weight"]), dim=1)
    angle = s["positions"].double()[:, None] * s["freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turned = x[..., :rot]
    if case["interleaved"]:
        u, v = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((u * cos - v * sin, v * cos + u * sin), dim=-1).flatten(-2)
    else:
        u, v = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((u * cos - v * sin, v * cos + u * sin), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1).to(proj.dtype).view(n, -1)


def _plain_cache(s):
    case = s["case"]
    dim = case["dim"]
    kc, ks = _codes(s["k"])
    vc, vs = _codes(s["v"])
    record = s["pool"].view(-1, case["kv_heads"], 68 * dim)
    lp = s["positions"].long()
    page, row = s["table"][s["token_seq"].long(), lp // PAGE].long(), lp % PAGE
    codes = record[..., :64 * dim].unflatten(-1, (2, PAGE, dim // 2))          # [pages, kv, k | v, 64, bytes]
    scales = record[..., 64 * dim:].unflatten(-1, (2, PAGE, dim // GROUP))
    codes[page, :, 0, row], codes[page, :, 1, row] = kc, vc
    scales[page, :, 0, row], scales[page, :, 1, row] = ks, vs
    k = _values(codes[page, :, 0, row], scales[page, :, 0, row])
    v = _values(codes[page, :, 1, row], scales[page, :, 1, row])
    return k.to(s["k"].dtype), v.to(s["v"].dtype)


def _plain_attend(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    k, v = _pages_of(s["pool"], s["table"], dim)                                # [seqs, kv, keys, dim]
    seqs, new = case["seqs"], s["max_new"]
    token = s["seq_start"][:-1, None].long() + torch.arange(new, device="cuda")      # rows past a sequence's last are never taken
    q = s["q"].float()[token.clamp(max=s["n_tokens"] - 1)].view(seqs, new, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.reshape(seqs, kv, -1, dim), k.transpose(2, 3)).view(seqs, kv, heads // kv, new, -1) * s["scale"]
    at = s["past"][:, None].long() + torch.arange(new, device="cuda")           # a query's position
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= at[..., None]
    if case["window"]:
        seen = seen & ((key > at[..., None] - case["window"]) | (key < case["keep"]))
    seen = seen & (key < s["ctx"][:, None, None])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
    total = scores.sum(-1, keepdim=True)
    v = v.masked_fill(~(key < s["ctx"][:, None])[:, None, :, None], 0.0)
    mixed = torch.matmul(scores.view(seqs, kv, -1, scores.shape[-1]), v).view(seqs, kv, heads // kv, new, dim) / total
    mixed = mixed.permute(0, 3, 1, 2, 4).reshape(seqs, new, heads * dim)
    return mixed[s["token_seq"].long(), (s["positions"] - s["past"][s["token_seq"].long()]).long()].to(torch.bfloat16)


def run(s):
    case = s["case"]
    if own:
        from burn_transformers_b200 import kernels
        if case["kind"] == "rotary":
            kernels.qk_norm_rotary(s["proj"], s["positions"], s["freq"], n_tokens=case["tokens"], n_heads=case["heads"],
                                   n_kv_heads=case["kv_heads"], head_dim=case["dim"], rot_dims=case["rot"], q_weight=s["q_weight"],
                                   k_weight=s["k_weight"], eps=s["eps"], interleaved=case["interleaved"], out=s["out"])
            return s["out"]
        if case["kind"] == "cache":
            kernels.cache4_append(s["k"], s["v"], s["pool"], s["positions"], s["token_seq"], s["ctx"], s["table"], s["width"],
                                  n_tokens=s["n_tokens"])
            kernels.cache4_gather(s["pool"], s["positions"], s["token_seq"], s["table"], s["width"], s["k_out"], s["v_out"],
                                  n_tokens=s["n_tokens"])
            return s["k_out"], s["v_out"]
        sizes = dict(n_tokens=s["n_tokens"], n_seqs=case["seqs"], max_new=s["max_new"], max_ctx=s["max_ctx"], n_heads=case["heads"],
                     n_kv_heads=case["kv_heads"], head_dim=case["dim"], window=case["window"], keep_first=case["keep"])
        if "scratch" not in s:       # (a program keeps one for its largest step)
            s["scratch"] = torch.empty(max(1, kernels.cache4_attention_scratch_floats(**sizes)), device="cuda")
        kernels.cache4_attention(s["q"], s["out"], s["pool"], s["table"], s["width"], s["seq_start"], s["past"], scale=s["scale"],
                                 scratch=s["scratch"], **sizes)
        return s["out"]
    return {"rotary": _plain_rotary, "cache": _plain_cache, "attend": _plain_attend}[case["kind"]](s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _seen(position, window, keep):
    """How many keys a query at `position` sees."""
    if not window or window > position:
        return position + 1
    return window + min(keep, position + 1 - window)


def work(case):
    size = 4 if case.get("dtype") == "float32" else 2
    dim, kv = case["dim"], case["kv_heads"]
    if case["kind"] == "rotary":
        elements = case["tokens"] * (case["heads"] + kv) * dim
        return {"bytes": 2 * elements * size + 4 * case["tokens"], "flops": 10 * elements}
    pasts, news = _lengths(case)
    if case["kind"] == "cache":
        elements = 2 * sum(news) * kv * dim
        return {"bytes": elements * (2 * size + 17 / 32), "flops": 4 * elements}
    pairs = keys = 0
    for past, new in zip(pasts, news):
        window, keep = case["window"], case["keep"]
        pairs += sum(_seen(p, window, keep) for p in range(past, past + new))
        first = max(0, past - window + 1) if window else 0               # the first key in the first query's window
        keys += past + new - first + min(keep if window else 0, first)
    rows = 2 * sum(news) * case["heads"] * dim * 2
    return {"bytes": rows + keys * kv * dim * 2 * 17 / 32, "flops": 4 * pairs * case["heads"] * dim}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    dim, kv = case["dim"], case["kv_heads"]
    if case["kind"] == "rotary":
        return _exact_rotary(case, s)
    if case["kind"] == "cache":
        return tuple(_exact_held(t.double()) for t in (s["k"], s["v"]))
    heads, group = case["heads"], case["heads"] // kv
    out = torch.empty(s["n_tokens"], heads, dim, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, heads, dim)
    pasts, news = _lengths(case)
    if sum((p + n) * n for p, n in zip(pasts, news)) * heads * dim > 2e13:
        return None
    row = 0
    for i, (past, new) in enumerate(zip(pasts, news)):
        length = past + new
        pages = s["table"][i, :-(-length // PAGE)].long()
        for h in range(kv):
            k = _exact_rows(s["pool"][pages, h], dim, 0)[:length]
            v = _exact_rows(s["pool"][pages, h], dim, 1)[:length]
            for first in range(0, new, 512):
                last = min(new, first + 512)
                position = torch.arange(past + first, past + last, device="cuda")[:, None]
                key = torch.arange(length, device="cuda")[None]
                hidden = key > position
                if case["window"]:
                    hidden |= (position - key >= case["window"]) & (key >= case["keep"])
                x = q[row + first:row + last, h * group:(h + 1) * group]
                logits = torch.einsum("ngd,kd->gnk", x, k) / math.sqrt(dim)
                logits[:, hidden] = -math.inf
                weights = torch.softmax(logits, dim=-1)
                out[row + first:row + last, h * group:(h + 1) * group] = torch.einsum("gnk,kd->ngd", weights, v)
        row += new
    return out.view(s["n_tokens"], -1)


def _exact_rotary(case, s):
    n, heads, dim, rot = case["tokens"], case["heads"], case["dim"], case["rot"]
    rows = s["proj"].double().view(n, -1, dim)[:, :heads + case["kv_heads"]]
    gain = torch.cat((s["q_weight"].expand(heads, dim), s["k_weight"].expand(case["kv_heads"], dim))).double()
    rows = rows / torch.sqrt(rows.pow(2).sum(-1, keepdim=True) / dim + s["eps"]) * gain
    pair = torch.arange(rot, device="cuda").view(-1, 2) if case["interleaved"] else torch.arange(rot, device="cuda").view(2, -1).t()
    z = torch.complex(rows[..., pair[:, 0]], rows[..., pair[:, 1]])
    z = z * torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double().outer(s["freq"].double()))[:, None]
    rows[..., pair[:, 0]], rows[..., pair[:, 1]] = z.real, z.imag
    return rows.reshape(n, -1)


def _exact_scales():
    return torch.tensor([(8 + b % 8) * 2.0 ** (b // 8 - 23) for b in range(255)], dtype=torch.float64, device="cuda")


def _exact_held(x):
    """What the groups of 32 numbers are held as: multiples, from -7 to 7, of the first scale whose seventh multiple reaches."""
    parts = x.unflatten(-1, (x.shape[-1] // GROUP, GROUP))
    scales = _exact_scales()
    which = torch.searchsorted(7.0 * scales, parts.abs().max(-1).values.contiguous()).clamp(max=254)
    s = scales[which].unsqueeze(-1)
    return (torch.round(parts / s).clamp(-7.0, 7.0) * s).flatten(-2)


def _exact_rows(records, dim, which):
    """[pages, bytes] of one key head -> [positions, dim]."""
    codes = records[:, which * 32 * dim:(which + 1) * 32 * dim].reshape(-1, dim // 2).long()
    at = 64 * dim + which * 2 * dim
    bytes_ = records[:, at:at + 2 * dim].reshape(-1, dim // GROUP).long()
    rows = torch.empty(codes.shape[0], dim, dtype=torch.float64, device="cuda")
    rows[:, 0::2], rows[:, 1::2] = (codes % 16 - 8).double(), (codes // 16 - 8).double()
    return rows * _exact_scales()[bytes_].repeat_interleave(GROUP, dim=1)
