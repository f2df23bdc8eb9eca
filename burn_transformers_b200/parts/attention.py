"""Self-attention over the cache."""
from __future__ import annotations

import torch

from .. import kernels
from ..cache.spec import PAGE_SIZE, CacheNeed, KvSpec
from ..errors import CacheError, ShapeError
from ..weights.spec import MATRIX, VECTOR, TensorSpec
from .base import Mixer
from .linear import linear

_SM_COUNTS: dict = {}


def _sm_count(device) -> int:
    """Streaming multiprocessors of `device` (asked of the driver once)."""
    if device not in _SM_COUNTS:
        _SM_COUNTS[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return _SM_COUNTS[device]


class CausalSelfAttention(Mixer):
    """Multi-head (or grouped) attention with one fused query|key|value projection.

    [q|k|v] = x @ qkv.weight + qkv.bias with the weight stored [in, out]; head h owns channels
    h*head_dim..(h+1)*head_dim of its block; scores are (q . k) * scale, masked causally (and by
    `window` if given), softmax in 32-bit, then the value mix and the output projection, whose
    result is added to the residual stream (src/models/gpt2/model.rs:114-142, 218-261;
    src/attention/dispatch.rs:277-430 of the reference).  `n_kv_heads` < `n_heads` shares each key
    head among consecutive query heads.

    `qk_norm_eps`: every query and key head is normed, x / sqrt(mean(x^2) + eps) * weight ("q_norm.weight" and "k_norm.weight",
    [head_dim]), before `positions` turns it, in the same pass where `positions` offers it.

    `cache_bits` 4 (or `hold_cache_in(4)`): the cache holds keys and values in 4-bit codes (csrc/cache4.cuh).  Every query then attends over
    held values, the step's own too: a sequence's portions change nothing but roundings (of sums, and in bfloat16 of the softmax weights,
    which are rounded relative to the largest score that a warp or piece has met: up to 2^-8 of each).  With a `window` the cache keeps what
    the window needs, or every position where that takes no more than the window's ring in the model's type (cache/bank.py); positions below
    `keep_first` (of a cache in 4 bits only) stay visible beside the window, and the cache then keeps every position.
    """

    accepts_lazy_norm = True
    linear_weights = ("qkv.weight", "out.weight")
    MAX_HEAD_DIM = 256      # every head size up to this runs (the kernels made for 16-byte pieces where they fit)

    def __init__(self, width: int, n_heads: int, n_kv_heads: int, head_dim: int, scale: float, *,
                 causal: bool = True, window: int | None = None, bias: bool = True,
                 init_std: float = 0.02, out_init_std: float | None = None, positions=None, out_scale: float = 1.0,
                 qk_norm_eps: float | None = None, cache_bits: int | None = None, keep_first: int = 0):
        if n_heads <= 0 or n_kv_heads <= 0 or n_heads % n_kv_heads:
            raise ShapeError(f"{n_heads} query heads cannot share {n_kv_heads} key heads")
        if not 1 <= head_dim <= self.MAX_HEAD_DIM:
            raise ShapeError(f"head_dim {head_dim} is outside 1..{self.MAX_HEAD_DIM}, the head sizes the attention "
                             f"kernels take")
        self.width, self.n_heads, self.n_kv_heads, self.head_dim = width, n_heads, n_kv_heads, head_dim
        self.scale, self.causal, self.window, self.has_bias = float(scale), causal, window, bias
        # a position encoding that rotates (parts.base.PositionEncoding.rotates): applied to the new queries and
        # keys before the keys are filed, so that the cache holds rotated keys
        self.positions = positions if positions is not None and positions.rotates else None
        self.q_width = n_heads * head_dim
        self.kv_width = n_kv_heads * head_dim
        self.proj_width = self.q_width + 2 * self.kv_width
        self.init_std = init_std
        self.out_init_std = init_std if out_init_std is None else out_init_std
        # the mixer's result times this as it enters the residual stream: folded into the output projection when the
        # weights are bound (in 32-bit, rounded once to the compute type)
        self.out_scale = float(out_scale)
        self.qk_norm_eps = None if qk_norm_eps is None else float(qk_norm_eps)
        if keep_first < 0 or (keep_first and (window is None or cache_bits is None)):
            raise ShapeError(f"{keep_first} kept positions need a window and a cache in 4 bits")
        self.keep_first = int(keep_first)
        self.cache_bits = None
        if cache_bits is not None:
            self.hold_cache_in(cache_bits)

    def check_cache_bits(self, bits: int) -> None:
        """Raises what stands against holding this layer's keys and values in `bits` bits."""
        if bits != 4:
            raise ShapeError(f"a cache holds keys and values in the model's type or in 4 bits, not in {bits}")
        if self.head_dim % 32 or not self.causal:
            raise ShapeError(f"a cache in 4 bits takes causal attention over heads of a multiple of 32 channels, not of {self.head_dim}")

    def hold_cache_in(self, bits: int) -> None:
        """Has the cache hold this layer's keys and values in `bits` (4) bits; before the engine makes its cache."""
        self.check_cache_bits(bits)
        self.cache_bits = bits

    def bind(self, tensors):
        if self.positions is not None and hasattr(self.positions, "inv_freq"):
            for t in tensors.values():
                self.positions.inv_freq(t.device)
        if self.out_scale != 1.0:
            tensors = dict(tensors)
            for name in ("out.weight", "out.bias"):
                if name in tensors:
                    t = tensors[name]
                    tensors[name] = (t.to(torch.float32) * self.out_scale).to(t.dtype)
        super().bind(tensors)

    def specs(self):
        specs = {"qkv.weight": TensorSpec((self.width, self.proj_width), MATRIX, ("normal", self.init_std)),
                 "out.weight": TensorSpec((self.q_width, self.width), MATRIX, ("normal", self.out_init_std))}
        if self.has_bias:
            specs["qkv.bias"] = TensorSpec((self.proj_width,), VECTOR, ("zeros",))
            specs["out.bias"] = TensorSpec((self.width,), VECTOR, ("zeros",))
        if self.qk_norm_eps is not None:
            specs["q_norm.weight"] = TensorSpec((self.head_dim,), VECTOR, ("ones",))
            specs["k_norm.weight"] = TensorSpec((self.head_dim,), VECTOR, ("ones",))
        return specs

    def cache_need(self):
        if self.cache_bits is not None:
            # (kept first positions lie in pages that come round to nothing else)
            return CacheNeed(kv=KvSpec(self.n_kv_heads, self.head_dim, None if self.keep_first else self.window, bits=self.cache_bits))
        return CacheNeed(kv=KvSpec(self.n_kv_heads, self.head_dim, self.window))

    def _splits(self, ctx) -> int:
        """Blocks per (sequence, head) in a decode step: enough to fill the GPU about twice, none when the batch
        does that by itself (a split costs a merge); at most 8, so that they merge inside one thread-block
        cluster, and at most one per page."""
        units = max(1, ctx.n_seqs * self.n_heads)
        span = ctx.ctx_bound if self.window is None else min(ctx.ctx_bound, self.window)
        pages = max(1, -(-span // PAGE_SIZE))
        by_fill = -(-2 * _sm_count(ctx.ws.device) // units)
        return int(max(1, min(by_fill, pages, 8)))

    def _turn(self, ctx, proj) -> None:
        """Norms and turns the step's query and key heads in place."""
        heads = (self.n_heads, self.n_kv_heads, self.head_dim)
        if self.qk_norm_eps is None:
            if self.positions is not None:
                self.positions.rotate(ctx, proj, *heads)
            return
        norm = dict(q_weight=self.t_q_norm_weight, k_weight=self.t_k_norm_weight, eps=self.qk_norm_eps)
        if hasattr(self.positions, "norm_rotate"):
            self.positions.norm_rotate(ctx, proj, *heads, **norm)
            return
        kernels.qk_norm_rotary(proj, ctx.positions, None, n_tokens=ctx.n_tokens, n_heads=self.n_heads, n_kv_heads=self.n_kv_heads,
                               head_dim=self.head_dim, rot_dims=0, **norm)
        if self.positions is not None:
            self.positions.rotate(ctx, proj, *heads)

    def _step_pages(self, ctx):
        """Pages of the step's own for sequences that begin with it: (pool, table, table_len).  Sequence s has the pages from
        seq_start[s] // 64 + s on, as many as its tokens can fill."""
        table_len = -(-ctx.max_new // PAGE_SIZE)
        pool = ctx.ws.take((ctx.n_tokens // PAGE_SIZE + ctx.n_seqs, self.n_kv_heads, kernels.cache4_record_bytes(self.head_dim)), torch.uint8)
        table = ctx.ws.take((ctx.n_seqs, table_len), torch.int32)
        first, count = ctx.ws.take((ctx.n_seqs,), torch.int32), ctx.ws.take((max(ctx.n_seqs, table_len),), torch.int32)
        torch.arange(count.shape[0], out=count)
        torch.div(ctx.seq_start[:ctx.n_seqs], PAGE_SIZE, rounding_mode="floor", out=first)
        first.add_(count[:ctx.n_seqs])
        torch.add(first[:, None], count[:table_len], out=table)
        return pool, table, table_len

    def _forward_4_bits(self, ctx, proj, residual, entry, owns_cache) -> None:
        n = ctx.n_tokens
        pool, _, group, g = ctx.cache.layer_pools(entry)
        table, table_len = ctx.tables[g], group.table_len
        # prompts that a ring does not hold whole: their queries attend over pages that live as long as the step
        longer = group.is_ring and self.window is not None and not ctx.is_decode and ctx.max_new > table_len * PAGE_SIZE - self.window + 1
        if longer and not (ctx.fresh and owns_cache):
            # (the engine refuses such a step before the cache changes; this guards direct users of the part)
            raise CacheError("a step that brings this many tokens to sequences that already hold some would overwrite keys of a "
                             "windowed layer's ring that its first tokens still see")
        if owns_cache:
            k = proj[:n, self.q_width:self.q_width + self.kv_width].view(n, self.n_kv_heads, self.head_dim)
            v = proj[:n, self.q_width + self.kv_width:].view(n, self.n_kv_heads, self.head_dim)
            new = (ctx.positions, ctx.token_seq, ctx.ctx_len)
            kernels.cache4_append(k, v, pool, *new, table, table_len, n_tokens=n)
            if longer:
                pool, table, table_len = self._step_pages(ctx)
                kernels.cache4_append(k, v, pool, *new, table, table_len, n_tokens=n)
        # (where sequences go on, bounded by the cache's longest, not by the step's: how the keys are cut, and with it the last bits of the
        # results, is then the same for a step that is recorded and one that is not.  Prompts without a past are recorded by their sizes)
        max_ctx = ctx.max_new if ctx.fresh and not ctx.is_decode else ctx.cache.config.max_context
        sizes = dict(n_tokens=n, n_seqs=ctx.n_seqs, max_new=1 if ctx.is_decode else ctx.max_new, max_ctx=max_ctx,
                     n_heads=self.n_heads, n_kv_heads=self.n_kv_heads, head_dim=self.head_dim, window=self.window or 0, keep_first=self.keep_first)
        floats = kernels.cache4_attention_scratch_floats(**sizes)
        scratch = ctx.ws.take((floats,), torch.float32) if floats else None
        mixed = ctx.ws.take((n, self.q_width), ctx.dtype)
        kernels.cache4_attention(proj, mixed, pool, table, table_len, ctx.seq_start, ctx.past_len, scale=self.scale, scratch=scratch, **sizes)
        linear(ctx, mixed, self.t_out_weight, self.t_out_bias if self.has_bias else None, residual, m=n,
               residual=residual, w_is_nk=self.nk_out_weight)

    def forward(self, ctx, x, residual, entry, owns_cache=True):
        n = ctx.n_tokens
        dtype = ctx.dtype
        proj = ctx.ws.take((n, self.proj_width), dtype)
        linear(ctx, x, self.t_qkv_weight, self.t_qkv_bias if self.has_bias else None, proj, m=n,
               w_is_nk=self.nk_qkv_weight)
        program = getattr(ctx, "program", None)
        if self.positions is not None or self.qk_norm_eps is not None or self.cache_bits is not None:
            if program is not None:
                from ..engine.program import ProgramUnsupported
                raise ProgramUnsupported("a rotating position encoding, a norm of heads or a cache in 4 bits has no phase in the fused step")
            self._turn(ctx, proj)
        if self.cache_bits is not None:
            self._forward_4_bits(ctx, proj, residual, entry, owns_cache)
            return
        k_pool, v_pool, group, g = ctx.cache.layer_pools(entry)
        table = ctx.tables[g]
        window = self.window or 0
        # fresh sequences attend over the step's own projections; where the kernel can, it files their keys and values as it goes
        files = (owns_cache and ctx.fresh and not ctx.is_decode and not group.is_ring
                 and kernels.attention_prefill_files(proj, k_pool, self.head_dim, self.causal))
        if owns_cache and not ctx.is_decode and not files:
            side = getattr(ctx, "side", None) if ctx.fresh else None
            if side is not None:
                # fresh sequences attend over the step's own projections: nothing in this step reads the pages, so
                # the keys and values are filed beside the attention, on the step's second stream
                side.fork()
                with side.stream_context():
                    kernels.kv_append(proj, self.q_width, self.q_width + self.kv_width, ctx.positions, ctx.token_seq,
                                      ctx.ctx_len, table, group.table_len, k_pool, v_pool, n, self.n_kv_heads, self.head_dim)
            else:
                kernels.kv_append(proj, self.q_width, self.q_width + self.kv_width, ctx.positions, ctx.token_seq,
                                  ctx.ctx_len, table, group.table_len, k_pool, v_pool, n, self.n_kv_heads, self.head_dim)
        if program is not None and ctx.is_decode:
            # recorded as a phase of the fused step; its partial results are merged by the output projection
            mixed = program.add_attention(ctx, proj, k_pool, v_pool, table, group.table_len, n_heads=self.n_heads,
                                          n_kv_heads=self.n_kv_heads, head_dim=self.head_dim, scale=self.scale,
                                          window=window,
                                          new_kv_offsets=(self.q_width, self.q_width + self.kv_width) if owns_cache else None)
            linear(ctx, mixed, self.t_out_weight, self.t_out_bias if self.has_bias else None, residual, m=n,
                   residual=residual, w_is_nk=self.nk_out_weight)
            return
        mixed = ctx.ws.take((n, self.q_width), dtype)
        if ctx.is_decode and not kernels.attention_decode_supports(self.head_dim, proj.shape[1], dtype):
            # a head size whose rows are no whole 16-byte pieces: the step's keys and values are filed first, then
            # the kernel that reads element by element attends over the pages (one new token per sequence)
            kernels.kv_append(proj, self.q_width, self.q_width + self.kv_width, ctx.positions, ctx.token_seq,
                              ctx.ctx_len, table, group.table_len, k_pool, v_pool, n, self.n_kv_heads, self.head_dim)
            kernels.attention_prefill(proj, mixed, ctx.seq_start, ctx.past_len, ctx.n_seqs, 1, self.n_heads,
                                      self.n_kv_heads, self.head_dim, self.scale, causal=self.causal, window=window,
                                      k_pool=k_pool, v_pool=v_pool, table=table, table_len=group.table_len)
        elif ctx.is_decode:
            splits = self._splits(ctx)
            kernels.attention_decode(proj, mixed, k_pool, v_pool, table, group.table_len, ctx.ctx_len, ctx.n_seqs,
                                     self.n_heads, self.n_kv_heads, self.head_dim, self.scale, window=window,
                                     n_splits=splits, max_ctx=ctx.ctx_bound,
                                     new_kv_offsets=(self.q_width, self.q_width + self.kv_width) if owns_cache else None)
        elif ctx.fresh and owns_cache:
            # every sequence starts at position 0: keys and values are the step's own projections
            kernels.attention_prefill(proj, mixed, ctx.seq_start, ctx.past_len, ctx.n_seqs, ctx.max_new,
                                           self.n_heads, self.n_kv_heads, self.head_dim, self.scale,
                                           causal=self.causal, window=window,
                                           k_offset=self.q_width, v_offset=self.q_width + self.kv_width,
                                           **({"file": (k_pool, v_pool, table)} if files else {}))
        else:
            if group.is_ring and ctx.max_new > group.table_len * PAGE_SIZE - self.window + 1:
                # (the engine refuses such a step before the cache changes; this guards direct users of the part)
                raise CacheError("a step that brings this many tokens to sequences that already hold some would "
                                 "overwrite keys of a windowed layer's ring that its first tokens still see")
            kernels.attention_prefill(proj, mixed, ctx.seq_start, ctx.past_len, ctx.n_seqs, ctx.max_new,
                                           self.n_heads, self.n_kv_heads, self.head_dim, self.scale,
                                           causal=self.causal, window=window, k_pool=k_pool, v_pool=v_pool,
                                           table=table, table_len=group.table_len)
        linear(ctx, mixed, self.t_out_weight, self.t_out_bias if self.has_bias else None, residual, m=n,
               residual=residual, w_is_nk=self.nk_out_weight)
