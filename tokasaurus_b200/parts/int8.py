"""Attention and the gated feed-forward in 8 bits: matrices as 8-bit codes with a scale an output channel, made from the loaded
ones when a part is bound, against tokens that are brought to 8 bits one by one; keys and values as 8-bit codes with a scale a
page and kv head.  Norms, embedding, head and the residual stream stay as they are.  (The reference has no counterpart: its
weights and cache are bfloat16, tokasaurus/model/kv_cache.py:27-54.)

What a token's keys and values are held as goes by what shares their page: by the tokens behind them in the same portion (one
scale), and, where they topped the scale of those ahead, by one more rounding of those.  Results therefore depend, within the
codes' rounding, on how a prompt is cut into portions, which without an 8-bit cache they do not."""

from __future__ import annotations

import torch

from tokasaurus_b200.kernels import int8, ops
from tokasaurus_b200.kernels.modules import int8_modules
from tokasaurus_b200.parts.attention import PagedAttention
from tokasaurus_b200.parts.base import PagedCacheNeed
from tokasaurus_b200.parts.mlp import GatedMLP


class Int8PagedAttention(PagedAttention):
    def __init__(self, *args, int8_linears: bool = False, int8_cache: bool = False, **kw):
        super().__init__(*args, **kw)
        if self.qkv_stage is not None:
            raise ValueError("attention in 8 bits has no stage between the projections and the rotation")
        self.int8_linears, self.int8_cache = bool(int8_linears), bool(int8_cache)
        self.qkv_codes = self.o_codes = None  # (codes, scales) of the matrices

    def kernel_modules(self, dtype):
        return int8_modules((self.head_dim,) if self.int8_cache else ())

    def cache_need(self):
        return PagedCacheNeed(self.n_kv_heads, self.head_dim, self.window, eight_bits=self.int8_cache)

    def plan_key(self):
        return None if self.int8_cache else super().plan_key()  # (the work over an 8-bit cache is cut on the device)

    def bind(self, weights, rt) -> None:
        super().bind(weights, rt)
        if self.int8_linears:
            self.qkv_codes, self.o_codes = int8.quantise_rows(self.w_qkv), int8.quantise_rows(self.w_o)
            self.w_qkv = self.w_o = None

    def _project(self, ctx, h, w, codes):
        return ops.linear(h, w) if codes is None else int8.linear_int8(h, *codes, ctx.status)

    def _project_out(self, ctx, attn):
        if self.o_codes is None and ops.can_use_few_rows(attn, self.w_o, ops.ATTN_FEW_ROWS_MAX):
            return ops.linear_few_rows(attn, self.w_o, ctx.status)  # (slices, which the norm behind adds up)
        return self._project(ctx, attn, self.w_o, self.o_codes)

    def forward(self, ctx, h, cache, out_rows=None):
        hd, nh, nkv = self.head_dim, self.n_heads, self.n_kv_heads
        tables = ctx.tables[cache.group]
        rot = self.position.rotary_dim if self.position.kind == "rotary" else 0
        qkv = self._project(ctx, h, self.w_qkv, self.qkv_codes)
        if not self.int8_cache:
            ops.rope_kv_write(qkv, ctx.positions, ctx.token_seq, tables.indptr, tables.page_ids, self.inv_freq, cache.k, cache.v,
                              nh, nkv, hd, rot, cache.page_size, cache.writable, ctx.status)
            return self._project_out(ctx, self.attend(ctx, qkv, cache, out_rows))
        int8.rope_kv8_write(qkv, ctx.positions, ctx.token_seq, tables.indptr, tables.page_ids, self.inv_freq, cache.k, cache.v,
                            cache.k_scale, cache.v_scale, nh, nkv, hd, rot, cache.page_size, cache.writable, ctx.status)
        attn = torch.empty((h.shape[0], nh * hd), dtype=h.dtype, device=h.device)
        int8.attn_kv8(qkv, attn, cache.k, cache.v, cache.k_scale, cache.v_scale, ctx.seq_q_start, ctx.seq_q_len, ctx.seq_kv_len,
                      tables.indptr, tables.page_ids, nh, nkv, hd, cache.page_size, self.scale, self.window, ctx.status,
                      **self._bounds(ctx, tables, cache.page_size))
        if out_rows is not None:
            wanted = torch.empty((out_rows.numel(), nh * hd), dtype=h.dtype, device=h.device)
            ops.gather_rows(attn, out_rows, wanted)
            attn = wanted
        return self._project_out(ctx, attn)

    @staticmethod
    def _bounds(ctx, tables, page_size: int) -> dict:
        """What the launches are sized by: the step's own lengths, or, in a step graph, the most of any step it is replayed for."""
        if ctx.lengths is None:
            # (contexts grow up to what the table holds, which a graph stages at the size of the whole pool)
            return dict(max_q_len=1 if ctx.decode_graph else ctx.n_tokens, max_kv_len=tables.page_ids.shape[0] * page_size,
                        single_tokens=ctx.n_seqs, portions=0 if ctx.decode_graph else ctx.n_seqs)
        q_len = ctx.lengths
        return dict(max_q_len=int(q_len.max()), max_kv_len=int(ctx.host.seq_kv_len.max()), single_tokens=int((q_len == 1).sum()))


class Int8GatedMLP(GatedMLP):
    """``down(silu(gate(h)) * up(h))`` with its three matrices in 8 bits; the product of gate and up applies the SiLU gate."""

    def kernel_modules(self, dtype):
        return int8_modules()

    def bind(self, weights, rt) -> None:
        g, u, d = self.names
        if self.activation != "silu" or self.inner % 8:
            raise ValueError("a feed-forward in 8 bits has the SiLU gate and a width that is a multiple of 8")
        self.gate_up_codes = int8.quantise_rows(ops.interleave_gate_up(weights[g], weights[u]))
        self.down_codes = int8.quantise_rows(weights[d].contiguous())

    def forward(self, ctx, h):
        act = int8.linear_int8(h, *self.gate_up_codes, ctx.status, gated=True)
        return int8.linear_int8(act, *self.down_codes, ctx.status, out_dtype=torch.float32 if self.out_f32 else None)
