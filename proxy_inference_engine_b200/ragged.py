"""Ragged continuous batching: one model step over a mix of prefill chunks and decode rows.

``BatchDetails`` carries the fields of the reference's descriptor (CORE/include/engine/batch_details.hpp:10-90): the
concatenated ``token_ids`` / ``positions`` of the step, per-sequence ``input_lengths`` / ``context_lengths``, the
``consolidated_block_table`` of page ids (this build: 2-D ``[num_sequences, max_blocks]``, pages of 64 tokens from
``paging.PageAllocator``) and the prefill / decode counts.  The reference declares the descriptor but no kernel consumes
it yet (its scheduler is a skeleton); here ``ragged_step`` runs it:

* every token of the step is one row of the activation matrix, so the quantized matmuls see M = total_tokens_in_step;
* ``pie_rope_kv_append`` rotates q and k at each token's own position and appends k, v through the token's row of a
  per-token block table (the sequence's row, repeated) -- per-sequence positions, no uniform ``offset``
  (lifting PIE/cache/kv_cache/reusable.py:139);
* ``pie_decode_attn`` then gives every token the context ``position + 1`` of its own sequence: inside a prefill chunk
  that is exactly the causal mask of create_attention_mask (PIE/models/base.py:18-53), because the chunk's keys were
  appended before any of its queries attends.

Same arithmetic as the per-sequence path (Model.__call__ over a PagedKVCache); tests/test_gpu_ragged.py compares the two.

``StepPlan`` is the descriptor built on the device from lengths that live there: rows, slots and block table in one launch, one attention launch a layer that
reads a request's keys once for all its new tokens, and drafted tokens among them (``speculative_step``).  Its cache may be of 8 bits (``fp8_pools``), and the model's
linears of 8-bit integers (``llama.Model.to_int8``).
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from dataclasses import dataclass, field

import torch

from . import _lib, nn, ops
from .llama import MLP
from .ops import _p, _stream

PAGE_TOKENS = 64


def to_device(t: torch.Tensor, device) -> torch.Tensor:
    """A host tensor on the device, in stream order and without waiting for what is queued before it, as a plain copy would, so that a step can be
    prepared under the one before (which helps only callers that do not read a result in between).  The driver has taken the values when the call returns:
    9 to 60 us for 64 bytes to 800 KB.  (Page-locked memory: 18 to 43 us, and 1 to 3 ms after every graph capture, which empties torch's cache of it.)"""
    return t.to(device, non_blocking=torch.device(device).type == "cuda")


@dataclass
class BatchDetails:
    token_ids: torch.Tensor                     # int32 [total_tokens_in_step]
    positions: torch.Tensor                     # int32 [total_tokens_in_step]
    sequence_ids: list = field(default_factory=list)
    input_lengths: list = field(default_factory=list)
    context_lengths: list = field(default_factory=list)
    consolidated_block_table: torch.Tensor | None = None   # int32 [num_sequences, max_blocks]
    num_prefill_sequences: int = 0
    num_decode_sequences: int = 0
    total_tokens_in_step: int = 0
    state_slots: list = field(default_factory=list)        # per sequence: slot of its recurrent state (hybrid models)

    @classmethod
    def build(cls, sequences, device="cuda") -> "BatchDetails":
        """sequences: iterable of (sequence_id, new_token_ids, context_length, page_ids).  ``context_length`` = tokens of
        the sequence already in the cache; ``page_ids`` must cover context_length + len(new_token_ids) tokens."""
        ids, pos, sids, ins, ctxs, rows = [], [], [], [], [], []
        n_pre = n_dec = 0
        slots = []
        for sid, toks, ctx, pages, *rest in sequences:
            slots.append(int(rest[0]) if rest else 0)
            toks = [int(t) for t in toks]
            if not toks:
                raise ValueError(f"sequence {sid}: no tokens in this step")
            if ctx < 0:
                raise ValueError(f"sequence {sid}: negative context length")
            if sid in sids:
                raise ValueError(f"sequence {sid} appears twice in one step")
            need = (ctx + len(toks) + PAGE_TOKENS - 1) // PAGE_TOKENS
            if len(pages) < need:
                raise ValueError(f"sequence {sid}: {len(pages)} pages for {ctx + len(toks)} tokens (needs {need})")
            ids += toks
            pos += list(range(ctx, ctx + len(toks)))
            sids.append(sid); ins.append(len(toks)); ctxs.append(int(ctx)); rows.append([int(p) for p in pages])
            if len(toks) > 1 or ctx == 0:
                n_pre += 1
            else:
                n_dec += 1
        if not sids:
            raise ValueError("empty batch")
        width = max(1, max(len(r) for r in rows))
        table = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32)
        # tokens | positions | block table: one copy
        T = len(ids)
        dev = to_device(torch.cat([torch.tensor(ids + pos, dtype=torch.int32), table.flatten()]), device)
        return cls(dev[:T], dev[T:2 * T], sids, ins, ctxs, dev[2 * T:].view(table.shape), n_pre, n_dec, T, slots)

    def validate(self) -> None:
        n = len(self.sequence_ids)
        if len(self.input_lengths) != n or len(self.context_lengths) != n:
            raise ValueError("BatchDetails: per-sequence vectors differ in length")
        if sum(self.input_lengths) != self.total_tokens_in_step or self.token_ids.numel() != self.total_tokens_in_step \
                or self.positions.numel() != self.total_tokens_in_step:
            raise ValueError("BatchDetails: total_tokens_in_step != sum(input_lengths) / len(token_ids)")
        if self.num_prefill_sequences + self.num_decode_sequences != n:
            raise ValueError("BatchDetails: prefill + decode counts != number of sequences")
        if self.consolidated_block_table is None or self.consolidated_block_table.shape[0] != n:
            raise ValueError("BatchDetails: block table needs one row per sequence")
        width = self.consolidated_block_table.shape[1]
        for sid, inp, ctx in zip(self.sequence_ids, self.input_lengths, self.context_lengths):
            if inp <= 0 or ctx < 0 or (ctx + inp + PAGE_TOKENS - 1) // PAGE_TOKENS > width:
                raise ValueError(f"BatchDetails: sequence {sid} does not fit its block-table row")

    def last_token_rows(self) -> torch.Tensor:
        """Row of each sequence's last token in the step (the rows whose logits the sampler reads)."""
        ends, acc = [], 0
        for n in self.input_lengths:
            acc += n
            ends.append(acc - 1)
        return torch.tensor(ends, dtype=torch.long, device=self.token_ids.device)

    def hybrid_descriptor(self):
        """The step as libpie_b200_hybrid.so reads it (pieh_batch): per-row sequence index and position, per-sequence
        first row / rows / context / state slot, and the block table.  One host-to-device copy; returns (struct, keepalive)."""
        from ._lib import HybBatch
        if getattr(self, "_static_descriptor", None) is not None:   # a captured decode step: fixed buffers, refilled in place
            return self._static_descriptor
        n, T = len(self.sequence_ids), self.total_tokens_in_step
        starts, acc = [], 0
        for m in self.input_lengths:
            starts.append(acc)
            acc += m
        tok_seq = [i for i, m in enumerate(self.input_lengths) for _ in range(m)]
        slots = list(self.state_slots) if self.state_slots else [0] * n
        tile_seq, tile_row = [], []          # runs of <= 64 rows of one sequence: the query tiles of prompt attention
        for i, (s0, m) in enumerate(zip(starts, self.input_lengths)):
            for r0 in range(0, m, 64):
                tile_seq.append(i)
                tile_row.append(s0 + r0)
        nt = len(tile_seq)
        host = torch.tensor(tok_seq + starts + list(self.input_lengths) + list(self.context_lengths) + slots + tile_seq
                            + tile_row, dtype=torch.int32)
        dev = to_device(host, self.token_ids.device)
        ptr = lambda off: dev.data_ptr() + 4 * off
        d = HybBatch(T, n, ptr(0), self.positions.data_ptr(), ptr(T), ptr(T + n), ptr(T + 2 * n), ptr(T + 3 * n),
                     self.consolidated_block_table.data_ptr(), self.consolidated_block_table.stride(0), nt,
                     ptr(T + 4 * n), ptr(T + 4 * n + nt))
        return d, (dev, self.positions, self.consolidated_block_table)

    def token_block_table(self) -> torch.Tensor:
        """[total_tokens, max_blocks]: the block-table row of each token's sequence (what the kernels index by row)."""
        seq_of_token = torch.repeat_interleave(
            torch.arange(len(self.input_lengths), device=self.token_ids.device),
            torch.tensor(self.input_lengths, device=self.token_ids.device))
        return self.consolidated_block_table[seq_of_token].contiguous()


_DIMS = struct.Struct("7i").pack   # pie_step_dims


@dataclass
class StepPlan:
    """A ragged step described on the device: BatchDetails for callers whose requests' lengths live there -- after drafted tokens were verified, or in a captured
    step that runs again on other lengths.  One launch fills it; nothing is read back.  All int32, views of ``words``:

        row_starts [S + 1], contexts [S]     first row of each request, tokens it has in the cache
        sequences, positions, slots [T]      each row's request, position in it, and place in the pools (page * 64 + place in the page); -1, 0, -1 for rows behind the last
        block_table [S, max_blocks]          page ids, 0 behind a request's own
        logit_starts [S + 1], logit_rows [R] rows whose logits are wanted: each request's last 1 + drafted ones; 0 behind the last
        draft_tokens [R]                     the token each of them judges (verify_draft); -1 at a request's last
    """
    token_ids: torch.Tensor
    words: torch.Tensor
    dims: _lib.StepDims
    row_starts: torch.Tensor
    contexts: torch.Tensor
    sequences: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    block_table: torch.Tensor
    logit_starts: torch.Tensor
    logit_rows: torch.Tensor
    draft_tokens: torch.Tensor
    status: torch.Tensor

    FAULTS = {1: "a length is negative, or a request is longer than the step or its row of the block table", 2: "the requests have more tokens than token_ids",
              4: "the requests need more pages than there are page ids", 8: "a page id is outside the pools", 16: "a request's drafted tokens are not fewer than its new ones",
              32: "the requests have more logit rows than num_logits"}

    @classmethod
    def build(cls, token_ids, input_lengths, context_lengths, pages, *, num_pages: int, max_blocks: int, num_heads: int, num_kv_heads: int, draft_lengths=None,
              num_logits: int | None = None) -> "StepPlan":
        """token_ids int32 [T]: the requests' new tokens one behind the other; what is left of T belongs to nobody (ids of padding have to be tokens all the same).
        input_lengths, context_lengths int32 [S]: new tokens (0: the request sits this step out) and tokens in the cache.  pages: int32 page ids, ceil((cached + new) / 64) of
        each request one behind the other, or a table [S, columns] of them.  num_pages: of the pools.  max_blocks: columns of the plan's own block table.
        draft_lengths int32 [S]: how many of a request's new tokens are drafted ones (fewer than its new ones).  num_logits: logit rows to make room for (default: S, none drafted).
        Lengths that do not fit one another cannot be seen from here: check() tells, and until then nothing is read or written out of bounds."""
        S = input_lengths.numel()
        try:   # (packed, since a ctypes field takes what does not fit it modulo 2^32)
            dims = _lib.StepDims.from_buffer_copy(_DIMS(S, token_ids.numel(), S if num_logits is None else num_logits, max_blocks, num_pages, num_heads, num_kv_heads))
        except struct.error as e:
            raise ValueError(f"[StepPlan] not built here: numbers of anything have to be integers of 31 bits ({e})") from None
        got = ops.native_host().step_plan(token_ids, input_lengths, context_lengths, pages, draft_lengths, dims)
        if got is not None:
            return cls(token_ids, got[0], dims, *got[1:])
        what = "StepPlan"
        ops._step_ints(what, "token_ids", token_ids)
        ops._step_ints(what, "input_lengths", input_lengths, (S,))
        ops._step_ints(what, "context_lengths", context_lengths, (S,))
        if draft_lengths is not None:
            ops._step_ints(what, "draft_lengths", draft_lengths, (S,))
        if pages.dtype != torch.int32 or pages.dim() not in (1, 2) or (pages.dim() == 2 and pages.shape[0] != S):
            raise ValueError(f"[{what}] pages must be int32, a list or a table of {S} rows, but is {pages.dtype} {list(pages.shape)}")
        if pages.stride(-1) != 1 or (pages.dim() == 2 and pages.stride(0) < 1):
            pages = pages.contiguous()
        L = _lib.load()
        n = L.pie_step_plan_words(C.byref(dims))
        if token_ids.dim() != 1 or n == 0:
            raise ValueError(f"[{what}] not built here: {dims.requests} requests (1 to 4096), {dims.rows} rows, {dims.logit_rows} logit rows, {dims.blocks} blocks, "
                             f"{dims.pages} pages, {dims.Hq} query heads on {dims.Hkv}")
        given = [t for t in (token_ids, input_lengths, context_lengths, pages, draft_lengths) if t is not None]
        with ops._one_device(what, *given):
            words = torch.empty(n, dtype=torch.int32, device=token_ids.device)
            stride = 0 if pages.dim() == 1 else max(1, pages.stride(0))
            _lib.check(L.pie_step_plan_build(_p(words), C.byref(dims), _p(token_ids), _p(input_lengths), _p(context_lengths), _p(draft_lengths), _p(pages),
                                             pages.shape[-1], stride, _stream()), what)
        at = (C.c_longlong * 10)()
        _lib.check(L.pie_step_plan_offsets(C.byref(dims), at), what)
        T, R = dims.rows, dims.logit_rows
        part = lambda i, *shape: words[at[i]:at[i] + math.prod(shape)].view(shape)
        return cls(token_ids, words, dims, part(0, S + 1), part(1, S), part(2, T), part(3, T), part(4, T), part(5, S, dims.blocks), part(6, S + 1), part(7, R),
                   part(8, R), part(9, 192))

    def check(self) -> None:
        """Waits for the plan and raises ValueError for lengths and page ids that do not fit."""
        bits = 0
        for word in self.status.tolist():
            bits |= word
        if bits:
            raise ValueError("StepPlan: " + "; ".join(text for bit, text in self.FAULTS.items() if bits & bit))


def _planned_step(model, plan: StepPlan, pools, all_logits: bool) -> torch.Tensor:
    """ragged_step over a StepPlan: the rows' projections as there, keys and values through the slot map, attention of all rows in one launch a layer."""
    a, T = model.args, plan.dims.rows
    at0 = model.layers[0].self_attn
    Hq, Hkv, D = at0.num_heads, at0.n_kv_heads, at0.head_dim
    if getattr(at0.rope, "traditional", False) or getattr(getattr(model, "tp", None), "on", False):
        raise ValueError("[ragged_step] a StepPlan is for one GPU's whole model with rotation by halves")
    if len(pools) != len(model.layers):
        raise ValueError(f"[ragged_step] {len(pools)} pools for {len(model.layers)} layers")
    d = plan.dims   # (all of it before the first layer writes to its pools: slots of another plan's pools are other requests' places)
    for kp, vp in pools:
        if isinstance(kp, (tuple, list)):
            if len(kp) != 2 or not isinstance(vp, (tuple, list)) or len(vp) != 2:
                raise ValueError("[ragged_step] a StepPlan's attention reads bfloat16 pools, or fp8_pools; other 8-bit pools are for BatchDetails")
            if (d.Hq, d.Hkv) != (Hq, Hkv):
                raise ValueError(f"[ragged_step] the plan is for {d.Hq} heads on {d.Hkv}, but the model has {Hq} on {Hkv}")
            ops._fp8_pools("ragged_step", *kp, *vp, d, D)
            continue
        ops._slot_pools("ragged_step", kp, vp)
        if (d.Hq, d.Hkv, d.pages) != (Hq, Hkv, kp.shape[0]) or kp.shape[2:] != (Hkv, D):
            raise ValueError(f"[ragged_step] the plan is for {d.Hq} heads over {d.pages} pages of {d.Hkv} heads, but the model has {Hq} over {Hkv} of {D} features and a pool is "
                             f"{tuple(kp.shape)}")
    h = model.model.embed_tokens(plan.token_ids[None])
    for ly, (kp, vp) in zip(model.layers, pools):
        at, mlp = ly.self_attn, ly.mlp
        qkv = nn.int8_beside(h, (at.q_proj, at.k_proj, at.v_proj), norm=ly.input_layernorm)
        if qkv is None:
            x = ly.input_layernorm(h)
            qkv = at.q_proj(x), at.k_proj(x), at.v_proj(x)
        q, k, v = qkv[0].view(T, Hq, D), qkv[1].view(T, Hkv, D), qkv[2].view(T, Hkv, D)
        if isinstance(kp, (tuple, list)):
            q = ops.rope_kv_fp8(q, k, v, at.rope._freqs, plan, *kp, *vp)
            o = ops.chunk_attention_fp8(q, *kp, *vp, plan, at.scale)
        else:
            q = ops.rope_kv_slots(q, k, v, at.rope._freqs, plan.positions, plan.slots, kp, vp)
            o = ops.chunk_attention(q, kp, vp, plan, at.scale)
        h = at.o_proj(o[None], residual=h) if type(at.o_proj) is nn.Int8Linear else ops.add(h, at.o_proj(o[None]))
        both = None
        if type(mlp) is MLP and type(mlp.down_proj) is nn.Int8Linear:   # (a class made from it may put something else between the matrices)
            both = nn.int8_beside(h, (mlp.gate_proj, mlp.up_proj), norm=ly.post_attention_layernorm)
        if both is not None:
            h = mlp.down_proj(ops.silu_mul(*both), residual=h)
        else:
            h = ops.add(h, mlp(ly.post_attention_layernorm(h)))
    if not all_logits:
        h = h.index_select(1, plan.logit_rows)
    w, s, b = model.head_slices()
    qz = a.quantization
    return ops.quantized_matmul(model.model.norm(h), w, s, b, transpose=True, group_size=qz["group_size"], bits=qz["bits"])[0]


def fp8_pools(model, num_pages: int, device="cuda") -> list:
    """Pools of a cache of 8 bits for the steps of a StepPlan, per layer ((k_codes, k_scales), (v_codes, v_scales)): float8_e4m3fn [num_pages, n_kv, 64, D] and a float32 scale for each
    page and head (ops.rope_kv_fp8).  Half the bytes of bfloat16 pools, and a two-thousandth."""
    pair = lambda at: (torch.zeros((num_pages, at.n_kv_heads, PAGE_TOKENS, at.head_dim), dtype=torch.float8_e4m3fn, device=device),
                       torch.zeros((num_pages, at.n_kv_heads), dtype=torch.float32, device=device))
    return [(pair(ly.self_attn), pair(ly.self_attn)) for ly in model.layers]


def speculative_step(model, plan: StepPlan, pools, *, max_draft: int, temp: float = 0.0, uniforms=None, noise=None, draft_logits=None):
    """One step of drafting decode: ragged_step over a plan whose requests bring their last token and some drafted ones (draft_lengths), then verify_draft.
    Returns its (tokens, counts, logprobs).  A request that took part then has context + new - drafted + counts - 1 tokens in the cache -- what lies behind them
    there is written over -- and its last token, tokens[s, counts[s] - 1], is the next step's first; of one that sat the step out (counts 0) nothing changed."""
    logits = ragged_step(model, plan, pools)
    return ops.verify_draft(logits, plan.draft_tokens, plan.logit_starts, max_draft=max_draft, temp=temp, uniforms=uniforms, noise=noise, draft_logits=draft_logits)


def ragged_step(model, batch: BatchDetails, pools, all_logits: bool = False) -> torch.Tensor:
    """One forward step of ``model`` over ``batch``.  pools: per layer (k_pool, v_pool) bf16 [n_pages, 64, n_kv, D] --
    the pools the block table's page ids index -- or, for the 8-bit KV cache of cache.PagedQuantizedKVCache, per layer
    ((k_quants, k_scales, k_biases), (v_quants, v_scales, v_biases)) [n_pages, n_kv, 64, .].
    Returns logits [num_sequences, vocab] of each sequence's last token (all_logits: [total_tokens, vocab]).
    ``batch`` may be a StepPlan (bfloat16 pools, or fp8_pools): logits [num_logits, vocab] of its logit rows."""
    if isinstance(batch, StepPlan):
        return _planned_step(model, batch, pools, all_logits)
    batch.validate()
    L = _lib.load()
    a = model.args
    T = batch.total_tokens_in_step
    at0 = model.layers[0].self_attn
    Hq, Hkv, D = at0.num_heads, at0.n_kv_heads, at0.head_dim
    table = batch.token_block_table()
    pos = batch.positions
    h = model.model.embed_tokens(batch.token_ids[None])          # [1, T, hidden]
    q = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=h.device)
    max_ctx = max(c + n for c, n in zip(batch.context_lengths, batch.input_lengths))
    for ly, (kp, vp) in zip(model.layers, pools):
        at = ly.self_attn
        x = ly.input_layernorm(h)
        qkv = torch.cat([at.q_proj(x), at.k_proj(x), at.v_proj(x)], dim=-1).view(T, (Hq + 2 * Hkv) * D)
        if isinstance(kp, (tuple, list)):   # quantised pools: (quants, scales, biases) [n_pages, n_kv, 64, .] per K and V
            desc = ops.kvq_desc(tuple(kp), tuple(vp), table, PAGE_TOKENS)
            ops.kvq_append(qkv, desc, pos, at.rope._freqs, Hq, Hkv, D, q_out=q)
            o = ops.decode_attention_q8(q, desc, pos, at.scale, Hkv, max_context=max_ctx)
        else:
            lay = ops.kv_layout(kp, table, PAGE_TOKENS)
            _lib.check(L.pie_rope_kv_append(_p(q), _p(qkv), _p(kp), _p(vp), C.byref(lay), _p(pos), _p(at.rope._freqs), T,
                                            Hq, Hkv, D, _stream()), "rope_kv_append")
            o = ops.decode_attention(q, kp, vp, lay, pos, at.scale, max_context=max_ctx)     # [T, Hq * D]
        h = ops.add(h, at.o_proj(o[None]))
        h = ops.add(h, ly.mlp(ly.post_attention_layernorm(h)))
    if not all_logits:
        h = h[:, batch.last_token_rows()]
    out = model.model.norm(h.contiguous())
    w, s, b = model.head_slices()
    qz = a.quantization
    return ops.quantized_matmul(out, w, s, b, transpose=True, group_size=qz["group_size"], bits=qz["bits"])[0]
