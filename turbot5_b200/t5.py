"""A thin T5 encoder / decoder stack around the fused-bias kernels.

Only what is needed to drive the attention path end to end (and to measure
encoder tokens/s): embeddings, pre-norm blocks (RMSNorm -> attention -> residual,
RMSNorm -> feed-forward -> residual), final norm, LM head.  Linear layers are
plain `nn.Linear` (cuBLAS); attention, RMSNorm and decoding go through the
library.  Module and parameter names follow the Hugging Face / TurboT5 layout
(`shared`, `encoder.block.N.layer.0.SelfAttention.q`, `...layer.1.DenseReluDense.wi_0`,
`decoder.block.N.layer.1.EncDecAttention.k`, `lm_head`), so a T5 state dict
loads with `load_state_dict`.

Restates the control flow of `T5Stack` / `T5Block` / `T5LayerSelfAttention` /
`T5LayerCrossAttention` / `T5LayerFF` (src/turbot5/model/modeling.py:63-342,
352-632) and the LM head of `T5ForConditionalGeneration`
(src/turbot5/heads/t5_heads.py:132-260).  Differences: the decoder uses the
flash module too (the reference hard-wires its `basic` attention there,
modeling.py:134-135,170) and generation keeps a preallocated K/V cache that the
split-KV decoding kernel reads in place, instead of `torch.cat` per step
(src/turbot5/model/attentions.py:198).
"""
from dataclasses import dataclass
from typing import List, Optional

import torch
from torch import nn

from . import _native as nat
from .attention import (flash_attention_with_fusing_bias, flash_attention_with_fusing_bias_varlen,
                        flash_decoding_quantized_with_fusing_bias, flash_decoding_with_fusing_bias)
from .generation import (CACHE_BLOCK, MAX_BEAMS, beam_search_sequences, beam_search_step, quantize_into_cache,
                         reorder_beam_cache)
from .modules import (T5ATTENTION_TYPES, T5FlashAttention, T5LayerNorm, add_rms_layer_norm, gated_gelu,
                      rms_layer_norm)
from .padding import get_unpad_plan, pad_rows, unpad_rows

_host = nat.host
_HALF = (torch.bfloat16, torch.float16)


@dataclass
class T5StackConfig:
    vocab_size: int = 32128
    d_model: int = 768
    d_kv: int = 64
    d_ff: int = 2048
    num_layers: int = 12
    num_decoder_layers: int = 12
    num_heads: int = 12
    relative_attention_num_buckets: int = 32
    relative_attention_max_distance: int = 128
    dropout_rate: float = 0.0
    layer_norm_epsilon: float = 1e-6
    feed_forward_proj: str = "gated-gelu"      # or "relu"
    tie_word_embeddings: bool = False
    is_decoder: bool = False
    decoder_start_token_id: int = 0
    attention_type: str = "flash"              # encoder self-attention: "flash" (full) or "local" (block-local)
    sliding_window: int = 512                  # block length of the "local" type
    eos_token_id: int = 1
    pad_token_id: int = 0


class _FusedOps:
    """Library operators behind `T5Stack.forward_fused`."""
    from .sequence_parallel import _DeviceOps as _sp
    rms_layer_norm = staticmethod(rms_layer_norm)
    add_rms_layer_norm = staticmethod(add_rms_layer_norm)
    gated_gelu = staticmethod(gated_gelu)
    attention = _sp.attention
    partial = _sp.partial
    merge = _sp.merge


class T5DenseGatedActDense(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.wi_0 = nn.Linear(cfg.d_model, cfg.d_ff, bias=False)
        self.wi_1 = nn.Linear(cfg.d_model, cfg.d_ff, bias=False)
        self.wo = nn.Linear(cfg.d_ff, cfg.d_model, bias=False)

    def forward(self, x):
        return self.wo(nn.functional.gelu(self.wi_0(x), approximate="tanh") * self.wi_1(x))


class T5DenseActDense(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.wi = nn.Linear(cfg.d_model, cfg.d_ff, bias=False)
        self.wo = nn.Linear(cfg.d_ff, cfg.d_model, bias=False)

    def forward(self, x):
        return self.wo(torch.relu(self.wi(x)))


class T5LayerFF(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        gated = cfg.feed_forward_proj.startswith("gated")
        self.DenseReluDense = T5DenseGatedActDense(cfg) if gated else T5DenseActDense(cfg)
        self.layer_norm = T5LayerNorm(cfg.d_model, eps=cfg.layer_norm_epsilon)

    def forward(self, hidden):
        return hidden + self.DenseReluDense(self.layer_norm(hidden).to(hidden.dtype))


class T5LayerSelfAttention(nn.Module):
    def __init__(self, cfg, has_relative_attention_bias):
        super().__init__()
        # the decoder always attends fully (as in the reference, src/turbot5/model/modeling.py:134-135)
        kind = T5FlashAttention if cfg.is_decoder else T5ATTENTION_TYPES[cfg.attention_type]
        self.SelfAttention = kind(cfg, has_relative_attention_bias=has_relative_attention_bias)
        self.layer_norm = T5LayerNorm(cfg.d_model, eps=cfg.layer_norm_epsilon)


class T5LayerCrossAttention(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.EncDecAttention = T5FlashAttention(cfg, cross_attention=True, has_relative_attention_bias=False)
        self.layer_norm = T5LayerNorm(cfg.d_model, eps=cfg.layer_norm_epsilon)


class T5Block(nn.Module):
    def __init__(self, cfg, has_relative_attention_bias):
        super().__init__()
        layers = [T5LayerSelfAttention(cfg, has_relative_attention_bias)]
        if cfg.is_decoder:
            layers.append(T5LayerCrossAttention(cfg))
        layers.append(T5LayerFF(cfg))
        self.layer = nn.ModuleList(layers)


class DecoderCache:
    """Preallocated K/V cache of one generation: self-attention keys/values grow in place,
    cross-attention keys/values are projected once from the encoder output.  Keys and values of a
    layer's self-attention live in ONE tensor (2, B, H, max_len, D), so that a decoding step appends
    both with one copy; `self_k[i]` / `self_v[i]` are its two halves.

    With `beams` the self-attention has a row for each of a sentence's beams, while the cross-attention's rows are the
    sentences: their beams read them together."""
    scales = ()
    workspace = None        # split scratch of this cache's own, or the one kept per stream

    def __init__(self, n_layers, batch, heads, d_kv, max_len, dtype, device, beams=1):
        self.self_kv = [torch.empty((2, batch * beams, heads, max_len, d_kv), dtype=dtype, device=device)
                        for _ in range(n_layers)]
        self.self_k = [kv[0] for kv in self.self_kv]
        self.self_v = [kv[1] for kv in self.self_kv]
        self.cross_k: List[Optional[torch.Tensor]] = [None] * n_layers
        self.cross_v: List[Optional[torch.Tensor]] = [None] * n_layers
        self.length = 0
        self.max_len = max_len
        self.beams = beams

    def set_cross(self, i, k, v, seqlens=None):
        self.cross_k[i], self.cross_v[i] = k, v

    def own_workspace(self):
        """Scratch for the split-KV launches that no other cache shares: captured graphs of two caches may then run at
        the same time."""
        L, (_, rows, H, cap, D) = nat.lib(), self.self_kv[0].shape
        need = L.t5b_decode_workspace_bytes(rows, H, 1, D, max(1, L.t5b_decode_num_splits(rows, H, cap)))
        for k in self.cross_k:
            if k is not None:
                B, _, N, _ = k.shape
                need = max(need, L.t5b_decode_workspace_bytes(B, H, self.beams, D, max(1, L.t5b_decode_num_splits(B, H, N))))
        self.workspace = torch.zeros(max(need, 256), dtype=torch.uint8, device=self.self_kv[0].device)

    def append(self, i, k, v, start):
        """New keys and values (B, H, M, D) at `start`: a number, or an int64 tensor for a single token."""
        if torch.is_tensor(start):
            self.self_k[i].index_copy_(2, start, k)
            self.self_v[i].index_copy_(2, start, v)
        else:
            self.self_k[i][:, :, start:start + k.shape[2]] = k
            self.self_v[i][:, :, start:start + k.shape[2]] = v

    def append_stacked(self, i, kv, pos):
        """The single new token's key and value, side by side (B, 1, 2, H, D): one copy."""
        self.self_kv[i].index_copy_(3, pos, kv.permute(2, 0, 3, 1, 4))

    def attend_self(self, i, q, table, nb, md, kv_len=None, seqlens=None, num_splits=0):
        return flash_decoding_with_fusing_bias(q, self.self_k[i], self.self_v[i], table, causal=True, sm_scale=1.0,
                                               NUM_BUCKETS=nb, MAX_DISTANCE=md, kv_len=kv_len, seqlens_k=seqlens,
                                               num_splits=num_splits, workspace=self.workspace)

    def attend_cross(self, i, q, seqlens=None):
        return flash_decoding_with_fusing_bias(q, self.cross_k[i], self.cross_v[i], None, causal=False, sm_scale=1.0,
                                               seqlens_k=seqlens, q_pos_offset=0, workspace=self.workspace)

    def reorder(self, parents, seqlens=None):
        """Let the self-attention rows follow their beams (`reorder_beam_cache`)."""
        reorder_beam_cache(self.self_kv, parents, seqlens=seqlens, scales=self.scales)


class QuantizedDecoderCache(DecoderCache):
    """A `DecoderCache` in 8 bits: float8_e4m3fn with a scale per 64 tokens and head, half of the memory and of the
    bytes that a step reads.  For 16-bit models."""

    def __init__(self, n_layers, batch, heads, d_kv, max_len, dtype, device, beams=1):
        if dtype not in _HALF:
            raise ValueError("an 8-bit cache belongs to a float16 or bfloat16 model, got %s" % dtype)
        if d_kv not in (16, 32, 64, 128):
            raise ValueError("an 8-bit cache takes head dims 16, 32, 64 and 128, got %d" % d_kv)
        blocks = -(-max_len // CACHE_BLOCK)
        super().__init__(n_layers, batch, heads, d_kv, blocks * CACHE_BLOCK, torch.float8_e4m3fn, device, beams)
        self.max_len = max_len
        self.scales = [torch.ones((2, batch * beams, heads, blocks), dtype=torch.float32, device=device)
                       for _ in range(n_layers)]
        self.cross_scales: List[Optional[torch.Tensor]] = [None] * n_layers
        self.cross_len = 0

    def set_cross(self, i, k, v, seqlens=None):
        B, H, N, D = k.shape
        blocks = max(1, -(-N // CACHE_BLOCK))
        kv = torch.empty((2, B, H, blocks * CACHE_BLOCK, D), dtype=torch.float8_e4m3fn, device=k.device)
        scale = torch.ones((2, B, H, blocks), dtype=torch.float32, device=k.device)
        quantize_into_cache(k, v, kv[0], scale[0], kv[1], scale[1], 0, seqlens=seqlens)
        self.cross_k[i], self.cross_v[i], self.cross_scales[i], self.cross_len = kv[0], kv[1], scale, N

    def append(self, i, k, v, start):
        s = self.scales[i]
        quantize_into_cache(k, v, self.self_k[i], s[0], self.self_v[i], s[1], start)

    def append_stacked(self, i, kv, pos):
        k, v = kv.transpose(1, 3).unbind(2)              # (B, H, 1, D) each
        self.append(i, k, v, pos)

    def attend_self(self, i, q, table, nb, md, kv_len=None, seqlens=None, num_splits=0):
        s = self.scales[i]
        return flash_decoding_quantized_with_fusing_bias(q, self.self_k[i], s[0], self.self_v[i], s[1], table, causal=True,
                                                         sm_scale=1.0, NUM_BUCKETS=nb, MAX_DISTANCE=md, kv_len=kv_len,
                                                         seqlens_k=seqlens)

    def attend_cross(self, i, q, seqlens=None):
        s = self.cross_scales[i]
        return flash_decoding_quantized_with_fusing_bias(q, self.cross_k[i], s[0], self.cross_v[i], s[1], None, sm_scale=1.0,
                                                         kv_len=self.cross_len, seqlens_k=seqlens, q_pos_offset=0)


def _cache_class(cache_dtype):
    if cache_dtype is None:
        return DecoderCache
    if cache_dtype == torch.float8_e4m3fn:
        return QuantizedDecoderCache
    raise ValueError("cache_dtype is None (the model's type) or torch.float8_e4m3fn, got %s" % cache_dtype)


class _NativeState:
    """What the native passes keep with a stack (stacked weights of the last `forward_fused`).  Copies and
    pickles of the module start without it."""

    def __init__(self):
        self.cache = _host.new_stack_cache()

    def __deepcopy__(self, memo):
        return _NativeState()

    def __reduce__(self):
        return _NativeState, ()


class T5Stack(nn.Module):
    def __init__(self, cfg: T5StackConfig, embed_tokens: nn.Embedding, is_decoder: bool):
        super().__init__()
        cfg = T5StackConfig(**{**cfg.__dict__, "is_decoder": is_decoder})
        self.cfg = cfg
        self.is_decoder = is_decoder
        self.embed_tokens = embed_tokens
        n = cfg.num_decoder_layers if is_decoder else cfg.num_layers
        self.block = nn.ModuleList([T5Block(cfg, has_relative_attention_bias=(i == 0)) for i in range(n)])
        self.final_layer_norm = T5LayerNorm(cfg.d_model, eps=cfg.layer_norm_epsilon)

    def _table(self):
        return self.block[0].layer[0].SelfAttention.relative_attention_bias.weight

    def forward(self, input_ids=None, attention_mask=None, inputs_embeds=None, encoder_hidden_states=None,
                encoder_attention_mask=None):
        """Full (uncached) pass.  `attention_mask` is the raw 0/1 (B, L) mask or None.

        A stack of 16-bit full-attention blocks runs as one native launch sequence (one autograd node in
        training); everything else (float32, block-local attention, replaced modules, hooks) runs
        module by module."""
        hidden = self.embed_tokens(input_ids) if inputs_embeds is None else inputs_embeds
        native = self._forward_native(hidden, attention_mask, encoder_hidden_states, encoder_attention_mask)
        if native is not None:
            return native
        table = self._table()
        for blk in self.block:
            sa = blk.layer[0]
            normed = sa.layer_norm(hidden).to(hidden.dtype)
            hidden = hidden + sa.SelfAttention(normed, mask=None if self.is_decoder else attention_mask,
                                               position_bias=table)[0]
            if self.is_decoder:
                ca = blk.layer[1]
                normed = ca.layer_norm(hidden).to(hidden.dtype)
                hidden = hidden + ca.EncDecAttention(normed, mask=encoder_attention_mask,
                                                     key_value_states=encoder_hidden_states)[0]
            hidden = blk.layer[-1](hidden)
        return self.final_layer_norm(hidden).to(hidden.dtype)

    def _forward_native(self, hidden, attention_mask, encoder_hidden_states, encoder_attention_mask):
        """`forward` as one launch sequence, or None when this call is not one it covers."""
        if self.is_decoder:
            if encoder_hidden_states is None or encoder_hidden_states.dim() != 3:
                return None
            if encoder_attention_mask is None:
                return self._run_native(hidden, enc=encoder_hidden_states)
            if encoder_attention_mask.dim() != 2 or not hidden.is_cuda:
                return None
            plan = get_unpad_plan(encoder_attention_mask)
            return self._run_native(hidden, enc=encoder_hidden_states, enc_cu=plan.cu_seqlens, enc_dest=plan.dest,
                                    enc_max=plan.seqlen)
        if attention_mask is None:
            return self._run_native(hidden)
        if attention_mask.dim() != 2 or not hidden.is_cuda:
            return None
        plan = get_unpad_plan(attention_mask)
        return self._run_native(hidden, mode=2, cu=plan.cu_seqlens, dest=plan.dest, max_len=plan.seqlen)

    def _run_native(self, x, mode=0, cu=None, dest=None, max_len=0, zero_tail=False, enc=None, enc_cu=None, enc_dest=None,
                    enc_max=0, need_plain=True):
        """One native pass over the rows x (B, S, d_model); modes as in csrc/host/stack.cpp.  None: not covered."""
        if not x.is_cuda or x.dtype not in _HALF or torch.is_autocast_enabled():
            return None
        if torch.nn.modules.module._has_any_global_hook():
            return None
        cfg = self.cfg
        return _host.stack_forward(self, _STACK_CLASSES, None if need_plain else self._native_cache(), self.is_decoder,
                                   cfg.num_heads, cfg.d_kv, cfg.relative_attention_num_buckets,
                                   cfg.relative_attention_max_distance, cfg.layer_norm_epsilon, need_plain, x, mode, cu,
                                   dest, max_len, zero_tail, enc, enc_cu, enc_dest, enc_max)

    # ---- inference pass of an encoder with the token-wise work fused around the attention path
    def _stacked_weights(self, i):
        """Per block: [q; k; v], [k; v], the cross-attention [k; v] and [wi_0; wi_1] weights stacked once,
        so each group is one matrix product.  Rebuilt when a parameter has been modified in place or
        replaced."""
        blk = self.block[i]
        att, ff = blk.layer[0].SelfAttention, blk.layer[-1].DenseReluDense
        gated = hasattr(ff, "wi_0")
        groups = dict(qkv=[att.q.weight, att.k.weight, att.v.weight], kv=[att.k.weight, att.v.weight])
        if self.is_decoder:
            catt = blk.layer[1].EncDecAttention
            groups["ckv"] = [catt.k.weight, catt.v.weight]
        if gated:
            groups["wi"] = [ff.wi_0.weight, ff.wi_1.weight]
        key = tuple((w.data_ptr(), w._version, w.dtype, w.device) for ws in groups.values() for w in ws)
        cache = self.__dict__.setdefault("_stacked", {})
        hit = cache.get(i)
        if hit is None or hit[0] != key:
            with torch.no_grad():
                cache[i] = hit = (key, {name: torch.cat(ws, 0) for name, ws in groups.items()})
        return hit[1]

    @torch.no_grad()
    def forward_fused(self, input_ids=None, inputs_embeds=None, seq_len=None, group=None, overlap=True, ops=None,
                      encoder_hidden_states=None, attention_mask=None, packed_rows=None, return_packed=False,
                      encoder_plan=None):
        """Forward pass without gradients, with the token-wise work fused around the attention path, as one
        native launch sequence where that covers the call and operator by operator otherwise: per encoder
        block eight launches -- stacked q/k/v projection,
        attention, output projection, residual add fused with the next RMSNorm, stacked wi_0|wi_1
        projection, gated GELU, wo projection, residual add + RMSNorm -- and five more per decoder
        block for the cross attention (q projection, stacked k/v projection of the encoder states,
        attention, output projection, residual add + RMSNorm).  Same arithmetic and rounding points
        as `forward` (the blocks of src/turbot5/model/modeling.py:124-128,142-164,166-219,221-342).

        With `seq_len` given the pass is sequence parallel (encoder stacks): `input_ids` /
        `inputs_embeds` hold this rank's token shard (B, S), S = ceil(seq_len / world), every
        token-wise operation runs on the shard, and each attention layer gathers the other ranks'
        keys and values (see `sequence_parallel_attention_overlapped`; `overlap=False` gathers first
        and attends once).  Returns the normed hidden states of the rows this call was given.
        With `attention_mask` (encoder stacks; the raw 0/1 (B, L) mask, right-padded) the valid tokens
        are packed ONCE, after the embedding: every projection, norm and feed-forward layer then runs
        on the packed rows only, the attention layers use the packed-sequence kernel, and the result is
        scattered back at the end (zeros at padded positions) -- where the reference unpads and pads
        around every attention call and does everything else on the padded batch
        (src/turbot5/model/attentions.py:405-470, model/padding.py:113-150).  `packed_rows` is an
        upper bound on the number of valid tokens known to the caller (e.g. from the tokenizer; with a bound
        below the true count the result is all NaN); without it the count is read back from the device once
        per call.
        `return_packed=True` skips the final scatter and returns (packed states (T, d_model), plan): a
        decoder stack takes them as `encoder_hidden_states` (2-D) with `encoder_plan=plan` and its cross
        attention then reads the packed keys directly (packed-sequence kernel, no bias), so the encoder
        output is never padded again.

        `ops` replaces the library operators (an object with rms_layer_norm, add_rms_layer_norm,
        gated_gelu, attention and the partial / merge pair of the sequence-parallel path): tests of
        the sharding logic on CPU ranks pass reference implementations.
        """
        if self.is_decoder and (encoder_hidden_states is None or seq_len is not None):
            raise ValueError("a decoder stack needs encoder_hidden_states and is not sequence parallel")
        if (encoder_plan is not None) != (encoder_hidden_states is not None and encoder_hidden_states.dim() == 2):
            raise ValueError("packed encoder states (T, d_model) go together with encoder_plan")
        if attention_mask is not None and (self.is_decoder or seq_len is not None):
            raise ValueError("attention_mask is taken by unsharded encoder stacks")
        for blk in self.block:
            if type(blk.layer[0].SelfAttention) is not T5FlashAttention:
                raise ValueError("forward_fused covers full attention (attention_type='flash')")
        if seq_len is not None or ops is not None:
            return self._forward_fused_ops(input_ids, inputs_embeds, seq_len, group, overlap, ops or _FusedOps,
                                           encoder_hidden_states, attention_mask, packed_rows, return_packed, encoder_plan)
        by_operators = lambda: self._forward_fused_ops(input_ids, inputs_embeds, None, None, False, _FusedOps,
                                                       encoder_hidden_states, attention_mask, packed_rows, return_packed,
                                                       encoder_plan)
        if attention_mask is not None:
            out = self._forward_fused_packed(input_ids, inputs_embeds, attention_mask, packed_rows, return_packed)
            return by_operators() if out is None else out
        x = self.embed_tokens(input_ids) if inputs_embeds is None else inputs_embeds
        if encoder_plan is None:
            out = self._run_native(x, enc=encoder_hidden_states, need_plain=False)
        else:
            # packed encoder states: every decoder sequence has S query rows, its keys are the valid
            # encoder tokens of the same batch row
            if encoder_plan.batch != x.shape[0]:
                raise ValueError("encoder_plan was made for another batch size")
            out = self._run_native(x, enc=encoder_hidden_states, enc_cu=encoder_plan.cu_seqlens, enc_max=encoder_plan.seqlen,
                                   need_plain=False)
        return by_operators() if out is None else out

    def _native_cache(self):
        state = self.__dict__.get("_native_state")
        if state is None:
            state = self.__dict__["_native_state"] = _NativeState()
        return state.cache

    def _forward_fused_packed(self, input_ids, inputs_embeds, attention_mask, packed_rows, return_packed):
        """The native encoder pass over the valid tokens of a padded batch, packed once; None: not covered."""
        plan = get_unpad_plan(attention_mask)
        B, L = plan.batch, plan.seqlen
        tail, cu = False, plan.cu_seqlens
        if packed_rows is None:
            # the valid tokens' ids (or rows) selected by the mask: the one read-back of the pass
            src = input_ids if inputs_embeds is None else inputs_embeds
            rows = src[attention_mask != 0]
            if rows.shape[0] == 0:
                rows, tail = src.flatten(0, 1)[:1], True
            x = self.embed_tokens(rows) if inputs_embeds is None else rows
        else:
            # With a caller's bound there may be rows past the last token.  The attention kernel does not
            # write them, and whatever the allocation held there must not reach a later matrix product
            # as the value row of a masked key (0 x NaN): the pass keeps them zero after attention.  No row past
            # the buffers is ever touched, whatever the bound: the attention calls see the sequences cut
            # at it (the result is then marked below).
            n = min(max(int(packed_rows), 1), B * L)
            x = self.embed_tokens(input_ids) if inputs_embeds is None else inputs_embeds
            x = unpad_rows(x, plan)[:n]                                    # kept tokens, zero tail
            tail, cu = True, plan.cu_seqlens.clamp(max=n)
        normed = self._run_native(x.unsqueeze(0), mode=1, cu=cu, max_len=L, zero_tail=tail, need_plain=False)
        if normed is None:
            return None
        return self._unpacked(normed[0], plan, packed_rows, return_packed)

    @staticmethod
    def _unpacked(normed, plan, packed_rows, return_packed):
        """Result of a packed pass from its rows (T, d_model)."""
        n, total = normed.shape[0], plan.batch * plan.seqlen
        if packed_rows is not None:
            # a bound below the true token count would silently drop tokens: make that loud (NaN
            # everywhere) without reading anything back
            normed = normed.masked_fill(plan.cu_seqlens[-1] > n, float("nan"))
        if return_packed:
            return normed, plan
        if packed_rows is not None and n < total:
            # the scatter reads the packed row of every valid token: give it all of them
            full = normed.new_full((total, normed.shape[-1]), float("nan"))
            full[:n] = normed
            normed = full
        return pad_rows(normed, plan)             # (B, L, d_model), zeros at padded positions

    def _forward_fused_ops(self, input_ids, inputs_embeds, seq_len, group, overlap, ops, encoder_hidden_states,
                           attention_mask=None, packed_rows=None, return_packed=False, encoder_plan=None):
        """The fused pass operator by operator: sequence-parallel encoders (a collective per layer), passes with
        other operators than the library's, and calls that the native pass does not take (autocast, norm weights
        or a bias table of another type than the matrices, weights that are not contiguous, replaced or hooked
        feed-forward layers)."""
        cfg = self.cfg
        x = self.embed_tokens(input_ids) if inputs_embeds is None else inputs_embeds
        plan = tail = None
        if attention_mask is not None:
            plan = get_unpad_plan(attention_mask)
            n = int(plan.cu_seqlens[-1]) if packed_rows is None else int(packed_rows)
            n = min(max(n, 1), plan.batch * plan.seqlen)
            x = unpad_rows(x, plan)[:n].unsqueeze(0)                  # (1, T, d_model): kept tokens, zero tail
            cu = plan.cu_seqlens
            if packed_rows is not None:
                # rows past the last token: as in `_forward_fused_packed`
                tail = (torch.arange(n, device=x.device) >= cu[-1])[:, None, None]
                cu = cu.clamp(max=n)
        B, S, _ = x.shape
        H, D = cfg.num_heads, cfg.d_kv
        HD = H * D
        nb, md = cfg.relative_attention_num_buckets, cfg.relative_attention_max_distance
        eps = cfg.layer_norm_epsilon
        table = self._table()
        heads = lambda t: t.unflatten(-1, (H, D)).transpose(1, 2)        # (B, L, H*D) -> (B, H, L, D) view
        x = x.contiguous() if (inputs_embeds is None or plan is not None) else x.clone(memory_format=torch.contiguous_format)
        normed = ops.rms_layer_norm(x, self.block[0].layer[0].layer_norm.weight, eps).to(x.dtype)
        if seq_len is not None:
            from . import sequence_parallel as sp
        if encoder_plan is not None:
            if encoder_plan.batch != B:
                raise ValueError("encoder_plan was made for another batch size")
            cu_dec = torch.arange(B + 1, dtype=torch.int32, device=x.device) * S
        for i, blk in enumerate(self.block):
            att, ffl = blk.layer[0].SelfAttention, blk.layer[-1]
            w = self._stacked_weights(i)
            if plan is not None:
                qkv = nn.functional.linear(normed, w["qkv"])[0]                           # (T, 3*H*D)
                q, k, v = (qkv[:, j * HD:(j + 1) * HD].unflatten(-1, (H, D)) for j in range(3))
                attn = flash_attention_with_fusing_bias_varlen(q, k, v, table, cu, cu, plan.seqlen, plan.seqlen,
                                                               causal=False, sm_scale=1.0, NUM_BUCKETS=nb, MAX_DISTANCE=md)
                if tail is not None:
                    attn = attn.masked_fill(tail, 0)
            elif seq_len is None:
                qkv = nn.functional.linear(normed, w["qkv"])
                q, k, v = (heads(qkv[..., j * HD:(j + 1) * HD]) for j in range(3))
                attn = ops.attention(q, k, v, table, self.is_decoder, 1.0, nb, md, 0).transpose(1, 2)
            else:
                q = nn.functional.linear(normed, att.q.weight).view(B, S, H, D)
                kv = nn.functional.linear(normed, w["kv"])
                if overlap:
                    attn = sp.sequence_parallel_attention_overlapped(q, kv, table, seq_len, sm_scale=1.0, NUM_BUCKETS=nb,
                                                                     MAX_DISTANCE=md, group=group, ops=ops)
                else:
                    k, v = kv[..., :HD].reshape(B, S, H, D), kv[..., HD:].reshape(B, S, H, D)
                    attn = sp.sequence_parallel_attention(
                        q, k, v, table, seq_len, sm_scale=1.0, NUM_BUCKETS=nb, MAX_DISTANCE=md, group=group,
                        attention_fn=lambda q_, k_, v_, b_, causal, sm_scale, NUM_BUCKETS, MAX_DISTANCE, q_pos_offset:
                        ops.attention(q_, k_, v_, b_, causal, sm_scale, NUM_BUCKETS, MAX_DISTANCE, q_pos_offset))
            o = nn.functional.linear(attn.reshape(B, S, HD), att.o.weight)
            if self.is_decoder:
                ca = blk.layer[1]
                x, normed = ops.add_rms_layer_norm(x, o, ca.layer_norm.weight, eps, inplace=True)
                catt = ca.EncDecAttention
                ckv = nn.functional.linear(encoder_hidden_states, w["ckv"])
                if encoder_plan is None:
                    q = heads(nn.functional.linear(normed, catt.q.weight))
                    attn = ops.attention(q, heads(ckv[..., :HD]), heads(ckv[..., HD:]), None, False, 1.0, nb, md, 0).transpose(1, 2)
                else:
                    # packed encoder states: every decoder sequence has S query rows, its keys are the valid
                    # encoder tokens of the same batch row
                    q = nn.functional.linear(normed, catt.q.weight).view(B * S, H, D)
                    attn = flash_attention_with_fusing_bias_varlen(
                        q, ckv[:, :HD].unflatten(-1, (H, D)), ckv[:, HD:].unflatten(-1, (H, D)), None, cu_dec,
                        encoder_plan.cu_seqlens, S, encoder_plan.seqlen, causal=False, sm_scale=1.0)
                o = nn.functional.linear(attn.reshape(B, S, HD), catt.o.weight)
            x, normed = ops.add_rms_layer_norm(x, o, ffl.layer_norm.weight, eps, inplace=True)
            ff = ffl.DenseReluDense
            if "wi" in w:
                f = nn.functional.linear(ops.gated_gelu(nn.functional.linear(normed, w["wi"])), ff.wo.weight)
            else:
                f = ff(normed)
            nxt = self.block[i + 1].layer[0].layer_norm if i + 1 < len(self.block) else self.final_layer_norm
            x, normed = ops.add_rms_layer_norm(x, f, nxt.weight, eps, inplace=True)
        return normed if plan is None else self._unpacked(normed[0], plan, packed_rows, return_packed)

    # ---- generation with a preallocated cache (decoder only)
    def new_cache(self, encoder_hidden_states, max_len, beams=1, cache_dtype=None, encoder_seqlens=None) -> DecoderCache:
        """A cache for `max_len` steps over these encoder states, in the model's type or (`cache_dtype`
        torch.float8_e4m3fn) in 8 bits; `beams` rows of self-attention per sentence.  `encoder_seqlens`: an 8-bit cache
        keeps only so many states of each sentence (a step that attends has to have these lengths or shorter ones)."""
        cfg = self.cfg
        B = encoder_hidden_states.shape[0]
        cache = _cache_class(cache_dtype)(len(self.block), B, cfg.num_heads, cfg.d_kv, max_len, encoder_hidden_states.dtype,
                                          encoder_hidden_states.device, beams)
        for i, blk in enumerate(self.block):
            att = blk.layer[1].EncDecAttention
            shape = lambda x: x.view(B, -1, cfg.num_heads, cfg.d_kv).transpose(1, 2)
            cache.set_cross(i, shape(att.k(encoder_hidden_states)), shape(att.v(encoder_hidden_states)), encoder_seqlens)
        return cache

    def decode_step_static(self, input_ids, cache: DecoderCache, pos, seqlens, encoder_seqlens=None):
        """One cached single-token step whose position lives on the device.

        `pos` (int64, shape (1,)) is the slot of the new token in the cache and `seqlens` (int32,
        shape (B,)) the number of cached keys including it; nothing in the launch sequence
        depends on their values, so the step can be captured once in a CUDA graph and replayed
        (the caller advances both tensors between replays).  Returns (B, 1, d_model).

        For 16-bit weights the step is fused like `forward_fused`: one stacked q|k|v projection, one
        copy that appends the new key and value to the cache, the split-KV kernel, the output
        projection, residual add + RMSNorm in one kernel -- thirteen launches per layer instead of
        twenty.

        With a cache of several beams, `input_ids` and `seqlens` have a row per beam and `encoder_seqlens` one per
        sentence.
        """
        cfg = self.cfg
        B = input_ids.shape[0]
        H, D = cfg.num_heads, cfg.d_kv
        HD = H * D
        nb, md = cfg.relative_attention_num_buckets, cfg.relative_attention_max_distance
        eps = cfg.layer_norm_epsilon
        hidden = self.embed_tokens(input_ids)
        table = self._table()
        fused = hidden.dtype in (torch.bfloat16, torch.float16) and cfg.d_model % 8 == 0
        shape = lambda x: x.view(B, 1, H, D).transpose(1, 2)
        # cross attention: the beams of a sentence are query rows over its keys
        K = cache.beams
        cross = shape if K == 1 else (lambda x: x.view(B // K, K, H, D).transpose(1, 2))
        # The split count of the self-attention launch comes from the cache CAPACITY, not from the
        # current length, so it is the same in every replay (a split beyond the cached keys is empty
        # and merges as such); a small batch then still fills the GPU late in a long generation.
        from . import _native as nat
        self_splits = max(1, nat.lib().t5b_decode_num_splits(B, H, cache.max_len))
        if fused:
            hidden = hidden.contiguous()
            normed = rms_layer_norm(hidden, self.block[0].layer[0].layer_norm.weight, eps)
        for i, blk in enumerate(self.block):
            sa, ca, ffl = blk.layer[0], blk.layer[1], blk.layer[-1]
            att, catt = sa.SelfAttention, ca.EncDecAttention
            if fused:
                w = self._stacked_weights(i)
                qkv = nn.functional.linear(normed, w["qkv"])                       # (B, 1, 3*H*D)
                q = shape(qkv[..., :HD])
                # new key and value -> slot `pos` of the stacked cache, one copy
                cache.append_stacked(i, qkv[..., HD:].view(B, 1, 2, H, D), pos)
            else:
                normed = sa.layer_norm(hidden).to(hidden.dtype)
                q = shape(att.q(normed))
                cache.append(i, shape(att.k(normed)), shape(att.v(normed)), pos)
            o = cache.attend_self(i, q, table, nb, md, seqlens=seqlens, num_splits=self_splits)
            o = att.o(o.transpose(1, 2).reshape(B, 1, HD))
            if fused:
                hidden, normed = add_rms_layer_norm(hidden, o, ca.layer_norm.weight, eps, inplace=True)
            else:
                hidden = hidden + o
                normed = ca.layer_norm(hidden).to(hidden.dtype)
            o = cache.attend_cross(i, cross(catt.q(normed)), encoder_seqlens)
            o = catt.o(o.transpose(1, 2).reshape(B, 1, HD))
            if fused:
                hidden, normed = add_rms_layer_norm(hidden, o, ffl.layer_norm.weight, eps, inplace=True)
                ff = ffl.DenseReluDense
                if "wi" in w:
                    f = nn.functional.linear(gated_gelu(nn.functional.linear(normed, w["wi"])), ff.wo.weight)
                else:
                    f = ff(normed)
                nxt = self.block[i + 1].layer[0].layer_norm if i + 1 < len(self.block) else self.final_layer_norm
                hidden, normed = add_rms_layer_norm(hidden, f, nxt.weight, eps, inplace=True)
            else:
                hidden = hidden + o
                hidden = ffl(hidden)
        return normed if fused else self.final_layer_norm(hidden).to(hidden.dtype)

    def decode_step(self, input_ids, cache: DecoderCache, encoder_seqlens=None):
        """One cached step for `input_ids` (B, M) (M new tokens, usually 1); returns (B, M, d_model).  Over an 8-bit cache
        every eight tokens read it again: for long prompts (hundreds of tokens) a 16-bit one is the faster."""
        cfg = self.cfg
        B, M = input_ids.shape
        H, D = cfg.num_heads, cfg.d_kv
        t0 = cache.length
        if t0 + M > cache.max_len:
            raise ValueError("decoder cache is full")
        if cache.beams != 1:
            raise ValueError("a cache of several beams belongs to decode_step_static")
        quantized = isinstance(cache, QuantizedDecoderCache)
        hidden = self.embed_tokens(input_ids)
        table = self._table()
        shape = lambda x: x.view(B, M, H, D).transpose(1, 2)
        for i, blk in enumerate(self.block):
            sa, ca = blk.layer[0], blk.layer[1]
            att = sa.SelfAttention
            normed = sa.layer_norm(hidden).to(hidden.dtype)
            q = shape(att.q(normed))
            cache.append(i, shape(att.k(normed)), shape(att.v(normed)), t0)
            if M <= att.decode_max_rows or quantized:
                o = cache.attend_self(i, q, table, cfg.relative_attention_num_buckets, cfg.relative_attention_max_distance,
                                      kv_len=t0 + M)
            else:
                o = flash_attention_with_fusing_bias(q, cache.self_k[i][:, :, :t0 + M], cache.self_v[i][:, :, :t0 + M],
                                                     table, causal=True, sm_scale=1.0,
                                                     NUM_BUCKETS=cfg.relative_attention_num_buckets,
                                                     MAX_DISTANCE=cfg.relative_attention_max_distance)
            hidden = hidden + att.o(o.transpose(1, 2).reshape(B, M, H * D))
            catt = ca.EncDecAttention
            normed = ca.layer_norm(hidden).to(hidden.dtype)
            q = shape(catt.q(normed))
            if M <= catt.decode_max_rows or quantized:
                o = cache.attend_cross(i, q, encoder_seqlens)
            else:
                o = flash_attention_with_fusing_bias(q, cache.cross_k[i], cache.cross_v[i], None, causal=False,
                                                     sm_scale=1.0, q_pos_offset=0)
            hidden = hidden + catt.o(o.transpose(1, 2).reshape(B, M, H * D))
            hidden = blk.layer[-1](hidden)
        cache.length = t0 + M
        return self.final_layer_norm(hidden).to(hidden.dtype)


# the classes of a plain stack, in the order of `Kind` in csrc/host/stack.cpp
_STACK_CLASSES = (T5Block, nn.ModuleList, T5LayerSelfAttention, T5LayerCrossAttention, T5LayerFF, T5FlashAttention,
                  T5LayerNorm, nn.Linear, T5DenseGatedActDense, T5DenseActDense, nn.Embedding)


def _native_decoding(model, encoder_hidden_states, max_len, encoder_seqlens=None):
    """A native decoding session for this model (caches, projected cross keys, one launch chain per token:
    csrc/decoder_step.cu), or None when the step kernels do not cover it: float32, more than 64 rows, replaced
    modules or hooks, sizes they do not take."""
    dec, head, emb, cfg = model.decoder, model.lm_head, model.decoder.embed_tokens, model.cfg
    plain = lambda m: not (m._forward_hooks or m._forward_pre_hooks or "forward" in m.__dict__)
    if type(model).logits is not T5ForConditionalGeneration.logits or "logits" in model.__dict__ or type(dec) is not T5Stack or \
            type(head) is not nn.Linear or type(emb) is not nn.Embedding or head.bias is not None or \
            emb.max_norm is not None or not (plain(head) and plain(emb) and plain(dec)) or \
            torch.nn.modules.module._has_any_global_hook() or torch.is_autocast_enabled() or \
            not encoder_hidden_states.is_cuda or encoder_hidden_states.dtype not in _HALF:
        return None
    scale = cfg.d_model ** -0.5 if cfg.tie_word_embeddings else 1.0
    return _host.new_decode_session(dec, _STACK_CLASSES, cfg.num_heads, cfg.d_kv,
                                    cfg.relative_attention_num_buckets, cfg.relative_attention_max_distance,
                                    cfg.layer_norm_epsilon, encoder_hidden_states, encoder_seqlens, max_len, head.weight,
                                    emb.weight, scale, cfg.decoder_start_token_id)


class GraphedDecoding:
    """Greedy generation whose single-token step is one CUDA graph; `cache_dtype` torch.float8_e4m3fn keeps the
    keys and values in 8 bits.

    The step (all decoder layers, LM head, argmax, token write-back, position update) is run
    once eagerly on a side stream (cuBLAS handles and stacked weights then exist), rewound,
    captured, and rewound again; `step()` then replays it.  Where the native step kernels cover the
    model the captured step is their launch chain; otherwise it is `decode_step_static`, whose split
    scratch is kept per stream: the capture stream gets its own, allocated and zeroed inside the
    graph's memory pool during capture.  The token position and the cached
    length live in device tensors that the graph itself advances, so no launch argument
    changes between replays.
    """

    def __init__(self, model, encoder_hidden_states, max_len, encoder_seqlens=None, cache_dtype=None):
        B = encoder_hidden_states.shape[0]
        dev = encoder_hidden_states.device
        self.model = model
        self.max_len = max_len
        self.steps_done = 0
        self.encoder_seqlens = encoder_seqlens
        with torch.no_grad():
            self.session = None
            if cache_dtype is None:
                self.session = _native_decoding(model, encoder_hidden_states, max_len, encoder_seqlens)
        if self.session is not None:
            self.tokens, self.last_logits = _host.decode_session_tensors(self.session)
        else:
            with torch.no_grad():
                self.cache = model.decoder.new_cache(encoder_hidden_states, max_len, cache_dtype=cache_dtype,
                                                     encoder_seqlens=encoder_seqlens)
            self.cur = torch.empty((B, 1), dtype=torch.long, device=dev)
            self.pos = torch.empty(1, dtype=torch.long, device=dev)
            self.seqlens = torch.empty(B, dtype=torch.int32, device=dev)
            self.tokens = torch.zeros((B, max_len), dtype=torch.long, device=dev)
        self.rewind()
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side), torch.no_grad():
            self._step()
        torch.cuda.current_stream(dev).wait_stream(side)
        self.rewind()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph), torch.no_grad():
            self.last_logits = self._step()
        self.rewind()

    def rewind(self):
        if self.session is not None:
            _host.decode_session_rewind(self.session)
        else:
            self.cur.fill_(self.model.cfg.decoder_start_token_id)
            self.pos.zero_()
            self.seqlens.fill_(1)
        self.steps_done = 0

    def _step(self):
        if self.session is not None:
            _host.decode_session_run(self.session, 1)
            return self.last_logits
        m = self.model
        logits = m.logits(m.decoder.decode_step_static(self.cur, self.cache, self.pos, self.seqlens,
                                                       self.encoder_seqlens))
        nxt = logits[:, -1:].argmax(-1)
        self.tokens.index_copy_(1, self.pos, nxt)
        self.cur.copy_(nxt)
        self.pos.add_(1)
        self.seqlens.add_(1)
        return logits

    def step(self):
        if self.steps_done >= self.max_len:
            raise RuntimeError("the cache is full: %d steps" % self.max_len)
        self.graph.replay()
        self.steps_done += 1


class BeamDecoding:
    """Beam search over a preallocated cache; the step is one CUDA graph (`use_cuda_graph=False`: launched one by one).

    A step runs the decoder on a row per beam (the beams of a sentence read its encoder keys together), the LM head,
    `beam_search_step` and `reorder_beam_cache`; positions, lengths, scores, the pool of finished sentences and the
    history of tokens and parents live on the device.  `cache_dtype` torch.float8_e4m3fn keeps keys and values in 8 bits.
    `sequences()` reads the best sentences back from the history at any time.
    """

    def __init__(self, model, encoder_hidden_states, max_len, num_beams, encoder_seqlens=None, length_penalty=1.0,
                 early_stopping=False, cache_dtype=None, use_cuda_graph=True):
        if not 1 <= num_beams <= MAX_BEAMS:
            raise ValueError("between 1 and %d beams, got %d" % (MAX_BEAMS, num_beams))
        if max_len < 1:
            raise ValueError("at least one step, got %d" % max_len)
        B, dev = encoder_hidden_states.shape[0], encoder_hidden_states.device
        self.model, self.max_len, self.batch, self.beams = model, max_len, B, num_beams
        self.encoder_seqlens = encoder_seqlens
        self.options = dict(eos_token_id=model.cfg.eos_token_id, pad_token_id=model.cfg.pad_token_id,
                            length_penalty=length_penalty)
        self.early_stopping = early_stopping
        with torch.no_grad():
            self.cache = model.decoder.new_cache(encoder_hidden_states, max_len, num_beams, cache_dtype, encoder_seqlens)
        if cache_dtype is None:
            self.cache.own_workspace()
        shape = (B, num_beams)
        self.cur = torch.empty(shape, dtype=torch.long, device=dev)
        self.parents = torch.empty(shape, dtype=torch.int32, device=dev)
        self.scores = torch.empty(shape, dtype=torch.float32, device=dev)
        self.finished_scores = torch.empty(shape, dtype=torch.float32, device=dev)
        self.finished_steps = torch.empty(shape, dtype=torch.int32, device=dev)
        self.finished_beams = torch.empty(shape, dtype=torch.int32, device=dev)
        self.done = torch.empty(B, dtype=torch.bool, device=dev)
        self.history = tuple(torch.empty((max_len, *shape), dtype=torch.int32, device=dev) for _ in range(2))
        self.pos = torch.empty(1, dtype=torch.long, device=dev)
        self.seqlens = torch.empty(B * num_beams, dtype=torch.int32, device=dev)
        self.graph = None
        self.rewind()
        if use_cuda_graph:
            with torch.cuda.device(dev):
                side = torch.cuda.Stream(dev)
                side.wait_stream(torch.cuda.current_stream(dev))
                with torch.cuda.stream(side), torch.no_grad():
                    self._step()                         # library handles and stacked weights exist from here on
                torch.cuda.current_stream(dev).wait_stream(side)
                self.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self.graph), torch.no_grad():
                    self._step()
            self.rewind()

    def rewind(self):
        """Back to the start of the search."""
        self.cur.fill_(self.model.cfg.decoder_start_token_id)
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0.0                          # the first step goes on from one beam of each sentence
        self.finished_scores.fill_(float("-inf"))
        for t in (self.finished_steps, self.finished_beams, self.done, self.pos):
            t.zero_()
        self.seqlens.fill_(1)
        self.steps_done = 0

    def _step(self):
        m = self.model
        hidden = m.decoder.decode_step_static(self.cur.view(-1, 1), self.cache, self.pos, self.seqlens, self.encoder_seqlens)
        state = (self.scores, self.finished_scores, self.finished_steps, self.finished_beams, self.done)
        beam_search_step(m.logits(hidden), *state, self.pos, early_stopping=self.early_stopping,
                         out=(self.cur, self.parents, *state), history=self.history, **self.options)
        self.cache.reorder(self.parents, self.seqlens)
        self.pos.add_(1)
        self.seqlens.add_(1)

    def step(self):
        if self.steps_done >= self.max_len:
            raise RuntimeError("the cache is full: %d steps" % self.max_len)
        if self.graph is not None:
            self.graph.replay()
        else:
            with torch.no_grad():
                self._step()
        self.steps_done += 1

    def sequences(self, num_return_sequences=1):
        """(ids (batch, num_return_sequences, steps done), scores) of the best sentences so far."""
        if self.steps_done == 0:
            raise RuntimeError("no step has been made")
        tokens, parents = (h[:self.steps_done] for h in self.history)
        return beam_search_sequences(tokens, parents, self.scores, self.finished_scores, self.finished_steps,
                                     self.finished_beams, self.done, num_return_sequences=num_return_sequences,
                                     **self.options)


class GraphedForward:
    """A whole teacher-forced forward pass (encoder, decoder, LM head) of fixed shapes as one CUDA graph.

    At small batches the pass is a few hundred short kernels and the host's launch rate, not the
    GPU, sets its duration (twelve decoder layers over 4 x 128 tokens: 4.4 ms of launches for well
    under 2 ms of work).  The pass is run once on a side stream (cuBLAS handles, stacked weights
    and the library's per-stream scratch then exist), captured, and replayed by `__call__`, which
    copies the token ids into the graph's input buffers and returns the graph's logits buffer (a
    static tensor: it is overwritten by the next call).  Inference only, unpadded inputs.
    """

    def __init__(self, model, batch, enc_len, dec_len, device=None):
        dev = torch.device(device) if device is not None else model.shared.weight.device
        self.model = model
        self.input_ids = torch.zeros((batch, enc_len), dtype=torch.long, device=dev)
        self.decoder_input_ids = torch.zeros((batch, dec_len), dtype=torch.long, device=dev)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side), torch.no_grad():
            model(self.input_ids, self.decoder_input_ids)
        torch.cuda.current_stream(dev).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph), torch.no_grad():
            self.logits = model(self.input_ids, self.decoder_input_ids)

    def __call__(self, input_ids, decoder_input_ids):
        if input_ids.shape != self.input_ids.shape or decoder_input_ids.shape != self.decoder_input_ids.shape:
            raise ValueError("GraphedForward was captured for ids of shapes %s and %s" %
                             (tuple(self.input_ids.shape), tuple(self.decoder_input_ids.shape)))
        self.input_ids.copy_(input_ids, non_blocking=True)
        self.decoder_input_ids.copy_(decoder_input_ids, non_blocking=True)
        self.graph.replay()
        return self.logits


class T5ForConditionalGeneration(nn.Module):
    def __init__(self, cfg: T5StackConfig):
        super().__init__()
        self.cfg = cfg
        self.shared = nn.Embedding(cfg.vocab_size, cfg.d_model)
        self.encoder = T5Stack(cfg, self.shared, is_decoder=False)
        self.decoder = T5Stack(cfg, self.shared, is_decoder=True)
        self.lm_head = nn.Linear(cfg.d_model, cfg.vocab_size, bias=False)

    def logits(self, decoder_hidden):
        if self.cfg.tie_word_embeddings:
            decoder_hidden = decoder_hidden * (self.cfg.d_model ** -0.5)
        return self.lm_head(decoder_hidden)

    def forward(self, input_ids, decoder_input_ids, attention_mask=None):
        if not torch.is_grad_enabled() and self.cfg.attention_type == "flash" and \
                input_ids.is_cuda and self.shared.weight.dtype in (torch.bfloat16, torch.float16):
            # inference: fused token-wise kernels in both stacks; a padded batch is packed once and the
            # decoder's cross attention reads the packed encoder states
            if attention_mask is None:
                enc = self.encoder.forward_fused(input_ids)
                return self.logits(self.decoder.forward_fused(decoder_input_ids, encoder_hidden_states=enc))
            enc, plan = self.encoder.forward_fused(input_ids, attention_mask=attention_mask, return_packed=True)
            return self.logits(self.decoder.forward_fused(decoder_input_ids, encoder_hidden_states=enc,
                                                          encoder_plan=plan))
        if attention_mask is not None:
            dec = self._packed_training_pass(input_ids, decoder_input_ids, attention_mask)
            if dec is not None:
                return self.logits(dec)
        enc = self.encoder(input_ids, attention_mask=attention_mask)
        dec = self.decoder(decoder_input_ids, encoder_hidden_states=enc, encoder_attention_mask=attention_mask)
        return self.logits(dec)

    def _packed_training_pass(self, input_ids, decoder_input_ids, attention_mask):
        """Decoder states of a padded batch in training: the valid tokens are packed once (padded rows get no
        gradient and give none), both stacks run as native passes and the cross attention reads the packed
        encoder states.  None when the stacks are not ones the native passes cover, and where nothing may be read
        back from the device (a capture, the synchronisation check): the padded passes read nothing back."""
        enc, dec = self.encoder, self.decoder
        if not input_ids.is_cuda or self.shared.weight.dtype not in _HALF or self.cfg.attention_type != "flash" or \
                attention_mask.shape != input_ids.shape or \
                any(type(m) is not T5Stack or "forward" in m.__dict__ or m._forward_hooks or m._forward_pre_hooks or
                    m._backward_hooks or m._backward_pre_hooks for m in (enc, dec)):
            return None
        if torch.cuda.is_current_stream_capturing() or torch.cuda.get_sync_debug_mode():
            return None                                  # packing reads the token count back: not here
        ids = input_ids[attention_mask != 0]             # the one read-back of the pass
        if ids.shape[0] == 0:
            return None
        plan = get_unpad_plan(attention_mask)
        states = enc._run_native(enc.embed_tokens(ids).unsqueeze(0), mode=1, cu=plan.cu_seqlens, max_len=plan.seqlen)
        if states is None:
            return None
        return dec._run_native(dec.embed_tokens(decoder_input_ids), enc=states[0], enc_cu=plan.cu_seqlens, enc_max=plan.seqlen)

    @torch.no_grad()
    def forward_cuda_graph(self, input_ids, decoder_input_ids):
        """`forward` for unpadded inference inputs through a CUDA graph kept per input shape (captured on
        first use; the returned logits live in the graph's buffer until the next call with that shape)."""
        key = (tuple(input_ids.shape), tuple(decoder_input_ids.shape), input_ids.device)
        graphs = self.__dict__.setdefault("_forward_graphs", {})
        if key not in graphs:
            graphs[key] = GraphedForward(self, input_ids.shape[0], input_ids.shape[1], decoder_input_ids.shape[1],
                                         input_ids.device)
        return graphs[key](input_ids, decoder_input_ids)

    @torch.no_grad()
    def generate(self, input_ids, attention_mask=None, max_new_tokens=32, use_cuda_graph=True, num_beams=1,
                 length_penalty=1.0, early_stopping=False, num_return_sequences=1, cache_dtype=None):
        """Generation for a (padded) batch of prompts: the encoder pass on the packed valid tokens
        (`forward_fused`), the cross-attention keys and values projected once into the preallocated cache,
        then one captured single-token step per new token.  Greedy, or with `num_beams` > 1 the best sentence of a beam
        search (`beam_search`, which takes the options after it).  `cache_dtype` torch.float8_e4m3fn keeps keys and values
        in 8 bits.  Returns the generated ids (B, max_new_tokens); (B, num_return_sequences, max_new_tokens) with more than
        one sentence."""
        if num_beams < 1:
            raise ValueError("between 1 and %d beams, got %d" % (MAX_BEAMS, num_beams))
        if num_beams == 1 and num_return_sequences != 1:
            raise ValueError("greedy generation has one sentence to return")
        fused = self.cfg.attention_type == "flash" and input_ids.is_cuda and \
            self.shared.weight.dtype in (torch.bfloat16, torch.float16)
        seqlens = None
        if attention_mask is not None:
            seqlens = attention_mask.to(torch.int32).sum(-1).to(torch.int32)
        if fused:
            enc = self.encoder.forward_fused(input_ids, attention_mask=attention_mask)
        else:
            enc = self.encoder(input_ids, attention_mask=attention_mask)
        if num_beams > 1:
            tokens, _ = self.beam_search(enc, max_new_tokens, num_beams, encoder_seqlens=seqlens, length_penalty=length_penalty,
                                         early_stopping=early_stopping, num_return_sequences=num_return_sequences,
                                         cache_dtype=cache_dtype, use_cuda_graph=use_cuda_graph)
            return tokens[:, 0] if num_return_sequences == 1 else tokens
        tokens, _ = self.greedy_decode(enc, max_new_tokens, encoder_seqlens=seqlens, use_cuda_graph=use_cuda_graph,
                                       cache_dtype=cache_dtype)
        return tokens

    @torch.no_grad()
    def beam_search(self, encoder_hidden_states, steps, num_beams, encoder_seqlens=None, length_penalty=1.0,
                    early_stopping=False, num_return_sequences=1, cache_dtype=None, use_cuda_graph=True):
        """Beam search from `decoder_start_token_id` (`BeamDecoding`): (ids (B, num_return_sequences, steps), scores
        (B, num_return_sequences)), best first, `pad_token_id` behind the end of a sentence.  A sentence's score is its
        log-probability over its length to the power of `length_penalty`; `early_stopping` ends a search as soon as
        num_beams sentences are finished.  Whether all searches have ended is looked up every 16 steps.  Capturing the step's
        graph takes as long as four to six steps launched one by one save (a 12-layer model)."""
        if not 1 <= num_return_sequences <= num_beams:
            raise ValueError("between 1 and num_beams = %d sentences, got %d" % (num_beams, num_return_sequences))
        search = BeamDecoding(self, encoder_hidden_states, steps, num_beams, encoder_seqlens, length_penalty, early_stopping,
                              cache_dtype, use_cuda_graph)
        for t in range(steps):
            search.step()
            if t % 16 == 15 and bool(search.done.all()):
                break
        tokens, scores = search.sequences(num_return_sequences)
        return nn.functional.pad(tokens, (0, steps - tokens.shape[-1]), value=self.cfg.pad_token_id), scores

    @torch.no_grad()
    def greedy_decode(self, encoder_hidden_states, steps, encoder_seqlens=None, use_cuda_graph=False, cache_dtype=None):
        """Greedy generation from `decoder_start_token_id` with the preallocated cache.

        Where the native step kernels cover the model (16-bit plain stacks, up to 64 rows, a cache in the model's
        type) every token is one native launch chain.  Otherwise, with `use_cuda_graph`, the whole single-token step
        (all layers, LM head, argmax, position update) is captured once after a warm-up step and replayed: one graph
        launch per token instead of a few hundred kernel launches issued from Python.  `cache_dtype`
        torch.float8_e4m3fn keeps keys and values in 8 bits.
        """
        session = None
        if cache_dtype is None:
            session = _native_decoding(self, encoder_hidden_states, steps, encoder_seqlens)
        if session is not None:
            _host.decode_session_run(session, steps)
            return _host.decode_session_tensors(session)
        if use_cuda_graph:
            session = GraphedDecoding(self, encoder_hidden_states, steps, encoder_seqlens, cache_dtype)
            for _ in range(steps):
                session.step()
            return session.tokens, session.last_logits
        B = encoder_hidden_states.shape[0]
        cache = self.decoder.new_cache(encoder_hidden_states, steps, cache_dtype=cache_dtype,
                                       encoder_seqlens=encoder_seqlens)
        cur = torch.full((B, 1), self.cfg.decoder_start_token_id, dtype=torch.long, device=encoder_hidden_states.device)
        tokens, last_logits = [], None
        for _ in range(steps):
            last_logits = self.logits(self.decoder.decode_step(cur, cache, encoder_seqlens))
            cur = last_logits[:, -1:].argmax(-1)
            tokens.append(cur)
        return torch.cat(tokens, dim=1), last_logits
