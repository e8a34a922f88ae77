"""Device state of one decode request.

Field-for-field the reference's Globals dataclass
(qimeng_megakernel/models/LLM/llama/llama3_2__1b/A100/single_batch/decode_schedule/globs.py:8-41):
same names, shapes, dtypes and layouts (Q/K weight rows and the K cache in the interleaved RoPE
layout, rope tables fp32 interleaved).  `instructions`, `barriers` and the split-KV intermediates stay
None: the B200 kernel owns its scheduler, counters and scratch.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch


@dataclass
class Globals:
    instructions: Optional[torch.Tensor] = None
    barriers: Optional[torch.Tensor] = None
    position_id: Optional[int] = None

    attn_norm_weights: Optional[torch.Tensor] = None     # [L, H]
    qkv_weights: Optional[torch.Tensor] = None           # [L, (NH+2NKV)*HD, H]
    rope_cos: Optional[torch.Tensor] = None              # [max_pos, HD] fp32
    rope_sin: Optional[torch.Tensor] = None
    o_proj_weights: Optional[torch.Tensor] = None        # [L, H, NH*HD]
    mlp_norm_weights: Optional[torch.Tensor] = None      # [L, H]
    up_proj_weights: Optional[torch.Tensor] = None       # [L, I, H]
    gate_proj_weights: Optional[torch.Tensor] = None     # [L, I, H]
    down_proj_weights: Optional[torch.Tensor] = None     # [L, H, I]
    lm_head_norm_weights: Optional[torch.Tensor] = None  # [H]
    lm_head_weights: Optional[torch.Tensor] = None       # [V, H]
    embed_tokens: Optional[torch.Tensor] = None          # [V, H] (tied to lm_head_weights for Llama-3.2-1B)

    k_cache: Optional[torch.Tensor] = None               # [L, B, S, NKV, HD]
    v_cache: Optional[torch.Tensor] = None
    hidden_states: Optional[torch.Tensor] = None         # [H]
    q_post_rope: Optional[torch.Tensor] = None           # [NH*HD]
    attn_out: Optional[torch.Tensor] = None              # [NH*HD]
    attn_out_intermediates: Optional[torch.Tensor] = None
    attn_lse_intermediates: Optional[torch.Tensor] = None
    silu_out: Optional[torch.Tensor] = None              # [I]
    logits: Optional[torch.Tensor] = None                # [V]

    # multi-batch fields of the reference (llama3_2__1b/A100/multi_batch/decode_schedule/globs.py:13-26); with B > 1
    # the state tensors above gain a leading [B] dimension
    position_ids: Optional[torch.Tensor] = None          # int32 [B]
    kv_lengths: Optional[torch.Tensor] = None
    active_mask: Optional[torch.Tensor] = None           # uint8 / bool [B]
    # B200 addition: the KV-cache sequence every row of the step belongs to (int32 [rows]); with it the rows may be
    # consecutive positions of one sequence (prefill) and the state tensors have `rows` rows while the cache has B sequences
    kv_slots: Optional[torch.Tensor] = None
    # B200 addition: a paged KV cache whose sequences share a prefix (paged.PagedState); k_cache / v_cache are then the pools
    # [L, num_pages, page_size, NKV, HD], and position_ids, active_mask and kv_slots are the buffers of the state's steps
    paged: Optional[object] = None
    # Qwen3 (qwen3__0_6b/A100/single_batch/decode_schedule/globs.py): per-head Q/K norm gains, interleaved order
    q_norm_weights: Optional[torch.Tensor] = None        # [L, HD]
    k_norm_weights: Optional[torch.Tensor] = None        # [L, HD]

    # MoE (qwen1_5_moe_a2_7b/A100/single_batch/decode_schedule/globs.py:30-34; no shared expert on this route)
    router_weights: Optional[torch.Tensor] = None                 # [L, E, H]
    expert_gate_up_proj_weights: Optional[torch.Tensor] = None    # [L, E, 2*Ie, H], gate rows then up rows
    expert_down_proj_weights: Optional[torch.Tensor] = None       # [L, E, H, Ie]

    # B200 additions (optional): device-resident greedy loop
    next_token: Optional[torch.Tensor] = None            # int64 [B], argmax of the last step
    token_in: Optional[torch.Tensor] = None              # int64 [B]; when set the kernel embeds it itself
    out_tokens: Optional[torch.Tensor] = None            # int64 [n] ([B, n]); kernel stores argmax at [pos+1]
