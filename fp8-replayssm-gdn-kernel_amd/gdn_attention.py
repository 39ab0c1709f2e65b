"""The full-attention layers between a hybrid model's GDN layers: their entry
(head norms, position rotation, append to a paged cache) and attention of new
tokens over that cache.

The reference leaves these layers to vLLM; its models interleave them with the
GDN layers this package serves, so a program that prefills and decodes such a
model through this package needs both. Kernels run on torch's current stream;
nothing synchronises.
"""

from __future__ import annotations

import torch

import gdnr_lib
from gdn_replayssm_fp8_kernel import _as_f32, _as_i32

__all__ = ["rope_table", "qkv_norm_rope_append", "paged_attention"]

_APPEND = gdnr_lib.ENTRY_IDS["gdnr_qkv_norm_rope_append"]
_ATTENTION = gdnr_lib.ENTRY_IDS["gdnr_paged_attention"]
_APPEND_NAMES = ("q", "k", "v", "q_weight", "k_weight", "cos_sin", "positions", "k_cache", "v_cache", "slot_mapping",
                 "q_out")
_ATTENTION_NAMES = ("q", "k_cache", "v_cache", "block_table", "cu_seqlens", "context_lens", "out", "workspace")


def rope_table(positions: int, rotary_dim: int, base: float = 10000.0, device="cuda",
               inv_freq: torch.Tensor | None = None, scale: float = 1.0) -> torch.Tensor:
    """cos_sin [positions, rotary_dim] (cosines, then sines) of the angles
    p * base ** (-2i / rotary_dim). A model whose long contexts scale the
    frequencies passes its own inv_freq [rotary_dim / 2], and scale multiplies
    both halves (the attention factor some of them carry). Angles are formed in
    float64."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    if inv_freq is None:
        inv_freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if tuple(inv_freq.shape) != (rotary_dim // 2,):
        raise ValueError("inv_freq must be [rotary_dim / 2]")
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv_freq.double().cpu()
    return (torch.cat([angle.cos(), angle.sin()], dim=-1) * scale).float().to(device)


def qkv_norm_rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos_sin: torch.Tensor,
    positions: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """q [T, HQ, D], k and v [T, HKV, D] (views of one row buffer are taken as
    they are) into an attention layer: RMS norm of every q and k head (with a
    weight [D], read as float32), rotation of the first cos_sin.shape[1]
    elements by the row positions[t] of cos_sin (rope_table; pairs half the
    width apart, or neighbours when interleaved), k and v to slot
    slot_mapping[t] (page * page_size + offset; negative: not appended) of
    k_cache and v_cache [pages, page_size, HKV, D]. Returns q_out [T, HQ, D]."""
    host = gdnr_lib.host()
    host.require(_APPEND_NAMES, (q, k, v, q_weight, k_weight, cos_sin, positions, k_cache, v_cache, slot_mapping, q_out))
    if q_out is None:
        q_out = host.empty(q, tuple(q.shape))
    host.call(_APPEND, (q, k, v, None if q_weight is None else _as_f32(q_weight),
                        None if k_weight is None else _as_f32(k_weight), cos_sin, _as_i32(positions), k_cache, v_cache,
                        _as_i32(slot_mapping), q_out), (int(bool(interleaved)),), (eps,), None)
    return q_out


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    context_lens: torch.Tensor,
    max_context: int | None = None,
    out: torch.Tensor | None = None,
    scale: float | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of new tokens over a paged cache. Sequence n owns rows
    cu_seqlens[n]:cu_seqlens[n+1] of q [T, HQ, D]; its context_lens[n] keys, the
    new tokens' last, lie in the pages block_table[n, :]. Token j of L new ones
    sees keys 0 .. context - L + j (none: it returns zeros). max_context, a host
    bound of context_lens, defaults to what block_table's width holds and sizes
    the launch; scale defaults to D ** -0.5. workspace: a uint8 tensor of at
    least gdnr_lib.paged_attention_workspace(...) bytes (allocated when not
    given)."""
    host = gdnr_lib.host()
    host.require(_ATTENTION_NAMES, (q, k_cache, v_cache, block_table, cu_seqlens, context_lens, out, workspace))
    if q.dim() != 3 or k_cache.dim() != 4 or block_table.dim() != 2:
        raise ValueError("q must be [T, HQ, D], k_cache [pages, page_size, HKV, D] and block_table [N, width]")
    tokens, heads, dim = q.shape
    if max_context is None:
        max_context = block_table.shape[1] * k_cache.shape[1]
    if out is None:
        out = host.empty(q, (tokens, heads, dim))
    if workspace is None:
        size = gdnr_lib.paged_attention_workspace(tokens, block_table.shape[0], heads, k_cache.shape[2], dim, max_context)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    host.call(_ATTENTION, (q, k_cache, v_cache, _as_i32(block_table), _as_i32(cu_seqlens), _as_i32(context_lens), out,
                           workspace), (int(max_context),), (dim ** -0.5 if scale is None else scale,), None)
    return out
