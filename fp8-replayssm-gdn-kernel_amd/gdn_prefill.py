"""Prefill of gated delta-rule (GDN) layers: the recurrence over packed
sequences of any length, in the production operator's contract.

What the decode step (gdn_replayssm_fp8_kernel) and its slot cache start from:
a prompt's outputs and the state after its last token. Also the form for a few
tokens at once (drafted tokens to verify, a prompt's short tail). The
recurrence is the reference's run_kernel
(prototype/gdn_replay_fp8_reference.py:137-163) on the raw rows of
prototype/gdn_replayssm_fp8_kernel.py:500-562; the reference has no kernel
for more than one token (its prompts run in vLLM).

Kernels run on torch's current stream; nothing synchronises.
"""

from __future__ import annotations

import torch

import gdnr_lib
from gdn_replayssm_fp8_kernel import _as_f32, _as_flag, _as_i32

__all__ = ["gdn_prefill"]

_PREFILL = gdnr_lib.ENTRY_IDS["gdnr_prefill"]
_NAMES = ("mixed_qkv", "a", "b", "a_log", "dt_bias", "initial_state", "ssm_state_indices", "cu_seqlens",
          "has_initial_state", "out", "workspace")


def gdn_prefill(
    mixed_qkv: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    a_log: torch.Tensor,
    dt_bias: torch.Tensor,
    initial_state: torch.Tensor,
    ssm_state_indices: torch.Tensor,
    cu_seqlens: torch.Tensor,
    has_initial_state: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    scale: float | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """The gated delta rule over N packed sequences. Sequence n owns rows
    cu_seqlens[n]:cu_seqlens[n+1] of mixed_qkv [T, 2HK + HV V] (q heads | k
    heads | v heads, raw), a and b [T, HV], and the state in slot
    ssm_state_indices[n] of initial_state [slots, HV, V, K] (bf16, f16 or f32;
    slot 0 the null slot), which is updated in place. With has_initial_state
    [N], a sequence whose entry is False starts from zeros. Returns out
    [T, HV, V] = scale (S q) of every token, in mixed_qkv's dtype; scale
    defaults to head_k_dim ** -0.5. workspace: a uint8 tensor of at least
    gdnr_lib.prefill_workspace(...) bytes (allocated when not given)."""
    host = gdnr_lib.host()
    host.require(_NAMES, (mixed_qkv, a, b, a_log, dt_bias, initial_state, ssm_state_indices, cu_seqlens,
                          has_initial_state, out, workspace))
    if initial_state.dim() != 4 or mixed_qkv.dim() != 2:
        raise ValueError("initial_state must be [slots, HV, V, K] and mixed_qkv [T, 2HK + HV V]")
    tokens, (_, value_heads, value_dim, key_dim) = mixed_qkv.shape[0], initial_state.shape
    if out is None:
        out = host.empty(mixed_qkv, (tokens, value_heads, value_dim))
    if workspace is None:
        heads = max(0, (mixed_qkv.shape[1] - value_heads * value_dim) // (2 * max(key_dim, 1)))
        size = gdnr_lib.prefill_workspace(tokens, max(cu_seqlens.shape[0] - 1, 0) if cu_seqlens.dim() else 0, heads,
                                          value_heads, value_dim, mixed_qkv.dtype, initial_state.dtype)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=mixed_qkv.device)
    flags = None if has_initial_state is None else _as_flag(has_initial_state)
    host.call(_PREFILL, (mixed_qkv, a, b, _as_f32(a_log), _as_f32(dt_bias), initial_state, _as_i32(ssm_state_indices),
                         _as_i32(cu_seqlens), flags, out, workspace), (),
              (key_dim ** -0.5 if scale is None else scale,), None)
    return out
