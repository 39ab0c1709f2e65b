"""The full-attention layers between a hybrid model's GDN layers: their entry
(head norms, position rotation, append to a paged cache) and attention of new
tokens over that cache.

The reference leaves these layers to vLLM; its models interleave them with the
GDN layers this package serves, so a program that prefills and decodes such a
model through this package needs both. Kernels run on torch's current stream;
nothing synchronises.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

import gdnr_lib
from gdn_replayssm_fp8_kernel import _as_f32, _as_i32

__all__ = ["rope_table", "qkv_norm_rope_append", "paged_attention", "PagedBatch", "PagedKVCache"]

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
        inv_freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device="cpu") / rotary_dim)
    if tuple(inv_freq.shape) != (rotary_dim // 2,):
        raise ValueError("inv_freq must be [rotary_dim / 2]")
    angle = torch.arange(positions, dtype=torch.float64, device="cpu")[:, None] * inv_freq.double().cpu()
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
        max_context = min(block_table.shape[1] * k_cache.shape[1], 2 ** 31 - 1)
    elif not 0 <= max_context < 2 ** 31:
        raise ValueError(f"max_context {max_context} outside [0, 2^31)")
    if out is None:
        out = host.empty(q, (tokens, heads, dim))
    if workspace is None:
        size = gdnr_lib.paged_attention_workspace(tokens, block_table.shape[0], heads, k_cache.shape[2], dim, max_context)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    host.call(_ATTENTION, (q, k_cache, v_cache, _as_i32(block_table), _as_i32(cu_seqlens), _as_i32(context_lens), out,
                           workspace), (int(max_context),), (dim ** -0.5 if scale is None else scale,), None)
    return out


@dataclass
class PagedBatch:
    """Device metadata of one step of PagedKVCache sequences, shared by every
    layer of the step."""

    positions: torch.Tensor     # [T] i32: position of each new token in its sequence
    slot_mapping: torch.Tensor  # [T] i32: its slot in the caches
    block_table: torch.Tensor   # [N, width] i32
    cu_seqlens: torch.Tensor    # [N + 1] i32
    context_lens: torch.Tensor  # [N] i32, new tokens included
    max_context: int


class PagedKVCache:
    """Keys and values of ``layers`` attention layers in pages of ``page_size``
    tokens that sequences take as they grow. Which pages a sequence holds is
    host state (as ReplaySSMCache keeps its ring fills), the same for every
    layer; step() turns a batch into the metadata its layers' two operators
    take."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, layers: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if num_pages < 1 or page_size < 1 or layers < 1:
            raise ValueError("num_pages, page_size and layers must be at least 1")
        self.page_size, self.device = page_size, torch.device(device)
        self.k = [torch.zeros(num_pages, page_size, kv_heads, head_dim, dtype=dtype, device=self.device) for _ in range(layers)]
        self.v = [torch.zeros_like(k) for k in self.k]
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict = {}   # sequence -> its pages, in order
        self._length: dict = {}  # sequence -> tokens it holds

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence) -> int:
        return self._length.get(sequence, 0)

    def release(self, sequence) -> None:
        """End a sequence: its pages are free."""
        self._free.extend(reversed(self._pages.pop(sequence, [])))
        self._length.pop(sequence, None)

    def step(self, sequences, new_tokens) -> PagedBatch:
        """Room for new_tokens[i] further tokens of each sequence (any hashable
        names, distinct; a new name starts a sequence) and the metadata of
        appending and attending them. Raises, with nothing taken, when the
        pages do not suffice."""
        new = [int(x) for x in new_tokens]
        if len(new) != len(sequences) or min(new, default=0) < 0:
            raise ValueError("new_tokens must hold a count of at least 0 for each sequence")
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence appears twice in the batch")
        lengths = [self.length(s) + x for s, x in zip(sequences, new)]
        held = [-(-x // self.page_size) for x in lengths]
        need = sum(h - len(self._pages.get(s, [])) for s, h in zip(sequences, held))
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} free")
        width = max(held, default=0)
        table = np.zeros((len(new), max(width, 1)), dtype=np.int32)
        positions, slots = [], []
        for i, (s, x, total, h) in enumerate(zip(sequences, new, lengths, held)):
            pages = self._pages.setdefault(s, [])
            while len(pages) < h:
                pages.append(self._free.pop())
            self._length[s] = total
            table[i, :h] = pages
            at = np.arange(total - x, total)
            positions.append(at)
            slots.append(table[i, at // self.page_size].astype(np.int64) * self.page_size + at % self.page_size)
        # one copy for all of it
        parts = [np.concatenate(positions or [[]]), np.concatenate(slots or [[]]), np.concatenate([[0], np.cumsum(new)]),
                 np.asarray(lengths), table.reshape(-1)]
        packed = torch.from_numpy(np.concatenate(parts).astype(np.int32)).to(self.device)
        pos, slot, cu, context, flat = packed.split([p.size for p in parts])
        return PagedBatch(pos, slot, flat.view(table.shape), cu, context, max(lengths, default=0))
