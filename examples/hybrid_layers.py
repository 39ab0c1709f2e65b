"""A hybrid stack's token mixers, prefilled and decoded: GDN layers on
ReplaySSMCache (prompts by gdn_prefill, then one fused decode step a token) and
full-attention layers on PagedKVCache (qkv_norm_rope_append, paged_attention).

    python examples/hybrid_layers.py [--tokens N]

The projections around the mixers are random matrices at a small width, so the
run needs no weights. It prefills three prompts of different lengths, one of
them in two chunks, decodes further tokens, and compares each decoded token's
hidden state with the same token's when the whole sequence is prefilled at
once; the difference is what the FP8 checkpoint of the GDN state costs.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

PKG = Path(__file__).resolve().parents[1] / "fp8-replayssm-gdn-kernel_amd"
if str(PKG) not in sys.path:
    sys.path.insert(0, str(PKG))

import gdn_attention as ga  # noqa: E402
import gdn_replayssm_cache as rc  # noqa: E402

WIDTH, H, HV, K, V = 256, 2, 4, 128, 128  # hidden width; GDN heads
HQ, HKV, D, ROTARY = 8, 2, 128, 64        # attention heads


class HybridStack:
    """``pattern`` of layers, "g" GDN and "a" full attention, over slots 1..n."""

    def __init__(self, pattern: str = "ggga", sequences: int = 4, window: int = 8, pages: int = 64, page_size: int = 16,
                 seed: int = 0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows, columns):
            return (torch.randn(rows, columns, generator=gen, device=device) * rows ** -0.5).to(torch.bfloat16)

        self.pattern = pattern
        self.layers, attention = [], 0
        for kind in pattern:
            if kind == "g":
                self.layers.append(dict(
                    mixed=matrix(WIDTH, 2 * H * K + HV * V), gates=matrix(WIDTH, 2 * HV), out=matrix(HV * V, WIDTH),
                    a_log=torch.rand(HV, generator=gen, device=device),
                    dt_bias=torch.rand(HV, generator=gen, device=device) - 4.0,
                    cache=rc.ReplaySSMCache(sequences, window, H, HV, K, V, device=device)))
            else:
                self.layers.append(dict(qkv=matrix(WIDTH, (HQ + 2 * HKV) * D), out=matrix(HQ * D, WIDTH), index=attention,
                                        q_weight=torch.ones(D, device=device), k_weight=torch.ones(D, device=device)))
                attention += 1
        self.pages = ga.PagedKVCache(pages, page_size, HKV, D, layers=max(attention, 1), device=device)
        self.table = ga.rope_table(pages * page_size, ROTARY, device=device)

    def _attention(self, layer, x, batch):
        q, k, v = (x @ layer["qkv"]).split([HQ * D, HKV * D, HKV * D], dim=-1)
        keys, values = self.pages.k[layer["index"]], self.pages.v[layer["index"]]
        q = ga.qkv_norm_rope_append(q.unflatten(-1, (HQ, D)), k.unflatten(-1, (HKV, D)), v.unflatten(-1, (HKV, D)),
                                    self.table, batch.positions, keys, values, batch.slot_mapping,
                                    q_weight=layer["q_weight"], k_weight=layer["k_weight"])
        o = ga.paged_attention(q, keys, values, batch.block_table, batch.cu_seqlens, batch.context_lens,
                               max_context=batch.max_context)
        return o.flatten(1) @ layer["out"]

    def _run(self, slots, lengths, x, gdn):
        batch = self.pages.step(slots, lengths)
        for kind, layer in zip(self.pattern, self.layers):
            y = x / x.float().square().mean(-1, keepdim=True).add(1e-6).sqrt().to(x.dtype)
            if kind == "a":
                x = x + self._attention(layer, y, batch)
                continue
            a, b = (y @ layer["gates"]).split(HV, dim=-1)
            o = gdn(layer["cache"], y @ layer["mixed"], a.contiguous(), b.contiguous(), layer["a_log"], layer["dt_bias"])
            x = x + o.flatten(1) @ layer["out"]
        return x

    def prefill(self, slots, lengths, x, continued=None):
        """x [sum(lengths), WIDTH]: the slots' prompts (or their next chunks)."""
        return self._run(slots, lengths, x, lambda cache, *rows: cache.prefill(slots, lengths, *rows, continued=continued))

    def decode(self, slots, x):
        """x [len(slots), WIDTH]: one token of each."""
        return self._run(slots, [1] * len(slots), x, lambda cache, *rows: cache.step(slots, *rows))

    def release(self, slot):
        for kind, layer in zip(self.pattern, self.layers):
            if kind == "g":
                layer["cache"].release(slot)
        self.pages.release(slot)


def main(tokens: int = 12, device="cuda") -> float:
    """Largest relative difference of a decoded token's hidden state."""
    gen = torch.Generator(device=device).manual_seed(1)
    prompts, slots = [70, 5, 133], [1, 2, 3]
    stack = HybridStack(device=device)
    x = [torch.randn(n + tokens, WIDTH, generator=gen, device=device).to(torch.bfloat16) for n in prompts]
    # the third prompt comes in two chunks, the second one beside the others' whole prompts
    stack.prefill([3], [64], x[2][:64])
    rows = torch.cat([x[0][:prompts[0]], x[1][:prompts[1]], x[2][64:prompts[2]]])
    stack.prefill(slots, [prompts[0], prompts[1], prompts[2] - 64], rows, continued=[False, False, True])
    decoded = []
    for t in range(tokens):
        decoded.append(stack.decode(slots, torch.stack([y[n + t] for y, n in zip(x, prompts)])))
    for slot in slots:
        stack.release(slot)
    whole = stack.prefill(slots, [y.shape[0] for y in x], torch.cat(x)).split([y.shape[0] for y in x])
    worst = 0.0
    for i, (y, n) in enumerate(zip(whole, prompts)):
        for t in range(tokens):
            got, want = decoded[t][i].float(), y[n + t].float()
            worst = max(worst, float((got - want).norm() / want.norm()))
    return worst


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--tokens", type=int, default=12)
    print(f"decoded against prefilled, largest relative difference: {main(parser.parse_args().tokens):.3e}")
