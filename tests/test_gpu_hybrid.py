"""Prefill into the slot cache and the operators run together, on the GPU."""

from __future__ import annotations

import importlib.util

import numpy as np
import pytest
import torch

import gdn_attention as ga
import gdn_replayssm_cache as rc
import gdn_replayssm_fp8_kernel as gk
from conftest import REPO, rel_l2
from oracle import sequence_oracle

pytestmark = pytest.mark.gpu

H, HV, K, V = 2, 4, 128, 128


def rows(tokens, device, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    return (rand(tokens, 2 * H * K + HV * V).to(torch.bfloat16), rand(tokens, HV).to(torch.bfloat16),
            rand(tokens, HV).to(torch.bfloat16))


def params(device):
    gen = torch.Generator(device=device).manual_seed(99)
    return torch.rand(HV, generator=gen, device=device), torch.rand(HV, generator=gen, device=device) - 4.0


def np64(t):
    return t.detach().cpu().double().numpy()


def exact(x, p, lengths, state=None):
    """Outputs and final states of packed sequences, in float64."""
    n = len(lengths)
    state = np.zeros((n, HV, V, K)) if state is None else state
    return sequence_oracle.gdn_sequences(*(np64(y) for y in x), *(np64(y) for y in p), state, np.arange(n),
                                         np.concatenate([[0], np.cumsum(lengths)]))


def test_prefill_is_load_state_of_the_final_state(device):
    """A prompt's checkpoint is the quantised final state: equal codes but for
    those at a rounding boundary (f32 sums against float64: under 1e-3)."""
    p, lengths = params(device), [70, 1, 0, 200]
    x = rows(sum(lengths), device, 1)
    cache = rc.ReplaySSMCache(6, 8, H, HV, K, V, device=device)
    cache.payload.view(torch.uint8).fill_(0x7F)  # (NaN codes: what was there is not read)
    cache.fill[:] = 5
    out = cache.prefill([4, 2, 5, 1], lengths, *x, *p)
    want, states = exact(x, p, lengths)
    assert rel_l2(np64(out), want) <= 2.0 ** -8
    for i, slot in enumerate([4, 2, 5, 1]):
        ref = gk.quantize_checkpoint(torch.tensor(states[i:i + 1], dtype=torch.float32, device=device), saturation=False)
        assert (cache.payload.view(torch.uint8)[slot] != ref.payload.view(torch.uint8)[0]).float().mean() < 1e-3
        assert torch.allclose(cache.scale[slot].float(), ref.scale[0].float(), rtol=2.0 ** -10)
        assert cache.fill[slot] == 0
    assert (cache.payload.view(torch.uint8)[[0, 3, 6]] == 0x7F).all() and cache.fill[3] == 5


@pytest.mark.parametrize("window,decoded", [(8, 5), (16, 16), (8, 0)])
def test_continued_prefill_takes_the_ring_along(device, window, decoded):
    """A new turn goes on from checkpoint and ring: its outputs are those of
    the state that they stand for, token by token in float64."""
    p = params(device)
    x, y = rows(90, device, 2), rows(2 * 40, device, 3)
    cache = rc.ReplaySSMCache(3, window, H, HV, K, V, device=device)
    cache.prefill([2, 3], [50, 40], *x, *p)
    base = gk.dequantize_checkpoint(gk.QuantizedCheckpoint(cache.payload[2:4], cache.scale[2:4], "vblock", 32, 0.0))
    steps = [rows(2, device, 10 + t) for t in range(decoded)]
    for s in steps[:min(decoded, window)]:
        cache.step([2, 3], *s, *p)
    if decoded == window:  # the ring flushed: a new checkpoint, an empty ring
        base = gk.dequantize_checkpoint(gk.QuantizedCheckpoint(cache.payload[2:4], cache.scale[2:4], "vblock", 32, 0.0))
        steps = []
    state = np64(base)
    if steps:
        packed = [torch.stack([s[i] for s in steps], 1).flatten(0, 1) for i in range(3)]
        _, state = exact(packed, p, [len(steps)] * 2, state)
    want, _ = exact(y, p, [40, 40], state)
    out = cache.prefill([2, 3], [40, 40], *y, *p, continued=[True, True])
    # (the ring holds its keys, values and gates in bfloat16: their rounding
    # and the output's)
    assert rel_l2(np64(out), want) <= 2.0 ** -7


def test_prefill_states_in_bf16(device):
    p, x = params(device), rows(300, device, 5)
    codes = []
    for dtype in (torch.float32, torch.bfloat16):
        cache = rc.ReplaySSMCache(1, 8, H, HV, K, V, device=device)
        cache.prefill([1], [300], *x, *p, state_dtype=dtype)
        ck = gk.QuantizedCheckpoint(cache.payload[1:], cache.scale[1:], "vblock", 32, 0.0)
        codes.append(np64(gk.dequantize_checkpoint(ck)))
    # codes a boundary's rounding apart: one e4m3 step (2^-3 of the value at
    # most) in the 2^-9 / 2^-4 that bfloat16's rounding can cross
    assert rel_l2(codes[1], codes[0]) <= 0.02


def test_prefill_refusals(device):
    p, x = params(device), rows(10, device, 4)
    cache = rc.ReplaySSMCache(3, 8, H, HV, K, V, device=device)
    for slots, lengths, continued in (([0], [10], None), ([4], [10], None), ([1, 1], [5, 5], None), ([1], [9], None),
                                      ([1, 2], [12, -2], None), ([1, 2], [10], None), ([1], [10], [True, False])):
        with pytest.raises(ValueError):
            cache.prefill(slots, lengths, *x, *p, continued=continued)


def test_paged_cache_tables(device):
    """Pages taken as sequences grow, given back when they end; the metadata
    of a step says where its tokens are."""
    cache = ga.PagedKVCache(6, 4, 1, 64, device=device)
    b = cache.step(["x", "y"], [5, 2])
    assert b.positions.tolist() == [0, 1, 2, 3, 4, 0, 1] and b.cu_seqlens.tolist() == [0, 5, 7]
    assert b.context_lens.tolist() == [5, 2] and b.max_context == 5 and cache.free_pages == 3
    table = b.block_table.tolist()
    assert b.slot_mapping.tolist() == [4 * table[0][i // 4] + i % 4 for i in range(5)] + [4 * table[1][0], 4 * table[1][0] + 1]
    b = cache.step(["y", "x"], [1, 4])
    assert b.positions.tolist() == [2, 5, 6, 7, 8] and b.context_lens.tolist() == [3, 9]
    assert b.block_table.tolist()[1][:2] == table[0][:2] and cache.free_pages == 2
    with pytest.raises(RuntimeError):
        cache.step(["z", "y"], [8, 2])
    assert cache.free_pages == 2 and cache.length("z") == 0 and cache.length("y") == 3
    for sequences, new in ((["x", "x"], [1, 1]), (["x"], [1, 2]), (["x"], [-1])):
        with pytest.raises(ValueError):
            cache.step(sequences, new)
    cache.release("x")
    assert cache.free_pages == 5 and cache.length("x") == 0


def test_example_runs(device):
    """The example's stack: three GDN layers and an attention layer, prompts in
    chunks, decode steps past a flush. e4m3 codes are off by 2^-4 at most and
    about 2^-5.5 in the mean; three such layers in a residual stream: 0.1."""
    spec = importlib.util.spec_from_file_location("hybrid_layers", REPO / "examples" / "hybrid_layers.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.main(tokens=12, device=device) <= 0.1
