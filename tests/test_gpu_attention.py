"""The attention-layer operators on the GPU against float64
(oracle/sequence_oracle.py), marked `gpu`.

Tolerances (rel-L2): a value stored in bf16 or f16 is off by its rounding, at
most u = 2^-9 or 2^-12 of it. qkv_norm_rope_append rounds once: 1.1 u.
paged_attention rounds its weights to the cache's type before their product
with the values, as much again and independent: 2 u with room for the sums."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import gdn_attention as ga
import gdnr_lib
from conftest import rel_l2
from oracle import sequence_oracle

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -9, F16: 2.0 ** -12}


def np64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def i32(x, device):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


# ---------------------------------------------------------------- append

def make_append(tokens, device, heads=4, kv_heads=2, dim=128, rotary=None, page=16, dtype=BF16, norm=True, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    pages = -(-tokens // page) + 2
    return dict(q=rand(tokens, heads, dim).to(dtype), k=rand(tokens, kv_heads, dim).to(dtype),
                v=rand(tokens, kv_heads, dim).to(dtype), cos_sin=ga.rope_table(300, rotary or dim, device=device),
                positions=torch.randint(0, 300, (tokens,), generator=gen, device=device, dtype=torch.int32),
                k_cache=rand(pages, page, kv_heads, dim).to(dtype), v_cache=rand(pages, page, kv_heads, dim).to(dtype),
                slot_mapping=torch.randperm(pages * page, generator=gen, device=device)[:tokens].to(torch.int32),
                q_weight=1 + 0.3 * rand(dim) if norm else None, k_weight=1 + 0.3 * rand(dim) if norm else None)


def check_append(x, interleaved=False, eps=1e-6, **kw):
    table, pos, tol = np64(x["cos_sin"]), x["positions"].cpu().numpy(), 1.1 * U[x["q"].dtype]
    keys, values = np64(x["k_cache"]), np64(x["v_cache"])
    page, slots = keys.shape[1], x["slot_mapping"].cpu().numpy()
    on = (slots >= 0) & (slots < keys.shape[0] * page)
    want_q = sequence_oracle.norm_rope(np64(x["q"]), np64(x["q_weight"]), table, pos, interleaved, eps)
    want_k = sequence_oracle.norm_rope(np64(x["k"]), np64(x["k_weight"]), table, pos, interleaved, eps)
    values[slots[on] // page, slots[on] % page] = np64(x["v"])[on]
    old = keys.copy()
    got = ga.qkv_norm_rope_append(**x, interleaved=interleaved, eps=eps, **kw)
    assert rel_l2(np64(got), want_q) <= tol
    now = np64(x["k_cache"])
    if on.any():
        assert rel_l2(now[slots[on] // page, slots[on] % page], want_k[on]) <= tol
    now[slots[on] // page, slots[on] % page] = old[slots[on] // page, slots[on] % page]
    assert np.array_equal(now, old)  # no other slot is touched
    assert np.array_equal(np64(x["v_cache"]), values)
    return got


@pytest.mark.parametrize("tokens", [1, 2, 7, 64, 333, 5000])
def test_append_tokens(device, tokens):
    check_append(make_append(tokens, device, seed=tokens))


@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (64, 32), (128, 128), (128, 32), (128, 48), (256, 256), (256, 64),
                                        (256, 208)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_append_layouts(device, dim, rotary, interleaved, norm):
    check_append(make_append(9, device, dim=dim, rotary=rotary, norm=norm, seed=dim + rotary), interleaved)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (16, 4), (5, 5), (32, 8)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_heads(device, heads, kv_heads, dtype):
    check_append(make_append(21, device, heads=heads, kv_heads=kv_heads, dtype=dtype, page=11, seed=heads))


def test_append_skips_and_clamps(device):
    """Slots outside the cache append nothing; positions outside the table
    are clamped to it."""
    x = make_append(12, device, seed=3)
    x["slot_mapping"][::3] = -1
    x["slot_mapping"][1] = 10 ** 6
    check_append(x)
    x["positions"][:2] = torch.tensor([-5, 10 ** 6], dtype=torch.int32, device=device)
    y = dict(x, positions=x["positions"].clamp(0, 299))
    assert torch.equal(ga.qkv_norm_rope_append(**x), ga.qkv_norm_rope_append(**y))


def test_append_one_norm_and_nonfinite(device):
    """A norm on the queries alone; a NaN shows in its own head alone."""
    x = make_append(5, device, seed=4)
    x["k_weight"] = None
    check_append(x)
    clean = ga.qkv_norm_rope_append(**x)
    x["q"][2, 1, 3] = float("nan")
    got = ga.qkv_norm_rope_append(**x)
    assert torch.isnan(got[2, 1]).any()
    got[2, 1] = clean[2, 1]
    assert torch.equal(got, clean)


def test_append_strides(device):
    """q, k, v as views of one row buffer, keys and values interleaved in one
    cache, a given q_out inside a larger buffer."""
    x = make_append(40, device, heads=4, kv_heads=2, seed=5)
    row = torch.randn(40, 8 * 128 + 64, device=device).to(BF16)
    x["q"], x["k"], x["v"] = (row[:, a:b].view(40, -1, 128) for a, b in ((0, 512), (512, 768), (768, 1024)))
    both = torch.randn(6, 2, 16, 2, 128, device=device).to(BF16)
    x["k_cache"], x["v_cache"] = both[:, 0], both[:, 1]
    x["positions"] = torch.stack([x["positions"]] * 2, 1)[:, 0]
    buffer = torch.zeros(40, 6, 192, dtype=BF16, device=device)
    check_append(x, q_out=buffer[:, 1:5, 32:160])
    assert (buffer[:, 0] == 0).all() and (buffer[:, :, :32] == 0).all()


def test_rope_table(device):
    table = np64(ga.rope_table(50, 32, base=500.0, device=device))
    angle = np.arange(50)[:, None] * 500.0 ** (-np.arange(0, 32, 2) / 32)
    assert np.abs(table - np.concatenate([np.cos(angle), np.sin(angle)], 1)).max() < 1e-7
    half = ga.rope_table(50, 32, device=device, inv_freq=torch.full((16,), 0.25), scale=2.0)
    assert torch.allclose(half[:, :16].cpu(), 2 * torch.cos(0.25 * torch.arange(50.0))[:, None].expand(-1, 16), atol=1e-6)


# ---------------------------------------------------------------- attention

def make_attention(new, contexts, device, heads=4, kv_heads=2, dim=128, page=16, dtype=BF16, seed=0, spread=1.5):
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    held = [-(-c // page) for c in contexts]
    pages = sum(held) + 2
    order = np.random.RandomState(seed).permutation(pages)
    table = np.zeros((len(new), max(max(held), 1)), np.int32)
    at = 0
    for n, h in enumerate(held):
        table[n, :h] = order[at:at + h]
        at += h
    return dict(q=(spread * rand(sum(new), heads, dim)).to(dtype), k_cache=rand(pages, page, kv_heads, dim).to(dtype),
                v_cache=rand(pages, page, kv_heads, dim).to(dtype), block_table=i32(table, device),
                cu_seqlens=i32(np.concatenate([[0], np.cumsum(new)]), device), context_lens=i32(contexts, device))


def expected(x, scale=None):
    return sequence_oracle.paged_attention(np64(x["q"]), np64(x["k_cache"]), np64(x["v_cache"]),
                                           x["block_table"].cpu().numpy(), x["cu_seqlens"].cpu().numpy(),
                                           x["context_lens"].cpu().numpy(), scale)


def check_attention(x, **kw):
    want = expected(x, kw.get("scale"))
    got = ga.paged_attention(**x, **kw)
    assert rel_l2(np64(got), want) <= 2 * U[got.dtype]
    return got


@pytest.mark.parametrize("context", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 1000, 3001])
def test_decode_contexts(device, context):
    check_attention(make_attention([1], [context], device, seed=context))


@pytest.mark.parametrize("new,contexts", [([4, 1, 1], [4, 90, 300]), ([1, 0, 5], [20, 0, 5]), ([17], [17]), ([64], [64]),
                                          ([65, 3], [129, 40]), ([200, 1, 33], [700, 512, 33]), ([130], [131]), ([0, 0], [3, 0])])
def test_chunks(device, new, contexts):
    check_attention(make_attention(new, contexts, device, seed=sum(new)))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (3, 1), (10, 2), (16, 1), (20, 1), (40, 2), (6, 6), (32, 8)])
def test_groups(device, heads, kv_heads):
    check_attention(make_attention([1, 6, 35], [70, 9, 300], device, heads=heads, kv_heads=kv_heads, seed=heads))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page", [1, 7, 16, 48, 256])
def test_types_and_pages(device, dim, dtype, page):
    check_attention(make_attention([2, 1, 70], [100, 515, 180], device, dim=dim, dtype=dtype, page=page, seed=dim + page))


def test_rows_without_keys(device):
    """Fewer keys than new tokens: the first tokens see none and give 0."""
    x = make_attention([6, 40, 2], [4, 10, 0], device, seed=2)
    got = check_attention(x)
    assert (got[:2] == 0).all() and (got[6:36] == 0).all() and (got[46:] == 0).all() and (got[2:6] != 0).any()


@pytest.mark.parametrize("pieces", [False, True])
def test_stale_and_masked_values(device, pieces):
    """NaN and infinities where nothing may be seen -- pages of nobody,
    offsets past the context, a later token's key and value -- change no bit of
    what must not see them."""
    contexts = [40, 75, 2000] if pieces else [40, 75, 80]
    x = make_attention([1, 30, 50], contexts, device, seed=3)
    clean = ga.paged_attention(**x)
    used = torch.zeros(x["k_cache"].shape[:2], dtype=torch.bool, device=device)
    for n, c in enumerate(contexts):
        at = torch.arange(c, device=device)
        used[x["block_table"][n].long()[at // 16], at % 16] = True
    for value in (float("nan"), float("inf")):
        for cache in (x["k_cache"], x["v_cache"]):
            cache[~used] = value
    assert torch.equal(ga.paged_attention(**x), clean)
    # key and value of token 20 of sequence 1 (key 75 - 30 + 20), of token 7 of sequence 2
    for n, key in ((1, 65), (2, contexts[2] - 50 + 7)):
        at = int(x["block_table"][n, key // 16]), key % 16
        x["k_cache"][at][0, 3] = float("nan")
        x["v_cache"][at][0, 5] = float("inf")
        x["v_cache"][at][1, 6] = float("nan")
    got = ga.paged_attention(**x)
    rows = torch.ones(81, dtype=torch.bool, device=device)
    rows[1 + 20:31] = False
    rows[31 + 7:] = False
    # (a step with such a value is summed key by key: equal up to rounding)
    assert torch.isfinite(got[rows]).all() and rel_l2(np64(got[rows]), np64(clean[rows])) <= 2 * U[BF16]
    assert torch.isnan(got[~rows][:, :2]).all() and torch.isnan(got[~rows][:, 2:, 6]).all()
    others = [d for d in range(128) if d != 6]
    assert torch.isfinite(got[~rows][:, 2:, others]).all()


def test_lowest_scores(device):
    """Scores at the ends of f32's range: sums of the largest finite products."""
    x = make_attention([1, 20], [50, 60], device, seed=4)
    x["q"] *= 1e18
    x["k_cache"] *= 1e16
    check_attention(x)
    x["q"].zero_()
    check_attention(x)


def test_sharp_and_growing_scores(device):
    """Scores of hundreds, growing along the keys: the running maximum moves
    at every step."""
    x = make_attention([1, 8], [900, 400], device, seed=5, spread=12.0)
    for n, c in enumerate((900, 400)):
        at = torch.arange(c, device=device)
        x["k_cache"][x["block_table"][n].long()[at // 16], at % 16] *= (0.2 + at / c)[:, None, None].to(BF16)
    check_attention(x)


def test_attention_strides(device):
    """Caches interleaved in one tensor, q and out inside larger rows, strided
    lengths, a wide block table with pages outside the cache past the context."""
    x = make_attention([1, 9], [45, 130], device, seed=6)
    both = torch.stack([x["k_cache"], x["v_cache"]], 1)
    x["k_cache"], x["v_cache"] = both[:, 0], both[:, 1]
    row = torch.zeros(10, 4, 3 * 128, dtype=BF16, device=device)
    row[:, :, 128:256] = x["q"]
    x["q"] = row[:, :, 128:256]
    table = torch.full((2, 64), 10 ** 9, dtype=torch.int32, device=device)
    table[:, :x["block_table"].shape[1]] = x["block_table"]
    x["block_table"] = table
    x["context_lens"] = torch.stack([x["context_lens"]] * 3, 1)[:, 1]
    buffer = torch.full((10, 4, 256), 3.0, dtype=BF16, device=device)
    check_attention(x, out=buffer[:, :, 64:192], scale=0.3)
    assert (buffer[:, :, :64] == 3).all() and (buffer[:, :, 192:] == 3).all()
    want = ga.paged_attention(**x)
    assert rel_l2(np64(ga.paged_attention(**x, max_context=130)), np64(want)) <= 2 * U[BF16]


def test_long_cache(device):
    """Caches that span more than 4 GiB: rows found by offsets that pass 32 bits."""
    pages, page = 2400, 2048
    x = make_attention([1, 3], [40, 3000], device, page=16, seed=7)
    big = torch.zeros(pages, 2, page, 2, 128, dtype=BF16, device=device)  # 2.3 GiB of keys, as much of values
    table = i32([[pages - 1, 5], [700, pages - 2]], device)
    for n, c in enumerate((40, 3000)):
        at = torch.arange(c, device=device)
        for i, cache in enumerate((x["k_cache"], x["v_cache"])):
            big[table[n].long()[at // page], i, at % page] = cache[x["block_table"][n].long()[at // 16], at % 16]
    want = ga.paged_attention(**x)
    y = dict(x, k_cache=big[:, 0], v_cache=big[:, 1], block_table=table)
    assert rel_l2(np64(ga.paged_attention(**y, max_context=3000)), np64(want)) <= 2 * U[BF16]


def test_attention_streams_and_graph(device):
    x = make_attention([1, 1, 70], [3000, 40, 200], device, seed=8)
    want = ga.paged_attention(**x)
    size = gdnr_lib.paged_attention_workspace(72, 3, 4, 2, 128, x["block_table"].shape[1] * 16)
    workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=device)
    out, stream = torch.zeros_like(want), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(ga.paged_attention(**x), want)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        ga.paged_attention(**x, out=out, workspace=workspace)
        graph.capture_end()
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_append_then_attend(device):
    """What one operator appends is what the other reads."""
    new, contexts, page = [3, 1, 40], [3, 30, 90], 16
    x = make_attention(new, contexts, device, page=page, seed=9)
    a = make_append(44, device, page=page, seed=9)
    starts = np.concatenate([[0], np.cumsum(new)])
    pos = np.concatenate([np.arange(c - l, c) for l, c in zip(new, contexts)])
    table = x["block_table"].cpu().numpy()
    slot = np.concatenate([table[n][p // page] * page + p % page
                           for n in range(3) for p in [pos[starts[n]:starts[n + 1]]]])
    a.update(positions=i32(pos, device), slot_mapping=i32(slot, device), k_cache=x["k_cache"], v_cache=x["v_cache"])
    x["q"] = check_append(a)
    check_attention(x)


@pytest.mark.parametrize("new,context,heads,kv_heads,dim", [(1030, 1100, 16, 8, 64), (2500, 2500, 8, 1, 128), (1100, 1130, 32, 32, 64),
                                                            (700, 720, 24, 8, 256)])
def test_many_tiles_of_one_sequence(device, new, context, heads, kv_heads, dim):
    """More tiles than compute units, and twice as many: every row once,
    whatever the order that the tiles are taken in."""
    check_attention(make_attention([new], [context], device, heads=heads, kv_heads=kv_heads, dim=dim, seed=new))


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (6, 2, 64), (40, 2, 64), (16, 2, 256)])
@pytest.mark.parametrize("new,contexts", [([1, 1, 300], [5000, 700, 900]), ([2, 600, 0, 1], [4000, 650, 0, 3]),
                                          ([90, 1], [3000, 6000])])
def test_pieces_of_either_kind(device, heads, kv_heads, dim, new, contexts):
    """Decodes beside a prompt's chunk, each kind in its own number of pieces:
    every piece lies inside the workspace that was asked for, and nothing that
    the workspace held before is read."""
    x = make_attention(new, contexts, device, heads=heads, kv_heads=kv_heads, dim=dim, seed=dim + sum(new))
    most = max(contexts)
    size = gdnr_lib.paged_attention_workspace(sum(new), len(new), heads, kv_heads, dim, most)
    assert size > 0
    workspace = torch.full((size + 4096,), 0xFF, dtype=torch.uint8, device=device)  # (NaN)
    check_attention(x, max_context=most, workspace=workspace[:size])
    assert (workspace[size:] == 0xFF).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("gap", [12.0, 18.0])
@pytest.mark.parametrize("new,contexts", [([1], [20000]), ([1, 1, 3], [6000, 3000, 4000]), ([300], [5000]), ([1, 100], [9000, 5000])])
def test_tail_under_a_dominant_key(device, new, contexts, dim, gap, dtype):
    """A key ahead of thousands of others by 12 or 18 (e^18 = 2^26), its value
    0: the output is the others' sum, whose weights keep their bits. (Values of
    some 2^12, so that such a sum is no subnormal number of f16's.)"""
    x = make_attention(new, contexts, device, dim=dim, dtype=dtype, seed=dim, spread=1.0)
    x["v_cache"] *= 4096
    u = torch.full((dim,), dim ** -0.5, device=device)
    q = x["q"].float()
    x["q"] = (q - (q @ u)[..., None] * u + 8 * u).to(dtype)
    for n in range(len(new)):
        at = int(x["block_table"][n, 0]), 5
        x["k_cache"][at] = (gap * dim ** 0.5 / 8 * u).to(dtype)
        x["v_cache"][at] = 0
    check_attention(x)


@pytest.mark.parametrize("scale", [1.0, 60.0, 8000.0])
def test_large_scores_in_f16(device, scale):
    """Scores of a few units, of 1e4 and of 2^27, where floats are 8 apart."""
    x = make_attention([1, 40, 2], [3000, 700, 50], device, dtype=F16, seed=21)
    x["q"] *= scale
    x["k_cache"] *= scale
    check_attention(x)


@pytest.mark.parametrize("dim,rotary", [(64, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("magnitude", [1e8, 1e18, 1e20, 1e30, 5e37])
def test_append_large_rows(device, dim, rotary, interleaved, magnitude):
    """Heads whose squares leave f32 are normed like any others, beside some
    that are not large and under a large eps too."""
    x = make_append(40, device, heads=6, kv_heads=2, dim=dim, rotary=rotary, seed=22)
    x["q"][::2] *= magnitude
    x["k"][1::3, 0] *= magnitude
    check_append(x, interleaved=interleaved)
    check_append(x, interleaved=interleaved, eps=1e10)


@pytest.mark.parametrize("new,context,heads,kv_heads,dim,turns", [
    (180, 190, 256, 64, 64, 1.5), (250, 256, 256, 64, 64, 2.0), (75, 200, 1024, 128, 64, 2.5), (250, 700, 256, 64, 128, 2.0),
    (33, 250, 1024, 128, 256, 2.5)])
def test_order_of_the_tiles_past_one_to_a_compute_unit(device, new, context, heads, kv_heads, dim, turns):
    """One sequence in one piece, with ``turns`` times as many tiles as one to
    each compute unit: the second ones are taken from the other end, the rest in order."""
    rows, group = 64 if dim == 256 else 128, heads // kv_heads
    tiles, places = -(-new // (rows // group)), torch.cuda.get_device_properties(device).multi_processor_count // kv_heads
    if torch.cuda.get_device_properties(device).multi_processor_count == 256:
        assert tiles == turns * places
    assert gdnr_lib.paged_attention_workspace(new, 1, heads, kv_heads, dim, context) == 0  # one piece
    check_attention(make_attention([new], [context], device, heads=heads, kv_heads=kv_heads, dim=dim, seed=new), max_context=context)
