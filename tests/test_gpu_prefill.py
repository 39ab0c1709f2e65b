"""gdn_prefill on the GPU against the token-by-token recurrence in float64
(oracle/sequence_oracle.py), marked `gpu`.

Tolerances (rel-L2 of the whole output or state), from the arithmetic: a value
stored in bf16 or f16 is off by its rounding, at most u = 2^-9 or 2^-12 of it
(about 0.85 u over many values), and the sums before it may add as much again:
2 u. f32 values come from f32 sums of at most 128 products and a chain of
decays and corrections that forgets within some 100 tokens: 100 roundings of
2^-24 that add up as a walk, 2e-6 with room for cancellation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import gdn_prefill as gp
import gdn_replayssm_fp8_kernel as gk
import gdnr_lib
from conftest import rel_l2
from oracle import sequence_oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TOL = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2e-6}


def make(lengths, device, seed=0, heads=2, value_heads=4, value_dim=128, act=BF16, state=BF16, gate=None, slots=None,
         started=None, reference_dist=True, pad_rows=0, key_mean=0.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    T, N = int(sum(lengths)) + pad_rows, len(lengths)
    a_log = torch.rand(value_heads, generator=gen, device=device)
    dt_bias = torch.rand(value_heads, generator=gen, device=device) - (4.0 if reference_dist else 0.0)
    mixed = rand(T, 2 * heads * 128 + value_heads * value_dim)
    if key_mean:  # keys that share a direction: the chunk's triangle is far from the identity
        mixed[:, heads * 128:2 * heads * 128] += key_mean * rand(heads * 128)
    S = N + 2
    return dict(mixed=mixed.to(act), a=rand(T, value_heads).to(gate or act), b=rand(T, value_heads).to(gate or act),
                a_log=a_log, dt_bias=dt_bias, state=(0.05 * rand(S, value_heads, value_dim, 128)).to(state),
                slots=torch.tensor(slots if slots is not None else np.random.RandomState(seed).permutation(N) + 1,
                                   dtype=torch.int32, device=device),
                cu=torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=device),
                started=None if started is None else torch.tensor(started, device=device))


def np64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def expected(x, scale=None):
    return sequence_oracle.gdn_sequences(np64(x["mixed"]), np64(x["a"]), np64(x["b"]), np64(x["a_log"]),
                                         np64(x["dt_bias"]), np64(x["state"]), x["slots"].cpu().numpy(),
                                         x["cu"].cpu().numpy(), None if x["started"] is None else x["started"].cpu().numpy(),
                                         scale)


def run(x, **kw):
    return gp.gdn_prefill(x["mixed"], x["a"], x["b"], x["a_log"], x["dt_bias"], x["state"], x["slots"], x["cu"],
                          has_initial_state=x["started"], **kw)


def check(x, **kw):
    want, want_state = expected(x, kw.get("scale"))
    before = x["state"].clone()
    out = run(x, **kw)
    n = int(x["cu"][-1])
    if n:
        assert rel_l2(np64(out[:n]), want[:n]) <= TOL[out.dtype]
    used = x["slots"].cpu().long().numpy()
    live = used[used != 0]
    got = np64(x["state"])
    if live.size:
        tol = max(TOL[x["state"].dtype], 0 if out.dtype == F32 or x["state"].dtype == BF16 else 2e-6)
        assert rel_l2(got[live], want_state[live]) <= tol
    others = np.setdiff1d(np.arange(got.shape[0]), used)
    assert torch.equal(x["state"][others], before[others])  # no other slot is touched
    return out


@pytest.mark.parametrize("lengths", [[1], [2], [4, 4, 4], [1, 0, 3], [15, 16, 17], [63], [64], [65], [127, 128, 129],
                                     [200, 0, 1, 90], [333]])
def test_lengths(device, lengths):
    check(make(lengths, device, seed=len(lengths) + lengths[0]))


@pytest.mark.parametrize("lengths", [[5, 1, 8], [100, 70, 1]])
@pytest.mark.parametrize("act,state,gate", [(BF16, F32, None), (F16, F16, None), (F16, F32, F32), (F32, F32, None),
                                            (BF16, BF16, F32), (F16, BF16, None), (F32, BF16, None), (BF16, F16, None)])
def test_types(device, lengths, act, state, gate):
    check(make(lengths, device, seed=3, act=act, state=state, gate=gate))


@pytest.mark.parametrize("lengths", [[3, 7], [130, 64]])
@pytest.mark.parametrize("heads,value_heads,value_dim", [(16, 32, 128), (4, 12, 128), (8, 8, 256), (8, 16, 64), (1, 1, 32),
                                                         (2, 2, 96), (3, 15, 128), (1, 16, 160)])
def test_heads(device, lengths, heads, value_heads, value_dim):
    check(make(lengths, device, seed=5, heads=heads, value_heads=value_heads, value_dim=value_dim))


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("lengths", [[6, 0, 2, 0], [90, 0, 70, 0]])
def test_zero_starts(device, lengths, act):
    """A sequence that starts from nothing does not read its slot (NaN there);
    one of no tokens leaves zeros, or its slot as it was."""
    x = make(lengths, device, seed=7, act=act, state=act, slots=[3, 1, 4, 2], started=[False, False, True, True])
    x["state"][3] = float("nan")
    x["state"][1] = float("nan")
    kept = x["state"][2].clone()
    check(x)
    assert torch.equal(x["state"][2], kept) and (x["state"][1] == 0).all()


def test_correlated_keys(device):
    """Keys that share most of their direction, beta near 1 and slow decay:
    the tokens of a chunk correct one another strongly."""
    x = make([150], device, seed=9, key_mean=2.0)
    x["b"] += 3.0
    x["a"] -= 3.0
    check(x)


@pytest.mark.parametrize("shift", [6.0, 40.0])
def test_strong_decay(device, shift):
    """Log decays of some -7 and -50 a token: products of decays underflow."""
    x = make([130], device, seed=10)
    x["a"] += shift
    check(x)


@pytest.mark.parametrize("magnitude", [1e-6, 1e6, 1e20])
@pytest.mark.parametrize("lengths", [[3], [100]])
def test_magnitudes(device, lengths, magnitude):
    """Rows far from 1, and a state to match: results scale with the values."""
    x = make(lengths, device, seed=11)
    x["mixed"][:, 512:] *= magnitude
    x["state"] *= magnitude
    check(x)


def test_rows_of_different_magnitude(device):
    """Each V-row's precision is its own: a row 1e12 above its neighbours
    does not cost them theirs."""
    x = make([100], device, seed=12)
    v = x["mixed"][:, 512:].view(100, 4, 128)
    v[:, :, 1::2] *= 1e-12
    x["state"][:, :, 1::2] *= 1e-12
    want, _ = expected(x)
    out = np64(run(x))
    for rows in (slice(0, None, 2), slice(1, None, 2)):
        assert rel_l2(out[:, :, rows], want[:, :, rows]) <= TOL[BF16]


def test_continued(device):
    """A prompt in two calls gives what one call gives, up to the state's rounding between them."""
    whole = make([171], device, seed=13, state=F32, act=F32)
    first = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in whole.items()}
    out = run(whole)
    parts = []
    for rows in (slice(0, 77), slice(77, 171)):
        piece = dict(first, mixed=first["mixed"][rows], a=first["a"][rows], b=first["b"][rows],
                     cu=torch.tensor([0, rows.stop - rows.start], dtype=torch.int32, device=device))
        parts.append(run(piece))
    assert rel_l2(np64(torch.cat(parts)), np64(out)) <= TOL[F32]
    assert rel_l2(np64(first["state"]), np64(whole["state"])) <= TOL[F32]


def test_one_token_is_the_packed_step(device):
    """A call of one token per sequence is the full-state decode step."""
    x = make([1] * 5, device, seed=14, heads=16, value_heads=32)
    state = x["state"].clone()
    step = gk.gdn_bf16_step_packed(x["mixed"], x["a"], x["b"], x["a_log"], x["dt_bias"], state, x["slots"])
    out = run(x)
    assert rel_l2(np64(out), np64(step[:, 0])) <= TOL[BF16]
    assert rel_l2(np64(x["state"]), np64(state)) <= TOL[BF16]


@pytest.mark.parametrize("lengths", [[9], [140]])
def test_strides(device, lengths):
    """Rows inside wider buffers, a state between other layers', strided
    indices, rows past the last sequence, a given out and scale."""
    T = sum(lengths)
    x = make(lengths, device, seed=15, pad_rows=3)
    wide = torch.randn(T + 3, x["mixed"].shape[1] + 128, device=device).to(BF16)
    wide[:, 64:-64] = x["mixed"]
    x["mixed"] = wide[:, 64:-64]
    gates = torch.randn(4, T + 3, 2, device=device).to(BF16)
    x["a"], x["b"] = gates[:, :, 0].t(), gates[:, :, 1].t()
    layers = torch.randn(x["state"].shape[0], 3, *x["state"].shape[1:], device=device).to(BF16) * 0.05
    x["state"] = layers[:, 1]
    x["slots"] = torch.stack([x["slots"], x["slots"] + 7], 1)[:, 0]
    others = layers[:, 0].clone(), layers[:, 2].clone()
    buffer = torch.full((T + 3, 4, 160), 7.0, dtype=BF16, device=device)
    out = check(x, out=buffer[:, :, 16:144], scale=0.25)
    assert torch.equal(layers[:, 0], others[0]) and torch.equal(layers[:, 2], others[1])
    assert (buffer[:, :, :16] == 7).all() and (buffer[:, :, 144:] == 7).all() and (out[T:] == 7).all()


def test_slots_out_of_range_are_the_null_slot(device):
    x = make([3, 3, 80], device, seed=16, slots=[2, -1, 99])
    kept = x["state"].clone()
    run(x)
    assert torch.equal(x["state"][1], kept[1]) and torch.equal(x["state"][3:], kept[3:])
    assert not torch.equal(x["state"][2], kept[2])


def test_offsets_are_clamped(device):
    """Offsets past the rows there are end at the last row."""
    x = make([70, 5], device, seed=17)
    x["cu"] = torch.tensor([0, 70, 5000], dtype=torch.int32, device=device)
    y = dict(x, cu=torch.tensor([0, 70, 75], dtype=torch.int32, device=device), state=x["state"].clone())
    assert torch.equal(run(x), run(y)) and torch.equal(x["state"], y["state"])


@pytest.mark.parametrize("lengths", [[12], [150]])
@pytest.mark.parametrize("what", ["v", "k", "q", "a", "state"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_nonfinite_values_stay_behind_their_token(device, lengths, what, value):
    """A value that is not finite shows in nothing before its token, in no
    other value head and, from v or the state, in no other V-row."""
    T, t, heads, hv = lengths[0], lengths[0] // 2 + 3, 2, 4
    x = make(lengths, device, seed=18, heads=heads, value_heads=hv)
    want, want_state = expected(x)
    clean = np.ones((T, hv, 128), bool)
    if what == "v":
        x["mixed"][t, 512 + 128 + 5] = value
        clean[t:, 1, 5] = False
    elif what == "state":
        x["state"][int(x["slots"][0]), 1, 5, 9] = value
        clean[:, 1, 5] = False
        t = 0
    elif what == "a":
        if value != value:
            x["a"][t, 1] = value
            clean[t:, 1] = False
        else:  # a log decay of -inf forgets the state: every output stays finite
            x["a"][t, 1] = value
            want, want_state = expected(x)
    else:
        x["mixed"][t, (256 if what == "k" else 0) + 5] = value
        clean[t if what == "q" else slice(t, None), 0:2] = False
    out = np64(run(x))
    assert np.isfinite(out[clean]).all()
    assert rel_l2(out[clean], want[clean]) <= TOL[BF16]
    if not clean.all():
        assert np.isnan(out[~clean]).any()
    state = np.isfinite(np64(x["state"])[int(x["slots"][0])])
    if what == "q":
        assert state.all()
    elif what == "k":
        assert state[2:].all() and not state[:2].any()
    elif what in ("v", "state"):
        assert not state[1, 5].any() and state.sum() == state.size - 128


def test_streams_and_graph(device):
    """On a stream of the caller's, and captured once and replayed."""
    x = make([5, 200, 66], device, seed=19)
    first = x["state"].clone()
    want = run(x)
    stream = torch.cuda.Stream()
    workspace = torch.empty(max(16, gdnr_lib.prefill_workspace(271, 3, 2, 4, 128, BF16, BF16)), dtype=torch.uint8, device=device)
    out = torch.empty_like(want)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x["state"].copy_(first)
        run(x, out=out, workspace=workspace)
        stream.synchronize()
        assert torch.equal(out, want)
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        run(x, out=out, workspace=workspace)
        graph.capture_end()
    for _ in range(3):
        x["state"].copy_(first)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_repeatable(device):
    x = make([300, 64, 1, 0, 77], device, seed=20, heads=16, value_heads=32)
    first = x["state"].clone()
    want, state = run(x), x["state"].clone()
    x["state"].copy_(first)
    assert torch.equal(run(x), want) and torch.equal(x["state"], state)


def sizes(count, low, high, seed):
    return np.random.RandomState(seed).randint(low, high, count).tolist()


@pytest.mark.parametrize("count,value_heads,act,state", [
    (2, 16, BF16, BF16), (7, 8, BF16, BF16), (20, 8, BF16, BF16), (70, 4, BF16, BF16),  # 3 roles, 4 waves, 8 waves
    (2, 16, F16, F32), (6, 8, F16, F32), (12, 8, F32, F32), (70, 4, F16, F16)])         # 3 roles, 2 waves, 4, 8
def test_scan_forms(device, count, value_heads, act, state):
    """Every width of the scan, each with empty sequences, single tokens and
    lengths that tie; 70 sequences are two groups of its longest-first order."""
    lengths = sizes(count, 20, 150, count)
    lengths[0], lengths[count // 2], lengths[-1] = 64, 0 if count > 2 else 1, 64
    check(make(lengths, device, seed=count, heads=value_heads // 2, value_heads=value_heads, act=act, state=state))


def test_order_of_the_batch(device):
    """What a sequence gets does not depend on where it stands in the batch."""
    lengths = [70, 200, 1, 130, 64]
    x = make(lengths, device, seed=40)
    whole = run(x)
    rows = torch.split(torch.arange(sum(lengths), device=device), lengths)
    order = [3, 0, 4, 2, 1]
    y = make(lengths, device, seed=40)
    at = torch.cat([rows[i] for i in order])
    for name in ("mixed", "a", "b"):
        y[name] = y[name][at]
    y["slots"] = y["slots"][order]
    y["cu"] = torch.tensor(np.concatenate([[0], np.cumsum([lengths[i] for i in order])]), dtype=torch.int32, device=device)
    assert torch.equal(run(y), whole[at]) and torch.equal(y["state"], x["state"])


@pytest.mark.parametrize("heads,value_heads", [(1, 3), (2, 10), (4, 16), (1, 32)])
@pytest.mark.parametrize("act,state", [(BF16, BF16), (F16, F32)])
def test_value_heads_in_parts(device, heads, value_heads, act, state):
    """Few chunks of key heads with several value heads each: the preparation's
    workgroups share a key head."""
    check(make([70, 40], device, seed=value_heads, heads=heads, value_heads=value_heads, act=act, state=state))


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("lengths", [[9], [100]])
@pytest.mark.parametrize("magnitude", [1e8, 1e18, 1e20, 1e30, 5e37])
def test_large_keys_and_queries(device, lengths, act, magnitude):
    """Keys and queries whose squares leave f32: their unit rows are what they
    are at any magnitude, some rows large and some not."""
    x = make(lengths, device, seed=41, act=act, state=act)
    x["mixed"][::2, :512] *= magnitude
    x["mixed"][1::4, :256] *= magnitude  # (queries alone)
    check(x)


# fewer than 16 tokens a sequence on average (32 with wider results), some of a chunk and more among them
SHORT_AND_LONG = {"one": [150] + [1] * 20, "edges": [1, 63, 64, 0, 65] + [2] * 30, "last": [1] * 40 + [0, 333],
                  "groups": [1] * 60 + [70, 130, 1, 64, 64, 128] + [0, 3] * 40 + [65] + [1] * 9, "none long": [9] * 20,
                  "all in one": [0] * 70 + [200] + [0] * 5}


@pytest.mark.parametrize("name", SHORT_AND_LONG)
@pytest.mark.parametrize("act,state", [(BF16, BF16), (F16, F32), (F32, F32), (BF16, F32)])
def test_long_sequences_among_short(device, name, act, state):
    """Short sequences token by token and long ones in chunks, in one call:
    nothing past the workspace that was asked for is written, nothing that it held is
    read."""
    lengths = SHORT_AND_LONG[name]
    assert 128 <= sum(lengths) < 16 * len(lengths)
    x = make(lengths, device, seed=42, act=act, state=state, started=[n % 3 != 1 for n in range(len(lengths))])
    x["state"][x["slots"][1::3].long()] = float("nan")  # (their sequences start from nothing)
    size = gdnr_lib.prefill_workspace(sum(lengths), len(lengths), 2, 4, 128, act, state)
    assert size > 0
    workspace = torch.full((size + 4096,), 0xFF, dtype=torch.uint8, device=device)
    check(x, workspace=workspace[:size])
    assert (workspace[size:] == 0xFF).all()


def test_long_among_short_is_the_long_one_alone(device):
    """What a long sequence gets does not depend on the short ones beside it."""
    x = make([1] * 30 + [200], device, seed=43, heads=8, value_heads=16)
    y = dict(x, mixed=x["mixed"][30:], a=x["a"][30:], b=x["b"][30:], slots=x["slots"][30:],
             cu=torch.tensor([0, 200], dtype=torch.int32, device=device), state=x["state"].clone())
    whole, alone = run(x), run(y)
    slot = int(x["slots"][30])
    assert torch.equal(whole[30:], alone) and torch.equal(x["state"][slot], y["state"][slot])


@pytest.mark.parametrize("act,state", [(BF16, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("sequences", [1, 9, 40])  # (roles; several waves a workgroup)
@pytest.mark.parametrize("token", [1, 4, 50, 63])
@pytest.mark.parametrize("magnitude", [1e2, 1e4, 1e6, 1e8, 1e12, 1e30])
def test_a_large_value_costs_earlier_tokens_nothing(device, act, state, sequences, token, magnitude):
    """One V-row's v far above everything at one token: the outputs before it, of
    that row alone, are as good as without it, and so is what follows."""
    x = make([70] * sequences, device, seed=44, heads=1, value_heads=2, act=act, state=state)
    at = torch.arange(sequences, device=device) * 70 + token
    x["mixed"][at, 256 + 5] = magnitude
    want, _ = expected(x)
    out = np64(check(x)).reshape(sequences, 70, 2, 128)[:, :token, 0, 5]
    assert rel_l2(out, want.reshape(sequences, 70, 2, 128)[:, :token, 0, 5]) <= TOL[act]


@pytest.mark.parametrize("act,state", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("magnitude", [1e4, 1e8, 1e15])
def test_a_state_forgotten_costs_later_tokens_nothing(device, act, state, magnitude):
    """A large state that the first tokens' decay forgets: what is left is as
    precise as if it had never been there."""
    x = make([100], device, seed=45, act=act, state=state)
    x["state"] *= magnitude
    x["a"][3:20] += 20.0  # (log decays of some -17 to -50 each)
    want, _ = expected(x)
    out = np64(check(x))
    assert rel_l2(out[20:], want[20:]) <= TOL[act]


@pytest.mark.parametrize("act,state", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("sequences", [1, 40])
def test_large_and_nonfinite_values_in_one_chunk(device, act, state, sequences):
    """A V-row that is NaN from its token on, and a key head whose key is, in
    chunks that are walked token by token for another row's large value."""
    x = make([90] * sequences, device, seed=46, heads=2, value_heads=4, act=act, state=state)
    want, want_state = expected(x)
    rows = torch.arange(sequences, device=device) * 90
    x["mixed"][rows + 40, 512 + 5] = 1e12  # value head 0
    x["mixed"][rows + 50, 512 + 9] = float("nan")
    x["mixed"][rows + 60, 256 + 128 + 3] = float("inf")  # the key of value heads 2 and 3
    x["mixed"][rows + 20, 512 + 2 * 128 + 7] = 1e12  # value head 2
    large, _ = expected(x)
    out = np64(run(x)).reshape(sequences, 90, 4, 128)
    want, large = want.reshape(out.shape), large.reshape(out.shape)
    assert np.isnan(out[:, 50:, 0, 9]).all() and np.isnan(out[:, 60:, 2:]).all()
    others = [r for r in range(128) if r not in (5, 9)]
    assert rel_l2(out[:, :, 0, others], want[:, :, 0, others]) <= TOL[act]
    assert rel_l2(out[:, :50, 0, 9], want[:, :50, 0, 9]) <= TOL[act]
    assert rel_l2(out[:, :, 1], want[:, :, 1]) <= TOL[act]
    assert rel_l2(out[:, :40, 0, 5], want[:, :40, 0, 5]) <= TOL[act]
    assert rel_l2(out[:, 40:, 0, 5], large[:, 40:, 0, 5]) <= TOL[act]
    assert rel_l2(out[:, :60, 3], want[:, :60, 3]) <= TOL[act]
    assert rel_l2(out[:, :20, 2, 7], want[:, :20, 2, 7]) <= TOL[act]
    states = np64(x["state"])[x["slots"].cpu().numpy()]
    assert np.isnan(states[:, 0, 9]).all() and np.isnan(states[:, 2:]).all() and np.isfinite(states[:, 0, others]).all()
