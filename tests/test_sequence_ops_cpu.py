"""The sequence operators on the CPU: what they refuse (before any HIP call, on
descriptors with addresses that are never read), their workspace counts, and
the oracle they are tested against."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import gdn_attention as ga
import gdn_prefill as gp
import gdn_replayssm_cache as rc
import gdnr_lib
from oracle import sequence_oracle
from test_abi_cpu import BF16, BOOL, F16, F32, FAKE, I32, I64, INVALID, OK, U8, UNSUPPORTED, desc


@pytest.fixture(scope="module")
def lib():
    return gdnr_lib.load_library()


def call(lib, name, tensors, numbers):
    args = [None if t is None else ctypes.byref(t) for t in tensors.values()]
    return getattr(lib, name)(*args, *numbers, None)


def prefill_case(T=10, N=2, H=2, HV=4, V=128, S=3, act=BF16, state=BF16):
    return dict(mixed=desc([T, 2 * H * 128 + HV * V], act), a=desc([T, HV], act), b=desc([T, HV], act),
                a_log=desc([HV], F32), dt_bias=desc([HV], F32), state=desc([S, HV, V, 128], state), slots=desc([N], I32),
                cu=desc([N + 1], I32), started=desc([N], BOOL), out=desc([T, HV, V], act), workspace=desc([1 << 30], U8))


def append_case(T=5, HQ=4, HKV=2, D=128, R=64, act=BF16):
    return dict(q=desc([T, HQ, D], act), k=desc([T, HKV, D], act), v=desc([T, HKV, D], act), q_weight=desc([D], F32),
                k_weight=None, cos_sin=desc([100, R], F32), positions=desc([T], I32), k_cache=desc([9, 16, HKV, D], act),
                v_cache=desc([9, 16, HKV, D], act), slots=desc([T], I32), q_out=desc([T, HQ, D], act))


def attention_case(T=5, N=2, HQ=4, HKV=2, D=128, width=4, act=BF16):
    return dict(q=desc([T, HQ, D], act), k_cache=desc([9, 16, HKV, D], act), v_cache=desc([9, 16, HKV, D], act),
                table=desc([N, width], I32), cu=desc([N + 1], I32), context=desc([N], I32), out=desc([T, HQ, D], act),
                workspace=None)


PREFILL_REFUSALS = {
    "heads do not divide": (dict(mixed=desc([10, 2 * 3 * 128 + 4 * 128], BF16)), INVALID),
    "width": (dict(mixed=desc([10, 1000], BF16)), INVALID),
    "rows": (dict(out=desc([9, 4, 128], BF16)), INVALID),
    "out dtype": (dict(out=desc([10, 4, 128], F32)), INVALID),
    "key dim": (dict(state=desc([3, 4, 128, 64], BF16)), UNSUPPORTED),
    "value dim": (dict(state=desc([3, 4, 100, 128], BF16), mixed=desc([10, 912], BF16)), UNSUPPORTED),
    "no slot": (dict(state=desc([0, 4, 128, 128], BF16)), INVALID),
    "gates": (dict(a=desc([10, 4], F16)), INVALID),
    "slots dtype": (dict(slots=desc([2], I64)), INVALID),
    "starts": (dict(cu=desc([0], I32)), INVALID),
    "starts and slots": (dict(cu=desc([4], I32)), INVALID),
    "flags": (dict(started=desc([2], F32)), INVALID),
    "workspace": (dict(mixed=desc([64, 1024], BF16), a=desc([64, 4], BF16), b=desc([64, 4], BF16),
                       out=desc([64, 4, 128], BF16), workspace=desc([64], U8)), INVALID),
    "no workspace": (dict(mixed=desc([64, 1024], BF16), a=desc([64, 4], BF16), b=desc([64, 4], BF16),
                          out=desc([64, 4, 128], BF16), workspace=None), INVALID),
    "alignment": (dict(mixed=desc([10, 1024], BF16, data=FAKE + 2)), INVALID),
    "inner stride": (dict(state=desc([3, 4, 128, 128], BF16, strides=[1 << 18, 1 << 16, 2, 2])), INVALID),
    "long rows": (dict(mixed=desc([10, 1024], BF16, strides=[1 << 24, 1])), UNSUPPORTED),
}


@pytest.mark.parametrize("name", PREFILL_REFUSALS)
def test_prefill_refusals(lib, name):
    changed, status = PREFILL_REFUSALS[name]
    assert call(lib, "gdnr_prefill", {**prefill_case(), **changed}, (ctypes.c_float(1.0),)) == status
    assert lib.gdnr_last_error()


def test_prefill_numbers(lib):
    for scale in (float("nan"), float("inf")):
        assert call(lib, "gdnr_prefill", prefill_case(), (ctypes.c_float(scale),)) == INVALID
    assert call(lib, "gdnr_prefill", prefill_case(T=0, N=0), (ctypes.c_float(1.0),)) == OK  # nothing to do
    assert call(lib, "gdnr_prefill", prefill_case(T=(1 << 23) + 1), (ctypes.c_float(1.0),)) == UNSUPPORTED
    assert call(lib, "gdnr_prefill", prefill_case(N=65536), (ctypes.c_float(1.0),)) == UNSUPPORTED


APPEND_REFUSALS = {
    "f32": (dict(q=desc([5, 4, 128], F32)), UNSUPPORTED),
    "head dim": (dict(q=desc([5, 4, 96], BF16)), UNSUPPORTED),
    "rows": (dict(k=desc([4, 2, 128], BF16)), INVALID),
    "value heads": (dict(v=desc([5, 1, 128], BF16)), INVALID),
    "rotary past the head": (dict(cos_sin=desc([100, 144], F32)), INVALID),
    "rotary": (dict(cos_sin=desc([100, 24], F32)), INVALID),
    "no positions": (dict(cos_sin=desc([0, 64], F32)), INVALID),
    "table dtype": (dict(cos_sin=desc([100, 64], BF16)), INVALID),
    "weight": (dict(q_weight=desc([64], F32)), INVALID),
    "weight dtype": (dict(k_weight=desc([128], BF16)), INVALID),
    "caches differ": (dict(v_cache=desc([8, 16, 2, 128], BF16)), INVALID),
    "cache heads": (dict(k_cache=desc([9, 16, 3, 128], BF16)), INVALID),
    "cache dtype": (dict(k_cache=desc([9, 16, 2, 128], F16)), INVALID),
    "empty pages": (dict(k_cache=desc([9, 0, 2, 128], BF16), v_cache=desc([9, 0, 2, 128], BF16)), INVALID),
    "cache span": (dict(k_cache=desc([9, 16, 2, 128], BF16, strides=[1 << 33, 256, 128, 1])), UNSUPPORTED),
    "slots": (dict(slots=desc([5], I64)), INVALID),
    "alignment": (dict(k=desc([5, 2, 128], BF16, strides=[260, 130, 1])), INVALID),
}


@pytest.mark.parametrize("name", APPEND_REFUSALS)
def test_append_refusals(lib, name):
    changed, status = APPEND_REFUSALS[name]
    assert call(lib, "gdnr_qkv_norm_rope_append", {**append_case(), **changed}, (0, ctypes.c_float(1e-6))) == status


def test_append_numbers(lib):
    for eps in (float("nan"), -1.0, float("inf")):
        assert call(lib, "gdnr_qkv_norm_rope_append", append_case(), (0, ctypes.c_float(eps))) == INVALID
    assert call(lib, "gdnr_qkv_norm_rope_append", append_case(T=0), (1, ctypes.c_float(0.0))) == OK


ATTENTION_REFUSALS = {
    "f32": (dict(q=desc([5, 4, 128], F32)), UNSUPPORTED),
    "head dim": (dict(q=desc([5, 4, 32], BF16)), UNSUPPORTED),
    "groups": (dict(q=desc([5, 5, 128], BF16)), INVALID),
    "out": (dict(out=desc([5, 4, 64], BF16)), INVALID),
    "table dtype": (dict(table=desc([2, 4], I64)), INVALID),
    "table rows": (dict(table=desc([3, 4], I32)), INVALID),
    "table stride": (dict(table=desc([2, 4], I32, strides=[8, 2])), INVALID),
    "contexts": (dict(context=desc([3], I32)), INVALID),
    "no pages": (dict(k_cache=desc([0, 16, 2, 128], BF16), v_cache=desc([0, 16, 2, 128], BF16)), INVALID),
    "cache alignment": (dict(v_cache=desc([9, 16, 2, 128], BF16, data=FAKE + 8)), INVALID),
}


@pytest.mark.parametrize("name", ATTENTION_REFUSALS)
def test_attention_refusals(lib, name):
    changed, status = ATTENTION_REFUSALS[name]
    assert call(lib, "gdnr_paged_attention", {**attention_case(), **changed}, (64, ctypes.c_float(0.1))) == status


def test_attention_numbers(lib):
    assert call(lib, "gdnr_paged_attention", attention_case(), (65, ctypes.c_float(0.1))) == INVALID  # past the table
    assert call(lib, "gdnr_paged_attention", attention_case(), (-1, ctypes.c_float(0.1))) == INVALID
    assert call(lib, "gdnr_paged_attention", attention_case(), (64, ctypes.c_float(float("nan")))) == INVALID
    assert call(lib, "gdnr_paged_attention", attention_case(T=0), (64, ctypes.c_float(0.1))) == OK
    long = attention_case(T=1, N=1, width=1 << 12)  # its pieces' workspace is missing
    assert call(lib, "gdnr_paged_attention", long, (1 << 16, ctypes.c_float(0.1))) == INVALID


def test_workspace_counts():
    assert gdnr_lib.prefill_workspace(8, 2, 16, 32, 128, torch.bfloat16, torch.bfloat16) == 0
    whole = gdnr_lib.prefill_workspace(4096, 1, 16, 32, 128, torch.bfloat16, torch.bfloat16)
    assert 0 < whole < gdnr_lib.prefill_workspace(4096, 1, 16, 32, 128, torch.bfloat16, torch.float32)
    assert gdnr_lib.paged_attention_workspace(1, 1, 16, 4, 128, 256) == 0
    assert gdnr_lib.paged_attention_workspace(1, 1, 16, 4, 128, 1 << 16) > 0
    for bad in ((-1, 1, 16, 32, 128, torch.bfloat16, torch.bfloat16),):
        with pytest.raises(gdnr_lib.GdnrError):
            gdnr_lib.prefill_workspace(*bad)
    for bad in ((1, 1, 16, 0, 128, 100), (1, 1, 16, 3, 128, 100), (1, 1, 16, 4, 128, -1), (1 << 24, 1, 16, 4, 128, 100)):
        with pytest.raises(gdnr_lib.GdnrError):
            gdnr_lib.paged_attention_workspace(*bad)


def test_host_tensors_are_refused():
    x = torch.zeros(4, 1024, dtype=torch.bfloat16)
    g = torch.zeros(4, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        gp.gdn_prefill(x, g, g, torch.zeros(4), torch.zeros(4), torch.zeros(2, 4, 128, 128), torch.ones(1, dtype=torch.int32),
                       torch.tensor([0, 4], dtype=torch.int32))
    q, cache = torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        ga.qkv_norm_rope_append(q, q, q, torch.zeros(8, 64), i, cache, cache, i)
    with pytest.raises(ValueError):
        ga.paged_attention(q, cache, cache, i[None], i[:2], i[:1])


def test_rope_table_refusals():
    for args in ((4, 7), (4, 0)):
        with pytest.raises(ValueError):
            ga.rope_table(*args, device="cpu")
    with pytest.raises(ValueError):
        ga.rope_table(4, 8, device="cpu", inv_freq=torch.zeros(3))


def test_paged_cache_and_prefill_refusals_on_the_host():
    with pytest.raises(ValueError):
        ga.PagedKVCache(0, 16, 1, 64, device="cpu")
    cache = ga.PagedKVCache(3, 4, 1, 64, device="cpu")
    batch = cache.step([7], [9])
    assert batch.max_context == 9 and cache.free_pages == 0
    with pytest.raises(RuntimeError):
        cache.step([8], [1])
    ssm = rc.ReplaySSMCache(2, 4, 1, 2, 128, 32, device="cpu")
    with pytest.raises(ValueError):
        ssm.prefill([1], [3], torch.zeros(4, 320), torch.zeros(4, 2), torch.zeros(4, 2), torch.zeros(2), torch.zeros(2))


def test_oracle_recurrence_is_the_step_oracle():
    """gdn_sequences against the step written with explicit matrices."""
    r = np.random.RandomState(0)
    H, HV, V, K, T = 2, 4, 32, 128, 6
    mixed, a, b = r.randn(T, 2 * H * K + HV * V), r.randn(T, HV), r.randn(T, HV)
    a_log, dt_bias, state = r.rand(HV), r.rand(HV) - 4, 0.1 * r.randn(3, HV, V, K)
    out, final = sequence_oracle.gdn_sequences(mixed, a, b, a_log, dt_bias, state, [2, 1], [0, 4, 6], [True, False])
    mine = state.copy()
    mine[1] = 0
    for slot, rows in ((2, range(0, 4)), (1, range(4, 6))):
        for t in rows:
            o, mine = _step(mixed[t], a[t], b[t], a_log, dt_bias, mine, slot, H)
            assert np.abs(o - out[t]).max() < 1e-12
    assert np.abs(mine - final).max() < 1e-12


def _step(row, a, b, a_log, dt_bias, state, slot, H):
    """One token of one sequence, written with explicit matrices: S (I - beta k k^T) e^g + beta v k^T."""
    HV, V, K = state.shape[1:]
    state, out = state.copy(), np.zeros((HV, V))
    for hv in range(HV):
        h = hv // (HV // H)
        q, k = row[h * K:(h + 1) * K], row[(H + h) * K:(H + h + 1) * K]
        q, k = q / np.sqrt(q @ q + 1e-6), k / np.sqrt(k @ k + 1e-6)
        v = row[2 * H * K + hv * V:2 * H * K + (hv + 1) * V]
        beta, g = 1 / (1 + np.exp(-b[hv])), -np.exp(a_log[hv]) * np.log1p(np.exp(a[hv] + dt_bias[hv]))
        state[slot, hv] = np.exp(g) * state[slot, hv] @ (np.eye(K) - beta * np.outer(k, k)) + beta * np.outer(v, k)
        out[hv] = state[slot, hv] @ q * K ** -0.5
    return out, state


def test_oracle_rotation_keeps_norms_and_relative_positions():
    """A rotation keeps lengths, and scores depend on the distance alone."""
    r = np.random.RandomState(1)
    table = np64(ga.rope_table(64, 32, base=100.0, device="cpu"))
    for interleaved in (False, True):
        x, y = r.randn(1, 1, 64), r.randn(1, 1, 64)
        turn = lambda v, p: sequence_oracle.norm_rope(v, None, table, np.array([p]), interleaved)[0, 0]  # noqa: E731
        assert abs(np.linalg.norm(turn(x, 9)) - np.linalg.norm(x)) < 1e-6  # (the table is float32)
        assert abs(turn(x, 9) @ turn(y, 4) - turn(x, 45) @ turn(y, 40)) < 1e-5
    w = r.rand(64)
    x = r.randn(3, 2, 64)
    normed = sequence_oracle.norm_rope(x, w, table, np.zeros(3, int), False)
    assert np.abs((normed / w / (x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6))) - 1).max() < 1e-9


def np64(t):
    return t.double().numpy()


def test_oracle_attention_on_one_page_is_softmax():
    r = np.random.RandomState(2)
    q, k, v = r.randn(3, 2, 8), r.randn(1, 5, 1, 8), r.randn(1, 5, 1, 8)
    out = sequence_oracle.paged_attention(q, k, v, np.array([[0]]), [0, 3], [5])
    for t in range(3):
        for h in range(2):
            p = np.exp(q[t, h] @ k[0, :3 + t, 0].T * 8 ** -0.5)
            assert np.abs(out[t, h] - p @ v[0, :3 + t, 0] / p.sum()).max() < 1e-12


@pytest.mark.parametrize("prompt", [1024, 8192])
@pytest.mark.parametrize("decodes", [1, 3, 40])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (64, 8, 256), (16, 2, 256), (8, 8, 64), (40, 2, 128)])
@pytest.mark.parametrize("context", [12000, 131072])
def test_mixed_batches_take_little_workspace(prompt, decodes, heads, kv_heads, dim, context):
    """A few decodes beside a prompt's chunk. Eight workgroups of 16 rows a
    compute unit hold the decodes' pieces and two of at most 128 the prompt's;
    rounding pieces up, and rows of a tile that are no token's, at most double
    either. 256 compute units; 4 (dim + 2) bytes a row."""
    size = gdnr_lib.paged_attention_workspace(prompt + decodes, decodes + 1, heads, kv_heads, dim, context)
    rows = 2 * (8 * 256 * 16 + 2 * 256 * 128)
    assert size <= rows * 4 * (dim + 2)


def test_a_prompt_in_one_piece_takes_none_beside_a_decode():
    """The decodes' pieces alone: at most eight workgroups of 16 rows a compute unit, rounded up."""
    assert gdnr_lib.paged_attention_workspace(8192, 1, 32, 8, 128, 131072) == 0
    size = gdnr_lib.paged_attention_workspace(8193, 2, 32, 8, 128, 131072)
    assert 0 < size <= 2 * 8 * 256 * 16 * 4 * (128 + 2)


@pytest.mark.parametrize("state", [torch.bfloat16, torch.float32])
def test_a_long_prompt_among_single_tokens_is_walked_in_chunks(state):
    """900 tokens beside 63 sequences of one: a workspace for the prompt's
    chunks, which its tokens alone would take too, and little more; none where no
    sequence can be long."""
    size = lambda tokens, sequences: gdnr_lib.prefill_workspace(tokens, sequences, 16, 32, 128, torch.bfloat16, state)  # noqa: E731
    assert size(900, 1) <= size(963, 64) <= 2 * size(900, 1)
    assert size(2000, 1000) <= 2 * size(2000, 1)
    assert size(8 * 4, 8) == size(64, 64) == 0


def test_rope_table_under_any_default_device():
    """The angles are formed on the host whatever torch's default device is."""
    want = ga.rope_table(20, 16, device="cpu")
    freq = 10000.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    with torch.device("meta"):
        got, given = ga.rope_table(20, 16, device="cpu"), ga.rope_table(20, 16, device="cpu", inv_freq=freq)
    assert torch.equal(got, want) and torch.equal(given, want)
