"""The sequence operators' cases: what a program that serves a hybrid language
model (GDN layers with full-attention layers between them) has the GPU do
around the decode step of its GDN layers.

A case is a dict of plain values. kind:
  "prefill"    gdn_prefill: the gated delta rule over packed sequences of any
               length, from raw mixed_qkv / a / b rows, on a slot-indexed state
  "append"     qkv_norm_rope_append: an attention layer's q/k head norms, the
               position rotation and the append of k, v to a paged cache
  "attention"  paged_attention: new tokens (a chunk of a prompt, or one token)
               over that cache

The GDN sizes are those of the repository's benchmark and tests (H=16, HV=32,
K=V=128, the Qwen3.5-4B GDN layer, and its V=64 / 256 and odd-group variants);
the attention sizes are generic: heads of 64, 128 and 256, groups of 1 to 8.

With ``own`` false ``run`` computes the operators in elementary torch
operations in float32, rounded once at the end; with ``own`` true it calls this
package.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

_PKG = Path.cwd() / "fp8-replayssm-gdn-kernel_amd"
if str(_PKG) not in sys.path:
    sys.path.insert(0, str(_PKG))

own = False

K = 128
CHUNK = 64
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _prefill(name, sequences, tokens, dtype="bf16", state="bf16", heads=16, value_heads=32, value_dim=128, ragged=True):
    return dict(name=name, kind="prefill", sequences=sequences, tokens=tokens, ragged=ragged, dtype=dtype, state=state,
                heads=heads, value_heads=value_heads, value_dim=value_dim)


def _append(name, tokens, dim, rotary, heads, kv_heads, page, interleaved=False, norm=True, dtype="bf16"):
    return dict(name=name, kind="append", tokens=tokens, head_dim=dim, rotary=rotary, heads=heads, kv_heads=kv_heads,
                page=page, interleaved=interleaved, norm=norm, dtype=dtype)


def _attention(name, sequences, tokens, context, dim, heads, kv_heads, page, decodes=0, dtype="bf16"):
    return dict(name=name, kind="attention", sequences=sequences, tokens=tokens, context=context, head_dim=dim,
                heads=heads, kv_heads=kv_heads, page=page, decodes=decodes, dtype=dtype)


def listed():
    return [
        # eight sequences whose four drafted tokens each are verified: the
        # recurrent form, a few tokens on states that are read and written once
        _prefill("verify drafts", 8, 32, ragged=False),
        # one user's prompt of 8192 tokens: a long chain of chunks, few heads
        # to spread over the card
        _prefill("one prompt", 1, 8192),
        # a scheduler's prefill batch: ragged prompts, an empty and a
        # one-token sequence among them, some of them continued from a state
        _prefill("ragged prompts", 24, 16384),
        # another layer shape (12 value heads on 4 key heads) in f16, its
        # state kept in f32
        _prefill("f32 state", 3, 1531, dtype="f16", state="f32", heads=4, value_heads=12),
        # one decoded token: what one call costs
        _append("append one token", 1, 128, 128, 16, 4, 16),
        # a decode step of 64 sequences, a quarter of wide heads rotated
        _append("append decode", 64, 256, 64, 16, 4, 64),
        # a prompt's chunk
        _append("append chunk", 8192, 128, 128, 32, 8, 16),
        # a throughput prefill: interleaved pairs, no head norms, f16, pages
        # of an odd size
        _append("append interleaved", 14001, 64, 32, 32, 32, 48, interleaved=True, norm=False, dtype="f16"),
        # one decoded token over a long context: few rows, a long axis
        _attention("decode one", 1, 1, 8192, 128, 16, 4, 16, decodes=1),
        # a decode step of 64 ragged sequences, wide heads
        _attention("decode batch", 64, 64, 8192, 256, 16, 2, 64, decodes=64),
        # a chunk of 2048 new tokens over a cached context
        _attention("prompt chunk", 1, 2048, 8192, 128, 32, 8, 16),
        # chunked prefill beside decodes in one call: three prompts' chunks
        # and thirteen decodes, f16, narrow heads, pages of an odd size
        _attention("mixed batch", 16, 1213, 4096, 64, 16, 4, 48, decodes=13, dtype="f16"),
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------

def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw(rng):
    kind = rng.choice(["prefill", "prefill", "append", "attention", "attention"])
    if kind == "prefill":
        h, hv, v = rng.choice([(16, 32, 128)] * 4 + [(8, 16, 128), (4, 12, 128), (8, 8, 256), (8, 16, 64)])
        dtype = rng.choice(["bf16"] * 4 + ["f16", "f32"])
        n = _log_int(rng, 1, 64)
        case = _prefill("", n, n * _log_int(rng, 1, 8192 // n if n < 32 else 256), dtype,
                        rng.choice([dtype, dtype, "f32"]), h, hv, v, ragged=rng.random() < 0.8)
    elif kind == "append":
        dim, hkv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
        case = _append("", _log_int(rng, 1, 12000), dim, rng.choice([dim, dim // 2, dim // 4]),
                       hkv * rng.choice([1, 2, 4, 8]), hkv, rng.choice([16, 32, 48, 64, 256]), rng.random() < 0.3,
                       rng.random() < 0.8, rng.choice(["bf16", "bf16", "f16"]))
    else:
        dim, hkv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
        n = _log_int(rng, 1, 64)
        decodes = rng.choice([n, n, n - 1, n // 2])
        tokens = decodes + (n - decodes) * _log_int(rng, 2, 1024)
        case = _attention("", n, tokens, _log_int(rng, 16, 12000), dim, hkv * rng.choice([1, 2, 4, 8]), hkv,
                          rng.choice([16, 16, 32, 48, 64, 256]), decodes, rng.choice(["bf16", "bf16", "f16"]))
    del case["name"]
    return case


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _cost(case):
    """Device cost of a case, as bytes: what the plain form keeps is padded to
    the longest sequence, so a ragged batch of many is dear."""
    if case["kind"] == "append":
        return work(case)["bytes"]
    if case["kind"] == "prefill":
        lengths = _lengths(case)
        return int(lengths.max()) * len(lengths) * case["value_heads"] * case["value_dim"] * 4
    new, context = _contexts(case)
    return (len(new) * int(context.max()) * case["heads"] * (4 * int(new.max()) + 8 * case["head_dim"])) // 4


# ---------------------------------------------------------------------------
# sizes that a case fixes by itself
# ---------------------------------------------------------------------------

def _lengths(case):
    """Tokens of each sequence. A ragged batch of eight or more holds an empty
    sequence and one of a single token."""
    n, total = case["sequences"], case["tokens"]
    if not case["ragged"]:
        return np.full(n, total // n, dtype=np.int64)
    part = np.random.RandomState(n).uniform(0.2, 1.0, n)
    if n >= 8:
        part[n // 3], part[n // 2] = 0.0, 0.0
    lengths = np.floor(part * total / part.sum()).astype(np.int64)
    if n >= 8:
        lengths[n // 2] = 1
    lengths[0] += total - lengths.sum()
    return np.maximum(lengths, 0)


def _contexts(case):
    """(new tokens, context length with them) of each sequence: the decodes
    first, then the prompts' chunks."""
    n, decodes = case["sequences"], case["decodes"]
    r = np.random.RandomState(n + decodes)
    new = np.ones(n, dtype=np.int64)
    if n > decodes:
        rest = case["tokens"] - decodes
        part = r.uniform(0.4, 1.0, n - decodes)
        new[decodes:] = np.maximum(1, np.floor(part * rest / part.sum())).astype(np.int64)
        new[n - 1] = max(1, rest - int(new[decodes:n - 1].sum()))
    past = np.floor(np.exp(r.uniform(np.log(0.3), 0, n)) * case["context"]).astype(np.int64)
    past[0] = case["context"]
    return new, np.maximum(past, new)


# ---------------------------------------------------------------------------
# inputs (plain torch, from the seed alone)
# ---------------------------------------------------------------------------

def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _i32(x):
    return torch.from_numpy(np.asarray(x).astype(np.int32)).cuda()


def _starts(lengths):
    return np.concatenate([[0], np.cumsum(lengths)])


def _prepare_prefill(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths = _lengths(case)
    n, T = len(lengths), int(lengths.sum())
    H, HV, V, dt = case["heads"], case["value_heads"], case["value_dim"], DTYPES[case["dtype"]]
    # long-memory gates (gamma around 0.95 a token), the benchmark's
    a_log = torch.rand(HV, generator=gen, device="cuda")
    dt_bias = torch.rand(HV, generator=gen, device="cuda") - 4.0
    mixed = _rand(gen, T, 2 * H * K + HV * V).to(dt)
    a, b = _rand(gen, T, HV).to(dt), _rand(gen, T, HV).to(dt)
    # a cache of slots, 0 the null slot, the sequences in shuffled slots;
    # every third sequence starts from nothing
    state = (0.02 * _rand(gen, n + 1, HV, V, K)).to(DTYPES[case["state"]])
    slots = torch.randperm(n, generator=gen, device="cuda").to(torch.int32) + 1
    started = torch.arange(n, device="cuda") % 3 != 2
    return dict(mixed=mixed, a=a, b=b, a_log=a_log, dt_bias=dt_bias, state=state, slots=slots, started=started,
                cu=_i32(_starts(lengths)), heads=H, longest=int(lengths.max()), gather=_padded(lengths))


def _padded(lengths):
    """Row of each (sequence, position) of the batch padded to its longest
    sequence, one past the last row where there is none."""
    n, longest, total = len(lengths), max(1, int(lengths.max())), int(lengths.sum())
    at = _starts(lengths)[:-1, None] + np.arange(longest)
    return torch.from_numpy(np.where(np.arange(longest) < lengths[:, None], at, total).reshape(n, longest)).cuda()


def _rope_table(positions, rotary, base=1e6):
    """[positions, rotary]: cosines, then sines."""
    freq = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=-1).float()


def _prepare_append(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, D, HQ, HKV, dt = case["tokens"], case["head_dim"], case["heads"], case["kv_heads"], DTYPES[case["dtype"]]
    q, k, v = _rand(gen, T, (HQ + 2 * HKV) * D).to(dt).split([HQ * D, HKV * D, HKV * D], dim=-1)
    pages = -(-T // case["page"]) + 3
    cache = [_rand(gen, pages, case["page"], HKV, D).to(dt) for _ in range(2)]
    slots = torch.randperm(pages * case["page"], generator=gen, device="cuda")[:T].to(torch.int32)
    positions = torch.randint(0, 16384, (T,), generator=gen, device="cuda", dtype=torch.int32)
    weights = [1.0 + 0.2 * _rand(gen, D) for _ in range(2)] if case["norm"] else [None, None]
    return dict(q=q.view(T, HQ, D), k=k.view(T, HKV, D), v=v.view(T, HKV, D), k_cache=cache[0], v_cache=cache[1],
                slots=slots, positions=positions, table=_rope_table(16384, case["rotary"]), q_weight=weights[0],
                k_weight=weights[1], interleaved=case["interleaved"])


def _prepare_attention(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, context = _contexts(case)
    n, T, page = len(new), int(new.sum()), case["page"]
    D, HQ, HKV, dt = case["head_dim"], case["heads"], case["kv_heads"], DTYPES[case["dtype"]]
    held = -(-context // page)
    # pages in shuffled order, three of them nobody's; a row of the table is
    # as wide as the longest sequence needs
    pages = int(held.sum()) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    at = _starts(held)[:-1, None] + np.arange(int(held.max()))
    table = order[torch.from_numpy(np.where(np.arange(int(held.max())) < held[:, None], at, 0)).cuda()]
    k_cache, v_cache = (torch.empty(pages, page, HKV, D, dtype=dt, device="cuda").normal_(generator=gen) for _ in range(2))
    # normed and rotated queries: scores of a few units, some keys far ahead
    q = (1.5 * _rand(gen, T, HQ, D)).to(dt)
    return dict(q=q, k_cache=k_cache, v_cache=v_cache, table=table.contiguous(), cu=_i32(_starts(new)),
                context=_i32(context), longest=int(new.max()), most=int(context.max()), gather=_padded(new))


def prepare(case, seed):
    make = {"prefill": _prepare_prefill, "append": _prepare_append, "attention": _prepare_attention}[case["kind"]]
    return dict(make(case, seed), kind=case["kind"])


# ---------------------------------------------------------------------------
# the plain forms, in float32
# ---------------------------------------------------------------------------

def _plain_prefill(s):
    H, (slots_total, HV, V, _) = s["heads"], s["state"].shape
    G, (n, longest), T = HV // H, s["gather"].shape, s["mixed"].shape[0]
    C = min(CHUNK, longest)
    chunks = -(-longest // C)
    # the gates and the unit keys and queries of every token, then the batch
    # padded to whole chunks with tokens that change nothing
    x = s["mixed"].float()
    q, k, v = x.split([H * K, H * K, HV * V], dim=-1)
    q, k = q.reshape(T, H, K), k.reshape(T, H, K)
    q = q / ((q * q).sum(-1, keepdim=True) + EPS).sqrt()
    k = k / ((k * k).sum(-1, keepdim=True) + EPS).sqrt()
    z = s["a"].float() + s["dt_bias"]
    g = -s["a_log"].exp() * torch.where(z > 20.0, z, torch.log1p(z.clamp(max=20.0).exp()))
    beta = 1.0 / (1.0 + (-s["b"].float()).exp())

    rows = torch.nn.functional.pad(s["gather"], (0, chunks * C - longest), value=T)

    def chunked(y):  # [T, heads, width] -> [n, heads, chunks, C, width]
        y = torch.cat([y, y.new_zeros(1, *y.shape[1:])])[rows]
        return y.view(n, chunks, C, *y.shape[2:]).permute(0, 3, 1, 2, 4).contiguous()

    q, k, v = chunked(q), chunked(k), chunked(v.reshape(T, HV, V))
    g, beta = chunked(g[..., None])[..., 0], chunked(beta[..., None])[..., 0]
    total = g.cumsum(-1)
    t = torch.arange(C, device=x.device)
    decay = (total[..., :, None] - total[..., None, :]).masked_fill(t[:, None] < t, -math.inf).exp()
    kk = (k @ k.transpose(-1, -2).contiguous()).repeat_interleave(G, dim=1)
    a = (q @ k.transpose(-1, -2).contiguous()).repeat_interleave(G, dim=1) * decay
    m = (kk * decay * beta[..., None]).masked_fill(t[:, None] == t, 0.0)
    del kk, decay
    # (I + M)^-1 of a strictly lower M: the product of I + (-M)^(2^j)
    inverse, power = torch.eye(C, device=x.device) - m, m
    for _ in range(max(0, (C - 1).bit_length() - 1)):
        power = power @ power
        inverse = inverse + inverse @ power
    del m, power
    at = s["slots"].long()
    S = s["state"][at].float() * s["started"][:, None, None, None]
    outs = []
    for c in range(chunks):
        kc, qc = (y[:, :, c].repeat_interleave(G, dim=1) for y in (k, q))
        from_start = total[:, :, c, :, None].exp()
        u = inverse[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - from_start * (kc @ S.transpose(-1, -2).contiguous())))
        outs.append(from_start * (qc @ S.transpose(-1, -2).contiguous()) + a[:, :, c] @ u)
        to_end = (total[:, :, c, -1:] - total[:, :, c]).exp()[..., None]
        S = total[:, :, c, -1, None, None].exp() * S + u.transpose(-1, -2).contiguous() @ (to_end * kc)
    out = (torch.stack(outs, 1).transpose(2, 3).reshape(n, chunks * C, HV, V) * K ** -0.5)[:, :longest]
    packed = torch.empty(T + 1, HV, V, dtype=s["mixed"].dtype, device=x.device)
    packed[s["gather"].reshape(-1)] = out.reshape(-1, HV, V).to(packed.dtype)
    s["state"][at] = S.to(s["state"].dtype)
    return {"out": packed[:T], "state": s["state"]}


def _plain_append(s):
    row = s["table"][s["positions"].long()][:, None]
    half = row.shape[-1] // 2
    cos, sin = row[..., :half], row[..., half:]

    def rotated(x, weight):
        y = x.float()
        if weight is not None:
            y = y / ((y * y).mean(-1, keepdim=True) + EPS).sqrt() * weight
        first = slice(0, 2 * half, 2) if s["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if s["interleaved"] else slice(half, 2 * half)
        x0, x1 = y[..., first], y[..., second]
        z = y.clone()
        z[..., first], z[..., second] = x0 * cos - x1 * sin, x1 * cos + x0 * sin
        return z.to(x.dtype)

    at = s["slots"].long()
    s["k_cache"].view(-1, *s["k"].shape[1:])[at] = rotated(s["k"], s["k_weight"])
    s["v_cache"].view(-1, *s["v"].shape[1:])[at] = s["v"]
    return {"q": rotated(s["q"], s["q_weight"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    (T, HQ, D), (n, longest) = s["q"].shape, s["gather"].shape
    HKV = s["k_cache"].shape[2]
    G, most = HQ // HKV, s["most"]
    k, v = (c[s["table"].long()].reshape(n, -1, HKV, D)[:, :most].permute(0, 2, 1, 3).float() for c in
            (s["k_cache"], s["v_cache"]))
    q = torch.cat([s["q"], s["q"].new_zeros(1, HQ, D)])[s["gather"]].float()
    q = q.view(n, longest, HKV, G, D).permute(0, 2, 3, 1, 4).reshape(n, HKV, G * longest, D)
    p = (q @ k.transpose(-1, -2).contiguous() * D ** -0.5).view(n, HKV, G, longest, most)
    last = s["context"][:, None] - (s["cu"][1:] - s["cu"][:-1])[:, None] + torch.arange(longest, device=q.device)
    seen = torch.arange(most, device=q.device) <= last[..., None]
    seen = seen & (torch.arange(most, device=q.device) < s["context"][:, None, None])
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    norm = p.sum(-1, keepdim=True)
    o = p.view(n, HKV, G * longest, most) @ v.contiguous() / norm.view(n, HKV, -1, 1).clamp(min=1e-30)
    o = o.view(n, HKV, G, longest, D).permute(0, 3, 1, 2, 4).reshape(-1, HQ, D)
    packed = torch.empty(T + 1, HQ, D, dtype=s["q"].dtype, device=q.device)
    packed[s["gather"].reshape(-1)] = o.to(packed.dtype)
    return {"out": packed[:T]}


# ---------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------

def _own_prefill(s):
    from gdn_prefill import gdn_prefill

    out = gdn_prefill(s["mixed"], s["a"], s["b"], s["a_log"], s["dt_bias"], s["state"], s["slots"], s["cu"],
                      has_initial_state=s["started"])
    return {"out": out, "state": s["state"]}


def _own_append(s):
    from gdn_attention import qkv_norm_rope_append

    q = qkv_norm_rope_append(s["q"], s["k"], s["v"], s["table"], s["positions"], s["k_cache"], s["v_cache"], s["slots"],
                             q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, interleaved=s["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    from gdn_attention import paged_attention

    return {"out": paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["context"],
                                   max_context=s["most"])}


_PLAIN = {"prefill": _plain_prefill, "append": _plain_append, "attention": _plain_attention}
_OWN = {"prefill": _own_prefill, "append": _own_append, "attention": _own_attention}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---------------------------------------------------------------------------
# the work a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "prefill":
        lengths = _lengths(case)
        T, H, HV, V = int(lengths.sum()), case["heads"], case["value_heads"], case["value_dim"]
        cells = HV * V * K * DTYPES[case["state"]].itemsize
        read = int((np.arange(len(lengths)) % 3 != 2).sum())
        # S k, the rank-1 update and S q of every token
        return {"bytes": T * es * (2 * H * K + 2 * HV * V + 2 * HV) + cells * (read + len(lengths)),
                "flops": 6 * T * HV * V * K}
    D, HQ, HKV = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        T = case["tokens"]
        table = min(T, 16384) * 4 * case["rotary"]
        return {"bytes": 2 * T * es * D * (HQ + 2 * HKV) + 8 * T + table, "flops": 6 * T * D * (HQ + HKV)}
    new, context = _contexts(case)
    pairs = int((new * (2 * context - new + 1) // 2).sum())
    return {"bytes": es * D * (2 * HKV * int(context.sum()) + 2 * HQ * int(new.sum())), "flops": 4 * D * HQ * pairs}


# ---------------------------------------------------------------------------
# the same in 64 bits, written from the definitions
# ---------------------------------------------------------------------------

def _exact_prefill(case, seed):
    x = _prepare_prefill(case, seed)
    lengths = _lengths(case)
    H, HV, V = case["heads"], case["value_heads"], case["value_dim"]
    T, n, group = x["mixed"].shape[0], len(lengths), HV // H
    unit = lambda y: y / torch.sqrt((y * y).sum(-1, keepdim=True) + EPS)  # noqa: E731
    rows = x["mixed"].double()
    q = unit(rows[:, :H * K].reshape(T, H, K)).repeat_interleave(group, dim=1)
    k = unit(rows[:, H * K:2 * H * K].reshape(T, H, K)).repeat_interleave(group, dim=1)
    v = rows[:, 2 * H * K:].reshape(T, HV, V)
    gamma = (-x["a_log"].double().exp() * torch.nn.functional.softplus(x["a"].double() + x["dt_bias"].double())).exp()
    beta = torch.sigmoid(x["b"].double())
    state = x["state"].double()
    # longest sequences first, so that those still running are a prefix; one
    # token of each at a time
    order = np.argsort(-lengths, kind="stable")
    slots, start = x["slots"].long()[order], torch.from_numpy(_starts(lengths)[:-1][order]).cuda()
    S = state[slots] * x["started"].double()[order][:, None, None, None]
    out = torch.empty(T, HV, V, dtype=torch.float64, device="cuda")
    for t in range(int(lengths.max())):
        live = int((lengths > t).sum())
        at, P = start[:live] + t, S[:live]
        P.mul_(gamma[at][..., None, None])
        u = beta[at][..., None] * (v[at] - (P @ k[at][..., None])[..., 0])
        P.addcmul_(u[..., None], k[at][..., None, :])
        out[at] = (P @ q[at][..., None])[..., 0] * K ** -0.5
    state[slots] = S
    return {"out": out, "state": state}


def _exact_append(case, seed):
    x = _prepare_append(case, seed)
    half, D = case["rotary"] // 2, case["head_dim"]
    angle = torch.complex(*x["table"].double()[x["positions"].long()].split(half, dim=-1))[:, None]

    def turned(y, weight):
        y = y.double()
        if weight is not None:
            y = y * weight.double() * torch.rsqrt((y * y).sum(-1, keepdim=True) / D + EPS)
        head, tail = y[..., :2 * half], y[..., 2 * half:]
        pairs = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * angle)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, tail], dim=-1)

    page, at = case["page"], x["slots"].long()
    caches = [x["k_cache"].double(), x["v_cache"].double()]
    caches[0][at // page, at % page] = turned(x["k"], x["k_weight"])
    caches[1][at // page, at % page] = x["v"].double()
    return {"q": turned(x["q"], x["q_weight"]), "k_cache": caches[0], "v_cache": caches[1]}


def _exact_attention(case, seed):
    x = _prepare_attention(case, seed)
    new, context = _contexts(case)
    D, page, group = case["head_dim"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    for i, first in enumerate(_starts(new)[:-1]):
        L, C = int(new[i]), int(context[i])
        position = torch.arange(C, device="cuda")
        where = x["table"][i].long()[position // page], position % page
        k, v = x["k_cache"][where].double(), x["v_cache"][where].double()
        visible = position[None, :] <= (C - L + torch.arange(L, device="cuda"))[:, None]
        for h in range(case["heads"]):
            score = x["q"][first:first + L, h].double() @ k[:, h // group].T.contiguous() / math.sqrt(D)
            score = torch.where(visible, score, torch.full_like(score, -math.inf))
            out[first:first + L, h] = torch.softmax(score, dim=-1) @ v[:, h // group].contiguous()
    return {"out": out}


def exact(case, seed):
    return {"prefill": _exact_prefill, "append": _exact_append, "attention": _exact_attention}[case["kind"]](case, seed)
