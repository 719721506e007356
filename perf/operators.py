"""The operators of generation from a key/value cache, in their plain form and
as the framework's calls: writing a paged cache (rotary embedding included,
8-bit storage where asked for) and reading it back, attention of new tokens
over it, and the adjustment of logits before a token is chosen.

A cache layer is k and v, [pages, KV heads, page size, head dim], in the
model's type or in float8_e4m3fn with one exponent e for each (page, head,
token) in k_exp and v_exp (int8): the value is the stored number times 2^e.
Sequence b's token at position p is at [page_table[b, p // size], :, p % size].
The rows of a step are the new tokens, sequence after sequence: sequence b's
are row_start[b] .. row_start[b + 1] - 1, and they are its last tokens, so that
its length with them is kv_len[b].
"""
from __future__ import annotations

import functools
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# query heads, key/value heads, head dim of the model presets
HEADS = {"plumbing": (8, 4, 32), "tiny": (10, 2, 32), "125m": (12, 4, 64), "small": (18, 6, 64), "medium": (32, 8, 64),
         "1b": (16, 8, 128), "7b": (32, 8, 128)}
THETA = 10_000.0


def listed():
    return [
        # a single prompt's next token, on the smallest preset: latency alone
        {"name": "decode_plumbing", "kind": "attend", "size": "plumbing", "dtype": "bf16", "fp8": False, "batch": 1,
         "new": 1, "length": 128, "page": 16},
        # a batch of answers being written, lengths as they come
        {"name": "decode_1b_ragged", "kind": "attend", "size": "1b", "dtype": "bf16", "fp8": False, "batch": 32,
         "new": 1, "length": 2048, "page": 64},
        # a few long documents, cache in 8 bits
        {"name": "decode_7b_long_fp8", "kind": "attend", "size": "7b", "dtype": "bf16", "fp8": True, "batch": 4,
         "new": 1, "length": 32768, "page": 64},
        # long prompts taken in pieces: 1024 new tokens each over what is there
        {"name": "chunk_7b", "kind": "attend", "size": "7b", "dtype": "bf16", "fp8": False, "batch": 2, "new": 1024,
         "length": 8192, "page": 64},
        # a batch of whole prompts of different lengths
        {"name": "prompts_1b_fp16", "kind": "attend", "size": "1b", "dtype": "fp16", "fp8": False, "batch": 8,
         "new": 2048, "length": 2048, "page": 32},
        # a model kept in float32, a short follow-up of odd length
        {"name": "chunk_tiny_fp32", "kind": "attend", "size": "tiny", "dtype": "fp32", "fp8": False, "batch": 3,
         "new": 77, "length": 701, "page": 16},
        # the cache written for one new token of each of 32 answers
        {"name": "write_1b_decode", "kind": "write", "size": "1b", "dtype": "bf16", "fp8": False, "batch": 32,
         "new": 1, "length": 2048, "page": 64},
        # prompts written in 8 bits, and the sequences read back
        {"name": "restore_125m_fp8", "kind": "restore", "size": "125m", "dtype": "bf16", "fp8": True, "batch": 16,
         "new": 1024, "length": 1024, "page": 32},
        # one token appended to long sequences, which are then read back whole
        {"name": "restore_7b_fp16", "kind": "restore", "size": "7b", "dtype": "fp16", "fp8": False, "batch": 4,
         "new": 1, "length": 8192, "page": 128},
        # one answer's next token: penalties and a bias, no grammar
        {"name": "logits_one", "kind": "logits", "dtype": "bf16", "batch": 1, "vocab": 32000, "history": 200,
         "bias": "shared", "mask": "", "view": True},
        # a served batch with everything on: long histories, a grammar for each
        {"name": "logits_batch", "kind": "logits", "dtype": "bf16", "batch": 64, "vocab": 128256, "history": 2048,
         "bias": "rows", "mask": "bits", "view": False},
        # one layer's step as generation runs it: rotate and write, then attend
        {"name": "layer_7b_decode", "kind": "layer", "size": "7b", "dtype": "bf16", "fp8": False, "batch": 16, "new": 1,
         "length": 4096, "page": 64},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["attend", "attend", "attend", "write", "restore", "logits", "layer"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        if kind == "logits":
            return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, 64), "vocab": rng.choice(
                [8192, 32000, 128256, _log_int(rng, 500, 128256)]), "history": _log_int(rng, 1, 2048),
                "bias": rng.choice(["", "shared", "rows"]), "mask": rng.choice(["", "bits", "bools"]),
                "view": rng.random() < 0.5}
        case = {"kind": kind, "size": rng.choice(list(HEADS)), "dtype": dtype, "fp8": rng.random() < 0.4,
                "batch": _log_int(rng, 1, 64), "new": 1, "length": _log_int(rng, 1, 32768),
                "page": rng.choice([16, 32, 64, 128, 256])}
        if rng.random() < 0.5:  # a chunk, up to a whole prompt
            case["new"] = min(_log_int(rng, 2, 2048), case["length"])
        if kind in ("write", "layer"):  # what is stored in 8 bits is returned as values, by reading it back
            case["fp8"] = False
        H, KV, hd = HEADS[case["size"]]
        tokens = case["batch"] * case["length"]
        # what the plain form holds at once, and what float32 takes longer for
        if tokens * KV * hd > 2**27 or case["batch"] * case["new"] * case["length"] * H > 2**29:
            continue
        if work(case)["flops"] > (2.4e11 if dtype != "fp32" else 3e10):
            continue
        return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """(kv_len, new tokens) of each sequence: one is as long as the case says,
    the others are anything up to that."""
    rng = random.Random(f"{case['batch']} {case['new']} {case['length']}")
    kv, new = [case["length"]], [case["new"]]
    for _ in range(case["batch"] - 1):
        n = case["new"] if case["new"] == 1 else rng.randint(1, case["new"])
        new.append(n)
        kv.append(n if case["new"] == case["length"] else rng.randint(n, case["length"]))
    return kv, new


def work(case):
    esz = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "logits":
        B, V = case["batch"], case["vocab"]
        extra = {"": 0, "shared": 4 * V, "rows": 4 * B * V}[case["bias"]]
        extra += {"": 0, "bits": B * V / 8, "bools": B * V}[case["mask"]]
        return {"bytes": B * V * (esz + 4) + 8 * sum(_history_lengths(case)[0]) + extra, "flops": 6.0 * B * V}
    H, KV, hd = HEADS[case["size"]]
    kv, new = _lengths(case)
    T, L = sum(new), sum(kv)
    token = 2 * KV * (hd + 1 if case["fp8"] else hd * esz)  # a cached token, keys and values
    written = T * (esz * hd * (2 * H + 2 * KV) + 2 * esz * hd) + T * token  # qkv read, q and the cache written, tables
    seen = sum(n * l - n * (n - 1) // 2 for n, l in zip(new, kv))
    attend = {"bytes": 2 * T * H * hd * esz + L * token, "flops": 4.0 * H * hd * seen}
    if case["kind"] == "attend":
        return attend
    if case["kind"] == "write":
        return {"bytes": written, "flops": 6.0 * T * (H + KV) * hd}
    if case["kind"] == "restore":
        return {"bytes": written + L * (token + 2 * KV * hd * esz), "flops": 6.0 * T * (H + KV) * hd}
    # the layer's step: the cache that was there is read, the new tokens are only written
    return {"bytes": written + T * H * hd * esz + (L - T) * token, "flops": attend["flops"] + 6.0 * T * (H + KV) * hd}


def _history_lengths(case):
    rng = random.Random(f"{case['batch']} {case['history']}")
    n = [case["history"]] + [rng.randint(1, case["history"]) for _ in range(case["batch"] - 1)]
    return n, [rng.randint(0, x) for x in n]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "logits":
        return _prepare_logits(case, dtype, g)
    H, KV, hd = HEADS[case["size"]]
    kv, new = _lengths(case)
    B, T, page = len(kv), sum(new), case["page"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    per_seq = -(-max(kv) // page)
    n_pages = sum(-(-n // page) for n in kv) + 3
    # the pages lie in any order, as a pool that sequences come and go in has them
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros(B, per_seq, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(kv):
        m = -(-n // page)
        table[b, :m] = order[at : at + m]
        at += m
    shape = (n_pages, KV, page, hd)
    state = {"case": case, "heads": (H, KV, hd), "dtype": dtype, "rows": T, "max_new": max(new), "max_len": max(kv),
             "tokens": sum(kv), "table": table,
             "row_start": torch.tensor(starts, dtype=torch.int32, device=DEV),
             "kv_len": torch.tensor(kv, dtype=torch.int32, device=DEV),
             "kv_start": torch.tensor([sum(kv[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV),
             "k_exp": None, "v_exp": None}
    for name in ("k", "v"):
        x = torch.randn(shape, device=DEV, generator=g, dtype=dtype)
        if case["fp8"]:
            # heads and tokens of different sizes, as they are in a model
            x = x.float() * (0.25 + 2 * torch.rand(shape[:3], device=DEV, generator=g))[..., None]
            state[name], state[name + "_exp"] = _to_fp8(x, dtype)
        else:
            state[name] = x
    if case["kind"] == "attend":
        state["q"] = torch.randn(T, H * hd, device=DEV, generator=g, dtype=dtype)
    else:
        state["qkv"] = torch.randn(T, (H + 2 * KV) * hd, device=DEV, generator=g, dtype=dtype)
        inv = THETA ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
        angle = torch.arange(max(kv), device=DEV, dtype=torch.float64)[:, None] * inv
        angle = torch.cat([angle, angle], 1)
        state["cos"], state["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
    return state


def _prepare_logits(case, dtype, g):
    B, V, n = case["batch"], case["vocab"], case["history"]
    rows = 3 if case["view"] else 1  # the last position's rows of [B, 3, V], or a tensor of their own
    logits = (3 * torch.randn(B, rows, V, device=DEV, generator=g)).to(dtype)[:, -1]
    # texts repeat: most tokens are among the first few hundred ids
    far = torch.randint(0, V, (B, n), device=DEV, generator=g)
    near = torch.randint(0, min(V, 300), (B, n), device=DEV, generator=g)
    tokens = torch.where(torch.rand(B, n, device=DEV, generator=g) < 0.7, near, far)
    lengths, prompts = _history_lengths(case)
    rand = lambda lo, hi: lo + (hi - lo) * torch.rand(B, device=DEV, generator=g)  # noqa: E731
    state = {"case": case, "logits": logits, "tokens": tokens,
             "lengths": torch.tensor(lengths, device=DEV, dtype=torch.int32),
             "prompts": torch.tensor(prompts, device=DEV, dtype=torch.int32),
             "repetition": rand(1.0, 1.5), "presence": rand(0.0, 1.0), "frequency": rand(0.0, 0.5),
             "bias": None, "mask": None}
    if case["bias"]:
        shape = (V,) if case["bias"] == "shared" else (B, V)
        state["bias"] = torch.randn(shape, device=DEV, generator=g) * (torch.rand(shape, device=DEV, generator=g) < 0.05)
    if case["mask"] == "bits":
        state["mask"] = torch.randint(-(2**31), 2**31, (B, -(-V // 32)), device=DEV, generator=g).to(torch.int32)
    elif case["mask"] == "bools":
        state["mask"] = torch.rand(B, V, device=DEV, generator=g) < 0.5
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    ops, LayerCache, CacheStep = _framework()
    kind = s["case"]["kind"]
    if kind == "logits":
        return ops.process_logits(s["logits"], tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompts"],
                                  repetition_penalty=s["repetition"], presence_penalty=s["presence"],
                                  frequency_penalty=s["frequency"], bias=s["bias"], mask=s["mask"])
    H, KV, hd = s["heads"]
    layer = LayerCache(s["k"], s["v"], s["k_exp"], s["v_exp"])
    step = CacheStep(s["row_start"], s["kv_len"], s["table"], s["rows"], s["max_new"], s["max_len"])
    if kind == "attend":
        return ops.paged_attention(s["q"], layer, step, H, hd**-0.5)
    q = ops.kv_cache_write(s["qkv"], layer, step, H, s["cos"], s["sin"])
    if kind == "write":
        return q, s["k"], s["v"]
    if kind == "restore":
        return q, *ops.kv_cache_read(layer, s["table"], s["kv_start"], s["tokens"], s["dtype"])
    return q, ops.paged_attention(q, layer, step, H, hd**-0.5), s["k"], s["v"]


@functools.lru_cache(maxsize=None)
def _framework():
    package = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cs244c-llama-zero_amd")
    if os.path.abspath(package) not in sys.path:
        sys.path.insert(0, os.path.abspath(package))
    from lzhip import ops
    from lzhip.cache import CacheStep, LayerCache

    return ops, LayerCache, CacheStep


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "logits":
        return _plain_logits(s)
    if kind == "attend":
        return _plain_attention(s, s["q"])
    q = _plain_write(s)
    if kind == "write":
        return q, s["k"], s["v"]
    if kind == "restore":
        return q, *_plain_read(s)
    return q, _plain_attention(s, q), s["k"], s["v"]


def _pow2(e):
    """2^e for integers -126..127, as float32."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to_fp8(x, dtype):
    """x (float32) as (float8_e4m3fn, int8 exponents over the last dimension):
    the smallest exponent e with max |x| <= 448 * 2^e, 0 where all are zero;
    -120..120, and -15..7 for a model in float16, which holds every multiple of
    2^-24 up to 57344 (larger ones become that)."""
    m, ex = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0, ex - 9 + (m > 0.875), torch.zeros_like(ex))
    e = e.clamp(-15, 7) if dtype == torch.float16 else e.clamp(-120, 120)
    q = (x * _pow2(-e)[..., None]).clamp(-448, 448)
    return q.to(torch.float8_e4m3fn), e.to(torch.int8)


def _values(pages, exps):
    """The values of gathered pages, float32."""
    return pages.float() if exps is None else pages.view(torch.float8_e4m3fn).float() * _pow2(exps)[..., None]


def _rows_of(s):
    """(sequence, position) of each row of the step."""
    r = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(s["row_start"][1:], r.to(torch.int32), right=True)
    return b, s["kv_len"][b] - s["row_start"][b + 1] + r


def _plain_write(s):
    H, KV, hd = s["heads"]
    b, pos = _rows_of(s)
    x = s["qkv"].float().view(-1, H + 2 * KV, hd)
    c, sn = s["cos"].float()[pos][:, None], s["sin"].float()[pos][:, None]
    qk = x[:, : H + KV]
    half = torch.cat([-qk[..., hd // 2 :], qk[..., : hd // 2]], -1)
    qk = qk * c + half * sn
    size = s["case"]["page"]
    page, slot = s["table"][b, pos // size].long(), pos % size
    for name, y in (("k", qk[:, H:]), ("v", x[:, H + KV :])):
        if s["case"]["fp8"]:
            y, e = _to_fp8(y, s["dtype"])
            s[name].view(torch.uint8)[page, :, slot] = y.view(torch.uint8)
            s[name + "_exp"][page, :, slot] = e
        else:
            s[name][page, :, slot] = y.to(s["dtype"])
    return qk[:, :H].reshape(-1, H * hd).to(s["dtype"])


def _plain_read(s):
    KV, hd = s["heads"][1:]
    size = s["case"]["page"]
    r = torch.arange(s["tokens"], device=DEV)
    b = torch.searchsorted(s["kv_start"][1:], r.to(torch.int32), right=True)
    pos = r - s["kv_start"][b]
    page, slot = s["table"][b, pos // size].long(), pos % size
    out = []
    for name in ("k", "v"):
        p, e = s[name], s[name + "_exp"]
        p = (p if e is None else p.view(torch.uint8))[page, :, slot]
        out.append(_values(p, None if e is None else e[page, :, slot]).to(s["dtype"]).view(-1, KV * hd))
    return out


def _plain_attention(s, q):
    H, KV, hd = s["heads"]
    size, L, N, G = s["case"]["page"], s["max_len"], s["max_new"], H // KV
    table = s["table"][:, : -(-L // size)].long()
    B = table.shape[0]
    whole = []
    for name in ("k", "v"):
        p, e = s[name], s[name + "_exp"]
        x = _values((p if e is None else p.view(torch.uint8))[table], None if e is None else e[table])
        whole.append(x.transpose(1, 2).reshape(B, KV, -1, hd)[:, :, :L])
    k, v = whole
    new = s["row_start"][1:] - s["row_start"][:-1]
    i = torch.arange(N, device=DEV)
    row = (s["row_start"][:-1, None] + i).clamp(max=s["rows"] - 1).long()
    x = q.float()[row].view(B, N, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(B, KV, G * N, hd)
    score = (x @ k.transpose(2, 3).contiguous()).view(B, KV, G, N, L) * hd**-0.5
    last = s["kv_len"][:, None] - new[:, None] + i  # the last position that new token i sees
    hidden = torch.arange(L, device=DEV) > last[:, :, None]
    score = score.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    y = (p.view(B, KV, G * N, L) @ v.contiguous()).view(B, KV, G, N, hd) / p.sum(-1, keepdim=True)
    b, pos = _rows_of(s)
    y = y.permute(0, 3, 1, 2, 4).reshape(B, N, H * hd)
    return y[b, pos - (s["kv_len"] - new)[b]].to(q.dtype)


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    i = torch.arange(s["tokens"].shape[1], device=DEV)
    inside = (i < s["lengths"][:, None]).float()
    answer = inside * (i >= s["prompts"][:, None])
    seen = torch.zeros(B, V, device=DEV).scatter_add_(1, s["tokens"], inside) > 0
    count = torch.zeros(B, V, device=DEV).scatter_add_(1, s["tokens"], answer)
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        allowed = s["mask"]
        if allowed.dtype == torch.int32:
            v = torch.arange(V, device=DEV)
            allowed = (allowed[:, v // 32] >> (v % 32)) & 1 != 0
        x = x.masked_fill(~allowed, -math.inf)
    return x


# ---------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logits":
        return _exact_logits(s)
    H, KV, hd = s["heads"]
    kv, new = _lengths(case)
    if case["kind"] == "attend":
        return _exact_attention(s, s["q"].double(), kv, new)
    x = s["qkv"].double().view(-1, H + 2 * KV, hd)
    rounded = x.clone()  # the rotation with its products and sums in 32 bits, from which 8 bits are formed
    at = 0
    for n, l in zip(new, kv):
        c, sn = s["cos"][l - n : l, None].double(), s["sin"][l - n : l, None].double()
        a, b = x[at : at + n, : H + KV, : hd // 2].clone(), x[at : at + n, : H + KV, hd // 2 :].clone()
        c1, c2, s1, s2 = *c.chunk(2, -1), *sn.chunk(2, -1)
        for y, f in ((x, lambda t: t), (rounded, lambda t: t.float().double())):
            y[at : at + n, : H + KV, : hd // 2] = f(f(a * c1) - f(b * s1))
            y[at : at + n, : H + KV, hd // 2 :] = f(f(b * c2) + f(a * s2))
        at += n
    q = x[:, :H].reshape(-1, H * hd)
    pages = {}
    for name, lo in (("k", H), ("v", H + KV)):
        y = (rounded if case["fp8"] else x)[:, lo : lo + KV]
        e = s[name + "_exp"]
        if case["fp8"]:
            m, ex = torch.frexp(y.abs().amax(-1, keepdim=True))
            unit = torch.where(m > 0, torch.where(m > 448 / 512, ex - 8, ex - 9), 0)
            unit = unit.clamp(-15, 7) if case["dtype"] == "fp16" else unit.clamp(-120, 120)
            unit = torch.ldexp(torch.ones_like(y[..., :1]), unit)
            y = (y / unit).clamp(-448, 448).float().to(torch.float8_e4m3fn).double() * unit
        there = s[name].double() if e is None else s[name].double() * torch.ldexp(
            torch.ones_like(e, dtype=torch.float64), e.int())[..., None]
        at = 0
        for b, (n, l) in enumerate(zip(new, kv)):
            p = torch.arange(l - n, l, device=DEV)
            there[s["table"][b, p // case["page"]].long(), :, p % case["page"]] = y[at : at + n]
            at += n
        pages[name] = there
    if case["kind"] == "write":
        return q, pages["k"], pages["v"]
    if case["kind"] == "restore":
        return q, *[torch.cat([_sequence(pages[n], s["table"][b], l) for b, l in enumerate(kv)]) for n in ("k", "v")]
    return q, _exact_attention({**s, **pages}, q, kv, new), pages["k"], pages["v"]


def _sequence(pages, table, length):
    """The first `length` tokens of one sequence, [length, KV * head dim]."""
    n, KV, size, hd = pages.shape
    return pages[table[: -(-length // size)].long()].transpose(1, 2).reshape(-1, KV * hd)[:length]


def _exact_attention(s, q, kv, new):
    H, KV, hd = s["heads"]
    if sum(n * l for n, l in zip(new, kv)) * H * hd > 4e11:
        return None
    G, out, at = H // KV, [], 0
    for b, (n, l) in enumerate(zip(new, kv)):
        heads = []
        hidden = torch.arange(l, device=DEV)[None] > torch.arange(l - n, l, device=DEV)[:, None]
        pages = s["table"][b, : -(-l // s["case"]["page"])].long()
        for g in range(KV):
            kv_of = []
            for name in ("k", "v"):
                t = s[name][pages, g].double()
                if s[name + "_exp"] is not None:
                    t = t * torch.ldexp(torch.ones_like(t[..., :1]), s[name + "_exp"][pages, g].int()[..., None])
                kv_of.append(t.reshape(-1, hd)[:l])
            for h in range(g * G, g * G + G):
                score = q[at : at + n, h * hd : (h + 1) * hd] @ kv_of[0].T / math.sqrt(hd)
                heads.append(torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ kv_of[1])
        out.append(torch.cat(heads, 1))
        at += n
    return torch.cat(out)


def _exact_logits(s):
    lengths, prompts = _history_lengths(s["case"])
    V, out = s["logits"].shape[1], []
    for b, (n, p) in enumerate(zip(lengths, prompts)):
        x = s["logits"][b].double()
        text = torch.bincount(s["tokens"][b, :n], minlength=V)
        count = torch.bincount(s["tokens"][b, p:n], minlength=V)
        r, f, a = (s[k][b].double() for k in ("repetition", "frequency", "presence"))
        x = torch.where(text > 0, torch.maximum(x / r, torch.zeros_like(x)) + torch.minimum(x * r, torch.zeros_like(x)), x)
        x = x - f * count - a * count.clamp(max=1)
        if s["bias"] is not None:
            x = x + (s["bias"] if s["bias"].dim() == 1 else s["bias"][b])
        if s["mask"] is not None:
            m = s["mask"][b]
            if m.dtype == torch.int32:
                m = ((m[:, None] >> torch.arange(32, device=DEV)) & 1).reshape(-1)[:V] != 0
            x[~m] = -math.inf
        out.append(x)
    return torch.stack(out)
