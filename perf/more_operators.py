"""The operators of drafted tokens over a paged key/value cache, in their plain
form and as the framework's calls: a step's tables made on the GPU from the
sequences' lengths, attention of a tree of drafted tokens over the cache, the
verification of the draft against the model's logits, and the move of the kept
tokens' keys and values to the slots that they keep.

A cache layer is k and v, [pages, KV heads, page size, head dim], in the
model's type or in float8_e4m3fn with one exponent e for each (page, head,
token) in k_exp and v_exp (int8): the value is the stored number times 2^e.
Sequence b's token in place p is at [page_table[b, p // size], :, p % size].
Its new tokens are rows row_start[b] .. row_start[b + 1] - 1 of a step, in its
last places, and kv_len[b] is its length with them.  They are the nodes of a
tree: a row sees the first base[b] places and, of those after them, place base
+ j where bit j of its mask words is set (its ancestors and itself).
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
LAYERS = {"plumbing": 4, "tiny": 8, "125m": 12, "small": 12, "medium": 24, "1b": 16, "7b": 32}
THETA = 10_000.0


def listed():
    return [
        # a single answer's draft of a few tokens, on the smallest preset: latency alone
        {"name": "tree_plumbing", "kind": "tree", "size": "plumbing", "dtype": "bf16", "fp8": False, "batch": 1,
         "nodes": 8, "length": 128, "page": 16},
        # a batch of answers being written, a small tree for each, lengths as they come
        {"name": "tree_1b_ragged", "kind": "tree", "size": "1b", "dtype": "bf16", "fp8": False, "batch": 32, "nodes": 16,
         "length": 2048, "page": 64},
        # a few long documents with wide trees, cache in 8 bits
        {"name": "tree_7b_long_fp8", "kind": "tree", "size": "7b", "dtype": "bf16", "fp8": True, "batch": 4, "nodes": 64,
         "length": 32768, "page": 64},
        # a model kept in float32, trees of an odd size
        {"name": "tree_tiny_fp32", "kind": "tree", "size": "tiny", "dtype": "fp32", "fp8": False, "batch": 3, "nodes": 33,
         "length": 701, "page": 16},
        # one answer, a chain of four drafted tokens, the arg-max at each place
        {"name": "verify_one", "kind": "verify", "dtype": "bf16", "batch": 1, "nodes": 5, "vocab": 32000,
         "mode": "greedy", "tree": False, "view": True},
        # a served batch: chains drawn from a draft model's probabilities
        {"name": "verify_drawn", "kind": "verify", "dtype": "fp32", "batch": 32, "nodes": 8, "vocab": 128256,
         "mode": "drawn", "tree": False, "view": False},
        # trees of likely tokens, the model's own choice at every node
        {"name": "verify_trees", "kind": "verify", "dtype": "bf16", "batch": 16, "nodes": 32, "vocab": 128256,
         "mode": "sample", "tree": True, "view": False},
        # a served batch's next step: what was rejected goes back, a tree each comes in
        {"name": "tables_trees", "kind": "tables", "batch": 64, "nodes": 24, "length": 4096, "page": 64, "tree": True,
         "scarce": False},
        # prompts taken in, more than the pool has pages for
        {"name": "tables_prompts", "kind": "tables", "batch": 48, "nodes": 2048, "length": 2048, "page": 16,
         "tree": False, "scarce": True},
        # the kept branches of one answer and of a served batch, in every layer
        {"name": "keep_plumbing", "kind": "keep", "size": "plumbing", "dtype": "fp32", "batch": 1, "nodes": 12,
         "length": 128, "page": 16},
        {"name": "keep_7b_batch", "kind": "keep", "size": "7b", "dtype": "bf16", "batch": 32, "nodes": 32,
         "length": 1024, "page": 64},
        # one layer's step with all that belongs to it: tables, write, attend, verify, keep
        {"name": "step_1b", "kind": "step", "size": "1b", "dtype": "bf16", "batch": 16, "nodes": 12, "length": 2048,
         "page": 64, "vocab": 32000},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["tree", "tree", "tree", "verify", "verify", "tables", "keep", "step"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        batch, nodes, page = _log_int(rng, 1, 64), _log_int(rng, 1, 160), rng.choice([16, 32, 64, 128, 256])
        length = max(nodes, _log_int(rng, 1, 32768))
        if kind == "verify":
            case = {"kind": kind, "dtype": dtype, "batch": batch, "nodes": _log_int(rng, 1, 64),
                    "vocab": rng.choice([8192, 32000, 128256, _log_int(rng, 500, 128256)]),
                    "mode": rng.choice(["greedy", "sample", "drawn"]), "view": rng.random() < 0.5}
            case["tree"] = case["mode"] != "drawn" and rng.random() < 0.6
            if batch * case["nodes"] * case["vocab"] <= 2**26:
                return case
            continue
        if kind == "tables":
            case = {"kind": kind, "batch": _log_int(rng, 1, 256), "nodes": nodes, "length": length, "page": page,
                    "tree": rng.random() < 0.6, "scarce": rng.random() < 0.3}
            if not case["tree"] and rng.random() < 0.5:  # whole prompts
                case["nodes"] = case["length"] = _log_int(rng, 1, 2048)
            if case["batch"] * case["length"] <= 2**20 and case["batch"] * case["nodes"] <= 98304:
                return case
            continue
        case = {"kind": kind, "size": rng.choice(list(HEADS)), "dtype": dtype, "batch": batch, "nodes": nodes,
                "length": length, "page": page}
        H, KV, hd = HEADS[case["size"]]
        cached = case["batch"] * length * KV * hd
        if kind == "keep":
            if cached * LAYERS[case["size"]] <= 2**31 and batch * nodes <= 1024:
                return case
            continue
        # what the plain form holds at once, and what float32 takes longer for
        if cached > 2**27 or batch * nodes * length * H > 2**29 or work({**case, "fp8": False, "vocab": 1})["flops"] > (
                1.2e11 if dtype != "fp32" else 1.5e10):
            continue
        if kind == "step":
            case["vocab"] = rng.choice([8192, 32000, _log_int(rng, 500, 32000)])
            if batch * nodes > 512 or batch * length > 65536:
                continue
        else:
            case["fp8"] = rng.random() < 0.4
        return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _counts(case):
    """(length before the step, new tokens) of each sequence: one is as long as
    the case says with its new tokens, the others are anything up to that."""
    rng = random.Random(f"{case['batch']} {case['nodes']} {case['length']}")
    new = [case["nodes"]] + [rng.randint(1, case["nodes"]) for _ in range(case["batch"] - 1)]
    kept = [case["length"] - new[0]] + [rng.randint(0, case["length"] - n) for n in new[1:]]
    return kept, new


def _accepted(case):
    """Tokens that each sequence keeps of its new ones."""
    _, new = _counts(case)
    rng = random.Random(f"accepted {case['batch']} {case['nodes']}")
    return [rng.randint(1, max(1, min(8, n // 2))) for n in new]


def work(case):
    kept, new = _counts(case) if case["kind"] != "verify" else (None, _new_rows(case))
    T = sum(new)
    if case["kind"] == "tables":
        pages = sum(-(-(k + n) // case["page"]) - k // case["page"] for k, n in zip(kept, new))
        words = -(-case["nodes"] // 32) if case["tree"] else 0
        return {"bytes": 8 * pages + 24 * len(new) + T * (12 + 4 * words + (4 if words else 0)), "flops": 0.0}
    esz = 4 if case.get("dtype") == "fp32" else 2
    verify = {"bytes": 0, "flops": 0.0}
    if case["kind"] in ("verify", "step"):
        V, drawn = case["vocab"], case.get("mode") == "drawn"
        # logits once; of a draft's probabilities one row a sequence
        verify = {"bytes": T * V * esz + T * 16 + (len(new) * V * 4 if drawn else 0) + len(new) * case["nodes"] * 12,
                  "flops": 4.0 * T * V}
        if case["kind"] == "verify":
            return verify
    H, KV, hd = HEADS[case["size"]]
    token = 2 * KV * (hd + 1 if case.get("fp8") else hd * esz)  # a cached token, keys and values
    if case["kind"] == "keep":
        moved = sum(max(0, a - 1) for a in _accepted(case))
        return {"bytes": 2 * moved * token * LAYERS[case["size"]] + 12 * T, "flops": 0.0}
    L = sum(kept) + T
    seen = sum(n * k + n * (1 + math.log(n)) for k, n in zip(kept, new))  # a node of these trees has about ln n ancestors
    attend = {"bytes": 2 * T * H * hd * esz + L * token + T * 4 * -(-case["nodes"] // 32), "flops": 4.0 * H * hd * seen}
    if case["kind"] == "tree":
        return attend
    written = T * (esz * hd * (2 * H + 2 * KV) + 2 * esz * hd) + T * token  # qkv read, q and the cache written, tables
    return {"bytes": attend["bytes"] - T * H * hd * esz - T * token + written + verify["bytes"] + 2 * len(new) * token,
            "flops": attend["flops"] + verify["flops"] + 6.0 * T * (H + KV) * hd}


def _new_rows(case):
    rng = random.Random(f"{case['batch']} {case['nodes']}")
    return [case["nodes"]] + [rng.randint(1, case["nodes"]) for _ in range(case["batch"] - 1)]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(new):
    return _i32([sum(new[:b]) for b in range(len(new) + 1)])


def _random_trees(batch, nodes, g):
    """Parents [batch, nodes]: the first node is the root, each other hangs
    from any node before it."""
    i = torch.arange(nodes, device=DEV)
    return torch.where(i > 0, (torch.rand(batch, nodes, device=DEV, generator=g) * i).to(torch.int32), -1).to(torch.int32)


def _closure(parents):
    """[B, N, N]: whether node j is i or an ancestor of i."""
    N = parents.shape[-1]
    i = torch.arange(N, device=DEV)
    p = torch.where((parents >= 0) & (parents < i), parents, -1)
    up = (p[..., None] == i).double() + torch.eye(N, device=DEV, dtype=torch.float64)
    return torch.linalg.matrix_power(up, max(N - 1, 1)) > 0


def _words(bits):
    """[..., N] truth values as int32 words of 32, lowest bit first."""
    n = bits.shape[-1]
    bits = torch.nn.functional.pad(bits, (0, -n % 32)).view(*bits.shape[:-1], -1, 32)
    return (bits.long() << torch.arange(32, device=DEV)).sum(-1).to(torch.int32)


def _pages_of(lengths, page, width, g):
    """A page table [B, width] with pages in any order, and the pages left over."""
    counts = [-(-n // page) for n in lengths]
    n_pages = sum(counts) + 3
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    table, at = torch.full((len(lengths), width), -1, dtype=torch.int32, device=DEV), 0
    for b, m in enumerate(counts):
        table[b, :m] = order[at : at + m]
        at += m
    return table, n_pages, order[at:]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": case}
    kind = case["kind"]
    if kind == "verify":
        _prepare_verify(s, _new_rows(case), g)
        return s
    kept, new = _counts(case)
    B, page, N = len(new), case["page"], case["nodes"]
    full = [k + n for k, n in zip(kept, new)]
    width = -(-max(full) // page)
    s |= {"new": _i32(new), "rows": sum(new), "max_new": N, "max_len": max(full)}
    if kind == "tables":
        # before the step each sequence holds a few tokens that it does not keep
        rng = random.Random(str(case))
        before = [min(k + rng.randint(0, min(N, 32)), width * page) if k else 0 for k in kept]
        table, n_pages, spare = _pages_of(before, page, width, g)
        asked = sum(-(-n // page) for n in full) + 4
        pool = n_pages + max(0, asked // 2 if case["scarce"] else asked)
        more = n_pages + torch.randperm(pool - n_pages, device=DEV, generator=g).to(torch.int32)
        free = torch.full((pool,), -1, dtype=torch.int32, device=DEV)
        n_free = spare.numel() + more.numel()
        free[:n_free] = torch.cat([spare, more])
        s |= {"table": table, "lengths": _i32(before), "free": free, "n_free": _i32([n_free]), "keep": _i32(kept),
              "parents": _random_trees(B, N, g) if case["tree"] else None}
        return s
    H, KV, hd = HEADS[case["size"]]
    dtype = DTYPES[case["dtype"]]
    table, n_pages, spare = _pages_of(full, page, width, g)
    s |= {"heads": (H, KV, hd), "dtype": dtype, "table": table, "row_start": _starts(new), "kv_len": _i32(full),
          "base": _i32(kept), "k_exp": None, "v_exp": None}
    stacked = (LAYERS[case["size"]],) if kind == "keep" else ()
    shape = (*stacked, n_pages, KV, page, hd)
    for name in ("k", "v"):
        x = torch.randn(shape, device=DEV, generator=g, dtype=dtype)
        if case.get("fp8"):
            # heads and tokens of different sizes, as they are in a model
            x = x.float() * (0.25 + 2 * torch.rand(shape[:-1], device=DEV, generator=g))[..., None]
            s[name], s[name + "_exp"] = _to_fp8(x, dtype)
        else:
            s[name] = x
    parents = _random_trees(B, N, g)
    b, place = _rows_of(s)
    node = place - s["base"][b]
    closure = _closure(parents)
    s |= {"parents": parents, "mask": _words(closure)[b, node], "positions": (place - node + closure.sum(-1)[b, node] - 1).to(
        torch.int32), "slots": s["table"][b, place // page].long() * page + place % page}
    if kind == "tree":
        s["q"] = torch.randn(sum(new), H * hd, device=DEV, generator=g, dtype=dtype)
    elif kind == "keep":
        # nodes in the order of their depth: those that are kept lie behind the places that they move to
        counts, rng = _accepted(case), random.Random(f"kept {seed}")
        rows = [[0] + sorted(rng.sample(range(c, n), c - 1)) + [-1] * (N - c) for c, n in zip(counts, new)]
        s |= {"counts": _i32(counts), "kept": _i32(rows)}
    else:
        s["qkv"] = torch.randn(sum(new), (H + 2 * KV) * hd, device=DEV, generator=g, dtype=dtype)
        inv = THETA ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
        angle = torch.arange(max(full), device=DEV, dtype=torch.float64)[:, None] * inv
        angle = torch.cat([angle, angle], 1)
        s |= {"cos": angle.cos().to(dtype), "sin": angle.sin().to(dtype)}
        # the step before had as many drafted tokens: their pages are there
        free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
        free[: spare.numel()] = spare
        s |= {"lengths": s["kv_len"].clone(), "keep": s["base"], "free": free, "n_free": _i32([spare.numel()])}
        _prepare_verify(s, new, g)
    return s


def _prepare_verify(s, new, g):
    case = s["case"]
    B, T, V, N, mode = len(new), sum(new), case["vocab"], case["nodes"], case.get("mode", "sample")
    wide = V + 64 if case.get("view") else V  # rows of their own, or of a head that is padded
    logits = (5 * torch.randn(T, wide, device=DEV, generator=g)).to(DTYPES[case["dtype"]])[:, :V]
    s |= {"logits": logits, "row_start": _starts(new), "rows": T, "max_new": N, "probs": None, "parents": s.get("parents"),
          "uniform": torch.rand(T, device=DEV, generator=g, dtype=torch.float64), "temperature": 0.0}
    if mode != "greedy":
        s["temperature"] = 0.5 + torch.rand(B, device=DEV, generator=g)
    if case.get("tree"):
        s["parents"] = _random_trees(B, N, g)
    # a row's token comes from the row of its parent: drawn, or one of the likely ones
    row = torch.arange(T, device=DEV)
    b = torch.searchsorted(s["row_start"][1:], row.to(torch.int32), right=True)
    start = s["row_start"][b].long()
    up = (row - 1).clamp(min=0) if s["parents"] is None else start + s["parents"][b, row - start].clamp(min=0)
    if mode == "drawn":
        noisy = logits.float() + torch.randn(T, V, device=DEV, generator=g)
        draft = torch.softmax(noisy / s["temperature"][b][:, None], -1)[up]
        s |= {"probs": draft, "tokens": torch.multinomial(draft, 1, generator=g)[:, 0]}
    else:
        likely = torch.topk(logits.float(), 3).indices[up]
        pick = (3 * torch.rand(T, device=DEV, generator=g) ** 2).long()
        s["tokens"] = likely.gather(1, pick[:, None])[:, 0].contiguous()


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    ops, LayerCache, DraftStep, PageTables = _framework()
    kind = s["case"]["kind"]
    step = None
    if kind in ("tables", "step"):
        tables = PageTables(s["table"], s["lengths"], s["free"], s["n_free"], s["case"]["page"])
        step = ops.cache_tables(tables, s["new"], s["rows"], s["max_new"], s["max_len"], keep=s["keep"],
                                parents=s["parents"])
        if kind == "tables":
            return (step.row_start, step.kv_len, step.base, step.positions, step.slots, step.mask, s["table"],
                    s["lengths"], s["free"], s["n_free"])
    elif kind in ("tree", "keep"):
        step = DraftStep(s["row_start"], s["kv_len"], s["table"], s["rows"], s["max_new"], s["max_len"], s["base"],
                         s["positions"], s["slots"], s["mask"])
    if kind == "verify":
        return ops.verify_draft(s["logits"], s["tokens"], s["row_start"], s["max_new"], s["uniform"],
                                temperature=s["temperature"], parents=s["parents"], draft_probs=s["probs"])
    layer = LayerCache(s["k"], s["v"], s["k_exp"], s["v_exp"])
    if kind == "keep":
        ops.kv_cache_keep(layer, step, s["kept"], s["counts"])
        return s["k"], s["v"]
    H, KV, hd = s["heads"]
    if kind == "tree":
        return ops.paged_attention(s["q"], layer, step, H, hd**-0.5)
    q = ops.kv_cache_write(s["qkv"], layer, step, H, s["cos"], s["sin"])
    y = ops.paged_attention(q, layer, step, H, hd**-0.5)
    counts, kept, tokens = ops.verify_draft(s["logits"], s["tokens"], step.row_start, s["max_new"], s["uniform"],
                                            temperature=s["temperature"], parents=s["parents"])
    ops.kv_cache_keep(layer, step, kept, counts)
    return y, counts, kept, tokens, s["k"], s["v"], s["lengths"]


@functools.lru_cache(maxsize=None)
def _framework():
    package = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cs244c-llama-zero_amd")
    if os.path.abspath(package) not in sys.path:
        sys.path.insert(0, os.path.abspath(package))
    from lzhip import ops
    from lzhip.cache import DraftStep, LayerCache, PageTables

    return ops, LayerCache, DraftStep, PageTables


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "tables":
        return _plain_tables(s)
    if kind == "verify":
        return _plain_verify(s, s["row_start"])
    if kind == "keep":
        return _plain_keep(s, s, s["kept"], s["counts"])
    if kind == "tree":
        return _plain_attention(s, s["q"], s)
    row_start, kv_len, base, positions, slots, mask = _plain_tables(s)[:6]
    step = {"row_start": row_start, "kv_len": kv_len, "base": base, "positions": positions, "slots": slots, "mask": mask}
    q = _plain_write(s, step)
    y = _plain_attention(s, q, step)
    counts, kept, tokens = _plain_verify(s, row_start)
    _plain_keep(s, step, kept, counts)
    return y, counts, kept, tokens, s["k"], s["v"], s["lengths"]


def _pow2(e):
    """2^e for integers -126..127, as float32."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to_fp8(x, dtype):
    """x (float32) as (float8_e4m3fn, int8 exponents over the last dimension):
    the smallest exponent e with max |x| <= 448 * 2^e, 0 where all are zero;
    -120..119, and -15..7 for a model in float16."""
    m, ex = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0, ex - 9 + (m > 0.875), torch.zeros_like(ex))
    e = e.clamp(-15, 7) if dtype == torch.float16 else e.clamp(-120, 119)
    q = (x * _pow2(-e)[..., None]).clamp(-448, 448)
    return q.to(torch.float8_e4m3fn), e.to(torch.int8)


def _values(pages, exps):
    """The values of gathered pages, float32."""
    return pages.float() if exps is None else pages.view(torch.float8_e4m3fn).float() * _pow2(exps)[..., None]


def _rows_of(s):
    """(sequence, place) of each row of the step."""
    r = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(s["row_start"][1:], r.to(torch.int32), right=True)
    return b, (s["kv_len"][b] - s["row_start"][b + 1] + r).long()


def _plain_tables(s):
    """Cuts each sequence to keep[b] tokens, puts the pages behind them on the
    stack of free ones (the first sequence's first on top) and takes pages for
    new[b] more, sequence after sequence; those whose tokens do not fit (into
    max_new, max_len, the table, or together with all that ask before them into
    the rows and the free pages) get none."""
    table, lengths, free, n_free = s["table"], s["lengths"], s["free"], s["n_free"].long()
    P, (B, width) = s["case"]["page"], table.shape
    cur = lengths.long().clamp(0, width * P)
    keep = torch.minimum(s["keep"].long().clamp(min=0), cur)
    new = s["new"].long()
    held, left, total = -(-cur // P), -(-keep // P), keep + new
    fits = (new > 0) & (new <= s["max_new"]) & (total <= min(s["max_len"], width * P))
    need = torch.where(fits, -(-total // P) - left, 0)
    top = n_free + (held - left).sum()
    served = fits & ((need == 0) | (need.cumsum(0) <= top)) & (torch.where(fits, new, 0).cumsum(0) <= s["rows"])
    new, take = torch.where(served, new, 0), torch.where(served, need, 0)
    c = torch.arange(width, device=DEV)
    given = (c >= left[:, None]) & (c < held[:, None])
    free[(top - 1 - (given.view(-1).cumsum(0) - 1).view(B, width))[given]] = table[given]
    table[given] = -1
    taken = (c >= left[:, None]) & (c < (left + take)[:, None])
    table[taken] = free[(top - 1 - (taken.view(-1).cumsum(0) - 1).view(B, width))[taken]]
    s["n_free"].copy_(top - take.sum())
    lengths.copy_(keep + new)
    row_start = torch.nn.functional.pad(new.cumsum(0), (1, 0)).to(torch.int32)
    kv_len, base = (keep + new).to(torch.int32), keep.to(torch.int32)
    r = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(row_start[1:], r.to(torch.int32), right=True)
    inside = b < B
    b = b.clamp(max=B - 1)
    place = torch.where(inside, keep[b] + r - row_start[b], 0)
    slots = torch.where(inside, table[b, place // P].long() * P + place % P, -1)
    position, mask = place, None
    if s["parents"] is not None:
        closure, node = _closure(s["parents"]), place - keep[b]
        node = torch.where(inside, node, 0)
        position = keep[b] + closure.sum(-1)[b, node] - 1
        mask = torch.where(inside[:, None], _words(closure)[b, node], 0)
    positions = torch.where(inside, position, -1).to(torch.int32)
    return row_start, kv_len, base, positions, slots, mask, table, lengths, free, s["n_free"]


def _plain_write(s, step):
    H, KV, hd = s["heads"]
    x = s["qkv"].float().view(-1, H + 2 * KV, hd)
    pos = step["positions"].long()
    c, sn = s["cos"].float()[pos][:, None], s["sin"].float()[pos][:, None]
    qk = x[:, : H + KV]
    half = torch.cat([-qk[..., hd // 2 :], qk[..., : hd // 2]], -1)
    qk = qk * c + half * sn
    size = s["case"]["page"]
    page, slot = step["slots"] // size, step["slots"] % size
    s["k"][page, :, slot] = qk[:, H:].to(s["dtype"])
    s["v"][page, :, slot] = x[:, H + KV :].to(s["dtype"])
    return qk[:, :H].reshape(-1, H * hd).to(s["dtype"])


def _plain_attention(s, q, step):
    H, KV, hd = s["heads"]
    size, L, N, G = s["case"]["page"], s["max_len"], s["max_new"], H // KV
    table = s["table"][:, : -(-L // size)].clamp(min=0).long()
    B = table.shape[0]
    whole = []
    for name in ("k", "v"):
        p, e = s[name], s[name + "_exp"]
        x = _values((p if e is None else p.view(torch.uint8))[table], None if e is None else e[table])
        whole.append(x.transpose(1, 2).reshape(B, KV, -1, hd)[:, :, :L])
    k, v = whole
    start, new = step["row_start"][:-1], step["row_start"][1:] - step["row_start"][:-1]
    i = torch.arange(N, device=DEV)
    row = (start[:, None] + i).clamp(max=s["rows"] - 1).long()
    x = q.float()[row].view(B, N, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(B, KV, G * N, hd)
    score = (x @ k.transpose(2, 3).contiguous()).view(B, KV, G, N, L) * hd**-0.5
    place = torch.arange(L, device=DEV)
    node = place - step["base"][:, None]  # [B, L]
    words = step["mask"][row]
    at = (node // 32).clamp(0, words.shape[2] - 1)[:, None].expand(B, N, L)
    bit = (words.gather(2, at) >> (node % 32)[:, None]) & 1
    seen = (node < 0)[:, None] | ((bit != 0) & (place < step["kv_len"][:, None])[:, None])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    y = (p.view(B, KV, G * N, L) @ v.contiguous()).view(B, KV, G, N, hd) / p.sum(-1, keepdim=True)
    r = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(step["row_start"][1:], r.to(torch.int32), right=True)
    y = y.permute(0, 3, 1, 2, 4).reshape(B, N, H * hd)
    return y[b, r - start[b]].to(q.dtype)


def _choose(weights, u):
    """The first token whose sum of weights up to it is over u times their sum."""
    sums = weights.cumsum(-1)
    return torch.searchsorted(sums, (u * sums[:, -1])[:, None], right=True)[:, 0].clamp(max=weights.shape[1] - 1)


def _plain_verify(s, row_start):
    """How many tokens each sequence gains, the nodes that it keeps (the root
    first) and the tokens: those of the kept nodes and the one that the last of
    them is followed by."""
    tokens, u, N = s["tokens"], s["uniform"], s["max_new"]
    T, V = s["logits"].shape
    B = row_start.shape[0] - 1
    start = row_start.long()
    r, i = torch.arange(T, device=DEV), torch.arange(N, device=DEV)
    b = torch.searchsorted(row_start[1:], r.to(torch.int32), right=True)
    there = i < (start[1:] - start[:-1])[:, None]  # [B, N]: the nodes that there are
    row = (start[:-1, None] + i).clamp(max=T - 1)
    x = s["logits"].double()
    sampled = torch.is_tensor(s["temperature"])
    w = torch.exp((x - x.amax(-1, keepdim=True)) / s["temperature"].double()[b][:, None]) if sampled else None
    if s["probs"] is None:
        choice = _choose(w, u) if sampled else s["logits"].float().argmax(-1)
        parents = (i - 1).expand(B, N) if s["parents"] is None else s["parents"].long()
        good = there & (i > 0) & (parents >= 0) & (parents < i)
        up = parents.clamp(min=0)
        match = good & (tokens[row] == choice[row].gather(1, up))
        # of children with the same token the first counts
        same = (up[:, :, None] == up[:, None]) & (i[:, None] > i) & match[:, None] & match[:, :, None]
        match &= ~same.any(-1)
        closure = _closure(torch.where(good, parents, -1))
        on_path = (there & ((match | (i == 0))[:, None] | ~closure).all(-1)) & closure[:, :, 0]
        counts = on_path.sum(-1)
        last = torch.where(on_path, i, 0).amax(-1)
        final = choice[row.gather(1, last[:, None])[:, 0]]
        order = torch.where(on_path, i, N).sort(-1).values
        kept = torch.where(order < N, order, -1)
    else:
        p = w / w.sum(-1, keepdim=True)
        q = s["probs"].double()
        prev = (r - 1).clamp(min=0)
        accept = u * q[r, tokens] < p[prev, tokens]
        ok = there & ((i == 0) | accept[row])
        counts = ok.long().cumprod(-1).sum(-1)
        kept = torch.where(i < counts[:, None], i, -1)
        last = row.gather(1, (counts - 1).clamp(min=0)[:, None])[:, 0]
        whole = counts == there.sum(-1)
        rest = (p[last] - torch.where(whole[:, None], 0, q[(last + 1).clamp(max=T - 1)])).clamp(min=0)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p[last])
        final = _choose(rest, u[row[:, 0]])
    shown = torch.where(kept >= 0, kept, 0)
    gained = tokens[row.gather(1, shown)].roll(-1, 1)  # the root's own token is not among them
    at_end = i == (counts - 1)[:, None]
    gained = torch.where(at_end, final[:, None], torch.where(i < (counts - 1)[:, None], gained, -1))
    return counts.to(torch.int32), kept.to(torch.int32), gained


def _plain_keep(s, step, kept, counts):
    start = step["row_start"].long()
    i = torch.arange(kept.shape[1], device=DEV)
    new = (start[1:] - start[:-1])[:, None]
    move = (i < counts[:, None]) & (i < new) & (kept >= 0) & (kept < new)
    src = step["slots"][(start[:-1, None] + kept)[move]]
    dst = step["slots"][(start[:-1, None] + i)[move]]
    size = s["case"]["page"]
    for x in (s["k"], s["v"]):
        x = x if x.dim() == 5 else x[None]
        x[:, dst // size, :, dst % size] = x[:, src // size, :, src % size]
    return s["k"], s["v"]


# ---------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "verify":
        return _exact_verify(s, _new_rows(case))
    kept, new = _counts(case)
    if kind == "tables":
        return _exact_tables(s, kept, new)
    if kind == "keep":
        counts, at = _accepted(case), 0
        size = case["page"]
        nodes = s["kept"].tolist()
        for b, (n, c) in enumerate(zip(new, counts)):
            where = s["slots"][at : at + n].tolist()
            for x in (s["k"], s["v"]):
                flat = [x[:, p // size, :, p % size].clone() for p in (where[j] for j in nodes[b][:c])]
                for j, value in enumerate(flat):
                    x[:, where[j] // size, :, where[j] % size] = value
            at += n
        return s["k"].double(), s["v"].double()
    if kind == "tree":
        return _exact_attention(s, s["q"].double(), kept, new)
    H, KV, hd = s["heads"]
    _exact_tables(s, kept, new)
    x = s["qkv"].double().view(-1, H + 2 * KV, hd)
    parents, size = s["parents"].tolist(), case["page"]
    k, v = s["k"].double(), s["v"].double()
    table = s["table"].tolist()
    at = 0
    for b, (l, n) in enumerate(zip(kept, new)):
        depth = _depths(parents[b][:n])
        where = l + torch.tensor(depth, device=DEV)
        c, sn = s["cos"][where, None].double(), s["sin"][where, None].double()
        lo, hi = x[at : at + n, : H + KV, : hd // 2].clone(), x[at : at + n, : H + KV, hd // 2 :].clone()
        x[at : at + n, : H + KV, : hd // 2] = lo * c[..., : hd // 2] - hi * sn[..., : hd // 2]
        x[at : at + n, : H + KV, hd // 2 :] = hi * c[..., hd // 2 :] + lo * sn[..., hd // 2 :]
        for j in range(n):
            p = table[b][(l + j) // size]
            k[p, :, (l + j) % size], v[p, :, (l + j) % size] = x[at + j, H : H + KV], x[at + j, H + KV :]
        at += n
    y = _exact_attention({**s, "k": k, "v": v}, x[:, :H].reshape(-1, H * hd), kept, new)
    counts, chosen, tokens = _exact_verify(s, new)
    for b, l in enumerate(kept):
        nodes = chosen[b, : counts[b]].tolist()
        for t in (k, v):
            flat = [t[table[b][(l + j) // size], :, (l + j) % size].clone() for j in nodes]
            for i, value in enumerate(flat):
                t[table[b][(l + i) // size], :, (l + i) % size] = value
    return y, counts, chosen, tokens, k, v, s["lengths"]


def _depths(parents):
    depth = []
    for i, p in enumerate(parents):
        depth.append(depth[p] + 1 if 0 <= p < i else 0)
    return depth


def _exact_tables(s, kept, new):
    P, width, pool = s["case"]["page"], s["table"].shape[1], s["free"].numel()
    table, lengths, free, top = s["table"].tolist(), s["lengths"].tolist(), s["free"].tolist(), int(s["n_free"])
    back = []
    for b, l in enumerate(kept):
        first = -(-l // P)
        for c in range(first, -(-lengths[b] // P)):
            back.append(table[b][c])
            table[b][c] = -1
    free[top : top + len(back)] = back[::-1]
    top += len(back)
    assert len(free) == pool
    asked, pages_asked, avail, starts = 0, 0, top, [0]
    positions, slots, masks, kv_len = [], [], [], []
    parents = None if s["parents"] is None else s["parents"].tolist()
    words = -(-s["max_new"] // 32)
    for b, (l, n) in enumerate(zip(kept, new)):
        need = -(-(l + n) // P) - -(-l // P)
        asked, pages_asked = asked + n, pages_asked + need
        if (need and pages_asked > avail) or asked > s["rows"] or l + n > width * P:
            n = 0
        for c in range(-(-l // P), -(-(l + n) // P)):
            top -= 1
            table[b][c] = free[top]
        ancestors, depth = [], _depths(parents[b][:n]) if parents else list(range(n))
        for i in range(n):
            p = parents[b][i] if parents else -1
            ancestors.append((ancestors[p] if 0 <= p < i else 0) | 1 << i)
            positions.append(l + depth[i])
            slots.append(table[b][(l + i) // P] * P + (l + i) % P)
            masks.append([(ancestors[i] >> 32 * w) & 0xFFFFFFFF for w in range(words)])
        starts.append(starts[-1] + n)
        kv_len.append(l + n)
    none = s["rows"] - starts[-1]
    mask = None
    if parents:
        mask = torch.tensor(masks + [[0] * words] * none, device=DEV, dtype=torch.int64).to(torch.int32)
    s["table"].copy_(_i32(table))
    s["lengths"].copy_(_i32(kv_len))
    s["free"].copy_(_i32(free))
    s["n_free"].fill_(top)
    return (_i32(starts), _i32(kv_len), _i32(kept), _i32(positions + [-1] * none),
            torch.tensor(slots + [-1] * none, device=DEV), mask, s["table"], s["lengths"], s["free"], s["n_free"])


def _exact_attention(s, q, kept, new):
    H, KV, hd = s["heads"]
    if sum(n * (k + n) for k, n in zip(kept, new)) * H * hd > 2e11:
        return None
    G, size, out, at = H // KV, s["case"]["page"], [], 0
    parents = s["parents"].tolist()
    for b, (l, n) in enumerate(zip(kept, new)):
        sees = torch.zeros(n, l + n, dtype=torch.bool, device=DEV)
        sees[:, :l] = True
        for i in range(n):
            p = parents[b][i]
            if 0 <= p < i:
                sees[i] |= sees[p]
            sees[i, l + i] = True
        pages = s["table"][b, : -(-(l + n) // size)].long()
        heads = []
        for g in range(KV):
            kv_of = []
            for name in ("k", "v"):
                t = s[name][pages, g].double()
                if s[name + "_exp"] is not None:
                    t = t * torch.ldexp(torch.ones_like(t[..., :1]), s[name + "_exp"][pages, g].int()[..., None])
                kv_of.append(t.reshape(-1, hd)[: l + n])
            for h in range(g * G, g * G + G):
                score = q[at : at + n, h * hd : (h + 1) * hd] @ kv_of[0].T / math.sqrt(hd)
                heads.append(torch.softmax(score.masked_fill(~sees, -math.inf), -1) @ kv_of[1])
        out.append(torch.cat(heads, 1))
        at += n
    return torch.cat(out)


def _exact_verify(s, new):
    N, V = s["max_new"], s["logits"].shape[1]
    tokens, u = s["tokens"].tolist(), s["uniform"].tolist()
    parents = None if s["parents"] is None else s["parents"].tolist()
    heat = s["temperature"].double().tolist() if torch.is_tensor(s["temperature"]) else [0.0] * len(new)
    counts, kept, gained, at = [], [], [], 0

    def pick(weights, x):
        sums = weights.cumsum(0)
        return min(int((sums <= x * sums[-1]).sum()), V - 1)

    def law(row, t):
        return torch.softmax(s["logits"][row].double() / t, 0)

    for b, n in enumerate(new):
        path, said = [0], []
        while True:
            node, t = path[-1], heat[b]
            if s["probs"] is not None:
                p = law(at + node, t)
                if node + 1 < n:
                    q = s["probs"][at + node + 1].double()
                    x = tokens[at + node + 1]
                    if u[at + node + 1] * float(q[x]) < float(p[x]):
                        path.append(node + 1)
                        said.append(x)
                        continue
                    rest = (p - q).clamp(min=0)
                    p = rest if float(rest.sum()) > 0 else p
                said.append(pick(p, u[at]))
                break
            choice = pick(law(at + node, t), u[at + node]) if t > 0 else int(torch.nonzero(
                s["logits"][at + node] == s["logits"][at + node].max())[0])
            said.append(choice)
            children = [i for i in range(node + 1, n) if (parents[b][i] if parents else i - 1) == node]
            matching = [i for i in children if tokens[at + i] == choice]
            if not matching:
                break
            path.append(matching[0])
        counts.append(len(path))
        kept.append(path + [-1] * (N - len(path)))
        gained.append(said + [-1] * (N - len(said)))
        at += n
    return _i32(counts), _i32(kept), torch.tensor(gained, device=DEV)
