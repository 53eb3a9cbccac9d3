"""Timed cases of the serving operators: attention of one new token over a
paged key-value cache, the append that fills the cache, the page operations
(reserve, fork, copy, free, compact) and the log probabilities of given tokens
(with entropy, top alternatives and gradient).

``run`` computes a case in plain torch where ``own`` is false and through
``adaattn_b200`` where it is true, on the inputs that ``prepare`` makes from a
seed; ``exact`` gives the computed outputs in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
ELT = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
IGNORE = -100


def listed():
    return [
        # One user's token through GPT-2-small's attention (12 heads of 64) early in a reply: latency.
        {"name": "attend_one_short", "op": "attend", "batch": 1, "heads": 12, "kv_heads": 12, "head_dim": 64,
         "page": 16, "min_len": 187, "max_len": 187, "dtype": "bf16", "mask": "none"},
        # GPT-2-small serving a batch of 16 left-padded prompts at every fill of its 1024 positions.
        {"name": "attend_batch_masked", "op": "attend", "batch": 16, "heads": 12, "kv_heads": 12, "head_dim": 64,
         "page": 16, "min_len": 1, "max_len": 1024, "dtype": "bf16", "mask": "bool"},
        # One very long document, grouped heads: the cache's length is the only axis to split.
        {"name": "attend_one_long", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 64, "min_len": 131071, "max_len": 131071, "dtype": "fp16", "mask": "none"},
        # A full serving batch of ragged lengths over an 8-bit cache with a scale per head.
        {"name": "attend_batch_e4m3", "op": "attend", "batch": 64, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 64, "min_len": 1, "max_len": 16384, "dtype": "e4m3", "mask": "none"},
        # One decode step's keys and values for 64 sequences.
        {"name": "append_token", "op": "append", "batch": 64, "kv_heads": 8, "head_dim": 128, "page": 16,
         "tokens": 1, "min_new": 1, "past": 900, "dtype": "bf16", "cache": "bf16"},
        # Right-padded prompts of up to 4096 tokens written to an 8-bit cache.
        {"name": "append_prompt", "op": "append", "batch": 8, "kv_heads": 8, "head_dim": 128, "page": 64,
         "tokens": 4096, "min_new": 77, "past": 0, "dtype": "bf16", "cache": "e4m3"},
        # Branching 32 sequences of a 12-layer decoder, some tokens each (copy on write), branches dropped.
        {"name": "pages_branch", "op": "branch", "seqs": 32, "planes": 24, "kv_heads": 12, "head_dim": 64,
         "page": 16, "min_len": 1, "max_len": 1024, "new": 3, "dtype": "bf16"},
        # Copies of 16 whole sequences that do not share pages with their originals.
        {"name": "pages_copy", "op": "copy", "seqs": 16, "planes": 8, "kv_heads": 8, "head_dim": 128,
         "page": 64, "min_len": 100, "max_len": 4096, "new": 0, "dtype": "bf16"},
        # Two groups of sequences leave and return in turn; the pool is compacted each time one has left.
        {"name": "pages_turns", "op": "turns", "seqs": 24, "planes": 8, "kv_heads": 8, "head_dim": 128,
         "page": 16, "min_len": 50, "max_len": 3000, "new": 0, "dtype": "fp16"},
        # One decode step's answer for 16 users: the chosen token's log probability and 20 alternatives.
        {"name": "score_step", "op": "score", "rows": 16, "vocab": 50257, "pad": 47, "top": 20, "dtype": "bf16"},
        # Scoring 16 x 1024 given tokens of GPT-2's vocabulary with 5 alternatives each.
        {"name": "score_prompts", "op": "score", "rows": 16384, "vocab": 50257, "pad": 47, "top": 5,
         "dtype": "bf16"},
        # A policy-gradient step's log probabilities and entropies with their gradient.
        {"name": "train_tokens", "op": "train", "rows": 4096, "vocab": 50257, "pad": 47, "top": 0,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "branch", "copy", "turns", "score", "train"])
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8, 12])
        d = rng.choice([64, 64, 128, 128, 128, 80, 32])
        dtype = rng.choice(["bf16", "bf16", "fp16", "e4m3", "e4m3", "fp32"])
        batch = _log_int(rng, 1, 200)
        most = max(1, min(100000, (1 << 29) // (batch * kv * d)))
        top = _log_int(rng, 1, most)
        return {"op": op, "batch": batch, "heads": kv * rng.choice([1, 1, 2, 4, 5, 7, 8, 16]), "kv_heads": kv,
                "head_dim": d, "page": rng.choice([8, 16, 16, 24, 32, 64, 128, 5]),
                "min_len": rng.choice([0, 1, top]) if top > 1 else top, "max_len": top, "dtype": dtype,
                "mask": rng.choice(["none", "none", "bool", "float"])}
    if op == "append":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        kv, d = rng.choice([1, 2, 4, 8, 12]), rng.choice([64, 128, 80, 33])
        batch = _log_int(rng, 1, 128)
        tokens = _log_int(rng, 1, max(1, min(8192, (1 << 25) // (batch * kv * d))))
        return {"op": op, "batch": batch, "kv_heads": kv, "head_dim": d, "page": rng.choice([8, 16, 24, 64, 128, 5]),
                "tokens": tokens, "min_new": rng.randint(0, tokens), "past": _log_int(rng, 1, 500) - 1,
                "dtype": dtype, "cache": rng.choice([dtype, "e4m3"])}
    if op in ("branch", "copy", "turns"):
        seqs = _log_int(rng, 2, 100)
        planes, kv, d = rng.choice([2, 8, 24]), rng.choice([1, 2, 8, 12]), rng.choice([64, 128, 33])
        dtype = rng.choice(["bf16", "fp16", "fp32", "e4m3"])
        top = _log_int(rng, 1, max(1, min(8192, (1 << 28) // (seqs * planes * kv * d))))
        return {"op": op, "seqs": seqs, "planes": planes, "kv_heads": kv, "head_dim": d,
                "page": rng.choice([8, 16, 24, 64, 128, 5]), "min_len": rng.choice([0, 1, top]) if top > 1 else top,
                "max_len": top, "new": rng.randint(1, 9) if op == "branch" else 0, "dtype": dtype}
    vocab = rng.choice([_log_int(rng, 64, 200000), 50257, 32000, 128256])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    most = (1 << 29 if op == "score" else 1 << 27) // (vocab * (2 if dtype == "fp32" else 1))
    return {"op": op, "rows": _log_int(rng, 1, max(1, min(most, 16384))), "vocab": vocab, "pad": rng.choice([0, 0, 7, 47]),
            "top": rng.choice([0, 1, 5, 20, 64]) if op == "score" else 0, "dtype": dtype}


# ---- inputs ------------------------------------------------------------------

def _lengths(case):
    """Evenly spread lengths, the same for every seed (their order is not)."""
    n, lo, hi = case.get("seqs", case.get("batch")), case["min_len"], case["max_len"]
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _spread(lo, hi, n):
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _held(lens, page):
    return [(n + page - 1) // page for n in lens]


def _random_pages(shape, dtype, gen):
    if dtype == torch.float32:
        return torch.randn(shape, generator=gen, device="cuda")
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).to(dtype)


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen, device="cuda")
    return torch.tensor(values, dtype=torch.int32, device="cuda")[order]


def _fill_table(table, rows, lens, page, ids):
    """Hands `ids` out to the sequences `rows` (lengths on the device) in order."""
    held = (lens.long() + page - 1) // page
    mask = torch.arange(table.shape[1], device="cuda") < held[:, None]
    part = torch.full((len(rows), table.shape[1]), -1, dtype=torch.int32, device="cuda")
    part[mask] = ids.to(torch.int32)
    table[rows] = part
    return int(mask.sum())


def _prepare_attend(case, gen):
    b, hkv, d, page = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    dt = DTYPES[case["dtype"]]
    qdt = torch.bfloat16 if case["dtype"] == "e4m3" else dt
    lens = _lengths(case)
    held = _held(lens, page)
    total, width = sum(held), max(1, max(held))
    n_pages = total + 3
    s = {"lens": _shuffled(lens, gen)}
    s["table"] = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    ids = torch.randperm(n_pages, generator=gen, device="cuda")[:total]
    _fill_table(s["table"], torch.arange(b, device="cuda"), s["lens"], page, ids)
    s["k"] = _random_pages((n_pages, hkv, page, d), dt, gen)
    s["v"] = _random_pages((n_pages, hkv, page, d), dt, gen)
    s["q"] = (1.5 * torch.randn(b, case["heads"], d, generator=gen, device="cuda")).to(qdt)
    s["scale"] = d ** -0.5
    s["ks"] = s["vs"] = s["mask"] = None
    if case["dtype"] == "e4m3":
        s["ks"] = 0.5 + torch.rand(hkv, generator=gen, device="cuda")
        s["vs"] = 0.5 + torch.rand(hkv, generator=gen, device="cuda")
    most = max(1, max(lens))
    if case["mask"] == "bool":  # left padding of up to a third of the sequence
        pad = (s["lens"].float() * torch.rand(b, generator=gen, device="cuda") / 3).int()
        s["mask"] = torch.arange(most, device="cuda") >= pad[:, None]
    elif case["mask"] == "float":  # a bias per key, some keys closed
        bias = torch.randn(b, most, generator=gen, device="cuda")
        closed = torch.rand(b, most, generator=gen, device="cuda") < 0.1
        s["mask"] = torch.where(closed, torch.full_like(bias, -math.inf), bias)
    return s


def _prepare_append(case, gen):
    b, hkv, d, page, n = case["batch"], case["kv_heads"], case["head_dim"], case["page"], case["tokens"]
    new = _shuffled(_spread(case["min_new"], n, b), gen)
    past = torch.randint(0, case["past"] + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
    width = (case["past"] + n + page - 1) // page
    n_pages = b * width + 2
    s = {"new": new, "lens": past + new}
    s["table"] = torch.randperm(n_pages, generator=gen, device="cuda")[:b * width].view(b, width).to(torch.int32)
    dt, cdt = DTYPES[case["dtype"]], DTYPES[case["cache"]]
    s["k_pages"] = _random_pages((n_pages, hkv, page, d), cdt, gen)
    s["v_pages"] = _random_pages((n_pages, hkv, page, d), cdt, gen)
    # a projection's output [B, N, (k, v), H, D], read through views
    kv = torch.randn(b, n, 2, hkv, d, generator=gen, device="cuda", dtype=dt)
    s["k"], s["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    s["ks"] = s["vs"] = None
    if case["cache"] == "e4m3":
        s["ks"] = 0.01 + 0.05 * torch.rand(hkv, generator=gen, device="cuda")
        s["vs"] = 0.005 + 0.05 * torch.rand(hkv, generator=gen, device="cuda")
    return s


def _prepare_pages(case, gen):
    n, page = case["seqs"], case["page"]
    lens = _lengths(case)
    total = sum(_held(lens, page))
    width = max(1, (case["max_len"] + case["new"] + page - 1) // page)
    s = {"page": page, "src": torch.arange(n, dtype=torch.int32, device="cuda"),
         "dst": torch.arange(n, 2 * n, dtype=torch.int32, device="cuda")}
    s["table"] = torch.full((2 * n, width), -1, dtype=torch.int32, device="cuda")
    s["lens"] = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
    first = _shuffled(lens, gen)
    s["lens"][:n] = first
    if case["op"] == "turns":  # the first group low in the pool, the second above it, both in order
        n_pages = 2 * total + 8
        s["lens"][n:] = _shuffled(lens, gen)
        _fill_table(s["table"], s["src"].long(), first, page, torch.arange(total, device="cuda"))
        _fill_table(s["table"], s["dst"].long(), s["lens"][n:], page, torch.arange(total, 2 * total, device="cuda"))
        s["len_a"], s["len_b"] = s["lens"][:n].clone(), s["lens"][n:].clone()
    else:
        n_pages = (2 * total if case["op"] == "copy" else total + n * (2 + case["new"] // page)) + 8
        _fill_table(s["table"], s["src"].long(), first, page,
                    torch.randperm(n_pages, generator=gen, device="cuda")[:total])
    s["refs"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    ids = s["table"][s["table"] >= 0].long()
    s["refs"][ids] = 1
    s["kv"] = _random_pages((case["planes"], n_pages, case["kv_heads"], page, case["head_dim"]),
                            DTYPES[case["dtype"]], gen)
    s["new"] = torch.randint(1, max(1, case["new"]) + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
    return s


def _prepare_logits(case, gen):
    rows, vocab, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    z = torch.randn(rows, vocab + case["pad"], generator=gen, device="cuda", dtype=dt)
    z *= (0.5 + 3.5 * torch.rand(rows, 1, generator=gen, device="cuda")).to(dt)  # flat and peaked rows
    s = {"logits": z[:, :vocab], "top": min(case["top"], vocab)}
    s["tokens"] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    ignored = torch.rand(rows, generator=gen, device="cuda") < 0.1
    if rows > 1:
        s["tokens"] = torch.where(ignored, torch.full_like(s["tokens"], IGNORE), s["tokens"])
    s["g_lp"] = torch.randn(rows, generator=gen, device="cuda")
    s["g_ent"] = 0.01 * torch.randn(rows, generator=gen, device="cuda")
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"attend": _prepare_attend, "append": _prepare_append, "branch": _prepare_pages, "copy": _prepare_pages,
            "turns": _prepare_pages, "score": _prepare_logits, "train": _prepare_logits}[case["op"]]
    s = make(case, gen)
    s["op"] = case["op"]
    return s


# ---- the plain forms ---------------------------------------------------------

def _gathered(pages, ids, scale):
    """[B, Hkv, W*page, D] in 32 bits: the pages of each sequence side by side."""
    raw = pages.view(torch.uint8) if pages.dtype == torch.float8_e4m3fn else pages
    x = raw[ids].permute(0, 2, 1, 3, 4)
    x = x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).view(pages.dtype).float()
    return x if scale is None else x * scale[:, None, None]


def _attend(s):
    q, ids = s["q"], s["table"].clamp_min(0).long()
    k, v = _gathered(s["k"], ids, s["ks"]), _gathered(s["v"], ids, s["vs"])
    b, hkv, n, d = k.shape
    x = torch.matmul(q.float().view(b, hkv, -1, d), k.transpose(2, 3)) * s["scale"]
    open_ = torch.arange(n, device=q.device) < s["lens"][:, None]
    if s["mask"] is not None:
        m = s["mask"][:, :n]
        rest = n - m.shape[1]
        if m.dtype == torch.bool:
            open_ = open_ & torch.cat([m, m.new_ones(b, rest)], 1)
        else:
            x = x + torch.cat([m.float(), m.new_zeros(b, rest).float()], 1)[:, None, None]
    x = torch.where(open_[:, None, None], x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(z > 0, z, torch.ones_like(z))
    return o.reshape(b, -1, d).to(q.dtype)


def _stored(x, scale, dtype):
    if scale is None:
        return x.to(dtype) if dtype != torch.float8_e4m3fn else x.float().clamp(-448, 448).to(dtype)
    return (x.float() / scale).clamp(-448, 448).to(dtype)


def _append(s):
    n, page = s["k"].shape[2], s["k_pages"].shape[2]
    j = torch.arange(n, device="cuda")
    b, t = torch.nonzero(j < s["new"][:, None], as_tuple=True)
    pos = (s["lens"] - s["new"]).long()[b] + t
    ids = s["table"][b, pos // page].long()
    for_h = (lambda c: None if c is None else c[:, None])
    for_raw = (lambda p: p.view(torch.uint8) if p.dtype == torch.float8_e4m3fn else p)
    k = _stored(s["k"][b, :, t], for_h(s["ks"]), s["k_pages"].dtype)
    v = _stored(s["v"][b, :, t], for_h(s["vs"]), s["v_pages"].dtype)
    for_raw(s["k_pages"])[ids, :, pos % page] = for_raw(k)
    for_raw(s["v_pages"])[ids, :, pos % page] = for_raw(v)
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _rows(s, seqs, lens):
    """The page ids of `seqs` [n, W] and which of them `lens` tokens fill."""
    held = (lens + s["page"] - 1) // s["page"]
    return s["table"][seqs], torch.arange(s["table"].shape[1], device="cuda") < held[:, None]


def _count(s, ids, mask, by):
    s["refs"].scatter_add_(0, ids.clamp_min(0).long().reshape(-1), (mask.int() * by).reshape(-1))


def _free(s, seqs):
    ids, mask = _rows(s, seqs, s["lens"][seqs])
    _count(s, ids, mask, -1)
    s["table"][seqs] = torch.where(mask, torch.full_like(ids, -1), ids)
    s["lens"][seqs] = 0


def _fork(s, src, dst):
    _free(s, dst)
    ids, mask = _rows(s, src, s["lens"][src])
    _count(s, ids, mask, 1)
    s["table"][dst] = torch.where(mask, ids, s["table"][dst])
    s["lens"][dst] = s["lens"][src]


def _free_pages(s):
    """Free page ids in ascending order first (the rest after them), and how many they are."""
    used = (s["refs"] > 0).int()
    return torch.argsort(used, stable=True), (1 - used).sum()


def _move(s, src, dst):
    raw = s["kv"].view(torch.uint8) if s["kv"].dtype == torch.float8_e4m3fn else s["kv"]
    raw[:, dst] = raw[:, src]


def _reserve(s, seqs, new):
    page, refs = s["page"], s["refs"]
    lens = s["lens"][seqs]
    old, full = (lens + page - 1) // page, (lens + new + page - 1) // page
    tail_at = (lens // page).clamp_max(s["table"].shape[1] - 1).long()
    tail = s["table"][seqs, tail_at].clamp_min(0).long()
    shared = (new > 0) & (lens % page != 0) & (refs[tail] > 1)
    # the last holder of a shared page keeps it when all the others of this call take copies
    i = torch.arange(len(seqs), device="cuda", dtype=torch.int32)
    sharers = torch.zeros_like(refs).scatter_add_(0, tail, shared.int())
    last = torch.full_like(refs, -1).scatter_reduce_(0, tail, torch.where(shared, i, torch.full_like(i, -1)), "amax")
    keeps = shared & (sharers[tail] == refs[tail]) & (last[tail] == i)
    copies = shared & ~keeps
    need = full - old + copies.int()
    free, n_free = _free_pages(s)
    end = need.cumsum(0)
    ok = (need == 0) | (end <= n_free)
    copied = torch.zeros_like(refs).scatter_add_(0, tail, (copies & ok).int())
    ok = ok & (~keeps | (copied[tail] == sharers[tail] - 1))
    copies = copies & ok
    first = end - need
    cols = torch.arange(s["table"].shape[1], device="cuda")
    fresh = ok[:, None] & (cols >= old[:, None]) & (cols < full[:, None])
    rank = (first + copies.int())[:, None] + cols - old[:, None]
    ids = free[rank.clamp(0, free.numel() - 1).long()].int()
    at_tail = copies[:, None] & (cols == tail_at[:, None])
    ids = torch.where(at_tail, free[first.clamp_max(free.numel() - 1).long()].int()[:, None], ids)
    taken = fresh | at_tail
    _count(s, ids, taken, 1)
    _count(s, tail, copies, -1)
    s["table"][seqs] = torch.where(taken, ids, s["table"][seqs])
    granted = torch.where(ok, new, torch.zeros_like(new))
    s["lens"][seqs] = lens + granted
    _move(s, tail[copies], free[first.long()[copies]])
    return granted


def _copy(s, src, dst):
    _free(s, dst)
    ids, mask = _rows(s, src, s["lens"][src])
    need = mask.sum(1)
    free, n_free = _free_pages(s)
    end = need.cumsum(0)
    ok = (need == 0) | (end <= n_free)
    mask = mask & ok[:, None]
    rank = (end - need)[:, None] + torch.arange(mask.shape[1], device="cuda")
    new = free[rank.clamp_max(free.numel() - 1)].int()
    _count(s, new, mask, 1)
    s["table"][dst] = torch.where(mask, new, s["table"][dst])
    s["lens"][dst] = torch.where(ok, s["lens"][src], torch.zeros_like(s["lens"][src]))
    _move(s, ids[mask].long(), new[mask].long())
    return ok


def _compact(s):
    used = s["refs"] > 0
    live = used.sum()
    at = torch.arange(len(used), device="cuda")
    holes, high = torch.nonzero(~used & (at < live))[:, 0], torch.nonzero(used & (at >= live))[:, 0]
    to = at.int()
    to[high] = holes.int()
    _move(s, high, holes)
    s["refs"][holes] = s["refs"][high]
    s["refs"][high] = 0
    seqs = torch.arange(s["table"].shape[0], device="cuda")
    ids, mask = _rows(s, seqs, s["lens"])
    s["table"].copy_(torch.where(mask, to[ids.clamp_min(0).long()], ids))
    return live.int().reshape(1)


def _pages(s):
    src, dst, out = s["src"].long(), s["dst"].long(), {}
    if s["op"] == "branch":
        _fork(s, src, dst)
        out["granted"] = _reserve(s, dst, s["new"])
        out["table_then"], out["refs_then"] = s["table"].clone(), s["refs"].clone()
        _free(s, dst)
    elif s["op"] == "copy":
        _copy(s, src, dst)
    else:
        _free(s, src)
        out["live_b"] = _compact(s)
        out["granted_a"] = _reserve(s, src, s["len_a"])
        _free(s, dst)
        out["live_a"] = _compact(s)
        out["granted_b"] = _reserve(s, dst, s["len_b"])
    return out | {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "kv": s["kv"]}


def _parts(z):
    """Row maximum, exp(z - maximum), its sum, and z - maximum (0 where the logit is -inf)."""
    top = z.amax(-1, keepdim=True)
    x = z - top
    e = torch.exp(x)
    return top, torch.where(e > 0, x, torch.zeros_like(x)), e, e.sum(-1, keepdim=True)


def _score(s):
    z, t = s["logits"].float(), s["tokens"]
    rows, vocab = z.shape
    top, x, e, total = _parts(z)
    lse = (top + torch.log(total))[:, 0]
    out = {"entropy": (torch.log(total) - (e * x).sum(-1, keepdim=True) / total)[:, 0], "lse": lse}
    chosen = z.gather(1, t.clamp_min(0)[:, None])[:, 0] - top[:, 0] - torch.log(total)[:, 0]
    out["logprobs"] = torch.where(t == IGNORE, torch.zeros_like(chosen), chosen)
    if s["top"]:
        # the value's order as an integer above the inverted index: equal values, lowest index first
        bits = (z + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32)
        key += (vocab - 1) - torch.arange(vocab, device="cuda")
        key = torch.topk(key, s["top"], dim=1).values
        out["top_tokens"] = (vocab - 1) - (key & 0xFFFFFFFF)
        out["top_logprobs"] = z.gather(1, out["top_tokens"]) - lse[:, None]
    return out


def _train(s):
    z, t = s["logits"].float(), s["tokens"]
    _, x, e, total = _parts(z)
    logp = x - torch.log(total)
    p = e / total
    entropy = -(p * logp).sum(-1)
    lp = logp.gather(1, t.clamp_min(0)[:, None])[:, 0]
    lp = torch.where(t == IGNORE, torch.zeros_like(lp), lp)
    g = torch.where(t == IGNORE, torch.zeros_like(lp), s["g_lp"])[:, None]
    grad = p * (-g - s["g_ent"][:, None] * (logp + entropy[:, None]))
    grad.scatter_add_(1, t.clamp_min(0)[:, None], g)
    return {"logprobs": lp, "entropy": entropy, "grad": grad.to(s["logits"].dtype)}


# ---- the framework's calls ---------------------------------------------------

def _own(s):
    import adaattn_b200 as ada
    op = s["op"]
    if op == "attend":
        return ada.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"],
                                   key_mask=s["mask"], k_scale=s["ks"], v_scale=s["vs"])
    if op == "append":
        ada.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["new"],
                         k_scale=s["ks"], v_scale=s["vs"])
        return {"k": s["k_pages"], "v": s["v_pages"]}
    if op in ("branch", "copy", "turns"):
        pool, out = (s["table"], s["lens"], s["refs"]), {}
        src, dst = s["src"], s["dst"]
        if op == "branch":
            ada.fork_pages(*pool, src, dst, page_size=s["page"])
            out["granted"] = ada.reserve_pages(s["kv"], *pool, dst, s["new"])
            out["table_then"], out["refs_then"] = s["table"].clone(), s["refs"].clone()
            ada.free_pages(*pool, dst, page_size=s["page"])
        elif op == "copy":
            ada.copy_pages(s["kv"], *pool, src, dst)
        else:
            ada.free_pages(*pool, src, page_size=s["page"])
            out["live_b"] = ada.compact_pages(s["kv"], *pool)
            out["granted_a"] = ada.reserve_pages(s["kv"], *pool, src, s["len_a"])
            ada.free_pages(*pool, dst, page_size=s["page"])
            out["live_a"] = ada.compact_pages(s["kv"], *pool)
            out["granted_b"] = ada.reserve_pages(s["kv"], *pool, dst, s["len_b"])
        return out | {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "kv": s["kv"]}
    if op == "score":
        r = ada.token_logprobs(s["logits"], s["tokens"], top_k=s["top"], ignore_index=IGNORE)
        out = {"logprobs": r.logprobs, "entropy": r.entropy, "lse": r.lse}
        return out | ({"top_tokens": r.top_tokens, "top_logprobs": r.top_logprobs} if s["top"] else {})
    x = s["logits"].detach().requires_grad_()
    r = ada.token_logprobs(x, s["tokens"], ignore_index=IGNORE)
    grad, = torch.autograd.grad((r.logprobs, r.entropy), x, (s["g_lp"], s["g_ent"]))
    return {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach(), "grad": grad}


def run(state):
    if own:
        return _own(state)
    plain = {"attend": _attend, "append": _append, "branch": _pages, "copy": _pages, "turns": _pages,
             "score": _score, "train": _train}
    return plain[state["op"]](state)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    op = case["op"]
    if op == "attend":
        keys, hkv, d = sum(_lengths(case)), case["kv_heads"], case["head_dim"]
        qelt = 2 if case["dtype"] == "e4m3" else ELT[case["dtype"]]
        mask = {"none": 0, "bool": 1, "float": 4}[case["mask"]] * keys
        io = 2 * case["batch"] * case["heads"] * d * qelt
        ids = 4 * (sum(_held(_lengths(case), case["page"])) + case["batch"])
        return {"bytes": 2 * keys * hkv * d * ELT[case["dtype"]] + mask + io + ids,
                "flops": 4 * keys * case["heads"] * d}
    if op == "append":
        tokens = sum(_spread(case["min_new"], case["tokens"], case["batch"]))
        cells = 2 * tokens * case["kv_heads"] * case["head_dim"]
        return {"bytes": cells * (ELT[case["dtype"]] + ELT[case["cache"]]) + 8 * case["batch"], "flops": 0}
    if op in ("branch", "copy", "turns"):
        page, lens = case["page"], _lengths(case)
        held = sum(_held(lens, page))
        block = case["planes"] * case["kv_heads"] * page * case["head_dim"] * ELT[case["dtype"]]
        moved = {"branch": sum(n % page != 0 for n in lens), "copy": held, "turns": 2 * held}[op]
        return {"bytes": 2 * moved * block + 24 * held + 16 * case["seqs"], "flops": 0}
    cells = case["rows"] * case["vocab"]
    passes = 1 if op == "score" else 2  # training writes the gradient once
    return {"bytes": passes * cells * ELT[case["dtype"]] + 24 * case["rows"], "flops": 6 * passes * cells}


# ---- 64 bits -----------------------------------------------------------------

def _exact_attend(s):
    q = s["q"].double()
    b, h, d = q.shape
    hkv, page = s["k"].shape[1], s["k"].shape[2]
    out = torch.zeros_like(q)
    for i, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        ids = s["table"][i, :(n + page - 1) // page].long()
        for j in range(hkv):
            cut = lambda p: p.view(torch.uint8)[ids, j].view(p.dtype) if p.element_size() == 1 else p[ids, j]
            k = cut(s["k"]).double().reshape(-1, d)[:n]
            v = cut(s["v"]).double().reshape(-1, d)[:n]
            if s["ks"] is not None:
                k, v = k * s["ks"][j].double(), v * s["vs"][j].double()
            heads = slice(j * (h // hkv), (j + 1) * (h // hkv))
            x = q[i, heads] @ k.T * s["scale"]
            if s["mask"] is not None:
                m = s["mask"][i, :n]
                x = x.masked_fill(~m, -math.inf) if m.dtype == torch.bool else x + m.double()
            if bool((x > -math.inf).any()):
                out[i, heads] = torch.softmax(x, -1) @ v
    return out


def _exact_append(case, s):
    if case["cache"] != "e4m3":
        return None
    out = {}
    page = s["k_pages"].shape[2]
    for name, pages, x, scale in (("k", s["k_pages"], s["k"], s["ks"]), ("v", s["v_pages"], s["v"], s["vs"])):
        y = pages.double()
        for i, (new, n) in enumerate(zip(s["new"].tolist(), s["lens"].tolist())):
            pos = torch.arange(n - new, n, device="cuda")
            ids = s["table"][i].long()[pos // page]
            y[ids, :, pos % page] = (x[i, :, :new].double() / scale.double()[:, None, None]).clamp(-448, 448).transpose(0, 1)
        out[name] = y
    return out


def _exact_logits(case, s):
    rows = s["logits"].shape[0]
    keep = {"logprobs": [], "entropy": [], "lse": [], "top_tokens": [], "top_logprobs": [], "grad": []}
    for a in range(0, rows, 1024):
        z, t = s["logits"][a:a + 1024].double(), s["tokens"][a:a + 1024]
        lse = torch.logsumexp(z, -1)
        logp = z - lse[:, None]
        p = torch.exp(logp)
        ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
        chosen = logp[torch.arange(len(t), device="cuda"), t.clamp_min(0)]
        given = (t != IGNORE).double()
        keep["logprobs"].append(chosen * given)
        keep["entropy"].append(ent)
        keep["lse"].append(lse)
        if case["op"] == "train":
            g = s["g_lp"][a:a + 1024].double() * given
            hit = torch.nn.functional.one_hot(t.clamp_min(0), z.shape[1])
            keep["grad"].append(g[:, None] * (hit - p)
                                - s["g_ent"][a:a + 1024].double()[:, None] * p * (logp + ent[:, None]))
        elif s["top"]:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :s["top"]]
            keep["top_tokens"].append(order)
            keep["top_logprobs"].append(logp.gather(1, order))
    out = {k: torch.cat(v) for k, v in keep.items() if v}
    if case["op"] == "train":
        del out["lse"]
    return out


def exact(case, seed):
    if case["op"] in ("branch", "copy", "turns"):
        return None  # whole numbers and moved data: no computed values
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        return _exact_append(case, s)
    return _exact_logits(case, s)
