"""What attention over selected blocks and sampling cost in a serving step, operator by operator.

Four operators: the bounds of a paged cache's keys, page by page ("bounds"), the choice of
the blocks that a query looks at, by those bounds ("select"), attention over the chosen
blocks ("blocks"), and a token drawn from a batch's logits with temperature, top-k, top-p
and min-p and a given random number, with the log of its probability ("sample").

With `own` false the plain forms run (elementary torch operations); with `own` true
the framework's kernels through aero_b200.pages and aero_b200.logits.

A pool holds K and V as (page, kv head, row in page, dim). table[s, i] is the page that
holds block i, positions [i * page, (i + 1) * page), of sequence s. bounds[page, head, 0]
and [.., 1] are the smallest and the largest value of each column of the page's keys.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # bounds for a batch whose pages came from elsewhere: short sequences
        {"name": "bounds_short", "op": "bounds", "dtype": "f16", "n_seq": 16, "kv_heads": 4, "dim": 128, "page": 16,
         "len_min": 1, "len_max": 1000},
        # the same for a pool of long contexts
        {"name": "bounds_long", "op": "bounds", "dtype": "bf16", "n_seq": 32, "kv_heads": 4, "dim": 128, "page": 64,
         "len_min": 8192, "len_max": 16384},
        # one long conversation's next token, small pages: latency
        {"name": "select_one", "op": "select", "dtype": "f16", "n_seq": 1, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 16, "len_min": 32768, "len_max": 32768, "new_max": 0, "blocks": 128, "first": 1, "recent": 2},
        # a batch of long contexts
        {"name": "select_batch", "op": "select", "dtype": "bf16", "n_seq": 48, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 64, "len_min": 8192, "len_max": 32768, "new_max": 0, "blocks": 32, "first": 1, "recent": 1},
        # drafts to be checked: a few tokens of each sequence, each with blocks of its own
        {"name": "select_drafts", "op": "select", "dtype": "f16", "n_seq": 8, "heads": 16, "kv_heads": 4, "dim": 64,
         "page": 32, "len_min": 500, "len_max": 20000, "new_max": 9, "blocks": 64, "first": 1, "recent": 2},
        # the attention that follows: one conversation, 2048 of its 32768 positions
        {"name": "blocks_one", "op": "blocks", "dtype": "f16", "n_seq": 1, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 16, "len_min": 32768, "len_max": 32768, "new_max": 0, "blocks": 128},
        # the batch
        {"name": "blocks_batch", "op": "blocks", "dtype": "bf16", "n_seq": 48, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 64, "len_min": 8192, "len_max": 32768, "new_max": 0, "blocks": 32},
        # drafts over wide heads, some of the sequences shorter than the list
        {"name": "blocks_drafts", "op": "blocks", "dtype": "bf16", "n_seq": 8, "heads": 16, "kv_heads": 2, "dim": 256,
         "page": 32, "len_min": 9, "len_max": 20000, "new_max": 9, "blocks": 64},
        # one conversation's next token, the usual settings: latency
        {"name": "sample_one", "op": "sample", "dtype": "f32", "rows": 1, "vocab": 32000, "style": "top_k",
         "masked": False},
        # a batch over the large vocabulary, nucleus sampling
        {"name": "sample_nucleus", "op": "sample", "dtype": "f32", "rows": 64, "vocab": 151936, "style": "nucleus",
         "masked": False},
        # many parallel samples, temperature alone, 16-bit logits with many ties
        {"name": "sample_free", "op": "sample", "dtype": "bf16", "rows": 256, "vocab": 32000, "style": "free",
         "masked": False},
        # requests of every kind in one batch, under a grammar that forbids half of the tokens
        {"name": "sample_mixed", "op": "sample", "dtype": "f32", "rows": 16, "vocab": 151936, "style": "mixed",
         "masked": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= limit["bytes"] and w["flops"] <= limit["flops"] and _pool_bytes(c) <= 3.0e9:
            return c


def _drawn(rng):
    op = rng.choice(["bounds", "select", "select", "blocks", "blocks", "sample", "sample", "sample"])
    if op == "sample":
        return {"op": op, "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "rows": _log(rng, 1, 256),
                "vocab": _log(rng, 1000, 152000), "style": rng.choice(["top_k", "nucleus", "free", "min_p", "mixed"]),
                "masked": rng.random() < 0.3}
    c = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "kv_heads": rng.choice([1, 2, 4, 8]),
         "dim": rng.choice([64, 128, 128, 192, 256]), "page": rng.choice([8, 16, 32, 64, 128, 256]),
         "n_seq": _log(rng, 1, 64), "len_max": _log(rng, 1, 32768)}
    c["len_min"] = max(1, int(c["len_max"] * rng.random()))
    if op == "bounds":
        return c
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 8, 16])
    c["new_max"] = rng.choice([0, 0, min(c["len_min"], rng.randint(1, 9))])
    c["blocks"] = _log(rng, 4, 128)
    if op == "select":  # a list that does not hold all blocks of the longest sequence
        c["first"], c["recent"] = rng.choice([0, 1, 1]), rng.choice([1, 2])
        c["len_max"] = max(c["len_max"], 16 * c["page"])
        c["blocks"] = min(c["blocks"], c["len_max"] // c["page"] // 2)
    return c


# Lengths, new tokens and the pages of each sequence: they follow from the case alone.
def _plan(case):
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    P, n = case["page"], case["n_seq"]
    lens = [r.randint(case["len_min"], case["len_max"]) for _ in range(n)]
    if n > 1:
        lens[r.randrange(n)] = case["len_max"]
    drafts = case.get("new_max", 0)
    new = [r.randint(1, drafts) if drafts else 1 for _ in range(n)]
    used = sum(-(-x // P) for x in lens)
    width = max(-(-x // P) for x in lens)
    order = list(range(used))
    r.shuffle(order)
    table, at = [], 0
    for x in lens:
        k = -(-x // P)
        table.append(order[at:at + k] + [-1] * (width - k))
        at += k
    return {"lens": lens, "new": new, "table": table, "refs": [1] * used, "n_page": used, "width": width}


def _pool_bytes(case):
    if case["op"] == "sample":
        return 0
    return _plan(case)["n_page"] * 2 * case["kv_heads"] * case["page"] * case["dim"] * 2


def work(case):
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": case["rows"] * case["vocab"] * 3}
    p = _plan(case)
    P, HK, D = case["page"], case["kv_heads"], case["dim"]
    row = HK * D * 2
    if case["op"] == "bounds":
        return {"bytes": row * sum(p["lens"]) + 2 * row * p["n_page"], "flops": 2 * HK * D * sum(p["lens"])}
    H, T = case["heads"], sum(p["new"])
    q = T * H * D * 2
    size = flops = 0
    for n, x in zip(p["lens"], p["new"]):
        blocks = [-(-(n - i) // P) for i in range(x)]  # visible to each new token, the last one first
        if case["op"] == "select":
            size += 2 * row * blocks[0]
            flops += 2 * H * D * sum(blocks)
        else:
            seen = [(min(b, case["blocks"]) - 1) * P + n - i - (b - 1) * P for i, b in enumerate(blocks)]
            size += 2 * row * min(sum(seen), n)
            flops += 4 * H * D * sum(seen)
    lists = T * HK * case["blocks"] * 4
    return {"bytes": size + lists + (1 if case["op"] == "select" else 2) * q, "flops": flops}


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "sample":
        return _prepare_sample(case, g, dt)
    p = _plan(case)
    P, HK, D = case["page"], case["kv_heads"], case["dim"]
    st = {"case": case, "plan": p, "table": _dev(p["table"]), "length": _dev(p["lens"]),
          "seqs": _dev(list(range(case["n_seq"]))), "scale": 1.0 / math.sqrt(D)}
    if own:
        from aero_b200.pages import PagedCache
        cache = st["cache"] = PagedCache(1, p["n_page"], P, HK, D, case["n_seq"], p["width"], dtype=dt, bounds=True)
        st["k"], st["v"] = cache.k(0), cache.v(0)
    else:
        st["k"] = torch.empty((p["n_page"], HK, P, D), dtype=dt, device="cuda")
        st["v"] = torch.empty_like(st["k"])
    # keys of a block are alike: a mean of their own and what each adds to it
    st["k"].normal_(generator=g)
    st["k"].add_(torch.empty((p["n_page"], HK, 1, D), dtype=dt, device="cuda").normal_(std=0.7, generator=g))
    if case["op"] == "blocks":
        st["v"].normal_(generator=g)
    if own:
        cache.set_tables(st["table"], st["length"], _dev(p["refs"]))
        st["bounds"] = cache.bounds(0)
        if case["op"] == "select":
            cache.set_bounds(0, st["seqs"])
    elif case["op"] == "select":
        st["bounds"] = _plain_bounds(st)
    if case["op"] != "bounds":
        T = sum(p["new"])
        st["q"] = torch.empty((T, case["heads"], D), dtype=dt, device="cuda").normal_(std=2.0, generator=g)
        start = [0]
        for x in p["new"]:
            start.append(start[-1] + x)
        st["q_start"] = _dev(start) if case["new_max"] else None
        st["row_seq"] = [s for s, x in enumerate(p["new"]) for _ in range(x)]
        st["row_len"] = [n - x + i + 1 for n, x in zip(p["lens"], p["new"]) for i in range(x)]
        if case["op"] == "blocks":
            st["lists"] = _lists(case, st["row_len"], g)
    torch.cuda.synchronize()
    return st


def _lists(case, row_len, g):
    """For each token and kv head as many of its blocks as the list holds, the first and its own
    among them, ascending, -1 behind."""
    nb = torch.tensor([-(-n // case["page"]) for n in row_len], device="cuda")[:, None, None]
    width, most = case["blocks"], max(-(-n // case["page"]) for n in row_len)
    at = torch.arange(max(most, width), device="cuda")[None, None, :]
    key = torch.rand((len(row_len), case["kv_heads"], at.shape[-1]), device="cuda", generator=g)
    key = torch.where((at == 0) | (at == nb - 1), torch.full_like(key, 2.0), key)
    key = torch.where(at < nb, key, torch.full_like(key, -1.0))
    value, number = key.topk(width, dim=-1)
    number = torch.where(value >= 0, number, torch.full_like(number, 1 << 30)).sort(-1).values
    return torch.where(number < (1 << 30), number, torch.full_like(number, -1)).to(torch.int32).contiguous()


def _prepare_sample(case, g, dt):
    B, V = case["rows"], case["vocab"]
    # a language model's logits: a broad mass of unlikely tokens, a few that stand out
    x = torch.empty((B, V), device="cuda").normal_(std=2.0, generator=g)
    likely = torch.randint(0, V, (B, 50), device="cuda", generator=g)
    x.scatter_add_(1, likely, 14.0 * torch.rand((B, 50), device="cuda", generator=g))
    if case["masked"]:
        x.masked_fill_(torch.rand((B, V), device="cuda", generator=g) < 0.5, -math.inf)
    st = {"case": case, "logits": x.to(dt), "u": torch.rand(B, device="cuda", generator=g),
          "temperature": 0.6 + 0.8 * torch.rand(B, device="cuda", generator=g), "top_k": None, "top_p": None, "min_p": None}
    kind, style = torch.arange(B, device="cuda"), case["style"]
    if style in ("top_k", "mixed"):
        st["top_k"] = torch.full((B,), 40, dtype=torch.int32, device="cuda")
    if style in ("top_k", "nucleus", "mixed"):
        st["top_p"] = 0.85 + 0.1 * torch.rand(B, device="cuda", generator=g)
    if style in ("min_p", "mixed"):
        st["min_p"] = 0.02 + 0.05 * torch.rand(B, device="cuda", generator=g)
    if style == "mixed":  # by turns: the largest, top-k and top-p, wide top-k, top-p alone, min-p alone, no limit
        kind = kind % 6
        st["temperature"] = torch.where(kind == 0, 0.0, st["temperature"])
        k = torch.tensor([0, 40, 5000, 0, 0, 0], dtype=torch.int32, device="cuda")
        st["top_k"] = k[kind].contiguous()
        st["top_p"] = torch.where((kind == 1) | (kind == 3), st["top_p"], 1.0)
        st["min_p"] = torch.where(kind == 4, st["min_p"], 0.0)
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        if op == "sample":
            from aero_b200.logits import sample
            return sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                          top_p=state["top_p"], min_p=state["min_p"], logprob=True)
        cache = state["cache"]
        if op == "bounds":
            cache.set_bounds(0, state["seqs"])
            return state["bounds"]
        if op == "select":
            return cache.select(0, state["q"], state["seqs"], state["q_start"], n_blocks=case["blocks"],
                                first=case["first"], recent=case["recent"])
        return cache.attend_blocks(0, state["q"], state["seqs"], state["lists"], state["q_start"])
    return {"sample": _plain_sample, "bounds": _plain_bounds, "select": _plain_select, "blocks": _plain_blocks}[op](state)


def _plain_bounds(st):
    case, p = st["case"], st["plan"]
    P, HK, D = case["page"], case["kv_heads"], case["dim"]
    out = torch.zeros((p["n_page"], HK, 2, D), dtype=st["k"].dtype, device="cuda")
    slot = torch.arange(p["width"], device="cuda")[None, :]
    length = st["length"][:, None].long()
    held = slot * P < length
    page = st["table"][held].long()
    rows = (length - slot * P).clamp(max=P)[held]
    step = max(1, int(2.5e8 // (HK * P * D)))
    for i in range(0, page.numel(), step):
        x = st["k"][page[i:i + step]].float()
        hidden = (torch.arange(P, device="cuda")[None, :] >= rows[i:i + step, None])[:, None, :, None]
        out[page[i:i + step], :, 0] = x.masked_fill(hidden, math.inf).amin(2).to(out.dtype)
        out[page[i:i + step], :, 1] = x.masked_fill(hidden, -math.inf).amax(2).to(out.dtype)
    return out


def _plain_select(st):
    """Scores in 64 bits: they say which block comes before which."""
    case, p = st["case"], st["plan"]
    P, HK, D, W = case["page"], case["kv_heads"], case["dim"], case["blocks"]
    G = case["heads"] // HK
    T, most = len(st["row_len"]), p["width"]
    q = st["q"].double().reshape(T, HK, G, D)
    out = torch.empty((T, HK, W), dtype=torch.int32, device="cuda")
    at = torch.arange(max(most, W), device="cuda")[None, None, :]
    row_seq = torch.tensor(st["row_seq"], device="cuda")
    nb = ((torch.tensor(st["row_len"], device="cuda") + P - 1) // P)[:, None, None]
    step = max(1, int(1.0e8 // (most * HK * D)))
    for t0 in range(0, T, step):
        t1 = min(T, t0 + step)
        b = st["bounds"][st["table"][row_seq[t0:t1]].clamp(min=0).long()].double()  # (t, block, head, 2, dim)
        lo, hi = b[:, :, :, 0].permute(0, 2, 3, 1), b[:, :, :, 1].permute(0, 2, 3, 1)
        qq, n = q[t0:t1], nb[t0:t1]
        score = (qq.clamp(min=0) @ hi + qq.clamp(max=0) @ lo).amax(2)
        key = torch.full((t1 - t0, HK, at.shape[-1]), -math.inf, dtype=torch.float64, device="cuda")
        key[:, :, :most] = score
        key = torch.where((at < case["first"]) | (at >= n - case["recent"]), torch.full_like(key, math.inf), key)
        key = torch.where(at < n, key, torch.full_like(key, -math.inf))
        number = key.sort(dim=-1, descending=True, stable=True).indices[:, :, :W]
        number = torch.where(number < n, number, torch.full_like(number, 1 << 30)).sort(-1).values
        out[t0:t1] = torch.where(number < (1 << 30), number, torch.full_like(number, -1)).to(torch.int32)
    return out


def _plain_blocks(st):
    case = st["case"]
    P, HK, D, W = case["page"], case["kv_heads"], case["dim"], case["blocks"]
    G, T = case["heads"] // HK, len(st["row_len"])
    out = torch.empty_like(st["q"])
    row_seq = torch.tensor(st["row_seq"], device="cuda")
    n = torch.tensor(st["row_len"], device="cuda")[:, None, None]
    head = torch.arange(HK, device="cuda")[None, :, None]
    step = max(1, int(2.0e8 // (HK * W * P * D)))
    for t0 in range(0, T, step):
        t1 = min(T, t0 + step)
        lists = st["lists"][t0:t1].long()
        page = st["table"][row_seq[t0:t1, None, None], lists.clamp(min=0)].long()
        at = (lists[..., None] * P + torch.arange(P, device="cuda")).reshape(t1 - t0, HK, W * P)
        seen = (lists >= 0).repeat_interleave(P, -1) & (at < n[t0:t1])
        K = st["k"][page, head].float().reshape(t1 - t0, HK, W * P, D)
        V = st["v"][page, head].float().reshape(t1 - t0, HK, W * P, D)
        S = (st["q"][t0:t1].float().reshape(-1, HK, G, D) @ K.transpose(-1, -2)) * st["scale"]
        S = S.masked_fill(~seen[:, :, None, :], -math.inf)
        w = torch.exp(S - S.amax(-1, keepdim=True))
        o = (w @ V) / w.sum(-1, keepdim=True)
        out[t0:t1] = o.reshape(-1, case["heads"], D).to(out.dtype)
    return out


def _plain_sample(st):
    """Weights and their running sums in 64 bits: a token is where a sum passes a border."""
    x = st["logits"].double()
    B, V = x.shape
    value, number = x.sort(dim=1, descending=True, stable=True)
    T = st["temperature"].double()[:, None]
    log_w = (value - value[:, :1]) / torch.where(T > 0, T, torch.ones_like(T))
    w = torch.exp(log_w)
    place = torch.arange(V, device="cuda")[None, :]
    kept = torch.where(T > 0, place >= 0, place < 1)
    if st["top_k"] is not None:
        k = st["top_k"][:, None]
        kept &= (place < k) | (k <= 0)
    if st["top_p"] is not None:
        run = torch.cumsum(w * kept, 1)
        p = st["top_p"].double()[:, None]
        kept &= (run - w < p * run[:, -1:]) | (p >= 1)
    if st["min_p"] is not None:
        kept &= w >= st["min_p"].double()[:, None]
    run = torch.cumsum(w * kept, 1)
    past = run > st["u"].double()[:, None] * run[:, -1:]
    at = past.to(torch.uint8).argmax(1, keepdim=True)
    return [number.gather(1, at)[:, 0].to(torch.int32), (log_w.gather(1, at) - torch.log(run[:, -1:]))[:, 0].float()]


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"sample": _exact_sample, "bounds": _exact_bounds, "select": _exact_select, "blocks": _exact_blocks}[case["op"]](st)


def _exact_bounds(st):
    case, p = st["case"], st["plan"]
    P = case["page"]
    out = torch.zeros((p["n_page"], case["kv_heads"], 2, case["dim"]), dtype=torch.float64, device="cuda")
    for s, n in enumerate(p["lens"]):
        full = p["table"][s][:n // P]
        if full:
            k = st["k"][torch.tensor(full, device="cuda")].double()
            out[torch.tensor(full, device="cuda")] = torch.stack([-(-k).max(2).values, k.max(2).values], 2)
        if n % P:
            k = st["k"][p["table"][s][n // P], :, :n % P].double()
            out[p["table"][s][n // P]] = torch.stack([-(-k).max(1).values, k.max(1).values], 1)
    return out


def _exact_select(st):
    """Token by token and head by head, the products' larger one taken column by column."""
    case, p = st["case"], st["plan"]
    P, HK, W = case["page"], case["kv_heads"], case["blocks"]
    G = case["heads"] // HK
    T = len(st["row_len"])
    out = np.full((T, HK, W), -1, dtype=np.int32)
    for t in range(T):
        nb = -(-st["row_len"][t] // P)
        b = st["bounds"][torch.tensor(p["table"][st["row_seq"][t]][:nb], device="cuda")].double()
        q = st["q"][t].double().reshape(HK, G, -1)
        best = None
        for g in range(G):
            s = torch.maximum(q[:, g] * b[:, :, 0], q[:, g] * b[:, :, 1]).sum(-1)  # (block, head)
            best = s if best is None else torch.maximum(best, s)
        best = best.cpu().numpy()
        number = np.arange(nb)
        always = (number < case["first"]) | (number >= nb - case["recent"])
        for h in range(HK):
            order = np.argsort(-best[:, h], kind="stable")
            got = np.sort(np.concatenate([number[always], order[~always[order]]])[:W])
            out[t, h, :len(got)] = got
    return out


def _exact_blocks(st):
    case, p = st["case"], st["plan"]
    P, HK = case["page"], case["kv_heads"]
    G = case["heads"] // HK
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lists = st["lists"].cpu().numpy()
    for t, (s, n) in enumerate(zip(st["row_seq"], st["row_len"])):
        for h in range(HK):
            at = np.concatenate([np.arange(b * P, min(n, (b + 1) * P)) for b in lists[t, h] if b >= 0])
            page = torch.tensor(np.array(p["table"][s])[at // P], device="cuda")
            row = torch.tensor(at % P, device="cuda")
            K, V = st["k"][page, h, row].double(), st["v"][page, h, row].double()
            z = (st["q"][t, h * G:(h + 1) * G].double() @ K.T) * st["scale"]
            out[t, h * G:(h + 1) * G] = torch.softmax(z, 1) @ V
    return out


def _exact_sample(st):
    x, u = st["logits"].double().cpu().numpy(), st["u"].double().cpu().numpy()
    T = st["temperature"].double().cpu().numpy()
    k, p, least = (None if st[n] is None else st[n].double().cpu().numpy() for n in ("top_k", "top_p", "min_p"))
    out, log_p = np.zeros(len(x), dtype=np.int32), np.zeros(len(x))
    for r in range(len(x)):
        order = np.argsort(-x[r], kind="stable")
        if T[r] <= 0:
            out[r] = order[0]
            continue
        w = np.exp((x[r][order] - x[r][order[0]]) / T[r])
        if k is not None and k[r] > 0:
            w = w[:int(k[r])]
        if p is not None and p[r] < 1:
            w = w[:1 + int(np.count_nonzero(np.cumsum(w)[:-1] < p[r] * w.sum()))]
        if least is not None:
            w = w[w >= least[r]]
        at = np.count_nonzero(np.cumsum(w) <= u[r] * w.sum())
        out[r], log_p[r] = order[at], (x[r][order[at]] - x[r][order[0]]) / T[r] - np.log(w.sum())
    return [out, log_p]
