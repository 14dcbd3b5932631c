"""What a serving step over a paged key/value cache costs, operator by operator.

Four operators: attention of one new token per sequence over a paged cache
("decode"), attention of several new tokens per sequence over the same cache, with
a sliding window and first tokens that stay visible ("prompt"), the cache's own
bookkeeping and page moves ("step", "fork", "compact"), and the logits of a batch
adjusted by repetition penalties, biases and grammar masks ("logits").

With `own` false the plain forms run (elementary torch operations in 32 bits);
with `own` true the framework's kernels through aero_b200.pages and
aero_b200.logits.

A pool holds K and V as (layer, page, kv head, row in page, dim). table[s, i] is the
page that holds positions [i * page, (i + 1) * page) of sequence s, or -1.
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
        # one conversation of the 48-layer decoder (32 query heads on 4 kv heads of 128,
        # a 4096-position cache), one token: latency
        {"name": "decode_one", "op": "decode", "dtype": "f16", "n_seq": 1, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 16, "len_min": 4096, "len_max": 4096, "window": 0, "sinks": 0},
        # the same decoder's batch of 16, sequences of every length up to the cache's end
        {"name": "decode_batch", "op": "decode", "dtype": "bf16", "n_seq": 16, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 64, "len_min": 1, "len_max": 4096, "window": 0, "sinks": 0},
        # long contexts, many at once: the cache is the whole cost
        {"name": "decode_long", "op": "decode", "dtype": "f16", "n_seq": 48, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 64, "len_min": 8192, "len_max": 32768, "window": 0, "sinks": 0},
        # wide heads, a window and four first tokens: long histories of which little is read
        {"name": "decode_window", "op": "decode", "dtype": "bf16", "n_seq": 64, "heads": 16, "kv_heads": 2, "dim": 256,
         "page": 32, "len_min": 2000, "len_max": 20000, "window": 1024, "sinks": 4},
        # short turns over short histories: drafts to be checked, tails of prompts
        {"name": "prompt_few", "op": "prompt", "dtype": "f16", "n_seq": 8, "heads": 16, "kv_heads": 4, "dim": 64,
         "page": 16, "new_min": 1, "new_max": 9, "past_min": 0, "past_max": 1000, "window": 0, "sinks": 0},
        # a chunk of several prompts in windowed layers
        {"name": "prompt_window", "op": "prompt", "dtype": "bf16", "n_seq": 4, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 64, "new_min": 500, "new_max": 2100, "past_min": 0, "past_max": 2000, "window": 1024, "sinks": 4},
        # one long prompt, causal
        {"name": "prompt_long", "op": "prompt", "dtype": "f16", "n_seq": 1, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 64, "new_min": 16384, "new_max": 16384, "past_min": 0, "past_max": 0, "window": 0, "sinks": 0},
        # what a decode step does to the cache: a row for each sequence, a page where one is full
        {"name": "step_rows", "op": "step", "dtype": "f16", "n_seq": 16, "layers": 4, "kv_heads": 4, "dim": 128,
         "page": 16, "len_min": 1, "len_max": 1000, "new_max": 1, "spare": 64},
        # four prompts continued four ways each (parallel samples, beams)
        {"name": "fork_beams", "op": "fork", "dtype": "bf16", "n_seq": 4, "ways": 4, "layers": 12, "kv_heads": 4,
         "dim": 128, "page": 16, "len_min": 100, "len_max": 1000, "spare": 64},
        # after half of the sequences ended: the live pages to the pool's front
        {"name": "compact_pool", "op": "compact", "dtype": "f16", "n_seq": 64, "ended": 32, "layers": 8, "kv_heads": 4,
         "dim": 128, "page": 32, "len_min": 100, "len_max": 1900, "spare": 0},
        # one conversation's next token: latency
        {"name": "logits_one", "op": "logits", "dtype": "f32", "rows": 1, "vocab": 32000, "history": 500, "biases": 8,
         "masked": True},
        # a batch over the large vocabulary, long histories
        {"name": "logits_batch", "op": "logits", "dtype": "f32", "rows": 64, "vocab": 151936, "history": 8192,
         "biases": 64, "masked": True},
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
    op = rng.choice(["decode", "decode", "prompt", "prompt", "step", "fork", "compact", "logits"])
    if op == "logits":
        return {"op": op, "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "rows": _log(rng, 1, 64),
                "vocab": _log(rng, 1000, 152000), "history": _log(rng, 1, 8192), "biases": rng.choice([0, 8, 64]),
                "masked": rng.random() < 0.6}
    c = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "kv_heads": rng.choice([1, 2, 4, 8]),
         "dim": rng.choice([64, 128, 128, 192, 256]), "page": rng.choice([8, 16, 32, 64, 128])}
    if op in ("decode", "prompt"):
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 8, 16])
        windowed = rng.random() < 0.5
        c["window"] = _log(rng, 16, 4096) if windowed else 0
        c["sinks"] = rng.choice([0, 1, 4, 100]) if windowed else 0
    if op == "decode":
        c["n_seq"] = _log(rng, 1, 64)
        c["len_max"] = _log(rng, 1, 32768)
        c["len_min"] = max(1, int(c["len_max"] * rng.random()))
    elif op == "prompt":
        c["n_seq"] = _log(rng, 1, 16)
        c["new_max"] = _log(rng, 1, 16384)
        c["new_min"] = max(1, int(c["new_max"] * rng.random()))
        c["past_max"] = _log(rng, 1, 16384) if rng.random() < 0.7 else 0
        c["past_min"] = int(c["past_max"] * rng.random())
    else:
        c["layers"] = _log(rng, 1, 12)
        c["n_seq"] = _log(rng, 2, 64)
        c["len_max"] = _log(rng, 2, 2000)
        c["len_min"] = max(1, int(c["len_max"] * rng.random()))
        c["spare"] = rng.choice([0, 17, 300])
        if op == "step":
            c["new_max"] = _log(rng, 1, 300)
            c["spare"] += c["n_seq"] * (c["new_max"] // c["page"] + 1)
        elif op == "fork":
            c["n_seq"] = min(c["n_seq"], 16)
            c["ways"] = rng.randint(1, 5)
            c["spare"] += c["n_seq"] * c["ways"]
        else:
            c["ended"] = rng.randint(1, c["n_seq"] - 1)
    return c


# Everything about a case but the values: lengths, the pages of each sequence, who is forked
# or has ended. It follows from the case alone.
def _plan(case):
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    op, P = case["op"], case["page"]
    n = case["n_seq"]
    new = [0] * n
    if op == "prompt":
        new = [r.randint(case["new_min"], case["new_max"]) for _ in range(n)]
        lens = [r.randint(case["past_min"], case["past_max"]) + x for x in new]
    else:
        lens = [r.randint(case["len_min"], case["len_max"]) for _ in range(n)]
        if op in ("decode", "prompt") and n > 1:
            lens[r.randrange(n)] = case["len_max"]
    rows = n * (1 + case.get("ways", 0))
    if op == "step":
        new = [r.randint(1, case["new_max"]) for _ in range(n)]
    used = sum(-(-x // P) for x in lens)
    n_page = used + case.get("spare", 0)
    width = max(-(-(x + y) // P) for x, y in zip(lens, new)) if op == "step" else max(-(-x // P) for x in lens)
    order = list(range(n_page))
    r.shuffle(order)
    table = [[-1] * width for _ in range(rows)]
    refs = [0] * n_page
    at = 0
    for s, x in enumerate(lens):
        for i in range(-(-x // P)):
            table[s][i] = order[at]
            refs[order[at]] = 1
            at += 1
    length = lens + [0] * (rows - n)
    ended = []
    if op == "compact":
        ended = sorted(r.sample(range(n), case["ended"]))
        for s in ended:
            for i in range(-(-lens[s] // P)):
                refs[table[s][i]] = 0
                table[s][i] = -1
            length[s] = 0
    parents = [s for s in range(n) for _ in range(case.get("ways", 0))]
    return {"lens": lens, "new": new, "length": length, "table": table, "refs": refs, "n_page": n_page, "width": width,
            "rows": rows, "parents": parents, "children": list(range(n, rows))}


def _page_bytes(case):
    return case.get("layers", 1) * 2 * case["kv_heads"] * case["page"] * case["dim"] * 2


def _pool_bytes(case):
    return 0 if case["op"] == "logits" else _plan(case)["n_page"] * _page_bytes(case)


def _visible(n, window, sinks):
    """Keys that the token at position n - 1 sees."""
    if not window or n <= window:
        return n
    return window + min(sinks, n - window)


def work(case):
    op = case["op"]
    if op == "logits":
        size = 4 if case["dtype"] == "f32" else 2
        per = 2 * case["vocab"] * size + case["history"] * 4 + case["biases"] * 8
        per += (case["vocab"] + 31) // 32 * 4 if case["masked"] else 0
        return {"bytes": case["rows"] * per, "flops": case["rows"] * case["vocab"] * 3}
    p = _plan(case)
    row = case["kv_heads"] * case["dim"] * 2
    if op in ("decode", "prompt"):
        new = p["new"] if op == "prompt" else [1] * case["n_seq"]
        pairs = keys = 0
        for n, x in zip(p["lens"], new):
            w, s = case["window"], case["sinks"]
            if not w:
                pairs += x * n - x * (x - 1) // 2
                keys += n
            else:
                pairs += sum(_visible(n - i, w, s) for i in range(x))
                low = max(0, n - x - w + 1)  # the first key in the first new token's window
                keys += n - low + min(s, low)
        q = sum(new) * case["heads"] * case["dim"] * 2
        return {"bytes": 2 * row * keys + 2 * q, "flops": 4 * pairs * case["heads"] * case["dim"]}
    books = (p["rows"] * p["width"] + p["rows"] + p["n_page"]) * 4
    if op == "step":
        return {"bytes": 2 * books + 2 * 2 * row * case["layers"] * sum(p["new"]), "flops": 0}
    if op == "fork":
        part = sum(p["lens"][s] % case["page"] for s in p["parents"])
        return {"bytes": 2 * books + 2 * 2 * row * case["layers"] * part, "flops": 0}
    live = sum(1 for x in p["refs"] if x)
    moved = sum(1 for x in p["refs"][live:] if x)
    return {"bytes": 2 * books + 2 * moved * _page_bytes(case), "flops": 0}


# ------------------------------------------------------------------ the inputs
def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _fill(t, g):
    """Normal values, a layer at a time (the same ones whoever owns the memory)."""
    for layer in range(t.shape[0]):
        t[layer].normal_(generator=g)


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "logits":
        return _prepare_logits(case, g, dt)
    p = _plan(case)
    P, HK, D, L = case["page"], case["kv_heads"], case["dim"], case.get("layers", 1)
    st = {"case": case, "plan": p, "table": _dev(p["table"]), "length": _dev(p["length"]), "refs": _dev(p["refs"]),
          "scale": 1.0 / math.sqrt(D)}
    if own:
        from aero_b200.pages import PagedCache
        st["cache"] = PagedCache(L, p["n_page"], P, HK, D, p["rows"], p["width"], dtype=dt)
        st["k"], st["v"] = st["cache"].k(), st["cache"].v()
    else:
        st["k"] = torch.empty((L, p["n_page"], HK, P, D), dtype=dt, device="cuda")
        st["v"] = torch.empty_like(st["k"])
    _fill(st["k"], g)
    _fill(st["v"], g)
    if case["op"] in ("decode", "prompt"):
        new = p["new"] if case["op"] == "prompt" else [1] * case["n_seq"]
        # normed and scaled queries of a trained head: scores of a few units
        st["q"] = torch.empty((sum(new), case["heads"], D), dtype=dt, device="cuda").normal_(std=2.0, generator=g)
        st["seqs"] = _dev(list(range(case["n_seq"])))
        start = [0]
        for x in new:
            start.append(start[-1] + x)
        st["start"], st["q_start"] = start, _dev(start)
        if own:
            st["cache"].set_tables(st["table"], st["length"], st["refs"])
    elif case["op"] == "step":
        T = sum(p["new"])
        st["new_k"] = torch.empty((L, T, HK, D), dtype=dt, device="cuda").normal_(generator=g)
        st["new_v"] = torch.empty((L, T, HK, D), dtype=dt, device="cuda").normal_(generator=g)
        st["seqs"] = _dev(list(range(case["n_seq"])))
        st["counts"] = _dev(p["new"])
        st["row_seq"] = _dev([s for s, x in enumerate(p["new"]) for _ in range(x)])
        st["row_pos"] = _dev([p["lens"][s] + i for s, x in enumerate(p["new"]) for i in range(x)])
    elif case["op"] == "fork":
        st["parents"], st["children"] = _dev(p["parents"]), _dev(p["children"])
    if own and case["op"] not in ("decode", "prompt"):
        st["books"] = st["cache"].tables()
    torch.cuda.synchronize()
    return st


def _prepare_logits(case, g, dt):
    B, V, Hn, nb = case["rows"], case["vocab"], case["history"], case["biases"]
    st = {"case": case}
    st["logits"] = torch.empty((B, V), device="cuda").normal_(std=3.0, generator=g).to(dt)
    # tokens of a text: few of them often
    u = torch.rand((B, Hn), device="cuda", generator=g)
    st["history"] = (u.pow(4) * V).to(torch.int32).clamp_(max=V - 1)
    st["n_history"] = torch.randint((Hn + 1) // 2, Hn + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    st["n_prompt"] = (st["n_history"] // 2).to(torch.int32)
    st["repetition"] = 1.0 + 0.3 * torch.rand(B, device="cuda", generator=g)
    st["frequency"] = 0.5 * torch.rand(B, device="cuda", generator=g)
    st["presence"] = 0.5 * torch.rand(B, device="cuda", generator=g)
    # each row's biases: tokens of its own, none twice
    step = V // max(nb, 1)
    at = torch.randint(0, max(step, 1), (B, nb), device="cuda", generator=g)
    st["bias_token"] = (at + torch.arange(nb, device="cuda") * step).to(torch.int32).reshape(-1).contiguous()
    st["bias_value"] = torch.empty(B * nb, device="cuda").normal_(std=2.0, generator=g)
    st["bias_start"] = torch.arange(B + 1, device="cuda", dtype=torch.int32) * nb
    st["mask"] = None
    if case["masked"]:  # one bit a token, set: allowed; half of the vocabulary
        st["mask"] = torch.randint(-2**31, 2**31, (B, (V + 31) // 32), device="cuda", generator=g).to(torch.int32)
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        if op == "logits":
            from aero_b200.logits import adjust
            return adjust(state["logits"], history=state["history"], n_history=state["n_history"],
                          n_prompt=state["n_prompt"], repetition=state["repetition"], frequency=state["frequency"],
                          presence=state["presence"], bias_start=state["bias_start"], bias_token=state["bias_token"],
                          bias_value=state["bias_value"], mask=state["mask"])
        cache = state["cache"]
        if op == "decode":
            return cache.attend(0, state["q"], state["seqs"], window=case["window"], sinks=case["sinks"])
        if op == "prompt":
            return cache.attend(0, state["q"], state["seqs"], state["q_start"], window=case["window"],
                                sinks=case["sinks"])
        cache.set_tables(state["table"], state["length"], state["refs"])
        if op == "step":
            cache.extend(state["seqs"], state["counts"])
            for layer in range(case["layers"]):
                cache.append(layer, state["new_k"][layer], state["new_v"][layer], state["row_seq"], state["row_pos"])
        elif op == "fork":
            cache.fork(state["parents"], state["children"])
        else:
            cache.compact()
        return [*state["books"], state["k"], state["v"]]
    if op == "logits":
        return _plain_logits(state)
    if op == "decode":
        return _plain_decode(state)
    if op == "prompt":
        return _plain_prompt(state)
    table, length, refs = state["table"].clone(), state["length"].clone(), state["refs"].clone()
    return {"step": _plain_step, "fork": _plain_fork, "compact": _plain_compact}[op](state, table, length, refs)


def _rows_of(pool, table_rows, P):
    """Rows of the pages in table_rows (b, n), in 32 bits: (b, kv head, n * page, dim)."""
    x = pool[table_rows.clamp(min=0).long()]  # (b, n, kv head, page, dim)
    b, n, HK, _, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, HK, n * P, D).float()


def _softmax_product(S, seen, V):
    S = S.masked_fill(~seen, -math.inf)
    m = S.amax(-1, keepdim=True)
    p = torch.exp(S - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return (p @ V) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_decode(st):
    case, p = st["case"], st["plan"]
    P, HK, D, H = case["page"], case["kv_heads"], case["dim"], case["heads"]
    out = torch.empty_like(st["q"])
    n = p["width"] * P
    at = torch.arange(n, device="cuda")
    batch = max(1, int(1.0e9 // (n * HK * D * 4)))
    for b0 in range(0, case["n_seq"], batch):
        seqs = st["seqs"][b0:b0 + batch].long()
        pages, lens = st["table"][seqs], st["length"][seqs]
        K, V = _rows_of(st["k"][0], pages, P), _rows_of(st["v"][0], pages, P)
        q = st["q"][b0:b0 + batch].float().reshape(-1, HK, H // HK, D)
        seen = at[None, :] < lens[:, None]
        if case["window"]:
            seen &= (at[None, :] >= lens[:, None] - case["window"]) | (at[None, :] < case["sinks"])
        o = _softmax_product((q @ K.transpose(-1, -2)) * st["scale"], seen[:, None, None, :], V)
        out[b0:b0 + batch] = o.reshape(-1, H, D).to(out.dtype)
    return out


def _plain_prompt(st):
    case, p = st["case"], st["plan"]
    P, HK, D, H = case["page"], case["kv_heads"], case["dim"], case["heads"]
    G = H // HK
    out = torch.empty_like(st["q"])
    for s in range(case["n_seq"]):
        n, x, t0 = p["lens"][s], p["new"][s], st["start"][s]
        pages = st["table"][s:s + 1, :-(-n // P)]
        K, V = _rows_of(st["k"][0], pages, P)[0, :, :n], _rows_of(st["v"][0], pages, P)[0, :, :n]
        at = torch.arange(n, device="cuda")
        step = max(1, int(2.5e8 // (n * H)))
        for r0 in range(0, x, step):
            r1 = min(x, r0 + step)
            q = st["q"][t0 + r0:t0 + r1].float().reshape(r1 - r0, HK, G, D).permute(1, 2, 0, 3)
            pos = torch.arange(n - x + r0, n - x + r1, device="cuda")[:, None]
            seen = at[None, :] <= pos
            if case["window"]:
                seen &= (at[None, :] > pos - case["window"]) | (at[None, :] < case["sinks"])
            o = _softmax_product((q @ K[:, None].transpose(-1, -2)) * st["scale"], seen, V[:, None])
            out[t0 + r0:t0 + r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, H, D).to(out.dtype)
    return out


def _lowest_free(refs, want, slots):
    """want (n,) pages for each of n rows, in order, out of the lowest free ones: (n, slots)
    page numbers (-1 past a row's want), and refs with them taken."""
    free = refs == 0
    rank = torch.cumsum(free, 0) - 1  # a free page's place among the free ones
    n_page = refs.numel()
    number = torch.arange(n_page, device=refs.device)
    by_rank = torch.full((n_page + 1,), -1, dtype=torch.long, device=refs.device)
    by_rank[torch.where(free, rank, torch.full_like(rank, n_page))] = number
    first = torch.cumsum(want, 0) - want
    slot = torch.arange(slots, device=refs.device)
    ask = (first[:, None] + slot[None, :]).clamp(max=n_page)
    got = torch.where(slot[None, :] < want[:, None], by_rank[ask], torch.full_like(ask, -1))
    taken = free & (rank < want.sum())
    return got, refs + taken.to(refs.dtype)


def _plain_step(st, table, length, refs):
    case, p = st["case"], st["plan"]
    P = case["page"]
    seqs, counts = st["seqs"].long(), st["counts"].long()
    before = length[seqs].long()
    have, need = (before + P - 1) // P, (before + counts + P - 1) // P
    slots = (case["new_max"] + P - 1) // P + 1
    got, refs = _lowest_free(refs, need - have, slots)
    wide = torch.cat([table, torch.full((table.shape[0], slots + 1), -1, dtype=table.dtype, device="cuda")], 1)
    at = have[:, None] + torch.arange(slots, device="cuda")[None, :]
    wide[seqs[:, None], torch.where(got >= 0, at, torch.full_like(at, wide.shape[1] - 1))] = got.to(table.dtype)
    table = wide[:, :table.shape[1]].contiguous()
    length[seqs] = (before + counts).to(length.dtype)
    pos = st["row_pos"].long()
    page = table[st["row_seq"].long(), pos // P].long()
    for layer in range(case["layers"]):
        st["k"][layer][page, :, pos % P] = st["new_k"][layer]
        st["v"][layer][page, :, pos % P] = st["new_v"][layer]
    return [table, length, refs, st["k"], st["v"]]


def _plain_fork(st, table, length, refs):
    case, p = st["case"], st["plan"]
    P = case["page"]
    parents, children = st["parents"].long(), st["children"].long()
    lens = length[parents].long()
    full, part = lens // P, lens % P
    slot = torch.arange(table.shape[1], device="cuda")
    rows = torch.where(slot[None, :] < full[:, None], table[parents], torch.full_like(table[parents], -1))
    shared = torch.where(rows >= 0, rows, torch.full_like(rows, refs.numel())).long().reshape(-1)
    more = torch.zeros(refs.numel() + 1, dtype=refs.dtype, device="cuda")
    more.index_add_(0, shared, torch.ones_like(shared, dtype=refs.dtype))
    got, refs = _lowest_free(refs, (part > 0).long(), 1)
    refs = refs + more[:-1]
    wide = torch.cat([rows, torch.full((rows.shape[0], 1), -1, dtype=rows.dtype, device="cuda")], 1)
    last = torch.where(part > 0, full, torch.full_like(full, table.shape[1]))
    source = torch.cat([table, torch.full_like(table[:, :1], -1)], 1)[parents, last].long()
    wide.scatter_(1, last[:, None], got.to(wide.dtype))
    table[children] = wide[:, :table.shape[1]]
    length[children] = length[parents]
    pick = part > 0
    src, dst, left = source[pick], got[:, 0][pick], part[pick]
    keep = (torch.arange(P, device="cuda")[None, :] < left[:, None])[:, None, :, None]
    for layer in range(case["layers"]):
        for pool in (st["k"][layer], st["v"][layer]):
            pool[dst] = torch.where(keep, pool[src], pool[dst])
    return [table, length, refs, st["k"], st["v"]]


def _plain_compact(st, table, length, refs):
    live = refs > 0
    n_page = refs.numel()
    number = torch.arange(n_page, device="cuda")
    n_live = live.sum()
    holes = (~live & (number < n_live)).nonzero()[:, 0]
    movers = (live & (number >= n_live)).nonzero()[:, 0]
    to = number.clone()
    to[movers] = holes
    for layer in range(st["case"]["layers"]):
        for pool in (st["k"][layer], st["v"][layer]):
            pool[holes] = pool[movers]
    new_refs = refs.clone()
    new_refs[holes] = refs[movers]
    new_refs[movers] = 0
    table = torch.where(table >= 0, to[table.clamp(min=0).long()].to(table.dtype), table)
    return [table, length, new_refs, st["k"], st["v"]]


def _plain_logits(st):
    case = st["case"]
    B, V, Hn = case["rows"], case["vocab"], case["history"]
    x = st["logits"].float()
    place = torch.arange(Hn, device="cuda")[None, :]
    given = place < st["n_history"][:, None]
    answered = given & (place >= st["n_prompt"][:, None])
    tok = st["history"].long()
    seen = torch.zeros((B, V), device="cuda").scatter_add_(1, tok, given.float())
    count = torch.zeros((B, V), device="cuda").scatter_add_(1, tok, answered.float())
    rep = st["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0).float()
    nb = case["biases"]
    if nb:
        bias = torch.zeros((B, V), device="cuda")
        bias.scatter_add_(1, st["bias_token"].long().reshape(B, nb), st["bias_value"].reshape(B, nb))
        x = x + bias
    if st["mask"] is not None:
        v = torch.arange(V, device="cuda")
        allowed = (st["mask"][:, v // 32] >> (v % 32).to(torch.int32)[None, :]) & 1
        x = torch.where(allowed > 0, x, torch.full_like(x, -math.inf))
    return x.to(st["logits"].dtype)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "logits":
        return _exact_logits(st)
    if case["op"] in ("decode", "prompt"):
        return _exact_attention(st)
    return _exact_books(st)


def _exact_attention(st):
    """Sequence by sequence: the visible keys' rows taken out by number, no mask but the causal one."""
    case, p = st["case"], st["plan"]
    P, HK, H = case["page"], case["kv_heads"], case["heads"]
    W, S = case["window"], case["sinks"]
    G = H // HK
    q = st["q"].double()
    out = torch.zeros_like(q)
    for s in range(case["n_seq"]):
        n = p["lens"][s]
        new = p["new"][s] if case["op"] == "prompt" else 1
        t0 = st["start"][s]
        pages = torch.tensor(p["table"][s], device="cuda")
        block = max(1, int(1.2e8 // (n * G)))
        for b0 in range(0, new, block):
            b1 = min(new, b0 + block)
            first, last = n - new + b0, n - new + b1 - 1  # positions of the block's tokens
            low = max(0, first - W + 1) if W else 0
            keys = torch.cat([torch.arange(min(S, low) if W else 0), torch.arange(low, last + 1)]).cuda()
            page, row = pages[keys // P], keys % P
            pos = torch.arange(first, last + 1, device="cuda")[:, None]
            hidden = keys[None, :] > pos
            if W:
                hidden |= (pos - keys[None, :] >= W) & (keys[None, :] >= S)
            for h in range(HK):
                K, V = st["k"][0][page, h, row].double(), st["v"][0][page, h, row].double()
                for g in range(G):
                    z = (q[t0 + b0:t0 + b1, h * G + g] @ K.T) * st["scale"]
                    z[hidden] = -math.inf
                    out[t0 + b0:t0 + b1, h * G + g] = torch.softmax(z, 1) @ V
    return out


def _exact_books(st):
    case, p = st["case"], st["plan"]
    P = case["page"]
    table, length, refs = [list(r) for r in p["table"]], list(p["length"]), list(p["refs"])
    k, v = st["k"].clone(), st["v"].clone()

    def take():
        page = refs.index(0)
        refs[page] = 1
        return page

    if case["op"] == "step":
        at = 0
        for s, x in enumerate(p["new"]):
            for _ in range(x):
                n = length[s]
                if n % P == 0:
                    table[s][n // P] = take()
                length[s] = n + 1
            idx = torch.arange(length[s] - x, length[s], device="cuda")
            page = torch.tensor(table[s], device="cuda")[idx // P]
            k[:, page, :, idx % P] = st["new_k"][:, at:at + x].transpose(0, 1)
            v[:, page, :, idx % P] = st["new_v"][:, at:at + x].transpose(0, 1)
            at += x
    elif case["op"] == "fork":
        for a, b in zip(p["parents"], p["children"]):
            n = length[a]
            for i in range(n // P):
                table[b][i] = table[a][i]
                refs[table[a][i]] += 1
            if n % P:
                new = take()
                table[b][n // P] = new
                old = table[a][n // P]
                k[:, new, :, :n % P] = k[:, old, :, :n % P]
                v[:, new, :, :n % P] = v[:, old, :, :n % P]
            length[b] = n
    else:
        live = sum(1 for x in refs if x)
        holes = [i for i in range(live) if not refs[i]]
        movers = [i for i in range(live, len(refs)) if refs[i]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            k[:, b], v[:, b] = k[:, a], v[:, a]
            refs[b], refs[a] = refs[a], 0
        table = [[to.get(x, x) for x in r] for r in table]
    return [np.array(table, dtype=np.int32), np.array(length, dtype=np.int32), np.array(refs, dtype=np.int32), k, v]


def _exact_logits(st):
    x = st["logits"].double().cpu().numpy()
    hist, n, np_ = (st[k].cpu().numpy() for k in ("history", "n_history", "n_prompt"))
    rep, freq, pres = (st[k].double().cpu().numpy() for k in ("repetition", "frequency", "presence"))
    b0, bt, bv = (st[k].cpu().numpy() for k in ("bias_start", "bias_token", "bias_value"))
    for r in range(x.shape[0]):
        seen = np.unique(hist[r, :n[r]])
        row = x[r]
        row[seen] = np.where(row[seen] > 0, row[seen] / rep[r], row[seen] * rep[r])
        tok, cnt = np.unique(hist[r, np_[r]:n[r]], return_counts=True)
        row[tok] -= freq[r] * cnt + pres[r]
        for i in range(b0[r], b0[r + 1]):
            row[bt[i]] += float(bv[i])
        if st["mask"] is not None:
            bits = st["mask"][r].cpu().numpy().view(np.uint8)
            row[np.unpackbits(bits, bitorder="little")[:row.size] == 0] = -np.inf
    return x
