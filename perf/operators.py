"""A decode step of many requests at once, operator by operator, as cases that can be timed.

  step    block tables, row starts, positions and cache slots from the requests' lengths and a stack of free pages: a step takes
          pages for its new tokens, then the step is rolled back (every draft rejected) and the pages return
  append  the step's K and V rows into their slots of a paged cache
  attn    the step's queries (one new token a request, or a verify block of a few) over the paged cache
  sample  the next tokens from logits, with temperature, top-k, top-p, min-p and given random numbers

Requests have ragged lengths, `low` x `longest` to `longest`, fixed by the case; contents, page order and random numbers come
from the seed.  Sizes are those of this repository's models (8 or 2 KV heads of 256, vocabularies of 262144 and 32768) or generic.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False             # False: the operators in plain torch; True: this framework's kernels

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # 48 chats, one new token each: the smallest step, all latency
        {"name": "step_chats", "op": "step", "requests": 48, "longest": 2000, "low": 0.1, "page": 16, "new": 1, "chunk": 0},
        # a full server: verify blocks of 4, and every 16th request brings in a part of its prompt
        {"name": "step_server", "op": "step", "requests": 2048, "longest": 8000, "low": 0.05, "page": 16, "new": 4, "chunk": 257},
        # the K and V rows of 48 chats: 32-bit projections into an f16 cache, 8 KV heads of 256
        {"name": "append_chats", "op": "append", "tokens": 48, "kv_heads": 8, "dim": 256, "page": 16, "type": "f32", "cache": "f16"},
        # prompts of many requests, bf16 throughout, an odd number of rows
        {"name": "append_prompts", "op": "append", "tokens": 8191, "kv_heads": 8, "dim": 256, "page": 64, "type": "bf16", "cache": "bf16"},
        # one chat at its beginning: latency
        {"name": "attn_one", "op": "attn", "requests": 1, "longest": 300, "low": 1.0, "page": 16, "new": 1, "heads": 16, "kv_heads": 8,
         "dim": 256, "type": "f32", "cache": "f16", "window": 0},
        # 48 chats on the model with two KV heads of 256
        {"name": "attn_chats", "op": "attn", "requests": 48, "longest": 4001, "low": 0.05, "page": 16, "new": 1, "heads": 8, "kv_heads": 2,
         "dim": 256, "type": "f32", "cache": "f16", "window": 0},
        # verify blocks of 4 on the model with eight KV heads of 256
        {"name": "attn_verify", "op": "attn", "requests": 32, "longest": 8190, "low": 0.2, "page": 32, "new": 4, "heads": 16, "kv_heads": 8,
         "dim": 256, "type": "f32", "cache": "f16", "window": 0},
        # a full server, grouped heads of 128, bf16
        {"name": "attn_server", "op": "attn", "requests": 96, "longest": 16383, "low": 0.1, "page": 16, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "bf16", "cache": "bf16", "window": 0},
        # two very long documents: the work has to be split over the length
        {"name": "attn_long", "op": "attn", "requests": 2, "longest": 120001, "low": 0.9, "page": 64, "new": 1, "heads": 32, "kv_heads": 4,
         "dim": 128, "type": "bf16", "cache": "bf16", "window": 0},
        # one row of a vocabulary of 262144 with the usual filters: latency
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 262144, "type": "f32", "top_k": 64, "top_p": 0.95, "min_p": 0.0},
        # 48 chats, top-p and min-p over the whole vocabulary
        {"name": "sample_chats", "op": "sample", "rows": 48, "vocab": 262144, "type": "f32", "top_k": 0, "top_p": 0.9, "min_p": 0.02},
        # many rows of a smaller vocabulary in 16 bits, temperature alone
        {"name": "sample_many", "op": "sample", "rows": 512, "vocab": 32768, "type": "bf16", "top_k": 0, "top_p": 1.0, "min_p": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("step", "append", "attn", "attn", "sample", "sample"))
    if op == "step":
        return {"op": op, "requests": _log(rng, 1, 2048), "longest": _log(rng, 1, 8000), "low": rng.choice((0.05, 0.5, 1.0)),
                "page": rng.choice((8, 16, 24, 64)), "new": rng.randint(1, 8), "chunk": rng.choice((0, 0, _log(rng, 9, 257)))}
    if op == "append":
        kind = rng.choice((("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")))
        return {"op": op, "tokens": _log(rng, 1, 8191), "kv_heads": rng.randint(1, 8), "dim": rng.choice((64, 80, 128, 256)),
                "page": rng.choice((1, 8, 16, 24, 64)), "type": kind[0], "cache": kind[1]}
    if op == "sample":
        vocab = _log(rng, 50, 262144)
        return {"op": op, "rows": _log(rng, 1, min(512, (512 * 32768) // vocab)), "vocab": vocab, "type": rng.choice(("f32", "f16", "bf16")),
                "top_k": rng.choice((0, 0, 1, _log(rng, 2, 2000))), "top_p": rng.choice((1.0, round(rng.uniform(0.3, 0.99), 3))),
                "min_p": rng.choice((0.0, round(rng.uniform(0.001, 0.2), 4)))}
    kind = rng.choice((("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")))
    kv_heads, dim = rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 80, 128, 256, 512))
    requests = _log(rng, 1, 96)
    room = (96 * 16383 * 8 * 128 * 2) // (4 * requests * kv_heads * dim * BYTES[kind[1]])
    new = rng.choice((1, 1, 1, rng.randint(2, 8)))
    return {"op": op, "requests": requests, "longest": _log(rng, new, max(new, min(131072, room))), "low": rng.choice((0.05, 0.5, 1.0)),
            "page": rng.choice((8, 16, 24, 64, 128)), "new": new, "heads": kv_heads * rng.choice((1, 2, 4, 7, 8)), "kv_heads": kv_heads,
            "dim": dim, "type": kind[0], "cache": kind[1], "window": rng.choice((0, 0, 0, _log(rng, 16, 2048)))}


def _spread(case, least=1):
    """The requests' lengths: longest first, the others spread evenly over low x longest .. longest in no order."""
    n, top = case["requests"], case["longest"]
    return [max(least, min(top, round(top * (1 - (1 - case["low"]) * ((i * 0.6180339887498949) % 1.0))))) for i in range(n)]


def _news(case):
    return [case["chunk"] if case["chunk"] and i % 16 == 15 else case["new"] for i in range(case["requests"])]


def _pages(lengths, page):
    return [-(-n // page) for n in lengths]


def work(case):
    op = case["op"]
    if op == "step":
        lens, news = _spread(case), _news(case)
        taken = sum(_pages([a + b for a, b in zip(lens, news)], case["page"])) - sum(_pages(lens, case["page"]))
        # lengths and new tokens in; page ids off the stack and into the tables; starts and three words a token out; lengths back
        return {"bytes": 4 * (4 * len(lens) + 1) + 12 * sum(news) + 16 * taken, "flops": 0}
    if op == "append":
        return {"bytes": case["tokens"] * (4 + 2 * case["kv_heads"] * case["dim"] * (BYTES[case["type"]] + BYTES[case["cache"]])), "flops": 0}
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * BYTES[case["type"]] + 28 * case["rows"], "flops": 4 * n}
    lens = _spread(case, case["new"])
    w, new = case["window"], case["new"]
    keys = sum(min(n, w + new - 1) if w else n for n in lens)          # rows that some query of the block sees
    seen = sum(min(n - new + 1 + t, w) if w else n - new + 1 + t for n in lens for t in range(new))
    rows = case["requests"] * new * case["heads"] * case["dim"]
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * BYTES[case["cache"]] + 2 * rows * BYTES[case["type"]] + 4 * keys // case["page"],
            "flops": 4 * seen * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(pages, columns, order):
    """Block table [requests][columns]: request r holds the next pages[r] ids of `order`, -1 behind them."""
    n = torch.tensor(pages, device="cuda")
    first = torch.cumsum(n, 0) - n
    col = torch.arange(columns, device="cuda")
    at = (first[:, None] + col).clamp(max=max(0, len(order) - 1))
    return torch.where(col < n[:, None], order[at], -1).to(torch.int32)


def _cache(g, n_pages, case):
    shape = (n_pages, case["page"], case["kv_heads"], case["dim"])
    return [torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["cache"]]) for _ in range(2)]


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"op": op, "case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # logits of a language model: a wide bulk, a few tokens far above it, some that a grammar rules out
        x = torch.randn((rows, vocab), generator=g, device="cuda") * 2.2
        x += torch.where(torch.rand((rows, vocab), generator=g, device="cuda") < 20.0 / vocab, 6.0, 0.0)
        x[:, 1:vocab:97] = -math.inf
        s["logits"] = x.to(DTYPES[case["type"]])
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        s["temperature"] = 0.6 + 0.8 * torch.rand(rows, generator=g, device="cuda")
        s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda") if case["top_k"] else None
        s["top_p"] = torch.full((rows,), case["top_p"], device="cuda") if case["top_p"] < 1 else None
        s["min_p"] = torch.full((rows,), case["min_p"], device="cuda") if case["min_p"] > 0 else None
        s["token"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["prob"] = torch.empty(rows, device="cuda")
        if own:
            s["lg"] = importlib.import_module("little-gemma_b200")
        return s
    page = case["page"]
    if op == "append":
        n, spare = case["tokens"], 3 * page
        s["k_cache"], s["v_cache"] = _cache(g, -(-(n + spare) // page), case)
        width = case["kv_heads"] * case["dim"]
        s["k"], s["v"] = (torch.randn((n, width), generator=g, device="cuda").to(DTYPES[case["type"]]) for _ in range(2))
        s["slot"] = torch.randperm(s["k_cache"].shape[0] * page, generator=g, device="cuda")[:n].to(torch.int32)
        lens, spare_pages, columns, order = [1], 0, 1, torch.zeros(1, dtype=torch.int64, device="cuda")
    else:
        new = _news(case) if op == "step" else [0] * case["requests"]
        lens = _spread(case, 1 if op == "step" else case["new"])
        spare_pages = sum(_pages([a + b for a, b in zip(lens, new)], page)) - sum(_pages(lens, page)) + 5
        columns = max(_pages([a + b for a, b in zip(lens, new)], page))
        order = torch.randperm(sum(_pages(lens, page)) + spare_pages, generator=g, device="cuda")
    held = sum(_pages(lens, page)) if op != "append" else 0
    s["len"] = _ints(lens)
    s["table"] = _table(_pages(lens, page), columns, order)
    s["free"] = torch.zeros(len(order), dtype=torch.int32, device="cuda")
    s["free"][: len(order) - held] = order[held:].to(torch.int32)
    s["n_free"] = _ints([len(order) - held])
    if op == "step":
        cap = sum(new)
        s["keep"], s["new"], s["none"] = s["len"].clone(), _ints(new), torch.zeros(len(lens), dtype=torch.int32, device="cuda")
        for name, n in (("start", len(lens) + 1), ("pos", cap), ("slot", cap), ("req", cap)):
            s[name] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["back"] = torch.empty(len(lens) + 1, dtype=torch.int32, device="cuda")
        # a step needs no rows of a cache: the smallest that has these pages
        s["k_cache"] = s["v_cache"] = torch.empty((len(order), page, 1, 8), dtype=torch.float16, device="cuda")
    if op == "attn":
        s["k_cache"], s["v_cache"] = _cache(g, len(order), case)
        rows = case["requests"] * case["new"]
        s["q"] = (torch.randn((rows, case["heads"], case["dim"]), generator=g, device="cuda") * 1.5).to(DTYPES[case["type"]])
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["lg"] = importlib.import_module("little-gemma_b200")
        stack = (s["free"], s["n_free"]) if op == "step" else ()
        s["cache"] = s["lg"].PagedCache(s["k_cache"], s["v_cache"], s["table"], s["len"], *stack)
        if op == "attn":
            s["work"] = torch.empty(s["cache"].attn_work(case["requests"], case["new"], case["heads"]), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------------

def run(s):
    return {"step": _step, "append": _append, "attn": _attn, "sample": _sample}[s["op"]](s)


def _step(s):
    if own:
        c = s["cache"]
        c.step(s["new"], s["start"], s["pos"], s["slot"], s["req"], stream=s["stream"])
        c.step(s["none"], s["back"], keep=s["keep"], stream=s["stream"])
        return {k: s[k] for k in ("start", "pos", "slot", "req", "back", "table", "len", "free", "n_free")}
    page, rows = s["case"]["page"], s["pos"].numel()
    old, new, keep, table, free, n_free = (s[k].long() for k in ("len", "new", "keep", "table", "free", "n_free"))
    col = torch.arange(table.shape[1], device="cuda")
    # pages from the top of the stack, in the order of the requests
    have, need = (old + page - 1) // page, (old + new + page - 1) // page
    take = need - have
    at = torch.cumsum(take, 0) - take
    fresh = (col >= have[:, None]) & (col < need[:, None])
    pop = at[:, None] + col - have[:, None]
    table = torch.where(fresh, free[(n_free - 1 - pop).clamp(0, len(free) - 1)], table)
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(new, 0)])
    token = torch.arange(rows, device="cuda")
    req = torch.searchsorted(start, token, right=True) - 1
    pos = old[req] + token - start[req]
    slot = table[req, pos // page] * page + pos % page
    length, n_free = old + new, n_free - take.sum()
    # the roll-back: what lies behind the kept rows returns, the last page first
    have, need = need, (keep + page - 1) // page
    give = have - need
    at = torch.cumsum(give, 0) - give
    gone = (col >= need[:, None]) & (col < have[:, None])
    push = n_free + give.sum() - 1 - (at[:, None] + col - need[:, None])
    free = torch.cat([free, free[:1]]).scatter(0, torch.where(gone, push, len(free)).reshape(-1), table.reshape(-1))[:-1]
    table = torch.where(gone, -1, table)
    length, n_free = torch.minimum(length, keep), n_free + give.sum()
    out = {"start": start, "pos": pos, "slot": slot, "req": req, "back": torch.zeros_like(start), "table": table, "len": length,
           "free": free, "n_free": n_free}
    return {k: v.to(torch.int32) for k, v in out.items()}


def _append(s):
    if own:
        s["cache"].append(s["k"], s["v"], s["slot"], stream=s["stream"])
    else:
        at = s["slot"].long()
        for cache, rows in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
            flat = cache.view(-1, cache.shape[2] * cache.shape[3])
            flat[at] = rows.to(cache.dtype)
    return {"k": s["k_cache"], "v": s["v_cache"]}


def _attn(s):
    c = s["case"]
    if own:
        s["cache"].attn(s["q"], s["out"], s["work"], n_new=c["new"], window=c["window"], stream=s["stream"])
        return s["out"]
    n, new, heads, kv, dim = c["requests"], c["new"], c["heads"], c["kv_heads"], c["dim"]
    pages = s["table"].long().clamp(min=0)
    k, v = (s[x][pages].reshape(n, -1, kv, dim).float() for x in ("k_cache", "v_cache"))
    q = s["q"].view(n, new, kv, heads // kv, dim).float()
    score = torch.einsum("rtkgd,rlkd->rktgl", q, k) * dim ** -0.5
    del k
    at = torch.arange(v.shape[1], device="cuda")
    top = s["len"][:, None] - new + torch.arange(new, device="cuda")             # position of each new token
    seen = at <= top[..., None]
    if c["window"]:
        seen &= at > top[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    score = torch.exp(score.sub_(score.amax(-1, keepdim=True)))
    score = score.div_(score.sum(-1, keepdim=True))
    out = torch.einsum("rktgl,rlkd->rtkgd", score, v)
    return out.reshape(n * new, heads, dim).to(s["q"].dtype)


def _sample(s):
    if own:
        s["lg"].sample(s["logits"], s["u"], s["token"], s["prob"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                       min_p=s["min_p"], stream=s["stream"])
        return {"token": s["token"], "prob": s["prob"]}
    # 64 bits throughout: a token is decided by where a running sum over the vocabulary passes a number
    x = s["logits"].double()
    w = torch.exp((x - x.amax(-1, keepdim=True)) / s["temperature"].double()[:, None])
    if s["top_k"] is not None or s["top_p"] is not None or s["min_p"] is not None:
        _, order = torch.sort(x, dim=-1, descending=True, stable=True)           # ties: the lowest index first
        sw = w.gather(-1, order)
        rank = torch.arange(x.shape[1], device="cuda")
        keep = torch.ones_like(sw, dtype=torch.bool)
        if s["top_k"] is not None:
            keep &= rank < s["top_k"][:, None]
        if s["top_p"] is not None:
            sw = sw * keep
            total = torch.cumsum(sw, -1)
            keep &= total - sw < s["top_p"].double()[:, None] * total[:, -1:]
        if s["min_p"] is not None:
            keep &= sw >= s["min_p"].double()[:, None]
        keep |= rank == 0
        w = w * torch.zeros_like(keep).scatter(-1, order, keep)
    total = torch.cumsum(w, -1)
    below = (total <= s["u"].double()[:, None] * total[:, -1:]).sum(-1, keepdim=True).clamp(max=x.shape[1] - 1)
    prob = w.gather(-1, below) / total[:, -1:]
    return {"token": below[:, 0].to(torch.int32), "prob": prob[:, 0].float()}


# ------------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "step":
        return None                                                              # whole numbers
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            cache = s[name + "_cache"].double().cpu().numpy()
            flat = cache.reshape(-1, case["kv_heads"] * case["dim"])
            flat[s["slot"].cpu().numpy()] = s[name].double().cpu().numpy()
            out[name] = cache
        return out
    if case["op"] == "sample":
        logits, u, temp = (s[k].double().cpu().numpy() for k in ("logits", "u", "temperature"))
        prob = np.empty(case["rows"])
        for r in range(case["rows"]):
            prob[r] = _drawn(logits[r], u[r], temp[r], case["top_k"], float(np.float32(case["top_p"])), float(np.float32(case["min_p"])))
        return {"token": None, "prob": prob}
    n, new, heads, kv, dim = (case[k] for k in ("requests", "new", "heads", "kv_heads", "dim"))
    out = torch.empty((n, new, heads, dim), dtype=torch.float64, device="cuda")
    lens = s["len"].tolist()
    for r in range(n):
        rows = s["table"][r, : -(-lens[r] // case["page"])].long()
        k, v = (s[x][rows].flatten(0, 1)[: lens[r]].double() for x in ("k_cache", "v_cache"))
        for t in range(new):
            hi = lens[r] - new + t + 1
            lo = max(0, hi - case["window"]) if case["window"] else 0
            q = s["q"][r * new + t].double().view(kv, heads // kv, dim)
            p = torch.softmax(q @ k[lo:hi].permute(1, 2, 0) / math.sqrt(dim), -1)
            out[r, t] = (p @ v[lo:hi].transpose(0, 1)).reshape(heads, dim)
    return out.view(n * new, heads, dim)


def _drawn(logits, u, temperature, top_k, top_p, min_p):
    """The probability of the token that one row of logits and one random number give, by sorting."""
    p = np.exp((logits - logits.max()) / temperature)
    order = np.lexsort((np.arange(len(p)), -logits))
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        run = np.cumsum(p[order])
        order = order[: max(1, int(np.searchsorted(np.concatenate([[0.0], run[:-1]]), top_p * run[-1], side="left")))]
    if min_p > 0:
        order = order[: max(1, int(np.count_nonzero(p[order] >= min_p)))]
    kept = np.sort(order)
    run = np.cumsum(p[kept])
    i = min(int(np.searchsorted(run, u * run[-1], side="right")), len(kept) - 1)
    return p[kept[i]] / run[-1]
