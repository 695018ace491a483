"""Operators of a language model's serving path, measured: attention under masks and score changes for prompts, and, for
token-by-token generation, the plan that gives new tokens their places in a paged cache, the append that quantises them
into it (8 bits, one scale for each page and head), and the attention that reads it.

Each operator has its plain form here (elementary torch operations in 32 bits); with `own` set, `run` makes the calls of
the framework instead. `exact` gives the same results from the definitions in 64 bits."""
import math
import os
import random
import sys

import torch

own = False

F8 = torch.float8_e4m3fn
TOP = 448.0         # largest e4m3 value
LEAST = -100        # exponent of the smallest scale
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A decode step of 64 requests: one new token each, a page boundary crossed now and then.
        dict(name="plan_decode", op="plan", requests=64, page=32, longest=4096, prompt=1),
        # Admission of a large mixed batch: prompts of all lengths beside requests that generate.
        dict(name="plan_prompts", op="plan", requests=1024, page=16, longest=8192, prompt=1024),
        # The new tokens of one decode step enter the cache.
        dict(name="append_decode", op="append", requests=64, page=32, longest=4096, prompt=1, kv_heads=8, dim=128, type="f16"),
        # Whole prompts enter the cache.
        dict(name="append_prompts", op="append", requests=24, page=64, longest=64, prompt=2600, kv_heads=8, dim=128, type="bf16"),
        # One user, a short context: latency is all.
        dict(name="paged_single", op="paged", requests=1, page=32, longest=2048, shortest=2048, queries=1, heads=32, kv_heads=8,
             dim=128, type="f16", cap=0.0, slopes=False),
        # A serving batch of ragged contexts, grouped heads.
        dict(name="paged_batch", op="paged", requests=64, page=32, longest=8192, shortest=1, queries=1, heads=32, kv_heads=8,
             dim=128, type="bf16", cap=0.0, slopes=False),
        # A few long contexts with capped scores.
        dict(name="paged_long_capped", op="paged", requests=3, page=64, longest=65536, shortest=30001, queries=1, heads=32, kv_heads=16,
             dim=128, type="bf16", cap=50.0, slopes=False),
        # Drafted tokens verified several at a time, one key head for each query head, bias by distance.
        dict(name="paged_drafts_slopes", op="paged", requests=16, page=16, longest=4096, shortest=17, queries=5, heads=16, kv_heads=16,
             dim=64, type="f16", cap=0.0, slopes=True),
        # A short packed prompt batch.
        dict(name="masked_short_documents", op="masked", batch=1, heads=8, kv_heads=8, rows=300, keys=300, dim=64, type="f16",
             causal=True, cap=0.0, slopes=False, documents=5, prefix=False, tokens_first=False),
        # Prompts of a model with capped scores and grouped heads, at the length of this repository's attention benchmark.
        dict(name="masked_capped", op="masked", batch=2, heads=32, kv_heads=8, rows=4096, keys=4096, dim=128, type="f16",
             causal=True, cap=50.0, slopes=False, documents=0, prefix=False, tokens_first=True),
        # Long packed documents with a bias by distance.
        dict(name="masked_documents_slopes", op="masked", batch=1, heads=32, kv_heads=32, rows=8192, keys=8192, dim=64, type="bf16",
             causal=True, cap=0.0, slopes=True, documents=11, prefix=False, tokens_first=False),
        # A prefix seen from everywhere, then text; a chunk of a prompt whose earlier keys are there already; odd sizes.
        dict(name="masked_prefix_chunk", op="masked", batch=4, heads=16, kv_heads=4, rows=1001, keys=2777, dim=128, type="bf16",
             causal=True, cap=0.0, slopes=False, documents=0, prefix=True, tokens_first=True),
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "append", "paged", "paged", "masked", "masked"])
    page = rng.choice([16, 32, 64, 128])
    kind = rng.choice(["f16", "bf16"])
    if op == "plan":
        requests = _spread(rng, 1, 1024)
        return dict(op=op, requests=requests, page=page, longest=_spread(rng, 64, 8192), prompt=rng.choice([1, _spread(rng, 2, 1024)]))
    if op == "append":
        requests, prompt = _spread(rng, 1, 256), rng.choice([1, _spread(rng, 2, 2600)])
        requests = max(1, min(requests, 60000 // prompt))
        return dict(op=op, requests=requests, page=page, longest=_spread(rng, 16, 1024), prompt=prompt,
                    kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), type=kind)
    if op == "paged":
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        longest = _spread(rng, 16, 32768)
        requests = max(1, min(_spread(rng, 1, 128), (1 << 21) // (longest * kv_heads)))
        return dict(op=op, requests=requests, page=page, longest=longest, shortest=rng.choice([1, longest, (longest + 1) // 2]),
                    queries=rng.choice([1, 1, 1, 2, 4, 7]), heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice([64, 128]),
                    type=kind, cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3)
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4])
    rows = _spread(rng, 1, 5000)
    heads = kv_heads * group
    dim = rng.choice([16, 32, 64, 64, 128, 128])
    rows = min(rows, math.isqrt(int(2e11) // (4 * dim * heads)))
    batch = max(1, min(rng.choice([1, 2, 3, 5]), (1 << 30) // (rows * rows * heads), int(2e11) // (4 * dim * heads * rows * rows)))
    kind_of = rng.choice(["plain", "documents", "documents", "prefix"])
    causal = kind_of == "prefix" or rng.random() < 0.7
    keys = rows if kind_of == "documents" or rng.random() < 0.6 else rows + rng.randrange(1, 700)
    return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, rows=rows, keys=keys, dim=dim,
                type=kind, causal=causal, cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.35,
                documents=rng.randrange(1, 16) if kind_of == "documents" else 0, prefix=kind_of == "prefix", tokens_first=rng.random() < 0.5)


# ---- sizes that follow from a case -----------------------------------------------------

def _requests(case):
    """(tokens in the cache, new tokens) of each request: part of the case, not of the seed."""
    rng = random.Random(case["requests"] * 7919 + case["longest"])
    if case["op"] == "paged":
        new = [case["queries"] if case["requests"] == 1 else rng.randrange(1, case["queries"] + 1) for _ in range(case["requests"])]
        whole = [max(n, rng.randrange(case["shortest"], case["longest"] + 1)) for n in new]
        whole[0] = max(new[0], case["longest"])
        return [w - n for w, n in zip(whole, new)], new
    if case["prompt"] == 1:
        return [rng.randrange(0, case["longest"]) for _ in range(case["requests"])], [1] * case["requests"]
    new = [1 if rng.random() < 0.25 else rng.randrange(1, case["prompt"] + 1) for _ in range(case["requests"])]
    new[0] = case["prompt"]
    return [rng.randrange(0, case["longest"]) if rng.random() < 0.5 else 0 for _ in range(case["requests"])], new


def _documents(case):
    """The lengths of the documents of each packed row; a last one is padding where it fits."""
    rng = random.Random(case["rows"] * 31 + case["documents"])
    rows = []
    for _ in range(case["batch"]):
        cuts = sorted(rng.randrange(0, case["rows"] + 1) for _ in range(case["documents"] - 1))
        rows.append([b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])])
    return rows


def _prefix(case):
    rng = random.Random(case["rows"] + 5 * case["keys"])
    return [rng.randrange(0, case["keys"] + 1) for _ in range(case["batch"])]


def _pages(n, page):
    return -(-n // page)


def _pairs(case):
    """Allowed (row, key) pairs of one head, over the batch."""
    rows, keys = case["rows"], case["keys"]
    if case["documents"]:
        return sum(n * (n + 1) // 2 if case["causal"] else n * n for lens in _documents(case) for n in lens)
    if not case["causal"]:
        return case["batch"] * rows * keys
    start = _prefix(case) if case["prefix"] else [0] * case["batch"]
    return sum(max(p, keys - rows + i + 1) for p in start for i in range(rows))


def work(case):
    op = case["op"]
    if op == "masked":
        d, b = case["dim"], case["batch"]
        size = 2 * d * b * (2 * case["heads"] * case["rows"] + 2 * case["kv_heads"] * case["keys"])
        return {"bytes": size, "flops": 4.0 * d * case["heads"] * _pairs(case)}
    old, new = _requests(case)
    total = sum(new)
    if op == "plan":
        added = sum(_pages(o + n, case["page"]) - _pages(o, case["page"]) for o, n in zip(old, new))
        return {"bytes": 4 * 4 * len(old) + 4 + 8 * added + 8 * total, "flops": 0}
    if op == "append":
        touched = sum(_pages(o + n, case["page"]) - o // case["page"] for o, n in zip(old, new))
        elements = 2 * total * case["kv_heads"] * case["dim"]
        return {"bytes": 3 * elements + 8 * total + 2 * 4 * touched * case["kv_heads"], "flops": 0}
    d = case["dim"]
    whole = [o + n for o, n in zip(old, new)]
    pairs = sum(n * o + n * (n + 1) // 2 for o, n in zip(old, new))
    pages = sum(_pages(w, case["page"]) for w in whole)
    size = 2 * d * case["kv_heads"] * sum(whole) + pages * (4 + 8 * case["kv_heads"]) + 4 * d * case["heads"] * total
    return {"bytes": size, "flops": 4.0 * d * case["heads"] * pairs}


# ---- inputs ----------------------------------------------------------------------------

def _ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device="cuda")


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s, not below 2^-100."""
    mantissa, exponent = torch.frexp(amax)
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    exponent = torch.where(amax > 0, exponent, LEAST).clamp(min=LEAST)
    return torch.ldexp(torch.ones_like(amax), exponent)


def _filled_cache(gen, n_pages, kv_heads, page, dim, spread):
    """A cache as earlier appends left it: values of ordinary size, and heads that differ in theirs."""
    x = torch.randn(n_pages, kv_heads, page, dim, generator=gen, device="cuda")
    x *= spread * torch.exp2(torch.randint(-2, 3, (1, kv_heads, 1, 1), generator=gen, device="cuda").float() * 0.5)
    scale = _scale_of(x.abs().amax((2, 3)))
    return (x / scale[:, :, None, None]).to(F8).view(torch.uint8), scale


def _table(gen, n_pages, counts, width):
    """A block table over pages in random order, and the pages that stay free."""
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = _ints(counts, torch.int64)
    col = torch.arange(width, device="cuda")[None]
    index = (at.cumsum(0) - at)[:, None] + col
    used = col < at[:, None]
    table = torch.where(used, order[index.clamp(max=n_pages - 1)], table)
    return table.contiguous(), order[sum(counts):].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    s = dict(case=case)
    if case["op"] == "masked":
        kind = TYPES[case["type"]]

        def tensor(heads, rows, spread):
            shape = (case["batch"], rows, heads, case["dim"]) if case["tokens_first"] else (case["batch"], heads, rows, case["dim"])
            x = (torch.randn(shape, generator=gen, device="cuda") * spread).to(kind)
            return x.transpose(1, 2) if case["tokens_first"] else x

        # Queries large enough that the cap is felt where there is one.
        s["q"] = tensor(case["heads"], case["rows"], 6.0 if case["cap"] else 1.5)
        s["k"] = tensor(case["kv_heads"], case["keys"], 1.0)
        s["v"] = tensor(case["kv_heads"], case["keys"], 1.0)
        s["scale"] = 1 / math.sqrt(case["dim"])
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"]).float() if case["slopes"] else None
        s["documents"] = _ints([[i for i, n in enumerate(lens) for _ in range(n)] for lens in _documents(case)]) if case["documents"] else None
        s["prefix"] = _ints(_prefix(case)) if case["prefix"] else None
        return s
    old, new = _requests(case)
    page = case["page"]
    s["cached"], s["new"] = _ints(old), _ints(new)
    s["total"] = sum(new)
    width = max(_pages(o + n, page) for o, n in zip(old, new)) + 1
    if case["op"] == "plan":
        counts = [_pages(o, page) for o in old]
        grown = sum(_pages(o + n, page) for o, n in zip(old, new))
        s["table"], s["free"] = _table(gen, grown + 5, counts, width)
        s["n_free"] = _ints([s["free"].numel()])
        return s
    counts = [_pages(o + n, page) for o, n in zip(old, new)]
    s["table"], _ = _table(gen, sum(counts) + 3, counts, width)
    s["k_cache"], s["k_scale"] = _filled_cache(gen, sum(counts) + 3, case["kv_heads"], page, case["dim"], 1.0)
    s["v_cache"], s["v_scale"] = _filled_cache(gen, sum(counts) + 3, case["kv_heads"], page, case["dim"], 0.7)
    ends = s["new"].long().cumsum(0)
    s["starts"] = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    if case["op"] == "append":
        at = torch.arange(s["total"], device="cuda")
        r = torch.searchsorted(ends, at, right=True)
        where = s["cached"].long()[r] + at - s["starts"].long()[r]
        s["slots"] = s["table"][r, where // page].long() * page + where % page
        shape = (s["total"], case["kv_heads"], case["dim"])
        # Now and then a token is larger than its page's earlier ones, and the page's scale has to grow.
        size = torch.exp2(torch.randn(s["total"], 1, 1, generator=gen, device="cuda"))
        s["k"] = (torch.randn(shape, generator=gen, device="cuda") * size).to(TYPES[case["type"]])
        s["v"] = (torch.randn(shape, generator=gen, device="cuda") * size).to(TYPES[case["type"]])
        return s
    s["lens"] = s["cached"] + s["new"]
    s["max_len"] = max(o + n for o, n in zip(old, new))
    s["max_new"] = max(new)
    shape = (s["total"], case["heads"], case["dim"])
    s["q"] = (torch.randn(shape, generator=gen, device="cuda") * (6.0 if case["cap"] else 1.5)).to(TYPES[case["type"]])
    s["scale"] = 1 / math.sqrt(case["dim"])
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"]).float() if case["slopes"] else None
    return s


# ---- one pass --------------------------------------------------------------------------

def _framework():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thunderkittens-sm7x_b200"))
    import tk_b200
    return tk_b200


def run(s):
    op = s["case"]["op"]
    if own:
        tk_b200 = sys.modules.get("tk_b200") or _framework()
        if op == "masked":
            return tk_b200.attention_masked(s["q"], s["k"], s["v"], scale=s["scale"], causal=s["case"]["causal"], softcap=s["case"]["cap"],
                                            alibi_slopes=s["slopes"], doc_ids=s["documents"], prefix_lens=s["prefix"])
        if op == "plan":
            lens, seq_lens, starts, slots, n_free = tk_b200.kv_plan(s["cached"], s["new"], s["table"], s["free"], s["n_free"],
                                                                    page_size=s["case"]["page"], max_tokens=s["total"])
            return {"lens": lens, "seq_lens": seq_lens, "starts": starts, "slots": slots, "n_free": n_free, "table": s["table"]}
        if op == "append":
            tk_b200.kv_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
            return {"k": s["k_cache"].view(F8), "v": s["v_cache"].view(F8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        return tk_b200.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["starts"],
                                       scale=s["scale"], softcap=s["case"]["cap"], alibi_slopes=s["slopes"], max_query_len=s["max_new"],
                                       max_seq_len=s["max_len"])
    return {"masked": _masked, "plan": _plan, "append": _append, "paged": _paged}[op](s)


def _softmax_weights(x):
    """exp(x - max) / sum over the last axis; a row of -inf gives zeros."""
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = x.sum(-1, keepdim=True)
    return x.div_(torch.where(total == 0, 1.0, total))


def _runs(ids):
    """The number of each position's run of equal ids; -1 where the id is negative."""
    edge = torch.zeros_like(ids)
    edge[:, 1:] = (ids[:, 1:] != ids[:, :-1]).to(ids.dtype)
    return torch.where(ids >= 0, edge.cumsum(1).to(ids.dtype), -1)


def _allowed(s, rows, keys):
    """[batch or 1, 1, 1, rows, keys] truth values."""
    at = torch.arange(rows, device="cuda")[:, None] + (keys - rows)
    key = torch.arange(keys, device="cuda")[None]
    allowed = (key <= at if s["case"]["causal"] else torch.ones(rows, keys, dtype=torch.bool, device="cuda"))[None]
    if s["prefix"] is not None:
        allowed = allowed | (key[None] < s["prefix"][:, None, None])
    if s["documents"] is not None:
        run_of = _runs(s["documents"])
        allowed = allowed & (run_of[:, :, None] == run_of[:, None, :]) & (run_of >= 0)[:, :, None]
    return allowed[:, None, None]


def _masked(s):
    q, k, v, cap = s["q"], s["k"], s["v"], s["case"]["cap"]
    b, h, rows, d = q.shape
    g, keys = k.shape[1], k.shape[2]
    x = torch.matmul(q.float().reshape(b, g, h // g, rows, d), k.float()[:, :, None].transpose(-1, -2)) * s["scale"]
    if cap:
        x = torch.tanh_(x.div_(cap)).mul_(cap)
    if s["slopes"] is not None:
        far = (torch.arange(rows, device="cuda")[:, None] + (keys - rows) - torch.arange(keys, device="cuda")[None]).abs().float()
        x -= s["slopes"].reshape(g, h // g, 1, 1) * far
    x.masked_fill_(~_allowed(s, rows, keys), -math.inf)
    return torch.matmul(_softmax_weights(x), v.float()[:, :, None]).reshape(b, h, rows, d).to(q.dtype)


def _plan(s):
    page, table, width = s["case"]["page"], s["table"], s["table"].shape[1]
    cached, new = s["cached"].long(), s["new"].long()
    whole, ends = cached + new, new.cumsum(0)
    fits = (new > 0) & (whole <= width * page) & (ends <= s["total"])
    have, want = (cached + page - 1) // page, (whole + page - 1) // page
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    n_free = s["n_free"].long()
    taken = fits & ((need == 0) | (upto <= n_free))
    lens, seq_lens = torch.where(taken, whole, cached), torch.where(taken, whole, 0)
    left = n_free - torch.where(taken & (need > 0), upto, 0).amax()
    col = torch.arange(width, device="cuda")[None]
    fresh = taken[:, None] & (col >= have[:, None]) & (col < want[:, None])
    index = n_free - 1 - ((upto - need)[:, None] + col - have[:, None])
    table.copy_(torch.where(fresh, s["free"][index.clamp(0, s["free"].numel() - 1)], table))
    at = torch.arange(s["total"], device="cuda")
    r = torch.searchsorted(ends, at, right=True).clamp(max=cached.numel() - 1)
    where = cached[r] + at - (ends - new)[r]
    owner = table[r, (where // page).clamp(max=width - 1)].long()
    slots = torch.where(taken[r] & (at < ends[-1]) & (owner >= 0), owner * page + where % page, -1)
    starts = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return {"lens": lens.to(torch.int32), "seq_lens": seq_lens.to(torch.int32), "starts": starts, "slots": slots,
            "n_free": left.to(torch.int32), "table": table}


def _append_one(x, slots, cache, scale):
    n_pages, heads, page, dim = cache.shape
    x, owner, at = x.float(), slots // page, slots % page
    amax = torch.zeros_like(scale).scatter_reduce_(0, owner[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    first = torch.full((n_pages,), page, device="cuda").scatter_reduce_(0, owner, at, "amin")
    old = torch.where((first > 0)[:, None], scale, 0.0)
    now = torch.where((first < page)[:, None], torch.maximum(old, _scale_of(amax)), scale)
    # The tokens that a page already holds move to its new scale.
    lead = owner[torch.cat([owner.new_ones(1, dtype=torch.bool), owner[1:] != owner[:-1]])]
    held = cache[lead].view(F8).float() * (scale[lead] / now[lead])[:, :, None, None]
    kept = torch.arange(page, device="cuda")[None] < first[lead][:, None]
    cache[lead] = torch.where(kept[:, None, :, None], held.to(F8).view(torch.uint8), cache[lead])
    cache[owner, :, at] = (x / now[owner][:, :, None]).to(F8).view(torch.uint8)
    scale.copy_(now)


def _append(s):
    _append_one(s["k"], s["slots"], s["k_cache"], s["k_scale"])
    _append_one(s["v"], s["slots"], s["v_cache"], s["v_scale"])
    return {"k": s["k_cache"].view(F8), "v": s["v_cache"].view(F8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gathered(cache, scale, table, pages):
    """[requests, heads, tokens, dim] in 32 bits."""
    owner = table[:, :pages].long().clamp(min=0)
    x = cache[owner].view(F8).float() * scale[owner][..., None, None]
    r, n, h, p, d = x.shape
    return x.transpose(1, 2).reshape(r, h, n * p, d)


def _paged(s):
    q, cap, page, most = s["q"], s["case"]["cap"], s["case"]["page"], s["max_new"]
    pages = _pages(s["max_len"], page)
    k, v = _gathered(s["k_cache"], s["k_scale"], s["table"], pages), _gathered(s["v_cache"], s["v_scale"], s["table"], pages)
    r, g, keys, d = k.shape
    h = q.shape[1]
    lens, starts = s["lens"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    step = torch.arange(most, device="cuda")[None]
    x = q.float()[(starts[:-1, None] + step).clamp(max=q.shape[0] - 1)]                  # [r, most, h, d]
    x = x.reshape(r, most, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(r, g, -1, d)
    x = (torch.matmul(x, k.transpose(-1, -2)) * s["scale"]).reshape(r, g, h // g, most, keys)
    at = (lens - new)[:, None] + step                                                    # [r, most]
    key = torch.arange(keys, device="cuda")
    if cap:
        x = torch.tanh(x / cap) * cap
    if s["slopes"] is not None:
        x -= s["slopes"].reshape(1, g, h // g, 1, 1) * (at[:, :, None] - key).abs().float()[:, None, None]
    x.masked_fill_((key > at[:, :, None])[:, None, None], -math.inf)
    y = torch.matmul(_softmax_weights(x).reshape(r, g, -1, keys), v).reshape(r, g, h // g, most, d)
    y = y.permute(0, 3, 1, 2, 4).reshape(r, most, h, d)
    token = torch.arange(q.shape[0], device="cuda")
    owner = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    return y[owner, token - starts[owner]].to(q.dtype)


# ---- the definitions in 64 bits ---------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"masked": _exact_masked, "plan": _exact_plan, "append": _exact_append, "paged": _exact_paged}[case["op"]](s, case)


def _exact_row(x, allowed, v):
    x = torch.where(allowed, x, -math.inf)
    some = allowed.any(-1, keepdim=True)
    w = torch.softmax(torch.where(some, x, 0.0), -1) * some
    return w @ v


def _exact_score(q, k, scale, cap, slope, at, key):
    x = (q @ k.T) * scale
    if cap:
        x = cap * torch.tanh(x / cap)
    if slope is not None:
        x = x - slope.double() * (at[:, None] - key[None]).abs().double()
    return x


def _exact_masked(s, case):
    rows, keys = case["rows"], case["keys"]
    key = torch.arange(keys, device="cuda")
    at = torch.arange(rows, device="cuda") + keys - rows
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        allowed = key[None] <= at[:, None] if case["causal"] else torch.ones(rows, keys, dtype=torch.bool, device="cuda")
        if case["prefix"]:
            allowed = allowed | (key < s["prefix"][b])[None]
        if case["documents"]:
            number = torch.repeat_interleave(torch.arange(case["documents"], device="cuda"), _ints(_documents(case)[b]))
            allowed = allowed & (number[:, None] == number[None])
        for h in range(case["heads"]):
            g = h * case["kv_heads"] // case["heads"]
            x = _exact_score(s["q"][b, h].double(), s["k"][b, g].double(), s["scale"], case["cap"], s["slopes"][h] if case["slopes"] else None, at, key)
            out[b, h] = _exact_row(x, allowed, s["v"][b, g].double())
    return out


def _exact_paged(s, case):
    old, new = _requests(case)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for r, (o, n) in enumerate(zip(old, new)):
        key = torch.arange(o + n, device="cuda")
        at = torch.arange(o, o + n, device="cuda")
        owner, inside = s["table"][r].long()[key // case["page"]], key % case["page"]
        k = s["k_cache"][owner, :, inside].view(F8).double() * s["k_scale"][owner].double()[..., None]
        v = s["v_cache"][owner, :, inside].view(F8).double() * s["v_scale"][owner].double()[..., None]
        for h in range(case["heads"]):
            g = h * case["kv_heads"] // case["heads"]
            x = _exact_score(s["q"][first:first + n, h].double(), k[:, g], s["scale"], case["cap"], s["slopes"][h] if case["slopes"] else None, at, key)
            out[first:first + n, h] = _exact_row(x, key[None] <= at[:, None], v[:, g])
        first += n
    return out


def _exact_plan(s, case):
    return None  # whole numbers


def _exact_e4m3(x):
    """The nearest value of e4m3, ties to the even one: steps of 2^(e-3), none below 2^-9."""
    exponent = (torch.frexp(x.abs())[1] - 1).clamp(min=-6).double()
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _exact_append(s, case):
    page = case["page"]
    old, new = _requests(case)
    out = {}
    for name in ("k", "v"):
        values, scale = s[name + "_cache"].view(F8).double(), s[name + "_scale"].double()
        x, first = s[name].double(), 0
        for r, (o, n) in enumerate(zip(old, new)):
            for p in range(o // page, _pages(o + n, page)):
                a, b = max(o, p * page), min(o + n, (p + 1) * page)
                owner = s["slots"][first + a - o] // page
                part = x[first + a - o:first + b - o].transpose(0, 1)       # [heads, tokens, dim]
                wanted = part.abs().amax((1, 2)) / TOP
                half, power = torch.frexp(wanted)                            # wanted = half 2^power, 1/2 <= half < 1
                power = torch.where(wanted > 0, power - (half == 0.5).to(power.dtype), LEAST)
                now = torch.ldexp(torch.ones_like(wanted), power.clamp(min=LEAST))
                if a > p * page:
                    now = torch.maximum(now, scale[owner])
                    held = values[owner, :, :a - p * page]
                    values[owner, :, :a - p * page] = _exact_e4m3(held * (scale[owner] / now)[:, None, None])
                values[owner, :, a - p * page:b - p * page] = _exact_e4m3(part / now[:, None, None])
                scale[owner] = now
            first += n
        out[name], out[name + "_scale"] = values, scale
    return out
