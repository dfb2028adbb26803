"""Performance cases of the attention side of a serving step: block tables, batch layout and attention over the paged KV cache.

Four kinds of work, each through the entry point that a serving program calls:

``tables``  ``kv_cache_ops.resize_block_tables``: the requests of a step get the cache pages that their new length needs from a
            stack of free pages, finished ones give theirs back.
``layout``  ``kv_cache_ops.batch_layout``: from the lengths and block tables of a step the index arrays that its kernels read:
            row offsets, page lists, the request, position and cache slot of every token.
``attn``    ``attention_ops.paged_attention``: causal attention of a step's new tokens (prompt chunks and single decoded tokens
            in one batch) over the paged cache, for one layer.  The plan is made once a step and used by all of its layers, so it
            is part of what the program has in hand.
``step``    what a step does before its first layer and in it: layout, plan, append of its keys and values, attention.

Plain forms are elementary torch operations in 32 bits; ``exact`` is the definition in 64.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PAGE = 16  # tokens per page in the benchmark configurations

# q heads, kv heads, head size: the layer shapes of the benchmark, one rank of eight of the larger one, the small fp32 layer
SHAPES = {
    "llama3-8b": (32, 8, 128),
    "llama3-70b-tp8": (8, 1, 128),
    "small": (16, 4, 64),
}


def listed():
    return [
        # a decode-only step of 128 running requests (the scheduler's default limit): a few of them start a page
        {"name": "tables_decode_128", "kind": "tables", "requests": 128, "arrive": 0, "finish": 0, "max_len": 8192, "page": 16},
        # the largest: prompts arrive and requests finish among 512, so that tens of thousands of pages change hands
        {"name": "tables_mixed_512", "kind": "tables", "requests": 512, "arrive": 40, "finish": 33, "max_len": 32768, "page": 16},
        # index arrays of a decode-only step with an odd number of requests, padded to 64 tokens
        {"name": "layout_decode_61", "kind": "layout", "chunks": 0, "chunk": 0, "decodes": 61, "max_len": 8192, "page": 16},
        # the largest scheduler budget, not quite full: three prompt chunks and 209 decodes
        {"name": "layout_mixed_1999", "kind": "layout", "chunks": 3, "chunk": 596, "decodes": 209, "max_len": 32768, "page": 16},
        # a lightly loaded server: eight decoding requests, latency counts
        {"name": "attn_decode_8", "kind": "attn", "shape": "llama3-8b", "dtype": "bf16", "chunks": 0, "chunk": 0, "start": 0,
         "decodes": 8, "min_len": 200, "max_len": 2048, "page": 16, "window": 0},
        # a loaded one: 209 decoding requests with contexts up to the model's 8192 positions
        {"name": "attn_decode_209", "kind": "attn", "shape": "llama3-8b", "dtype": "bf16", "chunks": 0, "chunk": 0, "start": 0,
         "decodes": 209, "min_len": 512, "max_len": 8192, "page": 16, "window": 0},
        # the mixed chunk of the headline benchmark: 448 prompt tokens behind 1024 earlier ones, and 64 decodes
        {"name": "attn_mixed_512", "kind": "attn", "shape": "llama3-8b", "dtype": "bf16", "chunks": 1, "chunk": 448, "start": 1024,
         "decodes": 64, "min_len": 512, "max_len": 8192, "page": 16, "window": 0},
        # a chunk of the largest budget, far into a long prompt: the tensor cores' case
        {"name": "attn_chunk_1999_long", "kind": "attn", "shape": "llama3-8b", "dtype": "bf16", "chunks": 1, "chunk": 1999,
         "start": 29001, "decodes": 0, "min_len": 0, "max_len": 0, "page": 16, "window": 0},
        # one of eight ranks of the 70B-shaped layer on its chunk of 1792 prompt tokens (two prompts) and 256 decodes, fp16
        {"name": "attn_70b_tp8_2048", "kind": "attn", "shape": "llama3-70b-tp8", "dtype": "fp16", "chunks": 2, "chunk": 896,
         "start": 511, "decodes": 256, "min_len": 2048, "max_len": 8192, "page": 16, "window": 0},
        # heads of 64, pages of 24 tokens (no power of two), a sliding window and ragged prompts
        {"name": "attn_window_fp16", "kind": "attn", "shape": "small", "dtype": "fp16", "chunks": 3, "chunk": 333, "start": 1500,
         "decodes": 37, "min_len": 1, "max_len": 4097, "page": 24, "window": 1000},
        # the fp32 parity configuration: 256 prompt tokens and 32 decodes of a small layer
        {"name": "attn_fp32_288", "kind": "attn", "shape": "small", "dtype": "fp32", "chunks": 1, "chunk": 256, "start": 0,
         "decodes": 32, "min_len": 256, "max_len": 2048, "page": 16, "window": 0},
        # layout, plan, append and attention of one layer for a ragged mixed batch
        {"name": "step_mixed_300", "kind": "step", "shape": "llama3-8b", "dtype": "bf16", "chunks": 2, "chunk": 131, "start": 640,
         "decodes": 38, "min_len": 100, "max_len": 2048, "page": 16, "window": 0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "layout", "attn", "attn", "attn", "attn", "step", "step"])
    if kind == "tables":
        requests = _log_int(rng, 1, 512)
        return {"kind": kind, "requests": requests, "arrive": rng.randint(0, requests // 8), "finish": rng.randint(0, requests // 8),
                "max_len": _log_int(rng, 256, 32768), "page": rng.choice([8, 16, 16, 24, 32, 64])}
    chunks = rng.choice([0, 1, 1, 2, 3])
    chunk = _log_int(rng, 2, 2048) // max(1, chunks) if chunks else 0
    decodes = _log_int(rng, 1, 209) if not chunks or rng.random() < 0.7 else 0
    if kind == "layout":
        return {"kind": kind, "chunks": chunks, "chunk": max(chunk, 1) if chunks else 0, "decodes": decodes,
                "max_len": _log_int(rng, 256, 32768), "page": rng.choice([8, 16, 16, 24, 32, 64])}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    shape = "small" if dtype == "fp32" else rng.choice(["llama3-8b", "llama3-8b", "llama3-70b-tp8", "small"])
    max_len = _log_int(rng, 16, 2048 if dtype == "fp32" else 8192)
    if dtype == "fp32":
        chunk, decodes = min(chunk, 256), min(decodes, 64)
    if kind == "step":
        max_len, decodes = min(max_len, 2048), min(decodes, 64)
    return {"kind": kind, "shape": shape, "dtype": dtype, "chunks": chunks, "chunk": max(chunk, 1) if chunks else 0,
            "start": rng.choice([0, rng.randint(1, max_len)]) if chunks else 0, "decodes": decodes, "min_len": rng.randint(1, max_len // 8),
            "max_len": max_len, "page": rng.choice([8, 16, 16, 16, 24, 32, 64, 128]), "window": rng.choice([0, 0, 0, 100, 1000])}


# ------------------------------------------------------------------ inputs
def _lengths(case, gen):
    """Per request: new tokens of this step and tokens that were cached before it (host lists, made from the case and seed)."""
    query, context = [], []
    for i in range(case["chunks"]):
        query.append(case["chunk"] - (i * 7) % max(1, case["chunk"] // 4))  # ragged
        context.append(case.get("start", 0) * (case["chunks"] - i) // max(1, case["chunks"]))
    for _ in range(case["decodes"]):
        query.append(1)
        lo, hi = case.get("min_len", 1), case["max_len"]
        context.append(int(gen.integers(min(lo, hi), hi + 1)) - 1)
    return query, [max(0, c) for c in context]


def _table(lens, page, gen, width, pool=None):
    """Block tables of requests with these lengths: pages in shuffled order from a pool (a little larger than they need)."""
    need = [-(-n // page) for n in lens]
    pool = pool or sum(need) + 5
    order = gen.permutation(pool)
    table = np.full((len(lens), width), -1, dtype=np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, pool, order[at:]


def _gpu(a, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a), dtype=dtype).cuda()


def prepare(case, seed):
    gen = np.random.default_rng(seed)
    if case["kind"] == "tables":
        n, page = case["requests"], case["page"]
        width = -(-(case["max_len"] + 1) // page)
        now = gen.integers(1, case["max_len"] + 1, n)
        lens = now + 1                                     # every running request appends a token
        which = gen.permutation(n)
        now[which[:case["arrive"]]] = 0                    # prompts that arrive have no pages yet
        lens[which[n - case["finish"]:]] = 0               # requests that have finished keep none
        table, pool, free = _table(now.tolist(), page, gen, width, n * width)
        stack = np.concatenate([free, np.full(pool - len(free), -1)])
        parts = [table.ravel(), -(-now // page), stack, np.array([len(free)])]
        given = _gpu(np.concatenate(parts))
        work = torch.empty_like(given)
        ends = np.cumsum([len(p) for p in parts]).tolist()
        views = [work[a:b] for a, b in zip([0] + ends[:-1], ends)]
        return {"kind": "tables", "given": given, "work": work, "tables": views[0].view(n, width), "num_blocks": views[1],
                "free": views[2], "num_free": views[3], "lens": _gpu(lens), "page": page}
    query, context = _lengths(case, gen)
    page = case["page"]
    width = -(-max(case["max_len"], case["chunk"] + case.get("start", 0)) // page)
    pool = len(query) * width + 5 if case["kind"] == "step" else None  # (the whole cache is an output there)
    table, pool, _ = _table([q + c for q, c in zip(query, context)], page, gen, width, pool)
    total = sum(query)
    s = {"kind": case["kind"], "query": _gpu(query), "context": _gpu(context), "table": _gpu(table), "page": page, "pages": pool,
         "tokens": -(-total // 8) * 8}                     # batches are padded to a multiple of eight tokens
    if case["kind"] == "layout":
        return s
    nq, nkv, hd = SHAPES[case["shape"]]
    dtype = DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    # the fused qkv rows of the step: q is a view of them, as a layer hands it over; queries are spread so that the scores are
    qkv = torch.randn(s["tokens"], (nq + 2 * nkv) * hd, generator=g, device="cuda", dtype=torch.float32)
    qkv[:, :nq * hd] *= 1.5
    qkv = qkv.to(dtype)
    cache = torch.empty(pool, 2, page, nkv, hd, dtype=dtype, device="cuda")
    for lo in range(0, pool, 4096):
        part = cache[lo:lo + 4096]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float32))
    s.update(q=qkv[:, :nq * hd], k=qkv[:, nq * hd:(nq + nkv) * hd], v=qkv[:, (nq + nkv) * hd:], cache=cache, nq=nq, nkv=nkv, hd=hd,
             scale=hd ** -0.5, window=case["window"], query_list=query, context_list=context)
    if own:  # what a program keeps: the index arrays of the step and the plan made from them, for all of its layers
        from sarathi_serve_b200 import attention_ops, kv_cache_ops
        s["plan"] = attention_ops.AttentionPlan(nq, nkv, hd, page, dtype, max_requests=len(query), max_tokens=s["tokens"],
                                                window=case["window"])
        s["layout"] = kv_cache_ops.batch_layout(s["query"], s["context"], s["table"], page, pool, s["tokens"])
        s["plan"].update(s["layout"])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if s["kind"] == "tables":
        s["work"].copy_(s["given"])  # the call works in place: every pass starts from the same tables
    if own:
        from sarathi_serve_b200 import attention_ops, kv_cache_ops
        if s["kind"] == "tables":
            granted = kv_cache_ops.resize_block_tables(s["tables"], s["num_blocks"], s["lens"], s["free"], s["num_free"], s["page"])
            return [s["tables"], s["num_blocks"], s["free"], s["num_free"], granted]
        if s["kind"] == "layout":
            return list(kv_cache_ops.batch_layout(s["query"], s["context"], s["table"], s["page"], s["pages"], s["tokens"]))
        if s["kind"] == "attn":
            return attention_ops.paged_attention(s["q"], s["cache"], s["plan"], s["scale"])
        layout = kv_cache_ops.batch_layout(s["query"], s["context"], s["table"], s["page"], s["pages"], s["tokens"], out=s["layout"])
        s["plan"].update(layout)
        kv_cache_ops.append_rows(s["cache"], s["k"], s["v"], layout.kv_slots)
        out = attention_ops.paged_attention(s["q"], s["cache"], s["plan"], s["scale"])
        return [out, s["cache"]]
    if s["kind"] == "tables":
        return _plain_tables(s)
    layout = _plain_layout(s["query"], s["context"], s["table"], s["page"], s["pages"], s["tokens"]) if s["kind"] != "attn" else None
    if s["kind"] == "layout":
        return layout
    if s["kind"] == "step":
        slots = layout[7]
        put = slots >= 0
        rows = s["cache"].view(-1, s["nkv"] * s["hd"])
        rows[slots[put]] = s["k"][put]
        rows[slots[put] + s["page"]] = s["v"][put]
        return [_plain_attention(s), s["cache"]]
    return _plain_attention(s)


def _plain_tables(s):
    table, have, free, count, page = s["tables"], s["num_blocks"], s["free"], s["num_free"], s["page"]
    n, width = table.shape
    want = (s["lens"] + page - 1) // page
    back = (have - want).clamp(min=0)
    need = torch.where(want <= width, (want - have).clamp(min=0), 0)
    column = torch.arange(width, device=table.device)
    # pages given back go on the stack, request by request
    gone = (column >= want[:, None]) & (column < have[:, None])
    pages = table[gone]
    free[count + torch.arange(pages.numel(), device=table.device)] = pages
    avail = count + pages.numel()
    # and are taken from its top
    fits = (need.cumsum(0) <= avail) & (want <= width)
    need = torch.where(fits, need, 0)
    first = need.cumsum(0) - need
    new = (column >= have[:, None]) & (column < (have + need)[:, None])
    at = avail - 1 - (first[:, None] + column - have[:, None])
    table[new] = free[at[new].long()]
    have.copy_(torch.where(fits, want, have))
    count.copy_(avail - need.sum())
    return [table, have, free, count, fits.int()]


def _plain_layout(query, context, table, page, num_pages, tokens):
    n, width = table.shape
    ends = query.cumsum(0)
    kv = query + context
    pages = (kv + page - 1) // page
    zero = torch.zeros(1, dtype=torch.int64, device=query.device)
    qo_indptr = torch.cat([zero, ends])
    kv_indptr = torch.cat([zero, pages.cumsum(0)])
    kv_indices = torch.full((n * width,), -1, dtype=torch.int32, device=query.device)
    column = torch.arange(width, device=query.device)
    used = column < pages[:, None]
    kv_indices[(kv_indptr[:-1, None] + column)[used]] = table[used]
    last = torch.where(kv > 0, kv - (pages - 1) * page, 0)
    t = torch.arange(tokens, device=query.device)
    req = torch.searchsorted(ends, t, right=True)
    real = req < n
    req = req.clamp(max=n - 1)
    pos = torch.where(real, context[req] + t - qo_indptr[req], 0)
    block = table[req, pos // page].long()
    real_slot = real & (block >= 0) & (block < num_pages)
    slots = torch.where(real_slot, block * (2 * page) + pos % page, -1)
    return [qo_indptr.int(), kv.int(), kv_indptr.int(), kv_indices, last.int(), torch.where(real, req, -1).int(), pos.long(), slots]


def _plain_attention(s):
    q, cache, nq, nkv, hd, page = s["q"], s["cache"], s["nq"], s["nkv"], s["hd"], s["page"]
    group = nq // nkv
    out = torch.zeros(q.shape[0], nq * hd, dtype=q.dtype, device=q.device)
    row = 0
    for r, (new, before) in enumerate(zip(s["query_list"], s["context_list"])):
        length = new + before
        blocks = s["table"][r, :-(-length // page)].long()
        kv = cache[blocks].float()                                             # [blocks, 2, page, nkv, hd]
        k = kv[:, 0].reshape(-1, nkv, hd)[:length].permute(1, 2, 0)            # [nkv, hd, length]
        v = kv[:, 1].reshape(-1, nkv, hd)[:length].permute(1, 0, 2)            # [nkv, length, hd]
        x = q[row:row + new].float().reshape(new, nkv, group, hd).permute(1, 2, 0, 3).reshape(nkv, group * new, hd)
        scores = torch.matmul(x, k).view(nkv, group, new, length) * s["scale"]
        at = before + torch.arange(new, device=q.device)[:, None]
        key = torch.arange(length, device=q.device)
        hidden = key > at
        if s["window"]:
            hidden = hidden | (key <= at - s["window"])
        scores.masked_fill_(hidden, float("-inf"))
        scores -= scores.amax(-1, keepdim=True)
        p = scores.exp_()
        p /= p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(nkv, group * new, length), v).view(nkv, group, new, hd)
        out[row:row + new] = o.permute(2, 0, 1, 3).reshape(new, nq * hd).to(q.dtype)
        row += new
    return out


def _visible(case, query, context):
    """Sum over the new tokens of the keys each of them sees, and over the requests of the keys that any of them sees."""
    window = case["window"]
    pairs = keys = 0
    for new, before in zip(query, context):
        if not window or new + before <= window:
            pairs += new * before + new * (new + 1) // 2
            keys += new + before
        else:
            pairs += sum(min(window, before + i + 1) for i in range(new))
            keys += min(new + before, window + new - 1)
    return pairs, keys


def work(case):
    gen = np.random.default_rng(0)
    if case["kind"] == "tables":
        n, page = case["requests"], case["page"]
        arriving = case["arrive"] * (case["max_len"] / 2 / page)
        finishing = case["finish"] * (case["max_len"] / 2 / page)
        return {"bytes": int(4 * (4 * n + 2) + 8 * (arriving + finishing + n / page)), "flops": 0}
    query, context = _lengths(case, gen)
    total, n, page = sum(query), len(query), case["page"]
    pages = sum(-(-(q + c) // page) for q, c in zip(query, context))
    layout = 4 * 2 * n + 4 * 4 * (n + 1) + 8 * pages + 20 * total
    if case["kind"] == "layout":
        return {"bytes": layout, "flops": 0}
    nq, nkv, hd = SHAPES[case["shape"]]
    es = 4 if case["dtype"] == "fp32" else 2
    pairs, keys = _visible(case, query, context)
    moved = es * hd * (2 * nq * total + 2 * nkv * keys) + 4 * pages
    if case["kind"] == "step":
        moved += layout + 4 * es * hd * nkv * total
    return {"bytes": moved, "flops": 4 * pairs * nq * hd}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        given = s["given"].cpu().numpy().copy()
        n, width = s["tables"].shape
        table = given[:n * width].reshape(n, width)
        have = given[n * width:n * width + n]
        free = given[n * width + n:-1]
        count, page = int(given[-1]), s["page"]
        lens = s["lens"].cpu().numpy()
        want = [-(-int(x) // page) for x in lens]
        for r in range(n):
            for j in range(want[r], int(have[r])):
                free[count] = table[r, j]
                count += 1
        granted = np.ones(n, np.int32)
        for r in range(n):
            need = max(0, want[r] - int(have[r]))
            if want[r] > width:
                granted[r] = 0
                continue
            if need > count:  # the rest of those that grow gets nothing either
                granted[r:] = [0 if want[i] > have[i] else 1 for i in range(r, n)]
                break
            for j in range(need):
                count -= 1
                table[r, have[r] + j] = free[count]
        for r in range(n):
            if granted[r]:
                have[r] = want[r]
        return [table, have, free, np.array([count], np.int32), granted]
    query, context = s["query"].tolist(), s["context"].tolist()
    table, page, tokens = s["table"].cpu().numpy(), s["page"], s["tokens"]
    if case["kind"] in ("layout", "step"):
        qo, kv, indptr, last = [0], [], [0], []
        indices, req, pos, slots = [], [], [], []
        for r, (a, b) in enumerate(zip(query, context)):
            blocks = -(-(a + b) // page)
            qo.append(qo[-1] + a)
            kv.append(a + b)
            indptr.append(indptr[-1] + blocks)
            indices += table[r, :blocks].tolist()
            last.append(a + b - (blocks - 1) * page if a + b else 0)
            for p in range(b, b + a):
                req.append(r)
                pos.append(p)
                slots.append(int(table[r, p // page]) * 2 * page + p % page)
        pad = tokens - len(req)
        indices += [-1] * (table.size - len(indices))
        layout = [np.array(x, t) for x, t in ((qo, np.int32), (kv, np.int32), (indptr, np.int32), (indices, np.int32), (last, np.int32),
                                              (req + [-1] * pad, np.int32), (pos + [0] * pad, np.int64), (slots + [-1] * pad, np.int64))]
        if case["kind"] == "layout":
            return layout
        rows = s["cache"].view(-1, s["nkv"], s["hd"])
        for t, slot in enumerate(slots):
            rows[slot] = s["k"][t].view(s["nkv"], s["hd"])
            rows[slot + page] = s["v"][t].view(s["nkv"], s["hd"])
    nq, nkv, hd, window = s["nq"], s["nkv"], s["hd"], s["window"]
    out = torch.zeros(tokens, nq, hd, dtype=torch.float64, device="cuda")
    t = 0
    for r, (a, b) in enumerate(zip(query, context)):
        where = torch.tensor([int(table[r, j // page]) * 2 * page + j % page for j in range(a + b)], device="cuda")
        flat = s["cache"].view(-1, nkv, hd)
        keys, values = flat[where].double(), flat[where + page].double()
        for lo in range(0, a, 256):
            hi = min(a, lo + 256)
            x = s["q"][t + lo:t + hi].double().view(hi - lo, nq, hd)
            i = b + torch.arange(lo, hi, device="cuda").view(-1, 1)
            j = torch.arange(a + b, device="cuda").view(1, -1)
            seen = (j <= i) if not window else (j <= i) & (j > i - window)
            for h in range(nq):
                e = (x[:, h] @ keys[:, h // (nq // nkv)].T) / math.sqrt(hd)
                w = torch.softmax(torch.where(seen, e, torch.full_like(e, -math.inf)), dim=-1)
                out[t + lo:t + hi, h] = w @ values[:, h // (nq // nkv)]
        t += a
    out = out.view(tokens, nq * hd)
    return [out, s["cache"].double()] if case["kind"] == "step" else out
