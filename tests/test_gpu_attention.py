"""Attention over the paged KV cache, block tables and batch layout on the GPU, against plain implementations in 64 bits.

Tolerances (u(t) = eps(t) / 2, the most that one rounding is off, relative to the value):
  * the result is rounded once:                        u(dtype) |o|
  * fp16 / bf16 round the probabilities once:          u(dtype) W,  W = sum_j p_j |v_j|
  * a score is off by at most (hd + 16) 2^-24 A, A = scale max_j sum_i |q_i k_ji| (fp32 products summed in any order, scaling,
    the subtraction of the maximum), the power of two by 2^-21 relative (two units of its approximation); that moves numerator
    and denominator alike:                             2 ((hd + 16) 2^-24 A + 2^-21) W
  * fp32 sums over n keys, twice (numerator, denominator), and a join:  2 (n + 16) 2^-24 W
  * fp16 probabilities below its smallest step:        n 2^-25 max|v|   (the sum they are divided by is at least 1)
Nothing is compared where a result is not finite; non-finite results are expected exactly where 64 bits have them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(seed, dtype, heads, kv_heads, hd, page, batch, spread=1.5, pad=0, extra_pages=3, width=None, cache_fill=float("nan")):
    """A step of requests (new tokens, cached tokens): lengths, shuffled block tables and a cache whose slots behind the
    requests' tokens, and whose unused pages, hold ``cache_fill``."""
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in batch]
    need = [-(-n // page) for n in lens]
    pool = sum(need) + extra_pages
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    width = width or max([1] + need)
    table = torch.full((len(batch), width), -7, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    cache = torch.full((pool, 2, page, kv_heads, hd), cache_fill, dtype=dtype)
    for r, n in enumerate(lens):
        for b in range(need[r]):
            k = min(page, n - b * page)
            cache[table[r, b], :, :k] = torch.randn(2, k, kv_heads, hd, generator=g).to(dtype)
    total = sum(a for a, _ in batch)
    T = total + pad
    qkv = (torch.randn(T, (heads + 2 * kv_heads) * hd, generator=g) * spread).to(dtype)
    return dict(q=qkv.cuda()[:, :heads * hd], cache=cache.cuda(), table=table.cuda(), total=total, T=T, batch=batch, heads=heads,
                kv_heads=kv_heads, hd=hd, page=page, pool=pool, dtype=dtype,
                query=torch.tensor([a for a, _ in batch], dtype=torch.int32).cuda(),
                context=torch.tensor([b for _, b in batch], dtype=torch.int32).cuda())


def plan_of(c, window=0, max_requests=None, max_tokens=None):
    from sarathi_serve_b200 import attention_ops, kv_cache_ops
    layout = kv_cache_ops.batch_layout(c["query"], c["context"], c["table"], c["page"], c["pool"], c["T"])
    plan = attention_ops.AttentionPlan(c["heads"], c["kv_heads"], c["hd"], c["page"], c["dtype"], max_requests or len(c["batch"]),
                                       max_tokens or c["T"], window=window)
    return plan.update(layout), layout


def reference(c, scale, window=0):
    """(o, lse, tolerance) in 64 bits for the rows that belong to a request."""
    heads, kvh, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    group = heads // kvh
    dev = c["q"].device
    o = torch.zeros(c["total"], heads, hd, dtype=torch.float64, device=dev)
    lse = torch.full((c["total"], heads), -math.inf, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(o)
    u = half_step(c["dtype"])
    row = 0
    for r, (new, before) in enumerate(c["batch"]):
        n = new + before
        if new and n:
            where = torch.arange(n, device=dev)
            pages = c["table"][r].long()[where // page]
            k, v = (c["cache"][pages, i, where % page].double() for i in (0, 1))   # [n, kvh, hd]
            for lo in range(0, new, 512):
                hi = min(new, lo + 512)
                q = c["q"][row + lo:row + hi].double().view(hi - lo, heads, hd)
                pos = before + torch.arange(lo, hi, device=dev)[:, None]
                seen = where[None] <= pos
                if window:
                    seen = seen & (where[None] > pos - window)
                for h in range(heads):
                    kh, vh = k[:, h // group], v[:, h // group]
                    s = (q[:, h] @ kh.T * scale).masked_fill(~seen, -math.inf)
                    l = torch.logsumexp(s, 1)
                    p = torch.exp(s - l[:, None]).masked_fill(~seen, 0)
                    vz = torch.where(seen.any(0)[:, None], vh, 0)
                    # keys that a row does not see contribute nothing, whatever they hold
                    bad = ~torch.isfinite(vz)
                    res = p @ torch.where(bad, 0, vz)
                    if bad.any():
                        res = torch.where((seen.double() @ bad.double()) > 0, torch.nan, res)
                    va = torch.where(bad, 0, vz).abs()
                    W = p @ va
                    A = (q[:, h].abs() @ torch.where(torch.isfinite(kh), kh, 0).abs().T * abs(scale)).amax(1)
                    delta = (hd + 16) * 2.0 ** -24 * A + 2.0 ** -21
                    t = u * res.abs() + (2 * delta[:, None] + 2 * (n + 16) * 2.0 ** -24) * W
                    if c["dtype"] != torch.float32:
                        t = t + u * W
                    if c["dtype"] == torch.float16:
                        t = t + n * 2.0 ** -25 * va.amax() + 2.0 ** -25
                    o[row + lo:row + hi, h], lse[row + lo:row + hi, h], tol[row + lo:row + hi, h] = res, l, t
        row += new
    return o.view(c["total"], heads * hd), lse, tol.view(c["total"], heads * hd)


def check(c, out, scale, window=0, lse=None):
    want, l, tol = reference(c, scale, window)
    got = out[:c["total"]].double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), "finite results in other places"
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{((got - want).abs() / tol.clamp(min=1e-300))[fine].max().item():.2f} times the tolerance"
    if lse is not None:
        g = lse[:c["total"]].double()
        none = l == -math.inf
        assert torch.equal(g == -math.inf, none)
        d = (g - l)[~none].abs()
        assert d.numel() == 0 or d.max() < 1e-3 + 1e-5 * l[~none].abs().max()


MIXED = [(37, 0), (1, 0), (1, 1), (0, 0), (5, 300), (1, 127), (1, 128), (1, 900), (130, 257), (0, 40), (3, 126)]
DECODES = [(1, n) for n in (0, 15, 16, 17, 126, 127, 128, 255, 256, 1000, 3, 2047)]
LONG = [(1, 20000), (9, 7000)]


@pytest.mark.parametrize("batch", [MIXED, DECODES, LONG], ids=["mixed", "decodes", "long"])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (6, 6), (14, 2), (16, 2)])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_attention_against_64_bits(dtype, hd, heads, kv_heads, batch):
    from sarathi_serve_b200 import attention_ops
    c = make(1, dtype, heads, kv_heads, hd, 16, batch, pad=3)
    plan, _ = plan_of(c)
    lse = torch.full((c["T"], heads), 7.0, device="cuda")
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5, lse=lse)
    check(c, out, hd ** -0.5, lse=lse)
    assert out[c["total"]:].abs().sum() == 0 and (lse[c["total"]:] == -math.inf).all()


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 64, 128, 256, 100])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_page_sizes(dtype, hd, page):
    """Pages that end inside a block of keys, hold several, or are one token."""
    from sarathi_serve_b200 import attention_ops
    c = make(2, dtype, 8, 2, hd, page, [(150, 201), (1, 511), (1, 3), (33, 0), (64, 64)])
    plan, _ = plan_of(c)
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.11)
    check(c, out, 0.11)


@pytest.mark.parametrize("window", [1, 2, 64, 127, 128, 129, 500])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128)])
def test_sliding_window(dtype, hd, window):
    """Pages that have left every window may hold anything: here they are not in the cache at all."""
    from sarathi_serve_b200 import attention_ops
    c = make(3, dtype, 8, 2, hd, 16, [(200, 333), (1, 1000), (1, 5), (70, 0), (2, 640)])
    plan, layout = plan_of(c, window)
    for r, (new, before) in enumerate(c["batch"]):
        gone = max(0, before + 1 - window) // c["page"]
        at = int(layout.kv_indptr[r])
        layout.kv_indices[at:at + gone] = 10 ** 9
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5)
    check(c, out, hd ** -0.5, window)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_a_row_does_not_see(dtype, hd, bad):
    """A key or value that is not finite reaches the rows that see it and no others, neither in a chunk (later tokens of the
    same block) nor under a window (earlier ones)."""
    from sarathi_serve_b200 import attention_ops
    for window in (0, 40):
        for new, before, at in ((90, 100, 150), (3, 200, 201), (300, 0, 130), (1, 60, 5), (260, 20, 100)):
            c = make(4, dtype, 4, 2, hd, 16, [(new, before), (1, 77)])
            c["cache"][c["table"][0, at // 16], 1, at % 16, 1, 5] = bad
            plan, _ = plan_of(c, window)
            out = attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5)
            want, _, _ = reference(c, hd ** -0.5, window)
            got, fine = out[:c["total"]].double().view(-1, 4, hd), torch.isfinite(want).view(-1, 4, hd)
            # (which of the not finite values a row gets is left open, and so are its other columns' last bits)
            assert torch.equal(torch.isfinite(got), fine), (window, new, before, at)
            c2 = dict(c, cache=c["cache"].clone())
            c2["cache"][c["table"][0, at // 16], 1, at % 16, 1, 5] = 0
            clean, _, tol = reference(c2, hd ** -0.5, window)
            d = (got.view(c["total"], -1) - clean).abs() - tol
            assert d[fine.view(c["total"], -1)].max() <= 0, (window, new, before, at)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_a_value_that_is_not_finite_in_a_long_context(dtype, hd):
    """Seen by every row of a chunk: their results are not finite in its column, the other columns are as they were."""
    from sarathi_serve_b200 import attention_ops
    c = make(12, dtype, 4, 2, hd, 16, [(200, 5000), (1, 3000)])
    for r, at in ((0, 17), (1, 2990)):
        c["cache"][c["table"][r, at // 16], 1, at % 16, 0, 7] = float("inf")
    plan, _ = plan_of(c)
    check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5), hd ** -0.5)


@pytest.mark.parametrize("dtype,hd,kv_heads,pages", [(torch.bfloat16, 128, 8, 70000), (torch.float32, 64, 8, 140000)])
def test_cache_beyond_32_bits_of_elements(dtype, hd, kv_heads, pages):
    """Pages whose elements lie beyond 2^31, in all kinds of tiles."""
    from sarathi_serve_b200 import attention_ops
    batch, page = [(1, 300), (70, 130), (5, 20)], 16
    c = make(13, dtype, 2 * kv_heads, kv_heads, hd, page, batch)
    big = torch.empty(pages, 2, page, kv_heads, hd, dtype=dtype, device="cuda")
    assert big.numel() > 2 ** 31
    used = c["pool"]
    big[pages - used:] = c["cache"]
    c.update(cache=big, table=torch.where(c["table"] >= 0, c["table"] + (pages - used), c["table"]), pool=pages)
    plan, lay = plan_of(c)
    assert int(lay.kv_slots.max()) * kv_heads * hd > 2 ** 31 - 2 ** 24
    check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5), hd ** -0.5)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128)])
def test_keys_that_are_not_numbers(dtype, hd):
    """A NaN in a key makes the rows that see it NaN, wherever it lies in a block, and leaves the others alone."""
    from sarathi_serve_b200 import attention_ops
    for window in (0, 40):
        for new, before, at in [(200, 100, 131 + 7 * i) for i in range(9)] + [(3, 200, 201), (1, 60, 59), (260, 20, 100)]:
            c = make(11, dtype, 4, 2, hd, 16, [(new, before), (1, 77)], cache_fill=0.0)
            clean, _, tol = reference(c, hd ** -0.5, window)
            c["cache"][c["table"][0, at // 16], 0, at % 16, 1, 3] = float("nan")
            plan, _ = plan_of(c, window)
            lse = torch.zeros(c["T"], 4, device="cuda")
            out = attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5, lse=lse)
            pos = before + torch.arange(new, device="cuda")
            sees = (pos >= at) & ((pos < at + window) if window else (pos >= 0))
            got = out[:c["total"]].double().view(-1, 4, hd)
            assert torch.isnan(got[:new][sees][:, 2:]).all() and torch.isnan(lse[:new][sees][:, 2:]).all()
            got[:new, 2:][sees] = clean.view(-1, 4, hd)[:new, 2:][sees]
            assert ((got.view(c["total"], -1) - clean).abs() <= tol).all(), (window, new, before, at)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_extreme_scores(dtype, hd):
    """Maxima that grow from block to block by far more than a probability has bits, large negative scores, equal scores."""
    from sarathi_serve_b200 import attention_ops
    c = make(5, dtype, 4, 2, hd, 16, [(140, 500), (1, 700), (2, 0)], spread=0.5, cache_fill=0.0)
    flat = c["cache"].view(-1, 2, c["page"], 2, hd)
    for r in range(2):
        n = sum(c["batch"][r])
        for j in range(n):
            flat[c["table"][r, j // 16], 0, j % 16] *= 1 + j / 20.0
    plan, _ = plan_of(c)
    for scale in (1.0, -1.0, 0.0):
        check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, scale), scale)


def test_rows_behind_the_last_request_and_strides():
    """A given `out` keeps the rows of the padding, and a strided one what lies between its rows."""
    from sarathi_serve_b200 import attention_ops
    for dtype, hd in ((torch.bfloat16, 128), (torch.float32, 64)):
        c = make(6, dtype, 4, 2, hd, 16, [(20, 3), (1, 200), (140, 0)], pad=7)
        plan, _ = plan_of(c, max_requests=9, max_tokens=400)
        wide = torch.full((c["T"], 6 * hd), 3.0, dtype=dtype, device="cuda")
        lse = torch.full((c["T"], 4), 5.0, device="cuda")
        out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1, out=wide[:, :4 * hd], lse=lse)
        check(c, out, 0.1, lse=lse)
        assert (wide[:, 4 * hd:] == 3).all() and (wide[c["total"]:] == 3).all() and (lse[c["total"]:] == 5).all()


def test_queries_and_results_in_one_buffer():
    """Side by side they do not overlap; on top of each other they are refused."""
    from sarathi_serve_b200 import attention_ops
    c = make(16, torch.bfloat16, 4, 2, 128, 16, [(150, 30), (1, 200), (9, 0)])
    plan, _ = plan_of(c)
    wide = torch.zeros(c["T"], 1024, dtype=torch.bfloat16, device="cuda")
    wide[:, :512] = c["q"]
    out = attention_ops.paged_attention(wide[:, :512], c["cache"], plan, 0.1, out=wide[:, 512:])
    check(c, out, 0.1)
    assert torch.equal(wide[:, :512], c["q"])
    for out in (wide[:, :512], wide[:, 256:768], c["cache"].view(-1, 512)[:c["T"]]):
        with pytest.raises(RuntimeError, match="overlap"):
            attention_ops.paged_attention(wide[:, :512], c["cache"], plan, 0.1, out=out)


def test_lengths_that_the_caller_got_wrong():
    """More new tokens than the cache holds (their first rows see nothing), page ids outside the cache, q with fewer rows
    than planned, a list that ends early: defined results, nothing out of range."""
    from sarathi_serve_b200 import attention_ops
    for dtype, hd in ((torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 64)):
        c = make(7, dtype, 4, 2, hd, 16, [(10, 0), (150, 0)])
        plan, lay = plan_of(c)
        short = lay.kv_lens - 4
        plan.update(qo_indptr=lay.qo_indptr, kv_lens=short, kv_indptr=lay.kv_indptr, kv_indices=lay.kv_indices)
        out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1)
        for at, n in ((0, 10), (10, 150)):
            assert out[at:at + 4].abs().sum() == 0
            shifted = dict(c, batch=[(n - 4, 0)], total=n - 4, q=c["q"][at + 4:at + n], table=c["table"][0 if at == 0 else 1:])
            check(shifted, out[at + 4:at + n], 0.1)
        # pages that do not exist read as zeros
        zero = dict(c, cache=c["cache"].clone())
        zero["cache"][c["table"][1, 3]] = 0
        for wrong in (-1, c["pool"], 2 ** 31 - 1, -2 ** 31):
            lay.kv_indices[int(lay.kv_indptr[1]) + 3] = wrong
            plan.update(lay)
            check(zero, attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1), 0.1)
        lay.kv_indices[int(lay.kv_indptr[1]) + 3] = c["table"][1, 3]
        # fewer rows of q than planned
        few = attention_ops.paged_attention(c["q"][:77], c["cache"], plan, 0.1)
        whole = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1)
        want, _, tol = reference(c, 0.1)
        assert ((few.double() - want[:77]).abs() <= tol[:77]).all() and few.shape[0] == 77
        assert ((whole.double() - want).abs() <= tol).all()
        # lengths far beyond the listed pages are cut to them: 160 tokens have room in the second list
        plan.update(qo_indptr=lay.qo_indptr, kv_lens=torch.full_like(lay.kv_lens, 2 ** 31 - 1), kv_indptr=lay.kv_indptr, kv_indices=lay.kv_indices)
        attention_ops.paged_attention(c["q"], torch.nan_to_num(c["cache"]), plan, 0.1)
        torch.cuda.synchronize()


def test_nothing_to_do():
    from sarathi_serve_b200 import attention_ops
    for dtype in (torch.bfloat16, torch.float32):
        c = make(8, dtype, 4, 2, 128, 16, [(0, 0), (0, 30)], pad=5)
        plan, _ = plan_of(c)
        out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1)
        assert out.shape == (5, 512) and out.abs().sum() == 0
        assert attention_ops.paged_attention(c["q"][:0], c["cache"], plan, 0.1).shape == (0, 512)


def test_repeats_agree_and_shared_pages():
    """Repeats agree bit for bit (cut units are joined in the order of their keys), and requests may share pages."""
    from sarathi_serve_b200 import attention_ops
    for dtype in (torch.bfloat16, torch.float32):
        c = make(9, dtype, 8, 2, 128, 16, [(1, 5000), (1, 5000), (40, 1000)])
        c["table"][1] = c["table"][0]
        plan, _ = plan_of(c)
        first = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.09)
        check(c, first, 0.09)
        for _ in range(3):
            assert torch.equal(attention_ops.paged_attention(c["q"], c["cache"], plan, 0.09), first)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128)])
def test_values_before_and_behind_the_window(dtype, hd):
    """Values that are not finite at keys that leave the window inside a tile, that enter it there, and at both."""
    from sarathi_serve_b200 import attention_ops
    c = make(17, dtype, 8, 2, hd, 16, [(150, 300), (1, 700), (40, 90), (3, 250)])
    for r, keys in enumerate(((170, 299, 401, 449), (500, 612), (0, 60, 111), (120, 121, 252))):
        for i, j in enumerate(keys):
            c["cache"][c["table"][r, j // 16], 1, j % 16, i % 2, 5 * i:5 * i + 3] = (math.nan, math.inf)[i % 2]
    plan, _ = plan_of(c, window=130)
    check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1), 0.1, window=130)


@pytest.mark.parametrize("heads,hd", [(71, 64), (128, 128), (300, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_heads_on_one(dtype, heads, hd):
    """Groups wider than a tile of few rows, and than one of many: a token alone fills it; q with its heads apart."""
    from sarathi_serve_b200 import attention_ops
    c = make(18, dtype, heads, 1, hd, 16, [(1, 260), (3, 17), (1, 0), (2, 130)])
    plan, _ = plan_of(c)
    q = c["q"].unflatten(1, (heads, hd))
    check(c, attention_ops.paged_attention(q, c["cache"], plan, 0.1), 0.1)


@pytest.mark.parametrize("dtype,requests", [(torch.bfloat16, 3000), (torch.float32, 1500), (torch.float16, 8192)])
def test_thousands_of_requests(dtype, requests):
    """More tiles than the plan keeps near; the most requests that there can be."""
    from sarathi_serve_b200 import attention_ops
    g = torch.Generator().manual_seed(requests)
    now = torch.randint(0, 24, (requests,), generator=g).tolist()
    c = make(19, dtype, 2, 1, 64, 8, [(1, n) for n in now])
    plan, _ = plan_of(c)
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.125)
    few = list(range(0, requests, max(1, requests // 150)))
    part = dict(c, batch=[c["batch"][r] for r in few], total=len(few), q=c["q"][few], table=c["table"][few])
    check(part, out[few], 0.125)
    assert torch.isfinite(out).all()


# ------------------------------------------------------------------ block tables and layout
def layout_by_hand(query, context, table, page, pages, T):
    n, width = table.shape
    most = width * page
    ctx = [min(max(int(x), 0), most) for x in context]
    new = [min(max(int(x), 0), most - c) for x, c in zip(query, ctx)]
    qo = [0]
    for x in new:
        qo.append(min(qo[-1] + x, T))
    new = [b - a for a, b in zip(qo, qo[1:])]
    kv = [a + b for a, b in zip(new, ctx)]
    need = [-(-x // page) for x in kv]
    indptr, idx = [0], []
    for r, x in enumerate(need):
        indptr.append(indptr[-1] + x)
        idx += [int(v) for v in table[r, :x]]
    idx += [-1] * (n * width - len(idx))
    last = [x - (y - 1) * page if x else 0 for x, y in zip(kv, need)]
    req, pos, slot = [], [], []
    for r, x in enumerate(new):
        for i in range(x):
            p = ctx[r] + i
            b = int(table[r, p // page])
            req.append(r)
            pos.append(p)
            slot.append(b * 2 * page + p % page if 0 <= b < pages else -1)
    pad = T - len(req)
    return [qo, kv, indptr, idx, last, req + [-1] * pad, pos + [0] * pad, slot + [-1] * pad]


@pytest.mark.parametrize("n,width,page,T", [(1, 1, 1, 1), (1, 4, 16, 70), (7, 5, 24, 64), (61, 40, 16, 64), (600, 9, 8, 700),
                                           (3, 2000, 16, 30000), (8192, 2, 4, 9000), (5, 3, 16, 0), (4, 0, 16, 8)])
def test_batch_layout(n, width, page, T):
    from sarathi_serve_b200 import kv_cache_ops
    g = torch.Generator().manual_seed(n)
    table = torch.randint(-2, n * width + 2, (n, width), generator=g, dtype=torch.int32)
    context = torch.randint(-3, width * page + 20, (n,), generator=g, dtype=torch.int32)
    query = torch.randint(-1, max(2, 2 * T // n), (n,), generator=g, dtype=torch.int32)
    query[::5] = 1
    if n > 2:
        query[1], context[2] = 2 ** 31 - 1, 2 ** 31 - 1
    wide = torch.zeros(n, width + 3, dtype=torch.int32).cuda()
    wide[:, :width] = table.cuda()
    want = layout_by_hand(query.tolist(), context.tolist(), table, page, n * width, T)
    got = kv_cache_ops.batch_layout(query.cuda(), context.cuda(), wide[:, :width], page, n * width, T)
    for name, a, b in zip(got._fields, got, want):
        assert a.tolist() == b, name
    again = kv_cache_ops.batch_layout(query.cuda(), context.cuda(), wide[:, :width], page, n * width, T, out=got)
    assert all(a is b for a, b in zip(again, got)) and again.kv_slots.tolist() == want[7]


def test_layout_agrees_with_slots():
    """The slots are those that kv_cache_ops.slots computes from the same arrays."""
    from sarathi_serve_b200 import kv_cache_ops
    c = make(10, torch.float32, 2, 1, 64, 16, MIXED, pad=5)
    lay = kv_cache_ops.batch_layout(c["query"], c["context"], c["table"], 16, c["pool"], c["T"])
    s = kv_cache_ops.slots(lay.batch_indices, lay.positions.int(), lay.kv_indices, lay.kv_indptr, 16)
    assert torch.equal(s, lay.kv_slots)


def resize_by_hand(table, have, lens, free, count, page):
    n, width = table.shape
    table, have, free = table.clone(), [min(max(x, 0), width) for x in have], list(free)
    count = min(max(count, 0), len(free))
    want = [h if x < 0 else -(-x // page) for h, x in zip(have, lens)]
    granted = [1] * n
    full = False
    for r in range(n):
        if want[r] < have[r]:
            full = full or count + have[r] - want[r] > len(free)
            if full:
                granted[r] = 0
                continue
            for j in range(want[r], have[r]):
                free[count] = int(table[r, j])
                count += 1
    short = False
    for r in range(n):
        if want[r] > width:
            granted[r] = 0
        elif want[r] > have[r]:
            short = short or want[r] - have[r] > count
            if short:
                granted[r] = 0
                continue
            for j in range(have[r], want[r]):
                count -= 1
                table[r, j] = free[count]
    have = [w if k else h for w, h, k in zip(want, have, granted)]
    return table, have, free, count, granted


@pytest.mark.parametrize("n,width,page,spare,capacity", [(1, 1, 1, 1, 2), (5, 8, 16, 20, 60), (5, 8, 16, 3, 60), (128, 40, 16, 900, 6000),
                                                        (700, 64, 8, 9000, 40000), (33, 1000, 16, 7000, 40000), (33, 1000, 16, 700, 9000),
                                                        (8192, 4, 4, 5000, 40000), (64, 16, 16, 0, 2000), (6, 4, 16, 9, 9)])
def test_resize_block_tables(n, width, page, spare, capacity):
    from sarathi_serve_b200 import kv_cache_ops
    g = torch.Generator().manual_seed(n + spare)
    for trial in range(3):
        have = torch.randint(0, width + 1, (n,), generator=g)
        lens = torch.randint(0, width * page + 1, (n,), generator=g)
        keep = torch.rand(n, generator=g) < 0.5
        lens = torch.where(keep, have * page, lens)
        if n > 4:
            lens[3], lens[4] = -1, 2 ** 31 - 1
        pool = torch.randperm(n * width + capacity, generator=g).to(torch.int32)
        table = pool[:n * width].view(n, width).clone()
        free = torch.full((capacity,), -5, dtype=torch.int32)
        free[:spare] = pool[n * width:n * width + spare]
        want = resize_by_hand(table, have.tolist(), lens.tolist(), free.tolist(), spare, page)
        dev = [x.to(torch.int32).cuda() for x in (table, have, lens, free, torch.tensor([spare]))]
        granted = kv_cache_ops.resize_block_tables(dev[0], dev[1], dev[2], dev[3], dev[4], page)
        assert granted.tolist() == want[4]
        assert dev[1].tolist() == want[1] and int(dev[4]) == want[3]
        assert torch.equal(dev[0].cpu(), want[0]) and dev[3].tolist() == want[2]
        live = [dev[0][r, :int(dev[1][r])].tolist() for r in range(n)]
        ids = sum(live, []) + dev[3][:int(dev[4])].tolist()
        assert len(set(ids)) == len(ids), "a page has two owners"


def test_layout_of_the_next_step():
    """Last step's lengths are the next step's contexts: as a copy, not in place."""
    from sarathi_serve_b200 import kv_cache_ops
    i = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    table = torch.arange(40, dtype=torch.int32).view(4, 10).cuda()
    lay = kv_cache_ops.batch_layout(i([5, 1, 0, 30]), i([0, 9, 3, 40]), table, 8, 40, 40)
    with pytest.raises(RuntimeError, match="overlap"):
        kv_cache_ops.batch_layout(i([1, 1, 1, 1]), lay.kv_lens, table, 8, 40, 40, out=lay)
    kv_cache_ops.batch_layout(i([1, 1, 1, 1]), lay.kv_lens.clone(), table, 8, 40, 40, out=lay)
    assert lay.kv_lens.tolist() == [6, 11, 4, 71] and lay.positions[:4].tolist() == [5, 10, 3, 70]


def test_slots_of_very_large_pages():
    from sarathi_serve_b200 import kv_cache_ops
    i = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    lay = kv_cache_ops.batch_layout(i([2]), i([5]), i([[3]]), 1 << 30, 4, 3)
    assert lay.kv_slots.tolist() == [3 * 2 ** 31 + 5, 3 * 2 ** 31 + 6, -1]
