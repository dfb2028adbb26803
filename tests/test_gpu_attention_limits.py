"""Attention at the ends of what its arguments can be, on the GPU, against 64 bits (tolerances: test_gpu_attention.py)."""
import math

import pytest
import torch

from test_gpu_attention import check, make, plan_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 64)])
@pytest.mark.parametrize("window", [2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1])
def test_windows_wider_than_any_request(dtype, hd, window):
    """They hide nothing, of requests with more new tokens than the cache holds (negative positions) either."""
    from sarathi_serve_b200 import attention_ops
    c = make(21, dtype, 4, 2, hd, 16, [(10, 0), (150, 0), (3, 200), (300, 129)])
    plan, lay = plan_of(c, window)
    check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1), 0.1)
    plan.update(qo_indptr=lay.qo_indptr, kv_lens=torch.where(lay.kv_lens < 160, lay.kv_lens - 4, lay.kv_lens), kv_indptr=lay.kv_indptr,
                kv_indices=lay.kv_indices)
    lse = torch.zeros(c["T"], 4, device="cuda")
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1, lse=lse)
    for r, (at, n) in enumerate(((0, 10), (10, 150))):
        assert out[at:at + 4].abs().sum() == 0 and (lse[at:at + 4] == -math.inf).all()
        check(dict(c, batch=[(n - 4, 0)], total=n - 4, q=c["q"][at + 4:at + n], table=c["table"][r:]), out[at + 4:at + n], 0.1)
    check(dict(c, batch=c["batch"][2:], total=303, q=c["q"][160:], table=c["table"][2:]), out[160:], 0.1)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 256), (torch.float16, 64), (torch.float32, 64),
                                      (torch.float32, 128), (torch.float32, 256)])
@pytest.mark.parametrize("window", [0, 150])
def test_values_that_are_not_finite_under_weights_that_vanish(dtype, hd, window):
    """A key that a row sees takes part, however small its probability: a value there that is not finite makes the row's column so,
    wherever the key lies in a step of keys, in a tile or in a unit that is cut.  exp(-300 or less) is 0 in fp32."""
    from sarathi_serve_b200 import attention_ops
    for batch, far in (([(90, 100), (3, 200), (1, 150)], 1), ([(1, 20000), (2, 9000)], 4000), ([(300, 2000)], 700)):
        for at in (0, 17, 99, 100, 101, 130, 140):
            c = make(22, dtype, 4, 2, hd, 16, batch, cache_fill=0.0)
            c["q"][:, ::hd] = 8.0
            for r, (new, before) in enumerate(batch):
                lo = max(0, before - 120) + at if window else at
                for j in range(lo, min(lo + far, new + before)):
                    c["cache"][c["table"][r, j // 16], 0, j % 16, :, 0] = -400.0     # scores of -320 and less
                if lo < new + before:
                    c["cache"][c["table"][r, lo // 16], 1, lo % 16, 1, 5] = (math.nan, math.inf)[at % 2]
            plan, _ = plan_of(c, window)
            check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1), 0.1, window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 16), (256, 16), (128, 12)])
@pytest.mark.parametrize("batch", [[(1, 20000), (3, 9000)], [(200, 5000), (1, 300)]], ids=["decodes", "chunk"])
def test_one_key_that_outweighs_thousands(dtype, hd, page, batch):
    """One key has a value of 0 and a score 10 to 15 above the others', whose probabilities (2^-14 to 2^-22 of it) make the result.
    Tolerance: that of test_gpu_attention.py, but what fp16 loses below its full precision is 2^-32 of the largest a key (at worst
    2^-25 of 2^-7)."""
    from sarathi_serve_b200 import attention_ops
    heads, scale = 4, 1.0
    u = torch.finfo(dtype).eps / 2
    for sink in (0, 100):
        c = make(23, dtype, heads, 1, hd, page, batch, cache_fill=0.0)
        c["q"].zero_()
        a = (10 + 5 * torch.rand(c["T"], heads, generator=torch.Generator().manual_seed(5))).to(dtype).cuda()
        c["q"][:, ::hd] = a / 8
        plan, _ = plan_of(c)
        want = []
        for r, (new, before) in enumerate(batch):
            n = new + before
            where = torch.arange(n, device="cuda")
            pages = c["table"][r].long()[where // page]
            c["cache"][pages, 0, where % page] = 0
            c["cache"][pages[sink], 0, sink % page, 0, 0] = 8.0
            c["cache"][pages, 1, where % page] = c["cache"][pages, 1, where % page].abs().clamp(max=2.0)
            c["cache"][pages[sink], 1, sink % page] = 0
            v = c["cache"][pages, 1, where % page][:, 0].double()
            row = sum(b[0] for b in batch[:r])
            s = torch.zeros(new, heads, n, dtype=torch.float64, device="cuda")
            s[:, :, sink] = (c["q"][row:row + new, ::hd].double() * 8)
            s.masked_fill_((where > before + torch.arange(new, device="cuda")[:, None])[:, None], -math.inf)
            res = torch.softmax(s, 2) @ v
            delta = (hd + 16) * 2.0 ** -24 * 16 + 2.0 ** -21
            tol = (2 * u + 2 * delta + 2 * (n + 16) * 2.0 ** -24) * res + (n * 2.0 ** -32 * 2 + 2.0 ** -25 if dtype == torch.float16 else 0)
            want.append((res, tol))
        lse = torch.zeros(c["T"], heads, device="cuda")
        out = attention_ops.paged_attention(c["q"], c["cache"], plan, scale, lse=lse).view(-1, heads, hd).double()
        res, tol = (torch.cat(x) for x in zip(*want))
        worst = ((out - res).abs() / tol).max().item()
        assert worst <= 1, f"{worst:.2f} times the tolerance"
        check(c, out.view(-1, heads * hd), scale, lse=lse)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 64)])
def test_rows_ahead_of_the_first_request(dtype, hd):
    """Offsets that start behind row 0: the rows ahead belong to no request, as those behind the last one's."""
    from sarathi_serve_b200 import attention_ops
    c = make(24, dtype, 4, 2, hd, 16, [(20, 3), (1, 200), (140, 0)], pad=9)
    plan, lay = plan_of(c)
    plan.update(qo_indptr=lay.qo_indptr + 5, kv_lens=lay.kv_lens, kv_indptr=lay.kv_indptr, kv_indices=lay.kv_indices)
    part = dict(c, q=c["q"][5:166])
    lse = torch.full((c["T"], 4), 7.0, device="cuda")
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1, lse=lse)
    check(part, out[5:], 0.1, lse=lse[5:])
    for rows in (slice(0, 5), slice(166, c["T"])):
        assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()
    given, lse = torch.full_like(out, 3.0), torch.full_like(lse, 7.0)
    attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1, out=given, lse=lse)
    assert torch.equal(given[5:166], out[5:166])
    for rows in (slice(0, 5), slice(166, c["T"])):
        assert (given[rows] == 3).all() and (lse[rows] == 7).all()
