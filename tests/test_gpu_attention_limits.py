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
