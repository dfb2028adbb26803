"""The forms of the attention that test_gpu_attention.py takes at one type or head size only, at the others; long chunks, units cut into
many pieces, lengths beyond the listed pages, several plans at once.  Against 64 bits, with the tolerances of that file."""
import threading

import pytest
import torch

import test_gpu_attention as base

pytestmark = pytest.mark.gpu

OTHERS = [(torch.bfloat16, 64), (torch.bfloat16, 256), (torch.float16, 128), (torch.float16, 256), (torch.float32, 256)]
forms = pytest.mark.parametrize("dtype,hd", OTHERS)


@forms
@pytest.mark.parametrize("page", [1, 8, 12, 16, 24, 100, 256])
def test_page_sizes(dtype, hd, page):
    base.test_page_sizes(dtype, hd, page)


@forms
@pytest.mark.parametrize("window", [1, 64, 127, 129, 500])
def test_sliding_window(dtype, hd, window):
    base.test_sliding_window(dtype, hd, window)


@forms
@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_values_that_a_row_does_not_see(dtype, hd, bad):
    base.test_values_that_a_row_does_not_see(dtype, hd, bad)


@forms
def test_values_before_and_behind_the_window(dtype, hd):
    base.test_values_before_and_behind_the_window(dtype, hd)


@forms
def test_keys_that_are_not_numbers(dtype, hd):
    base.test_keys_that_are_not_numbers(dtype, hd)


@forms
def test_a_value_that_is_not_finite_in_a_long_context(dtype, hd):
    base.test_a_value_that_is_not_finite_in_a_long_context(dtype, hd)


@forms
def test_extreme_scores(dtype, hd):
    base.test_extreme_scores(dtype, hd)


@pytest.mark.parametrize("dtype,hd,page", [(torch.bfloat16, 128, 12), (torch.float16, 64, 3), (torch.bfloat16, 64, 1)])
def test_values_under_pages_that_are_no_multiple_of_8(dtype, hd, page):
    """(Chunks take the tiles of few rows then.)  Values that are not finite behind the window, before it and behind the end."""
    from sarathi_serve_b200 import attention_ops
    c = base.make(31, dtype, 8, 2, hd, page, [(150, 300), (1, 700), (40, 90), (3, 250)])
    for r, keys in enumerate(((170, 299, 401, 449), (500, 612), (0, 60, 111), (120, 121, 252))):
        for i, j in enumerate(keys):
            c["cache"][c["table"][r, j // page], 1, j % page, i % 2, 5 * i:5 * i + 3] = (float("nan"), float("inf"))[i % 2]
    for window in (0, 130):
        plan, _ = base.plan_of(c, window=window)
        base.check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1), 0.1, window=window)


@pytest.mark.parametrize("window", [0, 3000])
@pytest.mark.parametrize("dtype,hd,heads,kv_heads,batch", [
    (torch.bfloat16, 128, 4, 1, [(2500, 6001), (1, 500), (700, 0)]),
    (torch.float16, 64, 4, 2, [(1999, 9000), (3, 4000)]),
    (torch.bfloat16, 64, 2, 2, [(3500, 0), (64, 5000)]),
    (torch.float16, 128, 8, 1, [(1037, 7777)]),
    (torch.bfloat16, 256, 2, 1, [(700, 3000)]),
    (torch.float32, 64, 4, 1, [(1100, 4000)])])
def test_long_chunks(dtype, hd, heads, kv_heads, batch, window):
    from sarathi_serve_b200 import attention_ops
    c = base.make(32, dtype, heads, kv_heads, hd, 16, batch)
    plan, _ = base.plan_of(c, window)
    lse = torch.zeros(c["T"], heads, device="cuda")
    base.check(c, attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5, lse=lse), hd ** -0.5, window, lse=lse)


@pytest.mark.parametrize("window", [0, 20001])
@pytest.mark.parametrize("dtype,hd,heads,new", [(torch.bfloat16, 128, 2, 100), (torch.float16, 64, 3, 85), (torch.bfloat16, 64, 1, 129),
                                                (torch.float16, 128, 2, 64), (torch.bfloat16, 256, 2, 7), (torch.float32, 64, 2, 32)])
def test_one_unit_over_all_workers(dtype, hd, heads, new, window):
    """One tile (both halves, or one of them) against 40000 keys: as many pieces as there are workers; values that are not finite too."""
    from sarathi_serve_b200 import attention_ops
    c = base.make(33, dtype, heads, 1, hd, 16, [(new, 40000)])
    for bad in (False, True):
        if bad:
            for j in (25000, 40000 + new // 2):
                c["cache"][c["table"][0, j // 16], 1, j % 16, 0, 9] = float("nan")
        plan, _ = base.plan_of(c, window)
        out = attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5)
        base.check(c, out, hd ** -0.5, window)
        assert torch.equal(torch.nan_to_num(out, nan=77.0),
                           torch.nan_to_num(attention_ops.paged_attention(c["q"], c["cache"], plan, hd ** -0.5), nan=77.0))


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 64)])
def test_lengths_beyond_the_listed_pages(dtype, hd):
    """They are cut to what the pages have room for: the last new token stands in the last slot of the last listed page."""
    from sarathi_serve_b200 import attention_ops
    c = base.make(34, dtype, 4, 2, hd, 16, [(10, 0), (150, 0), (1, 99), (3, 205)], cache_fill=0.25)
    plan, lay = base.plan_of(c)
    plan.update(qo_indptr=lay.qo_indptr, kv_lens=torch.full_like(lay.kv_lens, 2 ** 31 - 1), kv_indptr=lay.kv_indptr, kv_indices=lay.kv_indices)
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1)
    room = [-(-sum(b) // 16) * 16 for b in c["batch"]]
    base.check(dict(c, batch=[(new, n - new) for (new, _), n in zip(c["batch"], room)]), out, 0.1)


def test_plans_of_several_threads():
    """Each with its own plan and stream; the library keeps nothing between calls that they could share."""
    from sarathi_serve_b200 import attention_ops
    kinds = [(torch.bfloat16, 128, [(300, 1000), (1, 4000)]), (torch.float16, 64, [(1, 700)] * 40), (torch.float32, 64, [(64, 300), (1, 900)]),
             (torch.bfloat16, 256, [(20, 500), (1, 30)])]
    cases = [base.make(35, dtype, 4, 2, hd, 16, batch) for dtype, hd, batch in kinds]
    single = []
    for c in cases:
        plan, _ = base.plan_of(c)
        single.append(attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1))
        base.check(c, single[-1], 0.1)
    torch.cuda.synchronize()
    failed = []

    def work(c, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                plan, layout = base.plan_of(c)
                for _ in range(50):
                    plan.update(layout)
                    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, want):
                    failed.append(c["dtype"])
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(cases, single)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_a_list_of_pages_is_not_given_away_while_it_is_read():
    """Layouts made on a side stream, the plan on the main one: what the plan has let go of stays out of the side stream's hands until
    the main stream has passed it."""
    from sarathi_serve_b200 import attention_ops, kv_cache_ops
    c = base.make(36, torch.bfloat16, 4, 2, 128, 16, [(1, 700), (9, 0)])
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    plan = attention_ops.AttentionPlan(4, 2, 128, 16, torch.bfloat16, 2, c["T"])

    def layout():
        with torch.cuda.stream(side):
            return kv_cache_ops.batch_layout(c["query"], c["context"], c["table"], 16, c["pool"], c["T"])
    side.wait_stream(main)
    first, second = layout(), layout()
    at = first.qo_indptr.untyped_storage().data_ptr()
    main.wait_stream(side)
    plan.update(first)
    torch.cuda._sleep(200_000_000)   # (0.1 s)
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1)
    del first
    plan.update(second)
    third = layout()
    busy = not main.query()
    assert not busy or third.qo_indptr.untyped_storage().data_ptr() != at
    assert busy, "the main stream was through too early to tell"
    base.check(c, out, 0.1)
