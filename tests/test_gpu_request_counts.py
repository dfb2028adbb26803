"""Plans, block tables and layouts of every number of requests up to the documented 8192, from a process that has made no larger
call before, and from two threads at once: what a launch is allowed depends neither on earlier calls nor on those beside it."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

PRELUDE = """
import sys, threading
sys.path[:0] = [{root!r}, {here!r}]
import torch
from sarathi_serve_b200 import attention_ops, kv_cache_ops
import test_gpu_attention as t


def attend(n):
    now = torch.randint(0, 24, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    c = t.make(19, torch.bfloat16, 2, 1, 64, 8, [(1, k) for k in now])
    plan, _ = t.plan_of(c)
    out = attention_ops.paged_attention(c["q"], c["cache"], plan, 0.125)
    few = list(range(0, n, 97)) + [n - 1]
    part = dict(c, batch=[c["batch"][r] for r in few], total=len(few), q=c["q"][few], table=c["table"][few])
    t.check(part, out[few], 0.125)


def lay_out(n):
    ints = lambda k: torch.full((n,), k, dtype=torch.int32, device="cuda")
    table = torch.arange(2 * n, dtype=torch.int32, device="cuda").view(n, 2)
    lay = kv_cache_ops.batch_layout(ints(1), ints(4), table, 4, 2 * n, n + 3)
    assert lay.qo_indptr.tolist() == list(range(n + 1)) and lay.kv_indptr.tolist() == list(range(0, 2 * n + 1, 2))
    assert torch.equal(lay.kv_indices, table.view(-1)) and lay.positions.tolist() == [4] * n + [0] * 3
    assert lay.kv_slots.tolist() == [(2 * r + 1) * 8 for r in range(n)] + [-1] * 3


def resize(n):
    ints = lambda k: torch.full((n,), k, dtype=torch.int32, device="cuda")
    table = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(n)
    free = torch.arange(n, 2 * n, dtype=torch.int32, device="cuda")
    count, have = torch.tensor([n], dtype=torch.int32, device="cuda"), ints(1)
    granted = kv_cache_ops.resize_block_tables(table, have, ints(5), free, count, 4)
    assert granted.tolist() == [1] * n and have.tolist() == [2] * n and int(count) == 0
    assert table[:, 1].tolist() == list(range(2 * n - 1, n - 1, -1))
"""


def run(body):
    script = PRELUDE.format(root=os.path.dirname(HERE), here=HERE) + body
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]


@pytest.mark.parametrize("call,counts", [("attend", (4185, 4186, 5000, 6143, 6144)), ("lay_out", (6109, 6110, 6143, 6144)),
                                         ("resize", (3054, 3055, 3063, 3071, 3500))])
def test_request_counts_in_a_fresh_process(call, counts):
    run("\n".join(f"{call}({n})" for n in sorted(set(counts))))


def test_request_counts_from_two_threads():
    """One thread plans and lays out as many requests as there can be while another one does fewer, which still are many."""
    run("""
failed = []


def many(n):
    try:
        ints = lambda k: torch.full((n,), k, dtype=torch.int32, device="cuda")
        table, one, four = torch.arange(2 * n, dtype=torch.int32, device="cuda").view(n, 2), ints(1), ints(4)
        plan = attention_ops.AttentionPlan(1, 1, 64, 4, torch.float16, n, n)
        free, count, have = ints(0), torch.zeros(1, dtype=torch.int32, device="cuda"), ints(2)
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            for _ in range(400):
                plan.update(kv_cache_ops.batch_layout(one, four, table, 4, 2 * n, n))
                kv_cache_ops.resize_block_tables(table, have, four + one, free, count, 4)
    except Exception as e:
        failed.append((n, e))


threads = [threading.Thread(target=many, args=(n,)) for n in (8192, 6200)]
for x in threads:
    x.start()
for x in threads:
    x.join()
torch.cuda.synchronize()
assert not failed, failed
""")
