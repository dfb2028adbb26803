"""Attention and batch layout without a GPU: argument checks of the C entry points and of the Python wrappers, the exactness
of the product that stands for a division, and a host model of the barriers inside a CTA of the tensor-core kernel."""
import ctypes
import random

import pytest
import torch

from sarathi_serve_b200 import _native as N


def shape(heads=8, kv=2, hd=128, page=16, dtype=2, window=0, requests=4, tokens=64):
    return N.AttentionShape(heads, kv, hd, page, dtype, window, requests, tokens)


@pytest.mark.parametrize("bad,status", [(dict(heads=6, kv=4), 1), (dict(kv=0), 1), (dict(page=0), 1), (dict(window=-1), 1),
                                        (dict(hd=96), 2), (dict(hd=512), 2), (dict(dtype=7), 2), (dict(requests=8193), 2),
                                        (dict(tokens=-1), 1), (dict(heads=1 << 16, kv=1, tokens=1 << 20), 1)])
def test_shapes_that_are_refused(bad, status):
    s = ctypes.byref(shape(**bad))
    assert N.lib().sb200_attention_plan_bytes(s) == -1 and N.lib().sb200_attention_workspace_bytes(s) == -1
    assert N.lib().sb200_attention_plan(16, 1 << 30, s, 16, 16, 16, 1, 1, None) == status
    assert N.lib().sb200_paged_attention(16, 4096, None, 16, 4096, 1, 16, 1, 16, s, 16, 1, 1.0, 0, 16, 1 << 40, None, None) == status


def test_sizes_of_plan_and_workspace():
    lib = N.lib()
    small, large = shape(), shape(requests=128, tokens=2048)
    assert 0 < lib.sb200_attention_plan_bytes(ctypes.byref(small)) < lib.sb200_attention_plan_bytes(ctypes.byref(large)) < 1 << 20
    assert lib.sb200_attention_workspace_bytes(ctypes.byref(small)) == lib.sb200_attention_workspace_bytes(ctypes.byref(large))
    assert lib.sb200_attention_plan_bytes(ctypes.byref(shape(requests=0, tokens=0))) > 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="makes calls on addresses that are not device memory")
def test_calls_that_are_refused():
    """Refused before any CUDA call: pointers, alignment, strides, sizes."""
    lib = N.lib()
    s = shape()
    sp = ctypes.byref(s)
    plan, ws = lib.sb200_attention_plan_bytes(sp), lib.sb200_attention_workspace_bytes(sp)
    good = dict(out=4096, ldo=1024, lse=None, q=4096, ldq=1536, T=8, cache=4096, pages=10, plan=4096, idx=4096, nidx=10, scale=0.1, zero=0,
                ws=4096, wsb=ws)
    call = lambda **k: lib.sb200_paged_attention(*[{**good, **k}[n] for n in ("out", "ldo", "lse", "q", "ldq", "T", "cache", "pages", "plan")],
                                                 sp, *[{**good, **k}[n] for n in ("idx", "nidx", "scale", "zero", "ws", "wsb")], None, None)
    for bad in (dict(out=None), dict(q=None), dict(cache=None), dict(plan=None), dict(idx=None), dict(q=4100), dict(out=4104),
                dict(cache=4104), dict(ldq=1020), dict(ldq=1028), dict(ldo=1000), dict(T=65), dict(T=-1), dict(pages=0), dict(pages=1 << 40),
                dict(ws=None), dict(wsb=ws - 1), dict(ws=4104), dict(scale=float("nan")), dict(scale=float("inf")), dict(nidx=-1)):
        assert call(**bad) == 1, bad
    assert call(T=0) == 0
    make = lambda p=4096, b=plan, qo=4096, kl=4096, kp=4096, n=2, m=10: lib.sb200_attention_plan(p, b, sp, qo, kl, kp, n, m, None)
    for bad in (dict(p=None), dict(p=4100), dict(b=plan - 1), dict(qo=None), dict(kl=None), dict(kp=None), dict(n=5), dict(n=-1), dict(m=-1)):
        assert make(**bad) == 1, bad
    tables = lambda t=4096, ld=8, nb=4096, sl=4096, f=4096, nf=4096, g=4096, n=4, w=8, c=100, pg=16: \
        lib.sb200_resize_block_tables(t, ld, nb, sl, f, nf, g, n, w, c, pg, None)
    for bad in (dict(t=None), dict(nb=None), dict(sl=None), dict(f=None), dict(nf=None), dict(g=None), dict(ld=7), dict(n=-1), dict(c=-1),
                dict(pg=0), dict(n=8000, w=1 << 20, ld=1 << 20)):
        assert tables(**bad) == 1, bad
    assert tables(n=8193) == 2 and tables(n=0) == 0
    lay = lambda q=4096, n=4, w=8, ld=8, pg=16, pages=10, T=8, cap=32, out=4096: \
        lib.sb200_batch_layout(q, 4096, 4096, ld, n, w, pg, pages, T, out, 4096, 4096, 4096, cap, 4096, 4096, 4096, 4096, None)
    for bad in (dict(q=None), dict(out=None), dict(cap=31), dict(ld=7), dict(pg=0), dict(T=-1), dict(pages=-1), dict(pages=1 << 33),
                dict(n=-1)):
        assert lay(**bad) == 1, bad
    assert lay(n=8193, w=0, ld=0) == 2


@pytest.mark.skipif(torch.cuda.is_available(), reason="makes calls on addresses that are not device memory")
def test_arrays_that_overlap_are_refused():
    """A result on top of its own input would be read by one SM after another has written it."""
    lib = N.lib()
    refused = lambda rc: rc == 1 and b"overlap" in lib.sb200_last_error()
    s = shape()
    sp, ws = ctypes.byref(s), lib.sb200_attention_workspace_bytes(ctypes.byref(s))
    page = 2 * 16 * 2 * 128 * 2  # bytes
    q, cache, far = 1 << 20, 1 << 30, 1 << 40
    call = lambda out, ldo=1280, T=8: lib.sb200_paged_attention(out, ldo, None, q, 1280, T, cache, 10, 4096, sp, 4096, 10, 0.1, 0, far, ws,
                                                                None, None)
    # 8 rows of 1024 elements of 2 bytes, 1280 elements apart
    for out in (q, q + 16, q + 2032, q - 2032, q + 7 * 2560, q + 2560 - 16, q + 3 * 2560 + 1040):
        assert refused(call(out)), out
    assert refused(call(q, T=1)) and refused(call(q + 2032, T=1)) and refused(call(q - 2 * 2560, ldo=2048))
    for out in (cache, cache + 10 * page - 16, cache - 7 * 2560):
        assert refused(call(out)), out

    a = [1 << (20 + i) for i in range(11)]
    tables = lambda t=a[0], nb=a[1], sl=a[2], f=a[3], nf=a[4], g=a[5]: lib.sb200_resize_block_tables(t, 8, nb, sl, f, nf, g, 4, 8, 100, 16, None)
    for bad in (dict(g=a[1]), dict(g=a[4] - 12), dict(nf=a[3] + 396), dict(sl=a[1] + 8), dict(f=a[0] + 31 * 4), dict(g=a[2])):
        assert refused(tables(**bad)), bad
    names = ("query", "context", "table", "qo", "kv", "indptr", "indices", "last", "req", "pos", "slot")
    good = dict(zip(names, a))

    def lay(**k):
        x = {**good, **k}
        return lib.sb200_batch_layout(x["query"], x["context"], x["table"], 8, 4, 8, 16, 10, 8, x["qo"], x["kv"], x["indptr"], x["indices"],
                                      40, x["last"], x["req"], x["pos"], x["slot"], None)
    for bad in (dict(context=good["kv"]), dict(query=good["kv"] + 12), dict(context=good["qo"] + 16), dict(table=good["indices"] + 39 * 4),
                dict(pos=good["slot"] + 56), dict(last=good["kv"]), dict(req=good["pos"] - 28)):
        assert refused(lay(**bad)), bad


def test_wrappers_want_gpu_tensors():
    from sarathi_serve_b200 import kv_cache_ops
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kv_cache_ops.batch_layout(i(2), i(2), i(2, 3), 16, 9, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kv_cache_ops.resize_block_tables(i(2, 3), i(2), i(2), i(9), i(1), 16)


def test_division_by_a_product():
    """FastDiv::of in csrc/attention.cuh: n / d for every d up to 2^16 at the numbers where it could be wrong."""
    rng = random.Random(0)
    for d in list(range(1, 2000)) + [rng.randint(2000, 1 << 20) for _ in range(2000)] + [1 << k for k in range(21)] + [65535, (1 << 20) - 1]:
        s = (d - 1).bit_length()
        mul = (1 << (31 + s)) // d + 1
        assert mul < 1 << 32
        top = (1 << 31) - 1
        for n in [0, 1, d - 1, d, d + 1, top, top // d * d, max(0, top // d * d - 1)] + [rng.randint(0, top) for _ in range(10)]:
            assert (n * mul) >> (31 + s) == n // d, (n, d)


class Barrier:
    """An mbarrier: a phase completes with its count of arrivals; `done(parity)` is what a wait for a phase of that parity sees."""

    def __init__(self, count=1):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def done(self, parity):
        return (self.phase & 1) != parity


def run_cta(pieces, seed):
    """One CTA of attn_tc_kernel (csrc/attention_tc.cu, many rows): the warp that issues products, the two groups that make
    probabilities, the two that load queries, and a tensor pipe that completes what was issued in order and arbitrarily late.
    ``pieces``: (blocks, halves).  Every wait has to end, and what a reader finds behind it has to be what it waited for."""
    rng = random.Random(seed)
    turn, q_full, q_empty = ([Barrier(), Barrier()] for _ in range(3))
    p_full = [[Barrier(), Barrier()], [Barrier(), Barrier()]]
    issued = []                                   # the tensor pipe's queue
    s_of, o_of = [None, None], [None, None]       # (piece, block) that S and O of a half stand at
    q_of = [None, None]

    def wait(bar, parity):
        while not bar.done(parity):
            yield

    def multiply():
        pp, qp = [[0, 0], [0, 0]], [0, 0]
        for i, (n, halves) in enumerate(pieces):
            if n == 0:
                continue
            for h in range(halves):
                yield from wait(q_full[h], qp[h])
                qp[h] ^= 1
                assert q_of[h] == i
                issued.append(("s", h, (i, 0)))
                issued.append(("turn", h))
                if n == 1:
                    issued.append(("q", h))
            for b in range(n):
                for h in range(halves):
                    for part in range(2):
                        yield from wait(p_full[h][part], pp[h][part])
                        pp[h][part] ^= 1
                        issued.append(("o", h, (i, b, part)))
                    if b + 1 < n:
                        issued.append(("s", h, (i, b + 1)))
                    issued.append(("turn", h))
                    if b + 2 == n:
                        issued.append(("q", h))
                    yield
            for h in range(halves):
                yield from wait(p_full[h][1], pp[h][1])
                pp[h][1] ^= 1

    def softmax(h):
        phase = 0
        for i, (n, halves) in enumerate(pieces):
            if h >= halves or n == 0:
                continue
            for b in range(n):
                yield from wait(turn[h], phase)
                phase ^= 1
                assert s_of[h] == (i, b) and (b == 0 or o_of[h] == (i, b - 1, 1))
                for part in range(2):
                    p_full[h][part].arrive()
                    yield
            yield from wait(turn[h], phase)
            phase ^= 1
            assert o_of[h] == (i, n - 1, 1)
            p_full[h][1].arrive()
            for _ in range(rng.randint(0, 5)):    # O is being read
                yield
                assert o_of[h] == (i, n - 1, 1)

    def queries(h):
        used = 0
        for i, (n, halves) in enumerate(pieces):
            if h >= halves or n == 0:
                continue
            yield from wait(q_empty[h], (used & 1) ^ 1)
            used += 1
            q_of[h] = i
            q_full[h].arrive()
            yield

    def pipe():
        if issued:
            what = issued.pop(0)
            if what[0] == "s":
                s_of[what[1]] = what[2]
            elif what[0] == "o":
                o_of[what[1]] = what[2]
            else:
                (turn if what[0] == "turn" else q_empty)[what[1]].arrive()

    roles = [multiply(), softmax(0), softmax(1), queries(0), queries(1)]
    speed = [rng.random() + 0.03 for _ in range(6)]
    for _ in range(200000):
        if not any(roles):
            return
        k = rng.choices(range(6), speed)[0]
        if k == 5:
            pipe()
        elif roles[k]:
            try:
                next(roles[k])
            except StopIteration:
                roles[k] = None
    raise AssertionError(f"a wait does not end: {pieces}")


def test_barriers_of_the_tensor_core_kernel():
    for seed in range(400):
        rng = random.Random(seed)
        run_cta([(rng.choice([0, 1, 1, 2, 3, 5]), rng.choice([1, 2])) for _ in range(rng.randint(1, 6))], seed)
