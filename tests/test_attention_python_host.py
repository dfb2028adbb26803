"""Python side of the attention plan, its wrapper and the layout, without a GPU: streams, lifetimes, devices, arguments.  The library and
the streams are stand-ins that write down what is asked of them."""
import contextlib

import pytest
import torch

from sarathi_serve_b200 import _native as N
from sarathi_serve_b200 import attention_ops, attention_wrapper, kv_cache_ops


class Stream:
    def __init__(self, number):
        self.cuda_stream, self.waited = number, []

    def wait_stream(self, other):
        self.waited.append(other)


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *a: 256
        return lambda *a: self.calls.append(name) or 0


class Machine:
    """The current stream, and which memory was recorded on which one."""

    def __init__(self):
        self.streams = [Stream(0), Stream(7), Stream(9)]
        self.now, self.recorded, self.capturing = self.streams[0], [], False
        self.library, self.device = Library(), 0

    @contextlib.contextmanager
    def on(self, stream):
        before, self.now = self.now, stream
        yield
        self.now = before

    def has(self, t, stream):
        return any(at == t.untyped_storage().data_ptr() and s is stream for at, s in self.recorded)


@pytest.fixture
def machine(monkeypatch):
    m = Machine()
    monkeypatch.setattr(N, "lib", lambda: m.library)
    monkeypatch.setattr(N, "require_cuda", lambda *t: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: m.device)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(N, "stream_ptr", lambda: m.now.cuda_stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: m.now)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: m.capturing)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: m.recorded.append((t.untyped_storage().data_ptr(), s)))
    return m


def plan():
    return attention_ops.AttentionPlan(2, 1, 64, 16, torch.float16, 4, 8, device=torch.device("cpu"))


def arrays():
    i = lambda n: torch.zeros(n, dtype=torch.int32)
    return dict(qo_indptr=i(3), kv_lens=i(2), kv_indptr=i(3), kv_indices=i(6))


def test_a_list_of_pages_is_recorded_where_it_is_read(machine):
    """Lists made on a side stream, the plan always on the main one: each list stays until the main stream has read it."""
    p = plan()
    lists = [arrays() for _ in range(3)]
    for a in lists:
        p.update(**a)
    assert all(machine.has(a["kv_indices"], machine.streams[0]) for a in lists)


def test_a_plan_used_first_on_another_stream_than_it_was_made_on(machine):
    """Its memory may still be in use by what the first stream did before, and may be given away while the second one works."""
    main, side, _ = machine.streams
    p = plan()
    with machine.on(side):
        p.update(**arrays())
    assert side.waited == [main]
    assert all(machine.has(t, side) for t in (p.buffer, p.workspace, p.kv_indices))


def test_a_plan_that_moves_between_streams(machine):
    main, side, third = machine.streams
    p = plan()
    a, b = arrays(), arrays()
    p.update(**a)
    with machine.on(side):
        p.stream()
        assert side.waited == [main] and machine.has(a["kv_indices"], side)
        p.update(**b)
    with machine.on(third):
        p.stream()
    assert third.waited == [side] and machine.has(b["kv_indices"], side) and machine.has(b["kv_indices"], third)
    assert not machine.has(a["kv_indices"], third)


def test_a_captured_call_leaves_order_and_lifetimes_to_the_caller(machine):
    main, side, _ = machine.streams
    p = plan()
    p.update(**arrays())
    machine.recorded.clear()
    machine.capturing = True
    with machine.on(side):
        p.update(**arrays())
    machine.capturing = False
    assert not machine.recorded and not side.waited and p.stream() == main.cuda_stream


def test_a_wrapper_that_is_used_on_another_stream_than_it_was_made_on(machine):
    """All that its kernels read there stays until they have: caches, layout, the step's lengths and tables."""
    main, side, _ = machine.streams
    w = attention_wrapper.PagedAttentionWrapper(2, 1, 64, 16, 5, 2, torch.float16, 4, 8, 3, device=torch.device("cpu"))
    i = lambda *s: torch.ones(*s, dtype=torch.int32)
    with machine.on(side):
        w.begin_forward(i(2), i(2), i(2, 1), 4)
    assert side.waited == [main]
    for t in (*w.kv_caches, *w.layout, w.query_lens, w.context_lens, w.block_tables, w.plan.buffer, w.plan.workspace):
        assert machine.has(t, side)


def test_a_wrapper_that_goes_back_and_forth_between_streams(machine):
    """Every change waits for the stream before; its memory is recorded once a stream, not every time."""
    main, side, _ = machine.streams
    w = attention_wrapper.PagedAttentionWrapper(2, 1, 64, 16, 5, 40, torch.float16, 4, 8, 3, device=torch.device("cpu"))
    i = lambda *s: torch.ones(*s, dtype=torch.int32)
    for _ in range(5):
        for stream in (side, main):
            with machine.on(stream):
                w.begin_forward(i(2), i(2), i(2, 1), 4)
    assert side.waited == [main] * 5 and main.waited == [side] * 5
    assert all(machine.has(t, side) for t in w.kv_caches) and len(machine.recorded) < 40 + 20


def test_a_wrapper_on_another_current_device_refuses_its_calls(machine):
    """Nothing is launched there, neither the append before the attention nor anything else, and the plan's stream stays."""
    w = attention_wrapper.PagedAttentionWrapper(2, 1, 64, 16, 5, 2, torch.float16, 4, 8, 3, device=torch.device("cpu"))
    i = lambda *s: torch.ones(*s, dtype=torch.int32)
    w.begin_forward(i(2), i(2), i(2, 1), 4)
    machine.library.calls.clear()
    machine.device = 1
    q, k = torch.zeros(4, 128, dtype=torch.float16), torch.zeros(4, 64, dtype=torch.float16)
    with machine.on(machine.streams[1]):
        for call in (lambda: w.fused_kv_append(0), lambda: w.forward(q, k, k, 0), lambda: w.begin_forward(i(2), i(2), i(2, 1), 4)):
            with pytest.raises(RuntimeError, match="current device"):
                call()
    assert not machine.library.calls and not machine.streams[1].waited


def test_numbers_that_do_not_fit_32_bits(machine):
    """The library takes C ints, of which ctypes would keep the low half."""
    make = lambda **k: attention_ops.AttentionPlan(**{**dict(num_heads=2, num_kv_heads=1, head_dim=64, page_size=16, dtype=torch.float16,
                                                             max_requests=4, max_tokens=8, device=torch.device("cpu")), **k})
    for name in ("num_heads", "num_kv_heads", "head_dim", "page_size", "max_requests", "max_tokens"):
        with pytest.raises(RuntimeError, match=name):
            make(**{name: 2 ** 32 + 64})
    with pytest.raises(RuntimeError, match="window"):
        make(window=-2 ** 32 + 5)
    assert make(window=2 ** 32 + 100).shape.window == make(window=2 ** 63 - 1).shape.window == 2 ** 31 - 1   # (wide, not 100 and -1)
    assert make(window=None).shape.window == 0 and make(window=100).shape.window == 100
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for call in (lambda: kv_cache_ops.batch_layout(i(2), i(2), i(2, 3), 2 ** 32 + 16, 9, 8),
                 lambda: kv_cache_ops.resize_block_tables(i(2, 3), i(2), i(2), i(9), i(1), 2 ** 32 + 16),
                 lambda: kv_cache_ops.slots(i(2), i(2), i(3), i(3), 2 ** 32 + 16)):
        with pytest.raises(RuntimeError, match="page_size"):
            call()
    assert not machine.library.calls


def test_a_layout_whose_arrays_were_exchanged(machine):
    """What is written is what the tuple holds now, whichever of its tensors got other memory or another length since."""
    written = []
    machine.library.sb200_batch_layout = lambda *a: written.append(a) or 0
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    step = lambda out=None: kv_cache_ops.batch_layout(i(2), i(2), i(2, 3), 16, 9, 8, out=out)
    lay = step()
    arrays = lambda: [*(x for x in written[-1][9:13]), *(x for x in written[-1][14:18])]
    assert arrays() == [t.data_ptr() for t in lay]
    assert step(lay) is lay and arrays() == [t.data_ptr() for t in lay]
    for k, name in enumerate(lay._fields):
        old = lay[k].data_ptr()
        lay[k].data = torch.zeros_like(lay[k])
        assert lay[k].data_ptr() != old
        step(lay)
        assert arrays() == [t.data_ptr() for t in lay], name
        whole = lay[k].data
        lay[k].data = whole[:-1]
        with pytest.raises(RuntimeError, match="out."):
            step(lay)
        lay[k].data = whole
        step(lay)
    wide = lay._replace(kv_indices=i(10))
    step(wide)
    assert arrays() == [t.data_ptr() for t in wide] and written[-1][13] == 10
    with pytest.raises(RuntimeError, match="kv_indices"):
        step(lay._replace(kv_indices=i(5)))
