"""The attention backend with the layers that call it: a small model served in chunks and single tokens over a paged cache, eagerly and
from CUDA graphs, against plain causal attention over the whole prompt; block tables, layout, append and attention of a step
captured together."""
import pytest
import torch

from helpers import TOL, rel_err
from oracle import tp_layer_oracle as O
from sarathi_serve_b200 import synthetic as S

pytestmark = pytest.mark.gpu


@pytest.fixture()
def tp1():
    from sarathi_serve_b200 import parallel_state as ps
    torch.cuda.set_device(0)
    ps.destroy_model_parallel()
    ps.initialize_model_parallel(1)
    yield ps
    ps.destroy_model_parallel()


def build_model(case, layers=2, vocab=500):
    from sarathi_serve_b200.decoder_layer import LlamaModel
    cfg = case.hf_config()
    cfg.num_hidden_layers, cfg.vocab_size = layers, vocab
    old = torch.get_default_dtype()
    torch.set_default_dtype(case.dtype)
    try:
        model = LlamaModel(cfg)
    finally:
        torch.set_default_dtype(old)
    t = S.generate(case)
    for layer in model.layers:
        S.load_layer(layer, S.shard(t, 0, 1))
    g = torch.Generator().manual_seed(3)
    model.embed_tokens.weight.data.copy_(torch.randn(512, case.hidden_size, generator=g).to(case.dtype))
    return model, t


def whole_prompt(model, t, case, ids):
    """norm(hidden states) of every token, attention over the whole prompt in 64 bits, the rest as the oracle's layer."""
    cache = O.cos_sin_cache(case.head_dim, case.head_dim, case.max_position, case.rope_theta, case.dtype)
    p = S.shard(t, 0, 1)
    h = model.embed_tokens.weight.data.cpu()[ids]
    n, nq, nkv, hd = ids.numel(), case.num_heads, case.num_kv_heads, case.head_dim
    pos = torch.arange(n)
    for _ in model.layers:
        x = O.rms_norm(h, p["input_layernorm.weight"], case.rms_norm_eps)
        qkv = O.linear(x, p["self_attn.qkv_proj.weight"])
        q, k, v = qkv.split([nq * hd, nkv * hd, nkv * hd], dim=-1)
        O.rotary_embedding(pos, q, k, hd, cache, True)
        qd, kd, vd = (z.double().view(n, -1, hd).transpose(0, 1) for z in (q, k, v))
        kd, vd = kd.repeat_interleave(nq // nkv, 0), vd.repeat_interleave(nq // nkv, 0)
        s = (qd @ kd.transpose(1, 2)) * hd ** -0.5
        s = s.masked_fill(pos[None, :] > pos[:, None], float("-inf"))
        a = (torch.softmax(s, -1) @ vd).transpose(0, 1).reshape(n, nq * hd).to(case.dtype)
        h = h + O.linear(a, p["self_attn.o_proj.weight"])
        y = O.rms_norm(h, p["post_attention_layernorm.weight"], case.rms_norm_eps)
        h = h + O.linear(O.silu_and_mul(O.linear(y, p["mlp.gate_up_proj.weight"])), p["mlp.down_proj.weight"])
    return O.rms_norm(h, torch.ones(case.hidden_size, dtype=case.dtype), case.rms_norm_eps)


@pytest.mark.parametrize("case_name", ["mini_bf16", "mini_f16", "mini_f32"])
@pytest.mark.parametrize("mode", ["eager", "unfused", "graph"])
def test_a_model_served_in_chunks(tp1, case_name, mode):
    """Two prompts in chunks of several steps, then single tokens, mixed: every row is what the whole prompt gives."""
    from sarathi_serve_b200 import kv_cache_ops
    from sarathi_serve_b200.attention_wrapper import PagedAttentionWrapper
    from sarathi_serve_b200.model_runner import ModelGraphRunner, prepare_inputs
    case = S.CASES[case_name]
    model, t = build_model(case)
    page, blocks, pool = 16, 20, 64
    attn = PagedAttentionWrapper(case.num_heads, case.num_kv_heads, case.head_dim, page, pool, len(model.layers), case.dtype,
                                 max_requests=4, max_tokens=128, max_blocks=blocks)
    for c in attn.kv_caches:
        c.fill_(float("nan"))  # slots that nothing has been stored to
    g = torch.Generator().manual_seed(5)
    ids = [torch.randint(0, 500, (n,), generator=g) for n in (150, 61)]
    want = [whole_prompt(model, t, case, x) for x in ids]
    steps = [[(100, 0), (7, 0)], [(40, 100), (50, 7)], [(7, 140), (1, 57)], [(1, 147), (1, 58)], [(0, 148), (1, 59)], [(1, 148), (1, 60)],
             [(1, 149), (0, 61)]]
    # block tables on the GPU, pages as the requests grow
    table = torch.full((2, blocks), -1, dtype=torch.int32, device="cuda")
    have = torch.zeros(2, dtype=torch.int32, device="cuda")
    free = torch.randperm(pool, generator=g).to(torch.int32).cuda()
    num_free = torch.tensor([pool], dtype=torch.int32, device="cuda")
    runner = ModelGraphRunner(model, attn, buckets=(8, 64, 128)) if mode == "graph" else None
    for step in steps:
        new = torch.tensor([a for a, _ in step], dtype=torch.int32, device="cuda")
        before = torch.tensor([b for _, b in step], dtype=torch.int32, device="cuda")
        assert kv_cache_ops.resize_block_tables(table, have, new + before, free, num_free, page).tolist() == [1, 1]
        chunks = [(ids[r][b:b + a].tolist(), b) for r, (a, b) in enumerate(step)]
        tok, pos, n = prepare_inputs(chunks, [], "cuda")
        rows = tok.numel() if runner is None else runner.bucket_for(n)
        attn.begin_forward(new, before, table, rows)
        assert torch.equal(attn.positions[:n], pos[:n])
        if runner is not None:
            out = runner.run(tok[:n], pos[:n])
        else:
            with torch.inference_mode():
                if mode == "eager":
                    out = model(tok, pos, attn)
                else:
                    h = model.embed_tokens(tok)
                    for i, layer in enumerate(model.layers):
                        h = layer.forward_unfused(pos, h, i, attn)
                    out = model.norm(h)
        attn.end_forward()
        at = 0
        for r, (a, b) in enumerate(step):
            if a:
                assert rel_err(out[at:at + a], want[r][b:b + a]) <= TOL[case.dtype] * 1.5, (step, r)
            at += a
    # both requests end: all pages come back, none twice
    kv_cache_ops.resize_block_tables(table, have, torch.zeros_like(have), free, num_free, page)
    assert int(num_free) == pool and sorted(free.tolist()) == list(range(pool))


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_a_captured_step_with_other_lengths(dtype, hd):
    """Block tables, layout, plan, append and attention captured once; replays with other lengths give what eager calls give."""
    from sarathi_serve_b200 import attention_ops, kv_cache_ops
    n, T, page, pool, nq, nkv, blocks = 5, 80, 16, 400, 8, 2, 64
    g = torch.Generator().manual_seed(1)
    i32 = dict(dtype=torch.int32, device="cuda")
    qkv = torch.zeros(T, (nq + 2 * nkv) * hd, dtype=dtype, device="cuda")
    fill = torch.randn(pool, 2, page, nkv, hd, generator=g).to(dtype).cuda()

    def fresh():
        return dict(new=torch.zeros(n, **i32), before=torch.zeros(n, **i32), table=torch.full((n, blocks), -1, **i32),
                    have=torch.zeros(n, **i32), free=torch.arange(pool, **i32), count=torch.tensor([pool], **i32), cache=fill.clone(),
                    granted=torch.zeros(n, **i32), lens=torch.zeros(n, **i32))

    def step(s, plan, layout, out):
        torch.add(s["new"], s["before"], out=s["lens"])
        kv_cache_ops.resize_block_tables(s["table"], s["have"], s["lens"], s["free"], s["count"], page, granted=s["granted"])
        kv_cache_ops.batch_layout(s["new"], s["before"], s["table"], page, pool, T, out=layout)
        plan.update(layout)
        kv_cache_ops.append_rows(s["cache"], qkv[:, nq * hd:(nq + nkv) * hd], qkv[:, (nq + nkv) * hd:], layout.kv_slots)
        attention_ops.paged_attention(qkv[:, :nq * hd], s["cache"], plan, hd ** -0.5, out=out)

    def parts(s):
        plan = attention_ops.AttentionPlan(nq, nkv, hd, page, dtype, n, T)
        return plan, kv_cache_ops.batch_layout(s["new"], s["before"], s["table"], page, pool, T), torch.zeros(T, nq * hd, dtype=dtype, device="cuda")

    a, b = fresh(), fresh()
    pa, pb = parts(a), parts(b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(a, *pa)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(a, *pa)
    torch.cuda.current_stream().wait_stream(stream)
    lens = [0] * n
    for k in range(12):
        new = [[60, 1, 0, 7, 12], [1, 1, 70, 1, 0], [1, 0, 1, 1, 1]][k % 3]
        for s in (a, b):
            s["new"].copy_(torch.tensor(new, **i32))
            s["before"].copy_(torch.tensor(lens, **i32))
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(dtype))
        graph.replay()
        step(b, *pb)
        lens = [x + y for x, y in zip(lens, new)]
        used = sum(new)
        assert torch.equal(pa[2][:used], pb[2][:used]) and torch.isfinite(pa[2].float()).all()
        for name in ("table", "have", "free", "count", "granted"):
            assert torch.equal(a[name], b[name]), name
        assert torch.equal(a["cache"], b["cache"])


def test_two_plans_on_two_streams():
    """Every plan has its own buffers: calls of different plans may overlap."""
    from sarathi_serve_b200 import attention_ops
    from test_gpu_attention import make, plan_of
    jobs = []
    for seed, batch in ((1, [(1, 3000), (200, 500)]), (2, [(90, 1000), (1, 700), (1, 64)])):
        c = make(seed, torch.bfloat16, 8, 2, 128, 16, batch)
        plan, layout = plan_of(c)
        jobs.append((c, plan, layout, attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    outs = [[], []]
    for _ in range(20):
        for i, (c, plan, _, _) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                outs[i].append(attention_ops.paged_attention(c["q"], c["cache"], plan, 0.1))
    torch.cuda.synchronize()
    for i, (_, _, _, want) in enumerate(jobs):
        assert all(torch.equal(o, want) for o in outs[i])


def test_a_plan_used_on_another_stream_than_it_was_made_on():
    """The plan, and the wrapper's index arrays, are still being written when the other stream's call is issued: it waits."""
    from sarathi_serve_b200 import attention_ops, kv_cache_ops
    from sarathi_serve_b200.attention_wrapper import PagedAttentionWrapper
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    w = PagedAttentionWrapper(8, 2, 128, 16, 64, 1, torch.bfloat16, max_requests=3, max_tokens=128, max_blocks=20)
    g = torch.Generator().manual_seed(2)
    cache = torch.randn(w.kv_caches[0].shape, generator=g).bfloat16().cuda()
    q, k, v = (torch.randn(128, n, generator=g).bfloat16().cuda() for n in (1024, 256, 256))
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(3, 20)
    steps = [(i([100, 1, 3]), i([20, 300, 0]), table), (i([1, 1, 90]), i([120, 7, 200]), table.flip(0).contiguous())]
    want = []
    for s in steps:
        w.kv_caches[0].copy_(cache)
        w.begin_forward(*s, 128)
        want.append(w.forward(q, k, v, 0, 0.1))
    w.kv_caches[0].copy_(cache)
    other = torch.cuda.Stream()
    a, b = torch.randn(2, 4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for s, x in zip(steps, want):
        for _ in range(20):
            a = torch.tanh(a @ b)  # some milliseconds on the current stream
        w.begin_forward(*s, 128)
        with torch.cuda.stream(other):
            got = w.forward(q, k, v, 0, 0.1)
            w.kv_caches[0].copy_(cache)
            assert torch.equal(got, x)
    lay = kv_cache_ops.batch_layout(*steps[0], 16, 64, 128)
    plan = attention_ops.AttentionPlan(8, 2, 128, 16, torch.bfloat16, 3, 128)
    torch.cuda.synchronize()
    for _ in range(20):
        a = torch.tanh(a @ b)
    plan.update(lay)
    with torch.cuda.stream(other):
        got = attention_ops.paged_attention(q, cache, plan, 0.1)
    plan.update(kv_cache_ops.batch_layout(*steps[1], 16, 64, 128))  # (back again: behind that call)
    torch.cuda.synchronize()
    assert torch.equal(got, attention_ops.paged_attention(q, cache, plan.update(lay), 0.1))


def test_a_step_with_fewer_pages_than_the_one_before():
    """Block tables that get narrower leave nothing behind: what a request is short of are zeros, not the pages of another."""
    from sarathi_serve_b200.attention_wrapper import PagedAttentionWrapper
    w = PagedAttentionWrapper(4, 2, 64, 16, 10, 1, torch.float16, max_requests=2, max_tokens=8, max_blocks=4)
    i = lambda x: torch.tensor(x, dtype=torch.int32)
    g = torch.Generator().manual_seed(8)
    w.kv_caches[0].copy_(torch.randn(w.kv_caches[0].shape, generator=g))
    w.begin_forward(i([1, 1]), i([60, 50]), i([[1, 2, 3, 4], [5, 6, 7, 8]]), 8)
    assert w.layout.kv_slots.tolist() == [4 * 32 + 12, 8 * 32 + 2] + [-1] * 6
    w.begin_forward(i([1, 1]), i([20, 50]), i([[1, 2], [5, 6]]), 8)  # the second has 51 tokens, and pages for 32
    assert w.layout.kv_slots.tolist() == [2 * 32 + 4] + [-1] * 7
    cache = w.kv_caches[0].clone()
    q = torch.randn(8, 4 * 64, generator=g).half().cuda()
    got = w.forward(q, torch.ones(8, 128, dtype=torch.float16, device="cuda"), torch.ones(8, 128, dtype=torch.float16, device="cuda"), 0, 0.1)
    assert torch.equal(w.kv_caches[0][7:], cache[7:]) and torch.equal(w.kv_caches[0][5:7], cache[5:7])
    keys = torch.cat([cache[5:7].transpose(0, 1).reshape(2, 32, 2, 64), torch.zeros(2, 19, 2, 64, dtype=torch.float16, device="cuda")], 1).double()
    k, v = keys.repeat_interleave(2, dim=2)
    q1 = q[1].double().view(4, 64)
    p = torch.softmax(0.1 * torch.einsum("hd,khd->hk", q1, k), -1)
    want, W = torch.einsum("hk,khd->hd", p, v).reshape(-1), torch.einsum("hk,khd->hd", p, v.abs()).reshape(-1)
    # roundings of the result and the probabilities; scores, powers of two and sums in fp32; probabilities below fp16's smallest step
    A = 0.1 * torch.einsum("hd,khd->hk", q1.abs(), k.abs()).max()
    tol = 2.0 ** -11 * (want.abs() + W) + 2 * ((80 * A + 67) * 2.0 ** -24 + 2.0 ** -21) * W + 51 * 2.0 ** -25 * v.abs().max()
    assert ((got[1].double() - want).abs() <= tol).all()


def test_wrapper_refusals():
    from sarathi_serve_b200 import attention_ops, kv_cache_ops
    from sarathi_serve_b200.attention_wrapper import PagedAttentionWrapper
    w = PagedAttentionWrapper(4, 2, 64, 16, 10, 1, torch.float16, max_requests=2, max_tokens=16, max_blocks=4)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    for bad in ((i(3), i(3), i(3, 4), 8), (i(2), i(2), i(2, 5), 8), (i(2), i(1), i(2, 4), 8), (i(2), i(2), i(1, 4), 8), (i(2), i(2), i(2, 4), 17),
                (i(2).long(), i(2), i(2, 4), 8), (i(2), i(2), i(2, 4), -1)):
        with pytest.raises(RuntimeError):
            w.begin_forward(*bad)
    with pytest.raises(RuntimeError, match="rows"):
        w.forward(*(torch.zeros(17, n, dtype=torch.float16, device="cuda") for n in (256, 128, 128)), 0)
    q, plan, cache = torch.zeros(8, 256, dtype=torch.float16, device="cuda"), w.plan, w.kv_caches[0]
    fresh = attention_ops.AttentionPlan(4, 2, 64, 16, torch.float16, 2, 16)
    for call in (lambda: attention_ops.paged_attention(q, cache, fresh, 1.0), lambda: attention_ops.paged_attention(q[:, :128], cache, plan, 1.0),
                 lambda: attention_ops.paged_attention(q.float(), cache, plan, 1.0), lambda: attention_ops.paged_attention(q, cache[:, :1], plan, 1.0),
                 lambda: attention_ops.paged_attention(q, cache.bfloat16(), plan, 1.0),
                 lambda: attention_ops.paged_attention(q, cache, plan, 1.0, out=q[:7]),
                 lambda: attention_ops.paged_attention(q, cache, plan, 1.0, lse=torch.zeros(8, 5, device="cuda")),
                 lambda: attention_ops.paged_attention(q, cache[:0], plan, 1.0),
                 lambda: attention_ops.paged_attention(torch.zeros(17, 256, dtype=torch.float16, device="cuda"), cache, plan, 1.0),
                 lambda: attention_ops.AttentionPlan(4, 3, 64, 16, torch.float16, 2, 16),
                 lambda: attention_ops.AttentionPlan(4, 2, 80, 16, torch.float16, 2, 16),
                 lambda: attention_ops.AttentionPlan(4, 2, 64, 16, torch.float64, 2, 16),
                 lambda: plan.update(qo_indptr=i(3), kv_lens=i(2)), lambda: plan.update(qo_indptr=i(2), kv_lens=i(2), kv_indptr=i(3), kv_indices=i(4)),
                 lambda: plan.update(qo_indptr=i(4), kv_lens=i(3), kv_indptr=i(4), kv_indices=i(4)),
                 lambda: kv_cache_ops.batch_layout(i(2).long(), i(2), i(2, 3), 16, 9, 8), lambda: kv_cache_ops.batch_layout(i(2), i(3), i(2, 3), 16, 9, 8),
                 lambda: kv_cache_ops.batch_layout(i(2), i(2), i(3, 2).t(), 16, 9, 8), lambda: kv_cache_ops.batch_layout(i(2), i(2), i(2, 3), 0, 9, 8),
                 lambda: kv_cache_ops.batch_layout(i(2), i(2), i(2, 3), 16, 9, 8, out=w.layout),
                 lambda: kv_cache_ops.resize_block_tables(i(2, 3), i(2), i(3), i(9), i(1), 16),
                 lambda: kv_cache_ops.resize_block_tables(i(2, 3), i(2), i(2), i(9), i(2), 16)):
        with pytest.raises(RuntimeError):
            call()
    torch.cuda.synchronize()
