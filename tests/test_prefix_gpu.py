"""Attention of a batch behind one prompt (pkv_prefix_*) against the definition in 64 bits, and against the
ordinary decode path."""
import numpy as np
import pytest

from tests.segment_util import Step

pytestmark = pytest.mark.gpu

QWEN, TINY, WIDE = (14, 2, 64), (32, 4, 64), (32, 8, 128)


def make(torch, dtype, geom, n, shared, tails, bs, seed, **kw):
    tails = (list(tails) * n)[:n]
    return Step(torch, dtype, geom, [1] * n, [shared + t for t in tails], bs, seed, shared=shared // bs * bs, **kw)


def run(pkv, step, shared, pos=None, **kw):
    torch = step.torch
    plan = pkv.PrefixPlan(step.n, step.qh, step.kvh, step.hd, step.bs, step.q.dtype, num_blocks=step.num_blocks)
    plan.build_host([k - 1 for k in step.kv_len] if pos is None else pos, shared)
    step.token_seq = torch.arange(step.n, device="cuda", dtype=torch.int32)
    plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.token_seq, step.out, step.scale, **kw)
    return plan


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("geom", [QWEN, TINY, WIDE, (5, 5, 64), (24, 1, 64), (16, 1, 128)])
@pytest.mark.parametrize("n,shared,tails", [
    (2, 16, [1]), (3, 128, [5, 1, 300]), (9, 1024, [16, 1, 77]), (40, 2000, [3, 500, 64, 1]), (130, 640, [20, 9]), (4, 9008, [40]),
])
@pytest.mark.parametrize("tiles", ["", "1"])
def test_against_definition(pkv, torch_cuda, monkeypatch, tiles, dtype, geom, n, shared, tails):
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    step = make(torch_cuda, dtype, geom, n, shared, tails, 16, seed=n)
    plan = run(pkv, step, shared)
    assert plan.plan.n_tiles > 0 or tiles == ""
    step.check(pkv)


@pytest.mark.parametrize("bs", [32, 64, 256])
def test_block_sizes(pkv, torch_cuda, monkeypatch, bs):
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    for geom in (TINY, WIDE):
        step = make(torch_cuda, "bf16", geom, 20, 1024, [1, 40, 333], bs, seed=bs)
        run(pkv, step, 1024)
        step.check(pkv)


@pytest.mark.parametrize("dtype,geom,bs", [("f32", QWEN, 16), ("f32", WIDE, 32), ("bf16", TINY, 8), ("f16", (6, 2, 96), 16), ("bf16", (6, 3, 40), 48)])
def test_geometries_without_tiles(pkv, torch_cuda, dtype, geom, bs):
    step = make(torch_cuda, dtype, geom, 11, 6 * bs * 8, [1, 40, 200], bs, seed=1)
    plan = run(pkv, step, 6 * bs * 8)
    assert plan.plan.n_tiles == 0
    step.check(pkv)


def test_no_prefix_and_one_token(pkv, torch_cuda):
    for n, shared in ((12, 0), (1, 512), (12, 15)):
        step = make(torch_cuda, "bf16", TINY, n, shared, [50, 900], 16, seed=n)
        run(pkv, step, shared)
        step.check(pkv)


@pytest.mark.parametrize("tiles", ["", "1"])
def test_tokens_inside_the_prefix(pkv, torch_cuda, monkeypatch, tiles):
    """A fully cached prompt computes its last token again: its position is the prefix's last, or any before."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    shared = 512
    for geom in (TINY, WIDE):
        step = make(torch, "bf16", geom, 8, shared, [0, 30, 0, 1, 0, 0, 16, 200], 16, seed=2)
        pos = [k - 1 for k in step.kv_len]
        pos[2], pos[4], pos[5] = 0, 300, 510
        run(pkv, step, shared, pos=pos)
        step.check(pkv, limits=[p + 1 for p in pos])


def test_prefix_that_ends_inside_a_block(pkv, torch_cuda, monkeypatch):
    """Keys the sequences agree on need not fill whole blocks or boxes."""
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    step = make(torch_cuda, "f16", TINY, 10, 1024, [30, 5, 100], 32, seed=3)
    for shared in (1001, 1023, 1024, 1008):
        step.out.copy_(step.mark)
        run(pkv, step, shared)
        step.check(pkv)


def test_against_the_ordinary_path_and_captured(pkv, torch_cuda, monkeypatch):
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    torch = torch_cuda
    step = make(torch, "bf16", WIDE, 70, 3000 // 16 * 16, [64, 1, 500], 16, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    shared = 3000 // 16 * 16
    with torch.cuda.stream(side):
        plan = run(pkv, step, shared)
    side.synchronize()
    step.check(pkv)
    first = step.out.clone()
    pos = torch.tensor([k - 1 for k in step.kv_len], dtype=torch.int32, device="cuda")
    ws = pkv.alloc_decode_workspace(step.n, step.qh, step.kvh, step.hd)
    other = step.mark.clone()
    pkv.launch_attention_decode(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.token_seq, pos, other, step.n, step.qh,
                                step.kvh, step.hd, 16, step.scale, workspace=ws)
    step.check(pkv, out=other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.token_seq, step.out, step.scale)
    for _ in range(3):
        step.out.copy_(step.mark)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step.out, first)


def test_two_plans_on_two_streams(pkv, torch_cuda, monkeypatch):
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    torch = torch_cuda
    steps = [make(torch, "bf16", TINY, 33 + i, 1600, [30, 5], 16, seed=5 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    plans = []
    for step, s in zip(steps, streams):
        with torch.cuda.stream(s):
            plans.append(run(pkv, step, 1600))
    torch.cuda.synchronize()
    for _ in range(20):
        for step, s, p in zip(steps, streams, plans):
            with torch.cuda.stream(s):
                p.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.token_seq, step.out, step.scale)
    for step in steps:
        step.check(pkv)


@pytest.mark.parametrize("tiles", ["", "1"])
def test_layer_with_norms_prefix_and_encoder(pkv, torch_cuda, monkeypatch, tiles):
    """One layer's run as a model makes it: norms + rotation + append of the step's tokens, attention over the shared
    prompt and their own keys, then attention to an encoder's states, every layer through the same two plans."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    qh, kvh, hd = TINY
    n, shared, bs = 24, 320, 16
    step = make(torch, "bf16", TINY, n, shared, [40, 7, 90], bs, seed=6)
    source = Step(torch, "bf16", TINY, [1] * n, [200 + 13 * i for i in range(n)], bs, seed=7)
    rng = np.random.default_rng(0)
    prefix = pkv.PrefixPlan(n, qh, kvh, hd, bs, step.q.dtype, num_blocks=step.num_blocks).build_host([k - 1 for k in step.kv_len], shared)
    cross = pkv.CrossPlan(n, n, qh, kvh, hd, bs, step.q.dtype, num_blocks=source.num_blocks).build_host(source.q_len, source.kv_len)
    seq = torch.arange(n, device="cuda", dtype=torch.int32)
    pos = torch.tensor([k - 1 for k in step.kv_len], dtype=torch.int32, device="cuda")
    slots = torch.stack([s[-1] for s in step.slots]).int()
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(600, device="cuda", dtype=torch.float64)[:, None] * inv
    cos, sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    for layer in range(2):
        rows = torch.from_numpy(rng.standard_normal((n, (qh + 2 * kvh) * hd))).cuda().to(step.q.dtype)
        q, k, v = rows.split([qh * hd, kvh * hd, kvh * hd], dim=1)
        w = torch.from_numpy(1 + 0.1 * rng.standard_normal((2, hd))).cuda().to(step.q.dtype)
        pkv.launch_qk_norm_rope_store_kv(q, k, v, w[0], w[1], 1e-6, pos, cos, sin, slots, step.q, step.kc, step.vc, n, qh, kvh, hd)
        prefix.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, seq, step.out, step.scale)
        source.q.copy_(step.out)
        cross.attention(source.q, source.kc, source.vc, source.block_tables, source.table_offset, source.out, source.scale)
        step.check(pkv)
        source.check(pkv)
        # what the attention read is what the norm pass is to have left
        x = q.double().view(n, qh, hd)
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w[0].double()
        c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
        a, b = y.chunk(2, -1)
        want = torch.cat([a * c - b * s, b * c + a * s], -1).flatten(1)
        size = torch.cat([(a * c).abs() + (b * s).abs()] * 2, -1).flatten(1) + torch.cat([(b * c).abs() + (a * s).abs()] * 2, -1).flatten(1)
        assert bool(((step.q.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).all())
        assert torch.equal(step.vc[slots.long()], v)


@pytest.mark.parametrize("tiles", ["1", "0"])
def test_pools_of_more_than_four_billion_elements(pkv, torch_cuda, monkeypatch, tiles):
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    step = make(torch_cuda, "bf16", WIDE, 12, 512, [1 + 30 * i for i in range(12)], 16, 20)
    step.move_behind(2 ** 32 // (8 * 128 * 16))
    run(pkv, step, 512)
    step.check(pkv)
