"""Corners of the unmasked attention forms (pkv_cross_*, pkv_prefix_*): scores that overflow for some rows of a warp only, outputs off
their natural alignment, plans made anew while earlier steps are under way."""
import pytest

from tests.segment_util import Step

pytestmark = pytest.mark.gpu

QWEN, TINY, WIDE, PAIRED = (14, 2, 64), (32, 4, 64), (32, 8, 128), (16, 16, 64)


def cross(pkv, step):
    plan = pkv.CrossPlan(step.n, len(step.q_len), step.qh, step.kvh, step.hd, step.bs, step.q.dtype, num_blocks=step.num_blocks)
    return plan.build_host(step.q_len, step.kv_len, q_start=step.q_start)


def attend(plan, step):
    plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.out, step.scale)


@pytest.mark.parametrize("geom", [PAIRED, TINY, WIDE])
@pytest.mark.parametrize("shut", [300, 520])
def test_rows_of_a_warp_without_a_finite_score_yet(pkv, torch_cuda, monkeypatch, geom, shut):
    """Every third token's scores overflow to -inf for the first `shut` keys; those of its neighbours, in the same warp, stay finite and
    rise from tile to tile, so that the accumulators are rescaled while the first have seen nothing yet."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    step = Step(torch, "bf16", geom, [150, 9], [1500, 700], 16, seed=shut)
    late = torch.arange(step.n, device="cuda") % 3 == 0
    q, k = step.q.view(step.n, step.qh, step.hd), step.kc.view(-1, step.kvh, step.hd)
    q[:, :, 0] = torch.where(late, 2.0 ** 100, 2.0 ** -100)[:, None].to(q.dtype)
    q[:, :, 1] = 16.0
    for rows in step.slots:
        k[rows, :, 0] = 0.0
        k[rows[:shut], :, 0] = -2.0 ** 100                   # times 2^100: beyond fp32; times 2^-100: -1
        k[rows, :, 1] = (torch.arange(len(rows), device="cuda") / 16.0).to(k.dtype)[:, None]
    plan = cross(pkv, step)
    assert plan.plan.n_tiles > 0 and plan.plan.n_items == 0
    attend(plan, step)
    torch.cuda.synchronize()
    rows, want, bound = step.expected()
    assert torch.equal(rows, torch.arange(step.n, device="cuda"))
    step.slots = [s[shut:] for s in step.slots]              # a weight of exp(-inf) is exactly none
    _, want_late, bound_late = step.expected()
    want, bound = torch.where(late[:, None], want_late, want), torch.where(late[:, None], bound_late, bound)
    bad = ~((step.out.double() - want).abs() <= bound)
    assert not bool(bad.any()), f"{int(bad.any(1)[late].sum())} late rows and {int(bad.any(1)[~late].sum())} others of {step.n}"
    assert pkv.debug_device_flags() == 0


def off_by(torch, t, elements):
    """The same values, `elements` past a 16-byte boundary."""
    store = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    at = store[elements:elements + t.numel()].view(t.shape)
    at.copy_(t)
    return at


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("geom", [(6, 2, 36), (4, 4, 20), (3, 1, 100)])
@pytest.mark.parametrize("elements", [1, 2, 3, 4])
def test_rows_of_other_than_16_byte_multiples_may_begin_anywhere(pkv, torch_cuda, dtype, geom, elements):
    """Heads of 8-byte multiples in tensors that are aligned to an element only; tokens cut in pieces and tokens without keys, which the
    merge writes."""
    torch = torch_cuda
    step = Step(torch, dtype, geom, [1, 2, 1], [3000, 0, 900], 16, seed=elements)
    for name in ("q", "kc", "vc", "out", "mark"):
        setattr(step, name, off_by(torch, getattr(step, name), elements))
    plan = cross(pkv, step)
    assert plan.plan.n_parts > 0 and plan.plan.n_merged > 2 * step.kvh
    attend(plan, step)
    step.check(pkv)

    step = Step(torch, dtype, geom, [1] * 3, [2500, 2401, 2900], 16, seed=elements, shared=2400)
    for name in ("q", "kc", "vc", "out", "mark"):
        setattr(step, name, off_by(torch, getattr(step, name), elements))
    plan = pkv.PrefixPlan(step.n, *geom, 16, step.q.dtype, num_blocks=step.num_blocks).build_host([k - 1 for k in step.kv_len], 2400)
    assert plan.plan.n_merged > 0
    plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, torch.arange(3, device="cuda", dtype=torch.int32), step.out,
                   step.scale)
    step.check(pkv)


def prefix_step(torch, geom, n, shared, tail, seed):
    step = Step(torch, "bf16", geom, [1] * n, [shared + tail + 3 * (i % 5) for i in range(n)], 16, seed=seed, shared=shared)
    step.token_seq = torch.arange(n, device="cuda", dtype=torch.int32)
    return step


def prefix_plan(pkv, step):
    return pkv.PrefixPlan(step.n, step.qh, step.kvh, step.hd, 16, step.q.dtype, num_blocks=step.num_blocks)


def attend_prefix(plan, step, **kw):
    plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.token_seq, step.out, step.scale, **kw)


BUSY = 100_000_000      # cycles, 50 ms and more: time for the host to plan the steps behind


@pytest.mark.parametrize("tiles", ["", "1"])
@pytest.mark.parametrize("drop", [False, True])
def test_plans_of_steps_that_the_gpu_has_not_reached(pkv, torch_cuda, monkeypatch, tiles, drop):
    """The host plans three steps ahead, through one object or through objects it drops."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    steps = [prefix_step(torch, TINY, 60, 640, 20 + 150 * i, seed=30 + i) for i in range(3)]
    sources = [Step(torch, "bf16", TINY, [1 + (j + i) % 4 for j in range(20)], [50 + 300 * i + 7 * j for j in range(20)], 16, seed=40 + i)
               for i in range(3)]
    rows = max(s.n for s in sources)
    plan, other = prefix_plan(pkv, steps[0]), pkv.CrossPlan(rows, 20, *TINY, 16, torch.bfloat16)
    for s in sources:                                            # every step as many rows: the last ones of no sequence
        extra = rows - s.n
        s.q, s.mark = (torch.cat([t, t[:extra]]) for t in (s.q, s.mark))
        s.out, s.n = s.mark.clone(), rows
    torch.cuda.synchronize()
    torch.cuda._sleep(BUSY)
    for step, source in zip(steps, sources):
        if drop:
            plan, other = prefix_plan(pkv, step), pkv.CrossPlan(rows, 20, *TINY, 16, torch.bfloat16)
        plan.num_blocks = step.num_blocks
        plan.build_host([k - 1 for k in step.kv_len], 640)
        other.build_host(source.q_len, source.kv_len)
        attend_prefix(plan, step)
        attend(other, source)
    for x in steps + sources:
        x.check(pkv)


def test_workspace_of_a_plan_dropped_on_another_stream(pkv, torch_cuda, monkeypatch):
    """Its memory is not handed out again while that stream's calls are to come."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    step = prefix_step(torch, TINY, 60, 640, 50, seed=50)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for named in (False, True):
        step.out.copy_(step.mark)
        plan = prefix_plan(pkv, step).build_host([k - 1 for k in step.kv_len], 640)
        size = plan.workspace.numel()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(BUSY)
            if not named:
                attend_prefix(plan, step)
        if named:
            attend_prefix(plan, step, stream=side)
        del plan
        others = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
        step.check(pkv)
        del others


def test_plans_around_a_capture(pkv, torch_cuda):
    """Made anew, made and dropped while a stream is being captured: nothing of it ends the capture."""
    torch = torch_cuda
    step = prefix_step(torch, TINY, 60, 640, 50, seed=60)
    pos = [k - 1 for k in step.kv_len]
    plan = prefix_plan(pkv, step).build_host(pos, 640)
    attend_prefix(plan, step)
    dropped = prefix_plan(pkv, step).build_host(pos, 640)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        del dropped
        plan.build_host(pos, 640)                                # its copy is a node of the graph
        attend_prefix(plan, step)
    for _ in range(2):
        step.out.copy_(step.mark)
        graph.replay()
        step.check(pkv)


def captured(torch, call):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


def replace_image(plan, n):
    plan.workspace[:n].copy_(plan.staging[:n])


OTHER_PLAN = 64


@pytest.mark.parametrize("geom,dtype,tiles", [(TINY, "bf16", "1"), (WIDE, "f16", "1"), (TINY, "bf16", "0"), (WIDE, "f32", ""),
                                              ((6, 2, 40), "f16", ""), ((20, 1, 64), "bf16", "1"), ((24, 1, 128), "f16", "0")])
def test_replay_over_another_steps_plan_does_nothing_and_says_so(pkv, torch_cuda, monkeypatch, geom, dtype, tiles):
    """A captured call is made for the counts of its step: over an image of others it leaves the output alone."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    monkeypatch.setenv("PKV_DECODE_CLUSTER", "0")
    n, shared = 70, 512
    step = Step(torch, dtype, geom, [1] * n, [shared + 10 + 29 * i for i in range(n)], 16, seed=70, shared=shared)
    step.token_seq = torch.arange(n, device="cuda", dtype=torch.int32)
    plan = prefix_plan(pkv, step).build_host([k - 1 for k in step.kv_len], shared)
    graph = captured(torch, lambda: attend_prefix(plan, step))
    step.out.copy_(step.mark)
    graph.replay()
    step.check(pkv)
    first = pkv._lib.SegmentPlan.from_buffer_copy(plan.plan)
    shorter = [shared + (k - shared) // 3 for k in step.kv_len]
    image = plan.build_host_image([k - 1 for k in shorter], shared)
    assert first.n_items != plan.plan.n_items
    replace_image(plan, image)
    step.out.copy_(step.mark)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(step.out, step.mark)
    assert pkv.debug_device_flags() == OTHER_PLAN
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(pkv.PkvError, match="0x40"):                  # told by the next call, which runs nothing
        attend_prefix(plan, step)
    attend_prefix(plan, step)                                        # the present plan, called for itself
    assert pkv.debug_device_flags() == OTHER_PLAN                    # (the device's own record of the replay before)
    step.check(pkv, limits=shorter)
    # the captured step's image again: the replay is whole again
    image = plan.build_host_image([k - 1 for k in step.kv_len], shared)
    replace_image(plan, image)
    step.out.copy_(step.mark)
    graph.replay()
    step.check(pkv)


def test_replay_over_an_image_of_the_same_layout(pkv, torch_cuda, monkeypatch):
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    step = Step(torch, "bf16", TINY, [40, 40], [383, 1000], 16, seed=71)
    plan = cross(pkv, step)
    graph = captured(torch, lambda: attend(plan, step))
    replace_image(plan, plan.build_host_image([40, 40], [300, 910]))
    step.out.copy_(step.mark)
    graph.replay()
    step.check(pkv, limits=[300, 910])


@pytest.mark.parametrize("geom,dtype", [(QWEN, "bf16"), (QWEN, "f32"), ((8, 2, 128), "f16")])
def test_replays_of_the_cluster_form(pkv, torch_cuda, geom, dtype):
    """Small steps read their positions only: captured once, they follow the images of later steps as long as every row has keys."""
    torch = torch_cuda
    n, shared, most = 3, 64, 700
    step = Step(torch, dtype, geom, [1] * n, [shared + most] * n, 16, seed=73, shared=shared)
    step.token_seq = torch.arange(n, device="cuda", dtype=torch.int32)
    plan = prefix_plan(pkv, step).build_host([shared + 399, shared + 410, shared + 415], shared)
    assert plan.plan.cluster > 0
    before = pkv.lib().pkv_debug_cluster_launches()
    graph = captured(torch, lambda: attend_prefix(plan, step))
    assert pkv.lib().pkv_debug_cluster_launches() == before + 2
    for grown in (0, 1, 60, 200, 284):
        pos = [shared + 399 + grown, shared + 410 + grown, shared + 415 + grown]
        replace_image(plan, plan.build_host_image(pos, shared))
        step.out.copy_(step.mark)
        graph.replay()
        step.check(pkv, limits=[p + 1 for p in pos])

    step = Step(torch, dtype, geom, [1] * n, [600, 500, 640], 16, seed=74)
    plan = cross(pkv, step)
    assert plan.plan.cluster > 0
    graph = captured(torch, lambda: attend(plan, step))
    replace_image(plan, plan.build_host_image([1] * n, [600, 0, 640]))       # a row without keys
    step.out.copy_(step.mark)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(step.out, step.mark) and pkv.debug_device_flags() == OTHER_PLAN
    replace_image(plan, plan.build_host_image([1] * n, [333, 20, 640]))
    graph.replay()
    step.check(pkv, limits=[333, 20, 640])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("geom", [(256, 1, 64), (256, 1, 128), (200, 1, 64), (129, 1, 128), (128, 1, 64), (130, 2, 64), (256, 2, 128)])
def test_many_query_heads_to_a_kv_head(pkv, torch_cuda, monkeypatch, dtype, geom):
    """Up to a whole tile of one token's heads; pairs of kv heads with a full group each."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    step = Step(torch, dtype, geom, [1, 3, 2], [700, 129, 1], 16, seed=80)
    plan = cross(pkv, step)
    assert plan.plan.n_tiles > 0 and plan.plan.n_items == 0
    attend(plan, step)
    step.check(pkv)
    step = prefix_step(torch, geom, 3, 256, 40, seed=81)
    plan = prefix_plan(pkv, step).build_host([k - 1 for k in step.kv_len], 256)
    assert plan.plan.n_tiles > 0
    attend_prefix(plan, step)
    step.check(pkv)


def test_streams_by_handle(pkv, torch_cuda):
    """Plans made and used on a stream named by its handle, the default stream's among them."""
    torch = torch_cuda
    side = torch.cuda.Stream()
    for handle in (side.cuda_stream, 0, side):
        step = prefix_step(torch, TINY, 20, 128, 50, seed=82)
        source = Step(torch, "bf16", TINY, [2] * 10, [77 * i for i in range(10)], 16, seed=83)
        plan = prefix_plan(pkv, step)
        other = pkv.CrossPlan(source.n, 10, *TINY, 16, torch.bfloat16)
        decode = pkv.DecodePlan(step.n, *TINY)
        pos = torch.tensor([k - 1 for k in step.kv_len], dtype=torch.int32, device="cuda")
        out = step.mark.clone()
        torch.cuda.synchronize()
        for _ in range(2):
            plan.build_host([k - 1 for k in step.kv_len], 128, stream=handle)
            other.build_host(source.q_len, source.kv_len, stream=handle)
            decode.build_host([k - 1 for k in step.kv_len], stream=handle)
            attend_prefix(plan, step, stream=handle)
            other.attention(source.q, source.kc, source.vc, source.block_tables, source.table_offset, source.out, source.scale, stream=handle)
            decode.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.token_seq, pos, out, 16, step.scale, stream=handle)
        step.check(pkv)
        source.check(pkv)
        step.check(pkv, out=out)


@pytest.mark.parametrize("geom", [(1, 1, 64), (1, 1, 128), (3, 3, 64), (5, 5, 128), (2, 1, 64)])
def test_few_heads(pkv, torch_cuda, monkeypatch, geom):
    """A kv head without a partner; a tile of 128 or 256 tokens."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    step = Step(torch, "bf16", geom, [257, 1, 128, 300], [1000, 129, 64, 2000], 16, seed=84)
    attend(cross(pkv, step), step)
    step.check(pkv)
    step = prefix_step(torch, geom, 300, 1024, 30, seed=85)
    attend_prefix(prefix_plan(pkv, step).build_host([k - 1 for k in step.kv_len], 1024), step)
    step.check(pkv)


@pytest.mark.parametrize("geom,n,shared", [(TINY, 60, 640), (WIDE, 70, 2048), (QWEN, 3, 64)])
@pytest.mark.parametrize("tiles", ["", "1", "0"])
def test_layers_back_to_back_over_the_same_buffers(pkv, torch_cuda, monkeypatch, geom, n, shared, tiles):
    """Every layer writes q, and its tokens' rows of the pools, where the layer before had them, with launches of this library alone
    between: each sees what its own norm pass left, launched eagerly or replayed, as when the layers run one by one."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    qh, kvh, hd = geom
    layers = 12
    step = prefix_step(torch, geom, n, shared, 90, seed=90)
    plan = prefix_plan(pkv, step).build_host([k - 1 for k in step.kv_len], shared)
    source = Step(torch, "bf16", geom, [1 + i % 3 for i in range(n)], [40 + 13 * i for i in range(n)], 16, seed=91)
    encoder = cross(pkv, source)
    g = torch.Generator(device="cuda").manual_seed(92)
    rows = torch.randn((layers, n, (qh + 2 * kvh) * hd), generator=g, device="cuda").to(step.q.dtype)
    parts = [r.split([qh * hd, kvh * hd, kvh * hd], dim=1) for r in rows]
    w = torch.ones(hd, device="cuda", dtype=step.q.dtype)
    pos = torch.tensor([k - 1 for k in step.kv_len], dtype=torch.int32, device="cuda")
    slots = torch.stack([s[-1] for s in step.slots]).int()
    angle = torch.rand((max(step.kv_len), hd // 2), generator=g, device="cuda") * 6.28
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
    outs, encs = ([torch.empty_like(x.mark) for _ in range(layers)] for x in (step, source))

    def layer(i):
        q, k, v = parts[i]
        pkv.launch_qk_norm_rope_store_kv(q, k, v, w, w, 1e-6, pos, cos, sin, slots, step.q, step.kc, step.vc, n, qh, kvh, hd)
        plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.token_seq, outs[i], step.scale)
        encoder.attention(source.q, source.kc, source.vc, source.block_tables, source.table_offset, encs[i], source.scale)

    want = []
    for i in range(layers):
        layer(i)
        torch.cuda.synchronize()
        step.out.copy_(outs[i])
        step.check(pkv)
        want.append((outs[i].clone(), encs[i].clone()))

    def run():
        for i in range(layers):
            layer(i)

    graph = captured(torch, run)
    for go in (run, graph.replay) * 4:
        for t in outs + encs:
            t.fill_(float("nan"))
        go()
        torch.cuda.synchronize()
        assert all(torch.equal(a, x) and torch.equal(b, y) for a, b, (x, y) in zip(outs, encs, want))
    assert pkv.debug_device_flags() == 0
