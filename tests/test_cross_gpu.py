"""Attention to an encoder's states (pkv_cross_*) against the definition in 64 bits."""
import pytest

from tests.segment_util import Step

pytestmark = pytest.mark.gpu

QWEN, TINY, WIDE, PAIRED = (14, 2, 64), (32, 4, 64), (32, 8, 128), (16, 16, 64)


def run(pkv, step, **kw):
    plan = pkv.CrossPlan(step.n, len(step.q_len), step.qh, step.kvh, step.hd, step.bs, step.q.dtype, num_blocks=step.num_blocks)
    plan.build_host(step.q_len, step.kv_len, q_start=step.q_start)
    plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.out, step.scale, **kw)
    return plan


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("geom", [PAIRED, WIDE, QWEN, (48, 1, 64), (20, 1, 128)])
@pytest.mark.parametrize("q_len,kv_len", [
    ([1], [200]), ([4], [1]), ([130], [128]), ([5], [127]), ([300], [129]), ([9, 4, 33], [1500, 64, 16]), ([17], [5000]),
])
def test_tiles(pkv, torch_cuda, monkeypatch, dtype, geom, q_len, kv_len):
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    step = Step(torch_cuda, dtype, geom, q_len, kv_len, 16, seed=len(q_len) * 100 + q_len[0])
    plan = run(pkv, step)
    assert plan.plan.n_tiles > 0
    step.check(pkv)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("geom", [PAIRED, TINY, WIDE, (40, 2, 64), (6, 3, 40), (4, 2, 256)])
@pytest.mark.parametrize("q_len,kv_len", [
    ([1], [1]), ([1] * 40, [1 + 37 * i for i in range(40)]), ([1, 2, 3, 1], [700, 0, 65, 3000]),
    ([0, 60, 1, 0, 7, 200, 2], [100, 333, 1000, 0, 0, 1, 2049]),
])
@pytest.mark.parametrize("tiles", ["", "1"])
def test_ragged(pkv, torch_cuda, monkeypatch, tiles, dtype, geom, q_len, kv_len):
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    step = Step(torch_cuda, dtype, geom, q_len, kv_len, 16, seed=len(q_len))
    run(pkv, step)
    step.check(pkv)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bs", [1, 8, 24, 32, 64, 128, 512])
def test_block_sizes(pkv, torch_cuda, monkeypatch, dtype, bs):
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    for geom in (QWEN, WIDE):
        step = Step(torch_cuda, dtype, geom, [40, 1, 6, 150], [700, 901, 33, 128], bs, seed=bs)
        run(pkv, step)
        step.check(pkv)


def test_rows_of_no_sequence_stay(pkv, torch_cuda):
    step = Step(torch_cuda, "bf16", TINY, [50, 1, 9], [300, 77, 1000], 16, seed=3, q_start=[70, 3, 20], rows=140)
    run(pkv, step)
    step.check(pkv)


def test_large_scores_and_rising_maxima(pkv, torch_cuda, monkeypatch):
    """Rows whose maximum grows tile by tile, so that the accumulator is rescaled again and again."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    for geom in (PAIRED, WIDE):
        step = Step(torch, "bf16", geom, [140, 12], [1500, 900], 16, seed=4, sharp=6.0)
        for s in range(2):
            k = step.kc[step.slots[s]].float()
            ramp = torch.linspace(0.05, 3.0, k.shape[0], device="cuda")[:, None]
            step.kc[step.slots[s]] = (k.abs() * ramp).to(step.kc.dtype)
        step.q.abs_()
        run(pkv, step)
        step.check(pkv)


def test_scores_of_minus_infinity(pkv, torch_cuda, monkeypatch):
    """Keys that the values of K themselves shut out (weight zero), the whole first key tile of them and more."""
    torch = torch_cuda
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    for geom in (PAIRED, WIDE):
        for shut in (64, 128, 300):
            step = Step(torch, "bf16", geom, [150, 9], [1500, 700], 16, seed=shut)
            step.q.view(step.n, step.qh, step.hd)[:, :, 0] = 1.0
            for s in range(2):
                step.kc.view(-1, step.kvh, step.hd)[step.slots[s][:shut], :, 0] = -float("inf")
            run(pkv, step)
            for s in range(2):
                step.slots[s] = step.slots[s][shut:]             # the definition over the other keys: these add exact zeros
            step.check(pkv)


def test_many_items_on_every_block(pkv, torch_cuda):
    """More items than blocks: queues of several items each, of both kinds, with odd and even numbers of key tiles."""
    lens = [300 + 61 * (i % 7) for i in range(30)]
    step = Step(torch_cuda, "bf16", PAIRED, [130 + 40 * (i % 5) for i in range(30)], lens, 16, seed=5)
    plan = run(pkv, step)
    assert plan.plan.n_tiles > 148
    step.check(pkv)


def test_captured_and_on_a_side_stream(pkv, torch_cuda):
    torch = torch_cuda
    step = Step(torch, "bf16", WIDE, [1, 60, 2], [900, 700, 0], 16, seed=6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan = run(pkv, step)
    side.synchronize()
    step.check(pkv)
    first = step.out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(2):
            plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.out, step.scale)
    for _ in range(3):
        step.out.copy_(step.mark)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step.out, first)
    # another layer's tensors through the same plan
    other = Step(torch, "bf16", WIDE, [1, 60, 2], [900, 700, 0], 16, seed=7)
    plan.attention(other.q, other.kc, other.vc, other.block_tables, other.table_offset, other.out, other.scale)
    other.check(pkv)


def test_image_and_rebuilt_plan(pkv, torch_cuda):
    torch = torch_cuda
    step = Step(torch, "f16", TINY, [5, 1, 40], [600, 80, 129], 16, seed=8)
    plan = pkv.CrossPlan(step.n, 3, *TINY, 16, step.q.dtype)
    plan.build_host([1, 1, 1], [3, 3, 3])
    torch.cuda.synchronize()
    n = plan.build_host_image(step.q_len, step.kv_len)
    plan.workspace.fill_(255)
    plan.workspace[:n].copy_(plan.staging[:n])
    plan.attention(step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.out, step.scale)
    step.check(pkv)


def test_python_refusals(pkv, torch_cuda):
    torch = torch_cuda
    step = Step(torch, "bf16", TINY, [5], [60], 16, seed=9)
    plan = run(pkv, step)
    args = [step.q, step.kc, step.vc, step.block_tables, step.table_offset, step.out]
    with pytest.raises(TypeError):
        plan.attention(step.q.float(), *args[1:], step.scale)
    with pytest.raises(ValueError):
        plan.attention(step.q[:3], *args[1:], step.scale)
    with pytest.raises(ValueError):
        plan.attention(step.q.cpu(), *args[1:], step.scale)
    with pytest.raises(TypeError):
        plan.attention(*args[:3], step.block_tables.long(), *args[4:], step.scale)
    with pytest.raises(ValueError):
        plan.build_host([5, 1], [60, 3])
    with pytest.raises(ValueError):
        plan.attention(*args[:4], step.table_offset[:0], step.out, step.scale)
    fresh = pkv.CrossPlan(5, 1, *TINY, 16, step.q.dtype)
    with pytest.raises(pkv.PkvError):
        fresh.attention(*args, step.scale)                       # never built
    with pytest.raises(pkv.PkvError):
        plan.attention(*args, 0.0)


@pytest.mark.parametrize("dtype,tiles", [("bf16", "1"), ("bf16", "0"), ("f32", "")])
def test_pools_of_more_than_four_billion_elements(pkv, torch_cuda, monkeypatch, dtype, tiles):
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    step = Step(torch_cuda, dtype, WIDE, [70, 1, 3], [500, 900, 129], 16, seed=20)
    step.move_behind(2 ** 32 // (8 * 128 * 16))
    run(pkv, step)
    step.check(pkv)


def test_q_of_more_than_two_billion_elements(pkv, torch_cuda):
    """First and last rows of one long sequence."""
    torch = torch_cuda
    qh, kvh, hd = WIDE
    n, keys = 530001, 200
    small = Step(torch, "bf16", WIDE, [200], [keys], 16, seed=21)
    q, out = torch.empty((n, qh * hd), device="cuda", dtype=torch.bfloat16), torch.empty((n, qh * hd), device="cuda", dtype=torch.bfloat16)
    q.normal_()
    q[:100], q[-100:] = small.q[:100], small.q[100:]
    plan = pkv.CrossPlan(n, 1, qh, kvh, hd, 16, q.dtype, num_blocks=small.num_blocks).build_host([n], [keys])
    plan.attention(q, small.kc, small.vc, small.block_tables, small.table_offset, out, small.scale)
    small.out = torch.cat([out[:100], out[-100:]])
    small.check(pkv)
