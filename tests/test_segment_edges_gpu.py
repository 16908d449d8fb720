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
