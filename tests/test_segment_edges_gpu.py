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
