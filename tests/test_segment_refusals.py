"""What CrossPlan.attention and PrefixPlan.attention refuse before anything is enqueued.  No call of this file gets as far as a launch, so
the tensors may lie on the host: the checks see one device, that of the workspace."""
import importlib

import pytest


@pytest.fixture
def host(pkv, monkeypatch):
    torch = pytest.importorskip("torch")
    kernels = importlib.import_module("llm-engine_b200.kernels")
    monkeypatch.setattr(kernels, "_torch", torch)
    monkeypatch.setattr(kernels, "_ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(kernels, "_this_device", lambda device: None)
    monkeypatch.setattr(kernels, "_stream_of", lambda stream, device: 0)
    called = []
    monkeypatch.setattr(kernels, "_fn", lambda op, t: (op, lambda *a: called.append(op) or 0))
    return torch, called


def test_lengths_that_do_not_fit_are_refused(pkv, host):
    import numpy as np
    torch, _ = host
    ws = torch.zeros(1 << 22, dtype=torch.uint8)
    cross = pkv.CrossPlan(3, 3, 4, 2, 64, 16, torch.bfloat16, workspace=ws)
    prefix = pkv.PrefixPlan(3, 4, 2, 64, 16, torch.bfloat16, workspace=ws)
    good = cross.build_host_image([1] * 3, [5, 6, 7])
    for same in (np.array([5, 6, 7]), np.array([5, 6, 7], np.uint8), torch.tensor([5, 6, 7]), (5, 6, 7), np.arange(5, 8, dtype=np.uint64), np.array([5.0, 6.0, 7.0])):
        assert cross.build_host_image([1] * 3, same) == good
    every_second = np.array([5, 0, 6, 0, 7], np.int32)[::2]
    assert cross.build_host_image([1] * 3, every_second) == good and prefix.build_host_image(every_second, 0) > 0
    for bad in ([5, 6, 2 ** 32 + 7], np.array([5, 6, -2 ** 32]), np.array([5, 6, 2 ** 31]), np.array([2 ** 32 - 1] * 3, np.uint32), [5, 6, 7.5],
                np.array([5.0, 6.0, float("nan")]), ["5", "6", "7"]):
        for call in (lambda: cross.build_host_image([1] * 3, bad), lambda: cross.build_host_image(bad, [5, 6, 7]),
                     lambda: cross.build_host_image([1] * 3, [5, 6, 7], q_start=bad), lambda: prefix.build_host_image(bad, 0)):
            with pytest.raises(ValueError):
                call()


@pytest.mark.parametrize("kind", ["cross", "prefix"])
def test_pools_and_blocks_belong_together(pkv, host, kind):
    torch, called = host
    n, qh, kvh, hd, bs, blocks = 6, 4, 2, 64, 16, 30
    size = getattr(pkv.lib(), f"pkv_{kind}_workspace_bytes")(n, qh, kvh, hd)
    ws = torch.zeros(size, dtype=torch.uint8)
    if kind == "cross":
        plan = pkv.CrossPlan(n, n, qh, kvh, hd, bs, torch.bfloat16, num_blocks=blocks, workspace=ws)
        plan.build_host_image([1] * n, [100] * n)
    else:
        plan = pkv.PrefixPlan(n, qh, kvh, hd, bs, torch.bfloat16, num_blocks=blocks, workspace=ws)
        plan.build_host_image([100] * n, 64)
    q, out = (torch.zeros(n, qh * hd, dtype=torch.bfloat16) for _ in range(2))
    pool = torch.zeros(blocks, bs, kvh, hd, dtype=torch.bfloat16)
    index = [torch.zeros(n, dtype=torch.int32)] * (2 if kind == "cross" else 3)

    def call(k, v):
        plan.attention(q, k, v, *index, out, 0.125)

    call(pool, pool)
    assert len(called) == 1
    for k, v in ((pool, pool[:-1]), (pool[1:], pool), (pool[1:], pool[1:]), (pool[:0], pool[:0])):
        with pytest.raises(ValueError):
            call(k, v)
    assert len(called) == 1
    larger = torch.zeros(blocks + 3, bs, kvh, hd, dtype=torch.bfloat16)
    call(larger, larger)                                     # a pool beyond the plan's blocks is only not reached
    plan.plan.num_blocks = 0
    call(pool[1:], pool[1:])                                 # unknown
    assert len(called) == 3
