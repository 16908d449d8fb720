"""The pinned buffers that plans are uploaded from: a stream runs an upload when it gets there, and until then the buffer
holds what was planned for it, whatever is planned next."""
import ctypes as C
import gc
import importlib

import numpy as np
import pytest


class Uploads:
    """Stands in for the GPU: copies run when somebody waits for the event behind them, or at the end."""

    def __init__(self, real):
        self.real, self.pending, self.done, self.events = real, [], [], 0

    def __getattr__(self, name):
        return getattr(self.real, name)

    def pkv_cross_plan_host(self, *a):
        *lengths_and_sizes, staging, staging_bytes, _, ws_bytes, _, plan = a
        st = self.real.pkv_cross_plan_host_image(*lengths_and_sizes, staging, staging_bytes, ws_bytes, plan)
        self.pending.append((staging, plan._obj.image_bytes, C.string_at(staging, plan._obj.image_bytes)))
        return st

    def pkv_prefix_plan_host(self, *a):
        *lengths_and_sizes, staging, staging_bytes, _, ws_bytes, _, plan = a
        st = self.real.pkv_prefix_plan_host_image(*lengths_and_sizes, staging, staging_bytes, ws_bytes, plan)
        self.pending.append((staging, plan._obj.image_bytes, C.string_at(staging, plan._obj.image_bytes)))
        return st

    def pkv_decode_plan_host(self, *a):
        *sizes, staging, staging_bytes, _, ws_bytes, _, plan = a
        n = C.c_size_t(0)
        st = self.real.pkv_decode_plan_host_image(*sizes, staging, staging_bytes, ws_bytes, plan, C.byref(n))
        self.pending.append((staging, n.value, C.string_at(staging, n.value)))
        return st

    def run(self, up_to=None):
        while self.pending and (up_to is None or len(self.done) < up_to):
            staging, n, planned = self.pending.pop(0)
            self.done.append(C.string_at(staging, n) == planned)

    def mark(self, event, stream, device):
        return len(self.done) + len(self.pending)

    def passed(self, event, wait):
        if wait:
            self.run(event)
        return len(self.done) >= event


@pytest.fixture
def uploads(pkv, monkeypatch):
    kernels = importlib.import_module("llm-engine_b200.kernels")
    fake = Uploads(pkv.lib())
    monkeypatch.setattr(kernels._lib, "lib", lambda: fake)
    monkeypatch.setattr(kernels, "_ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(kernels, "_this_device", lambda device: None)
    monkeypatch.setattr(kernels, "_stream", lambda stream: 0)
    monkeypatch.setattr(kernels, "_stream_of", lambda stream, device: 0)
    monkeypatch.setattr(kernels, "_mark", fake.mark, raising=False)
    monkeypatch.setattr(kernels, "_passed", fake.passed, raising=False)
    yield fake
    fake.run()
    left = getattr(kernels, "_Staging", None)
    if left is not None:
        left._left.clear()


def cross(pkv, torch, n):
    ws = torch.zeros(pkv.lib().pkv_cross_workspace_bytes(n, 14, 2, 64), dtype=torch.uint8)
    return pkv.CrossPlan(n, n, 14, 2, 64, 16, torch.bfloat16, workspace=ws)


def prefix(pkv, torch, n):
    ws = torch.zeros(pkv.lib().pkv_prefix_workspace_bytes(n, 14, 2, 64), dtype=torch.uint8)
    return pkv.PrefixPlan(n, 14, 2, 64, 16, torch.bfloat16, workspace=ws)


def test_decode_plan_made_anew_or_dropped_while_its_upload_is_pending(pkv, uploads, monkeypatch):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    ws = torch.zeros(pkv.decode_workspace_bytes(40, 14, 2, 64), dtype=torch.uint8)
    for step in range(3):
        plan = pkv.DecodePlan(40, 14, 2, 64, workspace=ws)
        for again in range(2):
            plan.build_host([100 + 170 * i + 1000 * step + again for i in range(40)])
        del plan
        gc.collect()
    plan = pkv.DecodePlan(40, 14, 2, 64, workspace=ws).build_host([5000] * 40)
    plan.build_host_image([70] * 40)
    uploads.run()
    assert uploads.done == [True] * 7


def test_plan_made_anew_while_its_upload_is_pending(pkv, uploads):
    torch = pytest.importorskip("torch")
    plan, other = cross(pkv, torch, 40), prefix(pkv, torch, 40)
    for step in range(3):
        plan.build_host([1] * 40, [100 + 17 * i + step for i in range(40)])
        other.build_host([900 + i + step for i in range(40)], 512)
    plan.build_host_image([1] * 40, [50] * 40)
    other.build_host_image([50] * 40, 0)
    uploads.run()
    assert uploads.done == [True] * 6


def test_dropped_plan_keeps_its_bytes_until_the_upload(pkv, uploads):
    torch = pytest.importorskip("torch")
    kept = []
    for step in range(4):
        plan = prefix(pkv, torch, 64)
        plan.build_host([900 + i + step for i in range(64)], 512)
        kept.append(plan.staging.data_ptr())
        del plan
        gc.collect()
    assert len(set(kept)) == 4, "bytes of a pending upload were handed out again"
    uploads.run()
    assert uploads.done == [True] * 4
    kernels = importlib.import_module("llm-engine_b200.kernels")
    assert len(kernels._Staging._left) == 4
    again = prefix(pkv, torch, 64)                           # asks for its bytes: the uploads have run, the others are given back
    assert len(kernels._Staging._left) == 0 and again.staging.numel() > 0


def test_event_of_nobody_is_refused(pkv):
    assert pkv.lib().pkv_event_passed(None, 0) == pkv._lib.PKV_E_ARG
