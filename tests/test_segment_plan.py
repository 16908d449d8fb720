"""The host planners of pkv_cross_* and pkv_prefix_*: every (row, key) pair is listed exactly once, partials and the
merge agree, the bounds for workspace and staging hold, and bad arguments are refused before anything is enqueued."""
import ctypes as C
import random

import numpy as np
import pytest

from tests.segment_util import Image, check_cover

GEOMS = [(14, 2, 64), (32, 4, 64), (32, 8, 128), (16, 16, 64), (20, 1, 128), (7, 7, 96), (48, 1, 64)]


class Buffers:
    def __init__(self, pkv, n, qh, kvh, hd, prefix):
        L = pkv.lib()
        self.ws = L.pkv_prefix_workspace_bytes(n, qh, kvh, hd) if prefix else L.pkv_cross_workspace_bytes(n, qh, kvh, hd)
        self.staging = np.zeros(L.pkv_segment_staging_bytes(n, qh, kvh), np.uint8)


def cross(pkv, q_len, kv_len, n, geom, bs=16, elem=2, q_start=None, b=None):
    qh, kvh, hd = geom
    b = b or Buffers(pkv, n, qh, kvh, hd, False)
    plan = pkv._lib.SegmentPlan()
    arr = [None if a is None else np.ascontiguousarray(a, np.int32) for a in (q_start, q_len, kv_len)]
    st = pkv.lib().pkv_cross_plan_host_image(*[None if a is None else a.ctypes.data for a in arr], len(q_len), n, qh, kvh, hd, bs, elem,
                                             b.staging.ctypes.data, b.staging.size, b.ws, C.byref(plan))
    return st, plan, b


def prefix(pkv, pos, prefix_len, geom, bs=16, elem=2, b=None):
    qh, kvh, hd = geom
    n = len(pos)
    b = b or Buffers(pkv, n, qh, kvh, hd, True)
    plan = pkv._lib.SegmentPlan()
    p = np.ascontiguousarray(pos, np.int32)
    st = pkv.lib().pkv_prefix_plan_host_image(p.ctypes.data, n, prefix_len, qh, kvh, hd, bs, elem, b.staging.ctypes.data, b.staging.size, b.ws,
                                              C.byref(plan))
    return st, plan, b


def log_int(r, lo, hi):
    return int(round(lo * (hi / lo) ** r.random()))


@pytest.mark.parametrize("tiles", ["", "1", "0"])
@pytest.mark.parametrize("seed", range(60))
def test_cross_covers_every_pair(pkv, monkeypatch, seed, tiles):
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    r = random.Random(seed)
    geom = r.choice(GEOMS)
    n_seqs = log_int(r, 1, 60)
    top_q, top_k = log_int(r, 1, 600), log_int(r, 1, 9000)
    q_len = [r.choice([0, 1, r.randrange(1, top_q + 1), top_q]) for _ in range(n_seqs)]
    kv_len = [r.choice([0, 1, 127, 128, 129, r.randrange(1, top_k + 1), top_k]) for _ in range(n_seqs)]
    order = r.sample(range(n_seqs), n_seqs)
    start, at = [0] * n_seqs, r.randrange(3)
    for s in order:
        start[s] = at
        at += q_len[s] + r.randrange(2)
    n = max(at, 1)
    st, plan, b = cross(pkv, q_len, kv_len, n, geom, bs=r.choice([16, 64, 8, 48]), elem=r.choice([2, 2, 2, 4]), q_start=start)
    assert st == 0, pkv._lib.last_error()
    assert plan.workspace_bytes <= b.ws and plan.image_bytes <= b.staging.size
    image = Image(b.staging, plan)
    want = {start[s] + i: kv_len[s] for s in range(n_seqs) for i in range(q_len[s])}
    check_cover(image, plan, want)
    for s in range(n_seqs):
        for i in range(q_len[s]):
            assert image.seq[start[s] + i] == s and image.pos[start[s] + i] == kv_len[s] - 1
    assert (np.delete(image.seq, list(want)) == -1).all()


@pytest.mark.parametrize("tiles", ["", "1", "0"])
@pytest.mark.parametrize("seed", range(60))
def test_prefix_covers_every_pair(pkv, monkeypatch, seed, tiles):
    monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
    r = random.Random(1000 + seed)
    geom = r.choice(GEOMS)
    n = log_int(r, 1, 700)
    shared = r.choice([0, 1, 15, 16, 17, log_int(r, 16, 20000), 16 * log_int(r, 1, 1000)])
    tail = log_int(r, 1, 2000)
    pos = [shared + r.choice([0, 1, 15, 16, r.randrange(tail + 1)]) for _ in range(n)]
    for i in range(n):
        if r.random() < 0.05:
            pos[i] = r.randrange(shared + 1)
    st, plan, b = prefix(pkv, pos, shared, geom, bs=r.choice([16, 64, 8]), elem=r.choice([2, 2, 2, 4]))
    assert st == 0, pkv._lib.last_error()
    assert plan.workspace_bytes <= b.ws and plan.image_bytes <= b.staging.size
    image = Image(b.staging, plan)
    check_cover(image, plan, {t: p + 1 for t, p in enumerate(pos)})
    assert all(begin % 16 == 0 for _, begin, _, _ in image.items.tolist())


def test_packed_rows_without_starts_and_empty_steps(pkv):
    st, plan, b = cross(pkv, [3, 0, 5], [10, 10, 300], 9, GEOMS[0])
    assert st == 0
    image = Image(b.staging, plan)
    assert image.seq.tolist() == [0, 0, 0, 2, 2, 2, 2, 2, -1]
    for q_len, kv_len, n in (([0, 0], [5, 6], 4), ([], [], 4), ([1], [5], 0)):
        b = Buffers(pkv, max(n, 1), 14, 2, 64, False)
        st, plan, _ = cross(pkv, q_len, kv_len, n, GEOMS[0], b=b)
        assert st == 0 and plan.n_tiles == plan.n_items == plan.n_merged == 0
        assert pkv.lib().pkv_cross_attn_bf16(C.byref(plan), *[None] * 6, 1.0, None, 0, None) == 0


def test_plans_that_were_never_made_are_refused(pkv):
    L, E = pkv.lib(), pkv._lib
    plan = E.SegmentPlan()
    cross_args, prefix_args = (C.byref(plan), *[None] * 6, 1.0, None, 0, None), (C.byref(plan), *[None] * 7, 1.0, None, 0, None)
    assert L.pkv_cross_attn_bf16(*cross_args) == L.pkv_prefix_attn_bf16(*prefix_args) == E.PKV_E_ARG
    st, plan, b = cross(pkv, [1, -1], [5, 5], 4, GEOMS[0])
    assert st == E.PKV_E_ARG and L.pkv_cross_attn_bf16(C.byref(plan), *[None] * 6, 1.0, None, 0, None) == E.PKV_E_ARG
    st, plan, b = cross(pkv, [1], [5], 0, GEOMS[0], b=Buffers(pkv, 1, 14, 2, 64, False))
    assert st == 0 and L.pkv_prefix_attn_bf16(C.byref(plan), *[None] * 7, 1.0, None, 0, None) == E.PKV_E_ARG


def test_refusals(pkv):
    L, E = pkv.lib(), pkv._lib
    g = GEOMS[0]
    assert cross(pkv, [3, -1], [5, 5], 9, g)[0] == E.PKV_E_ARG
    assert cross(pkv, [3, 1], [5, -5], 9, g)[0] == E.PKV_E_ARG
    assert cross(pkv, [3, 7], [5, 5], 9, g)[0] == E.PKV_E_ARG                             # behind the last row
    assert cross(pkv, [3, 3], [5, 5], 9, g, q_start=[0, 2])[0] == E.PKV_E_ARG             # a row of two sequences
    assert cross(pkv, [3, 3], [5, 5], 9, g, q_start=[-1, 4])[0] == E.PKV_E_ARG
    assert cross(pkv, [2], [5], 9, g, elem=1)[0] == E.PKV_E_ARG
    assert cross(pkv, [2], [5], 9, (14, 4, 64), b=Buffers(pkv, 9, 14, 2, 64, False))[0] == E.PKV_E_UNSUPPORTED
    assert cross(pkv, [2], [5], 9, (2, 1, 512))[0] == E.PKV_E_UNSUPPORTED
    assert prefix(pkv, [5, -1], 0, g)[0] == E.PKV_E_ARG
    assert prefix(pkv, [5, 2 ** 31 - 1], 0, g)[0] == E.PKV_E_UNSUPPORTED and prefix(pkv, [5, 2 ** 30], 0, g)[0] == E.PKV_E_UNSUPPORTED
    assert cross(pkv, [2], [2 ** 30 + 1], 9, g)[0] == E.PKV_E_UNSUPPORTED and cross(pkv, [2], [2 ** 31 - 1], 9, g)[0] == E.PKV_E_UNSUPPORTED
    assert prefix(pkv, [5], -16, g)[0] == E.PKV_E_ARG
    small = Buffers(pkv, 64, 14, 2, 64, True)
    small.ws = 4096
    assert prefix(pkv, [5000] * 64, 4096, g, b=small)[0] == E.PKV_E_WORKSPACE
    small = Buffers(pkv, 64, 14, 2, 64, True)
    small.staging = np.zeros(512, np.uint8)
    assert prefix(pkv, [5000] * 64, 4096, g, b=small)[0] == E.PKV_E_WORKSPACE
    assert L.pkv_prefix_plan_host(None, 3, 0, 14, 2, 64, 16, 2, None, 0, None, 0, None, C.byref(E.SegmentPlan())) == E.PKV_E_ARG
    assert L.pkv_cross_plan_host(None, None, None, 3, 3, 14, 2, 64, 16, 2, None, 0, None, 0, None, None) == E.PKV_E_ARG
    # the attention calls look at everything before they enqueue
    st, plan, b = prefix(pkv, [500] * 9, 256, g)
    one, ws = 256, (1 << 20, b.ws)           # never dereferenced: every call below is refused on the host
    ok = [one] * 6 + [one]
    call = lambda kind, suffix, args, scale=1.0, w=ws, p=plan: getattr(L, f"pkv_{kind}_attn_{suffix}")(None if p is None else C.byref(p), *args, scale, *w, None)
    assert call("prefix", "bf16", ok, p=None) == E.PKV_E_ARG
    assert call("cross", "bf16", ok[:6]) == E.PKV_E_ARG                                    # a plan of the other kind
    assert call("prefix", "f32", ok) == E.PKV_E_ARG                                        # made for 16 bits
    for i in range(7):
        assert call("prefix", "f16", ok[:i] + [None] + ok[i + 1:]) == E.PKV_E_ARG
    assert call("prefix", "f16", ok, scale=0.0) == E.PKV_E_ARG
    assert call("prefix", "f16", ok, scale=float("nan")) == E.PKV_E_ARG
    assert call("prefix", "f16", ok, w=(None, b.ws)) == E.PKV_E_ARG
    assert call("prefix", "f16", ok, w=(264, b.ws)) == E.PKV_E_ARG
    assert call("prefix", "f16", ok, w=(256, 64)) == E.PKV_E_WORKSPACE
    for i in (0, 1, 2, 6):
        arg = list(ok)
        arg[i if i < 6 else 6] = 264
        assert call("prefix", "f16", arg) == E.PKV_E_ARG                                   # off a 16-byte boundary


def test_norm_refusals(pkv):
    L, E = pkv.lib(), pkv._lib
    one = 256
    base = dict(q=one, k=one, v=one, qs=896, ks=128, vs=128, qw=one, kw=one, eps=1e-6, pos=one, cos=one, sin=one, maxp=10, slots=one, qo=512,
                kc=one, vc=one, n_slots=64, n=3, qh=14, kvh=2, hd=64)

    def call(**kw):
        a = {**base, **kw}
        return L.pkv_qk_norm_rope_append_bf16(*[a[k] for k in base], None)

    for p in ("q", "k", "v", "qw", "kw", "pos", "cos", "sin", "slots", "qo", "kc", "vc"):
        assert call(**{p: None}) == E.PKV_E_ARG, p
    assert call(hd=65) == E.PKV_E_UNSUPPORTED
    assert call(eps=-1.0) == E.PKV_E_ARG and call(eps=float("nan")) == E.PKV_E_ARG
    assert call(qs=895) == E.PKV_E_ARG and call(ks=127) == E.PKV_E_ARG and call(vs=-128) == E.PKV_E_ARG
    assert call(maxp=0) == E.PKV_E_ARG and call(n_slots=0) == E.PKV_E_ARG and call(qh=-1) == E.PKV_E_ARG
    assert call(qo=one, qs=1024) == E.PKV_E_ARG                    # in place needs contiguous rows
    assert call(n=0, q=None) == 0 and call(qh=0, kvh=0, q=None) == 0


def test_longest_allowed_keys_are_planned(pkv):
    """2^30 keys, whose lengths in tiles and slabs stay within 32 bits."""
    for geom in (GEOMS[0], GEOMS[2]):
        st, plan, b = cross(pkv, [40, 1], [2 ** 30, 2 ** 30], 41, geom)
        assert st == 0, pkv._lib.last_error()
        check_cover(Image(b.staging, plan), plan, {t: 2 ** 30 for t in range(41)})
        st, plan, b = prefix(pkv, [2 ** 30 - 1] * 3, 2 ** 30 - 16, geom)
        assert st == 0, pkv._lib.last_error()
        check_cover(Image(b.staging, plan), plan, {t: 2 ** 30 for t in range(3)})


def test_plans_do_not_depend_on_what_was_planned_before(pkv):
    """The same lengths give the same image, whatever the staging buffer held."""
    b = Buffers(pkv, 100, 32, 8, 128, True)
    pos = [4096 + 7 * i for i in range(100)]
    st, plan, _ = prefix(pkv, pos, 4096, GEOMS[2], b=b)
    first = b.staging[:plan.image_bytes].copy()
    prefix(pkv, [50] * 100, 0, GEOMS[2], b=b)
    st, again, _ = prefix(pkv, pos, 4096, GEOMS[2], b=b)
    assert st == 0 and again.image_bytes == plan.image_bytes
    a, c = Image(first, plan), Image(b.staging, again)
    for name in ("items", "tiles", "merge", "pos"):
        assert np.array_equal(getattr(a, name), getattr(c, name)), name


def test_tensors_without_a_device_are_refused(pkv):
    """No CPU path: the Python calls say so before anything is launched."""
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    i, table = torch.zeros(2, dtype=torch.int32), torch.zeros(4, 32)
    with pytest.raises(ValueError, match="no CPU path"):
        pkv.launch_qk_norm_rope_store_kv(x, x, x, x[0, :64], x[0, :64], 1e-6, i, table, table, i, x, x, x, 2, 2, 2, 64)
    with pytest.raises(ValueError, match="no CPU path"):
        pkv.CrossPlan(2, 1, 2, 2, 64, 16, torch.bfloat16, workspace=torch.zeros(1 << 20, dtype=torch.uint8))


def test_waits_are_long_enough_for_what_is_planned(pkv):
    """Items that a bounded wait could take for a lost one are not planned: very long ones go to the decode kernels, a call of seconds
    is refused."""
    E = pkv._lib
    st, plan, _ = cross(pkv, [300], [2 ** 25], 300, GEOMS[2])
    assert st == 0 and plan.n_tiles > 0
    st, plan, _ = cross(pkv, [300], [2 ** 25 + 1], 300, GEOMS[2])
    assert st == 0 and plan.n_tiles == 0 and plan.n_items >= 300
    st, plan, _ = prefix(pkv, [2 ** 25 + 40] * 5, 2 ** 25 + 16, GEOMS[2])
    assert st == 0 and plan.n_tiles == 0
    st, plan, _ = cross(pkv, [2 ** 15], [2 ** 25], 2 ** 15, GEOMS[2])
    assert st == E.PKV_E_UNSUPPORTED and "split the step" in pkv._lib.last_error()


def test_recorded_give_up_is_reported_once(pkv):
    """What a kernel recorded is told by the next call of either form, which enqueues nothing; empty steps never look."""
    L, E = pkv.lib(), pkv._lib
    _, plan, _ = cross(pkv, [3, 40], [50, 700], 43, GEOMS[0])
    nothing = (C.byref(plan), *[None] * 6, 1.0, None, 0, None)
    _, other, _ = prefix(pkv, [600] * 9, 512, GEOMS[0])
    _, empty, _ = cross(pkv, [0], [5], 2, GEOMS[0])
    assert L.pkv_debug_set_reported_flags(32) == 0
    assert L.pkv_cross_attn_bf16(C.byref(empty), *[None] * 6, 1.0, None, 0, None) == 0
    assert L.pkv_cross_attn_bf16(*nothing) == E.PKV_E_CUDA and "0x20" in E.last_error()
    assert L.pkv_cross_attn_bf16(*nothing) == E.PKV_E_ARG            # cleared by the report: as far as the pointers
    assert L.pkv_debug_set_reported_flags(32) == 0
    assert L.pkv_prefix_attn_f16(C.byref(other), *[None] * 7, 1.0, None, 0, None) == E.PKV_E_CUDA
    assert L.pkv_prefix_attn_f16(C.byref(other), *[None] * 7, 1.0, None, 0, None) == E.PKV_E_ARG
