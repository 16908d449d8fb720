"""The stamp in a segment plan's image names the counts and offsets that the step's launches are made for, so that a captured call which is
replayed over another step's image can tell (tests/test_segment_edges_gpu.py replays some)."""
import numpy as np
import pytest

from tests.test_segment_plan import Buffers, GEOMS, cross, prefix


def stamps(b):
    """(of the whole image, of the cluster form)"""
    return tuple(b.staging[28:36].view(np.int32).tolist())


def layout(plan):
    return tuple(getattr(plan, name) for name, _ in plan._fields_ if name != "num_blocks")


def test_same_layout_same_stamp_and_other_layouts_others(pkv, monkeypatch):
    seen = {}
    for tiles in ("", "0", "1"):
        monkeypatch.setenv("PKV_SEGMENT_TILES", tiles)
        for geom in GEOMS[:4]:
            for n in (1, 5, 40, 130):
                for shared in (0, 64, 640, 5000):
                    for tail in (1, 2, 17, 400):
                        st, plan, b = prefix(pkv, [shared + tail + i % 3 for i in range(n)], shared, geom)
                        assert st == 0 and stamps(b)[0] != 0
                        seen.setdefault(layout(plan), set()).add(stamps(b)[0])
                st, plan, b = cross(pkv, [1 + i % 3 for i in range(n)], [50 + 40 * i for i in range(n)], 3 * n, geom)
                assert st == 0 and stamps(b)[0] != 0
                seen.setdefault(layout(plan), set()).add(stamps(b)[0])
    assert all(len(s) == 1 for s in seen.values())
    assert len(seen) > 200 and len({next(iter(s)) for s in seen.values()}) == len(seen)


def test_contents_alone_do_not_change_it(pkv, monkeypatch):
    """Lengths of as many key tiles each are dealt alike; a tile more is another unit for the dealer."""
    monkeypatch.setenv("PKV_SEGMENT_TILES", "1")
    images = [cross(pkv, [40, 40], kv, 80, GEOMS[1])[1:] for kv in ([300, 910], [383, 1000], [300, 1025])]
    a, c, d = [(layout(plan), stamps(b)) for plan, b in images]
    assert a == c and images[0][1].staging.tobytes() != images[1][1].staging.tobytes()
    assert (a[0] == d[0]) == (a[1] == d[1])


@pytest.mark.parametrize("geom", GEOMS[:2])
def test_cluster_form_asks_for_keys_in_every_row_only(pkv, geom):
    """It reads positions and sequences, which any image of as many rows holds if all of them have keys."""
    of = lambda *a, **kw: stamps(cross(pkv, *a, geom, **kw)[2])[1]
    n = 6
    same = of([1] * n, [900] * n, n)
    assert same != 0
    assert of([1] * n, [100 + i for i in range(n)], n) == same and of([2, 4], [3, 8000], n) == same
    assert of([1] * n, [900] * (n - 1) + [0], n) == 0               # a row without keys
    assert of([1] * (n - 1), [900] * (n - 1), n) == 0               # a row of no sequence
    assert of([1] * n, [900] * n, n, bs=32) != same
    assert stamps(prefix(pkv, [900] * n, 512, geom)[2])[1] not in (0, same)
    assert len({stamps(prefix(pkv, [900 + 37 * k] * n, s, geom)[2])[1] for k in range(4) for s in (0, 16, 512)}) == 1
