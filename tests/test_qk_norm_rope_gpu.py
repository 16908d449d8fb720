"""Per-head norms of q and k + rotation + append in one pass, against the formula in 64 bits.

Bounds, before any run.  u = 2^-24.  The sum of squares is a chain of at most 2 x 8 products and 5 additions a lane
(or D / 32 and 5): relative error under 21 u, halved by the root; the mean, eps, the root and its inverse add a
rounding each, the two products with inv and w one each, the rotation two: under 20 u of |n c| + |m s|, tested as 32 u.
Then one rounding to the element type: eps / 2 of the value, or half its smallest subnormal.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SUBNORMAL = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}


def make(torch, dtype, qh, kvh, hd, n, packed, seed, max_pos=700, n_slots=None, pad=0):
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = (qh + 2 * kvh) * hd
    rows = torch.randn((n, width + pad), generator=g, device="cuda") * torch.exp(torch.randn((n, 1), generator=g, device="cuda"))
    rows = rows.to(dt)
    q, k, v = rows[:, :qh * hd], rows[:, qh * hd:(qh + kvh) * hd], rows[:, (qh + kvh) * hd:width]
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    n_slots = n_slots or n + 37
    rng = np.random.default_rng(seed)
    d = {
        "q": q, "k": k, "v": v,
        "qw": (1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).to(dt), "kw": (1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).to(dt),
        "pos": torch.from_numpy(rng.integers(0, max_pos, n).astype(np.int32)).cuda(),
        "slots": torch.from_numpy(rng.permutation(n_slots)[:n].astype(np.int32)).cuda(),
        "cos": torch.cos(torch.rand((max_pos, hd // 2), generator=g, device="cuda") * 6.28), "sin": torch.sin(torch.rand((max_pos, hd // 2), generator=g, device="cuda") * 6.28),
        "qo": torch.randn((n, qh * hd), generator=g, device="cuda").to(dt),
        "kc": torch.randn((n_slots, kvh * hd), generator=g, device="cuda").to(dt), "vc": torch.randn((n_slots, kvh * hd), generator=g, device="cuda").to(dt),
    }
    return d


def formula(torch, d, heads, hd, which, eps):
    """(values, size of the terms) of the rotated heads in 64 bits."""
    x = d[which].double().reshape(d[which].shape[0], heads, hd)
    w = d[which + "w"].double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    pos = d["pos"].long().clamp(0, d["cos"].shape[0] - 1)
    c, s = d["cos"].double()[pos][:, None], d["sin"].double()[pos][:, None]
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    val = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    return val.flatten(1), size.flatten(1)


def near(torch, got, want, size, dtype):
    eps = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    bound = 32 * U * size + eps * (want.abs() + 32 * U * size) + SUBNORMAL[dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item():.3g} of the bound"


def launch(pkv, d, n, qh, kvh, hd, eps, **kw):
    pkv.launch_qk_norm_rope_store_kv(d["q"], d["k"], d["v"], d["qw"], d["kw"], eps, d["pos"], d["cos"], d["sin"], d["slots"],
                                     d.get("out", d["qo"]), d["kc"], d["vc"], n, qh, kvh, hd, **kw)


def check(torch, pkv, d, n, qh, kvh, hd, eps, dtype, **kw):
    before = {x: d[x].clone() for x in ("qo", "kc", "vc", "k", "v")}
    q_want, q_size = formula(torch, d, qh, hd, "q", eps)
    k_want, k_size = formula(torch, d, kvh, hd, "k", eps)
    launch(pkv, d, n, qh, kvh, hd, eps, **kw)
    torch.cuda.synchronize()
    pos, slots = d["pos"][:n].long(), d["slots"][:n].long()
    live = (pos >= 0) & (pos < d["cos"].shape[0])
    rows = torch.arange(n, device="cuda")[live]
    near(torch, d["qo"][rows], q_want[rows], q_size[rows], dtype)
    kept = torch.ones(d["qo"].shape[0], dtype=torch.bool, device="cuda")
    kept[rows] = False
    assert torch.equal(d["qo"][kept], before["qo"][kept])
    stored = live & (slots >= 0) & (slots < d["kc"].shape[0])
    at, src = slots[stored], torch.arange(n, device="cuda")[stored]
    near(torch, d["kc"][at], k_want[src], k_size[src], dtype)
    assert torch.equal(d["vc"][at], before["v"][src])
    kept = torch.ones(d["kc"].shape[0], dtype=torch.bool, device="cuda")
    kept[at] = False
    assert torch.equal(d["kc"][kept], before["kc"][kept]) and torch.equal(d["vc"][kept], before["vc"][kept])
    assert torch.equal(d["k"], before["k"]) and torch.equal(d["v"], before["v"])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("geom", [
    # q_heads, kv_heads, head_dim, tokens
    (14, 2, 64, 1), (14, 2, 64, 33), (32, 8, 128, 257), (4, 1, 256, 9),
    (32, 4, 64, 4400),            # several heads a lane
    (5, 4, 128, 5000),            # heads that do not divide by them
    (31, 9, 128, 6700),           # more rows than fit L2
    (3, 2, 32, 20), (6, 3, 40, 17), (4, 4, 6, 5), (1, 1, 2, 3), (2, 1, 96, 40),
])
def test_against_formula(pkv, torch_cuda, dtype, packed, geom):
    qh, kvh, hd, n = geom
    d = make(torch_cuda, dtype, qh, kvh, hd, n, packed, seed=qh * 1000 + n)
    check(torch_cuda, pkv, d, n, qh, kvh, hd, 1e-6, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 40])
def test_padding_rows_and_zero_rows(pkv, torch_cuda, dtype, hd):
    torch = torch_cuda
    qh, kvh, n = 6, 2, 50
    d = make(torch, dtype, qh, kvh, hd, n, True, seed=5)
    d["q"][4] = 0
    d["k"][4] = 0
    d["pos"][torch.tensor([0, 7, 49])] = torch.tensor([-1, 700, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    d["slots"][torch.tensor([1, 8, 48])] = torch.tensor([-1, d["kc"].shape[0], -2 ** 31], dtype=torch.int32, device="cuda")
    check(torch, pkv, d, n, qh, kvh, hd, 1e-5, dtype)
    # fewer tokens than rows: those behind stay as they were
    d = make(torch, dtype, qh, kvh, hd, n, True, seed=6)
    check(torch, pkv, d, 31, qh, kvh, hd, 1e-5, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,pad", [(64, 3), (40, 1), (128, 8)])
def test_odd_strides_and_offsets(pkv, torch_cuda, dtype, hd, pad):
    """Rows whose distance is no multiple of 16 bytes, and pointers that are off by one element."""
    torch = torch_cuda
    d = make(torch, dtype, 4, 2, hd, 60, True, seed=7, pad=pad)
    check(torch, pkv, d, 60, 4, 2, hd, 0.0, dtype)
    store = torch.empty(60 * 4 * hd + 1, dtype=d["qo"].dtype, device="cuda")
    d["qo"] = store[1:].view(60, 4 * hd)
    check(torch, pkv, d, 60, 4, 2, hd, 1e-6, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 40])
def test_in_place_and_captured(pkv, torch_cuda, dtype, hd):
    torch = torch_cuda
    d = make(torch, dtype, 8, 2, hd, 70, False, seed=8)
    want, size = formula(torch, d, 8, hd, "q", 1e-6)
    start = d["q"].clone()
    d["out"] = d["q"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        launch(pkv, d, 70, 8, 2, hd, 1e-6)
    side.synchronize()
    near(torch, d["q"], want, size, dtype)
    first = d["q"].clone(), d["kc"].clone()
    d["q"].copy_(start)
    d["kc"].zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch(pkv, d, 70, 8, 2, hd, 1e-6)
    for _ in range(2):
        d["q"].copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d["q"], first[0])
        assert torch.equal(d["kc"][d["slots"].long()], first[1][d["slots"].long()])


def test_not_a_number_stays_in_its_head(pkv, torch_cuda):
    torch = torch_cuda
    d = make(torch, "bf16", 4, 2, 64, 5, False, seed=9)
    d["q"][2, 70] = float("nan")
    d["k"][3, 5] = float("inf")
    launch(pkv, d, 5, 4, 2, 64, 1e-6)
    torch.cuda.synchronize()
    bad = torch.isnan(d["qo"].view(5, 4, 64)).any(-1)
    assert bad.nonzero().tolist() == [[2, 1]]
    kept = d["kc"][d["slots"].long()].view(5, 2, 64)
    assert torch.isnan(kept).any(-1).nonzero().tolist() == [[3, 0]]


@pytest.mark.parametrize("hd", [64, 40])
@pytest.mark.parametrize("qh,kvh", [(0, 3), (5, 0)])
def test_only_q_or_only_kv(pkv, torch_cuda, qh, kvh, hd):
    d = make(torch_cuda, "bf16", qh, kvh, hd, 21, True, seed=12)
    check(torch_cuda, pkv, d, 21, qh, kvh, hd, 1e-6, "bf16")


@pytest.mark.parametrize("hd", [128, 120])
def test_pools_of_more_than_four_billion_elements(pkv, torch_cuda, hd):
    torch = torch_cuda
    qh, kvh, n = 8, 8, 300
    d = make(torch, "bf16", qh, kvh, hd, n, True, seed=13)
    k_want, k_size = formula(torch, d, kvh, hd, "k", 1e-6)
    far = -(-2 ** 32 // (kvh * hd))
    d["kc"], d["vc"] = (torch.zeros((far + n + 37, kvh * hd), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    d["slots"] += far
    launch(pkv, d, n, qh, kvh, hd, 1e-6)
    at = d["slots"].long()
    near(torch, d["kc"][at], k_want, k_size, "bf16")
    assert torch.equal(d["vc"][at], d["v"])
    assert not bool(d["kc"][:far].any()) and not bool(d["vc"][:far].any())


def test_python_refusals(pkv, torch_cuda):
    torch = torch_cuda
    qh, kvh, hd, n = 4, 2, 64, 9
    good = make(torch, "bf16", qh, kvh, hd, n, True, seed=14)
    for name in good:
        bad = dict(good, **{name: good[name].cpu()})
        with pytest.raises(ValueError):
            launch(pkv, bad, n, qh, kvh, hd, 1e-6)
        with pytest.raises(TypeError):
            launch(pkv, dict(good, **{name: good[name].to(torch.float64)}), n, qh, kvh, hd, 1e-6)
    with pytest.raises(ValueError):
        launch(pkv, {k: v.cpu() for k, v in good.items()}, n, qh, kvh, hd, 1e-6)
    for name, bad in (("q", good["q"][:, :-1]), ("k", good["k"][:5]), ("v", good["v"][:, ::2]), ("qw", good["qw"][:32]), ("pos", good["pos"][:8]),
                      ("slots", good["slots"][::2]), ("cos", good["cos"][:, :16]), ("sin", good["sin"][:600]), ("qo", good["qo"][:8]),
                      ("vc", good["vc"][:-1]), ("kc", good["kc"][:, :64])):
        with pytest.raises(ValueError):
            launch(pkv, dict(good, **{name: bad}), n, qh, kvh, hd, 1e-6)
    check(torch, pkv, good, n, qh, kvh, hd, 1e-6, "bf16")
