"""Operators of one layer next to the paged K/V pools, as cases that can be timed one by one.

  norm    RMS norms of the query and key heads, the position rotation of both and the append of K and V
          to the pools, in one pass over the projection's output (its rows packed q | k | v, or apart)
  cross   attention of every sequence's new tokens to an encoder's states, held in blocks of the pools
          like any K/V, of a length of their own: no causal mask
  prefix  one new token per sequence for sequences that all start with the same long prompt: the shared
          keys are worked through once for all of them, each sequence's own keys follow

Head counts are those of Qwen2.5-0.5B (14 query heads, 2 kv heads, 64 dims) and TinyLlama-1.1B (32, 4,
64), a generic (32, 8, 128) and, for encoder-decoder attention, one key head per query head (16, 16, 64).
Lengths follow the case alone, so that every seed costs the same; values, block tables and the order of
the lengths follow the seed.  Pools hold what the step needs and a sixteenth more, in shuffled order.
"""
import importlib

import numpy as np
import torch

own = False      # True: the framework's operators; False: their plain form in elementary torch operations

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
QWEN = {"q_heads": 14, "kv_heads": 2, "head_dim": 64}
TINY = {"q_heads": 32, "kv_heads": 4, "head_dim": 64}
WIDE = {"q_heads": 32, "kv_heads": 8, "head_dim": 128}
PAIRED = {"q_heads": 16, "kv_heads": 16, "head_dim": 64}
EPS = 1e-6
ROPE_BASE = 1e6


def _norm(heads, dtype, tokens, packed=True, max_pos=8192):
    """tokens rows of a step; packed: q, k and v are column ranges of one projection's output."""
    return {"kind": "norm", **heads, "dtype": dtype, "tokens": tokens, "packed": packed, "max_pos": max_pos, "block": 16}


def _cross(heads, dtype, seqs, new, enc, block=16, lengths=1):
    """seqs sequences with new = (fewest, most) tokens each against enc = (shortest, longest) encoder states."""
    return {"kind": "cross", **heads, "dtype": dtype, "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "enc_lo": enc[0],
            "enc_hi": enc[1], "block": block, "lengths": lengths}


def _prefix(heads, dtype, seqs, shared, tail, block=16, lengths=1):
    """seqs sequences behind one prompt of `shared` tokens, each tail = (fewest, most) tokens past it."""
    return {"kind": "prefix", **heads, "dtype": dtype, "seqs": seqs, "shared": shared, "tail_lo": tail[0], "tail_hi": tail[1],
            "block": block, "lengths": lengths}


def listed():
    return [
        # a chat with one user: nothing but latency
        {"name": "norm_one", **_norm(QWEN, "bf16", 1)},
        # fp32, the precision the CPU engine checks against, q, k and v from projections of their own
        {"name": "norm_f32", **_norm(QWEN, "f32", 301, packed=False)},
        # a decode step of a full server on wider heads
        {"name": "norm_step", **_norm(WIDE, "f16", 256)},
        # prompts: the rows of a large prefill step
        {"name": "norm_prompts", **_norm(WIDE, "bf16", 8191)},
        # a transcription that has begun: one token against one recording's states
        {"name": "cross_one", **_cross(PAIRED, "f16", 1, (1, 1), (1500, 1500))},
        # a decode step of many: every sequence has read a source of its own length
        {"name": "cross_step", **_cross(TINY, "bf16", 96, (1, 1), (60, 3000), lengths=2)},
        # a few tokens a sequence (drafts, or beams that share their source), fp32
        {"name": "cross_f32", **_cross(QWEN, "f32", 7, (1, 6), (33, 900), lengths=3)},
        # the forced first tokens of a batch of targets, ragged on both sides
        {"name": "cross_prompts", **_cross(PAIRED, "bf16", 24, (3, 448), (100, 1500), lengths=4)},
        # long targets against long sources
        {"name": "cross_long", **_cross(WIDE, "bf16", 4, (1000, 2048), (4000, 6500), block=32, lengths=5)},
        # a handful of users of one assistant with a short system prompt
        {"name": "prefix_few", **_prefix(QWEN, "bf16", 6, 512, (5, 90), lengths=6)},
        # a full server behind one prompt
        {"name": "prefix_chat", **_prefix(TINY, "bf16", 128, 2048, (32, 600), lengths=7)},
        # many questions about one long document
        {"name": "prefix_document", **_prefix(WIDE, "f16", 200, 16384, (16, 400), block=32, lengths=8)},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["norm", "cross", "cross", "prefix", "prefix"])
    lengths = rng.randrange(1, 1 << 20)
    if kind == "norm":
        return _norm(rng.choice([QWEN, TINY, WIDE]), rng.choice(["bf16", "f16", "f32"]), _log_int(rng, 1, 8191), rng.random() < 0.6)
    if kind == "cross":
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        new_hi = rng.choice([1, _log_int(rng, 2, 32), _log_int(rng, 8, 2048)])
        enc_hi = _log_int(rng, 16, 6500)
        c = _cross(rng.choice([QWEN, TINY, WIDE, PAIRED]), dtype, _log_int(rng, 1, 96), (max(1, new_hi // rng.randrange(1, 32)), new_hi),
                   (max(1, enc_hi // rng.randrange(1, 32)), enc_hi), rng.choice([16, 16, 32, 64]), lengths)
        while not _affordable(c):
            c["seqs"] = (c["seqs"] + 1) // 2
            if c["seqs"] == 1:
                c["new_hi"] = max(1, c["new_hi"] // 2)
                c["new_lo"] = min(c["new_lo"], c["new_hi"])
        return c
    block = rng.choice([16, 16, 32])
    tail_hi = _log_int(rng, 2, 1000)
    c = _prefix(rng.choice([QWEN, TINY, WIDE]), rng.choice(["bf16", "f16"]), _log_int(rng, 2, 256), block * _log_int(rng, 2, 16384 // block),
                (max(1, tail_hi // rng.randrange(1, 32)), tail_hi), block, lengths)
    while not _affordable(c):
        c["seqs"] = (c["seqs"] + 1) // 2
    return c


def _affordable(c):
    most = 2e10 if c["dtype"] == "f32" else 6e11
    w = work(c)
    return w["flops"] <= most and w["bytes"] <= 1e9 and (c["kind"] != "prefix" or c["seqs"] * c["tail_hi"] <= 100000)


def _spread(c, lo, hi, n):
    """n lengths, spread over their logarithm; a case's longest is always among them."""
    rng = np.random.default_rng(c["lengths"])
    x = np.clip(np.round(np.exp(rng.uniform(np.log(lo), np.log(hi + 0.49), size=n))), lo, hi).astype(np.int64)
    x[-1] = hi
    return rng.permutation(x)


def _lengths(c):
    """(tokens, keys) of every sequence; for `prefix` the keys behind the shared ones, the new token's included."""
    if c["kind"] == "cross":
        return _spread(c, c["new_lo"], c["new_hi"], c["seqs"]), _spread(c, c["enc_lo"], c["enc_hi"], c["seqs"])
    return np.ones(c["seqs"], np.int64), _spread(c, c["tail_lo"], c["tail_hi"], c["seqs"])


def work(c):
    """norm: every row read and written once, tables of cos and sin once per position in use.  Attention:
    every key and value that some token attends read once, q read, the result written; the two products
    over all (row, key) pairs."""
    e = 4 if c["dtype"] == "f32" else 2
    qh, kvh, hd = c["q_heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] == "norm":
        n = c["tokens"]
        rows = 2 * n * (qh + 2 * kvh) * hd * e
        return {"bytes": rows + 8 * n + 4 * hd * min(n, c["max_pos"]) + 2 * hd * e, "flops": n * hd * (7 * (qh + kvh))}
    new, keys = _lengths(c)
    shared = c.get("shared", 0)
    held, pairs, n = int(keys.sum()) + shared, int((new * (keys + shared)).sum()), int(new.sum())
    blocks = int(((keys + c["block"] - 1) // c["block"]).sum()) + shared // c["block"]
    return {"bytes": 2 * held * kvh * hd * e + 2 * n * qh * hd * e + 4 * blocks, "flops": 4 * hd * qh * pairs}


class _State:
    pass


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _inputs(c, seed):
    """The tensors a layer finds before the call, from the seed alone."""
    s = _State()
    s.case = c
    rng = np.random.default_rng([seed, c.get("lengths", 1)])
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + c.get("lengths", 1))
    dt, qh, kvh, hd, bs = DTYPES[c["dtype"]], c["q_heads"], c["kv_heads"], c["head_dim"], c["block"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dt)

    if c["kind"] == "norm":
        n = c["tokens"]
        blocks = (n + bs - 1) // bs
        blocks += blocks // 16 + 2
        s.n, s.n_slots = n, blocks * bs
        # heads of one layer differ in size by an order of magnitude before they are normed
        size = torch.exp(torch.randn((1, qh + 2 * kvh, 1), generator=gen, device="cuda"))
        rows = (torch.randn((n, qh + 2 * kvh, hd), generator=gen, device="cuda") * size).to(dt).view(n, -1)
        parts = rows.split([qh * hd, kvh * hd, kvh * hd], dim=1)
        s.q, s.k, s.v = parts if c["packed"] else [p.contiguous() for p in parts]
        s.q_weight, s.k_weight = 1 + normal(hd, scale=0.2), 1 + normal(hd, scale=0.2)
        s.positions = _ints(rng.integers(0, c["max_pos"], size=n))
        inv = ROPE_BASE ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        angle = torch.arange(c["max_pos"], device="cuda", dtype=torch.float64)[:, None] * inv
        s.cos, s.sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        # a step's tokens fill blocks of the pool in the order the allocator gave them
        ids = rng.permutation(blocks)[:(n + bs - 1) // bs]
        s.slots = _ints((ids[:, None] * bs + np.arange(bs)).reshape(-1)[:n])
        s.q_out = torch.zeros((n, qh * hd), dtype=dt, device="cuda")
        s.k_cache, s.v_cache = normal(s.n_slots, kvh * hd), normal(s.n_slots, kvh * hd)
        return s
    new, keys = _lengths(c)
    order = rng.permutation(len(new))
    new, keys = new[order], keys[order]
    own_blocks, common = (keys + bs - 1) // bs, c.get("shared", 0) // bs
    nb = int(own_blocks.sum()) + common
    nb += nb // 16 + 2
    ids = rng.permutation(nb).astype(np.int32)
    at, tables = common, []
    for k in own_blocks:
        tables.append(np.concatenate([ids[:common], ids[at:at + k]]))
        at += k
    s.new, s.keys, s.num_blocks, s.n = new, keys, nb, int(new.sum())
    s.tables = _ints(np.concatenate(tables))
    s.table_offset = _ints(np.cumsum([0] + [len(t) for t in tables])[:-1])
    s.host_tables = tables
    s.k_cache, s.v_cache = normal(nb * bs, kvh * hd), normal(nb * bs, kvh * hd)
    s.q = normal(s.n, qh * hd, scale=1.5)
    s.out = torch.zeros_like(s.q)
    s.scale = hd ** -0.5
    # pool rows of each sequence's own keys, and of the shared ones, as int64 on the device
    s.rows = [torch.from_numpy((t[common:, None].astype(np.int64) * bs + np.arange(bs)).reshape(-1)[:k]).cuda() for t, k in zip(tables, keys)]
    s.shared_rows = torch.from_numpy((ids[:common, None].astype(np.int64) * bs + np.arange(bs)).reshape(-1)).cuda()
    return s


def prepare(c, seed):
    s = _inputs(c, seed)
    if c["kind"] == "prefix" and not own:
        # the plain form works on a batch padded to its longest tail
        most = int(s.keys.max())
        s.padded = torch.stack([torch.nn.functional.pad(r, (0, most - r.numel())) for r in s.rows])
        s.visible = torch.arange(most, device="cuda") < torch.from_numpy(s.keys).cuda()[:, None]
    if own and c["kind"] != "norm":
        # the work list that a server builds once a step and uses in every layer
        pkv = importlib.import_module("llm-engine_b200")
        heads = (c["q_heads"], c["kv_heads"], c["head_dim"], c["block"])
        if c["kind"] == "cross":
            s.plan = pkv.CrossPlan(s.n, len(s.new), *heads, s.q.dtype, num_blocks=s.num_blocks).build_host(s.new, s.keys)
        else:
            s.token_seq = _ints(np.arange(s.n))
            s.plan = pkv.PrefixPlan(s.n, *heads, s.q.dtype, num_blocks=s.num_blocks).build_host(c["shared"] + s.keys - 1, c["shared"])
    return s


def run(s):
    c = s.case
    if own:
        return _run_own(s, c)
    return {"norm": _plain_norm, "cross": _plain_cross, "prefix": _plain_prefix}[c["kind"]](s, c)


def _run_own(s, c):
    pkv = importlib.import_module("llm-engine_b200")
    if c["kind"] == "norm":
        pkv.launch_qk_norm_rope_store_kv(s.q, s.k, s.v, s.q_weight, s.k_weight, EPS, s.positions, s.cos, s.sin, s.slots, s.q_out,
                                         s.k_cache, s.v_cache, s.n, c["q_heads"], c["kv_heads"], c["head_dim"])
        return {"q": s.q_out, "k_cache": s.k_cache, "v_cache": s.v_cache}
    if c["kind"] == "cross":
        s.plan.attention(s.q, s.k_cache, s.v_cache, s.tables, s.table_offset, s.out, s.scale)
    else:
        s.plan.attention(s.q, s.k_cache, s.v_cache, s.tables, s.table_offset, s.token_seq, s.out, s.scale)
    return {"out": s.out}


def _plain_norm(s, c):
    hd, dt = c["head_dim"], s.q_out.dtype
    cos, sin = s.cos[s.positions.long()][:, None], s.sin[s.positions.long()][:, None]

    def turned(x, weight):
        x = x.float().unflatten(1, (-1, hd))
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(1).to(dt)

    slots = s.slots.long()
    s.q_out.copy_(turned(s.q, s.q_weight))
    s.k_cache[slots] = turned(s.k, s.k_weight)
    s.v_cache[slots] = s.v
    return {"q": s.q_out, "k_cache": s.k_cache, "v_cache": s.v_cache}


def _attend(scores, v):
    """softmax(scores) v over the last axis of scores, its maximum taken off first."""
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p @ v / p.sum(-1, keepdim=True)


def _plain_cross(s, c):
    qh, kvh, hd = c["q_heads"], c["kv_heads"], c["head_dim"]
    at = 0
    for n, rows in zip(s.new.tolist(), s.rows):
        k = s.k_cache[rows].float().view(-1, kvh, hd).transpose(0, 1)                      # [kvh, L, D]
        v = s.v_cache[rows].float().view(-1, kvh, hd).transpose(0, 1)
        q = s.q[at:at + n].float().view(n, kvh, qh // kvh, hd).permute(1, 2, 0, 3)         # [kvh, G, n, D]
        o = _attend(q.reshape(kvh, -1, hd) @ k.transpose(1, 2) * s.scale, v)
        s.out[at:at + n] = o.view(kvh, qh // kvh, n, hd).permute(2, 0, 1, 3).reshape(n, -1).to(s.out.dtype)
        at += n
    return {"out": s.out}


def _plain_prefix(s, c):
    qh, kvh, hd, n = c["q_heads"], c["kv_heads"], c["head_dim"], s.n
    g, shared = qh // kvh, c["shared"]
    ks = s.k_cache[s.shared_rows].float().view(shared, kvh, hd).transpose(0, 1)            # [kvh, P, D]
    vs = s.v_cache[s.shared_rows].float().view(shared, kvh, hd).transpose(0, 1)
    q = s.q.float().view(n, kvh, g, hd)
    first = (q.transpose(0, 1).reshape(kvh, n * g, hd) @ ks.transpose(1, 2) * s.scale).view(kvh, n, g, shared)
    k = s.k_cache[s.padded].float().view(n, -1, kvh, hd).transpose(1, 2)                   # [n, kvh, L, D]
    v = s.v_cache[s.padded].float().view(n, -1, kvh, hd).transpose(1, 2)
    tail = (q @ k.transpose(2, 3) * s.scale).masked_fill(~s.visible[:, None, None], float("-inf"))
    most = torch.maximum(first.amax(-1).transpose(0, 1), tail.amax(-1))                    # [n, kvh, g]
    first = torch.exp(first - most.transpose(0, 1)[..., None])
    tail = torch.exp(tail - most[..., None])
    o = (first.view(kvh, n * g, shared) @ vs).view(kvh, n, g, hd).transpose(0, 1) + tail @ v
    o = o / (first.sum(-1).transpose(0, 1) + tail.sum(-1))[..., None]
    s.out.copy_(o.reshape(n, -1))
    return {"out": s.out}


def exact(c, seed):
    """The definitions in 64 bits, one head or one sequence at a time."""
    s = _inputs(c, seed)
    qh, kvh, hd, f64 = c["q_heads"], c["kv_heads"], c["head_dim"], torch.float64
    if c["kind"] == "norm":
        half, pos = hd // 2, s.positions.long()
        cos, sin = s.cos.to(f64)[pos], s.sin.to(f64)[pos]

        def head(x, weight):
            x = x.to(f64)
            x = x / ((x ** 2).sum(1, keepdim=True) / hd + EPS).sqrt() * weight.to(f64)
            return torch.cat([x[:, :half] * cos - x[:, half:] * sin, x[:, half:] * cos + x[:, :half] * sin], 1)

        q = torch.cat([head(s.q[:, h * hd:(h + 1) * hd], s.q_weight) for h in range(qh)], 1)
        k = torch.cat([head(s.k[:, h * hd:(h + 1) * hd], s.k_weight) for h in range(kvh)], 1)
        kc, vc = s.k_cache.to(f64), s.v_cache.to(f64)
        kc[s.slots.long()], vc[s.slots.long()] = k, s.v.to(f64)
        return {"q": q, "k_cache": kc, "v_cache": vc}
    out, at = torch.zeros((s.n, qh, hd), dtype=f64, device="cuda"), 0
    for n, rows in zip(s.new.tolist(), s.rows):
        rows = torch.cat([s.shared_rows, rows])
        for h in range(kvh):
            heads = slice(h * (qh // kvh), (h + 1) * (qh // kvh))
            k, v = (x[rows, h * hd:(h + 1) * hd].to(f64) for x in (s.k_cache, s.v_cache))
            q = s.q[at:at + n].to(f64).view(n, qh, hd)[:, heads].reshape(-1, hd)
            w = torch.softmax(q @ k.T * s.scale, dim=1)
            out[at:at + n, heads] = (w @ v).view(n, -1, hd)
        at += n
    return {"out": out.flatten(1)}
