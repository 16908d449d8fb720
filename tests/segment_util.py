"""Reads the image a segment plan writes (include/pkv.h, pkv_segment_plan) back into Python, and the sizes of the
library's records (llm-engine_b200/csrc/segment_plan.hpp)."""
import numpy as np


class Image:
    def __init__(self, staging, plan):
        raw = staging.numpy() if hasattr(staging, "numpy") else staging
        p = plan
        assert raw[:4].view(np.int32)[0] == 0x706b7631
        self.n_shares = int(raw[24:28].view(np.int32)[0])

        def ints(off, n, width):
            return raw[off:off + 4 * n * width].copy().view(np.int32).reshape(n, width)

        self.items = ints(p.off_items, p.n_items, 4)                      # token, kv_begin, kv_len, part
        self.tiles = ints(p.off_tiles, p.n_tiles, 8)                      # tok0, n_tok, kvh, kv_begin, kv_len, part, flags, -
        self.merge = ints(p.off_merge, p.n_merged, 8)                     # token, kvh, tile row, stride, n, own part, n, -
        self.rows = raw[p.off_rows:p.off_items].view(np.int32)
        self.lists = ints(p.off_lists, p.n_lists + 1, 1)[:, 0] if p.n_lists else None
        self.seq = ints(p.off_seq, p.n_tokens, 1)[:, 0]
        self.pos = ints(p.off_pos, p.n_tokens, 1)[:, 0]
        first = p.off_items + 16 * p.n_items
        self.first = raw[first:first + 4 * (self.n_shares + 1)].copy().view(np.int32) if self.n_shares else None


def check_cover(image, plan, want):
    """want: {token: number of keys}.  Every (token, kv head, key) is worked on exactly once; what is done in one piece writes
    the output, and the merge reads every other piece's partial, each row and part used once."""
    group, kvh_n = plan.q_heads // plan.kv_heads, plan.kv_heads
    keys, direct, tile_rows, parts = {}, set(), {}, {}
    for token, begin, n, part in image.items.tolist():
        assert n > 0 and begin >= 0
        for h in range(kvh_n):
            keys.setdefault((token, h), []).append((begin, n))
            if part < 0:
                assert (token, h) not in direct
                direct.add((token, h))
        if part >= 0:
            parts.setdefault(token, []).append(part)
    used_rows = np.zeros(plan.n_tile_rows, np.int32)
    for tok0, n_tok, kvh, begin, n, part, flags, _ in image.tiles.tolist():
        pair = bool(flags & 2)
        rows = n_tok * group
        assert 1 <= rows <= (128 if pair else 256) and n > 0 and begin % 128 == 0 and kvh + pair < kvh_n
        tokens = image.rows[tok0:tok0 + n_tok]
        assert bool(flags & 1) == bool((np.diff(tokens) == 1).all())
        for h in range(1 + pair):
            for i, token in enumerate(tokens.tolist()):
                keys.setdefault((token, kvh + h), []).append((begin, n))
                if part < 0:
                    assert (token, kvh + h) not in direct
                    direct.add((token, kvh + h))
                else:
                    tile_rows.setdefault((token, kvh + h), []).append(part + h * rows + i * group)
        if part >= 0:
            used_rows[part:part + rows * (1 + pair)] += 1
    assert (used_rows == 1).all()
    merged = {}
    for token, kvh, row, stride, n_tile, own, n_own, _ in image.merge.tolist():
        assert (token, kvh) not in merged
        merged[token, kvh] = ([row + i * stride for i in range(n_tile)], list(range(own, own + n_own)))
    used_parts = []
    for token, n_keys in want.items():
        for h in range(kvh_n):
            got = sorted(keys.get((token, h), []))
            at = 0
            for begin, n in got:
                assert begin == at, (token, h, got)
                at += n
            assert at == n_keys, (token, h, at, n_keys)
            if (token, h) in direct:
                assert len(got) == 1 and (token, h) not in merged
            else:
                assert merged[token, h] == (sorted(tile_rows.get((token, h), [])), sorted(parts.get(token, [])))
                assert bool(n_keys) == bool(merged[token, h][0] or merged[token, h][1])
        used_parts += parts.get(token, [])
    assert set(t for t, _ in keys) <= set(want) and set(t for t, _ in merged) <= set(want)
    assert sorted(used_parts) == list(range(plan.n_parts))
    if image.first is not None:
        assert image.first[0] == 0 and image.first[-1] == len(image.items) and (np.diff(image.first) >= 0).all()
    if image.lists is not None:
        assert image.lists[0] == 0 and image.lists[-1] == len(image.tiles) and (np.diff(image.lists) > 0).all()


# ---- steps on the device, and the definition in 64 bits ----
U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


class Step:
    """Sequences with tables of their own over a pool in which every slot that no key occupies holds NaN.
    q_len[s] rows each; kv_len[s] keys each; `shared` leading keys are the same blocks for all (shared < every kv_len)."""

    def __init__(self, torch, dtype, geom, q_len, kv_len, bs, seed, q_start=None, rows=None, shared=0, sharp=1.0):
        self.torch, self.dtype, self.bs = torch, dtype, bs
        self.qh, self.kvh, self.hd = geom
        dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_len, self.kv_len = list(q_len), list(kv_len)
        self.q_start = list(q_start) if q_start is not None else np.cumsum([0] + self.q_len)[:-1].tolist()
        self.n = rows if rows is not None else max([a + b for a, b in zip(self.q_start, self.q_len)] + [1])
        common = shared // bs
        need = [max(-(-k // bs) - common, 0) for k in self.kv_len]
        nb = sum(need) + common + 3
        ids = rng.permutation(nb).astype(np.int32)
        self.tables, at = [], common
        for k in need:
            self.tables.append(np.concatenate([ids[:common], ids[at:at + k]]).astype(np.int32))
            at += k
        self.num_blocks = nb
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()
        flat = np.concatenate(self.tables) if self.tables else np.zeros(0, np.int32)
        self.block_tables = i32(flat if flat.size else np.zeros(1, np.int32))
        self.table_offset = i32(np.cumsum([0] + [len(t) for t in self.tables])[:-1] if self.tables else np.zeros(1))
        kv_dim = self.kvh * self.hd
        self.kc = torch.full((nb * bs, kv_dim), float("nan"), device="cuda", dtype=dt)
        self.vc = torch.full((nb * bs, kv_dim), float("nan"), device="cuda", dtype=dt)
        self.slots = []
        for t, k in zip(self.tables, self.kv_len):
            s = (t[:, None].astype(np.int64) * bs + np.arange(bs)).reshape(-1)[:k]
            self.slots.append(torch.from_numpy(s).cuda())
        every = torch.cat(self.slots).unique() if self.slots else torch.zeros(0, dtype=torch.long, device="cuda")
        self.kc[every] = torch.randn((len(every), kv_dim), generator=g, device="cuda").to(dt)
        self.vc[every] = torch.randn((len(every), kv_dim), generator=g, device="cuda").to(dt)
        self.q = (sharp * torch.randn((self.n, self.qh * self.hd), generator=g, device="cuda")).to(dt)
        self.mark = torch.randn((self.n, self.qh * self.hd), generator=g, device="cuda").to(dt)
        self.out = self.mark.clone()
        self.scale = self.hd ** -0.5

    def expected(self, limits=None):
        """(rows, want, bound): the definition in 64 bits, and how far fp32 arithmetic with 16-bit operands may be off it.

        With s the scores, A = sum w |v| and w the weights: a score is a sum of D products, off by under 4 D u scale sum|q k|
        (the tensor cores' sums keep at least 22 bits), which moves the result by twice that of A.  P is rounded to the element type
        before the second product, HALF_STEP A, absolutely by 2^-25 per key where it is subnormal in f16 (the sum of
        the P is at least 2^-8 of the largest, kept below 2^8: 2^-25 of at least 1).  fp32 sums of L terms: (L + 64) u A with
        the exponentials and the merge.  The result is rounded once more: HALF_STEP |want|."""
        torch, f64 = self.torch, self.torch.float64
        group = self.qh // self.kvh
        rows, want, bound = [], [], []
        for s, n in enumerate(self.q_len):
            if n == 0:
                continue
            at = self.q_start[s]
            q = self.q[at:at + n].to(f64).view(n, self.kvh, group, self.hd)
            k, v = (x[self.slots[s]].to(f64).view(-1, self.kvh, self.hd) for x in (self.kc, self.vc))
            if limits is not None:
                k, v = k[:limits[s]], v[:limits[s]]
            L = k.shape[0]
            rows.append(torch.arange(at, at + n, device="cuda"))
            if L == 0:
                want.append(torch.zeros((n, self.qh * self.hd), dtype=f64, device="cuda"))
                bound.append(torch.zeros_like(want[-1]))
                continue
            sc = torch.einsum("nhgd,lhd->nhgl", q, k) * self.scale
            size = torch.einsum("nhgd,lhd->nhgl", q.abs(), k.abs()).amax(-1, keepdim=True) * self.scale
            w = torch.softmax(sc, -1)
            o = torch.einsum("nhgl,lhd->nhgd", w, v)
            A = torch.einsum("nhgl,lhd->nhgd", w, v.abs())
            r = 8 * self.hd * U * size * A + (L + 64) * U * A
            if self.dtype != "f32":
                r = r + HALF_STEP[self.dtype] * A
            if self.dtype == "f16":
                r = r + 2.0 ** -25 * v.abs().sum(0)[None, :, None, :]
            r = r + HALF_STEP[self.dtype] * (o.abs() + r) + 2.0 ** -25
            want.append(o.reshape(n, -1))
            bound.append(r.reshape(n, -1))
        cat = lambda x, shape: torch.cat(x) if x else torch.zeros(shape, dtype=f64, device="cuda")
        width = self.qh * self.hd
        return (torch.cat(rows) if rows else torch.zeros(0, dtype=torch.long, device="cuda")), cat(want, (0, width)), cat(bound, (0, width))

    def check(self, pkv, out=None, limits=None):
        torch = self.torch
        torch.cuda.synchronize()
        out = self.out if out is None else out
        assert pkv.debug_device_flags() == 0
        rows, want, bound = self.expected(limits)
        off = (out[rows].to(torch.float64) - want).abs()
        bad = ~(off <= bound)
        assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} values off, rows {rows[bad.any(1).nonzero()[:8, 0]].tolist()}, "
                                     f"by up to {(off / (bound + 1e-300)).nan_to_num(1e9).max().item():.3g} bounds")
        rest = torch.ones(self.n, dtype=torch.bool, device="cuda")
        rest[rows] = False
        assert torch.equal(out[rest], self.mark[rest]), "rows of no sequence were written"

    def move_behind(self, blocks):
        """The same step in pools that begin with `blocks` blocks of nobody's."""
        for name in ("kc", "vc"):
            small = getattr(self, name)
            pool = self.torch.empty((blocks * self.bs + small.shape[0], small.shape[1]), device="cuda", dtype=small.dtype)
            pool[blocks * self.bs:] = small
            setattr(self, name, pool)
        self.block_tables += blocks
        self.slots = [s + blocks * self.bs for s in self.slots]
        self.num_blocks += blocks
