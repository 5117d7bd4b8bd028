"""Plain 64-bit forms of the quantised cache, the attention of drafted tokens and the logit
rules, on the CPU, and caches to run them on."""
import numpy as np
import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def bits(pool):
    return pool.view(torch.uint8) if pool.dtype.itemsize == 1 else pool


def nearest_e4m3(y):
    """Codes' values: the nearest of the type, of two as near the even code."""
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    above = torch.searchsorted(grid, y.abs().contiguous()).clamp(1, 126)
    low, high = grid[above - 1], grid[above]
    up, down = high - y.abs(), y.abs() - low
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, above - 1)
    return grid[code] * torch.where(y < 0, -1.0, 1.0)


def quantise(x, dtype):
    """Codes' values (fp64) and fp32 scales of x [..][D], any of its rows not finite: 0 and NaN."""
    x = x.double()
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, 0.0)
    top = x.abs().amax(-1)
    # (a product and a quotient in 64 bits: a half is a half still where x has 24 bits)
    y = x * LARGEST[dtype] / torch.where(top > 0, top, 1.0)[..., None]
    code = torch.round(y) if dtype == torch.int8 else nearest_e4m3(y)
    scale = (top / LARGEST[dtype]).float()
    return code, torch.where(fine, scale, torch.tensor(float("nan")))


class Cache:
    """Pools, scales and a page table on the CPU; slots of no token hold `stale`."""

    def __init__(self, dtype, B, heads, D, page, tokens, seed, stale=None, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.tiles = -(-tokens // page)
        self.pages = B * heads * self.tiles + spare
        self.page, self.dtype, self.heads, self.D = page, dtype, heads, D
        self.table = torch.randperm(self.pages, generator=g)[:B * heads * self.tiles] \
            .to(torch.int32).view(B, heads, self.tiles).contiguous()
        shape = (self.pages, page, D)
        self.scales = None
        if dtype in LARGEST:
            x = torch.randn(shape, generator=g)
            x *= LARGEST[dtype] / x.abs().amax(-1, keepdim=True)
            y = torch.randn(shape, generator=g)
            y *= LARGEST[dtype] / y.abs().amax(-1, keepdim=True)
            self.k = x.round().to(dtype) if dtype == torch.int8 else x.to(dtype)
            self.v = y.round().to(dtype) if dtype == torch.int8 else y.to(dtype)
            self.scales = [(0.2 + torch.rand((self.pages, page), generator=g)) * 3 / LARGEST[dtype]
                           for _ in "kv"]
        else:
            self.k = torch.randn(shape, generator=g).to(dtype)
            self.v = torch.randn(shape, generator=g).to(dtype)

    def slot(self, b, h, pos):
        """(page, slot) of a position, None where it has no page."""
        t = pos // self.page
        if pos < 0 or t >= self.tiles or not 0 <= b < self.table.shape[0]:
            return None
        p = int(self.table[b, h, t])
        return (p, pos % self.page) if 0 <= p < self.pages else None

    def held(self, name, b, h, n):
        """Values fp64 [n][D] of positions 0 .. n - 1, and which of them have a page."""
        pool = getattr(self, name)
        pos = torch.arange(n)
        tile = (pos // self.page)
        ok = tile < self.tiles
        page = self.table[b, h, tile.clamp(max=self.tiles - 1)].long()
        ok &= (page >= 0) & (page < self.pages)
        page = torch.where(ok, page, 0)
        x = bits(pool)[page, pos % self.page].view(pool.dtype).double()
        if self.scales is not None:
            x = x * self.scales["kv".index(name)][page, pos % self.page].double()[:, None]
        return x, ok

    def cuda(self):
        out = Cache.__new__(Cache)
        out.__dict__ = dict(self.__dict__)
        for name in ("k", "v", "table"):
            setattr(out, name, getattr(self, name).cuda())
        out.scales = None if self.scales is None else [s.cuda() for s in self.scales]
        return out


def seen_bits(words, n):
    """Truth values [..][n] of mask words."""
    w = words.cpu().long() & 0xffffffff
    return (w[..., None] >> torch.arange(32) & 1).flatten(-2)[..., :n].bool()


def tree(q, cache, contexts, lens, mask, beams, sm_scale):
    """pa_tree in 64 bits, and how far fp32 sums of its products may be from it: q [B][N][H][D]
    on the CPU, mask bool [B][N][N] or None.  Outputs of tokens past lens are NaN in both."""
    B, N, H, D = q.shape
    G = H // cache.heads
    room = cache.tiles * cache.page
    out = torch.full((B, N, H, D), float("nan"), dtype=torch.float64)
    room_for = torch.full((B, N, H, D), float("nan"), dtype=torch.float64)
    for b in range(B):
        n = min(max(lens[b], 0), N)
        C = min(max(contexts[b], 0), room)
        L = min(C + n, room)
        beam = beams[b] if beams else b
        for h in range(H):
            if L == 0 or not 0 <= beam < cache.table.shape[0]:
                out[b, :n, h] = room_for[b, :n, h] = 0.0
                continue
            k, ok = cache.held("k", beam, h // G, L)
            v, _ = cache.held("v", beam, h // G, L)
            for i in range(n):
                see = ok.clone()
                j = torch.arange(L) - C
                own = torch.tril(torch.ones(N, N, dtype=torch.bool))[i] if mask is None else mask[b, i]
                see &= (j < 0) | own[j.clamp(min=0)]
                if not see.any():
                    out[b, i, h] = room_for[b, i, h] = 0.0
                    continue
                x = q[b, i, h].double()
                s = (k[see] * x).sum(-1) * sm_scale
                p = torch.exp(s - s.max())
                w = p / (p.sum() + 1e-6)
                out[b, i, h] = (w[:, None] * v[see]).sum(0)
                # A score is off by its queries' halves (2^-22 of each product) and an fp32 sum of D
                # products (D / 2 roundings of 2^-24 on the way and back, taken as D), its exponent by the
                # roundings of (s - m) in log2 units; e^x by two steps; a probability's parts by 2^-18
                # (two of bf16, the coarsest) at most, the sums over the keys by len roundings of 2^-24.  For
                # results in bf16 over other pools a probability is one fp16: rounded by half a step, 2^-11.
                mags = (k[see].abs() * x.abs()).sum(-1).max() * abs(sm_scale)
                off = float(mags) * (2.0 ** -22 + (D + 4) * 2.0 ** -24) + \
                    4 * float(s.abs().max() + 1) * 2.0 ** -23 + 2.0 ** -22
                # (the products take fp16's subnormal numbers as 0)
                low = 2.0 ** -14 if cache.dtype == torch.float16 else 0.0
                off += float((torch.where(k[see].abs() < low, k[see].abs(), 0.0) * x.abs()).sum(-1).max()
                             * abs(sm_scale))
                one = q.dtype == torch.bfloat16 and cache.dtype != torch.bfloat16
                share = 2 * off + (2.0 ** -11 if one else 2.0 ** -18) + (int(see.sum()) + 16) * 2.0 ** -24
                room_for[b, i, h] = share * (w[:, None] * v[see].abs()).sum(0) + 1e-30 + \
                    (w[:, None] * torch.where(v[see].abs() < low, v[see].abs(), 0.0)).sum(0)
    return out, room_for


def adjust(logits, r):
    """logits_adjust in 64 bits; r: its arguments as tensors on the CPU."""
    R, V = logits.shape
    out = logits.double().clone()

    def row(name, i, default):
        t = r.get(name)
        return default if t is None else t[i] if t.dim() else t

    for i in range(R):
        x = out[i]
        if r.get("history") is not None:
            ids = r["history"][i] if r["history"].dim() == 2 else r["history"]
            n = min(max(int(row("history_lens", i, len(ids))), 0), len(ids))
            np_ = min(max(int(row("prompt_lens", i, 0)), 0), n)
            ids = ids[:n].long()
            ok = (ids >= 0) & (ids < V)
            late = torch.arange(n) >= np_
            c = torch.bincount(ids[ok & late], minlength=V).double()
            met = (c + torch.bincount(ids[ok & ~late], minlength=V)) > 0
            rep = float(row("repetition", i, 1.0))
            x = torch.where(met, torch.where(x > 0, x / rep, x * rep), x)
            x = x - torch.where(c > 0, float(row("frequency", i, 0.0)) * c + float(row("presence", i, 0.0)), 0.0)
        if r.get("bias_ids") is not None:
            ids = r["bias_ids"][i] if r["bias_ids"].dim() == 2 else r["bias_ids"]
            val = r["bias"][i] if r["bias"].dim() == 2 else r["bias"]
            last = {int(t): float(y) for t, y in zip(ids, val)}
            for t, y in last.items():
                if 0 <= t < V:
                    x[t] += y
        if r.get("allowed") is not None:
            at = int(r["allowed_rows"][i]) if r.get("allowed_rows") is not None else i
            if 0 <= at < r["allowed"].shape[0]:
                x = torch.where(seen_bits(r["allowed"][at], V), x, float("-inf"))
        out[i] = x
    return out


def close(got, want, room, dtype):
    """got (of dtype) within `room` of want, and half a step of dtype."""
    got = got.cpu().double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    half = torch.finfo(dtype).eps / 2
    ok = (got - want).abs() <= room + half * (want.abs() + room) + torch.finfo(dtype).smallest_normal
    bad = ~(same | ok)
    assert not bad.any(), (int(bad.sum()), got[bad][:5], want[bad][:5])
