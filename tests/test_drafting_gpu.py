"""The quantised cache, the attention of drafted tokens and the logit rules against plain
64-bit forms, at the sizes, masks and values where they can go wrong."""
import numpy as np
import pytest
import torch

import llm_capi
from _drafting import LARGEST, Cache, adjust, bits, close, quantise, seen_bits, tree

pytestmark = pytest.mark.gpu
I8, E4M3 = torch.int8, torch.float8_e4m3fn
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# -- the cache --------------------------------------------------------------------------

def special_rows(x):
    """Rows that are 0, tiny, huge, all ties, and not finite (x [rows][D], changed)."""
    D = x.shape[-1]
    big = torch.finfo(x.dtype).max
    x[0] = 0.0
    if len(x) > 1:
        x[1] = torch.finfo(x.dtype).tiny * 1.5 * torch.sign(x[1])
    if len(x) > 2:
        x[2] = big
        x[2, ::2] = -big / 2
    if len(x) > 3:  # codes of int8 that are halves: largest 254, odd numbers
        x[3] = torch.arange(D) % 128 * 2 - 127
        x[3, 0] = 254.0
    if len(x) > 4:  # halves of e4m3: largest 448, numbers between its steps of 32, 2 and 2^-9
        x[4] = torch.tensor([448.0, 272.0, 304.0, -272.0, 17.0, 19.0, -17.0, 2.0 ** -10] * (D // 8))
    if len(x) > 5:
        x[5, D // 2] = float("nan")
    if len(x) > 6:
        x[6, D - 1] = -float("inf")
    if len(x) > 7:
        x[7] = -0.0


@pytest.mark.parametrize("cache", [I8, E4M3])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("B,N,heads,D,page", [
    (1, 1, 1, 64, 16), (3, 1, 5, 128, 16), (2, 21, 12, 64, 16), (3, 7, 2, 256, 32), (1, 130, 3, 128, 5 * 16),
    (2, 17, 1, 8, 6), (2, 33, 3, 24, 4), (1, 40, 2, 200, 10)])
def test_write_and_read(gpu, cache, io, B, N, heads, D, page):
    c = Cache(cache, B, heads, D, page, 50 + N, seed=N + D)
    g = torch.Generator().manual_seed(D + N)
    k = (torch.randn((B, N, heads, D), generator=g) * 3).to(io)
    v = torch.randn((B, N, heads, D), generator=g).to(io)
    special_rows(k.view(-1, D))
    special_rows(v.view(-1, D).flip(0))
    starts = [0, 13, 50][:B]
    lens = [N, max(N // 2, 1), N + 5][:B]
    d = c.cuda()
    llm_capi.kv_quant_write(k.cuda(), v.cuda(), d.k, d.v, d.table, *d.scales, starts=i32(starts), lens=i32(lens))
    back = [torch.full((B, N, heads, D), 7.0, dtype=io, device="cuda") for _ in "kv"]
    llm_capi.kv_quant_read(d.k, d.v, d.table, *d.scales, starts=i32(starts), lens=i32(lens), out=back)
    for name, x, got in zip("kv", (k, v), back):
        code, scale = quantise(x, cache)
        pool, held = getattr(c, name).clone(), c.scales["kv".index(name)].clone()
        want = torch.full((B, N, heads, D), 7.0, dtype=io)
        for b in range(B):
            for j in range(min(lens[b], N)):
                for h in range(heads):
                    at = c.slot(b, h, starts[b] + j)
                    if at is None:
                        want[b, j, h] = 0.0
                        continue
                    pool[at] = code[b, j, h].to(cache)
                    held[at] = scale[b, j, h]
                    want[b, j, h] = (code[b, j, h].float() * scale[b, j, h]).to(io)
        # every code is that of exact arithmetic (e4m3's two zeros are one), and nothing else moved
        assert torch.equal(getattr(d, name).cpu().float(), pool.float()), name
        assert torch.equal(d.scales["kv".index(name)].cpu().nan_to_num(-1.0), held.nan_to_num(-1.0)), name
        assert torch.equal(got.cpu().nan_to_num(-1.0), want.nan_to_num(-1.0)), name


@pytest.mark.parametrize("cache", [I8, E4M3])
def test_codes_near_borders(gpu, cache):
    """fp32 values one step of fp32 on either side of where two codes meet."""
    D, rows = 256, 64
    g = torch.Generator().manual_seed(5)
    top = torch.rand((rows, 1), generator=g, dtype=torch.float64) * 5 + 0.1
    top = top.float().double()
    if cache == I8:
        border = torch.randint(-127, 127, (rows, D), generator=g) + 0.5
    else:
        grid = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
        at = torch.randint(0, 126, (rows, D), generator=g)
        border = (grid[at] + grid[at + 1]) / 2
    x = (border * top / LARGEST[cache]).float()
    step = torch.randint(-1, 2, (rows, D), generator=g)
    x = (x.view(torch.int32) + step.to(torch.int32)).view(F32)
    x[:, 0] = top[:, 0].float()
    c = Cache(cache, 1, 1, D, 16, rows, seed=1)
    d = c.cuda()
    k = x.view(1, rows, 1, D)
    llm_capi.kv_quant_write(k.cuda(), (-k).cuda(), d.k, d.v, d.table, *d.scales, starts=i32([0]))
    code, _ = quantise(x, cache)
    page = c.table[0, 0].long()
    assert torch.equal(d.k.cpu().float()[page].view(-1, D)[:rows], code.float())
    assert torch.equal(d.v.cpu().float()[page].view(-1, D)[:rows], -code.float())


def test_write_leaves_out(gpu):
    """Positions without a page, negative ones, beams that the table does not have, empty rows."""
    c = Cache(I8, 4, 2, 64, 16, 64, seed=3)
    c.table[1, 0, 2] = -1
    c.table[1, 1, 1] = c.pages
    c.table[2, :, 3] = -7
    d = c.cuda()
    B, N = 6, 40
    k = torch.randn((B, N, 2, 64), generator=torch.Generator().manual_seed(1))
    starts, lens, beams = [30, 10, -5, 2 ** 31 - 20, 0, 3], [40, 40, 20, 40, -3, 40], [0, 1, 2, 3, 0, 9]
    args = dict(starts=i32(starts), lens=i32(lens), beam_ids=i32(beams))
    llm_capi.kv_quant_write(k.cuda(), k.cuda(), d.k, d.v, d.table, *d.scales, **args)
    code, scale = quantise(k, I8)
    pool, held = c.k.clone(), c.scales[0].clone()
    want = torch.zeros((B, N, 2, 64))
    for b in range(B):
        for j in range(max(min(lens[b], N), 0)):
            for h in range(2):
                at = c.slot(beams[b], h, starts[b] + j)
                if at is not None:
                    pool[at], held[at] = code[b, j, h].to(I8), scale[b, j, h]
                    want[b, j, h] = code[b, j, h].float() * scale[b, j, h]
    assert torch.equal(d.k.cpu(), pool) and torch.equal(d.scales[0].cpu(), held)
    got, _ = llm_capi.kv_quant_read(d.k, d.v, d.table, *d.scales, N=N, **args)
    assert torch.equal(got.cpu(), want)


def test_later_row_of_a_beam_is_kept(gpu):
    B, N = 130, 5
    c = Cache(E4M3, 3, 2, 128, 16, 32, seed=4)
    g = torch.Generator().manual_seed(2)
    k = torch.randn((B, N, 2, 128), generator=g)
    starts, lens = torch.randint(0, 28, (B,), generator=g).tolist(), torch.randint(0, 6, (B,), generator=g).tolist()
    beams = torch.randint(0, 3, (B,), generator=g).tolist()
    code, scale = quantise(k, E4M3)
    pool, held = c.k.float(), c.scales[0].clone()
    for b in range(B):
        for j in range(lens[b]):
            for h in range(2):
                at = c.slot(beams[b], h, starts[b] + j)
                pool[at], held[at] = code[b, j, h].float(), scale[b, j, h]
    for _ in range(3):
        d = c.cuda()
        llm_capi.kv_quant_write(k.cuda(), k.cuda(), d.k, d.v, d.table, *d.scales, starts=i32(starts), lens=i32(lens),
                                beam_ids=i32(beams))
        assert torch.equal(d.k.cpu().float(), pool) and torch.equal(d.scales[0].cpu(), held)


def test_views(gpu):
    """K and V out of a fused projection, interleaved pages, strided scales."""
    B, N, H, D = 2, 9, 3, 64
    c = Cache(I8, B, H, D, 16, 40, seed=6)
    qkv = torch.randn((B, N, 3 * H * D), generator=torch.Generator().manual_seed(3)).to(F16)
    k, v = (qkv[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in (1, 2))
    kv = torch.stack((c.k, c.v), 1).cuda()
    sc = torch.stack(c.scales, 1).cuda()
    fused = qkv.cuda()
    kd, vd = (fused[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in (1, 2))
    args = (kv[:, 0], kv[:, 1], c.table.cuda(), sc[:, 0], sc[:, 1])
    llm_capi.kv_quant_write(kd, vd, *args, starts=i32([3, 20]))
    d = c.cuda()
    llm_capi.kv_quant_write(k.contiguous().cuda(), v.contiguous().cuda(), d.k, d.v, d.table, *d.scales,
                            starts=i32([3, 20]))
    assert torch.equal(kv, torch.stack((d.k, d.v), 1)) and torch.equal(sc, torch.stack(d.scales, 1))
    out = torch.zeros((B, N, 2 * H * D), device="cuda")
    parts = [out[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in (0, 1)]
    llm_capi.kv_quant_read(*args, starts=i32([3, 20]), out=parts)
    want = llm_capi.kv_quant_read(d.k, d.v, d.table, *d.scales, starts=i32([3, 20]), N=N)
    assert torch.equal(parts[0], want[0]) and torch.equal(parts[1], want[1])
    q = fused[..., :H * D].unflatten(-1, (H, D))
    ctx = i32([3, 20])
    a = llm_capi.pa_tree(q, *args[:3], T=32, context_lens=ctx, scales=args[3:])
    b = llm_capi.pa_tree(q.contiguous(), d.k, d.v, d.table, T=32, context_lens=ctx, scales=d.scales)
    assert torch.equal(a, b)


# -- drafted tokens ---------------------------------------------------------------------

def random_tree(B, N, g):
    parents = torch.stack([(torch.rand(N, generator=g) * (torch.arange(N) + 1)).long() - 1 for _ in range(B)])
    words = llm_capi.tree_mask(parents)
    return words, seen_bits(words, N)


def check_tree(c, q, contexts, lens, words, mask, T=None, beams=None, scale=None, fill=3.25):
    d = c.cuda()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.full(q.shape, fill, dtype=q.dtype, device="cuda")
    got = llm_capi.pa_tree(q.cuda(), d.k, d.v, d.table, T=max(contexts) if T is None else T,
                           context_lens=i32(contexts), tree_mask=None if words is None else words.cuda(),
                           tree_lens=None if lens is None else i32(lens),
                           beam_ids=None if beams is None else i32(beams), scales=d.scales, sm_scale=scale, out=out)
    assert got is out
    N = q.shape[1]
    n = lens or [N] * len(contexts)
    want, room = tree(q, c, contexts, n, mask, beams, scale)
    for b in range(len(contexts)):
        m = min(max(n[b], 0), N)
        close(got[b, :m], want[b, :m], room[b, :m], q.dtype)
        assert (got[b, m:] == fill).all()
    return got


TREES = [  # B, N, heads, group, D, page, contexts
    (1, 1, 1, 1, 64, 16, [0]),
    (1, 1, 2, 1, 128, 16, [1]),
    (2, 1, 2, 4, 64, 32, [31, 700]),
    (3, 8, 4, 1, 64, 16, [113, 0, 15]),
    (2, 21, 1, 8, 128, 16, [33, 260]),
    (2, 17, 2, 1, 256, 16, [100, 31]),
    (1, 63, 2, 1, 128, 32, [1000]),
    (2, 70, 1, 3, 64, 48, [64, 500]),
    (2, 5, 3, 1, 128, 16, [127, 128]),
]


@pytest.mark.parametrize("cache", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(TREES)))
def test_tree(gpu, cache, io, case):
    B, N, heads, group, D, page, contexts = TREES[case]
    g = torch.Generator().manual_seed(case)
    c = Cache(cache, B, heads, D, page, max(contexts) + N, seed=case)
    q = (1.5 * torch.randn((B, N, heads * group, D), generator=g)).to(io)
    words, mask = random_tree(B, N, g)
    lens = [max(1, N - 3 * b) for b in range(B)]
    check_tree(c, q, contexts, lens, words, mask)


@pytest.mark.parametrize("cache,D", [(F16, 64), (BF16, 128), (I8, 128), (E4M3, 64), (I8, 256)])
def test_long_rows_in_parts(gpu, cache, D):
    """Rows of very different lengths over many splits, and a T that is far too small."""
    g = torch.Generator().manual_seed(D)
    contexts = [9000, 0, 257, 4096]
    c = Cache(cache, 4, 1, D, 16, 9020, seed=D)
    q = (1.5 * torch.randn((4, 3, 2, D), generator=g)).to(F32)
    words, mask = random_tree(4, 3, g)
    a = check_tree(c, q, contexts, [3, 2, 3, 0], words, mask)
    for T in (1, 300, 100000):
        check_tree(c, q, contexts, [3, 2, 3, 0], words, mask, T=T)


FORMS = [  # beams, B, N, heads, group, D, contexts
    (4, 16, 2, 4, 1, 128, [700, 30, 513, 1]),  # 64 pairs of long rows
    (2, 2, 60, 4, 5, 64, [3000, 40]),  # groups of rows, many parts of them
    (2, 2, 25, 2, 1, 128, [1900, 900]),  # two tiles in parts
    (1, 1, 1024, 1, 1, 64, [1500]),  # the most tokens
    (4, 128, 1, 4, 2, 64, [2300, 2047, 100, 2048]),  # pairs that fill the card, in parts
]


@pytest.mark.parametrize("cache,io", [(F16, F32), (BF16, BF16), (I8, F16), (E4M3, F32), (E4M3, BF16)])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_forms(gpu, cache, io, form):
    """Batches that are split over keys, rows and waves in the different ways, several rows to a beam, the
    tokens in chains."""
    beams, B, N, heads, group, D, contexts = FORMS[form]
    g = torch.Generator().manual_seed(100 + form)
    c = Cache(cache, beams, heads, D, 16, max(contexts) + N, seed=form)
    q = (1.5 * torch.randn((B, N, heads * group, D), generator=g)).to(io)
    ids = [b % beams for b in range(B)]
    check_tree(c, q, [contexts[i] for i in ids], [N - b % 2 * (N // 3) for b in range(B)], None, None, beams=ids)


@pytest.mark.parametrize("cache", [F16, BF16, I8, E4M3])
def test_masks_and_missing_pages(gpu, cache):
    """Rows that see nothing, trees of several words, pages that are missing under either half of
    a block, contexts past the table, beams in any order and outside it."""
    g = torch.Generator().manual_seed(11)
    N, D, B = 40, 64, 7
    c = Cache(cache, 4, 2, D, 16, 160, seed=12)
    c.table[0, 0, 1], c.table[0, 1, 2], c.table[1, :, :] = -1, c.pages, -5
    c.table[2, 0, 8] = -1
    contexts, lens, beams = [70, 50, 120, 0, -9, 1000, 20], [40, 40, 40, 40, 40, 40, 0], [0, 1, 2, 3, 3, 2, 9]
    q = torch.randn((B, N, 2, D), generator=g)
    mask = torch.rand((B, N, N), generator=g) < 0.2
    mask[:, 3] = False  # (sees the context alone, or nothing)
    mask[4] = False
    words = torch.zeros((B, N, 64), dtype=torch.int64)
    words[..., :N] = mask
    words = (words.view(B, N, 2, 32) << torch.arange(32)).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    got = check_tree(c, q, contexts, lens, words, mask, beams=beams, T=160)
    assert (got[1] == 0).sum() > 0 and (got[4] == 0).all()
    check_tree(c, q, contexts, lens, None, None, beams=beams, T=160)


@pytest.mark.parametrize("cache", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("group", [1, 8])
def test_what_is_not_seen_has_no_part(gpu, cache, group):
    """NaN and infinities behind the rows' ends, in pages of nobody and in drafted tokens that
    some rows see: those rows alone have them."""
    g = torch.Generator().manual_seed(21)
    N, D = 12, 64
    contexts = [50, 5]
    c = Cache(cache, 2, 1, D, 16, 70, seed=22)
    nan = torch.tensor(float("nan"))
    q = torch.randn((2, N, group, D), generator=g)
    words, mask = random_tree(2, N, g)
    used = torch.zeros((c.pages, 16), dtype=torch.bool)
    for b in range(2):
        for p in range(contexts[b] + N):
            used[c.slot(b, 0, p)] = True
    for pool in (c.k, c.v):
        if cache == E4M3:
            pool.view(torch.uint8)[~used] = 0x7f
        elif cache != I8:
            pool[~used] = nan.to(cache)
    if c.scales is not None:
        for s in c.scales:
            s[~used] = nan
    check_tree(c, q, contexts, None, words, mask)  # nothing of that arrives
    # drafted token 4 of row 0 has a NaN, token 7 of row 1 infinities of both signs
    n4, n7 = c.slot(0, 0, contexts[0] + 4), c.slot(1, 0, contexts[1] + 7)
    if cache in (F16, BF16):
        c.v[n4][3] = nan.to(cache)
        c.v[n7][5], c.v[n7][6] = float("inf"), -float("inf")
        c.k[n7][0] = nan.to(cache)
    elif cache == E4M3:
        c.v.view(torch.uint8)[n4][3] = 0xff
        c.scales[0][n7] = nan
    else:
        c.scales[1][n4] = nan
        c.scales[0][n7] = float("inf")
    d = c.cuda()
    got = llm_capi.pa_tree(q.cuda(), d.k, d.v, d.table, T=64, context_lens=i32(contexts), tree_mask=words.cuda(),
                           scales=d.scales, sm_scale=0.125).cpu()
    for b, j in ((0, 4), (1, 7)):
        assert mask[b, :, j].any() and not mask[b, :, j].all()
        sees = mask[b, :, j]
        assert torch.isfinite(got[b][~sees]).all()
        # (an infinite key scale: a score of -infinity weighs nothing, the formula's own result)
        key = bits(c.k)[c.slot(b, 0, contexts[b] + j)].view(cache).double()
        gone = (q[b][sees].double() @ key < 0) & (cache == I8) & (b == 1)
        assert ((~torch.isfinite(got[b][sees])).any(-1) ^ gone).all()
    # rows that do not see them are as if they were not there; of the dims, the NaN's own alone
    clean = Cache(cache, 2, 1, D, 16, 70, seed=22)
    want, room = tree(q, clean, contexts, [N, N], mask, None, 0.125)
    for b, j in ((0, 4), (1, 7)):
        close(got[b][~mask[b, :, j]], want[b][~mask[b, :, j]], room[b][~mask[b, :, j]], F32)
    if cache in (F16, BF16, E4M3):
        hurt = ~torch.isfinite(got[0][mask[0, :, 4]])
        assert hurt[..., 3].all() and hurt.sum() == hurt[..., 3].sum()


def test_scores_and_scales_at_their_ends(gpu):
    """Large scores, a negative and a zero scale, queries of any size, value scales far apart."""
    g = torch.Generator().manual_seed(31)
    c = Cache(I8, 1, 1, 64, 16, 300, seed=32)
    q = torch.randn((1, 4, 2, 64), generator=g)
    for scale in (20.0, -0.5, 0.0, 1e-3):
        check_tree(c, q, [290], None, None, None, scale=scale)
    for size in (1e-20, 1e12, 0.0):
        check_tree(c, q * size, [290], None, None, None, scale=0.125 / size if size else 0.125)
    c.scales[1] *= 10.0 ** torch.linspace(-6, 6, 16)
    check_tree(c, q, [290], None, None, None)
    c.scales[1].zero_()
    check_tree(c, q, [290], None, None, None)
    # small value scales behind blocks that hold none, a first page that is missing, queries of any size
    for cache in (I8, E4M3):
        c = Cache(cache, 1, 1, 64, 16, 300, seed=33)
        c.scales[1] *= 1e-6
        c.table[0, 0, :4] = -1
        check_tree(c, q, [290], None, None, None)
        c.scales[1][c.table[0, 0, 4:9].long()] = 0.0
        check_tree(c, q, [290], None, None, None)
        check_tree(c, q.repeat(1, 1, 20, 1), [290], None, None, None)
    c = Cache(F16, 1, 1, 64, 16, 300, seed=34)
    check_tree(c, q * 1e32, [290], None, None, None, scale=1e-33)
    raw = Cache(I8, 1, 1, 64, 16, 300, seed=32)  # without scales: the codes themselves
    raw.scales = None
    check_tree(raw, q * 0.01, [290], None, None, None)


def test_single_tokens_are_pa_decode(gpu):
    """N = 1 over fp16 pages: the step of single tokens, as pa_decode has it."""
    B, H, D = 5, 3, 128
    c = Cache(F16, B, H, D, 16, 600, seed=41)
    q = torch.randn((B, 1, H, D), generator=torch.Generator().manual_seed(42))
    d = c.cuda()
    ctx = [599, 0, 16, 31, 300]
    got = llm_capi.pa_tree(q.cuda(), d.k, d.v, d.table, T=600, context_lens=i32(ctx), sm_scale=0.09)
    same = llm_capi.pa_decode(q[:, 0].cuda(), d.k, d.v, d.table, T=600, context_lens=i32([x + 1 for x in ctx]),
                              sm_scale=0.09)
    want, room = tree(q, c, ctx, [1] * B, None, None, 0.09)
    close(got, want, room, F32)
    close(same[:, None], want, room, F32)


@pytest.mark.parametrize("cache,D", [(F16, 256), (I8, 256)])
def test_pools_past_32_bits(gpu, cache, D):
    """Pages that lie more than 4 GiB into a pool."""
    size = torch.empty(0, dtype=cache).element_size() * 16 * D
    pages = (5 << 30) // size
    small = Cache(cache, 1, 1, D, 16, 100, seed=51)
    far = torch.randperm(1000)[:small.tiles] + pages - 1000
    pools = []
    for x in (small.k, small.v):
        pool = torch.empty((pages, 16, D), dtype=cache, device="cuda")
        pool[far.cuda()] = x[small.table[0, 0].long()].cuda()
        pools.append(pool)
    table = far.to(torch.int32).view(1, 1, -1).cuda()
    scales = None
    if small.scales is not None:
        scales = []
        for s in small.scales:
            t = torch.zeros((pages, 16), device="cuda")
            t[far.cuda()] = s[small.table[0, 0].long()].cuda()
            scales.append(t)
    q = torch.randn((1, 3, 2, D), generator=torch.Generator().manual_seed(1))
    got = llm_capi.pa_tree(q.cuda(), *pools, table, T=90, context_lens=i32([90]), scales=scales, sm_scale=0.06)
    want, room = tree(q, small, [90], [3], None, None, 0.06)
    close(got, want, room, F32)
    if scales:
        k = torch.randn((1, 20, 1, D), generator=torch.Generator().manual_seed(2))
        llm_capi.kv_quant_write(k.cuda(), k.cuda(), *pools, table, *scales, starts=i32([70]))
        code, scale = quantise(k, cache)
        back, _ = llm_capi.kv_quant_read(*pools, table, *scales, starts=i32([70]), N=20)
        assert torch.equal(back.cpu(), code.float() * scale[..., None])


# -- logits -----------------------------------------------------------------------------

def rules(R, V, L, n, M, seed, shared=False):
    g = torch.Generator().manual_seed(seed)
    r = {}
    if L:
        shape = (L,) if shared else (R, L)
        r["history"] = (V * torch.rand(shape, generator=g) ** 4 - 1).round().to(torch.int32)
        r["history"].view(-1)[::17] = V + 3  # outside the vocabulary, as -1 is
        r["history_lens"] = torch.randint(-2, L + 3, (R,), generator=g, dtype=torch.int32)
        r["prompt_lens"] = torch.randint(-1, L + 1, (R,), generator=g, dtype=torch.int32)
        r["repetition"] = 0.7 + torch.rand(R, generator=g)
        r["frequency"] = torch.rand(R, generator=g) - 0.2
        r["presence"] = torch.rand(R, generator=g) - 0.2
    if n:
        shape = (n,) if shared else (R, n)
        r["bias_ids"] = torch.randint(-1, V + 1, shape, generator=g, dtype=torch.int32)
        r["bias"] = 5 * torch.randn(shape, generator=g)
    if M:
        r["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (M, -(-V // 32)), generator=g).to(torch.int32)
        r["allowed"][0] = 0
        r["allowed_rows"] = torch.randint(-1, M + 1, (R,), generator=g, dtype=torch.int32)
    return r


def check_logits(logits, r, out=None, on=None):
    args = {k: t.cuda() for k, t in r.items()}
    x = logits.cuda() if on is None else on
    got = llm_capi.logits_adjust(x, out=out, **args)
    want = adjust(logits, r)
    # fp32: a quotient or product, the sum c frequency + presence, two additions: 5 roundings of what
    # they meet at most, |x| times the penalty, c frequency + presence, the bias
    size = logits.double().abs() * 2 + want.abs().nan_to_num(0, 0, 0)
    if "frequency" in r:
        size = size + r["history"].shape[-1] + 1
    if "bias" in r:
        size = size + 30
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got.cpu()), fine) and torch.equal(got.cpu()[~fine].double().nan_to_num(1.5),
                                                                        want[~fine].nan_to_num(1.5))
    close(torch.where(fine, got.cpu(), 0), torch.where(fine, want, 0), torch.where(fine, 5 * size * 2.0 ** -24, 0),
          logits.dtype)
    return got


@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("R,V,L,n,M", [(1, 1, 1, 1, 1), (2, 31, 5, 0, 2), (3, 257, 40, 9, 0), (5, 4097, 700, 33, 5),
                                       (2, 50257, 3000, 300, 2), (7, 32768, 0, 5, 3), (3, 8195, 64, 0, 0),
                                       (64, 1000, 129, 3, 64), (1, 200003, 999, 40, 1), (2, 3, 0, 0, 0)])
def test_logits(gpu, io, R, V, L, n, M):
    g = torch.Generator().manual_seed(V)
    logits = (4 * torch.randn((R, V), generator=g)).to(io)
    logits.view(-1)[::7] = 0.0
    if V > 30:
        logits[0, 3], logits[0, 5], logits[0, 7] = float("inf"), -float("inf"), float("nan")
    check_logits(logits, rules(R, V, L, n, M, seed=V + L))
    if L and n:
        check_logits(logits, rules(R, V, L, n, M, seed=V, shared=True))


def test_logits_rules_by_themselves(gpu):
    logits = torch.randn((6, 1003), generator=torch.Generator().manual_seed(1))
    full = rules(6, 1003, 50, 9, 6, seed=2)
    for keep in (["history", "repetition"], ["history", "frequency"], ["history", "presence", "history_lens"],
                 ["history", "history_lens", "prompt_lens", "repetition", "presence"], ["bias_ids", "bias"],
                 ["allowed"], ["allowed", "allowed_rows"], ["history"]):
        check_logits(logits, {k: full[k] for k in keep})
    empty = {**full, "history": torch.zeros((6, 0), dtype=torch.int32), "bias_ids": torch.zeros((6, 0), dtype=torch.int32),
             "bias": torch.zeros((6, 0))}
    check_logits(logits, empty)
    with pytest.raises(llm_capi.LlmError):
        llm_capi.logits_adjust(logits.cuda(), repetition=torch.ones(6, device="cuda"))


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_logits_in_place_and_strided(gpu, io, shift):
    R, V = 4, 2001
    logits = torch.randn((R, V), generator=torch.Generator().manual_seed(3)).to(io)
    r = rules(R, V, 60, 5, 4, seed=4)
    wide = torch.full((R, V + 9), 3.0, dtype=io, device="cuda")
    mine = wide[:, shift:shift + V]
    mine.copy_(logits)
    other = torch.full((R, V + 9), 4.0, dtype=io, device="cuda")  # another alignment
    a = check_logits(logits, r, out=other[:, 2:2 + V], on=mine)
    assert torch.equal(mine.cpu(), logits) and (other[:, :2] == 4).all() and (other[:, 2 + V:] == 4).all()
    b = check_logits(logits, r, out=mine, on=mine)
    assert torch.equal(a, b) and b is mine
    assert (wide[:, :shift] == 3).all() and (wide[:, shift + V:] == 3).all()


# -- together ---------------------------------------------------------------------------

class Step:
    """A verification step: drafted keys and values written, attention, logits, rules, tokens."""

    def __init__(self, cache=I8, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.B, self.N, self.H, self.D, V = 3, 6, 4, 64, 513
        self.contexts = [100, 37, 260]
        self.c = Cache(cache, self.B, self.H, self.D, 16, 300, seed=seed)
        self.d = self.c.cuda()
        self.qkv = torch.randn((self.B, self.N, 3, self.H, self.D), generator=g).to(F16).cuda()
        self.words, self.mask = random_tree(self.B, self.N, g)
        self.wd, self.ctx = self.words.cuda(), i32(self.contexts)
        self.emb = (0.1 * torch.randn((V, self.H * self.D), generator=g)).to(F16).cuda()
        self.rules = rules(self.B * self.N, V, 30, 4, 5, seed=seed + 1)
        self.rules["allowed"][0] = -1
        self.rd = {k: t.cuda() for k, t in self.rules.items()}

    def run(self, stream=None):
        q, k, v = self.qkv.unbind(2)
        d = self.d
        llm_capi.kv_quant_write(k, v, d.k, d.v, d.table, *d.scales, starts=self.ctx, stream=stream)
        att = llm_capi.pa_tree(q, d.k, d.v, d.table, T=300, context_lens=self.ctx, tree_mask=self.wd,
                               scales=d.scales, sm_scale=0.125, stream=stream)
        x = att.view(self.B * self.N, -1).float()
        logits = llm_capi.lm_head(x, self.emb, stream=stream)
        llm_capi.logits_adjust(logits, out=logits, stream=stream, **self.rd)
        return att, logits, llm_capi.argmax_rows(logits, stream=stream)


@pytest.mark.parametrize("cache", [I8, E4M3])
def test_a_step_together(gpu, cache):
    s = Step(cache)
    att, logits, ids = s.run()
    q, k, v = (t.cpu() for t in s.qkv.unbind(2))
    for name, x in (("k", k), ("v", v)):  # the pages as they should be
        code, scale = quantise(x, cache)
        for b in range(s.B):
            for j in range(s.N):
                for h in range(s.H):
                    at = s.c.slot(b, h, s.contexts[b] + j)
                    getattr(s.c, name)[at] = code[b, j, h].to(cache)
                    s.c.scales["kv".index(name)][at] = scale[b, j, h]
        assert torch.equal(bits(getattr(s.d, name).cpu()), bits(getattr(s.c, name)))
    want, room = tree(q, s.c, s.contexts, [s.N] * s.B, s.mask, None, 0.125)
    close(att, want, room, F16)
    raw = att.cpu().double().view(s.B * s.N, -1) @ s.emb.cpu().double().T
    final = adjust(raw, s.rules)
    fine = torch.isfinite(final)
    assert torch.equal(torch.isfinite(logits.cpu()), fine)
    # lm_head's halves and sums of 256 fp32 products, then the rules' roundings
    size = (att.cpu().double().abs().view(s.B * s.N, -1) @ s.emb.cpu().double().abs().T) * 2 + 70
    close(torch.where(fine, logits.cpu(), 0), torch.where(fine, final, 0), torch.where(fine, size * 2.0 ** -16, 0), F32)
    assert torch.equal(ids.cpu().long(), logits.cpu().argmax(-1))


def test_another_stream(gpu):
    a, b = Step(seed=3), Step(seed=3)
    want = a.run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b.qkv += 0
    s.synchronize()
    with torch.cuda.stream(s):  # (the step's own torch operations follow the current stream)
        got = b.run(stream=s)
    s.synchronize()
    for x, y in zip(want, got):
        assert torch.equal(x, y)


def test_captured_steps(gpu):
    """Two captured steps of different rows, replayed in turn with eager work between, each as the
    eager step: new queries, contexts and rules reach the replays."""
    steps = [Step(seed=5), Step(E4M3, seed=6)]
    for s in steps:
        s.run()
    torch.cuda.synchronize()
    graphs = []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.out = s.run()
        graphs.append(g)
    for turn in range(4):
        for s, g in zip(steps, graphs):
            s.qkv.copy_(torch.randn(s.qkv.shape, generator=torch.Generator().manual_seed(turn)).to(F16))
            s.ctx += 1
            s.rd["frequency"] += 0.1
            g.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in s.out]
            pools = [bits(s.d.k).clone(), s.d.scales[1].clone()]
            want = s.run()
            for x, y in zip(want, got):
                assert torch.equal(x, y)
            assert torch.equal(pools[0], bits(s.d.k)) and torch.equal(pools[1], s.d.scales[1])


def test_python_refusals(gpu):
    s = Step()
    d = s.d
    q, k, v = s.qkv.unbind(2)
    cache = (d.k, d.v, d.table)
    ok = dict(starts=s.ctx)
    for bad in (dict(starts=s.ctx.long()), dict(starts=s.ctx.cpu()), dict(starts=s.ctx[:2]),
                dict(starts=s.ctx, lens=s.ctx[None])):
        with pytest.raises((TypeError, ValueError)):
            llm_capi.kv_quant_write(k, v, *cache, *d.scales, **bad)
    for kk, vv in ((k, v[:, :3]), (k, v.float()), (k.cpu(), v.cpu()), (k.transpose(1, 2), v.transpose(1, 2)),
                   (k[..., :32], v[..., :32]), (k.int(), v.int())):
        with pytest.raises((TypeError, ValueError)):
            llm_capi.kv_quant_write(kk, vv, *cache, *d.scales, **ok)
    with pytest.raises((TypeError, ValueError)):
        llm_capi.kv_quant_write(k, v, *cache, d.scales[0].half(), d.scales[1], **ok)
    with pytest.raises((TypeError, ValueError)):
        llm_capi.kv_quant_write(k, v, *cache, d.scales[0][:5], d.scales[1][:5], **ok)
    for bad in (dict(tree_mask=s.wd[:, :2]), dict(tree_mask=s.wd.long()), dict(context_lens=s.ctx.float()),
                dict(out=torch.empty_like(q, dtype=F32)), dict(tree_lens=s.ctx[:1])):
        with pytest.raises((TypeError, ValueError)):
            llm_capi.pa_tree(q, *cache, T=300, scales=d.scales, **bad)
    with pytest.raises((TypeError, ValueError)):  # more rows than the table has
        llm_capi.pa_tree(q.repeat(2, 1, 1, 1), *cache, T=300, scales=d.scales)
    with pytest.raises(llm_capi.LlmError):
        llm_capi.pa_tree(q[..., :3, :], d.k, d.v, d.table, T=300, scales=d.scales)
    x = torch.zeros((2, 40), device="cuda")
    for bad in (dict(history=x), dict(history=i32([[1]])), dict(allowed=i32([[1], [1]])), dict(bias=x),
                dict(out=x[:1]), dict(history=i32([1]), frequency=x[0])):
        with pytest.raises((TypeError, ValueError)):
            llm_capi.logits_adjust(x, **bad)


def test_scales_go_together(gpu):
    s = Step()
    q = torch.zeros((s.d.table.shape[0], 1, s.d.table.shape[1], s.d.k.shape[2]), device="cuda")
    for bad in ((s.d.scales[0], None), (None, s.d.scales[1])):
        with pytest.raises(ValueError):
            llm_capi.pa_tree(q, s.d.k, s.d.v, s.d.table, T=1, scales=bad)
