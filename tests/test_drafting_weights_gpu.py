"""What each key weighs in the attention of drafted tokens: results whose values nearly cancel, and keys
whose value scales or scores lie far from the others'.

Tolerances.  With w the weights of a row's keys (they add up to 1) and v their values, a result is off
by at most
    sum(w |v|) (2 off + 2^-17 + (keys + 16) 2^-24)
and half a step of its type: `off` is the error of a score (queries in two halves, 2^-22 of each product,
D sums of 2^-24, the exponent's roundings), counted twice for a key and the sum; a weight enters the products in
two parts of 8 bits at least (half a step of the first is 2^-9 of it, of the second 2^-9 of what is left, 2^-18)
and its roundings ahead of them, 2^-18 in all; sums of fp32 are off by 2^-24 a key.  Over fp16 pages the parts
are fp16: half of the smallest step, 2^-25, of probabilities times 2^11, relative to at most twice the
row's largest, is 2^-35 of it, so 2^-35 max(w) sum |v| more."""
import pytest
import torch

import llm_capi
from _drafting import Cache, close

pytestmark = pytest.mark.gpu
I8, E4M3 = torch.int8, torch.float8_e4m3fn
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def put(c, name, b, pos, codes, scale=None):
    """Codes (and the scale) of one token of head 0."""
    at = c.slot(b, 0, pos)
    getattr(c, name)[at] = codes.to(c.dtype)
    if scale is not None and c.scales is not None:
        c.scales["kv".index(name)][at] = scale


def attention(q, c, contexts, mask, sm_scale, beams=None):
    """(results, room) in 64 bits of chains or masks [B][N][N], one key head: q [B][N][H][D]."""
    B, N, H, D = q.shape
    out, room = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        L = contexts[b] + N
        k, ok = c.held("k", beams[b] if beams else b, 0, L)
        v, _ = c.held("v", beams[b] if beams else b, 0, L)
        j = torch.arange(L) - contexts[b]
        for i in range(N):
            own = torch.arange(N) <= i if mask is None else mask[b, i]
            see = ok & ((j < 0) | own[j.clamp(min=0)])
            x = q[b, i].double()
            s = x @ k[see].T.contiguous() * sm_scale  # [H][keys]
            p = torch.exp(s - s.amax(1, keepdim=True))
            w = p / (p.sum(1, keepdim=True) + 1e-6)
            out[b, i] = w @ v[see]
            off = (x.abs() @ k[see].abs().T.contiguous()).amax(1) * abs(sm_scale) * (2.0 ** -22 + (D + 4) * 2.0 ** -24) \
                + 4 * (s.abs().amax(1) + 1) * 2.0 ** -23 + 2.0 ** -22
            share = 2 * off + 2.0 ** -17 + (int(see.sum()) + 16) * 2.0 ** -24
            room[b, i] = share[:, None] * (w @ v[see].abs())
            if c.dtype == F16:
                room[b, i] += 2.0 ** -35 * w.amax(1)[:, None] * v[see].abs().sum(0)
    return out, room


def check(c, q, contexts, words=None, mask=None, T=None, sm_scale=None, fill=None):
    d = c.cuda()
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    got = llm_capi.pa_tree(q.cuda(), d.k, d.v, d.table, T=max(contexts) if T is None else T,
                           context_lens=i32(contexts), tree_mask=None if words is None else words.cuda(),
                           scales=d.scales, sm_scale=sm_scale)
    want, room = attention(q, c, contexts, mask, sm_scale)
    close(got, want, room, q.dtype)
    return got, want


ROWS = [(3, 2), (21, 2), (50, 2), (40, 5)]  # tokens, query heads: one tile of rows, four, eight


@pytest.mark.parametrize("io", [BF16, F16, F32])
@pytest.mark.parametrize("cache", [F16, I8, E4M3])
@pytest.mark.parametrize("N,H", ROWS)
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_nearly_cancel(gpu, cache, io, N, H, D):
    """Every value meets its negative under almost the same weight: what is left is as small as the
    difference of two probabilities, and as exact as they are."""
    g = torch.Generator().manual_seed(N + D)
    C = 200
    c = Cache(cache, 1, 1, D, 16, C + N, seed=N)
    for pos in range(1, C, 2):
        for name in "kv":
            first = getattr(c, name)[c.slot(0, 0, pos - 1)].float()
            x = -first if name == "v" else first
            s = None if c.scales is None else c.scales["kv".index(name)][c.slot(0, 0, pos - 1)].clone()
            if name == "k":  # (a score next to the first's)
                x[pos % D] += 1.0 if cache == I8 else 0.25
                x = x.clamp(-127, 127) if cache == I8 else x
            put(c, name, 0, pos, x, s)
    for pos in range(C, C + N):  # (the drafts' own values do not count)
        put(c, "v", 0, pos, torch.zeros(D))
    q = (1.5 * torch.randn((1, N, H, D), generator=g)).to(io)
    check(c, q, [C])


def positive_rows(N, H, D, io, g):
    """Queries whose every element is positive, so that a key of one sign scores low for all of them."""
    return (0.5 + torch.rand((1, N, H, D), generator=g)).to(io)


@pytest.mark.parametrize("cache", [I8, E4M3])
@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("N,H", ROWS)
@pytest.mark.parametrize("far", [14, 25, 40, 80])
def test_unseen_drafts_of_large_scales(gpu, cache, io, N, H, far):
    """A drafted token whose value scale is 2^far times the others': rows that do not see it have
    their own values, rows that see it its."""
    g = torch.Generator().manual_seed(far + N)
    C = 77
    c = Cache(cache, 1, 1, 64, 16, C + N, seed=N)
    c.scales[1][c.slot(0, 0, C + 1)] *= 2.0 ** far
    q = (1.5 * torch.randn((1, N, H, 64), generator=g)).to(io)
    mask = torch.eye(N, dtype=torch.bool)[None].clone()
    mask[:, N - 1, 1] = True
    words = torch.zeros((1, N, -(-N // 32) * 32), dtype=torch.int64)
    words[..., :N] = mask
    words = (words.view(1, N, -1, 32) << torch.arange(32)).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    check(c, q, [C], words, mask)
    check(c, q, [C], words, mask, T=4000)


@pytest.mark.parametrize("cache", [I8, E4M3])
@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("N,H", [(1, 1)] + ROWS)
@pytest.mark.parametrize("far", [14, 25, 40, 80])
@pytest.mark.parametrize("pos", [0, 50, 158])
def test_keys_of_no_weight_and_large_scale(gpu, cache, io, N, H, far, pos):
    """A committed key whose score is some 70 below the others' and whose value scale 2^far times theirs,
    ahead of them, among them and behind them."""
    g = torch.Generator().manual_seed(far + N)
    C = 160
    c = Cache(cache, 1, 1, 64, 16, C + N, seed=N)
    q = positive_rows(N, H, 64, io, g)
    put(c, "k", 0, pos, torch.full((64,), -96.0), 70 * 8 / (64 * 96.0))
    c.scales[1][c.slot(0, 0, pos)] *= 2.0 ** far
    check(c, q, [C])


@pytest.mark.parametrize("cache", [I8, E4M3])
@pytest.mark.parametrize("N,H", [(1, 1)] + ROWS)
@pytest.mark.parametrize("up", [0.3, -0.3, 3.0])
def test_scores_that_rise_and_fall(gpu, cache, N, H, up):
    """Scores that go up (or down) by a step from key to key, over scales that go the other way."""
    g = torch.Generator().manual_seed(N)
    C = 320
    c = Cache(cache, 1, 1, 64, 16, C + N, seed=N)
    q = positive_rows(N, H, 64, F32, g)
    for t in range(C + N):
        put(c, "k", 0, t, torch.full((64,), 96.0), (t - C / 2) * up * 8 / (64 * 96.0))
        c.scales[1][c.slot(0, 0, t)] *= 2.0 ** (-(t - C / 2) * up / 4)
    check(c, q, [C])


@pytest.mark.parametrize("cache", [I8, E4M3])
@pytest.mark.parametrize("size", [-140, -120, -100, 100, 118])
def test_scales_of_any_size(gpu, cache, size):
    """Value scales from fp32's subnormal numbers to its largest ones, one of no weight among them."""
    c = Cache(cache, 1, 1, 64, 16, 300, seed=7)
    q = positive_rows(3, 2, 64, F32, torch.Generator().manual_seed(1))
    c.scales[1] = (c.scales[1].double() * 2.0 ** size).float()
    check(c, q, [290])
    c.scales[1][c.slot(0, 0, 40)] = 0.0
    c.scales[1][c.slot(0, 0, 41)] *= -1.0
    check(c, q, [290])


@pytest.mark.parametrize("cache", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("N,H", [(1, 1)] + ROWS)
@pytest.mark.parametrize("far", [12, 20, 26, 32, 60])
def test_many_keys_far_below_one_without_value(gpu, cache, io, N, H, far):
    """A key that has next to all the weight and the value 0: the result is the others', whose weights are 2^-far
    of its."""
    C, D = 700, 64
    c = Cache(cache, 1, 1, D, 16, C + N, seed=far)
    q = positive_rows(N, H, D, io, torch.Generator().manual_seed(far))
    low = 0.25 * far / 96 if cache in (I8, E4M3) else 0.25 * far
    for t in range(C + N):  # scores: far * log 2 and 0 for queries of 1, between half and twice that for these
        put(c, "k", 0, t, torch.full((D,), 96.0 if cache in (I8, E4M3) else low) * (t == 9), low)
    put(c, "v", 0, 9, torch.zeros(D))
    check(c, q, [C], sm_scale=0.6931 * 4 / D)


@pytest.mark.parametrize("io", [F32, F16])
def test_subnormal_elements_of_fp16_pages_count(gpu, io):
    c = Cache(F16, 1, 1, 64, 16, 100, seed=3)
    for x in (c.k, c.v):
        x.copy_((x.float() * 2.0 ** -18).half())
    q = 1000 * positive_rows(5, 4, 64, F32, torch.Generator().manual_seed(2))
    got, want = check(c, q.to(io), [90], sm_scale=4.0)
    assert want.abs().max() > 2.0 ** -21
    if io == F32:
        assert (got != 0).all()


NOT_NUMBERS = [  # beams, B, N, H, contexts of the beams: one tile in parts, by 8 waves, four tiles, eight
    (2, 2, 5, 2, [3060, 126]),
    (4, 64, 2, 2, [700, 638, 900, 520]),
    (1, 1, 30, 2, [3060]),
    (1, 1, 70, 2, [3060]),
]


@pytest.mark.parametrize("cache", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", range(len(NOT_NUMBERS)))
def test_drafts_that_are_not_numbers(gpu, cache, io, D, form):
    """A NaN in the second drafted token's values, infinities in the last one's: the rows that see them have what
    the formula gives, in those dims alone, the others their own results."""
    beams, B, N, H, contexts = NOT_NUMBERS[form]
    g = torch.Generator().manual_seed(D + form)
    c = Cache(cache, beams, 1, D, 16, max(contexts) + N, seed=form)
    for b in range(beams):
        second, last = c.slot(b, 0, contexts[b] + 1), c.slot(b, 0, contexts[b] + N - 1)
        if cache == I8:
            c.scales[1][second] = float("nan")
            c.v[last][7] = 0
        elif cache == E4M3:
            c.v.view(torch.uint8)[second][3] = 0xff
        else:
            c.v[second][3] = float("nan")
            c.v[last][5], c.v[last][6] = float("inf"), -float("inf")
        if c.scales is not None and N > 2:
            c.scales[1][last] = -float("inf")
    ids = [b % beams for b in range(B)]
    of_rows = [contexts[i] for i in ids]
    q = torch.randn((B, N, H, D), generator=g).to(io)
    d = c.cuda()
    got = llm_capi.pa_tree(q.cuda(), d.k, d.v, d.table, T=max(contexts), context_lens=i32(of_rows), beam_ids=i32(ids),
                           scales=d.scales, sm_scale=D ** -0.5).cpu()
    want, room = attention(q, c, of_rows, None, D ** -0.5, ids)
    fine = torch.isfinite(want)
    assert fine[:, 0].all() and not fine[:, 1:].all(-1).any()
    assert torch.equal(got[~fine].double().nan_to_num(7.0), want[~fine].nan_to_num(7.0))
    close(torch.where(fine, got, 0), torch.where(fine, want, 0), torch.where(fine, room, 0), io)


@pytest.mark.parametrize("cache", [F16, BF16, I8, E4M3])
@pytest.mark.parametrize("N,H,D,C,T", [(3, 2, 128, [2500, 31], 2500), (33, 2, 64, [700, 700], 5000),
                                       (5, 64, 128, [1, 200], 200), (100, 3, 256, [128], 1)])
def test_wide_rows_bits_behind_the_tree_and_one_context(gpu, cache, N, H, D, C, T):
    """q and out in wider rows (joined from parts as well), masks whose bits behind the last token are anything,
    pools without scales, and every row at T."""
    B = len(C)
    g = torch.Generator().manual_seed(N + D)
    c = Cache(cache, B, 1, D, 48, max(C) + N, seed=N)
    if cache == I8:
        c.scales = None
    q = ((0.02 if cache == I8 else 1.5) * torch.randn((B, N, H, D), generator=g)).to(BF16)
    words = -(-N // 32)
    full = torch.rand((B, N, words * 32), generator=g) < 0.5
    full[:, torch.arange(N), torch.arange(N)] = True
    w = (full.long().view(B, N, words, 32) << torch.arange(32)).sum(-1)
    w = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
    d = c.cuda()
    wide = torch.full((2, B, N, H * D + 16), 3.25, dtype=BF16, device="cuda")
    qd, out = (x[..., :H * D].unflatten(-1, (H, D)) for x in wide)
    qd.copy_(q)
    one = C[0] == T and len(set(C)) == 1
    got = llm_capi.pa_tree(qd, d.k, d.v, d.table, T=T, context_lens=None if one else i32(C), tree_mask=w.cuda(),
                           scales=d.scales, sm_scale=D ** -0.5, out=out)
    assert (wide[:, ..., H * D:] == 3.25).all() and torch.equal(qd.cpu(), q)
    want, room = attention(q, c, C, full[..., :N], D ** -0.5)
    close(got, want, room, BF16)
    if len(set(C)) == 1:
        got = llm_capi.pa_tree(qd, d.k, d.v, d.table, T=C[0], tree_mask=w.cuda(), scales=d.scales, sm_scale=D ** -0.5)
        close(got, want, room, BF16)


def test_two_calls_at_once(gpu):
    """Two streams with calls in parts, each with a workspace of its own, against the calls alone."""
    c = Cache(I8, 2, 1, 128, 16, 2600, seed=1).cuda()
    q = [torch.randn((2, n, 4, 128), generator=torch.Generator().manual_seed(n)).cuda() for n in (2, 30)]
    call = lambda x: llm_capi.pa_tree(x, c.k, c.v, c.table, T=2500, context_lens=i32([2500, 1900]), scales=c.scales,
                                      sm_scale=0.09)
    want = [call(x) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(q[i]))
    torch.cuda.synchronize()
    for x, ys in zip(want, got):
        assert all(torch.equal(x, y) for y in ys)
