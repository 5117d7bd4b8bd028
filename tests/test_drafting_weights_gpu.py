"""What each key weighs in the attention of drafted tokens: results whose values nearly cancel, and keys
whose value scales or scores lie far from the others'.

Tolerances.  With w the weights of a row's keys (they add up to 1) and v their values, a result is off
by at most
    sum(w |v|) (2 off + 2^-18 + (keys + 16) 2^-24) + 2^-34 max(w |scale|) sum |code|
and half a step of its type: `off` is the error of a score (queries in two halves, 2^-22 of each product,
D sums of 2^-24, the exponent's roundings), counted twice for a key and the sum; a probability enters
the products in two halves of 11 bits and its rescalings (2^-18 together), or with the smallest step of fp16 next
to a row's largest; sums of fp32 are off by 2^-24 a key.  Where values have no scales, scale = 1."""
import pytest
import torch

import llm_capi
from _drafting import Cache, bits, close

pytestmark = pytest.mark.gpu
I8, E4M3 = torch.int8, torch.float8_e4m3fn
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def put(c, name, b, pos, codes, scale=None):
    """Codes (and the scale) of one token of head 0."""
    at = c.slot(b, 0, pos)
    getattr(c, name)[at] = codes.to(c.dtype)
    if scale is not None:
        c.scales["kv".index(name)][at] = scale


def attention(q, c, contexts, mask, sm_scale):
    """(results, room) in 64 bits of chains or masks [B][N][N], one key head: q [B][N][H][D]."""
    B, N, H, D = q.shape
    out, room = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        L = contexts[b] + N
        k, ok = c.held("k", b, 0, L)
        v, _ = c.held("v", b, 0, L)
        at = torch.tensor([c.slot(b, 0, t) for t in range(L)])
        scale = c.scales[1][at[:, 0], at[:, 1]].double() if c.scales is not None else torch.ones(L).double()
        code = bits(c.v)[at[:, 0], at[:, 1]].view(c.dtype).double()
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
            share = 2 * off + 2.0 ** -18 + (int(see.sum()) + 16) * 2.0 ** -24
            tail = 2.0 ** -34 * (w * scale[see].abs()).amax(1)
            room[b, i] = share[:, None] * (w @ v[see].abs()) + tail[:, None] * code[see].abs().sum(0)
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
