"""The steps of a program that verifies drafted tokens over a quantised paged cache, as
cases that can be timed and compared.

    store    new keys and values quantised into pages (kv_quant_write) and read back
    read     a stretch of a quantised cache read back (kv_quant_read)
    tree     attention of drafted tokens over a paged cache (pa_tree)
    logits   penalties, biases and grammar masks on logits (logits_adjust)

Rows of a batch hold their tokens at starts[b] .. starts[b] + lens[b] - 1.  `prepare` makes
what a program holds before the call, `run` is one pass (the framework's entry points where
`own` is true, else elementary torch), `exact` the operators' definition in 64 bits.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
PKG = ROOT / "pagedattention-based-transformer-decoder-inference-framework_amd"
if str(PKG) not in sys.path:
    sys.path.insert(0, str(PKG))

own = False

VOCAB = 50257        # of the dense decoders
STACK_VOCAB = 32768  # of the layer-stack models
PAGE = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
LARGEST = {"i8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # a decode step's keys and values of a batch of 64, one token a sequence
        dict(name="store_step_64", kind="store", cache="i8", io="f16", rows=64, tokens=1, heads=16,
             dim=128, page=PAGE, context=1024),
        # drafted tokens of a small model, trees of their own sizes
        dict(name="store_draft", kind="store", cache="e4m3", io="f32", rows=16, tokens=21, heads=12,
             dim=64, page=PAGE, context=333),
        # a prompt taken in: 2048 tokens of one sequence
        dict(name="store_prompt_2048", kind="store", cache="i8", io="bf16", rows=1, tokens=2048,
             heads=16, dim=128, page=PAGE, context=0),
        # the last tokens of a batch, for a program that inspects its cache
        dict(name="read_tail", kind="read", cache="e4m3", io="f32", rows=16, tokens=113, heads=12,
             dim=64, page=PAGE, context=1900),
        # prefixes of a batch given to attention that knows 16-bit pages alone
        dict(name="read_prefix", kind="read", cache="i8", io="f16", rows=8, tokens=3840, heads=16,
             dim=128, page=PAGE, context=0),
        # one user's first drafts of a small model: launches and latency only
        dict(name="tree_first", kind="tree", cache="f16", io="f32", rows=1, tokens=8, heads=12, group=1,
             dim=64, page=PAGE, context=113),
        # grouped heads and ragged drafts in bf16, as a layer-stack model's heads lie
        dict(name="tree_grouped", kind="tree", cache="bf16", io="bf16", rows=16, tokens=21, heads=16,
             group=8, dim=128, page=PAGE, context=4096),
        # one long document and a wide tree of drafts
        dict(name="tree_long", kind="tree", cache="e4m3", io="bf16", rows=1, tokens=63, heads=16, group=1,
             dim=128, page=32, context=32768),
        # a batch of 64 at a context of 8192, no drafts: the step of single tokens
        dict(name="tree_step_64x8192", kind="tree", cache="i8", io="f32", rows=64, tokens=1, heads=16,
             group=1, dim=128, page=PAGE, context=8192),
        # one request's logits with the usual penalties
        dict(name="logits_one", kind="logits", io="f32", rows=1, vocab=VOCAB, history=130, biases=0,
             masks=0),
        # a batch whose requests have penalties, biases and grammars
        dict(name="logits_batch_64", kind="logits", io="f32", rows=64, vocab=VOCAB, history=4096,
             biases=37, masks=8),
        # drafts of a whole batch verified at once, under their grammars
        dict(name="logits_drafts", kind="logits", io="bf16", rows=336, vocab=STACK_VOCAB, history=1021,
             biases=0, masks=336),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["store", "read", "tree", "tree", "logits"])
    if kind == "logits":
        vocab = _log(rng, 1000, 65536)
        rows = _log(rng, 1, max(1, min(336, 64 * VOCAB // vocab)))
        return dict(kind=kind, io=rng.choice(["f32", "f16", "bf16"]), rows=rows, vocab=vocab,
                    history=_log(rng, 1, 4096), biases=rng.choice([0, _log(rng, 1, 300)]),
                    masks=rng.choice([0, 1, rows]))
    dim, page = rng.choice([64, 128, 256]), rng.choice([16, 32])
    io = rng.choice(["f32", "f16", "bf16"])
    if kind != "tree":
        heads = rng.choice([1, 2, 4, 12, 16])
        tokens = _log(rng, 1, 4096)
        rows = _log(rng, 1, max(1, min(64, 8 * 3840 * 16 * 128 // (tokens * heads * dim))))
        return dict(kind=kind, cache=rng.choice(["i8", "e4m3"]), io=io, rows=rows, tokens=tokens,
                    heads=heads, dim=dim, page=page, context=rng.choice([0, _log(rng, 1, 2000)]))
    group = rng.choice([1, 1, 2, 4, 8])
    heads = group * rng.choice([1, 2, 4, 12, 16])
    context = _log(rng, 1, 32768)
    rows = _log(rng, 1, max(1, min(64, 64 * 8192 * 16 * 128 // (context * heads * dim))))
    tokens = _log(rng, 1, max(1, min(64, (1 << 27) // (rows * heads * context))))
    return dict(kind=kind, cache=rng.choice(["f16", "bf16", "i8", "e4m3"]), io=io, rows=rows,
                tokens=tokens, heads=heads, group=group, dim=dim, page=page, context=context)


def _starts(case):
    """Tokens that each row holds before the call: the first row's is the longest."""
    return [int(case["context"] * (1.0 - (0.618 * b) % 1.0 * 0.9)) for b in range(case["rows"])]


def _lens(case):
    """New tokens of each row, the first row's all."""
    if case["tokens"] == 1 or case["rows"] == 1:
        return [case["tokens"]] * case["rows"]
    return [max(1, int(case["tokens"] * (1.0 - (0.382 * b) % 1.0 * 0.5))) for b in range(case["rows"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    if case["kind"] == "logits":
        return _prepare_logits(case, normal, whole, gen)
    tree = case["kind"] == "tree"
    B, N, D, ts = case["rows"], case["tokens"], case["dim"], case["page"]
    kv_heads = case["heads"] // case.get("group", 1)
    tiles = -(-(case["context"] + N) // ts)
    pages = B * kv_heads * tiles + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[:B * kv_heads * tiles]
    state = dict(case=case, table=table.to(torch.int32).view(B, kv_heads, tiles).contiguous(),
                 starts=torch.tensor(_starts(case), dtype=torch.int32, device="cuda"),
                 lens=torch.tensor(_lens(case), dtype=torch.int32, device="cuda"))
    for name in ("k", "v"):
        pool = torch.empty((pages, ts, D), dtype=TYPES[case["cache"]], device="cuda")
        for part in pool.split(1 << 14):
            x = normal(*part.shape)
            if case["cache"] in LARGEST:  # the largest of a row at the type's own largest, as written
                x *= LARGEST[case["cache"]] / x.abs().amax(-1, keepdim=True)
            part.copy_(x.round() if case["cache"] == "i8" else x)
        state[name + "_pool"] = pool
        if case["cache"] in LARGEST:
            state[name + "_scale"] = (0.5 + torch.rand((pages, ts), generator=gen, device="cuda")) \
                * 3.0 / LARGEST[case["cache"]]
    io = TYPES[case["io"]]
    if case["kind"] == "store":
        # some heads' keys are many times the others', as they are in earnest
        wide = 1.0 + 8.0 * torch.rand((kv_heads, 1), generator=gen, device="cuda")
        state["k"] = (normal(B, N, kv_heads, D) * wide).to(io)
        state["v"] = normal(B, N, kv_heads, D).to(io)
    if case["kind"] == "read" or case["kind"] == "store":
        state["k_back"] = torch.zeros((B, N, kv_heads, D), dtype=io, device="cuda")
        state["v_back"] = torch.zeros_like(state["k_back"])
    if tree:
        state["q"] = (1.5 * normal(B, N, case["heads"], D)).to(io)
        state["out"] = torch.zeros_like(state["q"])
        # token j's parent is one of the tokens ahead of it, or the context's last token
        seen = torch.eye(N, dtype=torch.bool, device="cuda").expand(B, N, N).clone()
        parent = torch.rand((B, N), generator=gen, device="cuda")
        for j in range(1, N):
            at = (parent[:, j] * (j + 1)).long() - 1
            seen[:, j] |= seen[torch.arange(B, device="cuda"), at.clamp(min=0)] & (at >= 0)[:, None]
        state["mask"] = _words(seen)
    return state


def _words(bits):
    """Truth values [..][n] as int32 words [..][ceil(n / 32)], value 0 in the lowest bit."""
    n = bits.shape[-1]
    full = torch.zeros((*bits.shape[:-1], -(-n // 32) * 32), dtype=torch.int64, device=bits.device)
    full[..., :n] = bits
    words = (full.view(*bits.shape[:-1], -1, 32) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _bits(words, n):
    at = torch.arange(32, device=words.device, dtype=torch.int32)
    return (words[..., None] >> at & 1).flatten(-2)[..., :n].bool()


def _prepare_logits(case, normal, whole, gen):
    R, V, L = case["rows"], case["vocab"], case["history"]
    # a text's tokens: few of them often, most hardly ever
    seen = (V * torch.rand((R, L), generator=gen, device="cuda") ** 3).to(torch.int32).clamp(max=V - 1)
    lens = whole(L // 2, L + 1, R)
    state = dict(case=case, logits=(3.0 * normal(R, V)).to(TYPES[case["io"]]), history=seen,
                 history_lens=lens, prompt_lens=(lens * 0.6).to(torch.int32),
                 repetition=1.0 + 0.3 * torch.rand(R, generator=gen, device="cuda"),
                 frequency=0.5 * torch.rand(R, generator=gen, device="cuda"),
                 presence=0.8 * torch.rand(R, generator=gen, device="cuda"), bias_ids=None, bias=None,
                 allowed=None, allowed_rows=None)
    if case["biases"]:
        ids = torch.randperm(V, generator=gen, device="cuda")[:case["biases"]]
        ids = (ids + 7919 * torch.arange(R, device="cuda")[:, None]) % V
        state["bias_ids"], state["bias"] = ids.to(torch.int32), 2.0 * normal(*ids.shape)
    if case["masks"]:
        M = case["masks"]
        # a grammar allows next to nothing (a bracket) or nearly everything (inside a text)
        share = torch.tensor([0.01, 0.95], device="cuda")[torch.arange(M, device="cuda") % 2]
        state["allowed"] = _words(torch.rand((M, V), generator=gen, device="cuda") < share[:, None])
        state["allowed_rows"] = whole(0, M, R)
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    import llm_capi
    kind = s["case"]["kind"]
    if kind == "logits":
        names = ("history", "history_lens", "prompt_lens", "repetition", "frequency", "presence",
                 "bias_ids", "bias", "allowed", "allowed_rows")
        return llm_capi.logits_adjust(s["logits"], **{n: s[n] for n in names})
    if kind == "tree":
        scales = (s["k_scale"], s["v_scale"]) if "k_scale" in s else None
        D = s["case"]["dim"]
        return llm_capi.pa_tree(s["q"], s["k_pool"], s["v_pool"], s["table"], T=s["case"]["context"],
                                context_lens=s["starts"], tree_mask=s["mask"], tree_lens=s["lens"],
                                scales=scales, sm_scale=D ** -0.5, out=s["out"])
    cache = (s["k_pool"], s["v_pool"], s["table"], s["k_scale"], s["v_scale"])
    if kind == "store":
        llm_capi.kv_quant_write(s["k"], s["v"], *cache, starts=s["starts"], lens=s["lens"])
    k, v = llm_capi.kv_quant_read(*cache, starts=s["starts"], lens=s["lens"],
                                  out=(s["k_back"], s["v_back"]))
    return (k, v) if kind == "read" else (k, v, s["k_scale"], s["v_scale"])


# -- the plain form ----------------------------------------------------------------------

def _plain(s):
    kind = s["case"]["kind"]
    if kind == "logits":
        return _plain_logits(s)
    if kind == "tree":
        return _plain_tree(s)
    if kind == "store":
        _plain_store(s)
        return (*_plain_read(s), s["k_scale"], s["v_scale"])
    return _plain_read(s)


def _places(s):
    """Page and slot of every token [B][N][heads], and whether the row has that token."""
    N, ts = s["case"]["tokens"], s["case"]["page"]
    at = torch.arange(N, device="cuda")
    pos = s["starts"][:, None] + at
    here = at < s["lens"][:, None]
    tile = torch.where(here, pos // ts, 0).long()
    page = torch.gather(s["table"].long(), 2, tile[:, None].expand(-1, s["table"].shape[1], -1))
    return page.transpose(1, 2), (pos % ts)[:, :, None].expand_as(page.transpose(1, 2)), here


def _codes(x, cache):
    """Values quantised along the last dimension: codes and scales."""
    x = x.double()  # in 32 bits some quotients next to a border between two codes cross it
    top, largest = x.abs().amax(-1, keepdim=True), LARGEST[cache]
    y = x * largest / torch.where(top > 0, top, 1.0)
    scale = (top[..., 0] / largest).float()
    if cache == "i8":
        return y.round().to(torch.int8), scale
    # e4m3: 3 bits behind the leading one, steps of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    return ((y / step).round() * step).float().to(torch.float8_e4m3fn), scale


def _plain_store(s):
    page, slot, here = _places(s)
    page, slot = page[here], slot[here]
    for name in ("k", "v"):
        code, scale = _codes(s[name][here], s["case"]["cache"])
        s[name + "_pool"].view(torch.uint8)[page, slot] = code.view(torch.uint8)
        s[name + "_scale"][page, slot] = scale


def _plain_read(s):
    page, slot, here = _places(s)
    back = []
    for name in ("k", "v"):
        code = s[name + "_pool"].view(torch.uint8)[page, slot].view(TYPES[s["case"]["cache"]])
        x = code.float() * s[name + "_scale"][page, slot][..., None]
        into = s[name + "_back"]
        into.copy_(torch.where(here[:, :, None, None], x.to(into.dtype), into))
        back.append(into)
    return tuple(back)


def _plain_tree(s):
    c = s["case"]
    B, N, H, D, ts = c["rows"], c["tokens"], c["heads"], c["dim"], c["page"]
    heads, tiles = s["table"].shape[1:]
    table = s["table"].long().flatten()

    def gathered(name):
        pool = s[name + "_pool"]
        x = pool.view(torch.uint8 if pool.dtype.itemsize == 1 else pool.dtype)[table]
        x = x.view(pool.dtype).float()
        if name + "_scale" in s:
            x *= s[name + "_scale"][table][..., None]
        return x.view(B, heads, tiles * ts, D)

    pos = torch.arange(tiles * ts, device="cuda")
    j = pos - s["starts"][:, None]  # the position's place among the drafts
    seen = torch.gather(_bits(s["mask"], N), 2, j.clamp(0, N - 1)[:, None].expand(-1, N, -1))
    seen = (seen & ((j >= 0) & (j < s["lens"][:, None]))[:, None]) | (j < 0)[:, None]
    # rows of a key/value head: its group's heads of every drafted token
    q = s["q"].float().view(B, N, heads, H // heads, D).permute(0, 2, 3, 1, 4).reshape(B, heads, -1, D)
    score = torch.matmul(q, gathered("k").transpose(2, 3)) * D ** -0.5
    seen = seen[:, None, None].expand(-1, 1, H // heads, -1, -1).reshape(B, 1, -1, tiles * ts)
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > float("-inf"), top, 0.0))
    out = torch.matmul(p, gathered("v")) / (p.sum(-1, keepdim=True) + 1e-6)
    out = out.view(B, heads, H // heads, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D)
    here = torch.arange(N, device="cuda") < s["lens"][:, None]
    s["out"].copy_(torch.where(here[:, :, None, None], out.to(s["out"].dtype), s["out"]))
    return s["out"]


def _plain_logits(s):
    c = s["case"]
    R, V = c["rows"], c["vocab"]
    x = s["logits"].float()
    at = torch.arange(c["history"], device="cuda")
    ids = s["history"].long()
    asked = at < s["prompt_lens"][:, None]
    said = (at < s["history_lens"][:, None]) & ~asked
    count = torch.zeros((R, V), device="cuda").scatter_add_(1, ids, said.float())
    met = torch.zeros((R, V), device="cuda").scatter_add_(1, ids, (asked | said).float()) > 0
    rep = s["repetition"][:, None]
    x = torch.where(met, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias"] is not None:
        x = x + torch.zeros((R, V), device="cuda").scatter_(1, s["bias_ids"].long(), s["bias"])
    if s["allowed"] is not None:
        x = x.masked_fill(~_bits(s["allowed"][s["allowed_rows"].long()], V), float("-inf"))
    return x.to(s["logits"].dtype)


# -- what a pass cannot do without ----------------------------------------------------------

def work(case):
    if case["kind"] == "logits":
        R, V = case["rows"], case["vocab"]
        masks = min(case["masks"], R)
        return {"bytes": 2 * R * V * SIZES[case["io"]] + 4 * R * case["history"] + 8 * R * case["biases"]
                + masks * (-(-V // 32)) * 4, "flops": 4 * R * V}
    D, starts, lens = case["dim"], _starts(case), _lens(case)
    heads, io, held = case["heads"], SIZES[case["io"]], SIZES[case["cache"]]
    row = D * held + (4 if case["cache"] in LARGEST else 0)
    new = sum(lens)
    if case["kind"] == "tree":
        kv = sum(a + n for a, n in zip(starts, lens)) * (heads // case["group"])
        flops = sum(4 * n * (a + n) * heads * D for a, n in zip(starts, lens))
        return {"bytes": 2 * kv * row + 2 * new * heads * D * io, "flops": flops}
    passes = 2 if case["kind"] == "store" else 1
    return {"bytes": passes * 2 * new * heads * (D * io + row), "flops": passes * 4 * new * heads * D}


# -- the definition in 64 bits -----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"logits": _exact_logits, "tree": _exact_tree}.get(case["kind"], _exact_cache)(s)


def _slots(s, b, lo, hi):
    """Flat slots [heads][hi - lo] of row b's positions lo .. hi - 1."""
    ts = s["case"]["page"]
    pos = torch.arange(lo, hi, device="cuda")
    return s["table"][b].long()[:, pos // ts] * ts + pos % ts


def _held(s, name, slots):
    pool = s[name + "_pool"]
    x = pool.view(-1, pool.shape[-1]).view(torch.uint8 if pool.dtype.itemsize == 1 else pool.dtype)[slots]
    x = x.view(pool.dtype).double()
    return x * s[name + "_scale"].view(-1)[slots].double()[..., None] if name + "_scale" in s else x


def _exact_cache(s):
    case = s["case"]
    found = []
    scales = []
    for name in ("k", "v"):
        back = s[name + "_back"].double()
        scale = s[name + "_scale"].double().clone()
        for b, (at, n) in enumerate(zip(_starts(case), _lens(case))):
            slots = _slots(s, b, at, at + n)
            if case["kind"] == "read":
                back[b, :n] = _held(s, name, slots).transpose(0, 1)
                continue
            x = s[name][b, :n].double()
            largest = LARGEST[case["cache"]]
            unit = x.abs().max(dim=-1).values / largest
            y = x / unit[..., None].clamp(min=1e-300)
            if case["cache"] == "i8":
                # the quotient of two rounded numbers may miss a half that the true one is
                y = (x * largest / x.abs().amax(-1, keepdim=True).clamp(min=1e-300)).round()
            else:
                y = _nearest_e4m3(x * largest / x.abs().amax(-1, keepdim=True).clamp(min=1e-300))
            back[b, :n] = y * unit[..., None]
            scale.view(-1)[slots] = unit.transpose(0, 1)
        found.append(back)
        scales.append(scale)
    return tuple(found) if case["kind"] == "read" else (*found, *scales)


def _nearest_e4m3(y):
    """The value of e4m3 that is nearest, of two as near the one with an even code."""
    grid = torch.arange(127, dtype=torch.uint8, device=y.device).view(torch.float8_e4m3fn).double()
    above = torch.searchsorted(grid, y.abs()).clamp(1, 126)  # codes in the order of their values
    low, high = grid[above - 1], grid[above]
    up, down = high - y.abs(), y.abs() - low
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, above - 1)
    return grid[code] * y.sign()


def _exact_tree(s):
    case = s["case"]
    H, N, D = case["heads"], case["tokens"], case["dim"]
    out = s["out"].double()
    seen = _bits(s["mask"], N)
    for b, (at, n) in enumerate(zip(_starts(case), _lens(case))):
        slots = _slots(s, b, 0, at + n)
        k, v = _held(s, "k", slots), _held(s, "v", slots)  # [kv heads][positions][D]
        for h in range(k.shape[0]):
            mine = slice(h * case["group"], (h + 1) * case["group"])
            q = s["q"][b, :n, mine].double().reshape(-1, D)
            x = q @ k[h].T.contiguous() / D ** 0.5
            x[:, at:].masked_fill_(~seen[b, :n, :n].repeat_interleave(case["group"], 0), float("-inf"))
            p = torch.exp(x - x.amax(1, keepdim=True))
            out[b, :n, mine] = (p @ v[h] / (p.sum(1, keepdim=True) + 1e-6)).view(n, -1, D)
    return out


def _exact_logits(s):
    case = s["case"]
    V = case["vocab"]
    out = s["logits"].double()
    said_to, asked_to = s["history_lens"].tolist(), s["prompt_lens"].tolist()
    masks = s["allowed_rows"].tolist() if s["allowed"] is not None else None
    at = torch.arange(V, device="cuda")
    for r in range(case["rows"]):
        ids = s["history"][r].long()
        said = torch.bincount(ids[asked_to[r]:said_to[r]], minlength=V).double()
        met = said + torch.bincount(ids[:asked_to[r]], minlength=V)
        x, rep = out[r], s["repetition"][r].double()
        x = torch.where(met > 0, torch.where(x > 0, x / rep, x * rep), x)
        x -= s["frequency"][r].double() * said + s["presence"][r].double() * (said > 0).double()
        if s["bias"] is not None:
            x[s["bias_ids"][r].long()] += s["bias"][r].double()
        if masks is not None:
            word = s["allowed"][masks[r]][at // 32]
            x[(word >> (at % 32).to(torch.int32) & 1) == 0] = float("-inf")
        out[r] = x
    return out
