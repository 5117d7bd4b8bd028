"""Refusals of the quantised cache, the drafted tokens' attention and the logit rules before
anything is launched, and the masks of drafted trees."""
import ctypes

import pytest
import torch

import llm_capi
from _drafting import seen_bits

P = ctypes.c_void_p(4096)  # an address that is never read


def view(**change):
    v = dict(k_pool=4096, v_pool=4096, page_table=4096, num_pages=8, page_size=16, head_dim=64, num_beams=2,
             num_heads=2, max_tiles=4, kv_dtype=llm_capi.LLM_I8, page_stride=0)
    return ctypes.byref(llm_capi.PaKvView(**{**v, **change}))


def scales(**change):
    s = dict(k_scale=4096, v_scale=4096, page_stride=0)
    return ctypes.byref(llm_capi.PaKvScales(**{**s, **change}))


VIEWS = [dict(k_pool=0), dict(page_table=0), dict(num_pages=0), dict(max_tiles=0), dict(num_heads=0),
         dict(kv_dtype=llm_capi.LLM_F32), dict(kv_dtype=9), dict(page_stride=24), dict(page_stride=512),
         dict(page_stride=-1024), dict(k_pool=4104), dict(max_tiles=1 << 28), dict(page_size=-16)]


@pytest.mark.parametrize("entry", ["kv_quant_write", "kv_quant_read"])
def test_cache_calls_refused(entry):
    call = getattr(llm_capi.load(), entry)

    def run(v=None, s=None, k=P, dtype=llm_capi.LLM_F16, step=0, starts=P, B=2, N=3):
        return call(v or view(), s or scales(), k, P, dtype, step, None, starts, None, B, N, None)

    for change in VIEWS:
        assert run(view(**change)) == llm_capi.LLM_ERR_INVALID, change
    assert call(None, scales(), P, P, 0, 0, None, P, None, 1, 1, None) == llm_capi.LLM_ERR_INVALID
    assert call(view(), None, P, P, 0, 0, None, P, None, 1, 1, None) == llm_capi.LLM_ERR_INVALID
    assert run(view(kv_dtype=llm_capi.LLM_F16)) == llm_capi.LLM_ERR_INVALID  # has no scales
    assert run(s=scales(k_scale=0)) == llm_capi.LLM_ERR_INVALID
    assert run(s=scales(page_stride=15)) == llm_capi.LLM_ERR_INVALID
    assert run(k=None) == run(starts=None) == llm_capi.LLM_ERR_INVALID
    assert run(k=ctypes.c_void_p(4104)) == llm_capi.LLM_ERR_INVALID
    assert run(dtype=llm_capi.LLM_I8) == run(step=127) == run(step=129) == llm_capi.LLM_ERR_INVALID
    assert run(B=-1) == run(N=-1) == run(B=65536) == llm_capi.LLM_ERR_INVALID
    assert run(N=(1 << 31) - 1) == llm_capi.LLM_ERR_INVALID
    assert run(view(head_dim=60, page_size=16)) == llm_capi.LLM_ERR_UNSUPPORTED
    assert run(view(head_dim=264)) == llm_capi.LLM_ERR_UNSUPPORTED
    assert run(B=0) == run(N=0) == llm_capi.LLM_OK
    assert entry.encode() in llm_capi.load().llm_last_error()


def test_tree_refused():
    lib = llm_capi.load()

    def run(v=None, s=scales(), q=P, q_step=0, out=P, out_step=0, dtype=llm_capi.LLM_F32, B=2, N=3, H=4, D=64,
            T=8, scale=1.0, ws=None, size=0):
        return lib.pa_tree(v or view(), s, q, q_step, out, out_step, dtype, None, None, None, None, B, N, H, D, T,
                           scale, ws, size, None)

    bad, no = llm_capi.LLM_ERR_INVALID, llm_capi.LLM_ERR_UNSUPPORTED
    for change in VIEWS:
        assert run(view(**change)) == bad, change
    assert run(view(kv_dtype=llm_capi.LLM_E4M3), s=None) == bad
    assert run(view(kv_dtype=llm_capi.LLM_F16)) == run(view(kv_dtype=llm_capi.LLM_BF16)) == bad
    assert run(q=None) == run(out=None) == run(q=ctypes.c_void_p(4100)) == bad
    assert run(H=3) == run(H=0) == run(D=128) == run(T=-1) == run(N=-1) == run(B=-1) == bad
    assert run(q_step=255) == run(out_step=258) == run(dtype=llm_capi.LLM_E4M3) == bad
    assert run(scale=float("nan")) == run(scale=float("inf")) == bad
    assert run(view(head_dim=96), D=96) == run(view(page_size=24)) == no
    assert run(N=1025) == run(H=130) == run(B=65536) == no
    assert run(B=0) == run(N=0) == llm_capi.LLM_OK
    # a long row is split, and its parts need room
    long = view(max_tiles=4096)
    need = lib.pa_tree_workspace_bytes(long, 2, 3, 4, 60000)
    assert need > 0 and need % 16 == 0
    assert run(long, T=60000) == run(long, T=60000, ws=P, size=need - 1) == bad
    assert run(long, T=60000, ws=ctypes.c_void_p(4100), size=need) == bad
    assert b"pa_tree_workspace_bytes" in lib.llm_last_error()
    assert lib.pa_tree_workspace_bytes(long, 2, 1025, 4, 60000) == 0
    assert lib.pa_tree_workspace_bytes(view(), 2, 3, 4, 64) == 0  # short: none


def test_logits_refused():
    lib = llm_capi.load()

    def run(x=P, out=P, dtype=llm_capi.LLM_F32, rows=2, V=10, step=0, **rules):
        return lib.logits_adjust(x, out, dtype, rows, V, step, ctypes.byref(llm_capi.LogitsRules(**rules)), None)

    bad = llm_capi.LLM_ERR_INVALID
    assert lib.logits_adjust(P, P, 2, 2, 10, 0, None, None) == bad
    assert run(x=None) == run(out=None) == run(rows=-1) == run(rows=65536) == run(V=0) == run(step=9) == bad
    assert run(dtype=llm_capi.LLM_I8) == run(x=ctypes.c_void_p(4098)) == bad
    assert run(repetition=4096) == run(history=4096, history_len=-1) == bad
    assert run(history=4096, history_len=5, history_stride=4) == bad
    assert run(bias_ids=4096) == run(bias=4096) == bad
    assert run(bias_ids=4096, bias=4096, bias_len=3, bias_stride=2) == bad
    assert run(allowed=4096) == run(allowed=4096, num_masks=1) == bad  # two rows, one mask
    assert run(rows=0) == llm_capi.LLM_OK
    assert b"logits_adjust" in lib.llm_last_error()


def test_decode_keeps_to_its_types():
    lib = llm_capi.load()
    v = view(kv_dtype=llm_capi.LLM_E4M3)
    assert lib.pa_decode(v, P, P, None, None, 1, 2, 64, 16, 1.0, 0, None, 0, None) == llm_capi.LLM_ERR_INVALID
    assert llm_capi.kv_dtype_of(torch.empty(1, dtype=torch.float8_e4m3fn)) == llm_capi.LLM_E4M3


def test_tree_mask():
    words = llm_capi.tree_mask([[-1, 0, 0, 1], [-1, -1, 1, 0]])
    assert words.shape == (2, 4, 1) and words.dtype == torch.int32
    assert words[..., 0].tolist() == [[1, 3, 5, 11], [1, 2, 6, 9]]
    chain = llm_capi.tree_mask(list(range(-1, 69)))
    assert chain.shape == (70, 3)
    assert torch.equal(seen_bits(chain, 70), torch.tril(torch.ones(70, 70, dtype=torch.bool)))
    assert llm_capi.tree_mask(torch.zeros((1, 0), dtype=torch.int32)).shape == (1, 0, 0)
    with pytest.raises(ValueError):
        llm_capi.tree_mask([0])
    with pytest.raises(ValueError):
        llm_capi.tree_mask([-1, -2])


def test_torch_calls_refuse_before_any_launch():
    """The tensors' own checks, on tensors of the CPU: no call gets as far as the library."""
    calls = llm_capi._torch_calls()
    pool, table = torch.zeros((4, 16, 64), dtype=torch.int8), torch.zeros((1, 2, 2), dtype=torch.int32)
    scale, x = torch.zeros((4, 16)), torch.zeros((1, 1, 2, 64))
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="current device"):
        llm_capi.kv_quant_write(x, x, pool, pool, table, scale, scale, starts=one)
    with pytest.raises(ValueError, match="current device"):
        llm_capi.pa_tree(x, pool, pool, table, T=1)
    with pytest.raises(ValueError, match="current device"):
        llm_capi.logits_adjust(scale)
    with pytest.raises(ValueError):
        calls.quant(True, x, x, pool, pool, table, scale, scale, one, None, None, 0)
    with pytest.raises(ValueError):
        calls.tree(x, pool, pool, table, None, None, None, None, None, None, 1, 1.0, None, 0)
    with pytest.raises(ValueError):
        calls.adjust(scale, *[None] * 11, 0)
