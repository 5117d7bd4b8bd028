"""Sizes at which the quantised cache and the logit rules refuse a call, before anything is launched."""
import ctypes

import llm_capi
from test_drafting import P, scales, view


def test_more_tokens_than_a_launch_has_workgroups():
    """256 threads a workgroup and less than 2^32 of them: 2^24 - 1 workgroups, of 16 tokens of two heads."""
    lib = llm_capi.load()
    most = 16 * ((1 << 24) - 1)
    for call in (lib.kv_quant_write, lib.kv_quant_read):
        for N in (most + 1, 2 * most, (1 << 31) - 1):
            assert call(view(), scales(), P, P, llm_capi.LLM_F16, 0, None, P, None, 1, N, None) == \
                llm_capi.LLM_ERR_INVALID, N
            assert b"too many tokens" in lib.llm_last_error()


def adjust(x=P, out=P, dtype=llm_capi.LLM_F32, rows=2, V=10, step=0, **rules):
    return llm_capi.load().logits_adjust(x, out, dtype, rows, V, step, ctypes.byref(llm_capi.LogitsRules(**rules)),
                                         None)


def test_lists_that_a_thread_could_not_count_to():
    """A thread steps 1024 entries at a time: past 2^31 - 1024 its place would leave 32 bits."""
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        assert adjust(history=4096, history_len=n) == llm_capi.LLM_ERR_INVALID
        assert adjust(bias_ids=4096, bias=4096, bias_len=n) == llm_capi.LLM_ERR_INVALID


def test_out_that_overlaps_the_logits():
    """Rows of another place that share elements with the logits' rows; in place is not one of them."""
    at = 1 << 20

    def overlaps(by, rows=4, V=10, step=32):
        # (with penalties that have no history: what does not overlap is refused for that)
        assert adjust(x=ctypes.c_void_p(at), out=ctypes.c_void_p(at + by), rows=rows, V=V, step=step,
                      repetition=4096) == llm_capi.LLM_ERR_INVALID
        error = llm_capi.load().llm_last_error()
        assert b"overlap" in error or b"history" in error
        return b"overlap" in error

    for by in (4, -4, 36, -36, 4 * 32, -4 * 32, 3 * 4 * 32 + 36, -(3 * 4 * 32 + 36), 4 * (2 * 32 - 9)):
        assert overlaps(by), by
    assert overlaps(4, rows=1) and overlaps(-36, rows=1) and overlaps(36, step=0)
    # in place, beside the logits' rows, in the gaps between them, behind them
    for by in (0, 40, -40, 88, 4 * 3 * 32 + 40, 4 * 4 * 32, -4 * 4 * 32, 4 * (32 + 10), 4 * (32 + 22)):
        assert not overlaps(by), by
    assert not overlaps(40, rows=1) and not overlaps(160, step=0)


def parts_of(B, N, heads, group, D, T, kv_dtype):
    """Parts that long rows are taken in, from what the call asks for them."""
    H = heads * group
    v = view(num_heads=heads, head_dim=D, kv_dtype=kv_dtype, max_tiles=4096)
    size = llm_capi.load().pa_tree_workspace_bytes(v, B, N, H, T)
    assert size % (B * N * H * (D + 2) * 4) == 0
    return size // (B * N * H * (D + 2) * 4)


def test_parts_of_batches_that_may_be_even():
    """Batches for which a plan for uneven rows alone has half a round too many when all are of one length, and
    gains nothing for it when they are not."""
    I8, F16, BF16 = llm_capi.LLM_I8, llm_capi.LLM_F16, llm_capi.LLM_BF16
    for most, batch in ((8, (4, 63, 16, 1, 128, 8192, I8)), (2, (64, 5, 4, 8, 128, 2048, F16)),
                        (8, (6, 24, 8, 2, 128, 3000, F16)), (7, (8, 128, 8, 1, 128, 4096, F16)),
                        (4, (4, 512, 2, 4, 128, 1024, BF16))):
        assert 1 < parts_of(*batch) <= most, batch
