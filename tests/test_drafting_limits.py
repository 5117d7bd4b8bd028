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
