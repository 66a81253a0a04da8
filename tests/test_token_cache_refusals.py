"""Refusals of the token cache's calls, before any device call (no GPU needed)."""
import pytest

from hnsw_amd import capi

BUFFERS = dict(lens=1 << 12, grow=2 << 12, table=3 << 12, ring=4 << 12, state=5 << 12, slots=6 << 12, cu_new=7 << 12, lens_out=8 << 12, state_out=9 << 12, status=10 << 12)
SIZES = dict(lens=12, grow=12, state=16, slots=40, cu_new=16, lens_out=12, state_out=16, status=4)      # 3 requests, 5 slots


def _plan(**at):
    b = dict(BUFFERS, **at)
    rc = capi.lib().hnsw_amd_cache_plan_device(b["lens"], b["grow"], 3, b["table"], 4, b["ring"], 8, b["state"], 16, 5, b["slots"], b["cu_new"], b["lens_out"], b["state_out"],
                                               b["status"], 0, None)
    return rc, capi.lib().hnsw_amd_last_error().decode()


@pytest.mark.parametrize("result", ["slots", "cu_new", "lens_out", "state_out", "status"])
@pytest.mark.parametrize("given", ["lens", "grow", "state"])
def test_plan_refuses_results_that_lie_in_what_it_reads(result, given):
    """Every workgroup reads lengths, growth and state, while others write."""
    for at in (BUFFERS[given], BUFFERS[given] + SIZES[given] - 4, BUFFERS[given] - SIZES[result] + 4):
        rc, why = _plan(**{result: at})
        assert rc == capi.E_ARG and "buffers of their own" in why, (result, given, at)
