"""How linear attention cuts a sequence into segments, as the C ABI reports it (no GPU needed)."""
import pytest

from swiftx_b200 import _lib


def _plan(heads, dk, dtype, L=4096):
    """(whether the forward is cut, the backward's segments)"""
    lib = _lib.load()
    a = _lib.LinattnArgs()
    a.batch, a.seqlen, a.heads, a.qk_heads, a.dk, a.dv, a.dtype = 1, L, heads, heads, dk, 64, dtype
    return lib.swx_linattn_fwd_workspace_bytes(a) > 0, lib.swx_linattn_segments(a)


@pytest.mark.parametrize("heads", [99, 100, 120, 148])
def test_fp32_walks_are_not_halved(heads):
    """One fp32 forward CTA fills an SM: 99 to 148 whole walks run in one round, their halves in two of the same
    length and with the states on top.  So does the backward above dk 64; up to dk 64 two of its CTAs fit."""
    assert _plan(heads, 64, 0) == (False, 2)
    assert _plan(heads, 128, 0) == (False, 1)


@pytest.mark.parametrize("heads,segments", [(149, 1), (98, 3), (74, 4), (40, 8), (6, 32)])         # 40: seven of 10 chunks and one of 4, made 8 of 8
def test_fp32_walks_of_other_counts(heads, segments):
    assert _plan(heads, 64, 0) == (segments > 1, segments)
    assert _plan(heads, 128, 0) == (segments > 1, segments)


@pytest.mark.parametrize("heads,L", [(149, 129), (149, 256), (200, 384), (222, 500)])
def test_pipelined_kernels_take_many_heads_uncut(heads, L):
    """bf16 heads of up to 64 in several rounds: from 129 tokens on the pipelined kernels, which walk them whole."""
    assert _plan(heads, 64, 1, L)[0] is False
