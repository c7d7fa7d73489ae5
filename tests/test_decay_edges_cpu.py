"""Boundary of decay linear attention where there are no rows or no tokens, without a GPU."""
import pytest

from linearnexus_amd import _lib
from test_decay_norm_paged_cpu import _decay, _refused


def test_a_gradient_for_each_head_is_required_without_rows_too():
    """Sums over no rows are zeros that the call writes."""
    a = _decay(B=0, g_per_head=1)
    a.d_g = None
    _refused(_lib.load().lnx_decay_bwd(a, None), -1, b"d_g")
    a = _decay(B=0, H=1 << 25, g_per_head=1)
    _refused(_lib.load().lnx_decay_bwd(a, None), -2, b"too many heads")


def test_a_gradient_without_elements_may_be_missing():
    """No tokens, a decay for each: d_g has no memory.  (Refused for the workspace, which comes after every tensor.)"""
    for kw in (dict(B=2, T=0), dict(T=0, nseq=3)):
        a = _decay(**kw)
        a.cu_seqlens = a.g  # any memory
        a.d_g = a.g = None
        _refused(_lib.load().lnx_decay_bwd(a, None), -4, b"workspace")
