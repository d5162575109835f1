"""The paged K/V cache's C entries without a GPU: sizes and factors at the edges.  No call here gets as far as a launch."""
import ctypes as C

from test_cache_host import INVALID, P, cache, chunk_args


def test_an_expansion_whose_size_does_not_fit_is_not_made(built_lib):
    """2^30 pages by 2^24 heads of 64 by 16 rows would be 2^66 bytes: past 2 GB, as 2^21 rows of 5 sequences are, not 0."""
    from fstattention_b200 import _lib
    size = _lib.lib().fst_attention_chunk_workspace_bytes
    few = size(C.byref(cache(table_stride=9)), 1, 4, 2, 2048, 64)
    for stride, Z, heads in ((1 << 20, 1 << 10, 1 << 24), (1 << 20, 2000, (1 << 31) - 1), (1 << 20, 1 << 10, 1 << 23)):
        c = cache(table_stride=stride, k_scale=P(512), v_scale=P(1024))
        assert size(C.byref(c), Z, heads, heads, 2048, 64) == few


def test_a_factor_that_overflows_in_base_two_is_refused(built_lib):
    """sm_scale * log2(e) has to be finite too."""
    from fstattention_b200 import _lib
    lib = _lib.lib()
    for scale in (2.4e38, 3.4e38):
        assert lib.fst_attention_chunk(*chunk_args(cache(), scale=scale)) == INVALID
