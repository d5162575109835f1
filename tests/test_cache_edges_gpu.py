"""The paged K/V cache on the GPU: lengths, scales and counts at the edges of what the calls allow.

Tolerances are those of ``test_cache_gpu.py`` where a test does not derive its own.
"""
import pytest
import torch

import fstattention_b200 as fst
from oracle import cache_oracle as orc
from test_cache_gpu import append, check, chunk, clean, int32, new_cache

pytestmark = pytest.mark.gpu


# ---- the ring of K and V tiles ------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N,H", [(1, 32), (2, 32), (4, 32)])
def test_long_items_whose_last_tile_is_nearly_empty(N, H, D, quantised):
    """Many tiles, then one of 1 to 16 keys, in which all warps but one have nothing to do: they must not give V's stage back for
    a warp that still reads an earlier tile out of it.  8, 16 and 32 rows of a head; the same bits every time."""
    gen = torch.Generator().manual_seed(D + N)
    H_kv, dtype = 4, torch.float16 if D == 64 else torch.bfloat16
    lens = [256 * 17 + 1, 256 * 12 + 16, 256 * 14 + 2, 256 * 9 + 7, 256 * 17 + 5, 256 + 1]
    cache = new_cache(gen, lens, H_kv, D, 64, "HND", dtype, quantised)
    q = torch.randn((len(lens), H, N, D), generator=gen).to(dtype).cuda()
    first, lse = chunk(q, cache, int32(lens), D ** -0.5, return_lse=True)
    check(first, lse, orc.attention(q, cache, lens, D ** -0.5), quantised, max(lens))
    for _ in range(50):
        again, lse_again = chunk(q, cache, int32(lens), D ** -0.5, return_lse=True)
        assert torch.equal(again, first) and torch.equal(lse_again, lse)
    clean()


# ---- lengths far past the table ----------------------------------------------------------------------------
INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("length", [1 << 30, INT_MAX - 127, INT_MAX - 14, INT_MAX])
def test_lengths_up_to_the_largest_are_cut(length, page):
    """Cut to what the table holds and reported: by an 8-bit cache that is expanded first (2048 rows of a head), and by the other kernels."""
    gen = torch.Generator().manual_seed(page)
    for N, H in ((1, 4), (12, 4), (100, 4), (520, 8)):
        cache = new_cache(gen, [600, 40], 2, 64, page, "NHD", torch.bfloat16, True)
        q = torch.randn((2, H, N, 64), generator=gen).to(torch.bfloat16).cuda()
        most = cache[2].shape[1] * page
        want = chunk(q, cache, int32([most, 40]), 0.125)
        clean()
        got = chunk(q, cache, int32([length, 40]), 0.125)
        assert fst.last_status(clear=True) == 18 and torch.equal(got, want)
        x = torch.zeros((2, 2, 1, 64), dtype=torch.bfloat16, device="cuda")
        append(x, x, cache, int32([length, 0]))
        assert fst.last_status(clear=True) == 18
