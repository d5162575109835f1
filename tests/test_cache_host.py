"""The paged K/V cache without a GPU: what its calls refuse, and the oracle's 8-bit arithmetic against torch's own."""
import ctypes as C

import pytest
import torch

from oracle import cache_oracle as orc

OK, INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE, TOO_LARGE = 0, 1, 2, 3, 4, 6
P = C.c_void_p


# ---- Python -------------------------------------------------------------------------------------
def test_python_refusals(built_lib):
    import fstattention_b200 as fst
    pool = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 3, 64), dtype=torch.float16)
    calls = (lambda **kw: fst.fst_cache_append(x, x, pool, pool, table, lens, **kw),
             lambda **kw: fst.fst_cache_read(pool, pool, table, lens, 5, **kw),
             lambda **kw: fst.fst_attention_chunk(x, pool, pool, table, lens, 0.1, **kw))
    for call in calls:
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
        with pytest.raises(ValueError, match="pool_layout"):
            call(pool_layout="HDN")
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        fst.fst_cache_read(pool, pool, table, lens, 5, dtype=torch.float32)
    with pytest.raises(TypeError):
        fst.fst_cache_append(None, x, pool, pool, table, lens)
    with pytest.raises(TypeError):
        fst.fst_attention_chunk(x, pool, pool, [[0]], lens, 0.1)


# ---- C --------------------------------------------------------------------------------------------
# Addresses below are made up: every call here returns before anything could be launched.
def cache(**kw):
    from fstattention_b200 import _lib
    f = dict(k_pool=P(4096), v_pool=P(8192), k_scale=P(None), v_scale=P(None), block_table=P(256), table_stride=8, page_size=16, n_pages=9,
             stride_page=16 * 2 * 64, stride_row=2 * 64, stride_head=64)
    f.update(kw)
    return _lib.PagedCache(**f)


BAD_CACHES = [
    (dict(k_pool=P(None)), INVALID), (dict(v_pool=P(None)), INVALID), (dict(block_table=P(None)), INVALID),
    (dict(table_stride=0), INVALID), (dict(table_stride=-1), INVALID), (dict(n_pages=0), INVALID),
    (dict(k_scale=P(512)), INVALID), (dict(v_scale=P(512)), INVALID),
    (dict(stride_page=0), INVALID), (dict(stride_row=0), INVALID), (dict(stride_head=-64), INVALID),
    (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED), (dict(page_size=256), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED),
    (dict(k_pool=P(4096 + 8)), ALIGNMENT), (dict(v_pool=P(8192 + 2)), ALIGNMENT),
    (dict(stride_page=16 * 2 * 64 + 4), ALIGNMENT), (dict(stride_row=2 * 64 + 1), ALIGNMENT), (dict(stride_head=65), ALIGNMENT),
    (dict(k_scale=P(512), v_scale=P(1024), stride_head=72), ALIGNMENT), (dict(k_scale=P(520), v_scale=P(1024)), ALIGNMENT),
    (dict(table_stride=(1 << 31) - 1), TOO_LARGE), (dict(table_stride=1 << 27), TOO_LARGE),
]


def append_args(c, k=4096, v=8192, start=256, lens=None, rows=None, Z=1, H_kv=2, N=3, M=3, D=64, strides=(384, 192, 64) * 2, dtype=0):
    return [C.byref(c) if c is not None else None, P(k), P(v), P(start), P(lens), P(rows), Z, H_kv, N, M, D, *strides, dtype, None, None]


def read_args(c, k=4096, v=8192, lens=256, Z=1, H_kv=2, M=3, D=64, strides=(384, 192, 64) * 2, dtype=0):
    return [C.byref(c) if c is not None else None, P(k), P(v), P(lens), Z, H_kv, M, D, *strides, dtype, None, None]


def chunk_args(c, q=4096, o=8192, lse=None, kv_lens=256, q_lens=None, Z=1, H=4, H_kv=2, n_q=3, D=64, strides=(768, 192, 64) * 2, scale=0.125,
               causal=1, dtype=0, workspace=4096, bytes=1 << 40):
    return [P(q), P(o), P(lse), C.byref(c) if c is not None else None, P(kv_lens), P(q_lens), Z, H, H_kv, n_q, D, *strides, scale, causal, dtype,
            P(workspace), bytes, None, None]


@pytest.mark.parametrize("case", range(len(BAD_CACHES)))
def test_caches_that_are_refused(built_lib, case):
    from fstattention_b200 import _lib
    lib = _lib.lib()
    fields, want = BAD_CACHES[case]
    c = cache(**fields)
    assert lib.fst_cache_append(*append_args(c)) == want
    assert lib.fst_cache_read(*read_args(c)) == want
    assert lib.fst_attention_chunk(*chunk_args(c)) == want
    assert lib.fst_attention_chunk_workspace_bytes(C.byref(c), 1, 4, 2, 3, 64) == 0


def test_arguments_that_are_refused(built_lib):
    from fstattention_b200 import _lib
    lib = _lib.lib()
    c = cache()
    for kw, want in [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(start=None), INVALID), (dict(Z=0), INVALID), (dict(H_kv=0), INVALID),
                     (dict(N=0), INVALID), (dict(M=0), INVALID), (dict(M=2), INVALID), (dict(D=96), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED),
                     (dict(dtype=-1), UNSUPPORTED), (dict(k=4100), ALIGNMENT), (dict(strides=(384, 192, 68, 384, 192, 64)), ALIGNMENT),
                     (dict(strides=(384, 192, 64, 384, 196, 64)), ALIGNMENT)]:
        assert lib.fst_cache_append(*append_args(c, **kw)) == want, kw
    for kw, want in [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(lens=None), INVALID), (dict(Z=-1), INVALID), (dict(H_kv=0), INVALID),
                     (dict(M=0), INVALID), (dict(D=32), UNSUPPORTED), (dict(dtype=3), UNSUPPORTED), (dict(v=8196), ALIGNMENT),
                     (dict(strides=(388, 192, 64, 384, 192, 64)), ALIGNMENT)]:
        assert lib.fst_cache_read(*read_args(c, **kw)) == want, kw
    for kw, want in [(dict(q=None), INVALID), (dict(o=None), INVALID), (dict(kv_lens=None), INVALID), (dict(Z=0), INVALID), (dict(H=0), INVALID),
                     (dict(H=5), INVALID), (dict(H_kv=0), INVALID), (dict(n_q=0), INVALID), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID),
                     (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(D=256), UNSUPPORTED),
                     (dict(dtype=2), UNSUPPORTED), (dict(n_q=(1 << 30), H=8), TOO_LARGE), (dict(q=4098), ALIGNMENT), (dict(o=8200), ALIGNMENT),
                     (dict(workspace=4096 + 128), ALIGNMENT), (dict(strides=(768, 192, 64, 768, 192, 60)), ALIGNMENT)]:
        assert lib.fst_attention_chunk(*chunk_args(c, **kw)) == want, kw
    for f, args in ((lib.fst_cache_append, append_args(None)), (lib.fst_cache_read, read_args(None)), (lib.fst_attention_chunk, chunk_args(None))):
        assert f(*args) == INVALID


def test_workspaces(built_lib):
    from fstattention_b200 import _lib
    lib = _lib.lib()
    size = lib.fst_attention_chunk_workspace_bytes
    small, large = cache(), cache(table_stride=9)                     # tables of 128 and 144 rows
    assert size(C.byref(small), 1, 4, 2, 3, 64) == 0
    need = size(C.byref(large), 1, 4, 2, 3, 64)
    assert need > 0 and size(C.byref(large), 1, 4, 2, 300, 64) > need
    # a number of pieces that does not depend on how many sequences, heads or rows there are
    assert size(C.byref(large), 64, 4, 2, 3, 64) == need == size(C.byref(cache(table_stride=4000)), 1, 4, 2, 3, 64)
    assert lib.fst_attention_chunk(*chunk_args(large, workspace=None)) == WORKSPACE
    assert lib.fst_attention_chunk(*chunk_args(large, bytes=need - 1)) == WORKSPACE
    # an 8-bit cache under 2048 rows of a head or more: its rows in 16 bits as well, two tensors of Z * pages pages, and a table
    quantised = cache(table_stride=9, k_scale=P(512), v_scale=P(1024))
    few, many = size(C.byref(quantised), 3, 4, 2, 1023, 64), size(C.byref(quantised), 3, 4, 2, 1024, 64)
    pages = 3 * 9
    assert few == size(C.byref(large), 3, 4, 2, 1023, 64)
    assert many - pages * (2 * 16 * 2 * 64 * 2 + 4) in range(few, few + 256)
    huge = cache(table_stride=1 << 17, k_scale=P(512), v_scale=P(1024))           # 2^21 rows of 2 heads of 64: 2 GB, and past that
    assert size(C.byref(huge), 2, 4, 2, 1024, 64) > 1 << 31 and size(C.byref(huge), 5, 4, 2, 1024, 64) == few


# ---- the oracle ---------------------------------------------------------------------------------
def test_oracle_rounds_as_torch_does():
    """e4m3 values of a row whose scale is one: the same as torch's conversion (nearest, ties to even)."""
    x = torch.cat([torch.linspace(-448, 448, 4001), torch.linspace(-0.05, 0.05, 2001), torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 17.0, 19.0])])
    row = torch.cat([x, torch.tensor([448.0])])
    values, e, finite = orc.quantise(row)
    assert int(e) == 0 and bool(finite)
    assert torch.equal(values, row.to(torch.float8_e4m3fn).double())
    for k in (-30, -3, 5, 100):                           # the same row at another power of two
        v2, e2, _ = orc.quantise(row.double() * 2.0 ** k)
        assert int(e2) == k and torch.equal(v2, values)


def test_oracle_scales():
    for a, e in [(448.0, 0), (448.1, 1), (447.0, 0), (224.0, -1), (225.0, 0), (0.0, -117), (1.0, -8), (1.75, -8), (1.76, -7), (2.0 ** -140, -117),
                 (3.3e38, 119)]:
        got = orc.quantise(torch.tensor([0.0, -a], dtype=torch.float64))
        assert int(got[1]) == e, a
    assert not orc.quantise(torch.tensor([1.0, float("nan")]))[2] and not orc.quantise(torch.tensor([float("-inf"), 1.0]))[2]
    b = torch.tensor([0, 1, 126, 127, 128, 254], dtype=torch.uint8)
    want = b.view(torch.float8_e8m0fnu).double()
    assert torch.equal(orc.pow2(b.long() - 127), want)
