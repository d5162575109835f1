"""The paged K/V cache on the GPU: calls that are refused, and legal ones off the beaten path.

Tolerances are those of ``test_cache_gpu.py``.
"""
import math
import threading

import pytest
import torch

import fstattention_b200 as fst
import test_cache_gpu as basics
from oracle import cache_oracle as orc
from test_cache_gpu import E4M3, E8M0, append, check, chunk, clean, int32, new_cache, read

pytestmark = pytest.mark.gpu


# ---- refusals -------------------------------------------------------------------------------------
def small(quantised=False, dtype=torch.float16, H_kv=2, D=64):
    gen = torch.Generator().manual_seed(0)
    cache = new_cache(gen, [40], H_kv, D, 16, "NHD", dtype, quantised)
    x = torch.randn((1, H_kv, 3, D), generator=gen).to(dtype).cuda()
    return cache, x


def every_call(cache, x, lens, **kw):
    return (lambda: append(x, x, cache, lens, **kw), lambda: read(cache, lens, 5, **kw), lambda: chunk(x, cache, lens, 0.1, **kw))


def swapped(cache, **kw):
    c = list(cache)
    for i, t in kw.items():
        c[("k", "v", "table", "ks", "vs", "layout").index(i)] = t
    return c


def test_caches_that_are_refused():
    cache, x = small()
    eight, _ = small(True)
    lens = int32([3])
    k, v, table = cache[:3]
    cases = [
        (swapped(cache, k=k.float(), v=v.float()), TypeError), (swapped(cache, v=v.bfloat16()), TypeError),
        (swapped(cache, v=v[:-1]), ValueError), (swapped(cache, v=v.transpose(1, 2).contiguous().transpose(1, 2)), ValueError),
        (swapped(cache, k=k[0], v=v[0]), ValueError), (swapped(cache, k=k[..., :32], v=v[..., :32]), ValueError),
        (swapped(cache, k=k[..., ::2], v=v[..., ::2]), ValueError), (swapped(cache, k=k[:, :8], v=v[:, :8]), ValueError),
        (swapped(cache, table=table.long()), ValueError), (swapped(cache, table=table[0]), ValueError),
        (swapped(cache, table=table.repeat(2, 1)), ValueError), (swapped(cache, table=table.repeat(1, 2)[:, ::2]), ValueError),
        (swapped(cache, ks=eight[3]), ValueError), (swapped(cache, ks=eight[3], vs=eight[4]), ValueError),
        (swapped(eight, ks=None), ValueError), (swapped(eight, vs=None), ValueError), (swapped(eight, ks=None, vs=None), ValueError),
        (swapped(eight, ks=eight[3].view(torch.uint8)), ValueError), (swapped(eight, vs=eight[4][:-1]), ValueError),
        (swapped(eight, ks=eight[3].transpose(1, 2)), ValueError), (swapped(cache, v=v.cpu()), RuntimeError),
        (swapped(cache, table=table.cpu()), RuntimeError), (swapped(eight, ks=eight[3].cpu()), RuntimeError),
        (swapped(cache, layout="HDN"), ValueError),
    ]
    for i, (bad, error) in enumerate(cases):
        for call in every_call(bad, x, lens):
            with pytest.raises(error):
                call()
                pytest.fail(f"case {i}")
    # strides that are no multiples of 16 bytes, a pool off a 16-byte boundary, and one that repeats itself
    wide = torch.zeros((5, 16, 2, 68), dtype=torch.float16, device="cuda")
    flat = torch.zeros(5 * 16 * 2 * 64 + 8, dtype=torch.float16, device="cuda")
    for pool in (wide[..., :64], flat[4:-4].view(5, 16, 2, 64), k[:, :, :1].expand(-1, -1, 2, -1), k[:1].expand(5, -1, -1, -1)):
        for call in every_call(swapped(cache, k=pool, v=pool), x, lens):
            with pytest.raises((ValueError, RuntimeError)):
                call()
    clean()


def test_arguments_that_are_refused():
    cache, x = small()
    eight, _ = small(True)
    lens = int32([3])
    refuse = lambda call, error=(ValueError, TypeError): pytest.raises(error, call)
    for bad in (lens.long(), int32([3, 3]), int32(3)):
        for call in every_call(cache, x, bad):
            refuse(call)
        refuse(lambda: append(x, x, cache, lens, lens=bad))
        refuse(lambda: chunk(x, cache, lens, 0.1, q_lens=bad))
    for call in every_call(cache, x, lens.cpu()):
        refuse(call, RuntimeError)
    # rows
    refuse(lambda: append(x, x[:, :, :2], cache, lens))
    refuse(lambda: append(x.bfloat16(), x.bfloat16(), cache, lens))
    refuse(lambda: append(x, x.bfloat16(), cache, lens))
    refuse(lambda: append(x.float(), x.float(), eight, lens))
    refuse(lambda: append(x[:, :1], x[:, :1], cache, lens))
    refuse(lambda: append(x[0], x[0], cache, lens))
    refuse(lambda: append(x[..., ::2], x[..., ::2], cache, lens))
    refuse(lambda: append(x.cpu(), x.cpu(), cache, lens), RuntimeError)
    refuse(lambda: append(x, x, cache, lens, rows=torch.zeros((1, 3), dtype=torch.int64, device="cuda")))
    refuse(lambda: append(x, x, cache, lens, rows=int32([0, 1, 2])))
    refuse(lambda: append(x[:, :, :0], x[:, :, :0], cache, lens, rows=int32([[0]])))
    # reading
    refuse(lambda: read(cache, lens, -1))
    refuse(lambda: read(cache, lens, 5, dtype=torch.bfloat16))
    refuse(lambda: read(eight, lens, 5, dtype=torch.float32))
    good = torch.empty((1, 2, 5, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (good[:, :, :4], good.half(), good[..., ::2], good[0]):
        refuse(lambda: read(eight, lens, 5, out=(good, bad)))
    refuse(lambda: read(eight, lens, 5, out=(good.cpu(), good)), RuntimeError)
    # queries
    for scale in (0.0, -0.1, math.nan, math.inf, 1e-60):
        refuse(lambda: chunk(x, cache, lens, scale))
    refuse(lambda: chunk(x.bfloat16(), cache, lens, 0.1))
    refuse(lambda: chunk(x.float(), eight, lens, 0.1))
    refuse(lambda: chunk(x[:, :1], cache, lens, 0.1))
    refuse(lambda: chunk(torch.cat([x, x[:, :1]], 1), cache, lens, 0.1))
    refuse(lambda: chunk(x[0], cache, lens, 0.1))
    refuse(lambda: chunk(x.repeat(1, 1, 1, 2), cache, lens, 0.1))
    refuse(lambda: chunk(x.cpu(), cache, lens, 0.1), RuntimeError)
    refuse(lambda: chunk(x, cache, lens, 0.1, out=torch.empty_like(x[:, :, :2])))
    refuse(lambda: chunk(x, cache, lens, 0.1, out=x.bfloat16()))
    refuse(lambda: chunk(x, cache, lens, 0.1, out=torch.empty_like(x).cpu()), RuntimeError)
    clean()


# ---- calls without work ----------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
def test_nothing_to_do(quantised):
    cache, x = small(quantised)
    lens, none = int32([3]), torch.zeros(0, dtype=torch.int32, device="cuda")
    empty = swapped(cache, table=cache[2][:0])
    was = cache[0].clone()
    append(x[:, :, :0], x[:, :, :0], cache, lens)
    append(x[:0], x[:0], empty, none)
    append(x, x, cache, lens, rows=int32([[0]])[:, :0])
    append(x, x, cache, lens, lens=int32([0]))
    append(x, x, cache, lens, lens=int32([-7]))
    assert torch.equal(was.view(torch.uint8), cache[0].view(torch.uint8))
    for got in (read(cache, lens, 0), read(empty, none, 4)):
        assert got[0].numel() == 0 and got[1].numel() == 0
    assert not read(cache, int32([-3]), 4)[0].any()
    out, lse = chunk(x[:, :, :0], cache, lens, 0.1, return_lse=True)
    assert out.shape == (1, 2, 0, 64) and lse.shape == (2, 0)
    out, lse = chunk(x[:0], empty, none, 0.1, return_lse=True)
    assert out.shape == (0, 2, 3, 64) and lse.shape == (0, 3)
    clean()


# ---- precision --------------------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 5, 12, 60])
def test_many_small_probabilities_beside_a_large_one(N, dtype, quantised):
    """One key whose value is zero has nearly all of the weight, 2^25.5 times that of any of the 60000 others, whose values are one (2^26
    times in 8 bits, which hold 51 as 52): what they leave of the result, 60000 * 2^-25.5 = 0.00126 or 60000 * 2^-26 = 0.00089, is there to the output's own rounding and that of the probabilities."""
    T, H, D = 60000, 2, 64
    gen = torch.Generator().manual_seed(N)
    cache = list(new_cache(gen, [T + N], 1, D, 64, "NHD", dtype, False))
    cache[0].zero_()
    cache[1].fill_(1.0)
    page, off = orc.row_of(cache, 0, torch.tensor([777], device="cuda"))
    cache[0][page, off, :, 5] = 51.0
    cache[1][page, off] = 0.0
    if quantised:
        for which in range(2):
            values, e, _ = orc.quantise(cache[which])
            cache[which], cache[3 + which] = values.to(E4M3), (e + 127).to(torch.uint8).transpose(1, 2).contiguous().view(E8M0)
    q = torch.zeros((1, H, N, D), dtype=dtype, device="cuda")
    q[..., 5] = 1.0
    out, lse = chunk(q, cache, int32([T + N]), math.log(2) / 2, causal=False, return_lse=True)
    clean()
    want = orc.attention(q, cache, [T + N], math.log(2) / 2, causal=False)
    assert 0.00085 < float(want[0].min()) and float(want[0].max()) < 0.0013
    check(out, lse, want, quantised, T + N)


@pytest.mark.parametrize("N", [1, 4, 12, 60])
def test_fp16_queries_over_an_8_bit_cache_keep_their_precision(N):
    """Probabilities and values are fp16, not bf16, where the queries are: the bounds of a 16-bit cache hold."""
    gen = torch.Generator().manual_seed(N)
    cache = new_cache(gen, [700, 333], 2, 128, 32, "NHD", torch.float16, True)
    q = torch.randn((2, 4, N, 128), generator=gen).to(torch.float16).cuda()
    out, lse = chunk(q, cache, int32([700, 333]), 0.1, return_lse=True)
    clean()
    check(out, lse, orc.attention(q, cache, [700, 333], 0.1), False, 700)


# ---- layouts --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("N,H,H_kv", [(1, 6, 2), (11, 6, 2), (150, 6, 2), (150, 8, 2), (600, 3, 3)])
def test_strided_tensors(N, H, H_kv, quantised):
    """Queries and outputs of [Z, N, H, D] layout inside wider tensors, pools that are one tensor, a block table's last columns unused."""
    gen = torch.Generator().manual_seed(N)
    Z, D, page, lens, dtype = 2, 128, 32, [N + 100, N + 7], torch.bfloat16
    cache = list(new_cache(gen, lens, H_kv, D, page, "HND", dtype, quantised, extra=100))
    both = torch.stack([cache[0].view(torch.uint8), cache[1].view(torch.uint8)], 1).view(cache[0].dtype)
    view = [both[:, 0], both[:, 1]] + cache[2:]
    wide = torch.randn((Z, N, H + 2 * H_kv, D), generator=gen).to(dtype).cuda()
    q = wide[:, :, :H].transpose(1, 2)
    k, v = wide[:, :, H:H + H_kv].transpose(1, 2), wide[:, :, H + H_kv:].transpose(1, 2)
    for c in (cache, view):
        append(k, v, c, int32([100, 7]))
    want = chunk(q.contiguous(), cache, int32(lens), 0.1)
    room = torch.full((Z, N, 2, H, D), 3.0, dtype=dtype, device="cuda")
    out = room[:, :, 1].transpose(1, 2)
    assert torch.equal(chunk(q, view, int32(lens), 0.1, out=out), want)
    assert (room[:, :, 0] == 3).all()
    clean()
    check(out, None, orc.attention(q, cache, lens, 0.1), quantised, max(lens))
    # broadcast queries
    for shape in ((Z, 1, N, D), (1, H, N, D), (Z, H, 1, D)):
        b = torch.randn(shape, generator=gen).to(dtype).cuda().expand(Z, H, N, D)
        assert torch.equal(chunk(b, view, int32(lens), 0.1), chunk(b.contiguous(), view, int32(lens), 0.1))
    clean()


def test_reading_into_given_tensors():
    gen = torch.Generator().manual_seed(2)
    for quantised in (False, True):
        cache = new_cache(gen, [70, 9], 3, 64, 16, "NHD", torch.float16, quantised)
        want = read(cache, int32([70, 9]), 75, dtype=torch.float16)
        room = torch.full((2, 2, 80, 3, 64), 5.0, dtype=torch.float16, device="cuda")
        k, v = (room[i, :, :75].transpose(1, 2) for i in range(2))
        got = read(cache, int32([70, 9]), 75, dtype=torch.float16, out=(k, v))
        assert got[0].data_ptr() == k.data_ptr() and torch.equal(k, want[0]) and torch.equal(v, want[1])
        assert (room[:, :, 75:] == 5).all()
        for M in (3, 70, 200):                            # fewer rows than the sequences have, and more than the tables can hold
            a = read(cache, int32([70, 9]), M, dtype=torch.float16)
            for x, y in zip(a, want):
                n = min(M, 75)
                assert torch.equal(x[:, :, :n], y[:, :, :n]) and not x[:, :, n:].any()
    clean()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("H,H_kv", [(1, 1), (33, 1), (128, 1), (200, 2), (48, 16)])
def test_groups_of_any_size(H, H_kv, quantised):
    gen = torch.Generator().manual_seed(H)
    for N, lens in ((1, [300, 0, 41]), (3, [3, 200, 130])):
        cache = new_cache(gen, lens, H_kv, 64, 16, "NHD", torch.float16, quantised)
        q = torch.randn((3, H, N, 64), generator=gen).to(torch.float16).cuda()
        out, lse = chunk(q, cache, int32(lens), 0.125, return_lse=True)
        clean()
        check(out, lse, orc.attention(q, cache, lens, 0.125), quantised, max(lens))


@pytest.mark.parametrize("quantised", [False, True])
def test_a_table_of_one_key_tile(quantised):
    """No item can be divided: no workspace, except for what an 8-bit cache is expanded into."""
    gen = torch.Generator().manual_seed(5)
    for lens, N, q_lens in (([128, 1, 77], 1, None), ([128, 30, 77], 20, [20, 20, 3]), ([128, 128, 65], 128, [128, 100, 65])):
        cache = new_cache(gen, [128] * 3, 2, 128, 128, "HND", torch.bfloat16, quantised)
        q = torch.randn((3, 8, N, 128), generator=gen).to(torch.bfloat16).cuda()
        out, lse = chunk(q, cache, int32(lens), 0.1, q_lens=None if q_lens is None else int32(q_lens), return_lse=True)
        clean()
        check(out, lse, orc.attention(q, cache, lens, 0.1, q_lens), quantised, 128)


@pytest.mark.parametrize("N", [2, 7, 12, 40, 140])
def test_a_query_that_is_not_finite_keeps_to_its_row(N):
    gen = torch.Generator().manual_seed(N)
    for quantised in (False, True):
        for dtype in (torch.float16, torch.bfloat16):
            cache = new_cache(gen, [400], 2, 64, 16, "NHD", dtype, quantised)
            q = torch.randn((1, 8, N, 64), generator=gen).to(dtype).cuda()
            want = chunk(q, cache, int32([400]), 0.1)
            odd = q.clone()
            odd[0, 1, N // 2, 3], odd[0, 6, 0, 60] = math.nan, math.inf
            got = chunk(odd, cache, int32([400]), 0.1)
            hit = torch.zeros((8, N), dtype=torch.bool, device="cuda")
            hit[1, N // 2] = hit[6, 0] = True
            assert torch.isnan(got[0][1, N // 2]).all()
            assert torch.equal(got[0][~hit], want[0][~hit])
    clean()


# ---- expanded 8-bit caches ---------------------------------------------------------------------------------
def test_an_expanded_cache():
    """2048 rows of a head and more: bad pages, sequences without queries or rows, and a graph whose lengths grow."""
    gen = torch.Generator().manual_seed(7)
    H, H_kv, D, N = 16, 2, 64, 260
    lens = [300, 0, 600, 17]
    cache = list(new_cache(gen, lens, H_kv, D, 16, "NHD", torch.bfloat16, True, extra=64))
    q = torch.randn((4, H, N, D), generator=gen).to(torch.bfloat16).cuda()
    kv, ql = int32(lens), int32([260, 260, 0, 17])
    out, lse = chunk(q, cache, kv, 0.125, q_lens=ql, return_lse=True)
    clean()
    check(out, lse, orc.attention(q, cache, lens, 0.125, ql.tolist()), True, 600)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = chunk(q, cache, kv, 0.125, q_lens=ql)
    for grown in (0, 1, 63):
        kv.copy_(int32([300 + grown, grown, 600, 17 + grown]))
        graph.replay()
        assert torch.equal(again, chunk(q, cache, kv, 0.125, q_lens=ql))
    clean()
    kv.copy_(int32(lens))
    table = cache[2].clone()
    for bad in (-1, cache[0].shape[0], 1 << 30):
        cache[2][0, 3] = bad
        got = chunk(q, cache, kv, 0.125, q_lens=ql)
        assert fst.last_status(clear=True) == 18 and torch.isfinite(got).all()
        assert torch.equal(got[1:], out[1:])
    # a bad page reads as zeros
    zeros = [t.clone() if torch.is_tensor(t) else t for t in cache]
    spare = sorted(set(range(cache[0].shape[0])) - set(table.flatten().tolist()))[0]
    for which in range(2):
        zeros[which].view(torch.uint8)[spare] = 0
        zeros[3 + which].view(torch.uint8)[spare] = 127
    zeros[2] = table.clone()
    zeros[2][0, 3] = spare
    assert torch.equal(chunk(q, zeros, kv, 0.125, q_lens=ql), got)
    clean()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_what_is_not_finite_in_an_expanded_cache(dtype):
    basics.test_what_is_not_finite_stays_where_it_is_seen(520, 8, 2, 64, dtype, True)


def test_queries_overwritten_by_their_results():
    """``out`` may be ``q``: the rows of an item are read before they are written, whoever divides them."""
    gen = torch.Generator().manual_seed(16)
    for quantised in (False, True):
        for N, lens in ((1, [5000, 30]), (7, [2000, 900]), (12, [3000, 12]), (300, [2500, 310])):
            cache = new_cache(gen, lens, 2, 128, 64, "NHD", torch.bfloat16, quantised)
            q = torch.randn((2, 8, N, 128), generator=gen).to(torch.bfloat16).cuda()
            want = chunk(q, cache, int32(lens), 0.1)
            for _ in range(3):
                same = q.clone()
                assert torch.equal(chunk(same, cache, int32(lens), 0.1, out=same), want)
    clean()


# ---- several at once -----------------------------------------------------------------------------------
def test_threads_on_streams_of_their_own():
    gen = torch.Generator().manual_seed(8)
    work = []
    for N, quantised in ((1, True), (6, False), (300, True), (90, False)):
        cache = new_cache(gen, [900, 500], 2, 128, 32, "NHD", torch.bfloat16, quantised)
        q = torch.randn((2, 4, N, 128), generator=gen).to(torch.bfloat16).cuda()
        kv = int32([900, 500])
        work.append((q, cache, kv, chunk(q, cache, kv, 0.1)))
    torch.cuda.synchronize()
    wrong = []

    def run(q, cache, kv, want):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [chunk(q, cache, kv, 0.1) for _ in range(20)]
            k = read(cache, kv, 900)[0]
            stream.synchronize()
        if not all(torch.equal(g, want) for g in got) or not k.any():
            wrong.append(q.shape)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    clean()


def test_calls_that_follow_each_other_see_each_others_rows():
    """Append, attention and append again in one queue: each starts early and still waits for what it reads and overwrites."""
    gen = torch.Generator().manual_seed(9)
    Z, H_kv, D, steps = 3, 2, 64, 40
    cache = new_cache(gen, [steps + 5] * Z, H_kv, D, 16, "NHD", torch.bfloat16, True)
    x = torch.randn((steps, 3, Z, H_kv, 1, D), generator=gen).to(torch.bfloat16).cuda()
    lens = torch.arange(steps + 6, dtype=torch.int32, device="cuda")[:, None].repeat(1, Z)
    torch.cuda.synchronize()
    outs = []
    for i in range(steps):
        append(x[i, 1], x[i, 2], cache, lens[5])          # the same place again and again
        outs.append(chunk(x[i, 0], cache, lens[6], 0.125))
    clean()
    for i in range(steps):
        append(x[i, 1], x[i, 2], cache, lens[5])
        torch.cuda.synchronize()
        assert torch.equal(chunk(x[i, 0], cache, lens[6], 0.125), outs[i])


def test_offsets_past_32_bits():
    """A pool of 2^32 bytes and more, a table that uses its last pages."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    gen = torch.Generator().manual_seed(10)
    H_kv, D, page = 2, 128, 128
    n_pages = (1 << 33) // (page * H_kv * D * 2) + 3
    k_pool, v_pool = (torch.zeros((n_pages, page, H_kv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = int32([[n_pages - 1, 0, n_pages - 3], [n_pages - 2, n_pages // 2 + 1, 7]])
    cache = (k_pool, v_pool, table, None, None, "NHD")
    k, v = (torch.randn((2, H_kv, 300, D), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    append(k, v, cache, int32([0, 17]))
    got = read(cache, int32([300, 317]), 317)
    assert torch.equal(got[0][0, :, :300], k[0]) and torch.equal(got[1][1, :, 17:], v[1])
    for N in (1, 5, 150):
        q = torch.randn((2, 4, N, D), generator=gen).to(torch.bfloat16).cuda()
        out, lse = chunk(q, cache, int32([300, 317]), 0.1, return_lse=True)
        check(out, lse, orc.attention(q, cache, [300, 317], 0.1), False, 317)
    clean()
