"""The paged K/V cache on the GPU: rows in, rows out, attention of new tokens over it.

Everything is compared with ``oracle/cache_oracle.py`` in 64 bits.  What is held or copied has to be equal.  An output of
the attention may be off by what its roundings add up to, with A the weighted mean of |v| and S the row's largest
sm_scale * sum_d |q_d k_d|:

* the output's own rounding, eps / 2 of its value, eps that of its type (an fp16 result below 2^-14: half of 2^-24);
* the rounding of the probabilities to 16 bits for the second product, eps / 2 of A (bf16's eps over an 8-bit cache);
* scores: fp32 sums of D products, D roundings of S (2^-23 each, the tensor cores may truncate), three more for the scale and
  the distance to the maximum, and the exponential's own error, below 2^-18; numerator and denominator are
  both off by that share: 2 A (2^-23 (D + 3) S + 2^-18);
* the sums over T keys in fp32: T + 64 roundings of 2^-23 at the most, of numerator and denominator: 2 A 2^-23 (T + 64).
"""
import math

import pytest
import torch

import fstattention_b200 as fst
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu

E4M3, E8M0 = orc.E4M3, orc.E8M0


def new_cache(gen, lens, H_kv, D, page, layout, dtype, quantised, extra=0, spread=0.5):
    """A cache whose pages hold random rows everywhere, and tables for sequences of ``lens`` rows."""
    width = max(1, -(-(max(lens) + extra) // page))
    n_pages = len(lens) * width + 2
    order = torch.randperm(n_pages, generator=gen)[:len(lens) * width].view(len(lens), width).to(torch.int32)
    shape = (n_pages, page, H_kv, D) if layout == "NHD" else (n_pages, H_kv, page, D)
    pools, scales = [], []
    for _ in range(2):
        x = (torch.randn(shape, generator=gen) * torch.exp(spread * torch.randn(D, generator=gen))).to(dtype)
        if quantised:
            values, e, _ = orc.quantise(x)
            pools.append(values.to(E4M3).cuda())
            e = (e + 127).to(torch.uint8)
            scales.append((e.transpose(1, 2) if layout == "NHD" else e).contiguous().cuda().view(E8M0))
        else:
            pools.append(x.cuda())
            scales.append(None)
    return pools[0], pools[1], order.cuda(), scales[0], scales[1], layout


def int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def chunk(q, cache, kv_lens, scale, **kw):
    return fst.fst_attention_chunk(q, cache[0], cache[1], cache[2], kv_lens, scale, k_scale=cache[3], v_scale=cache[4],
                                   pool_layout=cache[5], **kw)


def append(k, v, cache, start, **kw):
    fst.fst_cache_append(k, v, cache[0], cache[1], cache[2], start, k_scale=cache[3], v_scale=cache[4], pool_layout=cache[5], **kw)


def read(cache, lens, max_rows, **kw):
    return fst.fst_cache_read(cache[0], cache[1], cache[2], lens, max_rows, k_scale=cache[3], v_scale=cache[4], pool_layout=cache[5], **kw)


def check(got, lse, want, quantised, T):
    """got [Z, H, N, D] and lse [Z * H, N] against the oracle's four tensors."""
    out, ref_lse, mag, size = want
    eps = torch.finfo(got.dtype).eps
    p_eps = torch.finfo(torch.bfloat16).eps if quantised else eps
    D = got.shape[-1]
    share = 2.0 ** -23 * (D + 3) * size[..., None] + 2.0 ** -18
    tol = out.abs() * eps / 2 + mag * (p_eps / 2 + 2 * share + 2 * 2.0 ** -23 * (T + 64)) + 2.0 ** -25
    same = (out == got.double()) | (torch.isnan(out) & torch.isnan(got))
    far = torch.where(same, torch.zeros_like(out), (got.double() - out).abs() - tol)
    worst = float(torch.nan_to_num(far, nan=math.inf).max())
    assert worst <= 0, worst
    if lse is not None:
        lse = lse.view(ref_lse.shape).double()
        assert torch.equal(torch.isinf(lse), torch.isinf(ref_lse))
        fine = torch.isfinite(ref_lse)
        tol = (share[..., 0] + 2.0 ** -23 * (T + 64)) / math.log(2) + 2.0 ** -22 * ref_lse.abs()
        assert ((lse - ref_lse).abs() <= tol)[fine].all()


def clean():
    torch.cuda.synchronize()
    assert fst.last_status() == 0


# ---- append and read --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("page,layout,D,H_kv", [(16, "NHD", 128, 3), (64, "NHD", 64, 8), (32, "HND", 128, 1), (128, "HND", 64, 5)])
def test_append_then_read(dtype, quantised, page, layout, D, H_kv):
    gen = torch.Generator().manual_seed(page + D)
    start, lens, N = [0, 5, 15, 33, 130], [7, 1, 40, 0, 33], 40
    cache = new_cache(gen, [s + n for s, n in zip(start, lens)], H_kv, D, page, layout, dtype, quantised)
    before = [t.clone() for t in cache if torch.is_tensor(t)]
    wide = (torch.randn((5, N, H_kv, 2, D), generator=gen) * 3).to(dtype).cuda()
    k, v = wide[:, :, :, 0].transpose(1, 2), wide[:, :, :, 1].transpose(1, 2)           # strided
    append(k, v, cache, int32(start), lens=int32(lens))
    clean()
    total = [s + n for s, n in zip(start, lens)]
    out_type = dtype
    got = read(cache, int32(total), max(total) + 3, dtype=out_type if quantised else None)
    clean()
    written = torch.zeros(before[0].shape[:-1], dtype=torch.bool, device="cuda")
    for which, x in enumerate((k, v)):
        for z in range(5):
            want = x[z, :, :lens[z]]
            if quantised:
                values, e, _ = orc.quantise(want)
                want = (values * orc.pow2(e)[..., None]).to(out_type)
            assert torch.equal(got[which][z, :, start[z]:total[z]], want)
            assert not got[which][z, :, total[z]:].any()
            held = orc.rows(cache, z, total[z], which).to(out_type)
            assert torch.equal(got[which][z, :, :total[z]], held)
            at, off = orc.row_of(cache, z, torch.arange(start[z], total[z], device="cuda"))
            (written if layout == "NHD" else written.transpose(1, 2))[at, off] = True
    for was, now in zip(before[:2], cache[:2]):           # nothing else was touched
        assert torch.equal(was.view(torch.uint8).view(*was.shape[:-1], -1)[~written], now.view(torch.uint8).view(*was.shape[:-1], -1)[~written])
    if quantised:
        mask = written.transpose(1, 2) if layout == "NHD" else written
        for was, now in zip(before[3:], cache[3:5]):
            assert torch.equal(was.view(torch.uint8)[~mask], now.view(torch.uint8)[~mask])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantisation_at_its_edges(dtype):
    """Ties, the largest and smallest values, rows at and behind a change of the exponent, zeros, NaN and infinity."""
    D, rows = 64, []
    big = torch.finfo(dtype).max
    eps = torch.finfo(dtype).eps
    for top in (448.0, 448.0 * (1 + eps), 447.0, 1.75, 1.75 * (1 + eps), 2.0 ** -9, 2.0 ** -14, big, big / 2, 0.0, torch.finfo(dtype).tiny,
                torch.finfo(dtype).smallest_normal * eps, 3.0, 65000.0):
        x = torch.linspace(-1, 1, D, dtype=torch.float64) * top
        x[3], x[7] = top, -top
        rows.append(x)
    ties = torch.tensor([(1 + (2 * i + 1) / 16) * 2.0 ** j for j in range(-9, 8) for i in range(8)], dtype=torch.float64)[:D - 1]
    rows.append(torch.cat([ties, torch.tensor([448.0], dtype=torch.float64)]))
    sub = torch.arange(D, dtype=torch.float64) * 2.0 ** -10
    sub[0] = 448.0
    rows.append(sub)
    x = torch.stack(rows).to(dtype)
    odd = x[:4].clone()
    odd[0, 5], odd[1, 63], odd[2, 0], odd[3, 8] = math.nan, math.inf, -math.inf, math.nan
    x = torch.cat([x, odd]).cuda()[None, None]            # [1, 1, rows, D]
    n = x.shape[2]
    cache = new_cache(torch.Generator().manual_seed(1), [n], 1, D, 16, "NHD", dtype, True)
    append(x, -x, cache, int32([0]))
    clean()
    values, e, finite = orc.quantise(x[0, 0])
    for which, sign in ((0, 1.0), (1, -1.0)):
        at, off = orc.row_of(cache, 0, torch.arange(n, device="cuda"))
        b = cache[3 + which].view(torch.uint8)[at, 0, off].long()
        assert torch.equal(b, torch.where(finite, e + 127, torch.full_like(e, 255)))
        assert torch.equal(cache[which].view(torch.uint8)[at, off, 0].view(E4M3).double(), values * sign)
    for out_type in (torch.bfloat16, torch.float16):
        k, _ = read(cache, int32([n]), n, dtype=out_type)
        want = (values * orc.pow2(e)[:, None]).clamp(-torch.finfo(out_type).max, torch.finfo(out_type).max).to(out_type)
        want[~finite] = math.nan
        assert torch.equal(torch.isnan(k[0, 0]), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(k[0, 0]), torch.nan_to_num(want))


def test_every_byte_and_scale_reads_as_its_value():
    D, page = 128, 128
    pool = torch.arange(256, dtype=torch.uint8).repeat(page * D // 256).view(1, page, 1, D).cuda().view(E4M3)
    scale = torch.arange(page, dtype=torch.uint8).add(64).view(1, 1, page).cuda().view(E8M0)     # 2^-63 .. 2^64
    k, v = fst.fst_cache_read(pool, pool, int32([[0]]), int32([page]), page, k_scale=scale, v_scale=scale)
    want = (pool.double()[0, :, 0] * scale.double()[0, 0][:, None]).to(torch.bfloat16)
    for x in (k, v):
        assert torch.equal(torch.isnan(x[0, 0]), torch.isnan(want)) and torch.equal(torch.nan_to_num(x[0, 0]), torch.nan_to_num(want))


def test_append_of_a_tree_path():
    gen = torch.Generator().manual_seed(3)
    Z, H_kv, N, D, M = 6, 4, 50, 128, 9
    k, v = ((torch.randn((Z, H_kv, N, D), generator=gen)).to(torch.float16).cuda() for _ in range(2))
    path = torch.stack([torch.randperm(N, generator=gen)[:M] for _ in range(Z)]).to(torch.int32).cuda()
    start, lens = [3, 0, 100, 15, 16, 17], [9, 0, 4, 1, 9, 2]
    cache = new_cache(gen, [s + 9 for s in start], H_kv, D, 16, "HND", torch.float16, False)
    append(k, v, cache, int32(start), lens=int32(lens), rows=path)
    got = read(cache, int32([s + n for s, n in zip(start, lens)]), 110)
    clean()
    for z in range(Z):
        for x, y in zip(got, (k, v)):
            assert torch.equal(x[z, :, start[z]:start[z] + lens[z]], y[z][:, path[z, :lens[z]].long()])


def test_bad_places_are_reported_and_left_alone():
    gen = torch.Generator().manual_seed(4)
    k = torch.randn((1, 2, 4, 64), generator=gen).to(torch.bfloat16).cuda()
    for what in ("page", "past the table", "before", "row"):
        cache = list(new_cache(gen, [20], 2, 64, 16, "NHD", torch.bfloat16, False))
        start, rows = [14], None
        if what == "page":
            cache[2][0, 1] = cache[0].shape[0]
        elif what == "past the table":
            start = [30]
        elif what == "before":
            start = [-2]
        else:
            rows = int32([[0, 1, 4, -1]])
        was = cache[0].clone()
        append(k, k, cache, int32(start), rows=rows)
        assert fst.last_status(clear=True) == 18
        assert int((was != cache[0]).any(-1).sum()) == 2 * 2                 # two of the four rows, two heads
    cache[2][0, 0] = -5
    out = read(cache, int32([20]), 40)
    assert fst.last_status(clear=True) == 18
    assert not out[0][0, :, :16].any() and out[0][0, :, 16:20].all() and not out[0][0, :, 20:].any()
    read(cache, int32([33]), 40)                          # longer than its table
    assert fst.last_status(clear=True) == 18


# ---- attention --------------------------------------------------------------------------------
CASES = [
    # Z lengths, queries, q_lens, H, H_kv, D, page, layout
    ([77], 1, None, 32, 32, 128, 16, "NHD"),
    ([1], 1, None, 4, 2, 64, 16, "HND"),
    ([1000, 17, 4099], 1, None, 32, 8, 128, 64, "NHD"),
    ([2049, 300], 1, None, 10, 2, 64, 128, "HND"),
    ([640, 16, 129, 128, 127, 15], 1, None, 7, 1, 128, 32, "HND"),
    ([513, 90], 7, [7, 2], 32, 8, 64, 128, "HND"),
    ([1300, 700, 40], 13, [1, 13, 12], 8, 8, 128, 16, "NHD"),
    ([333], 5, None, 15, 3, 128, 64, "NHD"),
    ([150, 64], 64, [33, 64], 8, 2, 128, 32, "NHD"),
    ([70, 700], 70, [70, 65], 5, 1, 64, 64, "HND"),
    ([300, 1025], 300, [300, 17], 8, 2, 128, 64, "NHD"),
    ([1024, 511, 600], 511, [1, 511, 300], 4, 4, 64, 16, "NHD"),
    ([2500], 1111, None, 8, 1, 128, 128, "HND"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, dtype, quantised, causal):
    lens, N, q_lens, H, H_kv, D, page, layout = CASES[case]
    gen = torch.Generator().manual_seed(case)
    cache = new_cache(gen, lens, H_kv, D, page, layout, dtype, quantised)
    q = torch.randn((len(lens), H, N, D), generator=gen).to(dtype).cuda()
    ql = None if q_lens is None else int32(q_lens)
    out, lse = chunk(q, cache, int32(lens), D ** -0.5, q_lens=ql, causal=causal, return_lse=True)
    clean()
    check(out, lse, orc.attention(q, cache, lens, D ** -0.5, q_lens, causal), quantised, max(lens))


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("N,H,H_kv", [(1, 4, 4), (3, 8, 1), (40, 4, 2), (300, 2, 1)])
def test_lengths_of_nothing(N, H, H_kv, quantised):
    """Empty sequences, sequences without queries, more queries than rows."""
    lens = [0, 5, 0, 2, 64, 1, 0]
    q_lens = [N, 0, 0, N, N, 1, 1]
    gen = torch.Generator().manual_seed(N)
    cache = new_cache(gen, lens, H_kv, 64, 16, "NHD", torch.bfloat16, quantised)
    q = torch.randn((7, H, N, 64), generator=gen).to(torch.bfloat16).cuda()
    for causal in (True, False):
        out, lse = chunk(q, cache, int32(lens), 0.125, q_lens=int32(q_lens), causal=causal, return_lse=True)
        clean()
        check(out, lse, orc.attention(q, cache, lens, 0.125, q_lens, causal), quantised, 64)
        given = torch.full_like(q, 7.0)
        back = chunk(q, cache, int32(lens), 0.125, q_lens=int32(q_lens), causal=causal, out=given)
        assert back.data_ptr() == given.data_ptr()
        for z in range(7):
            assert (given[z, :, q_lens[z]:] == 7).all() and torch.equal(given[z, :, :q_lens[z]], out[z, :, :q_lens[z]])
    none = chunk(q, cache, int32([0] * 7), 0.125)
    assert not none.any()
    none = chunk(q, cache, int32(lens), 0.125, q_lens=int32([0] * 7))
    assert not none.any()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,H,H_kv,D", [(1, 8, 2, 128), (6, 4, 1, 64), (100, 4, 2, 128), (290, 2, 1, 64)])
def test_what_is_not_finite_stays_where_it_is_seen(N, H, H_kv, D, dtype, quantised):
    """NaN and infinities behind the sequences' ends, and in rows that only later queries attend to."""
    lens = [300, 290 + N % 7]
    gen = torch.Generator().manual_seed(D + N)
    cache = list(new_cache(gen, lens, H_kv, D, 32, "NHD", dtype, quantised))
    q = torch.randn((2, H, N, D), generator=gen).to(dtype).cuda()
    for z in range(2):                                    # everything behind the ends
        page, off = orc.row_of(cache, z, torch.arange(lens[z], cache[2].shape[1] * 32, device="cuda"))
        for which in range(2):
            if quantised:
                cache[which].view(torch.uint8)[page, off] = 0x7f
                cache[3 + which].view(torch.uint8).transpose(1, 2)[page, off] = 255
            else:
                cache[which][page, off] = math.nan
    out, lse = chunk(q, cache, int32(lens), D ** -0.5, return_lse=True)
    want = orc.attention(q, cache, lens, D ** -0.5)
    assert torch.isfinite(out).all()
    check(out, lse, want, quantised, 300)
    # rows of the chunk itself: row 300 - N / 2 of sequence 0, the last row of sequence 1
    for z, r in ((0, 300 - (N + 1) // 2), (1, lens[1] - 1)):
        page, off = orc.row_of(cache, z, torch.tensor([r], device="cuda"))
        if quantised:
            cache[1].view(torch.uint8)[page, off] = 0
            cache[4].view(torch.uint8).transpose(1, 2)[page, off] = 255
        else:
            cache[1][page, off, :, 3] = math.inf
            cache[1][page, off, 0, D - 2] = math.nan
            cache[1][page, off, H_kv - 1, D // 2] = -math.inf
    out, lse = chunk(q, cache, int32(lens), D ** -0.5, return_lse=True)
    clean()
    want = orc.attention(q, cache, lens, D ** -0.5)
    assert not torch.isfinite(want[0]).all() and (N == 1 or torch.isfinite(want[0]).any(-1).any())
    check(out, lse, want, quantised, 300)
    # K: a NaN score is a NaN for those who see it
    page, off = orc.row_of(cache, 1, torch.tensor([lens[1] - 1], device="cuda"))
    if quantised:
        cache[3].view(torch.uint8).transpose(1, 2)[page, off] = 255
        cache[0].view(torch.uint8)[page, off] = 0
    else:
        cache[0][page, off, :, 0] = math.nan
    out = chunk(q, cache, int32(lens), D ** -0.5)
    assert torch.isnan(out[1, :, -1]).all() and (N == 1 or torch.isfinite(out[1, :, :N - 1]).all())


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("N", [1, 9, 200])
def test_scores_of_any_size(N, quantised):
    """Scores in the thousands, rows of K and V many powers of two apart."""
    gen = torch.Generator().manual_seed(N)
    dtype, lens, H, H_kv, D = torch.bfloat16, [700, 260], 8, 2, 128
    cache = list(new_cache(gen, lens, H_kv, D, 64, "NHD", dtype, False, spread=0.2))
    power = torch.exp2(torch.randint(-20, 12, cache[1].shape[:2], generator=gen).float()).cuda()
    cache[1] = (cache[1] * power[:, :, None, None]).to(dtype)
    cache[0] = (cache[0] * torch.exp2(torch.randint(-6, 5, cache[0].shape[:2], generator=gen).float()).cuda()[:, :, None, None]).to(dtype)
    if quantised:
        for which in range(2):
            values, e, _ = orc.quantise(cache[which])
            cache[which], cache[3 + which] = values.to(E4M3), (e + 127).to(torch.uint8).transpose(1, 2).contiguous().view(E8M0)
    q = (torch.randn((2, H, N, D), generator=gen) * 4).to(dtype).cuda()
    out, lse = chunk(q, cache, int32(lens), 1.0, return_lse=True)
    clean()
    check(out, lse, orc.attention(q, cache, lens, 1.0), quantised, 700)


def test_strides_and_a_pool_inside_another_tensor():
    gen = torch.Generator().manual_seed(9)
    Z, H, H_kv, N, D, page = 2, 8, 2, 5, 128, 32
    lens = [200, 97]
    cache = list(new_cache(gen, lens, H_kv, D, page, "NHD", torch.float16, False))
    both = torch.stack([cache[0], cache[1]], 1)           # [n_pages, 2, page, H_kv, D]
    view = [both[:, 0], both[:, 1]] + cache[2:]
    q = torch.randn((Z, N, H, D), generator=gen).to(torch.float16).cuda().transpose(1, 2)
    want = chunk(q.contiguous(), cache, int32(lens), 0.1)
    assert torch.equal(chunk(q, view, int32(lens), 0.1), want)
    out = torch.empty((Z, N, H, 2 * D), dtype=torch.float16, device="cuda")[..., D:].transpose(1, 2)
    assert torch.equal(chunk(q, view, int32([200, 97, 0, 0])[:2], 0.1, out=out), want)
    every_other = torch.tensor([200, 1, 97, 1], dtype=torch.int32, device="cuda")[::2]
    assert torch.equal(chunk(q, view, every_other, 0.1), want)
    a, b = read(view, int32(lens), 200), read(cache, int32(lens), 200)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    clean()


def test_bad_pages_and_lengths_are_reported():
    gen = torch.Generator().manual_seed(10)
    for N in (1, 100):
        for quantised in (False, True):
            cache = list(new_cache(gen, [100], 2, 64, 16, "NHD", torch.bfloat16, quantised))
            q = torch.randn((1, 4, N, 64), generator=gen).to(torch.bfloat16).cuda()
            table = cache[2].clone()
            for bad in (-1, cache[0].shape[0], 1 << 30):
                cache[2][0, 2] = bad
                out = chunk(q, cache, int32([100]), 0.1)
                assert fst.last_status(clear=True) == 18 and torch.isfinite(out).all()
            cache[2].copy_(table)
            want = chunk(q, cache, int32([table.shape[1] * 16]), 0.1)
            clean()
            assert torch.equal(chunk(q, cache, int32([1 << 30]), 0.1), want)              # cut to what the table holds
            assert fst.last_status(clear=True) == 18
            assert not chunk(q, cache, int32([-4]), 0.1).any()
            assert fst.last_status(clear=True) == 18
            full = chunk(q, cache, int32([100]), 0.1)
            assert torch.equal(chunk(q, cache, int32([100]), 0.1, q_lens=int32([N + 5])), full)
            assert fst.last_status(clear=True) == 18


@pytest.mark.parametrize("N", [1, 150])
def test_streams_and_graphs(N):
    """On another stream, captured, and replayed after the sequences have grown; two graphs in turn."""
    gen = torch.Generator().manual_seed(11)
    H, H_kv, D, lens = 8, 2, 128, [400, 170]
    cache = new_cache(gen, lens, H_kv, D, 32, "NHD", torch.bfloat16, True, extra=200)
    q = torch.randn((2, H, N, D), generator=gen).to(torch.bfloat16).cuda()
    k, v = (torch.randn((2, H_kv, N, D), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    start, kv = int32([l - N for l in lens]), int32(lens)

    def step():
        append(k, v, cache, start)
        return chunk(q, cache, kv, D ** -0.5)

    want = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for i in range(3):
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert torch.equal(out, want)
        q.add_(0.25)
        k.mul_(-1.5)
        start.add_(31)
        kv.add_(31)
        want = step().clone()
    clean()


def test_results_do_not_change_from_run_to_run():
    gen = torch.Generator().manual_seed(12)
    for N in (1, 20, 400):
        cache = new_cache(gen, [3000, 700], 2, 128, 64, "NHD", torch.bfloat16, False)
        q = torch.randn((2, 8, N, 128), generator=gen).to(torch.bfloat16).cuda()
        first = chunk(q, cache, int32([3000, 700]), 0.1)
        for _ in range(5):
            assert torch.equal(chunk(q, cache, int32([3000, 700]), 0.1), first)


def test_many_sequences():
    gen = torch.Generator().manual_seed(13)
    lens = [int(x) for x in torch.randint(0, 90, (300,), generator=gen)]
    cache = new_cache(gen, lens, 2, 64, 16, "NHD", torch.float16, False)
    for N, q_lens in ((1, None), (9, [int(x) for x in torch.randint(0, 10, (300,), generator=gen)])):
        q = torch.randn((300, 4, N, 64), generator=gen).to(torch.float16).cuda()
        out, lse = chunk(q, cache, int32(lens), 0.125, q_lens=None if q_lens is None else int32(q_lens), return_lse=True)
        clean()
        check(out, lse, orc.attention(q, cache, lens, 0.125, q_lens), False, 90)


# ---- together -----------------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
def test_a_prompt_a_decode_step_and_a_tree(quantised):
    """Chunks of two prompts, a token each, then a token tree whose accepted path goes into the cache."""
    gen = torch.Generator().manual_seed(21)
    Z, H, H_kv, D, page, dtype = 2, 8, 2, 128, 32, torch.bfloat16
    lens, pieces = [0, 0], [[100, 64], [37, 100], [1, 1]]
    cache = new_cache(gen, [200, 200], H_kv, D, page, "NHD", dtype, quantised)
    for piece in pieces:
        N = max(piece)
        q = torch.randn((Z, H, N, D), generator=gen).to(dtype).cuda()
        k, v = (torch.randn((Z, H_kv, N, D), generator=gen).to(dtype).cuda() for _ in range(2))
        append(k, v, cache, int32(lens), lens=int32(piece))
        lens = [a + b for a, b in zip(lens, piece)]
        out, lse = chunk(q, cache, int32(lens), D ** -0.5, q_lens=int32(piece), return_lse=True)
        check(out, lse, orc.attention(q, cache, lens, D ** -0.5, piece), quantised, max(lens))
    parent = [-1] + [i // 2 for i in range(30)]
    meta = fst.build_tree_metadata(torch.tensor(parent, dtype=torch.int32, device="cuda"), 32, 32)
    n = len(parent)
    q = torch.randn((Z, H, n, D), generator=gen).to(dtype).cuda()
    k, v = (torch.randn((Z, H_kv, n, D), generator=gen).to(dtype).cuda() for _ in range(2))
    if not quantised:
        tree = fst.fst_attention_paged(q, k, v, meta, cache[0], cache[1], cache[2], int32(lens), D ** -0.5)
    # the tree behind the same prefix as contiguous tensors, one sequence at a time
    kp, vp = read(cache, int32(lens), max(lens))
    path = int32([[0, 1, 3, 7], [0, 2, 6, 13]])
    for z in range(Z):
        ka, va = (torch.cat([p[z:z + 1, :, :lens[z]], t[z:z + 1]], 2) for p, t in ((kp, k), (vp, v)))
        alone = fst.fst_attention(q[z:z + 1], ka, va, meta, sm_scale=D ** -0.5)
        if not quantised:
            assert (alone - tree[z:z + 1]).abs().max().item() <= 2 * 1.6e-2
        # a node attends to its ancestors: the same queries, one after the other, once the path is in the cache
        if z == 0:
            append(k, v, cache, int32(lens), rows=path)
            lens_after = [a + 4 for a in lens]
            qp = torch.stack([q[i][:, path[i].long()] for i in range(Z)])
            out, lse = chunk(qp, cache, int32(lens_after), D ** -0.5, return_lse=True)
            check(out, lse, orc.attention(qp, cache, lens_after, D ** -0.5), quantised, max(lens_after))
        if not quantised:                                 # (a quantised path is not the tree's own rows)
            assert (out[z] - alone[0][:, path[z].long()]).abs().max().item() <= 2 * 1.6e-2
    clean()
