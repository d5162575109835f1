"""The paged K/V cache on the GPU: lengths, scales and counts at the edges of what the calls allow.

Tolerances are those of ``test_cache_gpu.py`` where a test does not derive its own.
"""
import math

import pytest
import torch

import fstattention_b200 as fst
from oracle import cache_oracle as orc
from test_cache_gpu import append, check, chunk, clean, int32, new_cache, read

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


# ---- sequences without queries --------------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("N,H", [(1, 4), (12, 4), (100, 4), (520, 8)])
def test_a_sequence_without_queries_is_not_looked_at(N, H, quantised):
    """One whose pages have been taken away and whose length nobody has reset: nothing is reported, the others are as they are without it."""
    gen = torch.Generator().manual_seed(N)
    lens = [600, 700, 530]
    cache = new_cache(gen, lens, 2, 64, 16, "NHD", torch.bfloat16, quantised)
    q = torch.randn((3, H, N, 64), generator=gen).to(torch.bfloat16).cuda()
    want = chunk(q, cache, int32([600, 0, 530]), 0.125, q_lens=int32([N, 0, N]))
    cache[2][1] = -1
    for idle in (0, -3):
        got = chunk(q, cache, int32(lens), 0.125, q_lens=int32([N, idle, N]))
        clean()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_and_tokens_in_one_call(dtype):
    """A chunk of 520 tokens by 4 heads beside single tokens and an idle sequence: over 8 bits all of them go through the expanded copy."""
    gen = torch.Generator().manual_seed(31)
    lens, q_lens, H, H_kv, D = [900, 3000, 1, 2049, 77, 640], [520, 1, 1, 1, 0, 1], 8, 2, 128
    for quantised in (False, True):
        cache = new_cache(gen, lens, H_kv, D, 64, "NHD", dtype, quantised)
        q = torch.randn((6, H, 520, D), generator=gen).to(dtype).cuda()
        out, lse = chunk(q, cache, int32(lens), D ** -0.5, q_lens=int32(q_lens), return_lse=True)
        clean()
        check(out, lse, orc.attention(q, cache, lens, D ** -0.5, q_lens), quantised, 3000)


# ---- scales of V over all of their range ---------------------------------------------------------------------
def with_v_exponents(cache, low, high, gen):
    """The same cache with every V row's exponent drawn from [low, high]."""
    c = list(cache)
    c[4] = torch.randint(low + 127, high + 128, c[4].shape, generator=gen).to(torch.uint8).cuda().view(torch.float8_e8m0fnu)
    return c


def check_scaled(got, lse, want, T, p_eps, floor):
    """As ``check``, for outputs of any size: ``floor`` is half the smallest step of what the output and its sums are held in."""
    out, _, mag, size = want
    share = 2.0 ** -23 * (got.shape[-1] + 3) * size[..., None] + 2.0 ** -18
    tol = out.abs() * torch.finfo(got.dtype).eps / 2 + mag * (p_eps / 2 + 2 * share + 2 * 2.0 ** -23 * (T + 64)) + floor
    assert torch.isfinite(got).all()
    worst = float(((got.double() - out).abs() - tol).max())
    assert worst <= 0, (worst, float(out.abs().max()))
    check(torch.zeros_like(got), lse, (torch.zeros_like(out), *want[1:]), True, T)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 3, 7, 60])
def test_v_exponents_over_their_whole_range(N, dtype, D):
    """4, 12, 28 and 240 rows of a head.  bf16: rows of V up to 448 * 2^105, and one at 2^119 where no sum of many can leave fp32; fp16:
    up to 448 * 2^6, which its outputs hold.  Probabilities are off by bf16's rounding at the most."""
    gen = torch.Generator().manual_seed(N + D)
    lens, bf16 = [700, 333], dtype == torch.bfloat16
    base = new_cache(gen, lens, 2, D, 32, "NHD", dtype, True)
    q = torch.randn((2, 8, N, D), generator=gen).to(dtype).cuda()
    p_eps = torch.finfo(torch.bfloat16).eps
    floor = 2.0 ** -134 if bf16 else 2.0 ** -25
    for low, high, one in ((-117, 105 if bf16 else 6, None), (66, 70, None), (-90, -86, None), (-117, 60, 119)):
        if not bf16 and high > 6 or one is not None and N == 60:
            continue
        cache = with_v_exponents(base, low, high, gen)
        if one is not None:
            page, off = orc.row_of(cache, 0, torch.tensor([555], device="cuda"))
            cache[4].view(torch.uint8)[page, :, off] = one + 127
        out, lse = chunk(q, cache, int32(lens), D ** -0.5, return_lse=True)
        clean()
        check_scaled(out, lse, orc.attention(q, cache, lens, D ** -0.5), 700, p_eps, floor)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 3, 7, 60])
def test_rows_of_v_of_the_smallest_scales(N, dtype):
    """Values down to 2^-126 are bf16 numbers: they reach the output.  (fp16 outputs hold none of them.)"""
    gen = torch.Generator().manual_seed(N)
    lens = [700, 333]
    q = torch.randn((2, 8, N, 64), generator=gen).to(dtype).cuda()
    cache = with_v_exponents(new_cache(gen, lens, 2, 64, 32, "NHD", dtype, True), -117, -114, gen)
    out, lse = chunk(q, cache, int32(lens), 0.125, return_lse=True)
    clean()
    want = orc.attention(q, cache, lens, 0.125)
    if dtype == torch.float16:
        assert not out.any()
        return
    assert (want[0].abs() > 2.0 ** -126).any()
    check_scaled(out, lse, want, 700, torch.finfo(torch.bfloat16).eps, 2.0 ** -134)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [3, 4, 7, 8, 60])
def test_small_rows_of_v_beside_a_row_of_another_size(N, D):
    """A row 2^80 times as large as the others has one column: the others' columns are what they are without it (more than 8 rows of a head, bf16)."""
    gen = torch.Generator().manual_seed(N + D)
    lens = [700, 333]
    cache = with_v_exponents(new_cache(gen, lens, 2, D, 32, "NHD", torch.bfloat16, True), -22, -18, gen)
    for z in range(2):
        page, off = orc.row_of(cache, z, torch.tensor([17], device="cuda"))
        cache[1].view(torch.uint8)[page, off] = 0
        cache[1].view(torch.uint8)[page, off, :, 0] = 0x7e
        cache[4].view(torch.uint8)[page, :, off] = 127 + 60
    q = torch.randn((2, 8, N, D), generator=gen).to(torch.bfloat16).cuda()
    out, lse = chunk(q, cache, int32(lens), D ** -0.5, return_lse=True)
    clean()
    want = orc.attention(q, cache, lens, D ** -0.5)
    assert (want[0][..., 0] > 2.0 ** 50).all() and (want[0][..., 1:].abs() < 1).all()
    check_scaled(out, lse, want, 700, torch.finfo(torch.bfloat16).eps, 2.0 ** -134)


# ---- counts that a call does not have ------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("path", [False, True])
def test_a_count_above_the_rows_of_an_append_is_reported(path, quantised):
    """The rows that there are go into the pages, as they do without a count; one below zero is none."""
    gen = torch.Generator().manual_seed(6)
    k = torch.randn((3, 2, 4, 64), generator=gen).to(torch.bfloat16).cuda()
    rows = int32([[2, 0, 3]] * 3) if path else None
    M = 3 if path else 4
    cache = list(new_cache(gen, [20, 20, 20], 2, 64, 16, "NHD", torch.bfloat16, quantised))
    other = [t.clone() if torch.is_tensor(t) else t for t in cache]
    append(k, k, cache, int32([14, 3, 0]), rows=rows)
    append(k, k, other, int32([14, 3, 0]), rows=rows, lens=int32([M, M, M]))
    clean()
    for count in (M + 1, INT_MAX):
        append(k, k, other, int32([14, 3, 0]), rows=rows, lens=int32([M, count, M]))
        assert fst.last_status(clear=True) == 18
    append(k, k, other, int32([0, 0, 0]), rows=rows, lens=int32([-1, -INT_MAX - 1, 0]))
    clean()
    for a, b in zip(cache[:5], other[:5]):
        assert a is b or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---- every byte that a scale can be -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_byte_under_every_scale(dtype):
    """Two heads of 128 bytes have all 256 values, 256 rows all scales: 2^(b - 127) for b from 0 to 254, NaN for 255.  One rounding."""
    value = torch.arange(256, dtype=torch.uint8).view(1, 1, 2, 128).expand(2, 128, 2, 128).contiguous().cuda().view(torch.float8_e4m3fn)
    scale = torch.arange(256, dtype=torch.uint8).view(2, 1, 128).expand(2, 2, 128).contiguous().cuda().view(torch.float8_e8m0fnu)
    table, n = int32([[0, 1]]), int32([256])
    got = fst.fst_cache_read(value, value, table, n, 256, k_scale=scale, v_scale=scale, dtype=dtype)
    clean()
    power = torch.cat([orc.pow2(torch.arange(255) - 127), torch.tensor([float("nan")], dtype=torch.float64)]).cuda()
    want = value.view(256, 2, 128).double().transpose(0, 1) * power[None, :, None]
    most = torch.finfo(torch.float16).max
    want = (want.clamp(-most, most) if dtype == torch.float16 else want).to(dtype)
    for x in got:
        assert torch.equal(torch.isnan(x[0]), torch.isnan(want)) and torch.equal(torch.nan_to_num(x[0]), torch.nan_to_num(want))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [1, 3, 7, 60])
def test_the_smallest_scale_byte_means_the_same_to_every_kernel(N, D):
    """Rows of V under b = 0, 2^-127: up to 2^-118, of which sums may lose what lies below 2^-126, the smallest normal number."""
    gen = torch.Generator().manual_seed(N)
    lens = [700, 333]
    q = torch.randn((2, 8, N, D), generator=gen).to(torch.bfloat16).cuda()
    cache = with_v_exponents(new_cache(gen, lens, 2, D, 32, "NHD", torch.bfloat16, True), -127, -127, gen)
    cache[1].view(torch.uint8).fill_(0x7e)                # 448 everywhere
    out, lse = chunk(q, cache, int32(lens), D ** -0.5, return_lse=True)
    clean()
    want = orc.attention(q, cache, lens, D ** -0.5)
    assert (want[0] > 2.0 ** -119).all()
    check_scaled(out, lse, want, 700, torch.finfo(torch.bfloat16).eps, 2.0 ** -126)
    # K under it: scores of next to nothing, so that all weights are alike
    cache = list(new_cache(gen, lens, 2, D, 32, "NHD", torch.bfloat16, True))
    cache[3].view(torch.uint8).zero_()
    check(*chunk(q, cache, int32(lens), D ** -0.5, return_lse=True), orc.attention(q, cache, lens, D ** -0.5), True, 700)
    clean()


# ---- calls that read what the launch ahead of them writes ---------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("N", [1, 12, 40])
def test_a_chain_of_calls_without_a_pause(N, quantised):
    """Rows, lengths, tables and results that the kernel just ahead writes: each call starts early and still sees them."""
    gen = torch.Generator().manual_seed(N)
    Z, H, D, steps = 4, 2, 64, 12
    base = new_cache(gen, [steps * N + N] * Z, H, D, 16, "NHD", torch.bfloat16, quantised)
    q0 = torch.randn((Z, H, N, D), generator=gen).to(torch.bfloat16).cuda()

    def run(pause):
        cache = [t.clone() if torch.is_tensor(t) else t for t in base]
        start, kv, x = int32([0] * Z), int32([0] * Z), q0.clone()
        outs, first = [], cache[2].clone()
        for i in range(steps):
            cache[2].copy_(first.roll(1, 0))              # another table, and this one again
            cache[2].copy_(first)
            kv.add_(N)
            pause()
            append(x, x, cache, start)                    # x: what the attention ahead has written
            pause()
            x = chunk(x, cache, kv, D ** -0.5)
            pause()
            k, v = read(cache, kv, steps * N)
            pause()
            x = x + k[:, :, i * N:i * N + N] * 0.5        # (of a length that is known here)
            start.add_(N)
            outs += [x, k, v]
        return outs

    want = run(torch.cuda.synchronize)
    for _ in range(5):
        for a, b in zip(run(lambda: None), want):
            assert torch.equal(a, b)
    clean()


# ---- what small probabilities lose ----------------------------------------------------------------------------
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 5, 12, 60])
def test_small_probabilities_lose_no_more_than_their_step(N, dtype, quantised):
    """One key whose value is zero has nearly all of the weight, the 60000 others 2^-25.5 of it each (2^-26 over 8 bits) and the value one.

    The second product's probabilities are fp16 (bf16 for bf16 queries over 16 bits or of more than 32 rows of a head).  Rounding costs each
    eps / 2 of itself, or half of fp16's smallest step, 2^-24: of the largest weight that is 2^-40, and 2^-32 on tcgen05 (more than 32
    rows), where weights are 2^15 and 2^7 times too large.  Sums of 16 keys go into fp32 accumulators, two roundings each at the most."""
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
            cache[which], cache[3 + which] = values.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).transpose(1, 2).contiguous().view(torch.float8_e8m0fnu)
    q = torch.zeros((1, H, N, D), dtype=dtype, device="cuda")
    q[..., 5] = 1.0
    out = chunk(q, cache, int32([T + N]), math.log(2) / 2, causal=False)
    clean()
    want, _, mag, size = orc.attention(q, cache, [T + N], math.log(2) / 2, causal=False)
    tcgen05 = N * H > 32
    in_bf16 = dtype == torch.bfloat16 and (tcgen05 or not quantised)
    p_eps = torch.finfo(torch.bfloat16 if in_bf16 else torch.float16).eps
    share = 2.0 ** -23 * (D + 3) * size[..., None] + 2.0 ** -18
    tol = want * torch.finfo(dtype).eps / 2 + mag * (p_eps / 2 + 2 * share + 2 * 2.0 ** -23 * (T / 8 + 64)) + 2.0 ** -25
    if not in_bf16:
        tol = tol + (T + N) * 2.0 ** -(32 if tcgen05 else 40)
    worst = float(((out.double() - want).abs() - tol).max())
    assert worst <= 0, (worst, float(want.max()), float(out.double().max()))


# ---- many short items ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Z,H,H_kv,N,T", [(40, 8, 8, 300, 6), (64, 16, 8, 64, 100), (40, 10, 5, 1258, 17)])
def test_many_short_items_of_many_rows(Z, H, H_kv, N, T, D):
    """Items of one tile, some of rows that see nothing, one after the other: every wait ends, and every call gives the same."""
    gen = torch.Generator().manual_seed(D)
    lens = [int(x) for x in torch.randint(0, T + 1, (Z,), generator=gen)]
    cache = new_cache(gen, [T] * Z, H_kv, D, 32, "HND", torch.bfloat16, False, extra=200)
    q = torch.randn((Z, H, N, D), generator=gen).to(torch.bfloat16).cuda()
    kv = int32(lens)
    out, lse = chunk(q, cache, kv, D ** -0.5, return_lse=True)
    check(out, lse, orc.attention(q, cache, lens, D ** -0.5), False, T)
    clean()
    for _ in range(200):
        again = chunk(q, cache, kv, D ** -0.5)
    clean()
    assert torch.equal(again, out)
