"""A paged K/V cache and the attention over it, restated in 64 bits from the definitions (test infrastructure only).

Works on tensors of any device.  A cache is ``(k_pool, v_pool, block_table, k_scale, v_scale, layout)`` as the package
takes it; 16-bit caches have ``None`` for the scales.
"""
import math

import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def pow2(e):
    """2^e in float64, e integers in [-1022, 1023], from its bits (the device's pow and exp2 need not be exact)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x):
    """(values [.., D] float64, exponents [..] int64, finite [..]) that rows x [.., D] are held as."""
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, torch.zeros_like(x))
    a = x.abs().amax(-1)
    mant, expo = torch.frexp(a)                       # a = mant 2^expo, mant in [1/2, 1)
    e = expo.long() - 9 + (mant > 448 / 512).long()
    e = torch.where(a == 0, torch.full_like(e, -117), e).clamp(-117, 119)
    y = x * pow2(-e)[..., None]
    _, top = torch.frexp(y)                           # |y| in [2^(top - 1), 2^top)
    step = pow2(top.long().clamp(min=-5) - 4)             # subnormals: steps of 2^-9
    return (torch.round(y / step) * step).clamp(-448, 448), e, finite


def row_of(cache, z, r):
    """(page, row in the page) of rows r (a tensor) of sequence z."""
    k_pool, table, layout = cache[0], cache[2], cache[5]
    page = k_pool.shape[1 if layout == "NHD" else 2]
    return table[z].long()[r // page], r % page


def rows(cache, z, count, which):
    """float64 [H_kv, count, D]: the first ``count`` rows of K (which=0) or V (1) of sequence z."""
    pool, scale, layout = cache[which], cache[3 + which], cache[5]
    nhd = pool if layout == "NHD" else pool.transpose(1, 2)
    page, off = row_of(cache, z, torch.arange(count, device=pool.device))
    if pool.dtype != E4M3:
        return nhd[page, off].double().transpose(0, 1)
    x = nhd.view(torch.uint8)[page, off].view(E4M3).double()
    b = scale.view(torch.uint8).transpose(1, 2)[page, off].long()
    f = torch.where(b == 255, torch.full_like(b, math.nan, dtype=torch.float64), pow2(b - 127))
    return (x * f[..., None]).transpose(0, 1)


def attention(q, cache, kv_lens, sm_scale, q_lens=None, causal=True):
    """(out [Z, H, N, D], lse [Z, H, N] in base 2, and what error bounds are made of: weighted |v| [Z, H, N, D] and the
    largest sm_scale sum_d |q_d k_d| of a row [Z, H, N]), all float64.  Rows i >= q_lens[z] are zeros."""
    Z, H, N, D = q.shape
    out, mag = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    lse, size = torch.full((Z, H, N), -math.inf, dtype=torch.float64, device=q.device), torch.zeros((Z, H, N), dtype=torch.float64, device=q.device)
    for z in range(Z):
        T, n = int(kv_lens[z]), N if q_lens is None else int(q_lens[z])
        if T == 0 or n == 0:
            continue
        k, v = rows(cache, z, T, 0), rows(cache, z, T, 1)
        group = H // k.shape[0]
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        qz = q[z, :, :n].double()
        s = qz @ k.transpose(1, 2) * sm_scale
        seen = torch.ones((n, T), dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(T, device=q.device)[None] <= torch.arange(T - n, T, device=q.device)[:, None]
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(p), p / total)
        lse[z, :, :n] = torch.where(total == 0, torch.full_like(total, -math.inf), top + torch.log(total))[..., 0] / math.log(2)
        keep = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
        out[z, :, :n] = w @ keep
        odd = (~torch.isfinite(v)).any(0).any(-1).nonzero()[:, 0]                 # keys whose V is not finite somewhere
        for j in odd.tolist():
            extra = torch.where(torch.isfinite(v[:, j]), torch.zeros_like(v[:, j]), v[:, j])
            out[z, :, :n] += torch.where(seen[:, j][None, :, None], extra[:, None], torch.zeros_like(extra[:, None]))
        mag[z, :, :n] = w @ keep.abs()
        size[z, :, :n] = torch.where(seen, (qz.abs() @ k.abs().transpose(1, 2)) * sm_scale, torch.zeros_like(s)).amax(-1)
    return out, lse, mag, size
