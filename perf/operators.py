"""The operators around a paged K/V cache, as a list of measurable cases.

A decoder keeps the keys and values of its sequences in pages.  Three operators work on them:

  append    new K/V rows go into the pages behind a sequence's end: one row per sequence of a decode
            step, a chunk of a prompt, or the accepted path of a token tree; as they are, or quantised
            to e4m3 with one power of two per row and head
  read      the rows of sequences come back out of the pages as contiguous tensors, dequantised
  chunk     the queries of a chunk of new tokens (one token of a decode step, a few drafted ones, a
            piece of a prompt) attend to the cache, which holds the chunk's own rows too

``listed()`` names twelve cases over these, ``draw(rng)`` gives others of the same ranges.  With
``own`` false ``run`` computes the operators from elementary tensor operations in 32 bits; ``exact``
restates them in 64 bits.

Quantisation of a row x of one head: with a the largest |x_i|, the exponent e is the smallest
integer in [-117, 119] with a <= 448 * 2^e, element i is held as e4m3(x_i * 2^-e), rounded to the
nearest, ties to even, at most 448 in magnitude, and the row stands for e4m3 * 2^e.  (A row with an
element that is not finite has zeros and the scale NaN.)
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a few sequences, quantised as it is written: launch latency
        dict(name="append_token_e4m3", op="append", Z=8, N=1, rows=0, H_kv=8, D=128, dtype="bf16", quantised=True,
             page=64, layout="NHD", short=60, long=4000),
        # pieces of four prompts, the last one not full
        dict(name="append_chunk_e4m3", op="append", Z=4, N=2048, rows=0, H_kv=8, D=128, dtype="bf16", quantised=True,
             page=64, layout="NHD", short=0, long=3001),
        # the accepted paths of 64 token trees of 256 nodes, into a cache that holds the rows as they are
        dict(name="append_path_fp16", op="append", Z=64, N=256, rows=9, H_kv=32, D=128, dtype="fp16", quantised=False,
             page=16, layout="HND", short=31, long=2000),
        # a long prompt for calls that take contiguous K/V tensors
        dict(name="read_long_e4m3", op="read", Z=1, H_kv=8, D=128, dtype="bf16", quantised=True, page=64, layout="NHD",
             short=30011, long=30011),
        # a batch of prompts of different lengths, gathered as they are
        dict(name="read_ragged_fp16", op="read", Z=16, H_kv=8, D=64, dtype="fp16", quantised=False, page=32, layout="HND",
             short=501, long=3001),
        # one token of one short sequence, every query head with K/V of its own: launch latency
        dict(name="token_short", op="chunk", Z=1, N=1, H=32, H_kv=32, D=128, dtype="fp16", quantised=False, page=16,
             layout="NHD", short=77, long=77, ragged=False, causal=True),
        # a decode step of a full batch
        dict(name="token_batch", op="chunk", Z=64, N=1, H=32, H_kv=8, D=128, dtype="bf16", quantised=False, page=64,
             layout="NHD", short=1000, long=8191, ragged=False, causal=True),
        # a decode step behind very long prompts, quantised cache
        dict(name="token_long_e4m3", op="chunk", Z=2, N=1, H=64, H_kv=8, D=128, dtype="bf16", quantised=True, page=64,
             layout="NHD", short=100003, long=130001, ragged=False, causal=True),
        # drafted tokens being checked: a few queries per sequence, not the same number everywhere
        dict(name="draft_e4m3", op="chunk", Z=24, N=7, H=32, H_kv=8, D=64, dtype="fp16", quantised=True, page=128,
             layout="HND", short=500, long=4100, ragged=True, causal=True),
        # the first chunks of four prompts, nothing cached before them
        dict(name="chunk_first", op="chunk", Z=4, N=1024, H=32, H_kv=32, D=64, dtype="fp16", quantised=False, page=16,
             layout="NHD", short=1024, long=1024, ragged=False, causal=True),
        # a late chunk of a long prompt: the largest case
        dict(name="chunk_long", op="chunk", Z=1, N=4096, H=32, H_kv=8, D=128, dtype="bf16", quantised=False, page=64,
             layout="NHD", short=16400, long=16400, ragged=False, causal=True),
        # chunks of unlike lengths behind unlike prompts, quantised cache
        dict(name="chunk_ragged_e4m3", op="chunk", Z=3, N=2000, H=32, H_kv=4, D=128, dtype="bf16", quantised=True, page=64,
             layout="NHD", short=2001, long=9001, ragged=True, causal=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "read", "chunk", "chunk", "chunk"])
    D = rng.choice([64, 128, 128])
    H_kv = rng.choice([1, 2, 4, 8, 8, 12, 32])
    case = dict(op=op, H_kv=H_kv, D=D, dtype=rng.choice(["fp16", "bf16"]), quantised=rng.random() < 0.5,
                page=rng.choice([16, 32, 64, 128]), layout=rng.choice(["NHD", "HND"]))
    if op == "append":
        Z = _log_int(rng, 1, 96)
        N = _log_int(rng, 1, max(1, 8192 * 8 // (Z * max(8, H_kv))))
        rows = rng.randint(1, min(N, 12)) if rng.random() < 0.35 else 0
        short = rng.randint(0, 500)
        case.update(Z=Z, N=N, rows=rows, short=short, long=short + _log_int(rng, 1, 4000))
    elif op == "read":
        Z = _log_int(rng, 1, 32)
        long = _log_int(rng, 1, max(1, 30011 * 8 // (Z * max(8, H_kv))))
        case.update(Z=Z, short=rng.randint((long + 1) // 2, long), long=long)
    else:
        group = rng.choice([1, 2, 4, 5, 7, 8])
        H_kv = case["H_kv"] = min(H_kv, 64 // group)
        if rng.random() < 0.5:                        # a token, or a few
            N, Z = rng.choice([1, 1, 2, 4, 7, 13]), _log_int(rng, 1, 64)
            long = _log_int(rng, N, max(N, min(130001, 260000 * 8 // (Z * H_kv))))
        else:                                         # pieces of prompts
            N, Z = _log_int(rng, 16, 4096), _log_int(rng, 1, 8)
            long = _log_int(rng, N, max(N, min(16400, 4096 * 14000 * 32 // (Z * N * H_kv * group))))
            Z = max(1, min(Z, 4096 * 14000 * 32 // (N * long * H_kv * group)))
        ragged = Z > 1 and rng.random() < 0.5
        case.update(Z=Z, N=N, H=H_kv * group, short=rng.randint(max(N, long // 4), long), long=long, ragged=ragged,
                    causal=rng.random() < 0.85)
    return case


# ---------------------------------------------------------------------------------------------
# lengths of a case's sequences: spread evenly over the range, in no order
# ---------------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * (i * step % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _lengths(case):
    """(rows in the cache before an append, or in all, new rows or queries) of every sequence."""
    cached = _spread(case["short"], case["long"], case["Z"])
    if case["op"] == "append":
        top = case["rows"] or case["N"]
        return cached, _spread(max(1, top // 3), top, case["Z"])[::-1]
    if case["op"] == "read":
        return cached, [0] * case["Z"]
    top = case["N"]
    return cached, _spread(max(1, top // 7), top, case["Z"])[::-1] if case["ragged"] else [top] * case["Z"]


# ---------------------------------------------------------------------------------------------
# plain form of the quantisation
# ---------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e in float32, e in [-126, 127], by its bits."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x):
    """(e4m3 values, e8m0 scales) of rows along the last dimension."""
    x = x.float()
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, torch.zeros_like(x))
    amax = x.abs().amax(-1)
    mant, expo = torch.frexp(amax)                    # amax = mant * 2^expo, mant in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(mant <= 0.875, expo - 9, expo - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -117)).clamp(-117, 119).to(torch.int32)
    y = (x * _pow2(-e)[..., None]).clamp(-448.0, 448.0)
    return y.to(E4M3), torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8).view(E8M0)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _rows(gen, shape, dtype, channel):
    """Rows as projections give them: a few channels are several times larger than the others."""
    x = torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32)
    return (x * channel).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    Z, H_kv, D, page = case["Z"], case["H_kv"], case["D"], case["page"]
    dtype = DTYPES[case["dtype"]]
    cached, new = _lengths(case)
    append = case["op"] == "append"
    total = [c + n for c, n in zip(cached, new)] if append else cached
    width = -(-max(total) // page)
    n_pages = sum(-(-t // page) for t in total) + 3
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((Z, width), -1, dtype=torch.int32, device="cuda")
    first = 0
    for z, t in enumerate(total):                     # pages as an allocator hands them out: in no order
        used = -(-t // page)
        table[z, :used] = order[first:first + used]
        first += used
    state = dict(case=dict(case), table=table, width=width,
                 lens=torch.tensor(cached, dtype=torch.int32, device="cuda"),
                 new=torch.tensor(new, dtype=torch.int32, device="cuda"))

    shape = (n_pages, page, H_kv, D) if case["layout"] == "NHD" else (n_pages, H_kv, page, D)
    for name in ("k", "v"):
        channel = torch.exp(0.5 * torch.randn((D,), device="cuda", generator=gen))
        if append:
            pool = torch.zeros(shape, dtype=E4M3 if case["quantised"] else dtype, device="cuda")
            scale = torch.zeros((n_pages, H_kv, page), dtype=torch.uint8, device="cuda").view(E8M0)
            state[name] = _rows(gen, (Z, H_kv, case["N"], D), dtype, channel)
        else:
            pool = _rows(gen, shape, dtype, channel)
            scale = None
            if case["quantised"]:
                pool, scale = _quantise(pool)
                scale = scale.view(torch.uint8)
                scale = (scale.transpose(1, 2) if case["layout"] == "NHD" else scale).contiguous().view(E8M0)
        state[name + "_pool"], state[name + "_scale"] = pool, scale if case["quantised"] else None
    if append and case["rows"]:                       # the accepted path of every tree, its nodes ascending
        state["path"] = torch.sort(torch.rand((Z, case["N"]), device="cuda", generator=gen).argsort(-1)[:, :case["rows"]],
                                   -1).values.to(torch.int32)
    if case["op"] == "chunk":
        state["q"] = torch.randn((Z, case["H"], case["N"], D), device="cuda", generator=gen).to(dtype)
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"append": _append, "read": _read, "chunk": _chunk}[case["op"]](state, case)


def _append(s, case):
    pools = (s["k_pool"], s["v_pool"])
    scales = (s["k_scale"], s["v_scale"]) if case["quantised"] else ()
    if own:
        import fstattention_b200 as fst
        fst.fst_cache_append(s["k"], s["v"], *pools, s["table"], s["lens"], lens=s["new"], rows=s.get("path"),
                             k_scale=s["k_scale"], v_scale=s["v_scale"], pool_layout=case["layout"])
        return pools + scales
    # rows behind a sequence's count repeat its last one, which is then written several times
    j = torch.arange(case["rows"] or case["N"], device="cuda")[None, :].minimum(s["new"][:, None].long() - 1)
    at = s["lens"][:, None].long() + j
    page = s["table"].long().gather(1, at // case["page"])
    off = at % case["page"]
    src = s["path"].long().gather(1, j) if "path" in s else j
    for n, (x, pool) in enumerate(((s["k"], pools[0]), (s["v"], pools[1]))):
        x = x.gather(2, src[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3])).transpose(1, 2)     # [Z, M, H_kv, D]
        if case["quantised"]:
            x, scale = _quantise(x)
            scales[n].view(torch.uint8).transpose(1, 2)[page, off] = scale.view(torch.uint8)
            x, pool = x.view(torch.uint8), pool.view(torch.uint8)
        (pool if case["layout"] == "NHD" else pool.transpose(1, 2))[page, off] = x
    return pools + scales


def _gather(s, case, name):
    """float32 [Z, H_kv, width * page, D]: the rows of every sequence, past its end whatever a page holds, or page 0."""
    pages = s["table"].long().clamp(min=0)
    pool = s[name + "_pool"]
    if case["layout"] == "NHD":
        pool = pool.transpose(1, 2)
    x = (pool.view(torch.uint8)[pages].view(E4M3) if case["quantised"] else pool[pages]).float()    # [Z, width, H_kv, page, D]
    if case["quantised"]:
        x = x * s[name + "_scale"].view(torch.uint8)[pages].view(E8M0).float()[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _read(s, case):
    if own:
        import fstattention_b200 as fst
        return fst.fst_cache_read(s["k_pool"], s["v_pool"], s["table"], s["lens"], case["long"], k_scale=s["k_scale"],
                                  v_scale=s["v_scale"], dtype=DTYPES[case["dtype"]], pool_layout=case["layout"])
    there = (torch.arange(case["long"], device="cuda")[None, :] < s["lens"][:, None])[:, None, :, None]
    k, v = (_gather(s, case, name)[:, :, :case["long"]] for name in ("k", "v"))
    dtype = DTYPES[case["dtype"]]
    zero = torch.zeros((), device="cuda")
    return torch.where(there, k, zero).to(dtype), torch.where(there, v, zero).to(dtype)


def _chunk(s, case):
    q = s["q"]
    Z, H, N, D = q.shape
    if own:
        import fstattention_b200 as fst
        return fst.fst_attention_chunk(q, s["k_pool"], s["v_pool"], s["table"], s["lens"], D ** -0.5,
                                       q_lens=s["new"] if case["ragged"] else None, causal=case["causal"],
                                       k_scale=s["k_scale"], v_scale=s["v_scale"], pool_layout=case["layout"])
    H_kv = case["H_kv"]
    col = torch.arange(s["width"] * case["page"], device="cuda")
    k = _gather(s, case, "k")
    score = (q.float() * D ** -0.5).reshape(Z, H_kv, H // H_kv * N, D) @ k.transpose(2, 3)
    del k
    score = score.view(Z, H_kv, H // H_kv, N, -1)
    i = torch.arange(N, device="cuda")
    end = s["lens"][:, None] if not case["causal"] else (s["lens"] - s["new"])[:, None] + i + 1           # keys of query i
    end = torch.where(i < s["new"][:, None], end.expand(Z, N), torch.zeros_like(end.expand(Z, N)))
    seen = (col < end[..., None])[:, None, None]                                                        # [Z, 1, 1, N, T]
    score = torch.where(seen, score, torch.full((), -math.inf, device="cuda"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    del score
    total = p.sum(-1, keepdim=True)
    v = torch.where((col < s["lens"][:, None])[:, None, :, None], _gather(s, case, "v"), torch.zeros((), device="cuda"))
    out = (p.view(Z, H_kv, H // H_kv * N, -1) @ v).view(Z, H_kv, H // H_kv, N, D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.reshape(Z, H, N, D).to(q.dtype)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def _pairs(case):
    """(query, key) pairs of one query head."""
    cached, new = _lengths(case)
    if not case["causal"]:
        return sum(c * n for c, n in zip(cached, new))
    return sum(n * (c - n) + n * (n + 1) // 2 for c, n in zip(cached, new))


def work(case):
    cached, new = _lengths(case)
    width = case["H_kv"] * case["D"]
    held = 2 * (width + case["H_kv"]) if case["quantised"] else 4 * width          # bytes of a cached row, K and V
    index = 4 * sum(-(-c // case["page"]) for c in cached) + 8 * case["Z"]
    if case["op"] == "append":
        return {"bytes": sum(new) * (4 * width + held) + 8 * case["Z"] + 4 * sum(new), "flops": 2 * width * sum(new)}
    if case["op"] == "read":
        return {"bytes": sum(cached) * held + 4 * width * case["Z"] * case["long"] + index, "flops": 2 * width * sum(cached)}
    return {"bytes": sum(cached) * held + 4 * case["H"] * case["D"] * sum(new) + index,
            "flops": 4 * case["D"] * case["H"] * _pairs(case)}


# ---------------------------------------------------------------------------------------------
# the operators in 64 bits, from their definitions
# ---------------------------------------------------------------------------------------------
def _exact_pow2(e):
    """2^e in float64 by its bits: the device's exp2 need not be exact."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_e4m3(x):
    """(values that x's rows are held as, their exponents) in float64."""
    x = x.double()
    a = x.abs().amax(-1)
    e = torch.ceil(torch.log2(a / 448) - 1e-6).clamp(-117, 119)       # 16-bit values: the next above 448 * 2^e is 7e-4 off
    e = e.masked_fill(a == 0, -117)
    y = x / _exact_pow2(e)[..., None]
    step = _exact_pow2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -9))).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448), e


def _exact_rows(s, case, z, h, count, name):
    """float64 [count, D]: the first rows of sequence z, K/V head h, one by one out of their pages."""
    at = torch.arange(count, device="cuda")
    page, off = s["table"][z].long()[at // case["page"]], at % case["page"]
    pool = s[name + "_pool"]
    flat = pool.view(torch.uint8) if case["quantised"] else pool
    x = flat[page, off, h] if case["layout"] == "NHD" else flat[page, h, off]
    if not case["quantised"]:
        return x.double()
    scale = _exact_pow2(s[name + "_scale"].view(torch.uint8)[page, h, off].long() - 127)
    return x.view(E4M3).double() * scale[:, None]


def exact(case, seed):
    s = prepare(case, seed)
    cached, new = _lengths(case)
    if case["op"] == "append":
        outs = [s["k_pool"].double(), s["v_pool"].double()]
        outs += [s["k_scale"].double(), s["v_scale"].double()] if case["quantised"] else []
        for z in range(case["Z"]):
            take = s["path"][z, :new[z]].long() if "path" in s else torch.arange(new[z], device="cuda")
            at = cached[z] + torch.arange(new[z], device="cuda")
            page, off = s["table"][z].long()[at // case["page"]], at % case["page"]
            for n, name in enumerate(("k", "v")):
                x = s[name][z][:, take].transpose(0, 1)                       # [count, H_kv, D]
                if case["quantised"]:
                    x, e = _exact_e4m3(x)
                    outs[2 + n].transpose(1, 2)[page, off] = _exact_pow2(e)
                (outs[n] if case["layout"] == "NHD" else outs[n].transpose(1, 2))[page, off] = x.double()
        return tuple(outs)
    Z, H_kv, D = case["Z"], case["H_kv"], case["D"]
    if case["op"] == "read":
        outs = [torch.zeros((Z, H_kv, case["long"], D), dtype=torch.float64, device="cuda") for _ in range(2)]
        for z in range(Z):
            for h in range(H_kv):
                for out, name in zip(outs, ("k", "v")):
                    out[z, h, :cached[z]] = _exact_rows(s, case, z, h, cached[z], name)
        return tuple(outs)
    out = torch.zeros((Z, case["H"], case["N"], D), dtype=torch.float64, device="cuda")
    group = case["H"] // H_kv
    for z in range(Z):
        n, T = new[z], cached[z]
        hidden = torch.zeros((n, T), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden = torch.arange(T, device="cuda")[None, :] > torch.arange(T - n, T, device="cuda")[:, None]
        for h in range(H_kv):
            k, v = (_exact_rows(s, case, z, h, T, name) for name in ("k", "v"))
            q = s["q"][z, h * group:(h + 1) * group, :n].double()
            weight = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill_(hidden, -math.inf), -1)
            out[z, h * group:(h + 1) * group, :n] = weight @ v
    return out
