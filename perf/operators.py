"""The paged 8-bit cache of the serving path, operator by operator: block tables and slot maps from request
lengths, the quantising cache write, and attention over the cache.

The cache holds E4M3 codes, one FP32 scale for each page and key/value head: head h owns rows
[h * npages * page, (h + 1) * npages * page) of `q_k` / `q_v` (D bytes a row) and entries [h * npages, ...) of
`s_k` / `s_v`; position t of a sequence lives in row bt[t // page] * page + t % page of every head.

`listed()` and `draw()` give cases, `prepare()` the device arrays a serving loop holds before the call, `run()` one
call: in elementary torch operations (`own` false) or through the framework's entry points (`own` true)."""
import math

import torch

own = False

E4M3_MAX = 448.0
MIN_EXP, MAX_EXP = -60, 60  # range of the scales' exponents
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 64 requests: every request gets one token, one in `page` of them a new page
        dict(name="tables decode 64", op="tables", nseq=64, lo=1, hi=4096, fresh_lo=1, fresh_hi=1, page=16),
        # a mixed step of many requests: drafted tokens and short prompt pieces
        dict(name="tables mixed 500", op="tables", nseq=500, lo=0, hi=8192, fresh_lo=1, fresh_hi=64, page=16),
        # long prompts alone, at the largest token count of a step
        dict(name="tables prompts 8", op="tables", nseq=8, lo=0, hi=64, fresh_lo=4000, fresh_hi=8192, page=64),
        # the write of a decode step of 64 requests out of one fused projection row per token
        dict(name="write decode 64", op="write", nseq=64, lo=1, hi=4096, fresh_lo=1, fresh_hi=1, page=16, hq=64,
             hkv=8, d=128, dtype="f16"),
        # chunked prompts on top of short contexts, narrow heads
        dict(name="write chunks 1.5k", op="write", nseq=5, lo=3, hi=900, fresh_lo=100, fresh_hi=700, page=32, hq=12,
             hkv=4, d=64, dtype="f16"),
        # the largest prompt step
        dict(name="write prompts 16k", op="write", nseq=4, lo=0, hi=100, fresh_lo=2000, fresh_hi=6000, page=64, hq=32,
             hkv=8, d=128, dtype="bf16"),
        # one request, a short context: latency
        dict(name="attend 1 x 777", op="attend", nseq=1, kv_lo=777, kv_hi=777, q_lo=1, q_hi=1, hq=32, hkv=8, d=128,
             page=16, dtype="f16", causal=True),
        # a decode step over ragged contexts, 64 query heads on 8 key/value heads
        dict(name="attend 64 ragged", op="attend", nseq=64, kv_lo=100, kv_hi=8192, q_lo=1, q_hi=1, hq=64, hkv=8,
             d=128, page=16, dtype="bf16", causal=True),
        # a few long contexts
        dict(name="attend 4 x 128k", op="attend", nseq=4, kv_lo=131072, kv_hi=131072, q_lo=1, q_hi=1, hq=32, hkv=8,
             d=128, page=64, dtype="bf16", causal=True),
        # several drafted tokens a request, verified in one step
        dict(name="attend drafts 24", op="attend", nseq=24, kv_lo=300, kv_hi=5000, q_lo=2, q_hi=5, hq=12, hkv=4, d=64,
             page=32, dtype="f16", causal=True),
        # prompt chunks on top of a cached context
        dict(name="attend chunks 2 x 1k", op="attend", nseq=2, kv_lo=4096, kv_hi=6000, q_lo=1000, q_hi=1024, hq=32,
             hkv=8, d=128, page=64, dtype="bf16", causal=True),
        # cross attention: decoder prompts over the states of an encoder, which have lengths of their own
        dict(name="attend encoder 16", op="attend", nseq=16, kv_lo=400, kv_hi=1500, q_lo=1, q_hi=224, hq=16, hkv=16,
             d=64, page=32, dtype="f16", causal=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "write", "attend", "attend"])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if op in ("tables", "write"):
        nseq = _log_int(rng, 1, 500 if op == "tables" else 200)
        fresh_hi = _log_int(rng, 1, max(1, 16000 // nseq))
        case = dict(op=op, nseq=nseq, lo=rng.choice([0, 1, 40]), hi=_log_int(rng, 41, 8192 if op == "tables" else 2000),
                    fresh_lo=rng.randint(1, fresh_hi), fresh_hi=fresh_hi, page=page)
        if op == "write":
            hkv = rng.choice([1, 2, 4, 8])
            case.update(hq=hkv * rng.choice([1, 2, 3, 8]), hkv=hkv, d=rng.choice([64, 128]),
                        dtype=rng.choice(["f16", "bf16"]))
        return case
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8, 16])
    form = rng.choice(["decode", "decode", "drafts", "chunks", "encoder"])
    if form in ("decode", "drafts"):
        nseq = _log_int(rng, 1, 128)
        kv_hi = _log_int(rng, 20, max(40, min(131072, 2 ** 22 // (nseq * hkv))))
        q_lo, q_hi = (1, 1) if form == "decode" else (1, rng.randint(2, 8))
    else:
        nseq, hkv, group = _log_int(rng, 1, 16), rng.choice([2, 4, 8]), rng.choice([1, 2, 3, 4])
        kv_hi = _log_int(rng, 200, max(300, min(5000, 12000 // nseq)))
        q_hi = _log_int(rng, 17, max(20, 2048 // nseq))
        q_lo = rng.randint(1, q_hi)
    return dict(op="attend", nseq=nseq, kv_lo=rng.randint(1, kv_hi), kv_hi=kv_hi, q_lo=q_lo, q_hi=q_hi,
                hq=hkv * group, hkv=hkv, d=rng.choice([64, 128]), page=page, dtype=rng.choice(["f16", "bf16"]),
                causal=form != "encoder")


def _lengths(n, lo, hi, phase):
    """n whole numbers of lo..hi, spread over their logarithm, from the case alone."""
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [min(hi, max(lo, int(round(math.exp(a + (b - a) * ((0.6180339887498949 * (i + 1) + phase) % 1.0)) - 1))))
            for i in range(n)]


def _requests(case):
    """(cached positions, new tokens, positions attended to) of every request."""
    if case["op"] == "attend":
        fresh = _lengths(case["nseq"], case["q_lo"], case["q_hi"], 0.37)
        kv = _lengths(case["nseq"], case["kv_lo"], case["kv_hi"], 0.11)
        # causal: the new tokens are the last ones of the context; an encoder's states have lengths of their own
        return None, fresh, [a + b for a, b in zip(kv, fresh)] if case["causal"] else kv
    cached = _lengths(case["nseq"], case["lo"], case["hi"], 0.11)
    fresh = _lengths(case["nseq"], case["fresh_lo"], case["fresh_hi"], 0.37)
    return cached, fresh, [a + b for a, b in zip(cached, fresh)]


def _pages(n, page):
    return -(-n // page)


def work(case):
    cached, fresh, total = _requests(case)
    tokens, page = sum(fresh), case["page"]
    if case["op"] == "tables":
        new = sum(_pages(t, page) - _pages(c, page) for c, t in zip(cached, total))
        return {"bytes": 4 * (5 * case["nseq"] + 2 * new + 2 * tokens), "flops": 0}
    hkv, d = case["hkv"], case["d"]
    if case["op"] == "write":
        touched = sum(_pages(t, page) - c // page for c, t in zip(cached, total))
        return {"bytes": 2 * tokens * hkv * d * 3 + 2 * touched * hkv * 4 + 4 * tokens, "flops": 0}
    read = sum(total)
    scales = sum(_pages(t, page) for t in total)
    pairs = sum(q * t - (q * (q - 1) // 2 if case["causal"] else 0) for q, t in zip(fresh, total))
    return {"bytes": 2 * hkv * (read * d + 4 * scales) + 4 * scales + tokens * case["hq"] * (4 * d + 4),
            "flops": 4 * pairs * case["hq"] * d}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(counts):
    total, out = 0, [0]
    for c in counts:
        total += c
        out.append(total)
    return out


def _cache(gen, hkv, npages, page, d):
    """A pool of codes and scales: values of unit size, the scales of neighbouring pages up to a factor of four apart."""
    codes = torch.randn(2, hkv, npages * page, d, generator=gen, device="cuda", dtype=torch.float16)
    codes = (codes * 64).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.exp2(torch.randint(-7, -4, (2, hkv, npages), generator=gen, device="cuda").float())
    return {"q_k": codes[0], "q_v": codes[1], "s_k": scales[0].contiguous(), "s_v": scales[1].contiguous()}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    cached, fresh, total = _requests(case)
    nseq, page = case["nseq"], case["page"]
    stride = max(_pages(t, page) for t in total) + 1
    held = [_pages(t, page) for t in (cached if case["op"] == "tables" else total)]
    npages = sum(_pages(t, page) for t in total) + 7
    order = torch.randperm(npages, generator=gen, device="cuda").to(torch.int32)
    bt = torch.full((nseq, stride), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(stride, device="cuda")
    mine = col[None] < _ints(held)[:, None]
    bt[mine] = order[: sum(held)]
    s = {"case": case, "page": page, "npages": npages, "nseq": nseq, "bt": bt, "tokens": sum(fresh),
         "max_q": max(fresh), "max_len": max(total), "q_offsets": _ints(_offsets(fresh)), "seq_lens": _ints(total)}
    if case["op"] == "tables":
        s.update(cached=_ints(cached), fresh=_ints(fresh), free=order[sum(held):].contiguous(),
                 taken=_ints([0]), taken_out=_ints([0]), seq_lens=torch.empty_like(s["seq_lens"]),
                 q_offsets=torch.empty_like(s["q_offsets"]),
                 slots=torch.empty(sum(fresh) + 5, dtype=torch.int32, device="cuda"),
                 positions=torch.empty(sum(fresh) + 5, dtype=torch.int32, device="cuda"))
        return s
    hq, hkv, d, dtype = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    s.update(_cache(gen, hkv, npages, page, d), hq=hq, hkv=hkv, d=d, dtype=dtype)
    if case["op"] == "write":
        # one fused projection row a token: query heads, key heads, value heads; a token's own size varies
        rows = torch.randn(sum(fresh), (hq + 2 * hkv) * d, generator=gen, device="cuda")
        rows *= torch.exp2(torch.randn(sum(fresh), 1, generator=gen, device="cuda"))
        s["rows"] = rows.to(dtype)
        seq = torch.repeat_interleave(torch.arange(nseq, device="cuda"), _ints(fresh))
        pos = torch.arange(sum(fresh), device="cuda") - s["q_offsets"][seq] + _ints(cached)[seq]
        s["slots"] = (bt[seq, pos // page] * page + pos % page).to(torch.int32)
        return s
    s["q"] = (1.5 * torch.randn(sum(fresh), hq, d, generator=gen, device="cuda")).to(dtype)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(sum(fresh), hq, device="cuda")
    s["causal"] = case["causal"]
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------

def _plain_tables(s):
    page, bt, n = s["page"], s["bt"], s["slots"].numel()
    cached, fresh, free = s["cached"].long(), s["fresh"].long(), s["free"]
    total = cached + fresh
    first, last = (cached + page - 1) // page, (total + page - 1) // page
    need = last - first
    ahead = torch.cumsum(need, 0) - need + s["taken"].long()
    col = torch.arange(bt.shape[1], device="cuda")[None]
    at = ahead[:, None] + col - first[:, None]
    got = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    bt.copy_(torch.where((col >= first[:, None]) & (col < last[:, None]), got, bt))
    ends = torch.cumsum(fresh, 0)
    t = torch.arange(n, device="cuda")
    seq = torch.searchsorted(ends, t, right=True).clamp(max=s["nseq"] - 1)
    pos = t - (ends - fresh)[seq] + cached[seq]
    real = t < ends[-1]
    where = bt[seq, (pos // page).clamp(max=bt.shape[1] - 1)].long()
    slots = torch.where(real & (where >= 0), where * page + pos % page, -1)
    taken = (s["taken"].long() + need.sum()).clamp(max=free.numel())
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    return {"bt": bt, "seq_lens": total.int(), "q_offsets": offsets.int(), "slots": slots.int(),
            "positions": torch.where(real, pos, 0).int(), "taken": taken.int()}


def _plain_write_side(s, codes, scales, x):
    """One side (keys or values) of the write: x is [tokens][heads][D]."""
    page, npages, hkv, d = s["page"], s["npages"], s["hkv"], s["d"]
    slots = s["slots"].long()
    pages, place = torch.unique(slots // page, return_inverse=True)
    x = x.float().transpose(0, 1)
    amax = torch.zeros(hkv, pages.numel(), device="cuda")
    amax.index_reduce_(1, place, x.abs().amax(-1), "amax")
    first = torch.full((pages.numel(),), page, device="cuda", dtype=torch.int64)
    first.scatter_reduce_(0, place, slots % page, "amin")
    mantissa, exponent = torch.frexp(amax)
    need = (exponent - 9 + (mantissa > 0.875)).clamp(MIN_EXP, MAX_EXP)
    need = torch.exp2(torch.where(amax > 0, need, MIN_EXP).float())
    old = scales[:, pages]
    kept = (first > 0)[None]
    new = torch.where(kept & (amax <= E4M3_MAX * old), old, need)
    grown = kept & (new != old)
    view = codes.view(hkv, npages, page, d)
    held = view[:, pages]
    moved = (held.view(torch.float8_e4m3fn).float() * (old / new)[:, :, None, None]).to(torch.float8_e4m3fn)
    row = torch.arange(page, device="cuda")[None, :] < first[:, None]
    view[:, pages] = torch.where((grown[:, :, None] & row[None])[..., None], moved.view(torch.uint8), held)
    codes[:, slots] = (x / new[:, place, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[:, pages] = new


def _plain_write(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    heads = s["rows"].view(-1, hq + 2 * hkv, d)
    _plain_write_side(s, s["q_k"], s["s_k"], heads[:, hq:hq + hkv])
    _plain_write_side(s, s["q_v"], s["s_v"], heads[:, hq + hkv:])
    return _cache_outputs(s)


def _cache_outputs(s):
    return {"k": s["q_k"].view(torch.float8_e4m3fn), "v": s["q_v"].view(torch.float8_e4m3fn), "s_k": s["s_k"],
            "s_v": s["s_v"]}


def _plain_attend(s):
    nseq, page, hq, hkv, d, maxl, maxq = (s[k] for k in ("nseq", "page", "hq", "hkv", "d", "max_len", "max_q"))
    group = hq // hkv
    lens, offsets = s["seq_lens"].long(), s["q_offsets"].long()
    count = offsets[1:] - offsets[:-1]
    pos = torch.arange(maxl, device="cuda")
    pages = s["bt"][:, pos // page].long().clamp(min=0)
    rows = pages * page + pos % page

    def gathered(codes, scales):  # [nseq][hkv][maxl][d]
        v = codes[:, rows].view(torch.float8_e4m3fn).float()
        return v.mul_(scales[:, pages, None]).transpose(0, 1)

    tok = torch.arange(maxq, device="cuda")
    q = s["q"][(offsets[:-1, None] + tok).clamp(max=s["tokens"] - 1)].float()
    q = q.view(nseq, maxq, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(nseq, hkv, maxq * group, d)
    score = torch.matmul(q, gathered(s["q_k"], s["s_k"]).transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    seen = (pos < lens[:, None])[:, None]
    if s["causal"]:
        seen = seen & (pos <= (lens - count)[:, None, None] + tok[:, None])
    score = score.view(nseq, hkv, maxq, group, maxl).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    score = score.view(nseq, hkv, maxq * group, maxl)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    norm = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, gathered(s["q_v"], s["s_v"])) / torch.where(norm > 0, norm, 1.0)
    lse = (top + torch.log(norm)).squeeze(-1)
    # back to one row a token
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(offsets[1:].contiguous(), t, right=True)
    j = t - offsets[seq]
    out = out.view(nseq, hkv, maxq, group, d).permute(0, 2, 1, 3, 4).reshape(nseq, maxq, hq, d)
    lse = lse.view(nseq, hkv, maxq, group).permute(0, 2, 1, 3).reshape(nseq, maxq, hq)
    return {"out": out[seq, j].to(s["dtype"]), "lse": lse[seq, j]}


# ---- one pass ---------------------------------------------------------------------------------------------------

def _own_tables(s):
    import w4a16_dequant_gemm_b200 as w4
    w4.page_tables(s["cached"].data_ptr(), s["fresh"].data_ptr(), s["nseq"], s["page"], s["npages"],
                   s["free"].data_ptr(), s["free"].numel(), s["taken"].data_ptr(), s["taken_out"].data_ptr(),
                   s["bt"].data_ptr(), s["bt"].stride(0), s["seq_lens"].data_ptr(), s["q_offsets"].data_ptr(),
                   s["slots"].data_ptr(), s["positions"].data_ptr(), s["slots"].numel(),
                   torch.cuda.current_stream().cuda_stream)
    return {"bt": s["bt"], "seq_lens": s["seq_lens"], "q_offsets": s["q_offsets"], "slots": s["slots"],
            "positions": s["positions"], "taken": s["taken_out"]}


def _own_cache(s):
    import w4a16_dequant_gemm_b200 as w4
    return w4, w4.DeviceKVB8(s["hkv"], s["d"], s["page"], s["npages"], s["q_k"].data_ptr(), s["s_k"].data_ptr(),
                             s["q_v"].data_ptr(), s["s_v"].data_ptr())


def _own_write(s):
    w4, cache = _own_cache(s)
    rows, hq, hkv, d = s["rows"], s["hq"], s["hkv"], s["d"]
    w4.kv_write_b8(cache, s["slots"].data_ptr(), s["slots"].numel(), rows[:, hq * d:].data_ptr(),
                   rows[:, (hq + hkv) * d:].data_ptr(), rows.stride(0), rows.stride(0),
                   w4.DTYPE_BF16 if s["dtype"] == torch.bfloat16 else w4.DTYPE_F16,
                   stream=torch.cuda.current_stream().cuda_stream)
    return _cache_outputs(s)


def _own_attend(s):
    w4, cache = _own_cache(s)
    w4.attention_b8_paged(cache, s["bt"].data_ptr(), s["bt"].stride(0), s["seq_lens"].data_ptr(),
                          s["q_offsets"].data_ptr(), s["nseq"], s["max_q"], s["max_len"], s["q"].data_ptr(),
                          s["q"].stride(0), s["hq"], w4.DTYPE_BF16 if s["dtype"] == torch.bfloat16 else w4.DTYPE_F16,
                          s["out"].data_ptr(), s["out"].stride(0), lse=s["lse"].data_ptr(), causal=s["causal"],
                          stream=torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"], "lse": s["lse"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "write": _own_write, "attend": _own_attend}[op](state)
    return {"tables": _plain_tables, "write": _plain_write, "attend": _plain_attend}[op](state)


# ---- the definitions, in 64 bits --------------------------------------------------------------------------------

def _nearest_e4m3(v):
    """The E4M3 value nearest to v (64 bits, |v| <= 448), ties to the even code."""
    size = v.abs()
    _, e = torch.frexp(torch.where(size > 0, size, 1.0))
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def _exact_write_side(s, slots, codes, scales, x):
    page, value, scale = s["page"], codes.view(torch.float8_e4m3fn).double(), scales.double()
    at, n = 0, len(slots)
    while at < n:  # runs of tokens of one page
        end = at + 1
        while end < n and slots[end] // page == slots[at] // page:
            end += 1
        p, row = slots[at] // page, slots[at] % page
        part = x[at:end].double().transpose(0, 1)
        top = part.abs().amax((1, 2))
        need = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)))
        need = torch.where(need * (E4M3_MAX / 2) >= top, need / 2, need)
        need = torch.where(need * E4M3_MAX < top, need * 2, need).clamp(2.0 ** MIN_EXP, 2.0 ** MAX_EXP)
        if row:
            old = scale[:, p]
            keep = top <= E4M3_MAX * old
            new = torch.where(keep, old, need)
            held = value[:, p * page:p * page + row]
            value[:, p * page:p * page + row] = torch.where(keep[:, None, None], held,
                                                            _nearest_e4m3(held * (old / new)[:, None, None]))
            need = new
        scale[:, p] = need
        value[:, slots[at]:slots[at] + end - at] = _nearest_e4m3(part / need[:, None, None])
        at = end
    return value, scale


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    if case["op"] == "write":
        slots, heads = s["slots"].tolist(), s["rows"].view(-1, hq + 2 * hkv, d)
        k, s_k = _exact_write_side(s, slots, s["q_k"], s["s_k"], heads[:, hq:hq + hkv])
        v, s_v = _exact_write_side(s, slots, s["q_v"], s["s_v"], heads[:, hq + hkv:])
        return {"k": k, "v": v, "s_k": s_k, "s_v": s_v}
    _, fresh, total = _requests(case)
    out = torch.zeros(s["tokens"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], hq), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, length) in enumerate(zip(fresh, total)):
        pages = s["bt"][i, : _pages(length, page)].long()
        for h in range(hkv):
            def side(codes, scales):
                v = codes[h].view(-1, page, d)[pages].view(torch.float8_e4m3fn).double()
                return (v * scales[h][pages].double()[:, None, None]).view(-1, d)[:length]

            k, v = side(s["q_k"], s["s_k"]), side(s["q_v"], s["s_v"])
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            q = s["q"][at:at + n, heads].double()
            a = torch.einsum("tgd,ld->gtl", q, k) / math.sqrt(d)
            if case["causal"]:
                a = a.masked_fill(torch.arange(length, device="cuda") > length - n
                                  + torch.arange(n, device="cuda")[:, None], -math.inf)
            norm = torch.logsumexp(a, -1)
            lse[at:at + n, heads] = norm.T
            out[at:at + n, heads] = torch.einsum("gtl,ld->tgd", torch.exp(a - norm[..., None]), v)
        at += n
    return {"out": out, "lse": lse}
