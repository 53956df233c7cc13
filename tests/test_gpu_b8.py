"""GPU tests of the paged 8-bit cache operators (w4b_page_tables, w4b_kv_write_b8, w4b_attn_b8_paged) against plain
implementations of their definitions in 64 bits. None has a counterpart in the reference.

Tolerances. Tables and codes are exact. Attention: the kernel rounds each weight to FP16 (half a step: 2^-11 relative,
2^-25 absolute of the largest weight below the normal range) and the output to its type (2^-11 FP16, 2^-8 BF16); scores
are FP32 sums of exact products, whose error we bound by 2^-19 of the sum of magnitudes (128 terms, truncating adders)
and which moves a weight by that much relatively. So, with A = sum p |v|, S the largest sum of |q k| scale over a row
and n positions:
  |out - ref| <= A (2^-11 + 2 * 2^-19 S) + |ref| half_step + 2^-24 n max|v|
  |lse - ref| <= 2^-19 S + 2^-20 (1 + |ref|)"""
import math

import numpy as np
import pytest
import torch

import w4a16_dequant_gemm_b200 as w4

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
CODE = {F16: w4.DTYPE_F16, BF16: w4.DTYPE_BF16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


def offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(int).tolist()


# ---- block tables ------------------------------------------------------------------------------------------------

def plain_tables(cached, fresh, page, npages, free, taken, bt, max_tokens):
    bt, status = bt.copy(), 0
    slots, positions = [-1] * max_tokens, [0] * max_tokens
    lens, at, token = [], taken, 0
    over = False
    for i, (c, f) in enumerate(zip(cached, fresh)):
        fits = c >= 0 and f >= 0 and c + f <= min(bt.shape[1], npages) * page
        if not fits:
            over = True
            lens.append(0)
            token += max(f, 0)
            continue
        first, last = -(-c // page), -(-(c + f) // page)
        for col in range(first, last):
            p = free[at] if at < len(free) else -1
            bt[i, col] = p if 0 <= p < npages else -1
            at += 1
        for j in range(f):
            if token < max_tokens:
                pos = c + j
                positions[token] = pos
                p = bt[i, pos // page]
                slots[token] = p * page + pos % page if 0 <= p < npages else -1
            token += 1
        lens.append(c + f)
    if at > len(free):
        status = 601
    elif over or token > max_tokens:
        status = 602
    return bt, lens, offsets([max(f, 0) for f in fresh]), slots, positions, min(at, max(len(free), taken)), status


def run_tables(cached, fresh, page, npages, free, taken, bt, max_tokens, skew=0, in_place=False):
    n = len(cached)
    d = dict(cached=ints(cached), fresh=ints(fresh), free=ints(free), taken=ints([taken]), bt=ints(bt))
    lens = d["cached"] if in_place else ints([-7] * n)
    out = d["taken"] if in_place else ints([-7])
    off = ints([-7] * (n + 1))
    maps = torch.full((2, max_tokens + skew + 4), -7, dtype=torch.int32, device="cuda")
    slots, positions = maps[0, skew:], maps[1, skew:]
    w4.page_tables(d["cached"].data_ptr(), d["fresh"].data_ptr(), n, page, npages, d["free"].data_ptr() if free else None,
                   len(free), d["taken"].data_ptr(), out.data_ptr(), d["bt"].data_ptr(), d["bt"].stride(0), lens.data_ptr(),
                   off.data_ptr(), slots.data_ptr(), positions.data_ptr(), max_tokens, stream())
    status = w4.device_status()
    assert (maps[:, max_tokens + skew:] == -7).all() and (maps[:, :skew] == -7).all()
    return (d["bt"].cpu().numpy(), lens.tolist(), off.tolist(), slots[:max_tokens].tolist(), positions[:max_tokens].tolist(),
            int(out[0]), status)


def same_tables(args, **kw):
    want, got = plain_tables(*args), run_tables(*args, **kw)
    assert np.array_equal(want[0], got[0])
    assert list(want[1:6]) == list(got[1:6])
    assert want[6] == got[6]


def table_case(rng, n, page, cached_hi, fresh_hi, spare=3):
    cached = rng.integers(0, cached_hi + 1, n).tolist()
    fresh = rng.integers(0, fresh_hi + 1, n).tolist()
    total = [a + b for a, b in zip(cached, fresh)]
    cols = max(-(-t // page) for t in total) + 2
    held = sum(-(-c // page) for c in cached)
    need = sum(-(-t // page) for t in total) - held
    npages = held + need + spare + 1
    order = rng.permutation(npages).tolist()
    bt, k = np.full((n, cols), -3, dtype=np.int32), 0
    for i, c in enumerate(cached):
        m = -(-c // page)
        bt[i, :m] = order[k:k + m]
        k += m
    return cached, fresh, page, npages, order[held:], bt, need


@pytest.mark.parametrize("n,page,cached_hi,fresh_hi", [(1, 16, 0, 1), (1, 16, 40, 100), (7, 1, 5, 4), (64, 16, 300, 1),
                                                       (33, 48, 100, 200), (1025, 16, 50, 3), (2500, 32, 20, 9), (5, 64, 9, 9000)])
def test_tables(n, page, cached_hi, fresh_hi):
    rng = np.random.default_rng(n * 1000 + page)
    cached, fresh, page, npages, free, bt, need = table_case(rng, n, page, cached_hi, fresh_hi)
    tokens = sum(fresh)
    same_tables((cached, fresh, page, npages, free, 0, bt, tokens + 5))
    same_tables((cached, fresh, page, npages, [9999] * 2 + free, 2, bt, tokens), skew=1)
    same_tables((cached, fresh, page, npages, free, 0, bt, tokens + 3), in_place=True)


def test_tables_refused_steps():
    rng = np.random.default_rng(5)
    cached, fresh, page, npages, free, bt, need = table_case(rng, 40, 16, 60, 50)
    tokens = sum(fresh)
    same_tables((cached, fresh, page, npages, free[:need - 4], 0, bt, tokens))      # pages run out
    same_tables((cached, fresh, page, npages, [], 0, bt, tokens))
    same_tables((cached, fresh, page, npages, free[:5], 9, bt, tokens))             # taken behind the list's end
    same_tables((cached, fresh, page, npages, free, 0, bt, tokens - 7))             # more tokens than the maps hold
    same_tables((cached, fresh, page, npages, [npages, -1] + free, 0, bt, tokens))  # pages the pool does not have
    same_tables((cached, fresh, page, npages, free, 0, bt, 0))
    long = list(fresh)
    long[3], long[7] = 10 ** 9, -2                                                  # too long, negative
    same_tables((cached, long[:3] + [page * (bt.shape[1] + 1)] + fresh[4:], page, npages, free, 0, bt, 20))
    bad = list(cached)
    bad[0] = -1
    same_tables((bad, fresh, page, npages, free, 0, bt, tokens))
    got = run_tables(cached, long, page, npages, free, 0, bt, 64)
    assert got[6] == 602 and got[1][3] == 0 and got[1][7] == 0 and got[1][0] == cached[0] + fresh[0]


# ---- the write ---------------------------------------------------------------------------------------------------

def to_e4m3(v):
    """Nearest E4M3 value, ties to even, of |v| <= 448 (larger ones saturate); 64 bits."""
    v = np.clip(np.asarray(v, dtype=np.float64), -448.0, 448.0)
    _, e = np.frexp(np.where(v == 0, 1.0, np.abs(v)))
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(v / step) * step


def values(codes):
    return codes.view(torch.float8_e4m3fn).float().cpu().numpy().astype(np.float64)


def plain_write(val, scale, slots, x, page):
    """val [rows][D] and scale [npages] of one head, x [T][D]: in place."""
    status, T, t = 0, len(slots), 0
    if not np.isfinite(x).all():
        status = 501
        x = np.where(np.isfinite(x).all(1, keepdims=True), x, 0.0)
    while t < T:
        s = slots[t]
        if s < 0:
            t += 1
            continue
        n = 1
        while t + n < T and slots[t + n] == s + n and (s + n) % page:
            n += 1
        p, row = s // page, s % page
        amax = np.abs(x[t:t + n]).max()
        need = -60.0
        if amax > 0:
            need = math.ceil(math.log2(amax / 448.0)) - 1
            while amax > 448.0 * 2.0 ** need:
                need += 1
            if need > 60:
                status = 501
            need = min(max(need, -60), 60)
        new = np.float32(2.0 ** need)
        if row > 0:
            old = scale[p]
            if amax <= 448.0 * old:
                new = old
            else:
                r = np.float32(old / new)
                val[p * page:p * page + row] = to_e4m3(np.float32(val[p * page:p * page + row]) * r)
        scale[p] = new
        with np.errstate(over="ignore"):
            val[s:s + n] = to_e4m3(np.float32(x[t:t + n]) / new)
        t += n
    return status


def run_write(H, D, page, npages, slots, k, v, seed=0, scales=None, stride=None, expect=0, hold=None):
    """k, v: [T][H][D] CPU tensors. Compares codes, scales and status with plain_write."""
    gen = torch.Generator().manual_seed(seed)
    codes = (torch.randn(2, H, npages * page, D, generator=gen) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    sc = torch.exp2(torch.randint(-8, -3, (2, H, npages), generator=gen).float()) if scales is None else scales.clone()
    dc, ds = codes.view(torch.uint8).cuda(), sc.cuda()
    T, dtype = len(slots), k.dtype
    width = stride or H * D
    rows = torch.full((T, 2 * width), 777.0, dtype=dtype)
    rows[:, :H * D] = k.reshape(T, -1)
    rows[:, width:width + H * D] = v.reshape(T, -1)
    rows = rows.cuda()
    sl = ints(slots)
    p = w4.DeviceKVB8(H, D, page, npages, dc[0].data_ptr(), ds[0].data_ptr(), dc[1].data_ptr(), ds[1].data_ptr())
    w4.kv_write_b8(p, sl.data_ptr(), T, rows.data_ptr(), rows.data_ptr() + 2 * width, rows.stride(0), rows.stride(0), CODE[dtype], stream())
    got_status = w4.device_status()
    want_status = 0
    for side, x in enumerate((k, v)):
        val, scale = values(codes[side]).copy(), sc[side].numpy().copy()
        for h in range(H):
            want_status = plain_write(val[h], scale[h], slots, x[:, h].double().numpy(), page) or want_status
        assert np.array_equal(scale, ds[side].cpu().numpy())
        assert np.array_equal(val, values(dc[side]))
    assert got_status == (expect or want_status)


def new_rows(T, H, D, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(2, T, H, D, generator=gen) * torch.exp2(spread * torch.randn(2, T, H, 1, generator=gen))
    return x.to(dtype)


def runs(spec):
    """[(first slot, count)] -> slot list"""
    return [s + j for s, n in spec for j in range(n)]


WRITES = [
    (1, 64, 16, [(0, 1)]),                                            # one token, a fresh page
    (2, 128, 16, [(5, 1), (40, 1), (31, 1)]),                         # decode: pages continued
    (3, 64, 48, [(50, 46), (144, 48), (0, 7)]),                       # runs that end inside pages
    (2, 128, 64, [(70, 58), (192, 64), (256, 30), (3, 1), (320, 0)]),  # a prompt over several pages
    (1, 128, 256, [(3, 253), (512, 130)]),                            # pages larger than a CTA holds in registers
    (1, 64, 4096, [(100, 3000)]),
    (8, 128, 16, [(16 * i + (i * 7) % 16, 1) for i in range(90)]),    # a wide decode step
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(WRITES)))
def test_write(case, dtype):
    H, D, page, spec = WRITES[case]
    slots = runs(spec)
    npages = max(max(slots) // page + 2, 4)
    x = new_rows(len(slots), H, D, dtype, case)
    run_write(H, D, page, npages, slots, x[0], x[1], seed=case)
    padded = [-1] + [s for s in slots] + [-1, -1]                      # a padded batch
    z = torch.zeros(1, H, D, dtype=dtype)
    run_write(H, D, page, npages, padded, torch.cat([z, x[0], z, z]), torch.cat([z, x[1], z, z]), seed=case,
              stride=H * D + 8)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_write_values(dtype):
    """Zeros, tiny and large values, the border of a power of two, scales that are no powers of two, infinities and NaN."""
    H, D, page, npages = 1, 64, 16, 8
    slots = [0, 1, 2, 21, 35, 36, 48, 70, 80]
    x = new_rows(len(slots), H, D, dtype, 3, spread=0.5)
    x[0, 0:3] = 0
    x[0, 3] = 1e-7
    x[0, 4, 0, 5], x[0, 4, 0, 6] = 448.0, -0.0
    x[0, 5] = 0.5
    x[1, 0, 0, :4] = torch.tensor([448.0, -449.0, 60000.0, 2.0 ** -9])
    x[1, 6] = 6e-8
    run_write(H, D, page, npages, slots, x[0], x[1], seed=9)
    odd = torch.full((2, H, npages), 0.0123)
    run_write(H, D, page, npages, slots, x[0], x[1], seed=9, scales=odd)
    x[0, 4, 0, 7], x[1, 8, 0, 0], x[1, 2, 0, 63] = math.inf, math.nan, -math.inf
    run_write(H, D, page, npages, slots, x[0], x[1], seed=9)


def test_write_saturates_beyond_the_scales():
    x = torch.full((2, 2, 1, 64), 3e38).to(BF16)
    run_write(1, 64, 16, 2, [0, 17], x[0], x[1])


def test_write_bad_slots():
    """Slots outside the pool and tokens of a page that are out of order are reported and not written."""
    H, D, page, npages = 2, 64, 16, 4
    x = new_rows(6, H, D, F16, 4)
    keep = [0, 1, 3]
    codes = []
    for slots, use in (([3, 4, 64, 17, 10 ** 9, -1], slice(None)), ([3, 4, 17], keep)):
        q = torch.zeros(2, H, npages * page, D, dtype=torch.uint8, device="cuda")
        s = torch.full((2, H, npages), 2.0 ** -7, device="cuda")
        k, v = x[0][use].contiguous().cuda(), x[1][use].contiguous().cuda()
        sl = ints(slots)
        p = w4.DeviceKVB8(H, D, page, npages, q[0].data_ptr(), s[0].data_ptr(), q[1].data_ptr(), s[1].data_ptr())
        w4.kv_write_b8(p, sl.data_ptr(), len(slots), k.data_ptr(), v.data_ptr(), H * D, H * D, w4.DTYPE_F16, stream())
        codes.append((w4.device_status(), q.cpu(), s.cpu()))
    assert codes[0][0] == 603 and codes[1][0] == 0
    assert torch.equal(codes[0][1], codes[1][1]) and torch.equal(codes[0][2], codes[1][2])
    q = torch.zeros(2, H, npages * page, D, dtype=torch.uint8, device="cuda")
    sl = ints([3, 5, 4, 3, 18, 17])   # a gap, a step back, the same slot twice, descending
    k, v = x[0].contiguous().cuda(), x[1].contiguous().cuda()
    p = w4.DeviceKVB8(H, D, page, npages, q[0].data_ptr(), s[0].data_ptr(), q[1].data_ptr(), s[1].data_ptr())
    w4.kv_write_b8(p, sl.data_ptr(), 6, k.data_ptr(), v.data_ptr(), H * D, H * D, w4.DTYPE_F16, stream())
    assert w4.device_status() == 603
    written = (q.view(2, H, npages * page, D) != 0).any(-1).any(1).any(0).nonzero().flatten().tolist()
    assert written == [3, 18]


# ---- attention ---------------------------------------------------------------------------------------------------

class Problem:
    def __init__(self, lens, nq, hkv, group, d, page, dtype, causal, seed=0, spare=3, scale=None, scale_exp=(-7, -4), q_amp=1.5):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.nq, self.hkv, self.group, self.d, self.page = lens, nq, hkv, group, d, page
        self.dtype, self.causal, self.scale = dtype, causal, d ** -0.5 if scale is None else scale
        n = len(lens)
        need = [-(-x // page) for x in lens]
        self.npages = sum(need) + spare
        self.max_len = max(lens)
        order = torch.randperm(self.npages, generator=gen, device="cuda").tolist()
        self.stride = max(max(need), 1) + 2
        bt, k = [], 0
        for m in need:
            bt.append(order[k:k + m] + [-1] * (self.stride - m))
            k += m
        self.bt = ints(bt)
        c = torch.randn(2, hkv, self.npages * page, d, generator=gen, device="cuda") * 64
        self.codes = c.clamp(-448, 448).to(torch.float8_e4m3fn)
        self.scales = torch.exp2(torch.randint(scale_exp[0], scale_exp[1] + 1, (2, hkv, self.npages), generator=gen, device="cuda").float())
        self.offsets = offsets(nq)
        self.tokens = self.offsets[-1]
        self.q = (q_amp * torch.randn(self.tokens + 2, hkv * group, d, generator=gen, device="cuda")).to(dtype)
        self.poison = True

    def cache(self):
        codes = self.codes.view(torch.uint8)
        if self.poison:   # what lies behind a sequence's end is not read: NaN codes there, NaN in unused pages
            codes = codes.clone()
            used = torch.zeros(self.npages, dtype=torch.bool)
            for i, L in enumerate(self.lens):
                pages = self.bt[i, : -(-L // self.page)].tolist()
                used[pages] = True
                if L % self.page:
                    r = pages[-1] * self.page
                    codes[:, :, r + L % self.page: r + self.page] = 0x7F
            codes.view(2, self.hkv, self.npages, self.page, self.d)[:, :, ~used] = 0xFF
        return codes

    def reference(self, missing=()):
        """(out, lse, bound on out, bound on lse) in 64 bits; `missing`: (sequence, column) block-table entries left out."""
        T, hq = self.tokens, self.hkv * self.group
        out = torch.zeros(T, hq, self.d, dtype=torch.float64)
        lse = torch.full((T, hq), -math.inf, dtype=torch.float64)
        b_out, b_lse = torch.zeros_like(out), torch.zeros_like(lse)
        half = 2.0 ** -11 if self.dtype == F16 else 2.0 ** -8
        val = self.codes.double().view(2, self.hkv, self.npages, self.page, self.d) * self.scales.double()[..., None, None]
        val, q_all = val.cpu(), self.q.double().cpu()
        for i, (L, n) in enumerate(zip(self.lens, self.nq)):
            if L == 0 or n == 0:
                continue
            pages = self.bt[i, : -(-L // self.page)].tolist()
            kv = val[:, :, pages].reshape(2, self.hkv, -1, self.d)[:, :, :L]
            q = q_all[self.offsets[i]:self.offsets[i + 1]].view(n, self.hkv, self.group, self.d)
            a = torch.einsum("nhgd,hld->nhgl", q, kv[0]) * self.scale
            mag = torch.einsum("nhgd,hld->nhgl", q.abs(), kv[0].abs()) * self.scale
            pos = torch.arange(L)
            seen = pos[None] <= L - n + torch.arange(n)[:, None] if self.causal else torch.ones(n, L, dtype=torch.bool)
            for s, col in missing:
                if s == i:
                    seen = seen & ~((pos // self.page) == col)
            a = a.masked_fill(~seen[:, None, None], -math.inf)
            big = mag.masked_fill(~seen[:, None, None], 0).amax(-1)
            norm = torch.logsumexp(a, -1)
            p = torch.exp(a - torch.where(norm > -math.inf, norm, 0.0)[..., None])
            o = torch.einsum("nhgl,hld->nhgd", p, kv[1])
            mass = torch.einsum("nhgl,hld->nhgd", p, kv[1].abs())
            rows = slice(self.offsets[i], self.offsets[i + 1])
            out[rows], lse[rows] = o.reshape(n, hq, self.d), norm.reshape(n, hq)
            # the largest weight is at least the largest p * scale of V: relative to it the absolute rounding counts
            slack = 2.0 ** -24 * L * (p.amax(-1)[..., None] * kv[1].abs().amax(1)[None, :, None])
            b_out[rows] = (mass * (2.0 ** -11 + 2 * 2.0 ** -19 * big[..., None]) + o.abs() * half * 1.01 + slack + 2.0 ** -25).reshape(n, hq, self.d)
            b_lse[rows] = (2.0 ** -19 * big + 2.0 ** -20 * (1 + norm.abs())).reshape(n, hq)
        return out, lse, b_out, b_lse

    def run(self, out=None, lse=None, q=None, bt=None, codes=None, workspace=None, offsets=True, max_q=None):
        hq = self.hkv * self.group
        codes = self.cache() if codes is None else codes
        q = self.q if q is None else q
        out = torch.full((self.tokens + 2, hq, self.d), 9.0, dtype=self.dtype, device="cuda") if out is None else out
        lse = torch.full((self.tokens + 2, hq), 9.0, device="cuda") if lse is None else lse
        p = w4.DeviceKVB8(self.hkv, self.d, self.page, self.npages, codes[0].data_ptr(), self.scales[0].data_ptr(),
                          codes[1].data_ptr(), self.scales[1].data_ptr())
        bt = self.bt if bt is None else bt
        dl, do = ints(self.lens), ints(self.offsets)
        w4.attention_b8_paged(p, bt.data_ptr(), bt.stride(0), dl.data_ptr(), do.data_ptr() if offsets else None, len(self.lens),
                              max(self.nq + [1]) if max_q is None else max_q, self.max_len, q.data_ptr(), q.stride(0), hq,
                              CODE[self.dtype], out.data_ptr(), out.stride(0), lse.data_ptr(), self.scale, self.causal,
                              None if workspace is None else workspace.data_ptr(),
                              0 if workspace is None else workspace.numel(), stream())
        self.alive = (codes, dl, do, bt, q)
        return out, lse

    def check(self, out, lse, missing=()):
        ref, ref_lse, b_out, b_lse = self.reference(missing)
        T = self.tokens
        assert (out[T:] == 9).all() and (lse[T:] == 9).all()           # rows behind the last sequence
        o, s = out[:T].double().cpu(), lse[:T].double().cpu()
        empty = ref_lse == -math.inf
        assert (s[empty] == -math.inf).all() and (o[empty] == 0).all()
        off = (o - ref).abs() / b_out.clamp(min=1e-300)
        assert (off[~empty] <= 1).all(), (off[~empty].max(), (off > 1).nonzero()[:3])
        off = (s - ref_lse).abs()[~empty] / b_lse[~empty]
        assert (off <= 1).all(), off.max()


DECODES = [
    # lens, hkv, group, d, page
    ([1], 1, 1, 64, 16),
    ([17, 1, 16, 15], 2, 4, 128, 16),
    ([777], 8, 4, 128, 16),
    ([0, 5, 0, 64, 63, 65], 2, 8, 64, 32),
    ([300, 2000, 9, 1, 511], 4, 3, 128, 48),
    ([5000, 130], 1, 16, 128, 64),
    ([1000] * 3, 2, 5, 64, 128),
    ([4097, 4095], 2, 7, 128, 4096),
    ([33, 900], 1, 40, 64, 16),
    ([40000], 1, 2, 128, 256),
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_attention_single_tokens(case, dtype):
    lens, hkv, group, d, page = DECODES[case]
    p = Problem(lens, [1] * len(lens), hkv, group, d, page, dtype, True, seed=case)
    out, lse = p.run()
    p.check(out, lse)
    again = p.run(offsets=False)                                       # one token each, without offsets
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    assert w4.device_status() == 0


TOKENS = [
    # lens, query tokens, hkv, group, d, page
    ([3], [3], 1, 1, 64, 16),
    ([40, 100, 7, 0], [4, 5, 7, 0], 2, 3, 128, 16),
    ([2], [5], 1, 4, 64, 16),                     # causal: more tokens than positions, the first see nothing
    ([200, 0, 64, 65], [17, 3, 0, 33], 2, 2, 128, 32),
    ([700, 129, 128], [130, 129, 1], 1, 4, 128, 64),
    ([1500, 333], [60, 224], 4, 1, 64, 48),
    ([600, 80, 31], [257, 1, 2], 2, 8, 128, 16),
    ([512, 127], [300, 127], 2, 5, 64, 128),
]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(TOKENS)))
def test_attention_several_tokens(case, dtype, causal):
    lens, nq, hkv, group, d, page = TOKENS[case]
    p = Problem(lens, nq, hkv, group, d, page, dtype, causal, seed=100 + case)
    out, lse = p.run()
    p.check(out, lse)
    assert w4.device_status() == 0


@pytest.mark.parametrize("many", [1, 17], ids=["single", "rows"])
def test_attention_thousands_of_sequences(many):
    """5200 short sequences: every work range covers dozens, some of them without tokens or positions."""
    n = 5200
    rng = np.random.default_rng(7)
    nq = (rng.integers(0, 8, n) > 0).astype(int) * many
    p = Problem(rng.integers(0, 30, n).tolist(), nq.tolist(), 1, 2, 64, 16, F16, False, seed=30)
    p.check(*p.run())
    assert w4.device_status() == 0


def test_attention_mixed_batch():
    """Single tokens, drafts and prompt chunks side by side: both kernels in one call, sequences of one between the other's."""
    rng = np.random.default_rng(8)
    nq = [int(x) for x in rng.choice([1, 1, 1, 2, 5, 60, 300], 70)]
    lens = [int(x) + q for x, q in zip(rng.integers(0, 700, 70), nq)]
    p = Problem(lens, nq, 2, 4, 128, 32, BF16, True, seed=31)
    p.check(*p.run())
    assert w4.device_status() == 0


@pytest.mark.parametrize("nq", [1, 3, 70])
def test_attention_scales_far_apart(nq):
    """Pages whose scales differ by 2^50: the large ones decide the values, all decide the weights."""
    p = Problem([400, 64], [nq, nq], 2, 2, 64, 16, BF16, True, seed=3, scale_exp=(-14, -4), q_amp=1.0)
    gen = torch.Generator(device="cuda").manual_seed(4)
    p.scales[1] = torch.exp2(torch.randint(-45, 6, p.scales[1].shape, generator=gen, device="cuda").float())
    p.check(*p.run())


@pytest.mark.parametrize("nq", [1, 40])
def test_attention_scales_that_are_no_powers_of_two(nq):
    p = Problem([257, 30], [nq, nq], 2, 3, 128, 32, F16, True, seed=5)
    p.scales *= 1.2345
    p.check(*p.run())


@pytest.mark.parametrize("nq", [1, 33])
def test_attention_peaked_and_large(nq):
    """Scores of hundreds: one position carries the row, the reference point moves block by block."""
    p = Problem([900, 100], [nq, nq], 1, 4, 128, 16, BF16, True, seed=6, q_amp=60.0)
    p.check(*p.run())
    p = Problem([300], [nq], 1, 2, 64, 16, BF16, False, seed=7, q_amp=1e30, scale=1e-30)   # far beyond FP16's range
    p.check(*p.run())
    p = Problem([300], [nq], 1, 2, 64, 16, BF16, False, seed=7, q_amp=1e-25, scale=1e25)
    p.check(*p.run())


@pytest.mark.parametrize("nq", [1, 20])
def test_attention_missing_pages(nq):
    p = Problem([200, 50], [nq, nq], 2, 2, 128, 16, F16, False, seed=8)
    bt = p.bt.clone()
    bt[0, 3], bt[0, 12], bt[1, 0], bt[1, 1], bt[1, 2], bt[1, 3] = -1, p.npages, -5, 2 ** 31 - 1, -1, -1
    codes = p.cache()
    out, lse = p.run(bt=bt, codes=codes)
    assert w4.device_status() == 604
    p.check(out, lse, missing=[(0, 3), (0, 12), (1, 0), (1, 1), (1, 2), (1, 3)])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nq", [[2, 3], [40, 90]], ids=["few", "many"])
def test_attention_nan_stays_in_its_rows(nq, dtype):
    p = Problem([200, 160], nq, 2, 2, 64, 16, dtype, True, seed=9)
    clean, clean_lse = p.run()
    q = p.q.clone()
    q[1, 2, 5], q[3, 0, 0] = math.nan, math.inf
    out, lse = p.run(q=q)
    hit = torch.zeros(p.tokens + 2, 4, dtype=torch.bool, device="cuda")
    hit[1, 2] = hit[3, 0] = True
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])


@pytest.mark.parametrize("nq", [1, 50])
def test_attention_strides(nq):
    """Queries out of a fused projection row, outputs into a wider row."""
    p = Problem([300, 77], [nq, nq], 2, 3, 128, 32, BF16, True, seed=10)
    want, want_lse = p.run()
    wide = torch.zeros(p.tokens + 2, 12, 128, dtype=BF16, device="cuda")
    wide[:, 3:9] = p.q
    out = torch.full((p.tokens + 2, 10, 128), 9.0, dtype=BF16, device="cuda")
    got, lse = p.run(q=wide[:, 3:9], out=out[:, 1:7])
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    assert (out[:, 0] == 9).all() and (out[:, 7:] == 9).all()


@pytest.mark.parametrize("nq", [1, 30])
def test_attention_offsets_beyond_32_bits(nq):
    """A pool of more than 2^32 bytes a side: its last pages."""
    hkv, d, page, npages = 4, 128, 64, 160_000
    codes = torch.zeros(2, hkv, npages * page, d, dtype=torch.uint8, device="cuda")
    p = Problem([250], [nq], hkv, 2, d, page, F16, True, seed=11)
    scales = torch.ones(2, hkv, npages, device="cuda")
    small = p.codes.view(torch.uint8).view(2, hkv, p.npages, page, d)
    bt = torch.full_like(p.bt, -1)
    for j, pg in enumerate(p.bt[0, :4].tolist()):
        codes.view(2, hkv, npages, page, d)[:, :, npages - 1 - j] = small[:, :, pg]
        scales[:, :, npages - 1 - j] = p.scales[:, :, pg]
        bt[0, j] = npages - 1 - j
    want = p.reference()
    p.npages, p.scales, p.poison = npages, scales, False
    out, lse = p.run(bt=bt, codes=codes)
    T = p.tokens
    assert ((out[:T].double().cpu() - want[0]).abs() <= want[2]).all()
    assert ((lse[:T].double().cpu() - want[1]).abs() <= want[3]).all()


@pytest.mark.parametrize("nq", [1, 40])
def test_attention_same_bits_again_and_in_company(nq):
    p = Problem([2500, 100, 40], [nq] * 3, 2, 4, 128, 16, F16, True, seed=12)
    out, lse = p.run()
    for _ in range(3):
        o, s = p.run()
        assert torch.equal(o, out) and torch.equal(s, lse)
    codes = p.cache()
    pages = p.bt[1, :7].tolist()
    codes.view(2, 2, p.npages, 16, 128)[:, :, pages] = 0x31            # another sequence's values
    o, s = p.run(codes=codes)
    keep = list(range(nq)) + list(range(2 * nq, 3 * nq))
    assert torch.equal(o[keep], out[keep]) and torch.equal(s[keep], lse[keep])


@pytest.mark.parametrize("nq", [1, 40])
def test_attention_streams_and_graphs(nq):
    """Two captured graphs with a workspace each, replayed on two streams at once."""
    probs = [Problem([3000, 500], [nq, nq], 2, 4, 128, 16, F16, True, seed=20 + i) for i in range(2)]
    want = [p.run() for p in probs]
    size = w4.attention_b8_workspace(nq, 8, 2)
    graphs, got, keep = [], [], []
    for p in probs:
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        out, lse = torch.full_like(want[0][0], 9.0), torch.full_like(want[0][1], 9.0)
        codes = p.cache()
        dl, do = ints(p.lens), ints(p.offsets)
        desc = w4.DeviceKVB8(p.hkv, p.d, p.page, p.npages, codes[0].data_ptr(), p.scales[0].data_ptr(), codes[1].data_ptr(),
                             p.scales[1].data_ptr())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w4.attention_b8_paged(desc, p.bt.data_ptr(), p.bt.stride(0), dl.data_ptr(), do.data_ptr(), 2, nq, 3000, p.q.data_ptr(),
                                  p.q.stride(0), 8, w4.DTYPE_F16, out.data_ptr(), out.stride(0), lse.data_ptr(),
                                  workspace=ws.data_ptr(), workspace_bytes=size, stream=stream())
        graphs.append(graph)
        got.append((out, lse))
        keep.append((ws, codes, dl, do))
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, sides):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])


# ---- the three together ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_serving_loop(dtype):
    """Prompts, then decode steps of a batch: tables, write and attention as a serving loop calls them, in one captured
    step for the decode part; the attention's inputs are checked against the values that were written, in 64 bits."""
    hkv, group, d, page, npages, n = 2, 4, 128, 16, 64, 3
    hq = hkv * group
    width = (hq + 2 * hkv) * d
    gen = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.full((2, hkv, npages * page, d), 0x7F, dtype=torch.uint8, device="cuda")
    scales = torch.full((2, hkv, npages), math.nan, device="cuda")
    free = torch.randperm(npages, generator=gen, device="cuda").to(torch.int32)
    bt = torch.full((n, 20), -1, dtype=torch.int32, device="cuda")
    lens, taken = ints([0] * n), ints([0])
    off = ints([0] * (n + 1))
    cap = 128
    slots, positions = ints([0] * cap), ints([0] * cap)
    rows = torch.zeros(cap, width, dtype=dtype, device="cuda")
    out, lse = torch.zeros(cap, hq, d, dtype=dtype, device="cuda"), torch.zeros(cap, hq, device="cuda")
    fresh = ints([0] * n)
    cache = w4.DeviceKVB8(hkv, d, page, npages, codes[0].data_ptr(), scales[0].data_ptr(), codes[1].data_ptr(), scales[1].data_ptr())

    def step(max_q):
        st = stream()
        w4.page_tables(lens.data_ptr(), fresh.data_ptr(), n, page, npages, free.data_ptr(), npages, taken.data_ptr(), taken.data_ptr(),
                       bt.data_ptr(), bt.stride(0), lens.data_ptr(), off.data_ptr(), slots.data_ptr(), positions.data_ptr(), cap, st)
        w4.kv_write_b8(cache, slots.data_ptr(), cap, rows.data_ptr() + 2 * hq * d, rows.data_ptr() + 2 * (hq + hkv) * d, width, width,
                       CODE[dtype], st)
        w4.attention_b8_paged(cache, bt.data_ptr(), bt.stride(0), lens.data_ptr(), off.data_ptr(), n, max_q, 320, rows.data_ptr(), width,
                              hq, CODE[dtype], out.data_ptr(), out.stride(0), lse.data_ptr(), stream=st)

    history = [[[], []] for _ in range(n)]   # what was written, as values

    def verify(counts):
        torch.cuda.synchronize()
        assert w4.device_status() == 0
        at = 0
        for i, f in enumerate(counts):
            L = int(lens[i])
            pages = bt[i, : -(-L // page)].long()
            val = codes.view(torch.float8_e4m3fn).float().view(2, hkv, npages, page, d) * scales[..., None, None]
            kv = val[:, :, pages].reshape(2, hkv, -1, d)[:, :, :L].double()
            new = rows[at:at + f, hq * d:].view(f, 2, hkv, d).double().permute(1, 2, 0, 3)
            if f:
                # a code is off by half a step: 2^-4 of the value, or 2^-10 of the scale, a 448th of its range
                amax = scales[:, :, pages[(torch.arange(L - f, L, device="cuda") // page)]].double()[..., None] * 448
                assert ((kv[:, :, L - f:] - new).abs() <= new.abs() * 2.0 ** -4 + amax * 2.0 ** -18).all()
            q = rows[at:at + f, : hq * d].view(f, hkv, group, d).double()
            a = torch.einsum("nhgd,hld->nhgl", q, kv[0]) / math.sqrt(d)
            big = torch.einsum("nhgd,hld->nhgl", q.abs(), kv[0].abs()).amax(-1, keepdim=True) / math.sqrt(d) if f else 0
            seen = torch.arange(L, device="cuda")[None] <= L - f + torch.arange(f, device="cuda")[:, None]
            a = a.masked_fill(~seen[:, None, None], -math.inf)
            p = torch.softmax(a, -1)
            ref = torch.einsum("nhgl,hld->nhgd", p, kv[1])
            tol = torch.einsum("nhgl,hld->nhgd", p, kv[1].abs()) * (2.0 ** -11 + 2.0 ** -18 * big) + ref.abs() * (2.0 ** -8 if dtype == BF16 else 2.0 ** -11) * 1.01 + 1e-5
            assert ((out[at:at + f].view(f, hkv, group, d).double() - ref).abs() <= tol).all()
            at += f
        assert (slots[at:] == -1).all()

    def fill():
        rows.copy_((torch.randn(cap, width, generator=gen, device="cuda") * torch.exp2(torch.randn(cap, 1, generator=gen, device="cuda"))).to(dtype))

    fresh.copy_(ints([37, 16, 61]))
    fill()
    step(61)
    verify([37, 16, 61])
    fresh.copy_(ints([0, 40, 3]))
    fill()
    step(40)
    verify([0, 40, 3])
    fresh.copy_(ints([1, 1, 1]))
    fill()
    step(1)
    verify([1, 1, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(1)
    for _ in range(40):
        fill()
        graph.replay()
        verify([1, 1, 1])
    assert int(taken[0]) == sum(-(-int(x) // page) for x in lens.tolist())
