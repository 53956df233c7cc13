"""GPU tests of the paged 8-bit cache operators at the edges of what a call may say: bounds above and below what the
device-side counts ask for, table sizes around the shared memory's limits, values at the ends of their types. The plain
forms and the tolerances are those of test_gpu_b8.py; what a test adds to them it derives where it stands."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import w4a16_dequant_gemm_b200 as w4
from test_gpu_b8 import BF16, CODE, F16, Problem, ints, plain_tables, run_tables, same_tables, stream, table_case

pytestmark = pytest.mark.gpu


def check_rows(p, out, lse, tokens, missing=()):
    """`tokens` of the problem against its 64-bit form; all other rows as they were."""
    ref, ref_lse, b_out, b_lse = p.reference(missing)
    o, s = out[tokens].double().cpu(), lse[tokens].double().cpu()
    empty = ref_lse[tokens] == -math.inf
    assert (s[empty] == -math.inf).all() and (o[empty] == 0).all()
    assert ((o - ref[tokens]).abs() <= b_out[tokens])[~empty].all()
    assert ((s - ref_lse[tokens]).abs() <= b_lse[tokens])[~empty].all()
    rest = torch.ones(len(out), dtype=torch.bool)
    rest[tokens] = False
    assert (out[rest.cuda()] == 9).all() and (lse[rest.cuda()] == 9).all()


# ---- attention: max_q and max_seq_len are bounds -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("hkv,group,d", [(2, 4, 128), (2, 1, 64), (1, 40, 64)])
@pytest.mark.parametrize("n", [0, 1, 5, 8, 9, 32, 33])
def test_attention_max_q_above_every_count(n, hkv, group, d, dtype):
    """max_q = 64 whatever the counts: one sequence alone, and beside an empty and a short one."""
    for lens, nq in (([200 + n], [n]), ([100 + n, 0, 77], [n, 0, 2])):
        p = Problem(lens, nq, hkv, group, d, 32, dtype, True, seed=300 + n)
        p.check(*p.run(max_q=64))
    assert w4.device_status() == 0


@pytest.mark.parametrize("group", [1, 4])
def test_attention_counts_change_between_replays(group):
    """One captured call for up to 64 tokens of one request; the counts are written between its replays."""
    p = Problem([300], [64], 2, group, 128, 16, F16, True, seed=320)
    size = w4.attention_b8_workspace(64, 2 * group, 2)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    codes, hq = p.cache(), 2 * group
    out, lse = torch.empty(66, hq, 128, dtype=F16, device="cuda"), torch.empty(66, hq, device="cuda")
    dl, do = ints([300]), ints([0, 64])
    desc = w4.DeviceKVB8(2, 128, 16, p.npages, codes[0].data_ptr(), p.scales[0].data_ptr(), codes[1].data_ptr(), p.scales[1].data_ptr())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w4.attention_b8_paged(desc, p.bt.data_ptr(), p.bt.stride(0), dl.data_ptr(), do.data_ptr(), 1, 64, 300, p.q.data_ptr(),
                              p.q.stride(0), hq, w4.DTYPE_F16, out.data_ptr(), out.stride(0), lse.data_ptr(),
                              workspace=ws.data_ptr(), workspace_bytes=size, stream=stream())
    for n in (1, 64, 5, 0, 33, 9, 32, 64):
        p.nq, p.offsets, p.tokens = [n], [0, n], n
        do.copy_(ints([0, n]))
        out.fill_(9)
        lse.fill_(9)
        graph.replay()
        p.check(out, lse)
    assert w4.device_status() == 0


# ---- block tables --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n", [4051, 4052, 4053, 4095, 4096, 9001, 16384])
def test_tables_of_many_requests(n):
    """Around 48 KB of shared memory (12 n + 8 bytes and what the kernel holds besides), and the most there may be."""
    rng = np.random.default_rng(n)
    cached, fresh, page, npages, free, bt, need = table_case(rng, n, 16, 40, 2)
    tokens = sum(fresh)
    same_tables((cached, fresh, page, npages, free, 0, bt, tokens + 5))
    same_tables((cached, fresh, page, npages, free, 0, bt, tokens + 3), in_place=True)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
@pytest.mark.parametrize("nq,max_q,group", [([5, 2, 4], 3, 4), ([9], 1, 2), ([90, 20, 300], 40, 4), ([150], 70, 2), ([40, 3], 30, 1)], ids=str)
def test_attention_more_tokens_than_max_q(nq, max_q, group, causal, dtype):
    """The tokens behind the first max_q of a sequence are left out and reported; the others see what they would see."""
    lens = [300 + 7 * n for n in nq]
    p = Problem(lens, nq, 2, group, 128, 16, dtype, causal, seed=330)
    out, lse = p.run(max_q=max_q)
    kept = [p.offsets[i] + j for i, n in enumerate(nq) for j in range(min(n, max_q))]
    check_rows(p, out, lse, kept)
    assert w4.device_status() == 605
    p.check(*p.run(max_q=max(nq)))
    assert w4.device_status() == 0


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
@pytest.mark.parametrize("nq", [[1, 3], [60, 100], [130]], ids=str)
def test_attention_longer_than_max_seq_len(nq, causal):
    """Positions from max_seq_len on are left out and reported; a token's own position stays what it is."""
    cut, page = 192, 16
    lens = [250, 190][: len(nq)]
    p = Problem(lens, nq, 2, 2, 64, page, F16, causal, seed=340)
    p.max_len = cut
    out, lse = p.run()
    missing = [(i, c) for i in range(len(nq)) for c in range(cut // page, 20)]
    check_rows(p, out, lse, list(range(p.tokens)), missing)
    assert w4.device_status() == 605


# ---- the library's scratch -----------------------------------------------------------------------------------------

SCRATCH = """
import sys, threading, torch
sys.path[:0] = ["tests", "."]
import w4a16_dequant_gemm_b200 as w4
from test_gpu_b8 import Problem, F16
"""


def in_a_fresh_process(script):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", SCRATCH + script], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


def test_scratch_is_complete_after_the_first_call():
    """A process whose first call is a decode step, then captures a step of prompt chunks, both without a workspace."""
    in_a_fresh_process("""
one = Problem([500, 40], [1, 1], 2, 4, 128, 16, F16, True, seed=1)
one.check(*one.run())
p = Problem([500, 90], [70, 40], 2, 4, 128, 16, F16, True, seed=2)
hq, codes = 8, p.cache()
out, lse = torch.full((p.tokens + 2, hq, 128), 9.0, dtype=F16, device="cuda"), torch.full((p.tokens + 2, hq), 9.0, device="cuda")
dl, do = torch.tensor(p.lens, dtype=torch.int32, device="cuda"), torch.tensor(p.offsets, dtype=torch.int32, device="cuda")
desc = w4.DeviceKVB8(2, 128, 16, p.npages, codes[0].data_ptr(), p.scales[0].data_ptr(), codes[1].data_ptr(), p.scales[1].data_ptr())
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    w4.attention_b8_paged(desc, p.bt.data_ptr(), p.bt.stride(0), dl.data_ptr(), do.data_ptr(), 2, 70, 500, p.q.data_ptr(), p.q.stride(0),
                          hq, w4.DTYPE_F16, out.data_ptr(), out.stride(0), lse.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
graph.replay()
p.check(out, lse)
""")


def test_scratch_with_first_calls_of_several_threads():
    """Eight threads make their first calls at once (on one stream, as calls without a workspace have to be)."""
    in_a_fresh_process("""
probs = [Problem([500 + 30 * i, 40], [n, 1], 2, 4, 128, 16, F16, True, seed=i) for i, n in enumerate([1, 60, 1, 200, 3, 90, 1, 64])]
torch.cuda.synchronize()
got, gate = [None] * len(probs), threading.Barrier(len(probs))
def work(i):
    gate.wait()
    got[i] = probs[i].run()
threads = [threading.Thread(target=work, args=(i,)) for i in range(len(probs))]
[t.start() for t in threads]
[t.join() for t in threads]
for p, g in zip(probs, got):
    p.check(*g)
""")


# ---- attention: values ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,nseq", [(1, 80), (4, 80), (64, 20)])
def test_attention_first_position_outweighs_all_others(nq, nseq, dtype):
    """A first position e^18.75 = 2^27 above the others, whose own value is zero: the output is made of the others alone,
    each weighing 2^-27 of it. With L positions, value v and e = exp(-18.75): out = v (L - 1) e / (1 + (L - 1) e). The
    score is exact but for FP32 roundings (2^-19 of it, as elsewhere), the weights are rounded by 2^-11 relatively, or by
    2^-34 of the largest one where that is more: half of the smallest half, 2^-25, beside a largest weight of 2^9 or more; lse = 18.75 + log(1 + (L - 1) e)."""
    L, hkv, group, d, page, s, v = 2000, 8, 4, 64, 16, 18.75, 64.0
    p = Problem([L] * nseq, [nq] * nseq, hkv, group, d, page, dtype, False, seed=350, scale=1.0)
    codes = torch.zeros(2, hkv, p.npages, page, d, dtype=torch.uint8, device="cuda")
    codes[1] = 0x68                                                   # 64
    first = p.bt[:, 0].long()
    codes[1][:, first, 0] = 0
    codes[0][:, first, 0, 0] = 0x38                                   # 1
    p.codes = codes.view(2, hkv, -1, d).view(torch.float8_e4m3fn)
    p.scales.fill_(1.0)
    p.q.zero_()
    p.q[..., 0] = s
    out, lse = p.run()
    e = math.exp(-s)
    want, want_lse = v * (L - 1) * e / (1 + (L - 1) * e), s + math.log1p((L - 1) * e)
    half = 2.0 ** -11 if dtype == F16 else 2.0 ** -8
    tol = want * (2.0 ** -11 + 2 * 2.0 ** -19 * s + 1.01 * half) + 2.0 ** -34 * L * v
    assert ((out[:p.tokens].double() - want).abs() <= tol).all()
    assert ((lse[:p.tokens].double() - want_lse).abs() <= 2.0 ** -19 * s + 2.0 ** -20 * (1 + want_lse)).all()


def test_tables_in_place_keep_refused_requests():
    """A loop that advances in place: a request that does not fit keeps its cached length and its pages, and goes on when
    it is asked for something that fits."""
    rng = np.random.default_rng(6)
    cached, fresh, page, npages, free, bt, need = table_case(rng, 30, 16, 100, 30, spare=40)
    cached[3] = max(cached[3], 20)
    bt[3, :2] = free[-2:]
    free = free[:-2]
    fresh[3], fresh[7], cached[11] = page * bt.shape[1] + 1 - cached[3], -2, -4     # too long, negative counts
    tokens = sum(max(f, 0) for f in fresh)
    want = plain_tables(cached, fresh, page, npages, free, 0, bt, tokens)
    got = run_tables(cached, fresh, page, npages, free, 0, bt, tokens, in_place=True)
    refused = [3, 7, 11]
    lens = [c if i in refused else n for i, (c, n) in enumerate(zip(cached, want[1]))]
    assert got[6] == 602 and got[1] == lens
    assert np.array_equal(want[0], got[0]) and list(want[2:6]) == list(got[2:6])
    assert run_tables(cached, fresh, page, npages, free, 0, bt, tokens)[1] == want[1]   # into another array: 0
    again = [1] * 30
    again[11] = 0
    same_tables((lens[:11] + [0] + lens[12:], again, page, npages, free, got[5], got[0], 40))


def test_tables_in_place_go_on_after_the_pages_ran_out():
    """A request that got no page for some positions: its length set back to its first missing entry, it goes on with
    the pages of another list."""
    rng = np.random.default_rng(7)
    cached, fresh, page, npages, free, bt, need = table_case(rng, 20, 16, 100, 60, spare=80)
    tokens = sum(fresh)
    bt, lens, _, _, _, taken, status = run_tables(cached, fresh, page, npages, free[:need - 9], 0, bt, tokens, in_place=True)
    assert status == 601 and taken == need - 9
    for i, n in enumerate(lens):
        gone = [c for c in range(-(-n // page)) if bt[i, c] < 0]
        if gone:
            assert gone[0] * page >= cached[i]
            lens[i] = gone[0] * page
    left = [cached[i] + fresh[i] - n for i, n in enumerate(lens)]
    assert sum(left) > 0
    want = plain_tables(cached, fresh, page, npages, free, 0, bt, tokens)   # as if they had been there at once
    got = run_tables(lens, left, page, npages, free[need - 9:], 0, bt, sum(left), in_place=True)
    assert got[6] == 0 and got[1] == want[1] and np.array_equal(got[0], want[0])


# ---- the write -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("page", [16, 32, 48, 256])
def test_write_refuses_a_page_that_comes_back(page):
    """Slots of a page that stand apart - by tokens that are not written - are two runs of it: the first is written,
    the second is reported and not written."""
    H, D, npages = 2, 64, 8
    b = [i * page for i in range(npages)]
    cases = [
        ([5, -1, 7], [0]),
        ([5, -1, 6], [0]),
        ([5, 10 ** 9, 6, 7], [0]),
        ([b[1] + 4, 10 ** 9, -1, b[1] + 5, b[1] + 6], [0]),
        ([b[2] + 3, b[2] + 4, -1, b[2], b[2] + 1, b[5]], [0, 1, 5]),
        ([7] + [-1] * (page - 2) + [8], [0]),
        ([b[4] + 2, -1, b[5] + 2, -1, b[4] + 1, b[6] + 2], [0, 2, 5]),
    ]
    for slots, kept in cases:
        T = len(slots)
        gen = torch.Generator().manual_seed(len(slots))
        x = (torch.randn(2, T, H, D, generator=gen) + 3).to(F16).cuda()
        got = []
        for use in (slots, [s if i in kept else -1 for i, s in enumerate(slots)]):
            q = torch.zeros(2, H, npages * page, D, dtype=torch.uint8, device="cuda")
            sc = torch.full((2, H, npages), 2.0 ** -7, device="cuda")
            sl = ints(use)
            p = w4.DeviceKVB8(H, D, page, npages, q[0].data_ptr(), sc[0].data_ptr(), q[1].data_ptr(), sc[1].data_ptr())
            w4.kv_write_b8(p, sl.data_ptr(), T, x[0].data_ptr(), x[1].data_ptr(), H * D, H * D, w4.DTYPE_F16, stream())
            got.append((w4.device_status(), q.cpu(), sc.cpu()))
        assert got[0][0] == 603 and got[1][0] == 0, slots
        assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][2], got[1][2]), slots
        assert (got[0][1] != 0).any(-1).any(1).any(0).nonzero().flatten().tolist() == sorted(slots[i] for i in kept)


def test_write_takes_other_pages_in_any_order():
    """Runs of different pages in any order, with skipped tokens between them, are all written."""
    from test_gpu_b8 import new_rows, run_write, runs
    slots = runs([(100, 12), (16, 16), (3, 13)]) + [-1, -1] + runs([(64, 5)]) + [-1] + runs([(53, 2), (80, 16), (40, 1)])
    x = new_rows(len(slots), 2, 64, F16, 17)
    run_write(2, 64, 16, 8, slots, x[0], x[1])


@pytest.mark.parametrize("nq", [1, 5, 40])
def test_attention_bf16_queries_at_the_ends_of_the_type(nq):
    """Query values up to 2e38 and down to the subnormal ones, with scales that bring the scores back to a few units."""
    p = Problem([300, 70], [nq, nq], 2, 2, 64, 16, BF16, True, seed=360, q_amp=4e37, scale=2e-38)
    p.check(*p.run())
    p = Problem([300, 70], [nq, nq], 2, 2, 128, 16, BF16, True, seed=361, q_amp=1e36, scale=1e-36)
    p.check(*p.run())
    p = Problem([300, 70], [nq, nq], 2, 2, 64, 16, BF16, True, seed=362, q_amp=1e-37, scale=1e29, scale_exp=(18, 21))
    p.check(*p.run())


def test_tables_of_pages_near_2_to_31():
    """One page of 2^31 - 1 positions: the tokens of a request that holds it go into it."""
    page = 2 ** 31 - 1
    for cached, fresh in ((5, 3), (2 ** 30 + 1, 2), (page - 1, 1), (0, 4)):
        bt = np.full((1, 1), 0 if cached else -3, dtype=np.int32)
        same_tables(([cached], [fresh], page, 1, [] if cached else [0], 0, bt, fresh + 1))


def test_tables_with_token_sums_beyond_32_bits():
    """Refused requests whose counts sum up past 2^31: the lengths of the requests behind them are their own."""
    huge, page = 2 ** 31 - 1, 16
    cached, fresh = [20, 5, 0, 33, 7], [3, huge, huge, 5, 30]
    bt = np.array([[1, 2, -3, -3], [3, -3, -3, -3], [-3] * 4, [4, 5, 6, -3], [7, -3, -3, -3]], dtype=np.int32)
    got = run_tables(cached, fresh, page, 64, list(range(20, 40)), 0, bt, 10)
    assert got[6] == 602 and got[1] == [23, 0, 0, 38, 37]
    assert got[0][4].tolist() == [7, 20, 21, -3] and got[5] == 2
    assert got[3][:3] == [36, 37, 38] and got[3][3:] == [-1] * 7
