"""CPU tests of the paged 8-bit cache entries: malformed calls are rejected on the host before any pointer is read
(dummy addresses throughout; no GPU needed)."""
import pytest

import w4a16_dequant_gemm_b200 as w4

A = 256  # an aligned address that must never be read


def cache(H=2, D=128, page=16, npages=8, q_k=A, s_k=A, q_v=A, s_v=A):
    return w4.DeviceKVB8(H, D, page, npages, q_k, s_k, q_v, s_v)


BAD_CACHES = {"no heads": cache(H=0), "D 96": cache(D=96), "D 256": cache(D=256), "D 0": cache(D=0), "page 8": cache(page=8),
              "page 24": cache(page=24), "page 0": cache(page=0), "page 8192": cache(page=8192), "no pages": cache(npages=0),
              "rows 2^31": cache(page=4096, npages=1 << 19), "heads": cache(H=65536),
              "null codes": cache(q_k=None), "null value codes": cache(q_v=None), "null scales": cache(s_k=None),
              "null value scales": cache(s_v=None), "codes unaligned": cache(q_v=A + 8), "scales unaligned": cache(s_v=A + 2)}

TABLES = dict(cached=A, fresh=A, nseq=4, page=16, npages=8, free_pages=A, nfree=3, taken_in=A, taken_out=A, bt=A,
              bt_stride=4, seq_lens=A, q_offsets=A, slots=A, positions=A, max_tokens=8)
WRITE = dict(p=cache(), slots=A, T=3, k_new=A, v_new=A, k_stride=256, v_stride=256)
ATTEND = dict(p=cache(), bt=A, bt_stride=4, seq_lens=A, q_offsets=A, nseq=2, max_q=3, max_seq_len=64, q=A, q_stride=512,
              Hq=4, dtype=w4.DTYPE_F16, out=A, out_stride=512)


def refused(fn, base, **change):
    with pytest.raises(w4.InvalidArgument):
        fn(**{**base, **change})


@pytest.mark.parametrize("change", [
    dict(nseq=0), dict(nseq=16385), dict(page=0), dict(npages=0), dict(page=1 << 16, npages=1 << 15), dict(bt_stride=0),
    dict(nfree=-1), dict(max_tokens=-1), dict(cached=None), dict(fresh=None), dict(taken_in=None), dict(taken_out=None),
    dict(bt=None), dict(seq_lens=None), dict(q_offsets=None), dict(free_pages=None), dict(slots=None),
    dict(positions=None)], ids=str)
def test_page_tables_refusals(change):
    refused(w4.page_tables, TABLES, **change)


@pytest.mark.parametrize("name", BAD_CACHES)
def test_cache_descriptor_refusals(name):
    refused(w4.kv_write_b8, WRITE, p=BAD_CACHES[name])
    refused(w4.attention_b8_paged, ATTEND, p=BAD_CACHES[name])


@pytest.mark.parametrize("change", [
    dict(slots=None), dict(T=-1), dict(k_new=None), dict(v_new=None), dict(k_new=A + 8), dict(v_new=A + 2),
    dict(k_stride=255), dict(k_stride=260), dict(v_stride=248), dict(v_stride=-256), dict(dtype=2)], ids=str)
def test_write_refusals(change):
    refused(w4.kv_write_b8, WRITE, **change)


def test_write_of_no_tokens_is_no_launch():
    before = w4.launch_count()
    w4.kv_write_b8(**{**WRITE, "T": 0})
    assert w4.launch_count() == before


@pytest.mark.parametrize("change", [
    dict(bt=None), dict(seq_lens=None), dict(nseq=0), dict(max_q=0), dict(max_seq_len=-1), dict(max_seq_len=65535 * 256 + 1),
    dict(bt_stride=3), dict(q_offsets=None), dict(q=None), dict(out=None), dict(q=A + 8), dict(out=A + 4),
    dict(q_stride=511), dict(q_stride=504), dict(out_stride=8), dict(Hq=3), dict(Hq=0), dict(dtype=-1), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(lse=A + 2),
    dict(workspace=A + 16, workspace_bytes=1 << 30), dict(max_q=1 << 30)], ids=str)
def test_attention_refusals(change):
    refused(w4.attention_b8_paged, ATTEND, **change)


@pytest.mark.parametrize("shape", [(0, 4, 2), (1, 3, 2), (1, 0, 2), (1, 4, 0), (-5, 4, 2)], ids=str)
def test_workspace_refusals(shape):
    with pytest.raises(w4.InvalidArgument):
        w4.attention_b8_workspace(*shape)


def test_binding_refuses_what_the_abi_cannot_hold():
    """The binding of these entries checks its integers instead of cutting them off."""
    with pytest.raises(OverflowError):
        w4.page_tables(**{**TABLES, "nseq": 1 << 31})
    with pytest.raises(OverflowError):
        w4.kv_write_b8(**{**WRITE, "T": 1 << 40})
    with pytest.raises(OverflowError):
        w4.attention_b8_paged(**{**ATTEND, "q": -1})
    with pytest.raises(TypeError):
        w4.attention_b8_paged(**{**ATTEND, "max_q": 1.5})
    with pytest.raises(TypeError):
        w4.page_tables(**{**TABLES, "bt": "table"})
