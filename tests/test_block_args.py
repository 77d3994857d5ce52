"""Refusals of the operators around a block's linears (no GPU): every bad
argument is an error before anything touches a device."""
import ctypes

import pytest

import bonsai_b1
from bonsai_b1 import capi

P = 0x10000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return bonsai_b1.load()


@pytest.mark.parametrize("change", [
    dict(H=33), dict(H=0), dict(rows=-1), dict(x=None), dict(x=P + 4), dict(ldx=32), dict(ldx=66), dict(add=P + 8),
    dict(add=P, ld_add=60), dict(h=P + 4, ldh=64), dict(h=P, ldh=128), dict(weight=P + 4), dict(eps=-1.0),
    dict(eps=float("nan")), dict(y=None), dict(y=P + 4), dict(ldy=32)])
def test_rms_norm(lib, change):
    a = dict(x=P, ldx=64, add=None, ld_add=0, H=64, rows=2, weight=None, eps=1e-6, h=None, ldh=0, y=P * 2, ldy=64)
    a.update(change)
    assert lib.bonsai_b1_rms_norm_f32(*a.values(), None) == capi.ERR_ARG
    if "ldy" not in change:
        packed = list(a.values())[:-1]
        assert lib.bonsai_b1_rms_norm_pack_f16(*packed, None) == capi.ERR_ARG


def pages(**change):
    a = dict(k=P, v=P * 2, n_pages=4, page_size=16, page_stride=2 * 16 * 128, head_stride=16 * 128, row_stride=128,
             pages=P, ld_pages=8, max_pages=8, kv_len=P)
    a.update(change)
    return capi.KvPages(*a.values())


BAD_PAGES = [dict(k=None), dict(v=P + 8), dict(n_pages=0), dict(page_size=0), dict(page_size=24), dict(page_size=-16),
             dict(page_stride=100), dict(head_stride=-8), dict(row_stride=64), dict(row_stride=129),
             dict(page_stride=0), dict(pages=None), dict(pages=P + 2), dict(ld_pages=7), dict(max_pages=0),
             dict(kv_len=None), dict(kv_len=P + 1), dict(max_pages=1 << 26, ld_pages=1 << 26)]


def qkv(kv=None, **change):
    a = dict(q=P, k=P, v=P, ldq=512, ldk=256, ldv=256, tokens=3, heads=4, kv_heads=2, head_dim=128, q_weight=None,
             k_weight=None, eps=1e-6, rope=None, rope_rows=0, rope_dim=0, interleaved=0, positions=None, dtype=0,
             q_out=P, ld_q=512, k_out=P, v_out=P, ld_kv=256, pages=ctypes.pointer(kv) if kv else None, n_seqs=1,
             q_start=None, bad=None)
    a.update(change)
    return capi.QkvArgs(*a.values())


@pytest.mark.parametrize("change", [
    dict(q=None), dict(q=P + 4), dict(ldq=511), dict(ldq=510), dict(ldk=200), dict(ldv=258), dict(tokens=-1),
    dict(heads=0), dict(heads=3), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=32), dict(dtype=2),
    dict(dtype=-1), dict(q_weight=P + 4), dict(eps=-1.0), dict(rope=P, rope_rows=0, rope_dim=128),
    dict(rope=P, rope_rows=5, rope_dim=12), dict(rope=P, rope_rows=5, rope_dim=136),
    dict(rope=P + 4, rope_rows=5, rope_dim=128), dict(positions=P + 2), dict(q_out=None), dict(q_out=P + 8),
    dict(ld_q=508), dict(k_out=None), dict(v_out=P + 2), dict(ld_kv=128), dict(ld_kv=260), dict(bad=P + 1),
    dict(tokens=1 << 27)])
def test_qkv_rope(lib, change):
    assert lib.bonsai_b1_qkv_rope(ctypes.byref(qkv(**change)), None) == capi.ERR_ARG


@pytest.mark.parametrize("change", BAD_PAGES)
def test_bad_pages(lib, change):
    kv = pages(**change)
    assert lib.bonsai_b1_qkv_rope(ctypes.byref(qkv(kv)), None) == capi.ERR_ARG
    a = attention(kv)
    assert lib.bonsai_b1_attention(ctypes.byref(a), None, 0, None) == capi.ERR_ARG
    assert lib.bonsai_b1_attention_workspace_bytes(ctypes.byref(a)) == 0


def test_several_sequences_need_starts(lib):
    assert lib.bonsai_b1_qkv_rope(ctypes.byref(qkv(pages(), n_seqs=2)), None) == capi.ERR_ARG
    assert lib.bonsai_b1_qkv_rope(ctypes.byref(qkv(pages(), n_seqs=0, q_start=P)), None) == capi.ERR_ARG
    assert lib.bonsai_b1_attention(ctypes.byref(attention(pages(), n_seqs=2)), None, 0, None) == capi.ERR_ARG
    assert lib.bonsai_b1_attention(ctypes.byref(attention(n_seqs=2, q_start=P)), None, 0, None) == capi.ERR_ARG


def attention(kv=None, **change):
    a = dict(q=P, k=P, v=P, q_row=512, q_head=128, k_row=256, k_head=128, v_row=256, v_head=128, dtype=1, heads=4,
             kv_heads=2, head_dim=128, tokens=5, kv_tokens=9, n_seqs=1, q_start=None, kv_start=None,
             pages=ctypes.pointer(kv) if kv else None, causal=1, window=0, scale=0.1, out=P * 2, ldo=512, packed=0,
             bad=None)
    a.update(change)
    return capi.AttentionArgs(*a.values())


@pytest.mark.parametrize("change", [
    dict(q=None), dict(q=P + 8), dict(k=None), dict(v=P + 2), dict(q_row=100), dict(q_head=-8), dict(k_row=4),
    dict(k_head=12), dict(v_row=1 << 50), dict(v_head=2), dict(dtype=3), dict(heads=5), dict(heads=-4),
    dict(kv_heads=0), dict(head_dim=80), dict(tokens=-1), dict(kv_tokens=-1), dict(n_seqs=-1), dict(q_start=P + 2),
    dict(kv_start=P + 1), dict(window=-1), dict(window=5, causal=0), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None), dict(out=P + 8), dict(ldo=511),
    dict(ldo=508), dict(bad=P + 3), dict(tokens=1 << 26)])
def test_attention(lib, change):
    a = attention(**change)
    assert lib.bonsai_b1_attention(ctypes.byref(a), None, 0, None) == capi.ERR_ARG
    assert lib.bonsai_b1_attention_workspace_bytes(ctypes.byref(a)) == 0


@pytest.mark.parametrize("change", [
    dict(tokens=1 << 24), dict(heads=1 << 16, kv_heads=1 << 16), dict(tokens=1 << 22, heads=64, kv_heads=8),
    dict(n_seqs=1 << 22, q_start=P, kv_start=P), dict(n_seqs=1 << 30, q_start=P, kv_start=P), dict(kv_tokens=1 << 30),
    dict(k_row=(1 << 23) + 8), dict(v_row=1 << 24)])
def test_attention_too_large(lib, change):
    a = attention(**change)
    assert lib.bonsai_b1_attention(ctypes.byref(a), None, 0, None) == capi.ERR_ARG
    assert lib.bonsai_b1_attention_workspace_bytes(ctypes.byref(a)) == 0


def test_attention_misaligned_workspace(lib):
    assert lib.bonsai_b1_attention(ctypes.byref(attention()), P + 8, 1 << 20, None) == capi.ERR_ARG
    assert lib.bonsai_b1_attention(None, None, 0, None) == capi.ERR_ARG
    assert lib.bonsai_b1_qkv_rope(None, None) == capi.ERR_ARG


def test_python_refuses_what_is_no_cuda_tensor():
    import torch
    x = torch.zeros(2, 64)
    h = torch.zeros(2, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        bonsai_b1.rms_norm(x)
    with pytest.raises(ValueError):
        bonsai_b1.qkv_rope(x, x, x, 64)
    with pytest.raises(ValueError):
        bonsai_b1.attention(h, h, h)
    with pytest.raises(ValueError):
        bonsai_b1.attention_paged(h, h[None], h[None], None, x, x)


@pytest.mark.parametrize("h", [32, 512, 544, 2048, 2080, 4096, 4128, 8192, 8224, 16384, 16416, 32768, 32800, 70016])
def test_rms_norm_launches_fit(lib, h):
    """The rows of a launch keep its threads below the launch limit of 2^32,
    and cover a call of any number of rows in a few launches."""
    lib.b1_rms_norm_launch.restype = ctypes.c_int64
    threads, per = ctypes.c_int(0), ctypes.c_int(0)
    rows = lib.b1_rms_norm_launch(h, ctypes.byref(threads), ctypes.byref(per))
    assert rows % per.value == 0 and 1 << 21 <= rows < 1 << 31
    assert rows // per.value * threads.value < 1 << 32


def test_python_refuses_workspaces_smaller_than_their_elements():
    import torch
    buf = torch.zeros(64, dtype=torch.uint8)
    assert capi._workspace(None) == (None, 0)
    assert capi._workspace(buf[8:40]) == (buf.data_ptr() + 8, 32)
    assert capi._workspace(buf.float().view(8, 8)[2:4])[1] == 64
    for t in (buf[:1].expand(1 << 20), buf[::2], buf.view(8, 8).t()):
        with pytest.raises(ValueError):
            capi._workspace(t)
