"""Capped, biased and masked scores and the paged cache in 4 bits without a GPU: the refusals of the C ABI
and of the Python layer, all before any device is touched."""
from __future__ import annotations

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _lib
from test_operators_boundary import BAD, ODD, P, ST, append, attention, refused

FP4 = _lib.FP4
BYTE = P(0x1002)  # 2-byte aligned


def scored_attention(cap=0.0, slopes=None, **how):
    b, d = how.get("b", 1), how.get("d", 64)
    return _lib.lib().fattn_paged_scored_attention(0, how.get("cache", 0), b, 1, 1, d, BAD, ST, BAD,
                                                   how.get("kp", BAD), ST, BAD, ST, 1, 16, BAD, 0, 1, BAD, 1.0,
                                                   cap, slopes, BAD, 1 << 40, None)


def read(cache=0, dtype=0, b=1, hk=1, s=1, d=64, kp=BAD, pst=ST, pages=1, page=16, width=1, lengths=BAD, k=BAD):
    return _lib.lib().fattn_paged_read(cache, dtype, b, hk, s, d, kp, pst, BAD, pst, pages, page, BAD, 0, width,
                                       lengths, None, k, BAD, None)


@pytest.mark.parametrize("call,who", [(append, "paged_append"), (attention, "paged_attention")])
def test_four_bit_cache_refusals(call, who):
    refused(call(dtype=FP4), _lib.FATTN_EINVAL, who + ": f32, f16 or bf16")
    refused(call(cache=FP4, d=48), _lib.FATTN_EHEADDIM, "32, 64 or 128, got 48")
    refused(call(cache=FP4, page=24), _lib.FATTN_EINVAL, "multiple of 16 slots")
    refused(call(cache=FP4, kp=BYTE), _lib.FATTN_EALIGN, "4-byte aligned")
    refused(call(cache=FP4, pst=_lib.arr([0, 0, 38])), _lib.FATTN_EALIGN, "4-byte aligned")
    refused(call(cache=FP4, pst=_lib.arr([0, 0, 1 << 28])), _lib.FATTN_ERANGE, "2 GiB")
    refused(call(cache=FP4, kp=None), _lib.FATTN_EINVAL, "null operand")
    assert call(dtype=1, cache=FP4, b=0, kp=None) == 0


def test_four_bit_append_in_place_refused():
    refused(append(cache=FP4, heads=1), _lib.FATTN_EINVAL, "q_out must not be q")


@pytest.mark.parametrize("cap", [-1.0, 1e-31, 2e30, float("inf"), float("nan")])
def test_cap_refusals(cap):
    refused(scored_attention(cap=cap), _lib.FATTN_EINVAL, "paged_attention: a cap from 1e-30 to 1e30")
    x = torch.zeros(1, 1, 1, 64)
    with pytest.raises(cfa.FusedAttentionError, match="cap|not on a HIP device"):
        cfa.paged_attention(x, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1.0,
                            cap=cap)


def test_scored_attention_refusals():
    refused(scored_attention(cap=1.0, kp=None), _lib.FATTN_EINVAL, "null operand")
    refused(scored_attention(cap=1.0, kp=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    assert scored_attention(cap=1.0, slopes=BAD, b=0) == 0


def test_read_refusals():
    refused(read(dtype=FP4), _lib.FATTN_EINVAL, "paged_read: f32, f16 or bf16")
    refused(read(cache=4), _lib.FATTN_EINVAL, "paged_read: f32, f16 or bf16")
    refused(read(b=-1), _lib.FATTN_EINVAL, "negative size")
    refused(read(s=-1), _lib.FATTN_EINVAL, "negative size")
    refused(read(hk=1 << 16), _lib.FATTN_ERANGE, "heads")
    refused(read(d=96), _lib.FATTN_EHEADDIM, "32, 64 or 128, got 96")
    refused(read(page=8), _lib.FATTN_EINVAL, "multiple of 16 slots")
    refused(read(kp=None), _lib.FATTN_EINVAL, "null operand")
    refused(read(lengths=None), _lib.FATTN_EINVAL, "null operand")
    refused(read(k=None), _lib.FATTN_EINVAL, "null operand")
    refused(read(kp=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(read(cache=FP4, kp=BYTE), _lib.FATTN_EALIGN, "4-byte aligned")
    refused(read(k=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(read(s=1 << 27), _lib.FATTN_ERANGE, "32-bit")
    refused(read(b=1 << 20, hk=64), _lib.FATTN_ERANGE, "launch limit")
    refused(read(pst=_lib.arr([0, 0, -4])), _lib.FATTN_EINVAL, "negative strides")
    assert read(b=0, kp=None) == 0 and read(s=0, k=None) == 0 and read(hk=0, k=None) == 0


def test_fp4_row_bytes():
    assert [cfa.fp4_row_bytes(d) for d in (32, 64, 128)] == [20, 36, 68]
    with pytest.raises(cfa.FusedAttentionError, match="got 48"):
        cfa.fp4_row_bytes(48)


def test_python_refusals():
    q, ints = torch.randn(1, 2, 1, 64), torch.zeros(1, dtype=torch.int32)
    pages = torch.zeros(1, 2, 16, 36, dtype=torch.uint8)
    slopes = torch.zeros(2, requires_grad=True)
    for call, text in [
        (lambda: cfa.paged_append(q, q, pages, pages, ints[None], ints), "not on a HIP device"),
        (lambda: cfa.paged_attention(q, pages, pages, ints[None], ints, 1.0, cap=0.0), "a cap from"),
        (lambda: cfa.paged_attention(q, pages, pages, ints[None], ints, 1.0, slopes=slopes), "not on a HIP device"),
        (lambda: cfa.paged_read(pages, pages, ints[None], ints, 1), "not on a HIP device"),
        (lambda: cfa.paged_read(pages.double(), pages, ints[None], ints, 1), "must be float32"),
        (lambda: cfa.paged_read(pages, pages, ints[None], ints, 1, dtype=torch.float64), "dtype must be"),
        (lambda: cfa.paged_read(pages[0], pages, ints[None], ints, 1), "4 dimensions"),
    ]:
        with pytest.raises(cfa.FusedAttentionError, match=text):
            call()
    with pytest.raises(TypeError):
        cfa.paged_attention(q, pages, pages, ints[None], ints, 1.0, cap="much")


# --- Scored attention -------------------------------------------------------------------------------


def forward(b=1, heads=1, hk=1, sq=1, sk=1, d=64, q=BAD, k=BAD, qst=ST, kst=ST, cap=0.0, documents=None, dst=0,
            out=BAD, ws=BAD, size=1 << 40):
    return _lib.lib().fattn_scored_forward(q, qst, k, kst, k, kst, b, heads, hk, sq, sk, d, 1.0, 1, cap, None,
                                           documents, dst, None, out, BAD, ws, size, None)


def backward(b=1, heads=1, hk=1, sq=1, sk=1, d=64, q=BAD, k=BAD, qst=ST, kst=ST, cap=0.0, documents=None, dst=0,
             out=BAD, g=BAD, gst=ST, dq=BAD, dkv=BAD, ws=BAD, size=1 << 40):
    return _lib.lib().fattn_scored_backward(q, qst, k, kst, k, kst, b, heads, hk, sq, sk, d, 1.0, 1, cap, None,
                                            documents, dst, None, out, BAD, g, gst, dq, dkv, ws, size, None)


@pytest.mark.parametrize("call", [forward, backward])
def test_scored_refusals(call):
    refused(call(b=-1), _lib.FATTN_EINVAL, "fused_scored_attention: negative size")
    refused(call(sq=-1), _lib.FATTN_EINVAL, "negative size")
    refused(call(sq=3, sk=2), _lib.FATTN_EINVAL, "3 queries are more than the 2 positions")
    refused(call(d=48), _lib.FATTN_EHEADDIM, "32, 64 or 128, got 48")
    refused(call(heads=3, hk=2), _lib.FATTN_EINVAL, "3 query heads are no multiple of 2 key heads")
    refused(call(heads=0), _lib.FATTN_EINVAL, "0 query heads")
    for cap in (-1.0, 1e-31, float("inf"), float("nan")):
        refused(call(cap=cap), _lib.FATTN_EINVAL, "a cap from 1e-30 to 1e30")
    refused(call(q=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(k=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(out=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(q=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(k=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(out=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(documents=BAD, dst=-1), _lib.FATTN_EINVAL, "negative strides")
    refused(call(sk=2, kst=_lib.arr([0, 0, 66])), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(sk=2, kst=_lib.arr([0, 0, -4])), _lib.FATTN_EINVAL, "negative strides")
    refused(call(sk=5, kst=_lib.arr([0, 0, 1 << 28])), _lib.FATTN_ERANGE, "4 GiB")
    refused(call(b=1 << 16, heads=1 << 10, hk=1 << 10, sk=1 << 10), _lib.FATTN_ERANGE, "32-bit")
    refused(call(sk=(1 << 31) - 1), _lib.FATTN_ERANGE, "32-bit")
    assert call(b=0, q=None) == 0 and call(heads=0, hk=0) == 0 and call(sq=0, sk=0, k=None) == 0


def test_scored_workspace_and_gradient_refusals():
    L = _lib.lib()
    for size_of, call, more in ((L.fattn_scored_workspace_bytes, forward, ()),
                                (L.fattn_scored_backward_workspace_bytes, backward, (1,))):
        need = size_of(2, 4, 4, 1, 4096, 64, *more)
        assert need > 0
        for ws, size in ((None, need), (ODD, need), (BAD, need - 1)):
            refused(call(b=2, heads=4, hk=4, sk=4096, ws=ws, size=size), _lib.FATTN_EWORKSPACE, str(need))
        assert size_of(64, 8, 8, 4096, 4096, 64, *more) == 0
        assert size_of(2, 4, 3, 1, 4096, 64, *more) == 0
        assert size_of(2, 4, 4, 5000, 4096, 64, *more) == 0
        assert size_of(0, 4, 4, 1, 4096, 64, *more) == 0 and size_of(0, 4, 4, 0, 0, 64, *more) == 0
        assert size_of(2, 4, 4, 0, 0, 64, *more) == 0
    refused(backward(g=None), _lib.FATTN_EINVAL, "null operand")
    refused(backward(dq=None), _lib.FATTN_EINVAL, "null operand")
    refused(backward(dkv=None), _lib.FATTN_EINVAL, "null operand")
    refused(backward(g=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(backward(sq=2, sk=2, gst=_lib.arr([0, 0, 2])), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(backward(sq=5, sk=5, gst=_lib.arr([0, 0, 1 << 28])), _lib.FATTN_ERANGE, "4 GiB")


def test_scored_python_refusals():
    q, ids = torch.randn(1, 2, 3, 64), torch.zeros(1, 3, dtype=torch.int32)
    for call, text in [
        (lambda: cfa.fused_scored_attention(q, q, q, 1.0, True), "not on a HIP device"),
        (lambda: cfa.fused_scored_attention(q.double(), q, q, 1.0, True), "must be float32"),
        (lambda: cfa.fused_scored_attention(q[0], q, q, 1.0, True), "4 dimensions"),
        (lambda: cfa.fused_scored_attention(q, q, [1], 1.0, True), "must be a tensor"),
        (lambda: cfa.fused_scored_attention(q, q, q, 1.0, True, cap=-1.0), "a cap from"),
    ]:
        with pytest.raises(cfa.FusedAttentionError, match=text):
            call()
    with pytest.raises(TypeError):
        cfa.fused_scored_attention(q, q, q, None, True)


def test_forward_mode_refused():
    import torch.autograd.forward_ad as forward_ad

    x, ints, s = torch.randn(1, 2, 3, 64), torch.zeros(1, dtype=torch.int32), torch.zeros(2)
    with forward_ad.dual_level():
        dual, slopes = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(s, torch.ones_like(s))
        for call in (lambda: cfa.fused_scored_attention(dual, x, x, 1.0, True),
                     lambda: cfa.fused_scored_attention(x, dual, x, 1.0, True),
                     lambda: cfa.fused_scored_attention(x, x, dual, 1.0, True),
                     lambda: cfa.fused_scored_attention(x, x, x, 1.0, True, slopes=slopes),
                     lambda: cfa.paged_attention(x[:, :, :1], x, x, ints[None], ints, 1.0, slopes=slopes),
                     lambda: cfa.paged_read(dual, x, ints[None], ints, 1)):
            with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
                call()
