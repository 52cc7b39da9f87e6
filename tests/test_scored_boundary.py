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
