"""The operators around self-attention without a GPU: rotary frequencies against their formulas, and
the refusals of the C ABI and of the Python layer, all before any device is touched."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _lib

P = ctypes.c_void_p
BAD = P(0x1000)  # never dereferenced: every call below fails validation first
ODD = P(0x1008)  # 8-byte aligned
ST = _lib.arr([0, 0, 0])


def refused(rc, code, text):
    assert rc == code, (rc, _lib.last_error())
    assert text in _lib.last_error(), _lib.last_error()


# --- Frequencies ---------------------------------------------------------------------------------


def test_frequencies():
    f = cfa.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,)
    for i in (0, 1, 17, 31):
        assert f[i].item() == pytest.approx(10000.0 ** (-2 * i / 64), rel=1e-14)
    assert torch.equal(cfa.rotary_frequencies(64, scaling="linear", factor=4.0), f / 4)
    g = cfa.rotary_frequencies(64, scaling="base", factor=4.0)
    assert g[0].item() == 1.0 and g[31].item() == pytest.approx(f[31].item() / 4, rel=1e-12)
    r = cfa.rotary_frequencies(64, scaling="ramp", factor=4.0, original_length=4096, low=1.0, high=32.0)
    for i in range(32):
        turns = 4096 * f[i].item() / (2 * math.pi)
        keep = min(max((turns - 1) / 31, 0.0), 1.0)
        assert r[i].item() == pytest.approx(f[i].item() * (keep + (1 - keep) / 4), rel=1e-12)
    assert r[0] == f[0] and r[31].item() == pytest.approx(f[31].item() / 4, rel=1e-15)
    assert cfa.rotary_frequencies(2, scaling="base", factor=4.0).tolist() == [1.0]


@pytest.mark.parametrize("how", [dict(dim=3), dict(dim=0), dict(dim=8, base=0.0),
                                 dict(dim=8, factor=-1.0), dict(dim=8, scaling="other"),
                                 dict(dim=8, scaling="ramp", low=2.0, high=2.0),
                                 dict(dim=8, scaling="ramp", original_length=0)])
def test_frequencies_refused(how):
    with pytest.raises(cfa.FusedAttentionError, match="rotary_frequencies"):
        cfa.rotary_frequencies(**how)


# --- The C ABI -----------------------------------------------------------------------------------


def rotary(dtype=0, b=1, s=1, d=64, heads=(1, 0, 0), x=BAD, strides=(0,) * 9, bits=64, f=BAD, dim=64,
           pos=BAD):
    x3 = (P * 3)(*[x] * 3)
    return _lib.lib().fattn_rotary(dtype, b, s, d, _lib.arr(heads), x3, x3, _lib.arr(strides),
                                   _lib.arr([0] * 9), 1, pos, bits, _lib.arr([0, 0]), f, dim, 0, 1.0, 0,
                                   None)


def test_rotary_refusals():
    refused(rotary(dtype=3), _lib.FATTN_EINVAL, "fused_rotary: f32, f16 or bf16")
    refused(rotary(b=-1), _lib.FATTN_EINVAL, "expected")
    refused(rotary(bits=16), _lib.FATTN_EINVAL, "32 or 64 bits")
    refused(rotary(d=63), _lib.FATTN_EINVAL, "even head_dim")
    refused(rotary(d=2048), _lib.FATTN_EINVAL, "even head_dim")
    refused(rotary(dim=66), _lib.FATTN_EINVAL, "64")
    refused(rotary(dim=7), _lib.FATTN_EINVAL, "even part")
    refused(rotary(f=None), _lib.FATTN_EINVAL, "null frequencies")
    refused(rotary(pos=None), _lib.FATTN_EINVAL, "null positions")
    refused(rotary(x=None), _lib.FATTN_EINVAL, "null operand")
    refused(rotary(heads=(1 << 16, 0, 0)), _lib.FATTN_ERANGE, "heads")
    refused(rotary(b=1 << 13, s=1 << 13), _lib.FATTN_ERANGE, "tokens")
    refused(rotary(strides=(-1,) + (0,) * 8), _lib.FATTN_EINVAL, "negative strides")
    assert rotary(b=0) == 0 and rotary(s=0, x=None) == 0 and rotary(heads=(0, 0, 0)) == 0


def append(dtype=0, cache=0, b=1, heads=0, hk=1, s=1, d=64, k=BAD, pages=1, page=16, width=1, kp=BAD,
           lengths=BAD, st=ST, f=None, dim=0, pst=ST):
    return _lib.lib().fattn_paged_append(dtype, cache, b, heads, hk, s, d, BAD, st, BAD, ST, k, st, BAD,
                                         st, kp, pst, BAD, pst, pages, page, BAD, 0, width, lengths,
                                         None, f, dim, 0, 1.0, None)


def attention(dtype=0, cache=0, b=1, heads=1, hk=1, d=64, q=BAD, qst=ST, kp=BAD, pst=ST, pages=1, page=16,
              width=1, lengths=BAD, ws=BAD, size=1 << 40):
    return _lib.lib().fattn_paged_attention(dtype, cache, b, heads, hk, d, q, qst, BAD, kp, pst, BAD, pst,
                                            pages, page, BAD, 0, width, lengths, 1.0, ws, size, None)


@pytest.mark.parametrize("call,who", [(append, "paged_append"), (attention, "paged_attention")])
def test_cache_refusals(call, who):
    refused(call(dtype=9), _lib.FATTN_EINVAL, who + ": f32, f16 or bf16")
    refused(call(dtype=1, cache=0), _lib.FATTN_EINVAL, "another type")
    refused(call(dtype=1, cache=2), _lib.FATTN_EINVAL, "another type")
    refused(call(b=-1), _lib.FATTN_EINVAL, "negative size")
    refused(call(d=48), _lib.FATTN_EHEADDIM, "32, 64 or 128, got 48")
    refused(call(hk=0), _lib.FATTN_EINVAL, "multiple")
    refused(call(heads=3, hk=2), _lib.FATTN_EINVAL, "3 query heads are no multiple of 2 key heads")
    refused(call(hk=1 << 16, heads=1 << 16), _lib.FATTN_ERANGE, "heads")
    refused(call(page=8), _lib.FATTN_EINVAL, "multiple of 16 slots")
    refused(call(page=0), _lib.FATTN_EINVAL, "multiple of 16 slots")
    refused(call(pages=0), _lib.FATTN_EINVAL, "0 pages")
    refused(call(width=0), _lib.FATTN_EINVAL, "0 wide")
    refused(call(pages=1 << 31), _lib.FATTN_ERANGE, "32-bit")
    refused(call(kp=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(lengths=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(kp=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(pst=_lib.arr([0, 0, 66])), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(pst=_lib.arr([0, 0, 1 << 26])), _lib.FATTN_ERANGE, "2 GiB")
    refused(call(pst=_lib.arr([0, 0, -4])), _lib.FATTN_EINVAL, "negative strides")
    assert call(b=0, kp=None) == 0


def test_append_refusals():
    refused(append(s=-1), _lib.FATTN_EINVAL, "negative size")
    refused(append(k=None), _lib.FATTN_EINVAL, "null operand")
    refused(append(f=BAD, dim=65), _lib.FATTN_EINVAL, "even part")
    refused(append(f=BAD, dim=66), _lib.FATTN_EINVAL, "66 of 64")
    refused(append(b=1 << 13, s=1 << 13), _lib.FATTN_ERANGE, "tokens")
    assert append(s=0, k=None) == 0


def test_attention_refusals():
    refused(attention(q=None), _lib.FATTN_EINVAL, "null operand")
    refused(attention(q=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(attention(b=2, qst=_lib.arr([66, 0])), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(attention(width=1 << 28, page=16), _lib.FATTN_ERANGE, "32-bit")
    refused(attention(b=1 << 20, heads=64, hk=64), _lib.FATTN_ERANGE, "launch limit")
    L = _lib.lib()
    need = L.fattn_paged_attention_workspace_bytes(4, 8, 2, 64, 1 << 20)
    assert need > 0
    for ws, size in ((None, need), (ODD, need), (BAD, need - 1)):
        refused(attention(b=4, heads=8, hk=2, width=1 << 16, ws=ws, size=size), _lib.FATTN_EWORKSPACE,
                str(need))
    assert L.fattn_paged_attention_workspace_bytes(4, 8, 2, 64, 16) == 0
    assert L.fattn_paged_attention_workspace_bytes(4, 8, 3, 64, 1 << 20) == 0
    assert L.fattn_paged_attention_workspace_bytes(4, 8, 2, 48, 1 << 20) == 0
    refused(attention(heads=0), _lib.FATTN_EINVAL, "0 query heads")


def cross(b=1, heads=1, hk=1, sq=1, sk=1, d=64, q=BAD, k=BAD, qst=ST, kst=ST, out=BAD, ws=BAD,
          size=1 << 40):
    return _lib.lib().fattn_cross_forward(q, qst, k, kst, k, kst, b, heads, hk, sq, sk, d, None, 1.0, out,
                                          BAD, ws, size, None)


def cross_bwd(b=1, heads=1, hk=1, sq=1, sk=1, d=64, q=BAD, k=BAD, qst=ST, kst=ST, out=BAD, g=BAD, gst=ST,
              dq=BAD, dkv=BAD, ws=BAD, size=1 << 40):
    return _lib.lib().fattn_cross_backward(q, qst, k, kst, k, kst, b, heads, hk, sq, sk, d, None, 1.0, out,
                                           BAD, g, gst, dq, dkv, ws, size, None)


@pytest.mark.parametrize("call", [cross, cross_bwd])
def test_cross_refusals(call):
    refused(call(b=-1), _lib.FATTN_EINVAL, "fused_cross_attention: negative size")
    refused(call(sk=-1), _lib.FATTN_EINVAL, "negative size")
    refused(call(d=48), _lib.FATTN_EHEADDIM, "32, 64 or 128, got 48")
    refused(call(heads=3, hk=2), _lib.FATTN_EINVAL, "3 query heads are no multiple of 2 key heads")
    refused(call(heads=0), _lib.FATTN_EINVAL, "0 query heads")
    refused(call(hk=0), _lib.FATTN_EINVAL, "0 key heads")
    refused(call(q=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(k=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(out=None), _lib.FATTN_EINVAL, "null operand")
    refused(call(q=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(k=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(out=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(sk=2, kst=_lib.arr([0, 0, 66])), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(call(sk=2, kst=_lib.arr([0, 0, -4])), _lib.FATTN_EINVAL, "negative strides")
    refused(call(sk=5, kst=_lib.arr([0, 0, 1 << 28])), _lib.FATTN_ERANGE, "4 GiB")
    refused(call(b=1 << 16, heads=1 << 10, sq=1 << 10), _lib.FATTN_ERANGE, "32-bit")
    refused(call(sk=(1 << 31) - 1), _lib.FATTN_ERANGE, "32-bit")
    assert call(b=0, q=None) == 0 and call(heads=0, hk=0) == 0


def test_cross_workspace_and_gradient_refusals():
    L = _lib.lib()
    need = L.fattn_cross_workspace_bytes(2, 4, 4, 1, 4096, 64)
    assert need > 0
    for ws, size in ((None, need), (ODD, need), (BAD, need - 1)):
        refused(cross(b=2, heads=4, hk=4, sk=4096, ws=ws, size=size), _lib.FATTN_EWORKSPACE, str(need))
    assert L.fattn_cross_workspace_bytes(64, 8, 8, 1000, 4096, 64) == 0
    assert L.fattn_cross_backward_workspace_bytes(64, 8, 8, 1000, 4096, 64) == 0
    need = L.fattn_cross_backward_workspace_bytes(2, 4, 4, 100, 4096, 64)
    assert need > 0
    for ws, size in ((None, need), (ODD, need), (BAD, need - 1)):
        refused(cross_bwd(b=2, heads=4, hk=4, sq=100, sk=4096, ws=ws, size=size), _lib.FATTN_EWORKSPACE,
                str(need))
    assert L.fattn_cross_workspace_bytes(2, 4, 3, 1, 4096, 64) == 0
    refused(cross_bwd(g=None), _lib.FATTN_EINVAL, "null operand")
    refused(cross_bwd(dq=None), _lib.FATTN_EINVAL, "null operand")
    refused(cross_bwd(dkv=None), _lib.FATTN_EINVAL, "null operand")
    refused(cross_bwd(g=ODD), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(cross_bwd(sq=2, gst=_lib.arr([0, 0, 2])), _lib.FATTN_EALIGN, "16-byte aligned")
    refused(cross_bwd(sq=2, gst=_lib.arr([0, 0, -4])), _lib.FATTN_EINVAL, "negative strides")
    refused(cross_bwd(sq=5, gst=_lib.arr([0, 0, 1 << 28])), _lib.FATTN_ERANGE, "4 GiB")


# --- The Python layer ----------------------------------------------------------------------------


def test_python_refusals():
    q, f = torch.randn(1, 2, 3, 64), cfa.rotary_frequencies(64)
    pos, ints = torch.arange(3), torch.zeros(1, dtype=torch.int32)
    for call, text in [
        (lambda: cfa.fused_rotary(q, q, pos, f), "not on a HIP device"),
        (lambda: cfa.fused_rotary(q.double(), q, pos, f), "must be float32, float16, bfloat16"),
        (lambda: cfa.fused_rotary(q[0], q, pos, f), "4 dimensions"),
        (lambda: cfa.fused_rotary([1], q, pos, f), "must be a tensor"),
        (lambda: cfa.fused_rotary_qkv(q[0], 2, pos, f), "not on a HIP device"),
        (lambda: cfa.paged_append(q, q, q, q, ints[None], ints), "not on a HIP device"),
        (lambda: cfa.paged_attention(q[:, :, :1], q, q, ints[None], ints, 1.0), "not on a HIP device"),
        (lambda: cfa.fused_cross_attention(q, q, q, 1.0), "not on a HIP device"),
        (lambda: cfa.fused_cross_attention(q.half(), q, q, 1.0), "must be float32, got float16"),
    ]:
        with pytest.raises(cfa.FusedAttentionError, match=text):
            call()


def test_missing_binding_is_an_error(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_operators", None)
    monkeypatch.setattr(_lib, "OPERATORS_PATH", tmp_path / "absent.so")
    with pytest.raises(cfa.FusedAttentionError, match="not built"):
        cfa.fused_cross_attention(torch.zeros(1), torch.zeros(1), torch.zeros(1), 1.0)
    monkeypatch.setattr(_lib, "OPERATORS_PATH", tmp_path / "broken.so")
    (tmp_path / "broken.so").write_bytes(b"no library")
    with pytest.raises(cfa.FusedAttentionError, match="cannot load"):
        cfa.fused_cross_attention(torch.zeros(1), torch.zeros(1), torch.zeros(1), 1.0)


def test_binding_arguments():
    q, f = torch.randn(1, 2, 3, 64), cfa.rotary_frequencies(64)
    pos = torch.arange(3)
    with pytest.raises(cfa.FusedAttentionError, match="too few arguments"):
        _lib.operators().rotary(q, q, pos)
    with pytest.raises(TypeError):
        cfa.fused_rotary(q, q, pos, f, False, "one")
    with pytest.raises(TypeError):
        cfa.fused_cross_attention(q, q, q, None)
    with pytest.raises(cfa.FusedAttentionError) as e:
        cfa.fused_cross_attention(q, q, q, 1.0)
    assert e.value.code == 0


def test_forward_mode_refused():
    """An operand with a tangent of forward-mode differentiation: a result without one would be a
    derivative of 0."""
    import torch.autograd.forward_ad as forward_ad

    x, f, pos = torch.randn(1, 2, 3, 64), cfa.rotary_frequencies(64), torch.arange(3)
    ints = torch.zeros(1, dtype=torch.int32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        turning = forward_ad.make_dual(f, torch.ones_like(f))
        for call in (lambda: cfa.fused_rotary(dual, x, pos, f), lambda: cfa.fused_rotary(x, dual, pos, f),
                     lambda: cfa.fused_rotary(x, x, pos, turning),
                     lambda: cfa.fused_rotary_qkv(dual[0], 2, pos[:2], f),
                     lambda: cfa.fused_rotary_qkv(x[0], 2, pos[:2], turning),
                     lambda: cfa.paged_append(dual, x, x, x, ints[None], ints),
                     lambda: cfa.paged_append(x, dual, x, x, ints[None], ints),
                     lambda: cfa.paged_append(x, x, dual, x, ints[None], ints),
                     lambda: cfa.paged_append(x, x, x, dual, ints[None], ints),
                     lambda: cfa.paged_append(x, x, x, x, ints[None], ints, q=dual),
                     lambda: cfa.paged_append(x, x, x, x, ints[None], ints, frequencies=turning),
                     lambda: cfa.paged_attention(dual[:, :, :1], x, x, ints[None], ints, 1.0),
                     lambda: cfa.paged_attention(x[:, :, :1], dual, x, ints[None], ints, 1.0),
                     lambda: cfa.paged_attention(x[:, :, :1], x, dual, ints[None], ints, 1.0),
                     lambda: cfa.fused_cross_attention(dual, x, x, 1.0),
                     lambda: cfa.fused_cross_attention(x, dual, x, 1.0),
                     lambda: cfa.fused_cross_attention(x, x, dual, 1.0)):
            with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
                call()
            with torch.no_grad(), pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
                call()


def test_learned_frequencies_refused():
    """Frequencies that require a gradient would get none: refused, unless no graph is recorded or they are
    detached."""
    x, pos, ints = torch.randn(1, 2, 3, 64), torch.arange(3), torch.zeros(1, dtype=torch.int32)
    f = cfa.rotary_frequencies(64).requires_grad_()
    for call in (lambda f: cfa.fused_rotary(x, x, pos, f), lambda f: cfa.fused_rotary_qkv(x[0], 2, pos[:2], f),
                 lambda f: cfa.paged_append(x, x, x, x, ints[None], ints, frequencies=f)):
        with pytest.raises(cfa.FusedAttentionError, match="no gradient of the frequencies"):
            call(f)
        for fine in (lambda: call(f.detach()), lambda: torch.no_grad()(call)(f)):
            with pytest.raises(cfa.FusedAttentionError, match="not on a HIP device"):
                fine()
