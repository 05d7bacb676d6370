"""Calls of the 8-bit projections and adapters that are refused for their sizes or overlaps, through
the C ABI and the Python layer (no GPU needed)."""
import ctypes

import pytest

OK, INVALID, ALIGN, WORKSPACE, UNSUPPORTED = 0, 1, 2, 4, 6


@pytest.fixture(scope="module")
def lib():
    from tri_sds_b200 import _lib
    return _lib.load()


P = ctypes.c_void_p
A = 1 << 32            # stand-in addresses, far apart: every call below is refused before one is used
FAR = [A + (i << 36) for i in range(1, 12)]


def lora(lib, y=FAR[0], ldy=64, x=FAR[1], ldx=64, a=FAR[2], b=FAR[3], ad=FAR[4], out=FAR[5], ldo=64, M=2, K=64, N=64,
         n_ad=2, R=16, S=1, widths=None, ws=FAR[6], wsb=1 << 30, st=FAR[7]):
    w = None if widths is None else (ctypes.c_int32 * len(widths))(*widths)
    return lib.tsds_lora_add(P(y), ldy, P(x), ldx, P(a), P(b), P(ad), None, None, P(out), ldo, M, K, N, n_ad, R, S, w, P(ws),
                             wsb, P(st), None)


def test_width_of_a_single_slice(lib):
    for M in (0, 2, 2000):
        for widths in ([32], [0], [-64], [96]):
            assert lora(lib, M=M, widths=widths) == INVALID, (M, widths)
    assert lora(lib, M=0, widths=[64]) == OK and lora(lib, M=0, N=40, widths=[40]) == OK


def linear(lib, kind="store", x=FAR[0], ldx=64, sx=FAR[1], w=FAR[2], sw=FAR[3], out=FAR[4], ldo=32, M=2, n=32, K=64,
           st=FAR[5], res=FAR[6], ldr=32):
    if kind == "residual":
        return lib.tsds_linear_residual_fp8(P(x), ldx, P(sx), P(w), P(sw), P(res), ldr, P(out), ldo, M, n, K, P(st), None)
    f = lib.tsds_linear_fp8 if kind == "store" else lib.tsds_linear_swiglu_fp8
    return f(P(x), ldx, P(sx), P(w), P(sw), P(out), ldo, M, n, K, P(st), None)


@pytest.mark.parametrize("kind", ["store", "residual", "swiglu"])
def test_rows_and_k_whose_whole_blocks_pass_32_bits(lib, kind):
    for bad in (dict(M=2 ** 31 - 1), dict(M=2 ** 31 - 200), dict(K=2 ** 31 - 16, ldx=2 ** 31 - 16)):
        assert linear(lib, kind, **bad) == UNSUPPORTED, bad


def test_adapter_widths_whose_whole_blocks_pass_32_bits(lib):
    assert lora(lib, K=2 ** 31 - 8, ldx=2 ** 31 - 8) == UNSUPPORTED
    assert lora(lib, N=2 ** 31 - 8, ldy=2 ** 31 - 8, ldo=2 ** 31 - 8) == UNSUPPORTED


def test_sizes_and_strides_past_32_bits_raise(monkeypatch):
    """ctypes would pass their low 32 bits on: 2^32 + 64 columns apart would read as 64."""
    import torch
    from tri_sds_b200 import _lib, ops
    bf, f32, i32, e4 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn

    def t(dtype, *shape, ld=None):
        v = torch.empty(shape, dtype=dtype, device="meta")
        return v if ld is None else torch.empty_strided(shape, (ld, 1), dtype=dtype, device="meta")
    monkeypatch.setattr(ops, "_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "_bf16_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "_p", lambda v: None)
    monkeypatch.setattr(ops, "_one_device", lambda *a: -1)
    monkeypatch.setattr(ops._scratch, "status_word", lambda dev: None)
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("the library was called"))
    big = 2 ** 32 + 64
    x, w, q, s, wq, ws = t(bf, 4, 64), t(bf, 64), t(e4, 4, 64), t(f32, 4), t(e4, 32, 64), t(f32, 32)
    y, a, b, ad = t(bf, 4, 32), t(bf, 3, 16, 64), t(bf, 3, 32, 16), t(i32, 4)
    bad = [
        lambda: ops.quant_fp8(t(bf, 4, 64, ld=big)), lambda: ops.quant_fp8(t(bf, big, 64)),
        lambda: ops.quant_fp8(t(bf, 1, big)), lambda: ops.quant_fp8(x, out=t(e4, 4, 64, ld=big)),
        lambda: ops.add_rms_norm_fp8(t(bf, 4, 64, ld=big), w),
        lambda: ops.add_rms_norm_fp8(x, w, residual=t(bf, 4, 64, ld=big)),
        lambda: ops.add_rms_norm_fp8(x, w, residual=x, res_out=t(bf, 4, 64, ld=big)),
        lambda: ops.add_rms_norm_fp8(x, w, norm_out=t(bf, 4, 64, ld=big)),
        lambda: ops.linear_fp8(t(e4, 4, 64, ld=big), s, wq, ws), lambda: ops.linear_fp8(t(e4, big, 64), t(f32, big), wq, ws),
        lambda: ops.linear_fp8(q, s, t(e4, big, 64), t(f32, big)), lambda: ops.linear_fp8(q, s, wq, ws, out=t(bf, 4, 32, ld=big)),
        lambda: ops.linear_swiglu_fp8(q, s, t(e4, 2 * big, 64), t(f32, 2 * big)),
        lambda: ops.linear_residual_fp8(q, s, wq, ws, t(bf, 4, 32, ld=big)),
        lambda: ops.lora_add(t(bf, 4, 32, ld=big), x, a, b, ad), lambda: ops.lora_add(y, t(bf, 4, 64, ld=big), a, b, ad),
        lambda: ops.lora_add(y, x, a, b, ad, out=t(bf, 4, 32, ld=big)),
        lambda: ops.lora_add(y, x, t(bf, big, 16, 64), t(bf, big, 32, 16), ad),
        lambda: ops.lora_add(y, x, t(bf, 1, big, 64), t(bf, 1, 32, big), ad),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError, match="below 2"):
            call()
            pytest.fail(f"case {i} was accepted")
