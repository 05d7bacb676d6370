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
