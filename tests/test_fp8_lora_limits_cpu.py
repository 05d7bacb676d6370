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


# -- outputs over what a call reads ---------------------------------------------------

def quant(lib, x=FAR[0], q=FAR[1], s=FAR[2], rows=4, n=64, ldx=64, ldq=64):
    return lib.tsds_quant_fp8(P(x), P(q), P(s), rows, n, ldx, ldq, None)


def norm(lib, x=FAR[0], res=FAR[1], w=FAR[2], ro=FAR[3], q=FAR[4], s=FAR[5], no=FAR[6], rows=4, n=64, ldx=64, ldr=64,
         ldo=64, ldq=64, ldn=64):
    return lib.tsds_add_rms_norm_fp8(P(x), P(res), P(w), P(ro), P(q), P(s), P(no), rows, n, ldx, ldr, ldo, ldq, ldn, 1e-6,
                                     None)


def test_quantiser_over_its_input(lib):
    x = FAR[0]
    for bad in (dict(q=x), dict(q=x, ldq=128), dict(q=x + 64, ldq=128), dict(q=x - 16), dict(q=x + 128 * 3 + 112),
                dict(q=x, rows=1), dict(q=x + 16, ldq=256, ldx=128), dict(q=x + 144, ldq=240, ldx=128, rows=9)):
        assert quant(lib, **bad) == INVALID, bad


def test_norm_outputs_over_one_another_and_operands(lib):
    x, res, ro, q, no = FAR[0], FAR[1], FAR[3], FAR[4], FAR[6]
    for bad in (dict(no=ro), dict(no=ro + 16), dict(no=ro - 16), dict(no=res, ro=res), dict(no=x, ro=x),
                dict(q=x), dict(q=res), dict(q=ro), dict(q=no), dict(q=no + 128 * 3), dict(ro=res + 16), dict(ro=x - 16),
                dict(no=x + 32), dict(no=res + 128), dict(no=x, ldn=72)):
        assert norm(lib, **bad) == INVALID, bad
    assert norm(lib, no=x, res=None, ro=None, q=x) == INVALID


@pytest.mark.parametrize("kind", ["store", "residual", "swiglu"])
def test_projection_output_over_its_operands(lib, kind):
    x, w = FAR[0], FAR[2]
    for bad in (dict(out=x), dict(out=x + 64), dict(out=x - 4), dict(out=w), dict(out=w + 32 * 64 - 2), dict(out=w - 126)):
        assert linear(lib, kind, **bad) == INVALID, bad
    if kind == "swiglu":
        assert linear(lib, kind, out=w + 63 * 64) == INVALID     # 64 rows of gate and up
    if kind == "residual":
        for out in (FAR[6] + 2, FAR[6] - 2, FAR[6] + 64):
            assert linear(lib, kind, out=out) == INVALID
        assert linear(lib, kind, out=FAR[6] + 4, ldo=64, ldr=64) == INVALID


def test_adapter_output_over_its_operands(lib):
    y, x, a, b = FAR[0], FAR[1], FAR[2], FAR[3]
    for M in (2, 2000):
        for out in (x, x + 16, x - 16, y + 16, y - 16, y + 128, a, a + 2 * 16 * 64 * 2 - 16, b, b + 2 * 64 * 16 * 2 - 16):
            assert lora(lib, out=out, M=M) == INVALID, (M, hex(out))


# Row sets side by side, as a program that asks the same arithmetic of random ones would see them.
OVERLAP = r"""
#include <cstdio>
#include "common.cuh"
std::mutex& tsds_host_cache_lock() { static std::mutex m; return m; }
void tsds_count_launch() {}
int main() {
  long long a[4], b[4];
  while (std::scanf("%lld %lld %lld %lld %lld %lld %lld %lld", a, a + 1, a + 2, a + 3, b, b + 1, b + 2, b + 3) == 8)
    std::printf("%d\n", (int)tsds_overlap({(void*)a[0], a[1], a[2], a[3]}, {(void*)b[0], b[1], b[2], b[3]}));
}
"""


def test_overlap_of_random_row_sets(tmp_path):
    """Against sets of bytes, same and different strides, interleaved columns among them."""
    import os
    import random
    import subprocess
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / "overlap.cu", tmp_path / "overlap"
    src.write_text(OVERLAP)
    subprocess.run([nvcc, "-std=c++17", "-I", os.path.join(root, "tri_sds_b200", "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    rng = random.Random(5)
    cases, want = [], []
    for _ in range(4000):
        rows, ld = rng.randint(1, 6), rng.randint(1, 40)
        sets = [(rng.randint(200, 420), r, s, rng.randint(1, s))
                for r, s in ((rows, ld), (rng.choice([rows, rng.randint(1, 6)]), rng.choice([ld, ld, rng.randint(1, 40)])))]
        cases.append(" ".join(str(v) for s in sets for v in s))
        a, b = ({p + i * s + k for i in range(r) for k in range(w)} for p, r, s, w in sets)
        want.append(int(bool(a & b)))
    out = subprocess.run([str(exe)], input="\n".join(cases), capture_output=True, text=True, check=True).stdout.split()
    bad = [(c, w) for c, w, g in zip(cases, want, out) if w != int(g)]
    assert not bad, bad[:5]
    assert 0 < sum(want) < len(want)
