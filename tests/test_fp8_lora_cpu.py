"""Argument checks of the 8-bit projection and adapter operators: C-ABI codes
before any launch, and the Python layer's refusals (no GPU needed)."""
import ctypes

import pytest
import torch

INVALID, ALIGN, WORKSPACE, UNSUPPORTED = 1, 2, 4, 6
BF, F32, I32, E4M3 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    from tri_sds_b200 import _lib
    return _lib.load()


P = ctypes.c_void_p
A = 0x10000   # an aligned stand-in address: every call below is refused before it is used


def test_quant_codes(lib):
    def call(x=A, q=A, s=A, rows=2, n=64, ldx=64, ldq=64):
        return lib.tsds_quant_fp8(P(x), P(q), P(s), rows, n, ldx, ldq, None)
    assert call(rows=0) == 0 and call(rows=0, x=None, q=None, s=None) == 0
    for bad in (dict(rows=-1), dict(n=0), dict(n=40), dict(ldx=56), dict(ldq=48), dict(x=None), dict(q=None),
                dict(s=None)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(x=A + 2), dict(q=A + 8), dict(ldx=68), dict(ldq=72)):
        assert call(**bad) == ALIGN, bad


def test_norm_codes(lib):
    def call(x=A, res=A, w=A, ro=A, q=A, s=A, no=A, rows=2, n=64, ldx=64, ldr=64, ldo=64, ldq=64, ldn=64):
        return lib.tsds_add_rms_norm_fp8(P(x), P(res), P(w), P(ro), P(q), P(s), P(no), rows, n, ldx, ldr, ldo, ldq, ldn,
                                         1e-6, None)
    assert call(rows=0) == 0
    for bad in (dict(rows=-1), dict(n=72), dict(ldx=48), dict(ldr=48), dict(ldo=48), dict(ldq=48), dict(ldn=48),
                dict(x=None), dict(w=None), dict(q=None), dict(s=None), dict(ro=None),
                dict(ro=A, res=A, ldo=128), dict(ro=A, res=A + 4096, ldo=128)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(x=A + 8), dict(w=A + 2), dict(res=A + 2), dict(ro=A + 4), dict(q=A + 1), dict(no=A + 2),
                dict(ldx=68, ro=A + 4096), dict(ldr=68, res=A + 4096, x=A + 8192), dict(ldq=72), dict(ldn=68)):
        assert call(**bad) == ALIGN, bad


def test_linear_codes(lib):
    def store(x=A, ldx=64, sx=A, w=A, sw=A, out=A, ldo=32, M=2, n=32, K=64, st=A):
        return lib.tsds_linear_fp8(P(x), ldx, P(sx), P(w), P(sw), P(out), ldo, M, n, K, P(st), None)

    def swiglu(x=A, ldx=64, sx=A, w=A, sw=A, out=A, ldo=32, M=2, n=32, K=64, st=A):
        return lib.tsds_linear_swiglu_fp8(P(x), ldx, P(sx), P(w), P(sw), P(out), ldo, M, n, K, P(st), None)

    def residual(x=A, ldx=64, sx=A, w=A, sw=A, out=A, ldo=32, M=2, n=32, K=64, st=A, res=A, ldr=32):
        return lib.tsds_linear_residual_fp8(P(x), ldx, P(sx), P(w), P(sw), P(res), ldr, P(out), ldo, M, n, K, P(st),
                                            None)
    for call in (store, swiglu, residual):
        assert call(M=0) == 0
        for bad in (dict(M=-1), dict(n=0), dict(K=0), dict(K=72, ldx=80), dict(ldx=48), dict(ldo=31), dict(x=None),
                    dict(sx=None), dict(w=None), dict(sw=None), dict(out=None), dict(st=None),
                    dict(n=1 << 30, ldo=1 << 30)):
            assert call(**bad) == INVALID, (call, bad)
        for bad in (dict(x=A + 8), dict(w=A + 8), dict(ldx=72)):
            assert call(**bad) == ALIGN, (call, bad)
    assert residual(res=None) == INVALID and residual(ldr=16) == INVALID
    assert residual(out=A, res=A, ldr=40) == INVALID   # in place with two row strides


def test_lora_codes(lib):
    def call(y=A, ldy=64, x=A, ldx=64, a=A, b=A, ad=A, out=A + 65536, ldo=64, M=2, K=64, N=64, n_ad=2, R=16, S=1,
             widths=None, ws=A, wsb=1 << 30, st=A):
        w = None if widths is None else (ctypes.c_int32 * len(widths))(*widths)
        return lib.tsds_lora_add(P(y), ldy, P(x), ldx, P(a), P(b), P(ad), None, None, P(out), ldo, M, K, N, n_ad, R, S,
                                 w, P(ws), wsb, P(st), None)
    assert call(M=0) == 0
    for bad in (dict(M=-1), dict(K=0), dict(K=60), dict(N=0), dict(N=60), dict(n_ad=0), dict(R=0), dict(R=12),
                dict(ldx=56), dict(ldy=56), dict(ldo=56), dict(S=0), dict(S=2), dict(S=2, widths=[32, 16]),
                dict(S=2, widths=[48, 16]), dict(S=2, widths=[64, 32]), dict(S=2, widths=[-32, 96]),
                dict(S=3, widths=[32, 32, 0]), dict(y=None), dict(x=None), dict(a=None), dict(b=None), dict(ad=None),
                dict(out=None), dict(st=None), dict(out=A, ldo=72)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(M=2000, ws=None), dict(M=2000, wsb=64)):
        assert call(**bad) == WORKSPACE, bad
    assert lib.tsds_lora_workspace_bytes(8, 16, 3) == 0 and lib.tsds_lora_workspace_bytes(2000, 16, 3) > 0
    for bad in (dict(R=136), dict(S=5, widths=[32] * 5, N=160, ldy=160, ldo=160)):
        assert call(**bad) == UNSUPPORTED, bad
    for bad in (dict(y=A + 8), dict(x=A + 2), dict(a=A + 8), dict(b=A + 4), dict(out=A + 8), dict(ldx=68),
                dict(ldy=68), dict(ldo=68), dict(M=2000, ws=A + 8)):
        assert call(**bad) == ALIGN, bad


def test_lora_output_over_its_input_and_row_counts(lib):
    def call(M=2, n_ad=2, x=A, out=A + 65536, N=64):
        return lib.tsds_lora_add(P(A), N, P(x), 64, P(A), P(A), P(A), None, None, P(out), N, M, 64, N, n_ad, 16, 1, None,
                                 P(A), 1 << 30, P(A), None)
    assert call(out=A) == INVALID             # out = y is x as well
    assert call(x=A + 65536) == INVALID
    assert call(M=2000, n_ad=1 << 26) == UNSUPPORTED and call(M=2000, n_ad=1 << 20, N=2048) == UNSUPPORTED


# -- the Python layer -------------------------------------------------------------

def _cases(t):
    """(call, message) for tensors made by t(dtype, *shape)."""
    from tri_sds_b200 import ops
    x, w, q, s = t(BF, 4, 64), t(BF, 64), t(E4M3, 4, 64), t(F32, 4)
    wq, ws = t(E4M3, 32, 64), t(F32, 32)
    y, a, b, ad = t(BF, 4, 32), t(BF, 3, 16, 64), t(BF, 3, 32, 16), t(I32, 4)
    return ops, x, w, q, s, wq, ws, y, a, b, ad


def test_host_tensors_are_refused():
    ops, x, w, q, s, wq, ws, y, a, b, ad = _cases(lambda dt, *sh: torch.zeros(*sh).to(dt))
    for call in (lambda: ops.quant_fp8(x), lambda: ops.add_rms_norm_fp8(x, w), lambda: ops.linear_fp8(q, s, wq, ws),
                 lambda: ops.linear_residual_fp8(q, s, wq, ws, y), lambda: ops.linear_swiglu_fp8(q, s, wq, ws),
                 lambda: ops.lora_add(y, x, a, b, ad)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_shapes_and_types_are_checked(monkeypatch):
    """With the device checks reduced to dtypes, every mismatch raises before a pointer is taken."""
    from tri_sds_b200 import _lib, ops as o

    def dtype_only(dtype, *ts):
        for t in ts:
            o._need(t is None or t.dtype == dtype, f"expected {dtype}")
    monkeypatch.setattr(o, "_cuda", dtype_only)
    monkeypatch.setattr(o, "_bf16_cuda", lambda *ts: dtype_only(BF, *ts))
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("the library was called"))
    monkeypatch.setattr(o._scratch, "status_word", lambda dev: torch.zeros(1, dtype=I32))
    ops, x, w, q, s, wq, ws, y, a, b, ad = _cases(lambda dt, *sh: torch.zeros(*sh).to(dt))
    bad = [
        lambda: ops.quant_fp8(x.float()), lambda: ops.quant_fp8(x[0]), lambda: ops.quant_fp8(x.t()),
        lambda: ops.quant_fp8(x, out=q[:3]), lambda: ops.quant_fp8(x, out=q[:, :48]),
        lambda: ops.quant_fp8(x, scale=s[:3]), lambda: ops.quant_fp8(x, scale=s.double()),
        lambda: ops.quant_fp8(x, out=x),
        lambda: ops.add_rms_norm_fp8(x, w[:32]), lambda: ops.add_rms_norm_fp8(x, w, residual=x[:3]),
        lambda: ops.add_rms_norm_fp8(x, w, res_out=x), lambda: ops.add_rms_norm_fp8(x, w, residual=x, res_out=x[:2]),
        lambda: ops.add_rms_norm_fp8(x, w, norm_out=x[:, :32]), lambda: ops.add_rms_norm_fp8(x, w, residual=x.float()),
        lambda: ops.linear_fp8(x, s, wq, ws), lambda: ops.linear_fp8(q, s[:2], wq, ws),
        lambda: ops.linear_fp8(q, s, wq[:, :32], ws), lambda: ops.linear_fp8(q, s, wq, ws[:8]),
        lambda: ops.linear_fp8(q, s, wq.t(), ws), lambda: ops.linear_fp8(q, s, wq, ws, out=y[:, :16]),
        lambda: ops.linear_residual_fp8(q, s, wq, ws, y[:2]), lambda: ops.linear_residual_fp8(q, s, wq, ws, y.float()),
        lambda: ops.linear_swiglu_fp8(q, s, wq[:31], ws[:31]), lambda: ops.linear_swiglu_fp8(q, s, wq, ws[:16]),
        lambda: ops.lora_add(y, x[:3], a, b, ad), lambda: ops.lora_add(y, x, a[:2], b, ad),
        lambda: ops.lora_add(y, x, a, b[:, :16], ad), lambda: ops.lora_add(y, x, a, b, ad.long()),
        lambda: ops.lora_add(y, x, a, b, ad[:2]), lambda: ops.lora_add(y, x, a, b, ad, scale=s),
        lambda: ops.lora_add(y, x, a, b, ad, ranks=ad), lambda: ops.lora_add(y, x, a, b, ad, slices=[16, 16]),
        lambda: ops.lora_add(y, x, a, b, ad, out=y[:2]), lambda: ops.lora_add(y, x, a.transpose(1, 2), b, ad),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was accepted")


# -- torch.ops.tsds ------------------------------------------------------------------

_STREAM = object()


@pytest.fixture()
def recorded(monkeypatch):
    """Calls recorded instead of made; every pointer must reach the bytes its call's sizes say."""
    import tri_sds_b200.torch_ops  # noqa: F401
    from abi_extents import TRef
    from tri_sds_b200 import _lib, ops as o

    def dtype_only(dtype, *ts):
        for t in ts:
            o._need(t is None or t.dtype == dtype, f"expected {dtype}")
    calls = []

    def call(name, *a):
        assert a[-1] is _STREAM, name
        calls.append(name)
        need = _extents(name, a[:-1])
        assert need
        for i, nbytes in need:
            assert a[i] is None or a[i].bytes_left() >= nbytes, (name, i, nbytes)
    monkeypatch.setattr(o, "_p", lambda t: None if t is None else TRef(t))
    monkeypatch.setattr(o, "_stream", lambda: _STREAM)
    monkeypatch.setattr(o, "_cuda", dtype_only)
    monkeypatch.setattr(o, "_bf16_cuda", lambda *ts: dtype_only(BF, *ts))
    monkeypatch.setattr(_lib, "call", call)
    yield calls


def _extents(name, a):
    """[(argument, bytes it must reach)] from the meanings in include/tsds.h."""
    def rows(m, ld, n, size):
        return ((m - 1) * ld + n) * size
    if name == "tsds_quant_fp8":
        x, q, s, m, n, ldx, ldq = a
        return [(0, rows(m, ldx, n, 2)), (1, rows(m, ldq, n, 1)), (2, m * 4)]
    if name == "tsds_add_rms_norm_fp8":
        m, n, ldx, ldr, ldo, ldq, ldn = a[7:14]
        return [(0, rows(m, ldx, n, 2)), (1, rows(m, ldr, n, 2)), (2, n * 2), (3, rows(m, ldo, n, 2)),
                (4, rows(m, ldq, n, 1)), (5, m * 4), (6, rows(m, ldn, n, 2))]
    if name in ("tsds_linear_fp8", "tsds_linear_swiglu_fp8"):
        x, ldx, sx, w, sw, out, ldo, m, n, k, st = a
        wr = 2 * n if "swiglu" in name else n
        return [(0, rows(m, ldx, k, 1)), (2, m * 4), (3, wr * k), (4, wr * 4), (5, rows(m, ldo, n, 2)), (10, 4)]
    if name == "tsds_linear_residual_fp8":
        x, ldx, sx, w, sw, res, ldr, out, ldo, m, n, k, st = a
        return [(0, rows(m, ldx, k, 1)), (2, m * 4), (3, n * k), (4, n * 4), (5, rows(m, ldr, n, 2)),
                (7, rows(m, ldo, n, 2)), (12, 4)]
    if name == "tsds_lora_add":
        y, ldy, x, ldx, la, lb, ad, sc, rk, out, ldo, m, k, n, na, r, s, wd, ws, nb, st = a
        return [(0, rows(m, ldy, n, 2)), (2, rows(m, ldx, k, 2)), (4, na * s * r * k * 2), (5, na * n * r * 2),
                (6, m * 4), (7, na * 4), (8, na * 4), (9, rows(m, ldo, n, 2)), (18, nb), (20, 4)]
    return []


def test_torch_ops_calls_and_extents(recorded):
    import tri_sds_b200.torch_ops as T
    tsds = torch.ops.tsds
    for name in T.PROJECTION_OPS:
        schema = getattr(tsds, name).default._schema
        assert not any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments), name
    x, w, q, s = torch.zeros(5, 64).to(BF), torch.zeros(64).to(BF), torch.zeros(5, 64).to(E4M3), torch.zeros(5)
    wq, ws, y = torch.zeros(48, 64).to(E4M3), torch.zeros(48), torch.zeros(5, 48).to(BF)
    assert [t.shape for t in tsds.quant_fp8(x)] == [(5, 64), (5,)]
    assert [t.shape for t in tsds.add_rms_norm_fp8(x, x, w)] == [(5, 64), (5,), (5, 64), (5, 64)]
    assert tsds.linear_fp8(q, s, wq, ws).shape == (5, 48)
    assert tsds.linear_residual_fp8(q, s, wq, ws, y).shape == (5, 48)
    assert tsds.linear_swiglu_fp8(q, s, wq, ws).shape == (5, 24)
    for m in (5, 2000):   # one launch, and two with a workspace
        a, b, ad = torch.zeros(3, 32, 64).to(BF), torch.zeros(3, 96, 16).to(BF), torch.zeros(m, dtype=I32)
        out = tsds.lora_add(torch.zeros(m, 96).to(BF), torch.zeros(m, 64).to(BF), a, b, ad, torch.ones(3),
                            torch.ones(3, dtype=I32), [64, 32])
        assert out.shape == (m, 96)
    assert recorded == ["tsds_quant_fp8", "tsds_add_rms_norm_fp8", "tsds_linear_fp8", "tsds_linear_residual_fp8",
                        "tsds_linear_swiglu_fp8", "tsds_lora_add", "tsds_lora_add"]
