"""GPU checks of the 8-bit operators (row quantisation, residual + RMSNorm +
8 bits, the e4m3 projections) against their definitions in 64 bits."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from tri_sds_b200 import ops as o
    yield o
    o.check_status()


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *shape, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(BF)


def _quantised(g, rows, k, std=1.0):
    x = torch.randn(rows, k, device=DEV, generator=g) * std
    s = x.abs().amax(dim=1) / 448
    return (x / s[:, None]).to(E4M3), s


@pytest.mark.parametrize("rows,n", [(1, 16), (1, 5120), (3, 48), (7, 2064), (26, 25600), (2, 32768), (3, 40000),
                                    (300, 256)])
def test_quant(ops, rows, n):
    x = _rand(_gen(rows * n), rows, n, std=3.0)
    x[0, n // 2] = 1000.0
    q, s = ops.quant_fp8(x)
    ref.check_quant(q, s, x.double(), 2 * ref.F32)


@pytest.mark.parametrize("n", [8208, 9024, 16384, 16400, 21952, 32768, 32784])
def test_many_long_rows(ops, n):
    """Enough rows for the threads per row to follow the row's length."""
    g = _gen(n)
    x, w = _rand(g, 601, n, std=3.0), _rand(g, n, std=0.2) + 1
    x[600, n - 1] = 1000.0
    q, s = ops.quant_fp8(x)
    ref.check_quant(q, s, x.double(), 2 * ref.F32)
    no = torch.empty_like(x)
    q, s, ro = ops.add_rms_norm_fp8(x, w, residual=x, norm_out=no)
    _check_norm(x, x, w, 1e-6, q, s, ro, no)


def test_quant_ties_go_to_even(ops):
    """Half-way values: 448 fixes the scale at 1, so the sums 2^e (8 + m + 1/2) / 8 are exact ties."""
    vals = [2.0 ** e * (8 + m + 0.5) / 8 for e in range(-6, 8) for m in range(8)]
    row = torch.tensor([448.0] + vals + [-v for v in vals] + [0.0] * (240 - 2 * len(vals) - 1), device=DEV)
    x = (row[None] * torch.tensor([[1.0], [0.5], [3.0]], device=DEV)).to(BF)   # scales 1, 1/2, 3
    q, _ = ops.quant_fp8(x)
    v = row.double()
    step = ref.e4m3_step(v)
    want = torch.clamp(torch.round(v / step) * step, -448, 448)
    exact = (x.double() == row.double()[None] * torch.tensor([[1.0], [0.5], [3.0]], device=DEV).double())
    assert exact[:2].all() and (q.double()[:2] == want).all()
    assert (q.double()[2][exact[2]] == want[exact[2]]).all()


def test_quant_zero_tiny_and_nan_rows(ops):
    x = torch.zeros(6, 64, device=DEV, dtype=BF)
    x[1, 3] = 2.0 ** -120          # below the smallest scale: rounds to zero
    x[2, 5] = 2.0 ** -99
    x[3] = 1.0
    x[3, 7] = float("nan")
    x[4] = 1.0
    x[4, 0] = float("inf")
    x[5] = -2.0
    q, s = ops.quant_fp8(x)
    tiny = torch.tensor(ref.TINY / 448, device=DEV, dtype=torch.float64)
    assert (q[0].float() == 0).all() and (q[1].float() == 0).all()
    assert abs(s[0].double() / tiny - 1) < 1e-6 and s[0] == s[1]
    assert q[2, 5].float() == 448 and q[2].float().count_nonzero() == 1
    assert torch.isnan(s[3]) and torch.isnan(q[3].float()).all()
    assert not torch.isfinite(s[4]) and torch.isnan(q[4].float()).all()
    assert (q[5].float() == -448).all()


def test_quant_strides_and_neighbours(ops):
    g = _gen(5)
    big = _rand(g, 9, 200)
    out = torch.zeros(9, 256, device=DEV, dtype=torch.uint8).view(E4M3)
    scale = torch.full((9,), -1.0, device=DEV)
    ops.quant_fp8(big[2:7, 8:136], out=out[2:7, 16:144], scale=scale[2:7])
    ref.check_quant(out[2:7, 16:144], scale[2:7], big[2:7, 8:136].double(), 2 * ref.F32)
    o = out.view(torch.uint8)
    assert (o[:2] == 0).all() and (o[7:] == 0).all() and (o[:, :16] == 0).all() and (o[:, 144:] == 0).all()
    assert (scale[:2] == -1).all() and (scale[7:] == -1).all()


# the mean of squares: at most 70 additions one after another, halved by the square root
NORM_TOL = 40 * ref.F32


def _check_norm(x, res, w, eps, q, s, res_out, norm_out):
    r = x.float()
    if res is not None:
        r = (r + res.float()).to(BF).float()
        assert torch.equal(res_out, r.to(BF))
    r = r.double()
    y = r / torch.sqrt(r.square().mean(dim=1, keepdim=True) + eps) * w.double()
    ref.check_quant(q, s, y, NORM_TOL)
    if norm_out is not None:
        ref.check_bf16(norm_out, y, y.abs() * NORM_TOL)


@pytest.mark.parametrize("rows,n", [(1, 16), (1, 5120), (5, 2560), (26, 5120), (3, 8192), (2, 12288), (2, 40000),
                                    (513, 272)])
@pytest.mark.parametrize("res,norm", [(False, False), (True, False), (True, True), (False, True)])
def test_add_rms_norm(ops, rows, n, res, norm):
    g = _gen(rows + n)
    x, w = _rand(g, rows, n), _rand(g, n, std=0.2) + 1
    r = _rand(g, rows, n, std=4.0) if res else None
    no = torch.empty(rows, n, device=DEV, dtype=BF) if norm else None
    q, s, ro = ops.add_rms_norm_fp8(x, w, residual=r, eps=1e-6, norm_out=no)
    _check_norm(x, r, w, 1e-6, q, s, ro, no)
    if norm and n <= 8192:   # both sum the row with 256 threads in the same order; longer rows here with 1024
        assert torch.equal(no, ops.rms_norm(x if r is None else ro, w, 1e-6))


@pytest.mark.parametrize("n", [5120, 40000])
@pytest.mark.parametrize("target", ["residual", "x"])
def test_add_rms_norm_in_place(ops, n, target):
    g = _gen(7)
    x, r, w = _rand(g, 9, n), _rand(g, 9, n), _rand(g, n)
    q0, s0, ro0 = ops.add_rms_norm_fp8(x, w, residual=r)
    dst = r if target == "residual" else x
    q1, s1, ro1 = ops.add_rms_norm_fp8(x, w, residual=r, res_out=dst)
    assert ro1 is dst and torch.equal(ro0, dst)
    assert torch.equal(q0.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s0, s1)


def test_add_rms_norm_strides_zero_and_nan_rows(ops):
    g = _gen(8)
    x, r = _rand(g, 6, 512)[:, 128:384], _rand(g, 8, 320)[1:7, :256]
    x[2] = 0
    r[2] = 0
    x[4, 17] = float("nan")
    x[5, 3] = float("inf")
    w = _rand(g, 256)
    q, s, ro = ops.add_rms_norm_fp8(x, w, residual=r)
    ok = torch.tensor([0, 1, 3], device=DEV)
    _check_norm(x[ok], r[ok], w, 1e-6, q[ok], s[ok], ro[ok], None)
    assert (q[2].float() == 0).all() and torch.isfinite(s[2])
    for bad in (4, 5):
        assert torch.isnan(s[bad]) and torch.isnan(q[bad].float()).all()


def test_zero_rows(ops):
    e = torch.empty(0, 256, device=DEV, dtype=BF)
    w = torch.ones(256, device=DEV, dtype=BF)
    assert ops.quant_fp8(e)[0].shape == (0, 256)
    assert ops.add_rms_norm_fp8(e, w, residual=e)[2].shape == (0, 256)
    q, s = ops.quant_fp8(_rand(_gen(1), 32, 256))
    eq, es = ops.quant_fp8(e)
    assert ops.linear_fp8(eq, es, q, s).shape == (0, 32)
    assert ops.linear_swiglu_fp8(eq, es, q, s).shape == (0, 16)
    assert ops.linear_residual_fp8(eq, es, q, s, torch.empty(0, 32, device=DEV, dtype=BF)).shape == (0, 32)


# -- projections ------------------------------------------------------------------

def _check_linear(ops, kind, M, n, K, seed=0, out=None, res=None):
    g = _gen(seed + M + n + K)
    xq, xs = _quantised(g, M, K)
    wq, ws = _quantised(g, 2 * n if kind == "swiglu" else n, K, std=0.05)
    acc, err = ref.linear(xq, xs, wq, ws)
    if kind == "store":
        got = ops.linear_fp8(xq, xs, wq, ws, out=out)
    elif kind == "residual":
        res = _rand(g, M, n) if res is None else res
        acc, err = acc + res.double(), err + ref.F32 * (acc.abs() + res.double().abs())
        got = ops.linear_residual_fp8(xq, xs, wq, ws, res, out=out)
    else:
        acc, err = ref.silu_mul(acc[:, :n], err[:, :n], acc[:, n:], err[:, n:])
        got = ops.linear_swiglu_fp8(xq, xs, wq, ws, out=out)
    ops.check_status()
    ref.check_bf16(got, acc, err)
    return got


@pytest.mark.parametrize("kind", ["store", "residual", "swiglu"])
@pytest.mark.parametrize("M,n,K", [
    (1, 1, 16), (1, 128, 128), (2, 130, 256), (5, 1003, 144), (16, 64, 2576), (17, 640, 1280), (26, 5120, 2560),
    (37, 1003, 2576), (64, 768, 5120), (65, 257, 4096), (100, 333, 528), (128, 2048, 1040), (129, 96, 1024),
    (208, 5120, 2560), (255, 200, 272), (256, 1280, 2560), (257, 300, 400), (512, 640, 1024), (700, 1111, 1296),
    (2048, 128, 512)])
def test_linear(ops, kind, M, n, K):
    _check_linear(ops, kind, M, n, K)


@pytest.mark.parametrize("kind,M,n,K", [("store", 1, 10240, 5120), ("swiglu", 26, 25600, 5120),
                                        ("residual", 208, 5120, 25600), ("residual", 8, 5120, 8192),
                                        ("store", 3, 70000, 256)])
def test_linear_32b_shapes(ops, kind, M, n, K):
    _check_linear(ops, kind, M, n, K)


@pytest.mark.parametrize("kind", ["store", "residual", "swiglu"])
@pytest.mark.parametrize("M,n,K", [(20, 51201, 64), (33, 40004, 48), (100, 25602, 128), (128, 38400, 144),
                                   (129, 20001, 80), (300, 12801, 48), (513, 9732, 528), (2049, 5120, 272)])
def test_linear_many_whole_units(ops, kind, M, n, K):
    """More weight tiles than CTAs: whole units, odd, even and 8-byte aligned rows, rows past a multiple of 32."""
    _check_linear(ops, kind, M, n, K)


def test_linear_residual_in_place_many_units(ops):
    g = _gen(12)
    xq, xs = _quantised(g, 300, 96)
    wq, ws = _quantised(g, 12801, 96, std=0.05)
    res = _rand(g, 300, 12801)
    want = ops.linear_residual_fp8(xq, xs, wq, ws, res)
    assert torch.equal(ops.linear_residual_fp8(xq, xs, wq, ws, res, out=res), want)


def test_linear_strides_and_neighbours(ops):
    """x, res and out as column ranges of wider buffers; nothing outside out is written."""
    g = _gen(3)
    M, n, K = 21, 203, 384
    xq, xs = _quantised(g, M, 640)
    x = xq[:, 128:128 + K]
    wq, ws = _quantised(g, n, K, std=0.05)
    acc, err = ref.linear(x, xs, wq, ws)
    buf = torch.full((M + 2, 331), 7.0, device=DEV, dtype=BF)
    out = buf[1:-1, 5:5 + n]
    got = ops.linear_fp8(x, xs, wq, ws, out=out)
    ref.check_bf16(got, acc, err)
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[1:-1, 5:5 + n] = False
    assert (buf[keep] == 7).all()
    # the residual in place, odd stride
    out.copy_(_rand(g, M, n))
    before = out.double()
    ops.linear_residual_fp8(x, xs, wq, ws, out, out=out)
    ref.check_bf16(out, acc + before, err + ref.F32 * (acc.abs() + before.abs()))
    assert (buf[keep] == 7).all()


def test_linear_same_bits_every_time_and_rows_on_their_own(ops):
    """Repeated calls give the same bits (fixed summation order)."""
    g = _gen(4)
    xq, xs = _quantised(g, 208, 5120)
    wq, ws = _quantised(g, 1280, 5120, std=0.05)
    first = ops.linear_fp8(xq, xs, wq, ws)
    for _ in range(20):
        assert torch.equal(first, ops.linear_fp8(xq, xs, wq, ws))


def test_linear_nan_stays_in_its_row_and_channel(ops):
    g = _gen(6)
    xq, xs = _quantised(g, 30, 512)
    wq, ws = _quantised(g, 300, 512)
    xs[3] = float("nan")
    xq.view(torch.uint8)[7, 100] = 0x7F   # NaN
    ws[11] = float("inf")
    out = ops.linear_fp8(xq, xs, wq, ws).float()
    bad = torch.zeros(30, 300, dtype=torch.bool, device=DEV)
    bad[3] = bad[7] = True
    bad[:, 11] = True
    assert not torch.isfinite(out[bad]).any() and torch.isfinite(out[~bad]).all()


def test_weights_quantised_just_before_the_projection(ops):
    """The projection may start while the quantiser still runs: its weights are read after it."""
    g = _gen(9)
    xq, xs = _quantised(g, 4, 5120)
    ws = [_rand(g, 8192, 5120, std=0.02) for _ in range(3)]
    q, s = torch.empty(8192, 5120, device=DEV, dtype=E4M3), torch.empty(8192, device=DEV)
    outs = []
    for w in ws:
        ops.quant_fp8(w, out=q, scale=s)
        outs.append(ops.linear_fp8(xq, xs, q, s))
    torch.cuda.synchronize()
    for w, o in zip(ws, outs):
        q2, s2 = ops.quant_fp8(w)
        torch.cuda.synchronize()
        assert torch.equal(o, ops.linear_fp8(xq, xs, q2, s2))


def test_wait_limit_reports_and_recovers(ops):
    """A wait limit that a call of tens of microseconds cannot meet: it ends, the status is reported, the
    next call is right.  (A poll of the barrier itself lasts microseconds, so a small call may meet any limit.)"""
    from tri_sds_b200 import _lib
    lib = _lib.load()
    g = _gen(10)
    xq, xs = _quantised(g, 26, 5120)
    wq, ws = _quantised(g, 51200, 5120, std=0.05)
    want = ops.linear_fp8(xq, xs, wq, ws)
    limit = lib.tsds_get_wait_limit_ns()
    try:
        lib.tsds_set_wait_limit_ns(1)
        ops.linear_fp8(xq, xs, wq, ws)
        with pytest.raises(RuntimeError, match="timed out"):
            ops.check_status()
    finally:
        lib.tsds_set_wait_limit_ns(limit)
    assert torch.equal(want, ops.linear_fp8(xq, xs, wq, ws))
    ops.check_status()


# -- together ------------------------------------------------------------------------

def _block(ops, st, x, res):
    """A decoder layer's MLP over 8-bit weights with per-request adapters on the down projection."""
    q, s, res = ops.add_rms_norm_fp8(x, st["norm"], residual=res)
    h = ops.linear_swiglu_fp8(q, s, *st["gate_up"])
    hq, hs = ops.quant_fp8(h)
    out = ops.linear_residual_fp8(hq, hs, *st["down"], res)
    ops.lora_add(out, h, st["a"], st["b"], st["adapter"], scale=st["scale"], ranks=st["ranks"], out=out)
    return q, s, res, h, hq, hs, out


def _block_state(ops, g, M, N, I, R, n_ad):
    st = {"norm": _rand(g, N, std=0.1) + 1, "gate_up": ops.quant_fp8(_rand(g, 2 * I, N, std=0.02)),
          "down": ops.quant_fp8(_rand(g, N, I, std=0.02)), "a": _rand(g, n_ad, R, I, std=I ** -0.5),
          "b": _rand(g, n_ad, N, R, std=0.1), "scale": torch.rand(n_ad, device=DEV, generator=g) + 0.5,
          "ranks": torch.tensor([max(1, R >> (i % 3)) for i in range(n_ad)], dtype=torch.int32, device=DEV)}
    st["adapter"] = torch.tensor([(m // 5) % (n_ad + 1) - 1 for m in range(M)], dtype=torch.int32, device=DEV)
    return st


@pytest.mark.parametrize("M", [1, 26, 208])
def test_quantised_mlp_block_with_adapters(ops, M):
    """Each step of the block against its definition on the device's own inputs of that step."""
    g = _gen(M)
    N, I, R, n_ad = 640, 1280, 32, 3
    st = _block_state(ops, g, M, N, I, R, n_ad)
    x, r0 = _rand(g, M, N), _rand(g, M, N, std=4.0)
    q, s, res, h, hq, hs, out = _block(ops, st, x, r0)
    _check_norm(x, r0, st["norm"], 1e-6, q, s, res, None)
    acc, err = ref.linear(q, s, *st["gate_up"])
    ref.check_bf16(h, *ref.silu_mul(acc[:, :I], err[:, :I], acc[:, I:], err[:, I:]))
    ref.check_quant(hq, hs, h.double(), 2 * ref.F32)
    acc, err = ref.linear(hq, hs, *st["down"])
    proj = ops.linear_residual_fp8(hq, hs, *st["down"], res)
    ref.check_bf16(proj, acc + res.double(), err + ref.F32 * (acc.abs() + res.double().abs()))
    ref.check_bf16(out, *ref.lora(proj, h, st["a"], st["b"], st["adapter"], st["scale"], st["ranks"], None))
    ops.check_status()


def test_block_captured_and_replayed_on_a_side_stream(ops):
    """The block in a CUDA graph, replayed on other inputs, gives the eager bits; a second
    graph of the same operators shares nothing with it."""
    g = _gen(77)
    M, N, I = 26, 640, 1280
    st = _block_state(ops, g, M, N, I, 16, 4)
    xs = [(_rand(g, M, N), _rand(g, M, N)) for _ in range(4)]
    want = [_block(ops, st, *p)[-1].clone() for p in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        bx, br = xs[0][0].clone(), xs[0][1].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = _block(ops, st, bx, br)[-1]
        graphs.append((graph, bx, br, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(len(xs)):
        for k, (graph, bx, br, out) in enumerate(graphs):     # both at once, on different inputs
            p = xs[(i + k) % len(xs)]
            with torch.cuda.stream(streams[k]):
                bx.copy_(p[0])
                br.copy_(p[1])
                graph.replay()
        torch.cuda.synchronize()
        for k, (_, _, _, out) in enumerate(graphs):
            assert torch.equal(out, want[(i + k) % len(xs)]), (i, k)
    ops.check_status()


def test_torch_ops_give_the_ops_bits(ops):
    import tri_sds_b200.torch_ops  # noqa: F401
    tsds = torch.ops.tsds
    g = _gen(21)
    x, r, w = _rand(g, 26, 640), _rand(g, 26, 640), _rand(g, 640)
    no = torch.empty_like(x)
    want = ops.add_rms_norm_fp8(x, w, residual=r, norm_out=no)
    got = tsds.add_rms_norm_fp8(x, r, w)
    for a, b in zip(got, (*want, no)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    wq, ws = tsds.quant_fp8(_rand(g, 1280, 640))
    q, s = got[0], got[1]
    assert torch.equal(tsds.linear_fp8(q, s, wq, ws), ops.linear_fp8(q, s, wq, ws))
    assert torch.equal(tsds.linear_swiglu_fp8(q, s, wq, ws), ops.linear_swiglu_fp8(q, s, wq, ws))
    res = _rand(g, 26, 1280)
    assert torch.equal(tsds.linear_residual_fp8(q, s, wq, ws, res), ops.linear_residual_fp8(q, s, wq, ws, res))
    a, b = _rand(g, 3, 32, 640), _rand(g, 3, 1280, 16)
    ad = torch.tensor([m % 4 - 1 for m in range(26)], dtype=torch.int32, device=DEV)
    assert torch.equal(tsds.lora_add(res, x, a, b, ad, None, None, [1024, 256]),
                       ops.lora_add(res, x, a, b, ad, slices=[1024, 256]))
