"""GPU checks of the 8-bit operators where numbers, sizes or orders of work are extreme."""
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


def _norm_values(x, w, eps):
    r = x.double()
    return r / torch.sqrt(r.square().mean(dim=1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("n", [512, 40000])
@pytest.mark.parametrize("eps", [1e-6, 1e-12, 1e-20, 1e-38])
def test_norm_of_zero_rows_with_a_small_eps(ops, n, eps):
    """A padding row is zeros whatever eps lifts it by."""
    x = torch.randn(5, n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n)).to(BF)
    x[1] = x[3] = 0
    w = torch.ones(n, device=DEV, dtype=BF)
    no = torch.empty_like(x)
    q, s, _ = ops.add_rms_norm_fp8(x, w, eps=eps, norm_out=no)
    for row in (1, 3):
        assert (q[row].float() == 0).all() and (no[row] == 0).all()
        assert abs(s[row].double().item() / (ref.TINY / ref.TOP) - 1) < 1e-6
    assert torch.isfinite(q.float()).all() and torch.isfinite(s).all()


# The root's relative error is half of the sum's: at n = 512 (64 threads with a vector of 8, 8 warps) at
# most 8 + 5 + 8 additions, so 11 of 2^-24, then the mean, eps, root, reciprocal, the product with the largest value and
# the multiplier: 20 of 2^-24 in all.
RSTD = 20 * ref.F32


@pytest.mark.parametrize("eps,x_exp,w_exp", [(1e-12, -70, -45), (1e-12, -60, -59), (1e-14, -61, -60), (1e-14, -63, -62),
                                             (1e-20, -60, -55), (1e-20, -80, -46), (1e-6, -100, 0), (1e-12, -118, 2)])
def test_norm_of_tiny_rows_with_a_small_eps(ops, eps, x_exp, w_exp):
    """Values around the smallest magnitude a row is scaled to, lifted there by the norm alone."""
    g = torch.Generator(device=DEV).manual_seed(-x_exp)
    n = 512
    x = (torch.ldexp(torch.rand(4, n, device=DEV, generator=g, dtype=torch.float64) - 0.5,
                     torch.tensor(x_exp, device=DEV))).to(BF)
    w = torch.ldexp(torch.rand(n, device=DEV, generator=g, dtype=torch.float64) + 0.5,
                    torch.tensor(w_exp, device=DEV)).to(BF)
    q, s, _ = ops.add_rms_norm_fp8(x, w, eps=eps)
    v, s_ref = ref.quant(_norm_values(x, w, eps))
    assert ((s.double() - s_ref).abs() <= s_ref * RSTD).all()
    # (products below 2^-126 keep at least 2^-149; the largest here are above 2^-130)
    lim = ref.e4m3_step(v) / 2 + v.abs() * RSTD + ref.TOP * 2.0 ** -19
    off = (q.double() - v).abs()
    assert (off <= lim).all(), (off - lim).max()


def test_norm_weights_made_just_before_the_call(ops):
    """The norm may start while the kernel that makes its weights still runs: they are read after it."""
    g = torch.Generator(device=DEV).manual_seed(3)
    n = 5120
    x = torch.randn(4, n, device=DEV, generator=g).to(BF)
    gammas = [torch.randn(n, device=DEV, generator=g).to(BF) for _ in range(4)]
    wq, ws = ops.quant_fp8(torch.randn(n, n, device=DEV, generator=g).to(BF))
    xq, xs = ops.quant_fp8(x)
    w = torch.empty(n, device=DEV, dtype=BF)
    outs = []
    for i in range(40):
        ops.linear_fp8(xq, xs, wq, ws)            # keeps the stream busy
        torch.add(gammas[i % 4], 1.0, out=w)
        outs.append(ops.add_rms_norm_fp8(x, w))
    # the weights from a kernel of the library, which lets its successor start at once
    made = [ops.rms_norm(gammas[i][None], gammas[i])[0].clone() for i in range(4)]
    torch.cuda.synchronize()
    late = []
    for i in range(40):
        ops.rms_norm(gammas[i % 4][None], gammas[i % 4], out=w[None])
        late.append(ops.add_rms_norm_fp8(x, w))
    torch.cuda.synchronize()
    for i in range(4):
        for weights, got in (((gammas[i] + 1.0), outs[i::4]), (made[i], late[i::4])):
            q, s, _ = ops.add_rms_norm_fp8(x, weights.clone())
            torch.cuda.synchronize()
            for gq, gs, _ in got:
                assert torch.equal(gq.view(torch.uint8), q.view(torch.uint8)) and torch.equal(gs, s)


def test_columns_of_one_buffer_side_by_side(ops):
    """Operands and outputs as columns of the same wide rows share no byte and are served; norm_out over x or the
    residual gives the values it gives elsewhere."""
    g = torch.Generator(device=DEV).manual_seed(6)
    M, n = 300, 256
    wide = torch.randn(M, 5 * n, device=DEV, generator=g).to(BF)
    x, r, ro, no, qb = (wide[:, i * n:(i + 1) * n] for i in range(5))
    q = qb.view(E4M3)[:, :n]
    w = torch.randn(n, device=DEV, generator=g).to(BF)
    x0, r0 = x.clone(), r.clone()
    want_no = torch.empty(M, n, device=DEV, dtype=BF)
    want = ops.add_rms_norm_fp8(x0, w, residual=r0, norm_out=want_no)
    s = torch.empty(M, device=DEV)
    ops.add_rms_norm_fp8(x, w, residual=r, res_out=ro, norm_out=no, out=q, scale=s)
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])
    assert torch.equal(ro, want[2]) and torch.equal(no, want_no) and torch.equal(x, x0) and torch.equal(r, r0)
    wq, ws = ops.quant_fp8(torch.randn(n, n, device=DEV, generator=g).to(BF))
    proj = ops.linear_residual_fp8(q, s, wq, ws, r)
    ops.linear_residual_fp8(q, s, wq, ws, r, out=no)
    assert torch.equal(no, proj)
    for n in (256, 40000):
        x0, r0 = torch.randn(9, n, device=DEV, generator=g).to(BF), torch.randn(9, n, device=DEV, generator=g).to(BF)
        w, no = torch.randn(n, device=DEV, generator=g).to(BF), torch.empty(9, n, device=DEV, dtype=BF)
        want = ops.add_rms_norm_fp8(x0, w, residual=r0, norm_out=no)
        for over in range(2):
            xr = [x0.clone(), r0.clone()]
            got = ops.add_rms_norm_fp8(xr[0], w, residual=xr[1], norm_out=xr[over])
            assert torch.equal(xr[over], no) and torch.equal(got[2], want[2]) and torch.equal(got[1], want[1])
            assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))


@pytest.mark.parametrize("kind,M,n,K", [("residual", 208, 5120, 25600), ("store", 200, 10240, 5120), ("swiglu", 208, 25600, 5120),
                                        ("residual", 700, 5120, 8192)])
def test_wait_limit_of_cta_pairs_reports_and_recovers(ops, kind, M, n, K):
    """Above 128 rows two CTAs work on a unit: their waits run out at any moment of a call, the call ends, says so, and
    the next one is right."""
    from tri_sds_b200 import _lib
    lib = _lib.load()
    g = torch.Generator(device=DEV).manual_seed(M + n)
    xq, xs = ops.quant_fp8(torch.randn(M, K, device=DEV, generator=g).to(BF))
    wq, ws = ops.quant_fp8(torch.randn(2 * n if kind == "swiglu" else n, K, device=DEV, generator=g).to(BF))
    res = torch.randn(M, n, device=DEV, generator=g).to(BF)

    def call():
        if kind == "residual":
            return ops.linear_residual_fp8(xq, xs, wq, ws, res)
        return (ops.linear_fp8 if kind == "store" else ops.linear_swiglu_fp8)(xq, xs, wq, ws)
    want = call()
    ops.check_status()
    limit = lib.tsds_get_wait_limit_ns()
    for ns in (1, 500, 2000, 5000, 10000, 20000):
        try:
            lib.tsds_set_wait_limit_ns(ns)
            got = call()
            torch.cuda.synchronize()
        finally:
            lib.tsds_set_wait_limit_ns(limit)
        try:
            ops.check_status()
            assert torch.equal(got, want)    # every wait was met after all
            assert ns > 1
        except RuntimeError as e:
            assert "timed out" in str(e)
        assert torch.equal(call(), want)
        ops.check_status()


def _norm_tolerance(rows, n):
    """What the scale of a normalised row may be off by: the longest chain of additions of its squares (a thread's
    vectors of 8, five steps within a warp, the warps one after another; each off by 2^-24 of the sum, which the root
    halves together with the mean's and eps's rounding), then root, reciprocal, the product with the largest
    value and the division by 448."""
    if n <= 8192:
        threads = 256
    elif rows < 2 * 148 or n > 32768:
        threads = 1024
    else:
        threads = 512
    additions = 8 * -(-(n // 8) // threads) + 5 + threads // 32
    return ((additions + 2) / 2 + 4) * ref.F32 * (1 + 2.0 ** -10)


@pytest.mark.parametrize("rows,n", [(1, 16), (26, 5120), (3, 8192), (601, 8208), (601, 16384), (601, 16400), (601, 32768),
                                    (601, 32784), (2, 12288), (5, 32768), (2, 40000), (2, 262144)])
def test_norm_scales_within_their_additions(ops, rows, n):
    g = torch.Generator(device=DEV).manual_seed(rows + n)
    x, r = (torch.randn(rows, n, device=DEV, generator=g).to(BF) for _ in range(2))
    w = (1 + 0.2 * torch.randn(n, device=DEV, generator=g)).to(BF)
    q, s, ro = ops.add_rms_norm_fp8(x, w, residual=r)
    assert torch.equal(ro, (x.float() + r.float()).to(BF))
    ref.check_quant(q, s, _norm_values(ro, w, 1e-6), _norm_tolerance(rows, n))


@pytest.mark.parametrize("kind", ["store", "residual", "swiglu"])
@pytest.mark.parametrize("M,n,K", [(208, 1280, 5120), (40, 333, 528)])
def test_rows_of_a_batch_on_their_own(ops, kind, M, n, K):
    """A request's rows alone and inside a batch: other launch shapes, the same definition."""
    g = torch.Generator(device=DEV).manual_seed(M)
    xq, xs = ops.quant_fp8(torch.randn(M, K, device=DEV, generator=g).to(BF))
    wq, ws = ops.quant_fp8(torch.randn(2 * n if kind == "swiglu" else n, K, device=DEV, generator=g).to(BF))
    res = torch.randn(M, n, device=DEV, generator=g).to(BF)
    acc, err = ref.linear(xq, xs, wq, ws)
    if kind == "residual":
        acc, err = acc + res.double(), err + ref.F32 * (acc.abs() + res.double().abs())
    elif kind == "swiglu":
        acc, err = ref.silu_mul(acc[:, :n], err[:, :n], acc[:, n:], err[:, n:])
    for lo, hi in ((0, M), (0, 1), (M - 1, M), (7, 33), (3, 36)):
        a = (xq[lo:hi], xs[lo:hi], wq, ws)
        if kind == "residual":
            got = ops.linear_residual_fp8(*a, res[lo:hi])
        else:
            got = (ops.linear_fp8 if kind == "store" else ops.linear_swiglu_fp8)(*a)
        ref.check_bf16(got, acc[lo:hi], err[lo:hi])


def _exact_quant(x):
    """Rows of bf16 to the nearest e4m3 of x * 448 / max|x|, ties to even, without a rounding: |x| * 448 and a
    midpoint times max|x| have at most 17 and 13 significant bits, so fp64 compares them exactly."""
    a = x.double().abs()
    top = a.amax(dim=1, keepdim=True)
    v = a * ref.TOP / top * (1 - 2.0 ** -50)      # never above the value's grid cell
    step = ref.e4m3_step(v)
    lo = torch.floor(v / step)
    num, mid = a * ref.TOP, (lo + 0.5) * step * top
    up = (num > mid) | ((num == mid) & (lo % 2 == 1))
    return torch.copysign((lo + up) * step, x.double())


@pytest.mark.parametrize("rows,n", [(26, 25600), (1000, 5120), (513, 8208), (3, 32784)])
def test_quantiser_is_exact(ops, rows, n):
    """Every value, on rows with a few channels tens of times larger as a residual stream has them."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, n, device=DEV, generator=g)
    x[:, torch.randint(0, n, (n // 512,), device=DEV, generator=g)] *= 30.0
    x = x.to(BF)
    q, _ = ops.quant_fp8(x)
    assert torch.equal(q.double(), _exact_quant(x))
