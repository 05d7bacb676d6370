"""GPU checks of the per-request adapters at the ends of their ranges: infinities, numbers at bf16's end,
adapters that change between calls."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from tri_sds_b200 import ops as o
    yield o
    o.check_status()


def _case(M, R, used, seed=0, K=264, slices=(96, 160), n_ad=3):
    g = torch.Generator(device=DEV).manual_seed(seed + M + R)

    def rnd(*shape, std=1.0):
        v = torch.randn(*shape, device=DEV, generator=g) * std
        return torch.where(v.abs() < 1e-3, 1e-3, v).to(BF)   # no zero: an infinity times one would be NaN
    N = sum(slices)
    return dict(y=rnd(M, N), x=rnd(M, K), lora_a=rnd(n_ad, len(slices) * R, K, std=K ** -0.5), lora_b=rnd(n_ad, N, R, std=0.1),
                adapter=torch.tensor([m % (n_ad + 1) - 1 for m in range(M)], dtype=torch.int32, device=DEV),
                scale=torch.rand(n_ad, device=DEV, generator=g) + 0.5,
                ranks=torch.full((n_ad,), used, dtype=torch.int32, device=DEV), slices=list(slices))


def _check(ops, st):
    want, err = ref.lora(st["y"], st["x"], st["lora_a"], st["lora_b"], st["adapter"], st["scale"], st["ranks"], st["slices"])
    got = ops.lora_add(**st)
    fin = torch.isfinite(want)
    assert not fin.all()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got.double()[inf], want[inf])
    ref.check_bf16(got[fin], want[fin], err[fin])


# one launch and two; ranks that end inside and at the end of 8 and 16
SIZES = [(M, R, used) for M in (7, 40, 600, 1100) for R, used in ((8, 1), (16, 1), (16, 2), (24, 9), (64, 64), (128, 65))]


@pytest.mark.parametrize("M,R,used", SIZES)
def test_infinite_activation(ops, M, R, used):
    st = _case(M, R, used)
    st["x"][2, 100] = float("inf")
    st["x"][5, 263] = float("-inf")
    _check(ops, st)


@pytest.mark.parametrize("M,R,used", SIZES)
def test_infinite_scale_and_first_matrix(ops, M, R, used):
    st = _case(M, R, used, seed=1)
    st["scale"][1] = float("inf")
    st["lora_a"][2, 0, 17] = float("-inf")
    _check(ops, st)


@pytest.mark.parametrize("M,R", [(7, 8), (40, 64), (600, 24), (1100, 128)])
def test_first_product_between_the_largest_bf16_and_fp32(ops, M, R):
    """A first product that bf16 would round to an infinity: its two words still hold it."""
    st = _case(M, R, 1, seed=2)
    st["x"].zero_()
    st["lora_a"].zero_()
    st["lora_b"].fill_(2.0 ** -20)
    st["x"][:, 3] = 2.0 ** 64
    for s in range(2):
        st["lora_a"][:, s * R, 3] = 255 * 2.0 ** 56        # t = 255/256 2^128
    st["scale"][:] = 1 + 511 * 2.0 ** -17                  # times that: below 2^128 in fp32, 2^128 in bf16
    t = (torch.tensor(255 * 2.0 ** 120, device=DEV) * st["scale"][0])
    assert torch.isfinite(t) and torch.isinf(t.to(BF))
    want, err = ref.lora(st["y"], st["x"], st["lora_a"], st["lora_b"], st["adapter"], st["scale"], st["ranks"], st["slices"])
    ref.check_bf16(ops.lora_add(**st), want, err)


@pytest.mark.parametrize("M", [4, 40, 400, 1200])
def test_adapter_written_just_before_the_call(ops, M):
    """A slot of the adapters overwritten on the stream right before each call."""
    sts = [_case(M, 16, 16, seed=10 + i) for i in range(3)]
    want = [ops.lora_add(**st) for st in sts]
    live = {k: v.clone() if torch.is_tensor(v) else v for k, v in sts[0].items()}
    got = []
    for i in range(24):
        for name in ("y", "x", "lora_a", "lora_b", "scale", "ranks"):
            live[name].copy_(sts[i % 3][name])
        got.append(ops.lora_add(**live))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 3]), i


FIRST = r"""
import sys
import torch
sys.path.insert(0, REPO)
from tri_sds_b200 import ops
y, x = torch.ones(4, 64, device="cuda").bfloat16(), torch.ones(4, 64, device="cuda").bfloat16()
a, b = torch.ones(2, 8, 64, device="cuda").bfloat16(), torch.ones(2, 64, 8, device="cuda").bfloat16()
good = torch.zeros(4, device="cuda", dtype=torch.int32)
bad = torch.full((4,), 7, device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
graphs = []
for ids in (good, bad):          # the process's first calls
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.lora_add(y, x, a, b, ids)
    graphs.append((graph, out))
ops.check_status()
graphs[0][0].replay()
torch.cuda.synchronize()
assert (graphs[0][1] == 1 + 8 * 64).all()
ops.check_status()
graphs[1][0].replay()
graphs[0][0].replay()            # a later replay leaves the report alone
try:
    ops.check_status()
except RuntimeError as e:
    assert "status 10" in str(e)
else:
    raise SystemExit("the report of an index past the last adapter was lost")
graphs[1][0].replay()
ops.lora_add(y, x, a, b, good)
try:
    ops.check_status()
except RuntimeError:
    print("reported")
ops.check_status()
"""


def test_status_of_a_process_whose_first_calls_are_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST.replace("REPO", repr(root))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "reported" in r.stdout, r.stdout + r.stderr
