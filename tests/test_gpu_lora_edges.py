"""GPU checks of the per-request adapters at the ends of their ranges."""
import pytest
import torch

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
