"""GPU checks of the per-request low-rank adapters against their definition in 64 bits."""
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


def _case(M, K, slices, R, n_ad, adapters, seed=0, scale=True, ranks=True):
    g = torch.Generator(device=DEV).manual_seed(seed + M + K + R)

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * std).to(BF)

    N = sum(slices)
    st = dict(y=rnd(M, N), x=rnd(M, K), lora_a=rnd(n_ad, len(slices) * R, K, std=K ** -0.5),
              lora_b=rnd(n_ad, N, R, std=0.1), adapter=torch.tensor(adapters, dtype=torch.int32, device=DEV),
              slices=slices if len(slices) > 1 else None)
    st["scale"] = torch.rand(n_ad, device=DEV, generator=g) + 0.5 if scale else None
    st["ranks"] = torch.tensor([max(1, R - 3 * i) for i in range(n_ad)], dtype=torch.int32, device=DEV) \
        if ranks else None
    return st


def _check(ops, st, out=None):
    want, err = ref.lora(st["y"], st["x"], st["lora_a"], st["lora_b"], st["adapter"], st["scale"], st["ranks"],
                         st["slices"])
    got = ops.lora_add(out=out, **st)
    ref.check_bf16(got, want, err)
    none = st["adapter"] < 0
    assert torch.equal(got[none], st["y"][none]) if out is not st["y"] else True
    return got


@pytest.mark.parametrize("M,K,slices,R,n_ad", [
    (1, 8, [8], 8, 1), (1, 5120, [1024, 128, 128], 16, 2), (8, 5120, [8192, 1024, 1024], 16, 8), (3, 40, [200], 24, 4),
    (16, 264, [32, 64, 96, 32], 128, 2), (17, 1000, [1000], 48, 3), (26, 2560, [2560], 64, 1), (100, 512, [96, 32], 8, 16),
    (208, 25600, [5120], 64, 8), (1024, 128, [256], 16, 5), (1025, 136, [264], 24, 5), (1500, 640, [640, 128, 128], 32, 4),
    (2100, 72, [96, 96], 128, 3), (40, 264, [32, 64, 96, 32], 128, 2), (130, 1000, [1000], 128, 3),
    (257, 8, [8], 8, 2), (300, 1032, [2560], 64, 20), (520, 5120, [1024, 128, 128], 16, 70), (64, 640, [136], 128, 100), (1000, 264, [96, 32], 32, 3),
    (512, 520, [512], 64, 4), (1030, 5120, [640, 128, 128], 64, 2)])
@pytest.mark.parametrize("order", ["runs", "scattered"])
def test_lora(ops, M, K, slices, R, n_ad, order):
    if order == "runs":      # requests of 5 rows each, every (n_ad + 1)-th without an adapter
        ad = [(m // 5) % (n_ad + 1) - 1 for m in range(M)]
    else:
        g = torch.Generator().manual_seed(M)
        ad = torch.randint(-1, n_ad, (M,), generator=g).tolist()
    _check(ops, _case(M, K, slices, R, n_ad, ad))


@pytest.mark.parametrize("M,K,slices,R,n_ad", [
    (1, 8, [8], 128, 1), (2, 264, [96, 32, 32], 40, 3), (16, 520, [72], 64, 16), (17, 520, [72], 64, 17),
    (31, 5120, [1024, 128, 128], 32, 4), (64, 136, [1000], 64, 64), (65, 1288, [1288], 72, 9),
    (128, 5120, [5120], 16, 16), (200, 16000, [128], 48, 6), (256, 72, [64, 32], 24, 1), (511, 520, [256], 48, 3),
    (513, 264, [264], 8, 3)])
@pytest.mark.parametrize("step", [1, 26, 1000])
def test_lora_between_the_two_forms(ops, M, K, slices, R, n_ad, step):
    """Sizes on either side of the choice between one launch and two; rows that alternate, in runs, of one adapter."""
    _check(ops, _case(M, K, slices, R, n_ad, [(m // step) % n_ad if (m // step) % 5 != 4 else -1 for m in range(M)]))


@pytest.mark.parametrize("M,K,slices,R,n_ad", [
    (3600, 72, [96, 32], 24, 3), (3585, 520, [264], 8, 40), (4100, 264, [32, 64, 96, 32], 40, 130),
    (2048, 136, [160, 32], 128, 5), (150, 264, [1088, 32, 96], 64, 150), (600, 1032, [328], 96, 600)])
@pytest.mark.parametrize("step", [1, 70, 5000])
def test_lora_blocks_of_many_rows(ops, M, K, slices, R, n_ad, step):
    """Blocks of 128 rows with one adapter or up to 128, in and out of place, with and without rows that have none."""
    st = _case(M, K, slices, R, n_ad, [(m // step) % n_ad if (m // step) % 7 != 6 else -1 for m in range(M)])
    want = _check(ops, st)
    y = st["y"].clone()
    assert torch.equal(ops.lora_add(**dict(st, y=y), out=y), want)
    st["adapter"] = st["adapter"].clamp(min=0)
    want = _check(ops, st)
    y = st["y"].clone()
    assert torch.equal(ops.lora_add(**dict(st, y=y), out=y), want)


@pytest.mark.parametrize("M", [40, 1400])
def test_lora_in_place_leaves_other_rows_alone(ops, M):
    st = _case(M, 320, [288, 64], 16, 3, [(m % 4) - 1 for m in range(M)])
    want = _check(ops, st)
    y = st["y"].clone()
    st["y"] = y
    got = ops.lora_add(out=y, **st)
    assert got is y and torch.equal(got, want)


def test_lora_without_scale_and_ranks(ops):
    _check(ops, _case(19, 512, [512], 32, 4, [m % 4 for m in range(19)], scale=False, ranks=False))


@pytest.mark.parametrize("M", [16, 21, 300, 1100])
def test_lora_unused_ranks_are_not_read_into_the_sum(ops, M):
    """NaN past an adapter's rank (in A's rows and in B's columns) changes nothing."""
    for R, used in [(16, 1), (24, 7), (64, 33), (32, 0), (128, 66), (72, 64), (104, 97)]:
        st = _case(M, 264, [96, 160], R, 2, [m % 2 for m in range(M)])
        st["ranks"] = torch.tensor([used, R], dtype=torch.int32, device=DEV)
        for s in range(2):
            st["lora_a"][0, s * R + used:(s + 1) * R] = float("nan")
        st["lora_b"][0, :, used:] = float("inf")
        _check(ops, st)


def test_lora_ranks_out_of_range_are_clamped(ops):
    st = _case(5, 64, [64], 16, 2, [0, 1, 0, 1, -1])
    full = dict(st, ranks=torch.tensor([16, 0], dtype=torch.int32, device=DEV))
    wild = dict(st, ranks=torch.tensor([1000, -5], dtype=torch.int32, device=DEV))
    assert torch.equal(ops.lora_add(**full), ops.lora_add(**wild))


@pytest.mark.parametrize("M", [33, 1300])
def test_lora_index_past_the_last_adapter_is_reported(ops, M):
    ids = [m % 3 for m in range(M)]
    ids[7] = 3
    ids[20] = 2 ** 31 - 1
    st = _case(M, 128, [128], 16, 3, ids)
    got = ops.lora_add(**st)
    assert torch.equal(got[7], st["y"][7]) and torch.equal(got[20], st["y"][20])
    with pytest.raises(RuntimeError, match="status 10"):
        ops.check_status()
    want, err = ref.lora(st["y"], st["x"], st["lora_a"], st["lora_b"], st["adapter"], st["scale"], st["ranks"], None)
    ref.check_bf16(got, want, err)


@pytest.mark.parametrize("M", [30, 390, 1302])
def test_lora_strides_and_neighbours(ops, M):
    g = torch.Generator(device=DEV).manual_seed(2)
    st = _case(M, 256, [128, 64], 16, 3, [(m // (M // 4)) - 1 for m in range(M)])
    wide_x = torch.randn(M, 400, device=DEV, generator=g).to(BF)
    st["x"] = wide_x[:, 64:320]
    wide_y = torch.randn(M, 256, device=DEV, generator=g).to(BF)
    st["y"] = wide_y[:, 32:224]
    buf = torch.full((M + 2, 264), 5.0, device=DEV, dtype=BF)
    _check(ops, st, out=buf[1:M + 1, 8:200])
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[1:M + 1, 8:200] = False
    assert (buf[keep] == 5).all()
    with pytest.raises(RuntimeError, match="status 10"):   # the last rows name adapter 3 of 3
        ops.check_status()


@pytest.mark.parametrize("M", [40, 700])
def test_lora_nothing_to_add(ops, M):
    st = _case(M, 128, [128], 16, 2, [-1] * M)
    assert torch.equal(ops.lora_add(**st), st["y"])
    y = st["y"].clone()
    assert torch.equal(ops.lora_add(**dict(st, y=y, out=y)), st["y"])
    e = _case(0, 128, [128], 16, 2, [])
    assert ops.lora_add(**e).shape == (0, 128)


@pytest.mark.parametrize("M,R", [(208, 64), (1040, 32)])
def test_lora_same_bits_every_time(ops, M, R):
    st = _case(M, 5120, [1024], R, 8, [m // (M // 8) for m in range(M)])
    first = ops.lora_add(**st)
    for _ in range(20):
        assert torch.equal(first, ops.lora_add(**st))


def test_lora_offsets_past_32_bits(ops):
    """An adapter whose rows lie past 2^31 elements of lora_a."""
    K, R, n_ad = 4096, 64, 8200
    a = torch.zeros(n_ad, R, K, device=DEV, dtype=BF)
    assert a.numel() > 2 ** 31
    st = _case(6, K, [64], R, 1, [0] * 6, ranks=False)
    want = ops.lora_add(**st)
    a[-1] = st["lora_a"][0]
    b = torch.zeros(n_ad, 64, R, device=DEV, dtype=BF)
    b[-1] = st["lora_b"][0]
    scale = torch.ones(n_ad, device=DEV)
    scale[-1] = st["scale"][0]
    got = ops.lora_add(st["y"], st["x"], a, b, torch.full((6,), n_ad - 1, dtype=torch.int32, device=DEV), scale=scale)
    assert torch.equal(got, want)


@pytest.mark.parametrize("M", [12, 240, 1200])
def test_lora_streams_and_graphs_share_nothing(ops, M):
    """Two captured calls replayed at once on two streams, on changing inputs, beside eager calls."""
    sts = [_case(M, 640, [512, 128], 32, 4, [(m // 40) % 5 - 1 for m in range(M)], seed=i) for i in range(3)]
    want = [ops.lora_add(**st).clone() for st in sts]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        st = {k: v.clone() if torch.is_tensor(v) else v for k, v in sts[0].items()}
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = ops.lora_add(**st)
        graphs.append((graph, st, out, side))
    torch.cuda.synchronize()
    for i in range(6):
        for k, (graph, st, out, side) in enumerate(graphs):
            with torch.cuda.stream(side):
                for name, v in sts[(i + k) % 3].items():
                    if torch.is_tensor(v):
                        st[name].copy_(v)
                graph.replay()
        eager = ops.lora_add(**sts[(i + 2) % 3])
        torch.cuda.synchronize()
        for k, (_, _, out, _) in enumerate(graphs):
            assert torch.equal(out, want[(i + k) % 3])
        assert torch.equal(eager, want[(i + 2) % 3])


def test_lora_wait_limit_reports_and_recovers(ops):
    """A wait limit that the two-launch form cannot meet: the call ends, the status is reported, the
    next call is right."""
    from tri_sds_b200 import _lib
    lib = _lib.load()
    st = _case(2048, 25600, [512], 64, 4, [m // 512 for m in range(2048)])
    want = ops.lora_add(**st)
    ops.check_status()
    limit = lib.tsds_get_wait_limit_ns()
    try:
        lib.tsds_set_wait_limit_ns(1)
        ops.lora_add(**st)
        with pytest.raises(RuntimeError, match="timed out"):
            ops.check_status()
    finally:
        lib.tsds_set_wait_limit_ns(limit)
    assert torch.equal(want, ops.lora_add(**st))
    ops.check_status()
