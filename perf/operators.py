"""The operators of a quantised projection with per-request adapters, measured.

Four operators of a decoder layer that serves many requests over one 8-bit model:

  norm    residual addition + RMSNorm + e4m3 output with one scale per row
  quant   rows to e4m3 with one scale per row (weights once, activations each pass)
  linear  8-bit projection with row and channel scales: plain, + residual, SwiGLU
  lora    low-rank adapters of many requests added beside a shared projection

``run`` computes their plain form (fp32 torch operations) or, where ``own`` is true,
calls the framework's operators.
"""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
TOP = 448.0             # largest e4m3 value
TINY = 2.0 ** -100      # rows whose largest magnitude is below this are quantised against it
EPS = 1e-6


def listed():
    return [
        # a single-token decode step of one request at hidden 5120: latency only
        {"name": "norm_token", "op": "norm", "rows": 1, "n": 5120, "res": True, "norm_out": False},
        # a prompt's rows, the bf16 norm kept for the adapters beside the projection
        {"name": "norm_prompt", "op": "norm", "rows": 4096, "n": 5120, "res": True, "norm_out": True},
        # the SwiGLU output of one 26-node tree verify, before the down projection
        {"name": "quant_tree_down", "op": "quant", "rows": 26, "n": 25600},
        # a q/k/v weight matrix quantised at load
        {"name": "quant_weight", "op": "quant", "rows": 10240, "n": 5120},
        # q/k/v projection of a single token
        {"name": "linear_token_qkv", "op": "linear", "kind": "store", "rows": 1, "n": 10240, "k": 5120},
        # odd sizes: ragged rows, outputs off every tile, k off the 128-byte block
        {"name": "linear_odd", "op": "linear", "kind": "store", "rows": 37, "n": 1003, "k": 2576},
        # gate/up of one 26-node tree verify
        {"name": "linear_tree_gate_up", "op": "linear", "kind": "swiglu", "rows": 26, "n": 25600, "k": 5120},
        # down projection + residual of eight trees
        {"name": "linear_batch_down", "op": "linear", "kind": "residual", "rows": 208, "n": 5120, "k": 25600},
        # q/k/v projection of a prompt
        {"name": "linear_prompt_qkv", "op": "linear", "kind": "store", "rows": 2048, "n": 10240, "k": 5120},
        # q/k/v adapters of eight requests, one token each
        {"name": "lora_token_qkv", "op": "lora", "seqs": 8, "per_seq": 1, "adapters": 8, "rank": 16, "k": 5120,
         "q": 8192, "kv": 1024, "ragged": False},
        # down-projection adapters of eight requests' trees, ranks 64 / 32 / 16
        {"name": "lora_tree_down", "op": "lora", "seqs": 8, "per_seq": 26, "adapters": 8, "rank": 64, "k": 25600,
         "q": 5120, "kv": 0, "ragged": True},
        # q/k/v adapters of four prompts
        {"name": "lora_prompt_qkv", "op": "lora", "seqs": 4, "per_seq": 512, "adapters": 4, "rank": 32, "k": 5120,
         "q": 8192, "kv": 1024, "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quant", "linear", "linear", "linear", "lora", "lora"])
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 4096), "n": 16 * _log(rng, 16, 320), "res": rng.random() < 0.8,
                "norm_out": rng.random() < 0.5}
    if op == "quant":
        n = 16 * _log(rng, 16, 1600)
        return {"op": op, "rows": min(_log(rng, 1, 10240), 52428800 // n), "n": n}
    if op == "linear":
        n, k = _log(rng, 64, 25600), 16 * _log(rng, 16, 1600)
        n = max(64, min(n, 131072000 // k))
        rows = max(1, min(_log(rng, 1, 2048), 107374182400 // (2 * n * k)))
        return {"op": op, "kind": rng.choice(["store", "residual", "swiglu"]), "rows": rows, "n": n, "k": k}
    kv = 32 * _log(rng, 4, 32) if rng.random() < 0.5 else 0
    q = 32 * _log(rng, 4, 256) if kv else 8 * _log(rng, 16, 1024)
    seqs = _log(rng, 1, 32)
    return {"op": op, "seqs": seqs, "per_seq": _log(rng, 1, 2048 // seqs), "adapters": _log(rng, 1, 16),
            "rank": rng.choice([8, 16, 24, 32, 48, 64, 128]), "k": 16 * _log(rng, 16, 512), "q": q, "kv": kv,
            "ragged": rng.random() < 0.5}


def _ranks(case):
    return [max(1, case["rank"] >> (a % 3)) if case["ragged"] else case["rank"] for a in range(case["adapters"])]


def _activations(gen, rows, n):
    """Hidden states: unit rows with a few channels tens of times larger, as a residual stream has them."""
    x = torch.randn(rows, n, device="cuda", generator=gen)
    big = torch.randint(0, n, (max(1, n // 512),), device="cuda", generator=gen)
    x[:, big] *= 30.0
    return x.to(torch.bfloat16)


def _quantised(x):
    s = x.abs().amax(dim=1).clamp_min(TINY) / TOP
    return (x / s[:, None]).to(E4M3), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if op == "norm":
        rows, n = case["rows"], case["n"]
        st["x"] = (torch.randn(rows, n, device="cuda", generator=gen) * 0.5).to(torch.bfloat16)
        st["res"] = _activations(gen, rows, n) if case["res"] else None
        st["w"] = (1.0 + 0.1 * torch.randn(n, device="cuda", generator=gen)).to(torch.bfloat16)
        st["norm_out"] = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda") if case["norm_out"] else None
    elif op == "quant":
        st["x"] = _activations(gen, case["rows"], case["n"])
    elif op == "linear":
        m, n, k, kind = case["rows"], case["n"], case["k"], case["kind"]
        st["xq"], st["xs"] = _quantised(_activations(gen, m, k).float())
        w = torch.randn(2 * n if kind == "swiglu" else n, k, device="cuda", generator=gen) * 0.02
        st["wq"], st["ws"] = _quantised(w)
        st["res"] = _activations(gen, m, n) if kind == "residual" else None
    else:
        m, k, rank, na = case["seqs"] * case["per_seq"], case["k"], case["rank"], case["adapters"]
        slices = [case["q"], case["kv"], case["kv"]] if case["kv"] else [case["q"]]
        n = sum(slices)
        st["slices"] = slices
        st["x"] = torch.randn(m, k, device="cuda", generator=gen).to(torch.bfloat16)
        st["y"] = torch.randn(m, n, device="cuda", generator=gen).to(torch.bfloat16)
        st["a"] = (torch.randn(na, len(slices) * rank, k, device="cuda", generator=gen) * k ** -0.5).to(torch.bfloat16)
        st["b"] = (torch.randn(na, n, rank, device="cuda", generator=gen) * 0.1).to(torch.bfloat16)
        st["scale"] = 0.5 + torch.rand(na, device="cuda", generator=gen)
        st["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32, device="cuda")
        # requests take the adapters in turn, from a start of their own; one in eight has none
        first = int(torch.randint(0, na, (1,), device="cuda", generator=gen))
        seq = torch.arange(case["seqs"], device="cuda")
        of_seq = torch.where(seq % 8 == 7, -1, (seq + first) % na)
        st["adapter"] = of_seq.repeat_interleave(case["per_seq"]).to(torch.int32)
    return st


def work(case):
    op = case["op"]
    if op == "norm":
        r, n = case["rows"], case["n"]
        per = 2 + 1 + (4 if case["res"] else 0) + (2 if case["norm_out"] else 0)
        return {"bytes": r * (n * per + 4) + 2 * n, "flops": 8 * r * n}
    if op == "quant":
        r, n = case["rows"], case["n"]
        return {"bytes": r * (3 * n + 4), "flops": 3 * r * n}
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        w = 2 * n if case["kind"] == "swiglu" else n
        out = m * n * (4 if case["kind"] == "residual" else 2)
        return {"bytes": w * k + m * k + out + 4 * (m + w), "flops": 2 * m * w * k}
    m, k = case["seqs"] * case["per_seq"], case["k"]
    s = 3 if case["kv"] else 1
    n = case["q"] + 2 * case["kv"]
    with_one = case["seqs"] - case["seqs"] // 8
    used = sorted(_ranks(case))[:min(case["adapters"], with_one)]
    per_rank = s * k + n
    rows = with_one * case["per_seq"]
    mean = sum(used) / len(used)
    return {"bytes": rows * k * 2 + m * n * 4 + sum(used) * per_rank * 2 + 4 * m, "flops": 2 * rows * mean * per_rank}


# -- plain form --------------------------------------------------------------------

def _plain_quant(y):
    s = torch.clamp_min(y.abs().amax(dim=1), TINY) / TOP
    return torch.clamp(y / s[:, None], -TOP, TOP).to(E4M3), s


def _plain_norm(st):
    h = st["x"].float()
    res = None
    if st["res"] is not None:
        res = (h + st["res"].float()).to(torch.bfloat16)
        h = res.float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * st["w"].float()
    q, s = _plain_quant(y)
    return [q, s] + ([res] if res is not None else []) + ([y.to(torch.bfloat16)] if st["norm_out"] is not None else [])


def _plain_linear(st):
    kind = st["case"]["kind"]
    acc = (st["xq"].float() @ st["wq"].float().t()) * st["xs"][:, None] * st["ws"][None, :]
    if kind == "residual":
        acc = st["res"].float() + acc
    if kind == "swiglu":
        g, u = acc.chunk(2, dim=1)
        acc = g / (1.0 + torch.exp(-g)) * u
    return acc.to(torch.bfloat16)


def _plain_lora(st):
    case = st["case"]
    na, rank, s = case["adapters"], case["rank"], len(st["slices"])
    m = st["x"].shape[0]
    t = (st["x"].float() @ st["a"].float().reshape(-1, case["k"]).t()).reshape(m, na, s, rank)
    mine = st["adapter"][:, None] == torch.arange(na, device="cuda")
    used = torch.arange(rank, device="cuda") < st["ranks"][:, None]
    t = torch.where((mine[:, :, None] & used)[:, :, None, :], t * st["scale"][None, :, None, None], 0.0)
    b = torch.where(used[:, None, :], st["b"].float(), 0.0).split(st["slices"], dim=1)
    delta = torch.cat([torch.einsum("mar,anr->mn", t[:, :, i], b[i]) for i in range(s)], dim=1)
    return (st["y"].float() + delta).to(torch.bfloat16)


def _own(st):
    from tri_sds_b200 import ops
    case = st["case"]
    if case["op"] == "norm":
        q, s, res = ops.add_rms_norm_fp8(st["x"], st["w"], residual=st["res"], eps=EPS, norm_out=st["norm_out"])
        return [q, s] + ([res] if res is not None else []) + ([st["norm_out"]] if st["norm_out"] is not None else [])
    if case["op"] == "quant":
        return list(ops.quant_fp8(st["x"]))
    if case["op"] == "lora":
        return ops.lora_add(st["y"], st["x"], st["a"], st["b"], st["adapter"], scale=st["scale"], ranks=st["ranks"],
                            slices=st["slices"])
    if case["kind"] == "residual":
        return ops.linear_residual_fp8(st["xq"], st["xs"], st["wq"], st["ws"], st["res"])
    if case["kind"] == "swiglu":
        return ops.linear_swiglu_fp8(st["xq"], st["xs"], st["wq"], st["ws"])
    return ops.linear_fp8(st["xq"], st["xs"], st["wq"], st["ws"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "quant":
        return list(_plain_quant(state["x"].float()))
    return _plain_linear(state) if op == "linear" else _plain_lora(state)


# -- from the definition, in 64 bits -----------------------------------------------

def _e4m3_64(v):
    """The e4m3 value nearest to v (ties to even): 3 mantissa bits, exponents from -6, at most 448."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp_min(e - 1, -6) - 3)
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _quant_64(y):
    s = torch.maximum(y.abs().max(dim=1).values, torch.full((), TINY, dtype=y.dtype, device=y.device)) / TOP
    return [_e4m3_64(y / s.unsqueeze(1)), s]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        r = st["x"].double()
        out = []
        if st["res"] is not None:
            out = [r + st["res"].double()]
            r = out[0].to(torch.bfloat16).double()     # the residual stream is held in bf16
        y = r / torch.sqrt(r.square().sum(dim=1, keepdim=True) / case["n"] + EPS) * st["w"].double()
        return _quant_64(y) + out + ([y] if st["norm_out"] is not None else [])
    if op == "quant":
        return _quant_64(st["x"].double())
    if op == "linear":
        acc = torch.mm(st["xq"].double() * st["xs"].double()[:, None], (st["wq"].double() * st["ws"].double()[:, None]).t())
        if case["kind"] == "residual":
            return acc + st["res"].double()
        if case["kind"] == "swiglu":
            g, u = acc[:, :case["n"]], acc[:, case["n"]:]
            return g * torch.sigmoid(g) * u
        return acc
    out = st["y"].double()
    for a, r in enumerate(_ranks(case)):
        rows = (st["adapter"] == a).nonzero()[:, 0]
        x, at = st["x"][rows].double(), 0
        for i, width in enumerate(st["slices"]):
            first = i * case["rank"]
            t = x @ st["a"][a, first:first + r].double().t()
            out[rows, at:at + width] += st["scale"][a].double() * (t @ st["b"][a, at:at + width, :r].double().t())
            at += width
    return out
