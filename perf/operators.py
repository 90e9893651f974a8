"""What is measured of the operators around the experts: the residual's addition with RMSNorm
and 8-bit rows (``add_rms_norm``), products grouped by expert over bf16 or e4m3 banks
(``grouped_matmul``), SwiGLU into 8-bit rows (``swiglu_e4m3``) and the low-rank adapters of many
requests beside a projection (``lora_add``).

``run`` computes an operator in its plain form (elementary torch operations in float32) or, with
``own`` set, through the framework's entry point.  ``exact`` gives the same outputs in float64.
"""
import math
import os
import sys

import torch

own = False

E4M3_MAX = 448.0
TINY = 2.0 ** -126          # the smallest scale of a row: the smallest normal float32


def _vxmoe():
    """The framework's package, which lies in a folder of the repository; a program imports it once."""
    if "vxmoe" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "veystrix-core_b200"))
        import vxmoe  # noqa: F401
    return sys.modules["vxmoe"]


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # the norm before one layer's experts while one request decodes: the router reads bf16,
        # the experts read e4m3; latency is all there is
        dict(name="norm_decode_1", op="norm", tokens=1, width=2048, residual="bf16", output="both"),
        # a short prompt with a float32 residual stream and a width no vector divides
        dict(name="norm_odd_777", op="norm", tokens=777, width=1001, residual="f32", output="e4m3"),
        # a long prompt of the wider layer the loader reads (hidden size 2560)
        dict(name="norm_prefill_16384", op="norm", tokens=16384, width=2560, residual="bf16", output="both"),
        # between the two products of the experts, 64 decoding requests with 10 experts each
        dict(name="swiglu_decode_640", op="swiglu", rows=640, inner=512, halves=True),
        # the same for an 8,192-token prompt, experts of 640 wide
        dict(name="swiglu_prefill_81920", op="swiglu", rows=81920, inner=640, halves=True),
        # one decoding request: ten experts' gate and up rows, 8-bit, one row each
        dict(name="grouped_decode_1", op="grouped", kind="e4m3", tokens=1, slots=10, experts=512, inner=2048,
             outer=1024, gather=True, skew=False),
        # 64 decoding requests over unquantised experts: about 366 banks stream through once
        dict(name="grouped_decode_64", op="grouped", kind="bf16", tokens=64, slots=10, experts=512, inner=2048,
             outer=1024, gather=True, skew=False),
        # a 2,048-token prompt, 8-bit, about 40 rows an expert
        dict(name="grouped_prefill_2048", op="grouped", kind="e4m3", tokens=2048, slots=10, experts=512, inner=2048,
             outer=1024, gather=True, skew=False),
        # one of eight expert-parallel shards on a long prompt, with hot experts: rows already sorted
        dict(name="grouped_shard_40960", op="grouped", kind="bf16", tokens=40960, slots=1, experts=64, inner=2048,
             outer=1024, gather=False, skew=True),
        # one decoding request with an adapter beside a square projection
        dict(name="lora_decode_1", op="lora", tokens=1, inner=2048, outer=2048, adapters=8, rank=16, runs=False,
             ragged=False),
        # 64 decoding requests of 32 tenants, ranks as the tenants chose them
        dict(name="lora_decode_64", op="lora", tokens=64, inner=2048, outer=4096, adapters=32, rank=64, runs=False,
             ragged=True),
        # prompts of a few tenants packed one after the other
        dict(name="lora_prefill_8192", op="lora", tokens=8192, inner=2048, outer=4096, adapters=6, rank=32, runs=True,
             ragged=True),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over their logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "grouped", "grouped", "lora"])
    if op == "norm":
        width = _log(rng, 33, 16384)
        width = width if rng.random() < 0.4 else max(64, width // 8 * 8)
        tokens = _log(rng, 1, max(1, min(16384, 16384 * 2560 // width)))
        return dict(op=op, tokens=tokens, width=width, residual=rng.choice(["bf16", "f32", "none"]),
                    output=rng.choice(["bf16", "e4m3", "both"]))
    if op == "swiglu":
        inner = _log(rng, 17, 8192)
        inner = inner if rng.random() < 0.4 else max(32, inner // 8 * 8)
        return dict(op=op, rows=_log(rng, 1, max(1, min(81920, 81920 * 640 // inner))), inner=inner,
                    halves=rng.random() < 0.5)
    if op == "grouped":
        kind = rng.choice(["bf16", "e4m3"])
        experts, inner = _log(rng, 1, 512), _log(rng, 2, 256) * 16
        most = (512 * 1024 * 2048 // (1 if kind == "e4m3" else 2)) // (experts * inner)
        outer = _log(rng, 8, max(8, min(4096, most)))
        slots = min(experts, rng.choice([1, 2, 8, 10]))
        tokens = _log(rng, 1, max(1, min(40960, 40960 * 1024 * 2048 // (inner * outer)) // slots))
        return dict(op=op, kind=kind, tokens=tokens, slots=slots, experts=experts, inner=inner, outer=outer,
                    gather=slots > 1 or rng.random() < 0.5, skew=rng.random() < 0.4 and experts >= 16)
    tokens = _log(rng, 1, 8192)
    inner = _log(rng, 16, 512) * 8
    outer = _log(rng, 65, 4096)
    return dict(op=op, tokens=tokens, inner=inner, outer=outer if rng.random() < 0.3 else outer // 8 * 8,
                adapters=_log(rng, 1, 64), rank=8 * _log(rng, 1, 16), runs=rng.random() < 0.5,
                ragged=rng.random() < 0.6)


def work(case):
    op = case["op"]
    if op == "norm":
        t, d = case["tokens"], case["width"]
        res = {"bf16": 2, "f32": 4, "none": 0}[case["residual"]]
        out = {"bf16": 2, "e4m3": 1, "both": 3}[case["output"]]
        rows = 4 * t if case["output"] != "bf16" else 0
        return {"bytes": t * d * (2 + 2 * res + out) + 2 * d + rows, "flops": 7 * t * d}
    if op == "swiglu":
        p, i = case["rows"], case["inner"]
        return {"bytes": 5 * p * i + 4 * p, "flops": 8 * p * i}
    if op == "grouped":
        e, k, n, t, s = case["experts"], case["inner"], case["outer"], case["tokens"], case["slots"]
        size = 2 if case["kind"] == "bf16" else 1
        used = sum(1 - (1 - min(1.0, s * share)) ** t for share in _shares(case))   # experts that get a row
        scales = 0 if size == 2 else 4 * (t + used * n)
        index = 4 * t * s if case["gather"] else 0
        return {"bytes": size * (used * n * k + t * k) + 2 * t * s * n + scales + index + 4 * (e + 1),
                "flops": 2 * t * s * n * k}
    t, k, n, count = case["tokens"], case["inner"], case["outer"], case["adapters"]
    rank = (case["rank"] + 1) / 2 if case["ragged"] else case["rank"]
    requests = min(t, 2 * count) if case["runs"] else t
    used = count * (1 - (1 - 0.9 / count) ** requests)
    return {"bytes": 2 * t * (k + 2 * n) + 2 * used * rank * (k + n) + 4 * t, "flops": 2 * 0.9 * t * rank * (k + n)}


def _shares(case):
    """How likely a slot goes to each expert: evenly, or half of all to a sixteenth of them."""
    e = case["experts"]
    if not case["skew"]:
        return [1.0 / e] * e
    hot = max(1, e // 16)
    return [0.5 / hot] * hot + [0.5 / (e - hot)] * (e - hot)


# ---- inputs -----------------------------------------------------------------


def _rows_to_e4m3(v):
    scale = (v.abs().amax(-1) / E4M3_MAX).clamp_min(TINY)
    return (v / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, spread=1.0):
        return torch.randn(shape, device="cuda", generator=gen, dtype=dtype) * spread

    s = dict(case)
    op = case["op"]
    if op == "norm":
        t, d = case["tokens"], case["width"]
        s["x"] = normal(t, d, spread=0.5)
        s["gain"] = 1 + normal(d, spread=0.1)
        s["residual"] = (None if case["residual"] == "none" else
                         normal(t, d, dtype=torch.bfloat16 if case["residual"] == "bf16" else torch.float32,
                                spread=4.0))
        s["eps"] = 1e-6
    elif op == "swiglu":
        p, i = case["rows"], case["inner"]
        if case["halves"]:   # one product gives gate and up side by side
            both = normal(p, 2 * i, spread=1.5)
            s["gate"], s["up"] = both[:, :i], both[:, i:]
        else:
            s["gate"], s["up"] = normal(p, i, spread=1.5), normal(p, i, spread=1.5)
    elif op == "grouped":
        t, e, k, n, slots = (case[c] for c in ("tokens", "experts", "inner", "outer", "slots"))
        # distinct experts for each token, drawn without replacement by their shares
        share = torch.tensor(_shares(case), device="cuda")
        noise = torch.rand((t, e), device="cuda", generator=gen).clamp_min(1e-30)
        ids = (noise.log() / share).topk(slots, dim=1).indices.reshape(-1)
        del noise
        order = torch.sort(ids, stable=True)
        counts = torch.bincount(ids, minlength=e)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
        s["rows"] = order.indices.int() if case["gather"] else None
        s["most"] = int(counts.max())    # rows of the largest group, for the plain form's padding
        x = normal(t, k)
        w = normal(e, n, k, spread=0.02)
        if case["kind"] == "e4m3":
            s["x"], s["x_scales"] = _rows_to_e4m3(x.float())
            s["w"] = torch.empty((e, n, k), dtype=torch.float8_e4m3fn, device="cuda")
            s["w_scales"] = torch.empty((e, n), device="cuda")
            for first in range(0, e, 64):
                s["w"][first:first + 64], s["w_scales"][first:first + 64] = _rows_to_e4m3(w[first:first + 64].float())
        else:
            s["x"], s["w"], s["x_scales"], s["w_scales"] = x, w, None, None
    else:
        t, k, n, count, rank = (case[c] for c in ("tokens", "inner", "outer", "adapters", "rank"))
        s["y"], s["x"] = normal(t, n), normal(t, k)
        s["a"] = normal(count, rank, k, spread=k ** -0.5)
        s["b"] = normal(count, n, rank, spread=0.5 * rank ** -0.5)
        s["scales"] = torch.rand(count, device="cuda", generator=gen) * 1.5 + 0.5
        s["ranks"] = (torch.randint(1, rank + 1, (count,), device="cuda", generator=gen, dtype=torch.int32)
                      if case["ragged"] else None)
        # one request in ten has no adapter
        requests = min(t, 2 * count) if case["runs"] else t
        ids = torch.randint(0, count, (requests,), device="cuda", generator=gen, dtype=torch.int32)
        ids[torch.rand(requests, device="cuda", generator=gen) < 0.1] = -1
        s["adapters"] = ids[torch.arange(t, device="cuda") * requests // t] if case["runs"] else ids
    return s


# ---- one pass ---------------------------------------------------------------


def run(state):
    op = state["op"]
    if own:
        vx = _vxmoe()
        if op == "norm":
            return _norm_outputs(*vx.add_rms_norm(state["x"], state["residual"], state["gain"], state["eps"],
                                                  output=state["output"]))
        if op == "swiglu":
            return tuple(vx.swiglu_e4m3(state["gate"], state["up"]))
        if op == "grouped":
            return vx.grouped_matmul(state["x"], state["w"], state["offsets"], rows=state["rows"],
                                     slots=state["slots"], x_scales=state["x_scales"], w_scales=state["w_scales"])
        return vx.lora_add(state["y"], state["x"], state["a"], state["b"], state["adapters"],
                           scales=state["scales"], ranks=state["ranks"])
    return {"norm": _plain_norm, "swiglu": _plain_swiglu, "grouped": _plain_grouped, "lora": _plain_lora}[op](state)


def _norm_outputs(y, residual, q, scales):
    return {"y": y, "residual": residual, "q": q, "scales": scales}


def _plain_norm(s):
    v = s["x"].float()
    residual = None
    if s["residual"] is not None:
        v = v + s["residual"].float()
        residual = v.to(s["residual"].dtype)
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + s["eps"]) * s["gain"].float()
    q, scales = _rows_to_e4m3(v) if s["output"] != "bf16" else (None, None)
    return _norm_outputs(v.bfloat16() if s["output"] != "e4m3" else None, residual, q, scales)


def _plain_swiglu(s):
    g = s["gate"].float()
    return _rows_to_e4m3(g * torch.sigmoid(g) * s["up"].float())


def _plain_grouped(s):
    """Every group padded to the largest one's rows, one batched product, the padding left out."""
    offsets = s["offsets"].long()
    at = offsets[:-1, None] + torch.arange(s["most"], device="cuda")
    real = at < offsets[1:, None]
    at = torch.where(real, at, 0)
    rows = at if s["rows"] is None else s["rows"].long()[at] // s["slots"]
    x = s["x"].float()
    if s["x_scales"] is not None:
        x = x * s["x_scales"][:, None]
    y = torch.bmm(x[rows], s["w"].float().transpose(1, 2))
    if s["w_scales"] is not None:
        y = y * s["w_scales"][:, None, :]
    return y[real].bfloat16()


def _plain_lora(s):
    """All adapters as one wide one; a token's own columns are kept, the others are set to zero."""
    count, rank, inner = s["a"].shape
    h = s["x"].float() @ s["a"].float().reshape(count * rank, inner).T
    column = torch.arange(count * rank, device="cuda")
    mine = s["adapters"][:, None] == column // rank
    if s["ranks"] is not None:
        mine = mine & (column % rank < s["ranks"][column // rank])
    h = torch.where(mine, h * s["scales"][column // rank], 0.0)
    return (s["y"].float() + h @ s["b"].float().permute(0, 2, 1).reshape(count * rank, -1)).bfloat16()


# ---- the definitions in 64 bits ---------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        v = s["x"].double() + (0 if s["residual"] is None else s["residual"].double())
        z = v / ((v * v).sum(-1, keepdim=True) / v.shape[-1] + s["eps"]).sqrt() * s["gain"].double()
        scales = z.abs().max(-1).values.div(E4M3_MAX).clamp_min(TINY)
        wide, narrow = case["output"] != "e4m3", case["output"] != "bf16"
        return _norm_outputs(z if wide else None, v if s["residual"] is not None else None,
                             z / scales[:, None] if narrow else None, scales if narrow else None)
    if op == "swiglu":
        g = s["gate"].double()
        z = g / (1 + torch.exp(-g)) * s["up"].double()
        scales = z.abs().max(-1).values.div(E4M3_MAX).clamp_min(TINY)
        return z / scales[:, None], scales
    if op == "grouped":
        bounds = s["offsets"].tolist()
        row = torch.arange(bounds[-1], device="cuda") if s["rows"] is None else s["rows"].long() // case["slots"]
        out = torch.empty((bounds[-1], case["outer"]), dtype=torch.float64, device="cuda")
        for e, (first, last) in enumerate(zip(bounds, bounds[1:])):
            if last > first:
                x, w = s["x"][row[first:last]].double(), s["w"][e].double()
                if case["kind"] == "e4m3":
                    x = x * s["x_scales"][row[first:last]].double()[:, None]
                    w = w * s["w_scales"][e].double()[:, None]
                out[first:last] = x @ w.T
        return out
    out = s["y"].double()
    for i in range(case["adapters"]):
        at = (s["adapters"] == i).nonzero()[:, 0]
        if at.numel():
            r = case["rank"] if s["ranks"] is None else int(s["ranks"][i])
            h = s["x"][at].double() @ s["a"][i, :r].double().T
            out[at] += float(s["scales"][i]) * (h @ s["b"][i, :, :r].double().T)
    return out
