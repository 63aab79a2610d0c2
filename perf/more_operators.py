"""Layers on 8-bit weights and by experts, and sampling, as timed cases.

``mlir_edsl_hip.lm`` has, next to the operators of ``perf/operators.py`` and on
tensors and outputs that the caller owns, as there:

* ``i8_dense_launch``: the dense layer in 8-bit integers with a scale for each
  row of X (the 8-bit norm's) and each column of W, which ``i8_pack`` lays out
  once;
* ``grouped_dense_launch`` / ``grouped_dense_backward_launch``: the dense layer
  of experts, each on its own run of rows, run lengths known on the device only;
* ``sample_tokens_launch``: tokens from logits and given random numbers, with
  temperature, top-k, top-p and min-p for each row.

Where ``own`` is false ``run`` computes the same from elementary torch
operations in 32 bits (sampling in 64, since a token next to a border changes
with the last bits), rounded once at the end. Sizes come from this repository's
workloads and tests (4096, 8192, 4097, 2001, 50256), or are generic; ``draw``
spreads over the same ranges.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ALPHA = 0.01  # slope of the leaky epilogue

# A drawn case costs no more than the largest listed one of its kind.
MAX_I8_FLOPS = 2 * 4096 ** 3
MAX_I8_WEIGHTS = 4096 * 50256
MAX_GROUPED_FLOPS = 2 * 8192 * 4096 * 4096
MAX_GROUPED_WEIGHTS = 8 * 4096 * 4096
MAX_LOGITS = 256 * 50256


def listed():
    return [
        # One token's 8-bit row against a large layer: the weights' bytes are the time.
        {"name": "i8_token", "op": "i8", "M": 1, "K": 8192, "N": 8192, "y": "bf16", "epi": "none"},
        # A decode batch, odd width, bias and ReLU.
        {"name": "i8_batch", "op": "i8", "M": 33, "K": 4096, "N": 4097, "y": "f16", "epi": "bias_relu"},
        # A prompt through a square layer: matrix-core work.
        {"name": "i8_prompt", "op": "i8", "M": 4096, "K": 4096, "N": 4096, "y": "bf16", "epi": "none"},
        # One token at two experts of eight: latency and two experts' weights.
        {"name": "experts_token", "op": "grouped", "T": 2, "E": 8, "K": 4096, "N": 4096, "x": "bf16", "order": "kn",
         "epi": "none"},
        # A decode batch over many small experts, most with a row or two, some with none.
        {"name": "experts_batch", "op": "grouped", "T": 96, "E": 64, "K": 2048, "N": 1024, "x": "bf16", "order": "nk",
         "epi": "bias_leaky"},
        # A prompt's rows over eight experts: the largest forward product.
        {"name": "experts_prompt", "op": "grouped", "T": 8192, "E": 8, "K": 4096, "N": 4096, "x": "bf16", "order": "kn",
         "epi": "none"},
        # Full precision, odd sizes, rows off 16-byte lines.
        {"name": "experts_f32_odd", "op": "grouped", "T": 2001, "E": 5, "K": 1001, "N": 1003, "x": "f32", "order": "kn",
         "epi": "bias_relu"},
        # The training step's way back: rows, weights (in f32, as an optimizer keeps them) and biases.
        {"name": "experts_backward", "op": "grouped_back", "T": 8192, "E": 8, "K": 4096, "N": 4096, "x": "bf16",
         "order": "kn", "epi": "bias_relu", "grad": "f32"},
        # The same of many small experts in f16, gradients in the weights' type, odd sizes.
        {"name": "experts_backward_small", "op": "grouped_back", "T": 777, "E": 24, "K": 500, "N": 772, "x": "f16",
         "order": "nk", "epi": "none", "grad": "same"},
        # One answer's next token: latency.
        {"name": "sample_token", "op": "sample", "M": 1, "V": 50256, "x": "f32", "kinds": "all", "masked": 0.0},
        # A batch in which each request has its own settings.
        {"name": "sample_batch", "op": "sample", "M": 256, "V": 50256, "x": "bf16", "kinds": "mixed", "masked": 0.0},
        # Constrained answers: most of the vocabulary masked, some rows wholly, odd width.
        {"name": "sample_masked", "op": "sample", "M": 65, "V": 32001, "x": "f16", "kinds": "mixed", "masked": 0.9},
    ]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], spread over its logarithm; every third one a
    multiple of 64, as widths often are, the others as they come."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.randrange(3) == 0:
        v = (v + 32) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["i8", "i8", "grouped", "grouped", "grouped_back", "sample", "sample"])
    epi = rng.choice(["none", "relu", "bias", "bias_relu", "bias_leaky"])
    while True:
        if op == "i8":
            M = _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 65, 4096)
            c = {"op": "i8", "M": M, "K": _log_int(rng, 64, 8192), "N": _log_int(rng, 64, 50256),
                 "y": rng.choice(["f32", "bf16", "f16"]), "epi": epi}
            if 2 * M * c["K"] * c["N"] <= MAX_I8_FLOPS and c["K"] * c["N"] <= MAX_I8_WEIGHTS:
                return c
            continue
        if op == "sample":
            c = {"op": "sample", "M": _log_int(rng, 1, 1024), "V": _log_int(rng, 1000, 131072),
                 "x": rng.choice(["f32", "bf16", "f16"]),
                 "kinds": rng.choice(["plain", "k", "p", "min", "all", "mixed", "mixed", "greedy"]),
                 "masked": rng.choice([0.0, 0.0, 0.5, 0.95])}
            if c["M"] * c["V"] <= MAX_LOGITS:
                return c
            continue
        T = _log_int(rng, 1, 128) if rng.random() < 0.4 else _log_int(rng, 129, 8192)
        c = {"op": op, "T": T, "E": _log_int(rng, 1, 64), "K": _log_int(rng, 64, 8192), "N": _log_int(rng, 64, 8192),
             "x": rng.choice(["f32", "bf16", "bf16", "f16"]), "order": rng.choice(["kn", "kn", "nk"]), "epi": epi}
        if op == "grouped_back":
            c["grad"] = rng.choice(["same", "f32"])
        part = 4 if c["x"] == "f32" else 1
        if (2 * T * c["K"] * c["N"] <= MAX_GROUPED_FLOPS // part
                and c["E"] * c["K"] * c["N"] <= MAX_GROUPED_WEIGHTS // (2 if c["x"] == "f32" else 1)):
            return c


def work(case):
    if case["op"] == "i8":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": K * N + M * K + 4 * (M + N) + M * N * BYTES[case["y"]], "flops": 2 * M * K * N}
    if case["op"] == "sample":
        M, V = case["M"], case["V"]
        return {"bytes": M * V * BYTES[case["x"]] + M * 32, "flops": 6 * M * V}
    T, E, K, N, e = case["T"], case["E"], case["K"], case["N"], BYTES[case["x"]]
    used = E * (1 - (1 - 1 / E) ** T)  # experts that have rows, about
    if case["op"] == "grouped":
        return {"bytes": (used * K * N + T * (K + N)) * e, "flops": 2 * T * K * N}
    grad = 4 if case["grad"] == "f32" else e
    acts = 0 if case["epi"] in ("none", "bias") else T * N
    return {"bytes": (used * K * N + T * (2 * K + N) + acts) * e + E * (K * N + N) * grad, "flops": 4 * T * K * N}


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)


def _settings(g, case):
    """Each row's temperature, top-k, top-p and min-p; 1, 0, 1 and 0 where it has none."""
    M, kinds = case["M"], case["kinds"]
    uses = {"plain": (0, 0, 0), "k": (1, 0, 0), "p": (0, 1, 0), "min": (0, 0, 1), "all": (1, 1, 1)}.get(kinds)
    if uses is None:
        uses = [torch.rand(M, generator=g, device="cuda") < 0.5 for _ in range(3)]
    ks = torch.tensor([1, 5, 20, 40, 50, 200, 1000], dtype=torch.int32, device="cuda")
    k = ks[torch.randint(0, len(ks), (M,), generator=g, device="cuda")]
    p, m = 0.5 + 0.49 * _rand(g, M), 0.01 + 0.19 * _rand(g, M)
    temperature = 0.6 + 0.7 * _rand(g, M)
    if kinds == "greedy":
        temperature.zero_()
    elif kinds == "mixed":
        temperature[5::16] = 0.0
    on = [u if torch.is_tensor(u) else torch.full((M,), bool(u), device="cuda") for u in uses]
    return {"temperature": temperature, "top_k": torch.where(on[0], k, 0).to(torch.int32),
            "top_p": torch.where(on[1], p, 1.0), "min_p": torch.where(on[2], m, 0.0)}


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "i8":
        M, K, N = case["M"], case["K"], case["N"]
        x = _randn(g, M, K)
        xs = x.abs().amax(1) / 127
        s = {"x": (x / xs[:, None]).round().to(torch.int8), "x_scales": xs,
             "q": (32 * _randn(g, K, N)).round().clamp(-127, 127).to(torch.int8),
             "scales": (0.5 + _rand(g, N)) / (32 * math.sqrt(K))}
        if case["epi"].startswith("bias"):
            s["bias"] = _randn(g, N).to(DTYPES[case["y"]])
        return s
    if op == "sample":
        M, V = case["M"], case["V"]
        x = 2.5 * _randn(g, M, V)
        # A few likely tokens a row.
        x.scatter_add_(1, torch.randint(0, V, (M, 8), generator=g, device="cuda"), 6 * _rand(g, M, 8))
        if case["masked"]:
            x.masked_fill_(_rand(g, M, V) < case["masked"], -math.inf)
            x[7::16] = -math.inf
        return dict(_settings(g, case), x=x.to(DTYPES[case["x"]]), uniforms=_rand(g, M))
    T, E, K, N, dt = case["T"], case["E"], case["K"], case["N"], DTYPES[case["x"]]
    # Experts' shares of the rows differ by a few times, as a router's do.
    shares = torch.softmax(0.5 * _randn(g, E), 0)
    counts = torch.bincount(torch.multinomial(shares, T, replacement=True, generator=g), minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    if case["order"] == "kn":
        w = (_randn(g, E, K, N) / math.sqrt(K)).to(dt)
    else:
        w = (_randn(g, E, N, K) / math.sqrt(K)).to(dt).transpose(1, 2)
    s = {"x": _randn(g, T, K).to(dt), "w": w, "offsets": offsets, "most": int(counts.max())}
    if op == "grouped":
        if case["epi"].startswith("bias"):
            s["bias"] = _randn(g, E, N).to(dt)
    else:
        s["dy"] = _randn(g, T, N).to(dt)
        s["y"] = _randn(g, T, N).to(dt)
        if case["epi"].endswith("relu"):
            s["y"].clamp_(min=0)
    return s


def prepare(case, seed):
    """The inputs. The framework's side also has its outputs' memory, as a
    caller of its launches does, and the 8-bit weights in the layout that they
    are loaded into once."""
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    lm, op = _lm(), case["op"]
    s["lm"] = lm
    if op == "i8":
        s["packed"] = lm.i8_pack(s.pop("q"), s.pop("scales"))
        s["out"] = new(case["M"], case["N"], dtype=DTYPES[case["y"]])
    elif op == "grouped":
        s["out"] = new(case["T"], case["N"], dtype=DTYPES[case["x"]])
    elif op == "grouped_back":
        s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"], dtype=_grad_type(case))
        s["db"] = new(case["E"], case["N"], dtype=_grad_type(case)) if case["epi"].startswith("bias") else None
    else:
        s["tokens"], s["logprobs"] = new(case["M"], dtype=torch.int64), new(case["M"])
    return s


def _grad_type(case):
    return torch.float32 if case["grad"] == "f32" else DTYPES[case["x"]]


# ------------------------------------------------------------ the framework
# The dense layer's epilogue codes (include/edsl_hip_device.h).
_EPILOGUES = {"none": 0, "bias": 1, "relu": 2, "bias_relu": 3, "bias_leaky": 5}


def _lm():
    pkg = os.path.join(os.getcwd(), "ml-edsl_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mlir_edsl_hip import lm
    return lm


def _run_own(s):
    lm, case = s["lm"], s["case"]
    op = case["op"]
    if op == "i8":
        lm.i8_dense_launch(s["x"], s["packed"], s.get("bias"), s["out"], _EPILOGUES[case["epi"]], ALPHA,
                           x_scales=s["x_scales"])
        return {"y": s["out"]}
    if op == "grouped":
        lm.grouped_dense_launch(s["x"], s["w"], s["offsets"], s.get("bias"), s["out"], _EPILOGUES[case["epi"]], ALPHA)
        return {"y": s["out"]}
    if op == "grouped_back":
        lm.grouped_dense_backward_launch(s["dy"], s["x"], s["w"], s["offsets"], dX=s["dx"], dW=s["dw"], db=s["db"],
                                         Y=s["y"], epilogue=_EPILOGUES[case["epi"]], alpha=ALPHA)
        return {"dx": s["dx"], "dw": s["dw"], "db": s["db"]}
    lm.sample_tokens_launch(s["x"], s["uniforms"], s["tokens"], logprobs=s["logprobs"], temperature=s["temperature"],
                            top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"tokens": s["tokens"], "logprobs": s["logprobs"]}


# ------------------------------------------------------------ the plain form
def _activated(y, epi):
    if epi.endswith("relu"):
        return y.clamp(min=0)
    if epi.endswith("leaky"):
        return y.clamp(min=0) + ALPHA * y.clamp(max=0)
    return y


def _plain_i8(s):
    # Sums stay far under 2^24 here: 32-bit floats hold them exactly.
    y = (s["x"].float() @ s["q"].float()) * s["scales"].float() * s["x_scales"][:, None]
    if "bias" in s:
        y = y + s["bias"].float()
    return {"y": _activated(y, s["case"]["epi"]).to(DTYPES[s["case"]["y"]])}


def _places(s):
    """Each row's expert and its place among that expert's rows."""
    rows = torch.arange(s["case"]["T"], device="cuda", dtype=torch.int32)
    expert = torch.searchsorted(s["offsets"][1:], rows, right=True)
    return expert, rows - s["offsets"][expert]


def _padded(s, rows, expert, place):
    """Rows as one batch of each expert's, filled up with zeros."""
    out = rows.new_zeros(s["case"]["E"], s["most"], rows.shape[1], dtype=torch.float32)
    out[expert, place] = rows.float()
    return out


def _plain_grouped(s):
    case = s["case"]
    expert, place = _places(s)
    if case["T"] <= case["E"]:  # few rows: each one's own weights
        y = torch.bmm(s["x"].float()[:, None], s["w"][expert].float())[:, 0]
    else:
        y = torch.bmm(_padded(s, s["x"], expert, place), s["w"].float())[expert, place]
    if "bias" in s:
        y = y + s["bias"].float()[expert]
    return {"y": _activated(y, case["epi"]).to(s["x"].dtype)}


def _plain_grouped_back(s):
    case, dt = s["case"], _grad_type(s["case"])
    dz = s["dy"].float()
    if case["epi"].endswith("relu"):
        dz = torch.where(s["y"] > 0, dz, 0.0)
    elif case["epi"].endswith("leaky"):
        dz = torch.where(s["y"] > 0, dz, ALPHA * dz)
    expert, place = _places(s)
    x, dz = _padded(s, s["x"], expert, place), _padded(s, dz, expert, place)
    dx = torch.bmm(dz, s["w"].float().transpose(1, 2))[expert, place]
    db = dz.sum(1).to(dt) if case["epi"].startswith("bias") else None
    return {"dx": dx.to(s["x"].dtype), "dw": torch.bmm(x.transpose(1, 2), dz).to(dt), "db": db}


def _plain_sample(s):
    x = s["x"].double()
    greedy = s["temperature"] == 0
    l = x / torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    some = x.amax(1) > -math.inf
    l = torch.where(some[:, None], l, 0.0)
    ranked, order = l.sort(dim=1, descending=True, stable=True)
    w = (ranked - ranked[:, :1]).exp()
    rank = torch.arange(x.shape[1], device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1])[:, None]
    w = torch.where(rank < k, w, 0.0)
    mass = w.cumsum(1)
    keep = mass - w < s["top_p"].double()[:, None] * mass[:, -1:]
    keep |= s["top_p"][:, None] >= 1
    keep &= w >= s["min_p"].double()[:, None]
    keep &= torch.where(greedy[:, None], rank == 0, rank < k)
    kept = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))
    mass = kept.cumsum(1)
    tokens = (mass <= s["uniforms"].double()[:, None] * mass[:, -1:]).sum(1)
    tokens = tokens.clamp(max=x.shape[1] - 1)
    logprobs = (kept.gather(1, tokens[:, None]).squeeze(1) / mass[:, -1]).log()
    return {"tokens": torch.where(some, tokens, -1), "logprobs": torch.where(some, logprobs, -math.inf).float()}


_PLAIN = {"i8": _plain_i8, "grouped": _plain_grouped, "grouped_back": _plain_grouped_back, "sample": _plain_sample}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits
def _exact_act(z, epi):
    if epi in ("relu", "bias_relu"):
        return torch.where(z > 0, z, 0.0)
    return torch.where(z > 0, z, ALPHA * z) if epi == "bias_leaky" else z


def exact(case, seed):
    """From the definitions, in 64 bits, on the inputs as they are: expert by
    expert, and row by row for the samples."""
    s, op = _inputs(case, seed), case["op"]
    if op == "i8":
        x, q = s["x"].double() * s["x_scales"].double()[:, None], s["q"].double() * s["scales"].double()
        z = torch.mm(x, q)
        if "bias" in s:
            z += s["bias"].double()
        return {"y": _exact_act(z, case["epi"])}
    if op == "sample":
        # The row's kept logits from the largest down, then drawn in the order of their index.
        logprobs = torch.empty(case["M"], dtype=torch.float64, device="cuda")
        for m in range(case["M"]):
            v = s["x"][m].double()
            i = torch.nonzero(v > -math.inf).squeeze(1)
            if len(i) == 0:
                logprobs[m] = -math.inf
                continue
            t = s["temperature"][m].double()
            if t == 0:
                logprobs[m] = 0.0
                continue
            i = i[torch.sort(v[i].neg(), stable=True).indices]
            if s["top_k"][m] > 0:
                i = i[:int(s["top_k"][m])]
            p = torch.softmax(v[i] / t, 0)
            n = len(i)
            if s["top_p"][m] < 1:
                before = p.cumsum(0) - p
                n = int((before < s["top_p"][m].double()).sum())
            n = min(n, int((p >= s["min_p"][m].double() * p[0]).sum()))
            i = i[:n].sort().values
            logp = torch.log_softmax(v[i] / t, 0)
            at = torch.searchsorted(logp.exp().cumsum(0), s["uniforms"][m:m + 1].double(), right=True)
            logprobs[m] = logp[at.clamp(max=n - 1)[0]]
        return {"tokens": None, "logprobs": logprobs}
    off, d = s["offsets"].tolist(), {k: v.double() for k, v in s.items() if torch.is_tensor(v) and k != "w"}
    runs = [(e, slice(off[e], off[e + 1])) for e in range(case["E"])]
    if op == "grouped":
        y = torch.empty(case["T"], case["N"], dtype=torch.float64, device="cuda")
        for e, r in runs:
            y[r] = torch.mm(d["x"][r], s["w"][e].double())
            if "bias" in s:
                y[r] += d["bias"][e]
        return {"y": _exact_act(y, case["epi"])}
    slope = {"relu": 0.0, "bias_relu": 0.0, "bias_leaky": ALPHA}.get(case["epi"], 1.0)
    dz = d["dy"] * torch.where(d["y"] > 0, 1.0, slope)
    dx = torch.empty_like(d["x"])
    dw = torch.empty(case["E"], case["K"], case["N"], dtype=torch.float64, device="cuda")
    db = torch.empty(case["E"], case["N"], dtype=torch.float64, device="cuda")
    for e, r in runs:
        dx[r] = torch.mm(dz[r], s["w"][e].double().t())
        dw[e] = torch.mm(d["x"][r].t(), dz[r])
        db[e] = dz[r].sum(0)
    return {"dx": dx, "dw": dw, "db": db if case["epi"].startswith("bias") else None}
