"""The language-model operators around the dense layer, as timed cases.

``mlir_edsl_hip.lm`` has three operators, each called on tensors that live in
HBM with outputs that the caller owns, as ``device.dense_launch`` is:

* ``rms_norm_launch`` / ``rms_norm_backward_launch``: the root-mean-square norm
  with the residual's addition, its output in the input's type or in 8 bits
  with a scale for each row;
* ``q4_dense_launch``: the dense layer on 4-bit weights with group scales,
  laid out once by ``q4_pack``;
* ``token_logprobs_launch`` / ``token_logprobs_backward_launch``: log
  probabilities of given tokens with log-sum-exp, entropy and top alternatives.

Where ``own`` is false ``run`` computes the same from elementary torch
operations in 32 bits, rounded once at the end. Sizes come from this
repository's workloads and tests (4096, 8192, 4097, 2001, 50256), or are
generic; ``draw`` spreads over the same ranges.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "int8": torch.int8, "fp8": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "int8": 1, "fp8": 1}
QMAX = {"int8": 127.0, "fp8": 448.0}  # the largest value that 8 bits hold

# A drawn case costs no more than the largest listed one of its kind.
MAX_NORM = 4096 * 8192
MAX_Q4_FLOPS = 2 * 4096 ** 3
MAX_Q4_WEIGHTS = 4096 * 50256
MAX_LOGITS = 2048 * 50256


def listed():
    return [
        # One token's residual stream before a layer: latency.
        {"name": "norm_token", "op": "norm", "M": 1, "N": 4096, "x": "bf16", "y": "bf16", "residual": True},
        # A prompt's stream, the output in 8 bits for an 8-bit x 4-bit layer: the largest norm.
        {"name": "norm_8bit_prompt", "op": "norm", "M": 4096, "N": 8192, "x": "bf16", "y": "fp8", "residual": True},
        # An f32 stream of odd width, no residual: rows off 16-byte lines.
        {"name": "norm_odd", "op": "norm", "M": 2001, "N": 2001, "x": "f32", "y": "f32", "residual": False},
        # The training step's way back through the norm, weight gradient included.
        {"name": "norm_backward", "op": "norm_back", "M": 4096, "N": 4096, "x": "bf16", "stream_grad": True},
        # One token against a large layer: the weights' bytes are the time.
        {"name": "q4_token", "op": "q4", "M": 1, "K": 8192, "N": 8192, "x": "bf16", "y": "bf16", "scales": "bf16",
         "group": 128, "zeros": True, "epi": "none"},
        # A decode batch on the norm's 8-bit output, odd width, bias and ReLU.
        {"name": "q4_batch_8bit", "op": "q4", "M": 16, "K": 4096, "N": 4097, "x": "int8", "y": "bf16",
         "scales": "f16", "group": 64, "zeros": False, "epi": "bias_relu"},
        # A vocabulary-sized layer in f32 on a few dozen rows, f32 precision kept.
        {"name": "q4_vocabulary_f32", "op": "q4", "M": 48, "K": 4096, "N": 50256, "x": "f32", "y": "f32",
         "scales": "f32", "group": 128, "zeros": False, "epi": "bias"},
        # A prompt through a square layer: matrix-core work.
        {"name": "q4_prompt", "op": "q4", "M": 4096, "K": 4096, "N": 4096, "x": "bf16", "y": "bf16",
         "scales": "bf16", "group": 128, "zeros": True, "epi": "none"},
        # One token's logits, with alternatives: a long row on one card.
        {"name": "logprobs_token", "op": "lp", "M": 1, "V": 50256, "x": "f32", "k": 8, "masked": 0.0},
        # Scoring a prompt: every position's log probability, entropy, five alternatives.
        {"name": "logprobs_prompt", "op": "lp", "M": 2048, "V": 50256, "x": "bf16", "k": 5, "masked": 0.0},
        # Constrained sampling: most of the vocabulary masked by -inf, some rows wholly, padding tokens, odd width.
        {"name": "logprobs_masked", "op": "lp", "M": 65, "V": 32001, "x": "f16", "k": 20, "masked": 0.9},
        # The way back from log probabilities and entropies to the logits.
        {"name": "logprobs_backward", "op": "lp_back", "M": 2048, "V": 50256, "x": "bf16", "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], spread over its logarithm; every third one a
    multiple of 64, as widths often are, the others as they come."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.randrange(3) == 0:
        v = (v + 32) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_back", "q4", "q4", "q4", "lp", "lp", "lp_back"])
    x = rng.choice(["f32", "bf16", "bf16", "f16"])
    while True:
        if op in ("norm", "norm_back"):
            c = {"op": op, "M": _log_int(rng, 1, 8192), "N": _log_int(rng, 128, 16384), "x": x}
            if c["M"] * c["N"] > MAX_NORM or (op == "norm_back" and c["M"] * c["N"] > MAX_NORM // 2):
                continue
            if x == "f32" and c["M"] * c["N"] > MAX_NORM // 2:
                continue
            if op == "norm":
                c.update(y=rng.choice([x, x, "fp8"]), residual=rng.random() < 0.6)
            else:
                c["stream_grad"] = rng.random() < 0.5
            return c
        if op == "q4":
            small = rng.random() < 0.6
            c = {"op": "q4", "M": _log_int(rng, 1, 64) if small else _log_int(rng, 65, 4096),
                 "K": _log_int(rng, 128, 8192), "N": _log_int(rng, 128, 50256),
                 "x": rng.choice(["f32", "bf16", "bf16", "f16", "int8", "fp8"]),
                 "scales": rng.choice(["f32", "bf16", "f16"]), "group": rng.choice([32, 64, 128, 128, 256]),
                 "zeros": rng.random() < 0.5, "epi": rng.choice(["none", "relu", "bias", "bias_relu", "bias_leaky"])}
            c["y"] = c["x"] if c["x"] in ("f32", "bf16", "f16") else rng.choice(["f32", "bf16"])
            most = MAX_Q4_FLOPS // 4 if c["x"] == "f32" else MAX_Q4_FLOPS
            if 2 * c["M"] * c["K"] * c["N"] <= most and c["K"] * c["N"] <= MAX_Q4_WEIGHTS:
                return c
            continue
        c = {"op": op, "M": _log_int(rng, 1, 4096), "V": _log_int(rng, 1000, 131072), "x": x,
             "masked": rng.choice([0.0, 0.0, 0.5, 0.95])}
        if op == "lp":
            c["k"] = rng.choice([0, 1, 5, 8, 20, 32])
        if c["M"] * c["V"] <= MAX_LOGITS // (2 if x == "f32" else 1):
            return c


def work(case):
    op = case["op"]
    if op == "norm":
        M, N, e = case["M"], case["N"], BYTES[case["x"]]
        streams = 3 if case["residual"] else 1  # x; the residual and the sum that is written
        return {"bytes": M * N * (streams * e + BYTES[case["y"]]) + N * e + 4 * M, "flops": 6 * M * N}
    if op == "norm_back":
        M, N, e = case["M"], case["N"], BYTES[case["x"]]
        streams = 4 if case["stream_grad"] else 3  # dY, H, dX (and dH)
        return {"bytes": M * N * streams * e + N * e + 4 * N + 4 * M, "flops": 11 * M * N}
    if op == "q4":
        M, K, N, G = case["M"], case["K"], case["N"], -(-case["K"] // case["group"])
        per = BYTES[case["scales"]] + (0.5 if case["zeros"] else 0)
        return {"bytes": K * N / 2 + G * N * per + M * K * BYTES[case["x"]] + M * N * BYTES[case["y"]],
                "flops": 2 * M * K * N}
    M, V, e = case["M"], case["V"], BYTES[case["x"]]
    if op == "lp":
        return {"bytes": M * V * e + M * (8 + 12 + 12 * case["k"]), "flops": 6 * M * V}
    return {"bytes": 2 * M * V * e + M * 24, "flops": 9 * M * V}


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _logits(g, case):
    """Logits with the spread that a trained model's have; in a masked case
    that share of the vocabulary is -inf, and all of every 16th row."""
    M, V = case["M"], case["V"]
    x = 2.5 * _randn(g, M, V)
    tokens = torch.randint(0, V, (M,), generator=g, device="cuda")
    # Most given tokens are likely ones.
    likely = torch.rand(M, generator=g, device="cuda") < 0.7
    x[torch.arange(M, device="cuda"), tokens] += 9.0 * likely
    if case["masked"]:
        x.masked_fill_(torch.rand(M, V, generator=g, device="cuda") < case["masked"], -math.inf)
        x[7::16] = -math.inf
        tokens[3::8] = -100  # padding
    return x.to(DTYPES[case["x"]]), tokens


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    if op in ("norm", "norm_back"):
        M, N, dt = case["M"], case["N"], DTYPES[case["x"]]
        s = {"x": (1.5 * _randn(g, M, N)).to(dt), "weight": (1 + 0.1 * _randn(g, N)).to(dt)}
        if op == "norm":
            if case["residual"]:
                s["residual"] = (2 * _randn(g, M, N)).to(dt)
        else:
            s["dy"] = _randn(g, M, N).to(dt)
            if case["stream_grad"]:
                s["dh"] = _randn(g, M, N).to(dt)
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
        return s
    if op == "q4":
        M, K, N, group = case["M"], case["K"], case["N"], case["group"]
        G = -(-K // group)
        s = {"q": torch.randint(0, 16, (K, N), generator=g, device="cuda", dtype=torch.uint8),
             "scales": ((0.5 + torch.rand(G, N, generator=g, device="cuda")) / (4 * math.sqrt(K)))
             .to(DTYPES[case["scales"]])}
        if case["zeros"]:
            s["zeros"] = torch.randint(4, 12, (G, N), generator=g, device="cuda", dtype=torch.uint8)
        x = _randn(g, M, K)
        if case["x"] in QMAX:
            s["x_scales"] = x.abs().amax(1) / QMAX[case["x"]]
            x = x / s["x_scales"][:, None]
            x = x.round() if case["x"] == "int8" else x
        s["x"] = x.to(DTYPES[case["x"]])
        if case["epi"].startswith("bias"):
            s["bias"] = _randn(g, N).to(DTYPES[case["y"]])
        return s
    x, tokens = _logits(g, case)
    s = {"x": x, "tokens": tokens}
    if op == "lp_back":
        l = x.float()
        s["lse"], p = torch.logsumexp(l, 1), torch.softmax(l, 1)
        h = -torch.where(p > 0, p * (l - s["lse"][:, None]), 0.0).sum(1)
        s["entropy"] = torch.where(s["lse"] > -math.inf, h, 0.0)
        s["dlogprobs"], s["dentropy"] = _randn(g, case["M"]), 0.01 * _randn(g, case["M"])
    return s


ALPHA = 0.01  # slope of the leaky epilogue
SCALE = 1 / 0.8  # what the logits are multiplied by: a temperature of 0.8


def prepare(case, seed):
    """The inputs. The framework's side also has its outputs' memory, as a
    caller of its launches does, and the 4-bit weights in the layout that they
    are loaded into once."""
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    M, op = case["M"], case["op"]
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    lm = s["lm"] = _lm()
    if op == "norm":
        s["y"], s["rstd"] = new(M, case["N"], dtype=DTYPES[case["y"]]), new(M)
        s["total"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["y_scales"] = new(M) if case["y"] in QMAX else None
    elif op == "norm_back":
        s["dx"], s["dweight"] = torch.empty_like(s["x"]), new(case["N"])
    elif op == "q4":
        s["packed"] = lm.q4_pack(s.pop("q"), s.pop("scales"), s.pop("zeros", None), group_size=case["group"])
        s["y"] = new(M, case["N"], dtype=DTYPES[case["y"]])
    elif op == "lp":
        s["logprobs"], s["lse"], s["entropy"] = new(M), new(M), new(M)
        s["top"] = new(M, case["k"]) if case["k"] else None
        s["ids"] = new(M, case["k"], dtype=torch.int64) if case["k"] else None
    else:
        s["dlogits"] = torch.empty_like(s["x"])
    return s


# ------------------------------------------------------------ the framework
def _lm():
    pkg = os.path.join(os.getcwd(), "ml-edsl_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mlir_edsl_hip import lm
    return lm


def _run_own(s):
    lm, case = s["lm"], s["case"]
    op = case["op"]
    if op == "norm":
        lm.rms_norm_launch(s["x"], s["weight"], s["y"], residual=s.get("residual"), total=s["total"],
                           scales=s["y_scales"], rstd=s["rstd"], eps=EPS)
        return {"y": s["y"], "total": s["total"], "scales": s["y_scales"], "rstd": s["rstd"]}
    if op == "norm_back":
        lm.rms_norm_backward_launch(s["dy"], s["x"], s["weight"], s["rstd"], s["dx"], dweight=s["dweight"],
                                    dh=s.get("dh"))
        return {"dx": s["dx"], "dweight": s["dweight"]}
    if op == "q4":
        lm.q4_dense_launch(s["x"], s["packed"], s.get("bias"), s["y"], _EPILOGUES[case["epi"]], ALPHA,
                           x_scales=s.get("x_scales"))
        return {"y": s["y"]}
    if op == "lp":
        lm.token_logprobs_launch(s["x"], s["tokens"], s["logprobs"], lse=s["lse"], entropy=s["entropy"],
                                 top_logprobs=s["top"], top_ids=s["ids"], scale=SCALE)
        return {"logprobs": s["logprobs"], "lse": s["lse"], "entropy": s["entropy"], "top": s["top"],
                "ids": s["ids"]}
    lm.token_logprobs_backward_launch(s["x"], s["tokens"], s["lse"], s["dlogits"], dlogprobs=s["dlogprobs"],
                                      entropy=s["entropy"], dentropy=s["dentropy"])
    return {"dlogits": s["dlogits"]}


# The dense layer's epilogue codes (include/edsl_hip_device.h).
_EPILOGUES = {"none": 0, "bias": 1, "relu": 2, "bias_relu": 3, "bias_leaky": 5}


# ------------------------------------------------------------ the plain form
def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    total = None
    if "residual" in s:
        x = x + s["residual"].float()
        total = x.to(s["x"].dtype)
    rstd = torch.rsqrt(x.square().mean(1) + EPS)
    y, scales = x * rstd[:, None] * s["weight"].float(), None
    if case["y"] in QMAX:
        scales = y.abs().amax(1) / QMAX[case["y"]]
        y = torch.where(scales[:, None] > 0, y / scales[:, None], 0.0)
    return {"y": y.to(DTYPES[case["y"]]), "total": total, "scales": scales, "rstd": rstd}


def _plain_norm_back(s):
    dy, h, rstd = s["dy"].float(), s["x"].float(), s["rstd"][:, None]
    xh, t = h * rstd, dy * s["weight"].float()
    dx = (t - xh * (t * xh).mean(1, keepdim=True)) * rstd
    if "dh" in s:
        dx = dx + s["dh"].float()
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(0)}


def _plain_q4(s):
    case = s["case"]
    K, group = case["K"], case["group"]
    zeros = s["zeros"].float().repeat_interleave(group, 0)[:K] if case["zeros"] else 8.0
    w = (s["q"].float() - zeros) * s["scales"].float().repeat_interleave(group, 0)[:K]
    y = s["x"].float() @ w
    if "x_scales" in s:
        y = y * s["x_scales"][:, None]
    if "bias" in s:
        y = y + s["bias"].float()
    if case["epi"].endswith("relu"):
        y = y.clamp(min=0)
    elif case["epi"] == "bias_leaky":
        y = y.clamp(min=0) + ALPHA * y.clamp(max=0)
    return {"y": y.to(DTYPES[case["y"]])}


def _plain_lp(s):
    case, x, tokens = s["case"], s["x"].float(), s["tokens"]
    l = x * SCALE
    top = l.amax(1, keepdim=True)
    some = top > -math.inf
    e = torch.where(some, (l - top).exp(), 0.0)
    total = e.sum(1, keepdim=True)
    lse = torch.where(some, top + total.log(), -math.inf)
    entropy = torch.where(some, lse - torch.where(e > 0, e * l, 0.0).sum(1, keepdim=True) / total, 0.0)
    given = tokens.clamp(min=0)[:, None]
    lp = torch.where(some, l.gather(1, given) - lse, -math.inf).squeeze(1)
    lp = torch.where((tokens >= 0) & (tokens < case["V"]), lp, 0.0)
    out = {"logprobs": lp, "lse": lse.squeeze(1), "entropy": entropy.squeeze(1), "top": None, "ids": None}
    if case["k"]:
        # Unique keys: the value's order, then the lower index first.
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
        key = (order << 32) - torch.arange(case["V"], device=x.device)
        out["ids"] = key.topk(case["k"], 1).indices
        out["top"] = torch.where(some, l.gather(1, out["ids"]) - lse, -math.inf)
    return out


def _plain_lp_back(s):
    x, tokens, lse, h = s["x"].float(), s["tokens"], s["lse"][:, None], s["entropy"][:, None]
    some = lse > -math.inf
    given = ((tokens >= 0) & (tokens < x.shape[1]))[:, None]
    lp = torch.where(some, x - lse, -math.inf)
    p = lp.exp()
    g = torch.where(given & some, s["dlogprobs"][:, None], 0.0)
    d = -p * g - torch.where(p > 0, p * (lp + h), 0.0) * s["dentropy"][:, None]
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], g)
    return {"dlogits": d.to(s["x"].dtype)}


_PLAIN = {"norm": _plain_norm, "norm_back": _plain_norm_back, "q4": _plain_q4, "lp": _plain_lp,
          "lp_back": _plain_lp_back}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """From the definitions, in 64 bits, on the inputs as they are. What 8 bits
    hold is given unrounded, as a value of a narrower float type is."""
    s, op = _inputs(case, seed), case["op"]
    d = {k: v.double() for k, v in s.items() if v.is_floating_point() or k == "x"}
    if op == "norm":
        h = d["x"] + d["residual"] if case["residual"] else d["x"]
        norm = (torch.linalg.vector_norm(h, dim=1) ** 2 / case["N"] + EPS).sqrt()
        y, scales = d["weight"] * (h / norm[:, None]), None
        if case["y"] in QMAX:
            scales = torch.linalg.vector_norm(y, math.inf, dim=1) / QMAX[case["y"]]
            y = y / scales[:, None]
        return {"y": y, "total": h if case["residual"] else None, "scales": scales, "rstd": 1 / norm}
    if op == "norm_back":
        g, h, r = d["dy"] * d["weight"], d["x"], d["rstd"][:, None]
        dx = r * g - r ** 3 * h * ((g * h).sum(1, keepdim=True) / case["N"])
        if case["stream_grad"]:
            dx += d["dh"]
        return {"dx": dx, "dweight": (d["dy"] * h * r).sum(0)}
    if op == "q4":
        at = torch.arange(case["K"], device="cuda") // case["group"]
        n = s["q"].double()
        n -= s["zeros"].double()[at] if case["zeros"] else 8
        n *= d["scales"][at]
        x = d["x"] * d["x_scales"][:, None] if "x_scales" in s else d["x"]
        y = torch.mm(x, n)
        if "bias" in s:
            y += d["bias"]
        if case["epi"] in ("relu", "bias_relu"):
            y = torch.where(y > 0, y, 0.0)
        elif case["epi"] == "bias_leaky":
            y = torch.where(y > 0, y, ALPHA * y)
        return {"y": y}
    M, V, rows = case["M"], case["V"], torch.arange(case["M"], device="cuda")
    ok = (s["tokens"] >= 0) & (s["tokens"] < V)
    at = torch.where(ok, s["tokens"], 0)
    if op == "lp":
        l = d["x"] * SCALE
        lse = torch.logsumexp(l, 1)
        none = lse == -math.inf
        logp = torch.log_softmax(l, 1)
        entropy = torch.special.entr(logp.exp()).sum(1)
        lp = torch.where(ok, logp[rows, at], 0.0)
        lp[none & ok] = -math.inf
        entropy[none] = 0.0
        out = {"logprobs": lp, "lse": lse, "entropy": entropy, "top": None, "ids": None}
        if case["k"]:
            out["top"] = logp.topk(case["k"], 1).values
            out["top"][none] = -math.inf
        return out
    p = (d["x"] - d["lse"][:, None]).exp()
    p[d["lse"] == -math.inf] = 0.0
    logp = torch.where(p > 0, p, 1.0).log()
    out = -p * (torch.where(ok, d["dlogprobs"], 0.0)[:, None] + d["dentropy"][:, None] * (logp + d["entropy"][:, None]))
    gain = torch.where(ok & (d["lse"] > -math.inf), d["dlogprobs"], 0.0)
    out[rows, at] += gain
    return {"dlogits": out}
