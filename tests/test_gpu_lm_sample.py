"""Sampling against 64 bits, row by row from the definition.

Tokens are compared as they are: the kernel's masses are within 2^-46 V^(1/2) or so of
the largest weight, so that a random number or setting falls between two results'
borders with a chance of 1e-6 a row at most; where borders are met on purpose, weights
are powers of two and sums exact on both sides. Log probabilities: one rounding to
32 bits, and masses in units of 2^-46 of the largest weight: V 2^-46 / w relative."""
import math

import pytest
import torch

import lm_layers_reference as layers
from mlir_edsl_hip import last_plan, lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}
INF = math.inf


def logits(M, V, seed=0, dtype=F32, spread=2.5):
    return (spread * torch.randn(M, V, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def uniforms(M, seed=1):
    return torch.rand(M, generator=torch.Generator().manual_seed(seed)).cuda()


def draw(x, u, ids=torch.int64, **settings):
    tokens = torch.full((x.shape[0],), -9, dtype=ids, device="cuda")
    logprobs = torch.full((x.shape[0],), 9.0, device="cuda")
    lm.sample_tokens_launch(x, u, tokens, logprobs, **settings)
    return tokens, logprobs


def check(x, u, ids=torch.int64, **settings):
    tokens, logprobs = draw(x, u, ids, **settings)
    for m in range(x.shape[0]):
        row = {k: (v[m].item() if torch.is_tensor(v) else v) for k, v in settings.items()}
        token, logprob = layers.sample(x[m], u[m], **row)
        assert int(tokens[m]) == token, (m, row, int(tokens[m]), token)
        got = float(logprobs[m])
        if math.isfinite(logprob):
            bound = 2.0 ** -23 * abs(logprob) + x.shape[1] * 2.0 ** -45 * math.exp(-logprob)
            assert abs(got - logprob) <= bound, (m, got, logprob)
        else:
            assert got == logprob or (math.isnan(got) and math.isnan(logprob))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [1, 2, 7, 64, 513, 1000, 5000, 32001, 131072, 300000])
def test_lengths(dtype, V):
    x, u = logits(6, V, seed=V, dtype=TYPES[dtype]), uniforms(6, seed=V)
    check(x, u)
    check(x, u, temperature=0.7, top_k=50, top_p=0.9, min_p=0.02)


SETTINGS = {
    "plain": {}, "cold": dict(temperature=0.05), "hot": dict(temperature=30.0), "k1": dict(top_k=1),
    "k": dict(top_k=40), "k_large": dict(top_k=4000), "k_all": dict(top_k=10 ** 9), "p": dict(top_p=0.9),
    "p_small": dict(top_p=1e-6), "p_zero": dict(top_p=0.0), "p_negative": dict(top_p=-1.0), "p_near_1": dict(top_p=0.999999),
    "min": dict(min_p=0.05), "min_1": dict(min_p=1.0), "min_over": dict(min_p=3.0), "k_p": dict(top_k=20, top_p=0.5),
    "k_p_hot": dict(temperature=8.0, top_k=3000, top_p=0.95), "all": dict(temperature=0.8, top_k=100, top_p=0.95, min_p=0.01),
    "greedy": dict(temperature=0.0, top_k=5, top_p=0.5), "k_cold": dict(temperature=0.02, top_k=500, top_p=0.99),
}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("name", list(SETTINGS))
def test_settings(dtype, name):
    check(logits(24, 6001, seed=3, dtype=TYPES[dtype]), uniforms(24, seed=4), **SETTINGS[name])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_settings_of_each_row(dtype):
    M, g = 64, torch.Generator().manual_seed(7)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (M,), generator=g)].cuda()  # noqa: E731
    check(logits(M, 9000, seed=5, dtype=TYPES[dtype]), uniforms(M, seed=6), ids=torch.int32,
          temperature=pick(0.0, 0.3, 1.0, 1.7), top_k=pick(0, 1, 30, 2000, -4).int(), top_p=pick(1.0, 0.2, 0.9, 2.0),
          min_p=pick(0.0, 0.1, 0.5, -1.0))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("levels", [1, 2, 5])
@pytest.mark.parametrize("settings", [{}, dict(top_k=37), dict(top_p=0.5), dict(top_k=2500, top_p=0.25), dict(top_k=5003)],
                         ids=str)
def test_ties(dtype, levels, settings):
    """Few distinct logits, log 2 apart: long runs of equal ones at every border, more than a border's list holds."""
    V = 5003
    x = (torch.randint(0, levels, (8, V), generator=torch.Generator().manual_seed(levels)) * math.log(2)).to(TYPES[dtype]).cuda()
    check(x, uniforms(8, seed=9), **settings)


def test_ties_in_the_order_of_their_index():
    V = 3000
    x = torch.zeros(5, V, device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    assert draw(x, u)[0].tolist() == [0, 750, 1500, 2250, 2999]
    assert draw(x, u, top_k=8)[0].tolist() == [0, 2, 4, 6, 7]
    assert draw(x, u, top_p=0.5)[0].tolist() == [0, 375, 750, 1125, 1499]
    x[:, 1000:1004] = 1.0
    assert draw(x, u, top_k=4)[0].tolist() == [1000, 1001, 1002, 1003, 1003]
    assert draw(x, u, top_k=2)[0].tolist() == [1000, 1000, 1001, 1001, 1001]
    assert draw(x, u, temperature=0.0)[0].tolist() == [1000] * 5


def test_every_token_by_its_share():
    """Weights that are powers of two: the token at every 64th of the range."""
    x = torch.tensor([0.0, -INF, math.log(2), math.log(4), -INF, 0.0], dtype=torch.float64)
    x = x.float().expand(64, 6).contiguous().cuda()
    u = (torch.arange(64) / 64 + 2.0 ** -8).cuda()
    tokens = draw(x, u)[0].cpu()
    assert torch.bincount(tokens, minlength=6).tolist() == [8, 0, 16, 32, 0, 8]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("settings", [{}, dict(top_k=3), dict(top_p=0.3, min_p=0.01), dict(temperature=0.0),
                                      dict(top_k=200, top_p=0.9)], ids=str)
def test_masks_infinities_and_nan(dtype, settings):
    t = TYPES[dtype]
    low = torch.finfo(t).min
    x = logits(9, 700, seed=8, dtype=t)
    x[0] = -INF
    x[1] = -INF
    x[1, 699] = 3.0
    x[2, ::2] = -INF
    x[3] = low
    x[4, 100:] = low
    x[5, 50] = INF
    x[6, 60] = math.nan
    x[7] = -INF
    x[7, 5] = math.nan
    x[8, 1:] = -INF
    x[8, 0] = low
    check(x, uniforms(9, seed=2), **settings)


def test_settings_and_numbers_of_no_meaning():
    M = 10
    x, u = logits(M, 500), torch.full((M,), 0.5, device="cuda")
    t, p, m = (torch.full((M,), v, device="cuda") for v in (1.0, 1.0, 0.0))
    t[0], t[1], t[2], p[3], m[4], u[5] = -1.0, math.nan, INF, math.nan, math.nan, math.nan
    u[6], u[7], u[8] = -3.0, 1.0, INF
    tokens, logprobs = draw(x, u, temperature=t, top_p=p, min_p=m)
    assert tokens[:6].tolist() == [-1] * 6 and bool(logprobs[:6].isnan().all())
    for m in (6, 7, 8, 9):
        assert int(tokens[m]) == layers.sample(x[m], u[m])[0]


@pytest.mark.parametrize("temperature", [1e-38, 1e-20, 1e-3, 100.0, 1e6, 3e38])
def test_extreme_temperatures(temperature):
    check(logits(8, 2000, seed=11), uniforms(8, seed=12), temperature=temperature)
    check(logits(8, 2000, seed=11), uniforms(8, seed=12), temperature=temperature, top_k=10, top_p=0.8)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_alignments_and_outputs_left_out(dtype):
    M, V = 11, 1021
    big = torch.full((M, V + 9), INF, dtype=TYPES[dtype], device="cuda")
    x = big[:, 3:3 + V]
    x.copy_(logits(M, V, seed=13))
    check(x, uniforms(M), top_k=50, top_p=0.9)
    tokens = torch.zeros(M, dtype=torch.int32, device="cuda")
    lm.sample_tokens_launch(x, uniforms(M), tokens)
    assert "sample_tokens" in last_plan()
    assert [int(t) for t in tokens] == [layers.sample(x[m], uniforms(M)[m])[0] for m in range(M)]


def test_many_rows_and_the_same_bits():
    M, V = 3000, 400
    x, u = logits(M, V, seed=14, dtype=BF16), uniforms(M, seed=15)
    first = draw(x, u, temperature=0.9, top_k=30, top_p=0.8)
    for _ in range(3):
        again = draw(x, u, temperature=0.9, top_k=30, top_p=0.8)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    for m in range(0, M, 97):
        assert int(first[0][m]) == layers.sample(x[m], u[m], 0.9, 30, 0.8)[0]


def test_another_stream_and_graph_replays():
    M, V = 7, 3000
    x, u = logits(M, V), uniforms(M)
    tokens, logprobs = torch.zeros(M, dtype=torch.int64, device="cuda"), torch.zeros(M, device="cuda")
    k = torch.full((M,), 20, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    lm.sample_tokens_launch(x, u, tokens, logprobs, top_k=k, top_p=0.9, stream=side)
    side.synchronize()
    assert tokens.tolist() == [layers.sample(x[m], u[m], 1.0, 20, 0.9)[0] for m in range(M)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lm.sample_tokens_launch(x, u, tokens, logprobs, top_k=k, top_p=0.9)
    for i in range(4):
        x.copy_(logits(M, V, seed=20 + i))
        u.copy_(uniforms(M, seed=30 + i))
        k.fill_(5 * (i + 1))
        tokens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert tokens.tolist() == [layers.sample(x[m], u[m], 1.0, 5 * (i + 1), 0.9)[0] for m in range(M)]
        draw(logits(3, 900), uniforms(3), top_k=4)


def test_no_rows_and_refusals():
    x, u = logits(4, 30), uniforms(4)
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    f = lm.sample_tokens_launch
    f(x[:0], u[:0], tokens[:0])
    assert last_plan() == "empty"
    for call, error, text in (
            (lambda: f(x.int(), u, tokens), TypeError, "logits has dtype"),
            (lambda: f(x[0], u, tokens), ValueError, "logits must be 2-D"),
            (lambda: f(x.t(), u, tokens), ValueError, "unit inner stride"),
            (lambda: f(x[:, :0], u, tokens), RuntimeError, "no logits"),
            (lambda: f(x, u.double(), tokens), TypeError, "uniforms has dtype"),
            (lambda: f(x, u[:3], tokens), ValueError, "uniforms has shape"),
            (lambda: f(x, u, tokens.float()), TypeError, "tokens has dtype"),
            (lambda: f(x, u, tokens[:2]), ValueError, "tokens has shape"),
            (lambda: f(x, u, tokens, u.half()), TypeError, "logprobs has dtype"),
            (lambda: f(x, u, tokens, temperature=-1.0), RuntimeError, "temperature"),
            (lambda: f(x, u, tokens, temperature=INF), RuntimeError, "temperature"),
            (lambda: f(x, u, tokens, temperature=u.half()), TypeError, "temperature has dtype"),
            (lambda: f(x, u, tokens, top_k=u), TypeError, "top_k has dtype"),
            (lambda: f(x, u, tokens, top_k=2.5), TypeError, "integer"),
            (lambda: f(x, u, tokens, top_p=math.nan), RuntimeError, "top_p"),
            (lambda: f(x, u, tokens, min_p=u[:1]), ValueError, "min_p has shape"),
            (lambda: f(x, u.cpu(), tokens), ValueError, "uniforms must be a GPU tensor")):
        with pytest.raises(error, match=text):
            call()
