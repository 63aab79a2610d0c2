"""Log probabilities of given tokens, entropy, alternatives and the gradient of
the logits, against 64 bits.

Tolerances: with l the scaled logits of a row (their size L = max |l| over its
finite ones), the products scale * x and their difference from the maximum cost
a few roundings of 2^-24 of L, and the sums and the logarithm 40 more of their
results: 8 * 2^-24 * L + 40 * 2^-24 * (1 + |result|) bounds each value. A
gradient has that error relative to p, then one rounding to its type."""
import math

import pytest
import torch

import lm_reference as ref
from mlir_edsl_hip import last_plan, lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def make(M, V, dtype, pad=0, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    t = torch.zeros(M, V + pad, dtype=dtype, device="cuda")[:, pad:]
    t.copy_((spread * torch.randn(M, V, generator=g)).to(dtype))
    tokens = torch.randint(0, V, (M,), generator=g).cuda()
    return t, tokens


def call(x, tokens, k=0, scale=1.0, **kw):
    M = x.shape[0]
    ids = tokens.dtype if tokens is not None else torch.int64
    out = dict(logprobs=torch.full((M,), 7.0, device="cuda") if tokens is not None else None,
               lse=torch.full((M,), 7.0, device="cuda"), entropy=torch.full((M,), 7.0, device="cuda"),
               top_logprobs=torch.full((M, k), 7.0, device="cuda") if k else None,
               top_ids=torch.full((M, k), 77, dtype=ids, device="cuda") if k else None)
    lm.token_logprobs_launch(x, tokens, scale=scale, **out, **kw)
    return out


def same(got, want, L):
    got, want = ref.d(got), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok = ~torch.isnan(want) & ~inf
    bound = 8 * U * L.expand_as(want) + 40 * U * (1 + want.abs())
    worst = ((got - want).abs() - bound)[ok]
    assert worst.numel() == 0 or float(worst.max()) <= 0, float(worst.max())


def check(x, tokens, k=0, scale=1.0):
    out = call(x, tokens, k, scale)
    lp, lse, ent, top, ids = ref.token_logprobs(x, tokens, k, scale)
    l = scale * ref.d(x)
    L = torch.where(torch.isfinite(l), l.abs(), 0.0).amax(1)
    if tokens is not None:
        same(out["logprobs"], lp, L)
    same(out["lse"], lse, L)
    same(out["entropy"], ent, L)
    if k:
        assert torch.equal(out["top_ids"].cpu().long(), ids)
        same(out["top_logprobs"], top, L[:, None])
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 64, 32), (4, 100, 3), (7, 1000, 5),
                                   (2, 2049, 8), (1, 8191, 32), (3, 16385, 4), (300, 2500, 2), (1, 50256, 8),
                                   (270, 50257, 5), (2, 131072, 20), (260, 70001, 32),
                                   (3, 200003, 32), (300, 66000, 5)])
def test_sizes(M, V, k, dtype):
    x, tokens = make(M, V, dtype, V % 5, V)
    check(x, tokens, k, 1.25)


def test_one_launch_or_parts():
    x, tokens = make(1, 131073, BF16)
    call(x, tokens, 4)
    assert "+join" in last_plan()
    x, tokens = make(512, 4096, BF16)
    call(x, tokens, 4)
    assert "parts=1" in last_plan()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,V", [(9, 777), (6, 40000), (300, 5000)])
def test_masked_rows(M, V, dtype):
    """Rows with few values left, one, none; masks by -inf and by the type's lowest value."""
    x, tokens = make(M, V, dtype, 1, 3)
    x[1] = -math.inf
    x[2, 1:] = -math.inf
    x[3, :-1] = -math.inf
    x[4, torch.arange(V, device="cuda") % 97 != 5] = -math.inf
    x[5, 7:] = torch.finfo(dtype).min
    tokens[0], tokens[2], tokens[4] = -100, 0, V
    check(x, tokens, 20)


@pytest.mark.parametrize("scale", [0.25, 1.0])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_of_the_lowest_value(dtype, scale):
    """Equal logits, whatever they are, are equal probabilities."""
    V = 3000
    x = torch.full((3, V), torch.finfo(dtype).min, dtype=dtype, device="cuda")
    x[1] = 0.0
    x[2] = 100.0
    out = call(x, torch.tensor([5, 6, 7], device="cuda"), 6, scale)
    for key in ("logprobs", "top_logprobs"):
        assert (out[key] + math.log(V)).abs().max() <= 60 * U * math.log(V)
    assert (out["entropy"] - math.log(V)).abs().max() <= 60 * U * math.log(V)
    assert torch.equal(out["top_ids"].cpu(), torch.arange(6).expand(3, 6))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [500, 60000])
def test_ties_and_orders(V, dtype):
    """Equal values in many places, rising and falling rows, zeros of both signs,
    large values in few lanes: the lists that overflow among them."""
    x = torch.zeros(8, V, dtype=dtype, device="cuda")
    j = torch.arange(V, device="cuda")
    x[1] = (j // 7).to(dtype)
    x[2] = (-(j // 3)).to(dtype)
    x[3, ::2] = -0.0
    x[4] = (j % 512 < 8).to(dtype) * (1 + j % 13).to(dtype)
    x[5] = (j % 5).to(dtype)
    x[6] = torch.where(j % 2 == 0, -math.inf, 1.5)
    x[7, V // 2:] = 3.0
    check(x, (j[:8] * (V // 8)).clone(), 32)


def test_rows_that_are_not_numbers():
    for V in (600, 50000):
        x, tokens = make(6, V, F32, seed=4)
        x[1, V - 1], x[3, 0], x[4] = math.nan, math.inf, math.nan
        x[5, 2:] = -math.inf
        x[5, 1] = math.nan
        tokens[3] = -1
        check(x, tokens, 5)


def test_outputs_are_optional_and_ids_32_bits():
    x, tokens = make(5, 900, BF16, seed=5)
    out = check(x, tokens.int(), 7)
    assert out["top_ids"].dtype == torch.int32
    check(x, None, 3)
    lse = torch.empty(5, device="cuda")
    lm.token_logprobs_launch(x, lse=lse)
    assert torch.equal(lse, out["lse"])
    lm.token_logprobs_launch(x)  # nothing asked for
    lm.token_logprobs_launch(x[:0], tokens[:0], lse[:0])


def test_the_same_bits_again():
    x, tokens = make(64, 32001, F16, seed=6)
    a, b = call(x, tokens, 20), call(x, tokens, 20)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,V", [(1, 1), (3, 5), (4, 1000), (3, 8193), (2, 50257)])
@pytest.mark.parametrize("parts", ["both", "logprobs", "entropy"])
def test_backward(M, V, dtype, parts):
    x, tokens = make(M, V, dtype, 1, 7)
    if M > 2:
        x[1] = -math.inf
        x[2, : V // 2] = -math.inf
        tokens[0] = -100
    fwd = call(x, tokens, 0, 0.7)
    g = torch.Generator().manual_seed(8)
    a = dict(dlogprobs=torch.randn(M, generator=g).cuda() if parts != "entropy" else None,
             dentropy=torch.randn(M, generator=g).cuda() if parts != "logprobs" else None)
    dx = torch.full((M, V + 2), 7.0, dtype=dtype, device="cuda")[:, 2:]
    lm.token_logprobs_backward_launch(x, tokens, fwd["lse"], dx, entropy=fwd["entropy"], scale=0.7, **a)
    want = ref.token_logprobs_backward(x, tokens, fwd["lse"], entropy=fwd["entropy"], scale=0.7, **a)
    # p's relative error is the absolute one of its exponent: a few roundings of |l| + |lse| + 200 at most.
    lse = torch.where(torch.isfinite(ref.d(fwd["lse"])), ref.d(fwd["lse"]), 0.0)[:, None]
    l = torch.where(torch.isfinite(ref.d(x)), 0.7 * ref.d(x), 0.0)
    p = torch.where(torch.isfinite(ref.d(x)), (l - lse).exp(), 0.0)
    size = (0 if a["dlogprobs"] is None else ref.d(a["dlogprobs"]).abs()[:, None])
    if a["dentropy"] is not None:
        size = size + ref.d(a["dentropy"]).abs()[:, None] * ((l - lse).abs() + ref.d(fwd["entropy"]).abs()[:, None])
    bound = 8 * U * (2 + l.abs() + lse.abs()) * p * size + 4 * U * size * (p > 0) \
        + (ref.HALF_ULP[dtype] * 1.001 + 8 * U) * want.abs() + ref.TINY[dtype]
    got = ref.d(dx)
    assert not torch.isnan(got).any()
    worst = float(((got - want).abs() - bound).max())
    assert worst <= 0, worst
    same_place = x.clone()
    lm.token_logprobs_backward_launch(same_place, tokens, fwd["lse"], same_place, entropy=fwd["entropy"], scale=0.7, **a)
    assert torch.equal(same_place, dx)


def test_backward_against_differences():
    """The directional derivative of sum(g logprobs) + sum(gh entropy), by central differences in 64 bits."""
    M, V, scale = 4, 700, 1.3
    x, tokens = make(M, V, F32, seed=9)
    fwd = call(x, tokens, 0, scale)
    gen = torch.Generator().manual_seed(10)
    g, gh = torch.randn(M, generator=gen).cuda(), torch.randn(M, generator=gen).cuda()
    dx = torch.empty_like(x)
    lm.token_logprobs_backward_launch(x, tokens, fwd["lse"], dx, dlogprobs=g, entropy=fwd["entropy"], dentropy=gh,
                                      scale=scale)
    v = torch.randn(M, V, generator=gen, dtype=torch.float64)

    def value(x):
        lp, _, ent, _, _ = ref.token_logprobs(x, tokens.cpu(), 0, scale)
        return float((ref.d(g) * lp).sum() + (ref.d(gh) * ent).sum())
    e = 1e-5
    diff = (value(ref.d(x) + e * v) - value(ref.d(x) - e * v)) / (2 * e)
    got = float((ref.d(dx) * v).sum())
    assert abs(got - diff) <= 1e-4 * math.sqrt(M)


def test_another_stream_and_graph_replays():
    x, tokens = make(2, 50256, BF16, seed=11)
    lp, top, ids = torch.empty(2, device="cuda"), torch.empty(2, 4, device="cuda"), torch.empty(2, 4, dtype=torch.int64, device="cuda")
    step = lambda s=None: lm.token_logprobs_launch(x, tokens, lp, top_logprobs=top, top_ids=ids, stream=s)  # noqa: E731
    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    want = [t.clone() for t in (lp, top, ids)]
    torch.cuda.synchronize()
    lp.zero_()
    s.wait_stream(torch.cuda.current_stream())
    step(s)
    s.synchronize()
    assert torch.equal(lp, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        x.copy_(make(2, 50256, BF16, seed=40 + seed)[0])
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in (lp, top, ids)]
        top.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((lp, top, ids), want))


@pytest.mark.parametrize("change,error", [
    (dict(logits=lambda t: t.cpu()), ValueError), (dict(logits=lambda t: t.int()), TypeError),
    (dict(logits=lambda t: t[:, ::2]), ValueError), (dict(tokens=lambda t: t.float()), TypeError),
    (dict(tokens=lambda t: t[1:]), ValueError), (dict(tokens=lambda t: None), ValueError),
    (dict(logprobs=lambda t: t.half()), TypeError), (dict(top_logprobs=lambda t: None), ValueError),
    (dict(top_ids=lambda t: t.int()), TypeError), (dict(scale=lambda t: 0.0), RuntimeError),
    (dict(scale=lambda t: math.inf), RuntimeError),
    (dict(top_logprobs=lambda t: torch.empty(4, 33, device="cuda"),
          top_ids=lambda t: torch.empty(4, 33, device="cuda", dtype=torch.int64)), RuntimeError),
    (dict(logits=lambda t: t[:, :2]), RuntimeError)])
def test_refusals(change, error):
    a = dict(logits=torch.ones(4, 50, device="cuda"), tokens=torch.zeros(4, dtype=torch.int64, device="cuda"),
             logprobs=torch.empty(4, device="cuda"), top_logprobs=torch.empty(4, 3, device="cuda"),
             top_ids=torch.empty(4, 3, dtype=torch.int64, device="cuda"), scale=1.0)
    for name, f in change.items():
        a[name] = f(a[name])
    with pytest.raises(error):
        lm.token_logprobs_launch(**a)


def test_backward_refusals():
    x, tokens = make(4, 50, F32)
    v = torch.ones(4, device="cuda")
    for kw in (dict(tokens=None, dlogprobs=v), dict(dentropy=v), dict(dlogprobs=v[1:]), dict(lse=v.half()),
               dict(dlogits=x.half())):
        a = dict(logits=x, tokens=tokens, lse=v, dlogits=torch.empty_like(x)) | kw
        with pytest.raises((TypeError, ValueError)):
            lm.token_logprobs_backward_launch(**a)
