"""RMS norm with the residual's addition, 8-bit outputs and the backward pass,
against 64 bits.

Tolerances: a value that is computed in 32 bits and rounded once to its type is
within half a unit in the last place plus the 32-bit arithmetic, whose relative
error is at most (N / threads + 20) roundings of 2^-24 for the sum of squares
(halved by the root) and a few for the products: 32 roundings cover every size
here."""
import math

import pytest
import torch

import lm_reference as ref
from mlir_edsl_hip import last_plan, lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ARITH = 32 * 2.0 ** -24


def close(got, want, dtype, arith=ARITH, mag=None):
    """|got - want| within one rounding to dtype and `arith` of |want| (or of `mag`, what a sum's terms amount to)."""
    got, want = ref.d(got), ref.d(want)
    bound = (ref.HALF_ULP[dtype] * 1.001 + arith) * want.abs() + ref.TINY[dtype]
    if mag is not None:
        bound = bound + arith * ref.d(mag)
    worst = (got - want).abs() - bound
    assert not torch.isnan(worst).any()
    assert float(worst.max()) <= 0, f"off by {float(worst.max()):.3g} more than allowed"


def rows(M, N, dtype, pad=0, seed=0, scale=1.0):
    """[M, N] with a row stride of N + pad, starting `pad` elements into its memory."""
    g = torch.Generator().manual_seed(seed)
    t = torch.zeros(M, N + pad, dtype=dtype, device="cuda")[:, pad:]
    t.copy_((scale * torch.randn(M, N, generator=g)).to(dtype))
    return t


SIZES = [(1, 1), (3, 7), (5, 64), (37, 128), (41, 250), (2, 257), (7, 512), (4, 1000), (3, 2001), (2, 4096), (3, 8200), (2, 16384),
         (2, 32771), (1, 70001)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,N", SIZES)
def test_forward(M, N, dtype):
    pad = N % 3
    x, r = rows(M, N, dtype, pad, 1), rows(M, N, dtype, 2 * pad, 2, 2.0)
    w = (1 + 0.2 * torch.randn(N, generator=torch.Generator().manual_seed(3))).to(dtype).cuda()
    y, total, rstd = rows(M, N, dtype, pad + 1), rows(M, N, dtype, 1), torch.empty(M, device="cuda")
    lm.rms_norm_launch(x, w, y, residual=r, total=total, rstd=rstd, eps=1e-5)
    assert last_plan().startswith("rms_norm ")
    want, h, wr = ref.rms_norm(x, w, r, 1e-5)
    close(total, h, dtype, 2.0 ** -24)
    close(rstd, wr, F32)
    close(y, want, dtype, mag=(ref.d(x).abs() + ref.d(r).abs()) * wr[:, None] * ref.d(w).abs())
    lm.rms_norm_launch(x, w.float(), y, eps=1e-5)  # no residual, weight in f32
    close(y, ref.rms_norm(x, w, None, 1e-5)[0], dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("M,N", [(1, 1), (3, 7), (4, 1000), (3, 2001), (2, 8200), (1, 40000)])
def test_eight_bits(M, N, out, dtype):
    x, r = rows(M, N, dtype, 1, 4), rows(M, N, dtype, 0, 5)
    w = (1 + 0.2 * torch.randn(N, generator=torch.Generator().manual_seed(6))).cuda()
    x[-1, :] *= 0 if M > 1 else 1
    r[-1, :] *= 0 if M > 1 else 1
    y, scales = torch.empty(M, N + 3, dtype=torch.int8, device="cuda")[:, 3:].view(out), torch.empty(M, device="cuda")
    lm.rms_norm_launch(x, w, y, residual=r, scales=scales)
    want, _, _ = ref.rms_norm(x, w, r)
    top = 127.0 if out == torch.int8 else 448.0
    s = want.abs().amax(1) / top
    assert ((ref.d(scales) - s).abs() <= ARITH * s).all()
    codes, exact = ref.d(y.to(F32)), torch.where(s[:, None] > 0, want / s[:, None], 0.0)
    # Half a step of the code (integers; 1/16 of the value, 2^-10 near zero), and the 32-bit arithmetic before it.
    half = 0.5 if out == torch.int8 else (exact.abs() / 16).clamp(min=2.0 ** -10)
    assert ((codes - exact).abs() <= half + 2 * ARITH * (exact.abs() + top * 2.0 ** -12)).all()
    assert codes.abs().max() <= top


@pytest.mark.parametrize("out", [F32, torch.int8, torch.float8_e4m3fn])
def test_rows_that_are_not_numbers(out):
    x = rows(6, 300, F32, seed=7)
    x[1, 299], x[3, 0], x[4] = math.nan, math.inf, 0.0
    w = torch.ones(300, device="cuda")
    y = torch.empty(6, 300, device="cuda").to(out)
    scales = torch.empty(6, device="cuda") if out != F32 else None
    lm.rms_norm_launch(x, w, y, scales=scales)
    bad = torch.tensor([False, True, False, True, False, False])
    if out == F32:
        assert torch.equal(torch.isnan(y).any(1).cpu(), bad)
        assert (y[4] == 0).all()
    else:
        assert torch.equal(torch.isnan(scales).cpu(), bad)
        assert scales[4] == 0 and (y[4].float() == 0).all()


@pytest.mark.parametrize("N", [96, 5000, 40000])
def test_outputs_in_the_inputs_memory(N):
    x, r = rows(3, N, BF16, seed=8), rows(3, N, BF16, seed=9)
    w = torch.ones(N, device="cuda", dtype=BF16)
    y, total = torch.empty_like(x), torch.empty_like(x)
    lm.rms_norm_launch(x, w, y, residual=r, total=total)
    x2, r2 = x.clone(), r.clone()
    lm.rms_norm_launch(x2, w, x2, residual=r2, total=r2)
    assert torch.equal(x2, y) and torch.equal(r2, total)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,N", SIZES + [(1500, 130), (3000, 9), (300, 16384), (3, 12001)])
def test_backward(M, N, dtype):
    x, dy, dh = rows(M, N, dtype, 1, 10), rows(M, N, dtype, 0, 11), rows(M, N, dtype, 2, 12)
    w = (1 + 0.2 * torch.randn(N, generator=torch.Generator().manual_seed(13))).to(dtype).cuda()
    rstd = ref.rms_norm(x, w)[2].float().cuda()
    dx, dw = rows(M, N, dtype, 3), torch.full((N,), math.nan, device="cuda")
    lm.rms_norm_backward_launch(dy, x, w, rstd, dx, dweight=dw, dh=dh)
    wx, ww = ref.rms_norm_backward(dy, x, w, rstd, dh)
    # The terms of dx: t rstd, its mean against xh (|mean| <= the mean of |t xh|), and dh.
    t, xh = (ref.d(dy) * ref.d(w)).abs(), (ref.d(x) * ref.d(rstd)[:, None]).abs()
    terms = ref.d(rstd)[:, None] * (t + xh * (t * xh).mean(1, keepdim=True)) + ref.d(dh).abs()
    close(dx, wx, dtype, mag=terms)
    # A column's sum: at most M / groups + groups / 16 + 16 additions in a row.
    close(dw, ww, F32, (M + 64) * 2.0 ** -24, mag=(ref.d(dy).abs() * xh).sum(0))
    again = torch.empty_like(dw)
    lm.rms_norm_backward_launch(dy, x, w, rstd, dx, dweight=again)
    assert torch.equal(again, dw)
    close(dx, ref.rms_norm_backward(dy, x, w, rstd)[0], dtype, mag=terms)


def test_backward_against_differences():
    """The directional derivative of sum(y * g) + sum(total * gh), by central differences in 64 bits."""
    M, N = 5, 333
    x, r = rows(M, N, F32, seed=14), rows(M, N, F32, seed=15)
    w = (1 + 0.2 * torch.randn(N, generator=torch.Generator().manual_seed(16))).cuda()
    g, gh = rows(M, N, F32, seed=17), rows(M, N, F32, seed=18)
    y, total, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(M, device="cuda")
    lm.rms_norm_launch(x, w, y, residual=r, total=total, rstd=rstd)
    dx, dw = torch.empty_like(x), torch.empty(N, device="cuda")
    lm.rms_norm_backward_launch(g, total, w, rstd, dx, dweight=dw, dh=gh)

    def value(x, w):
        out, h, _ = ref.rms_norm(x, w, r)
        return float((out * ref.d(g)).sum() + (h * ref.d(gh)).sum())
    gen = torch.Generator().manual_seed(19)
    vx, vw = torch.randn(M, N, generator=gen, dtype=torch.float64), torch.randn(N, generator=gen, dtype=torch.float64)
    e = 1e-5
    diff = (value(ref.d(x) + e * vx, ref.d(w) + e * vw) - value(ref.d(x) - e * vx, ref.d(w) - e * vw)) / (2 * e)
    got = float((ref.d(dx) * vx).sum() + (ref.d(dw) * vw).sum())
    # 1665 products of size one, each with 32 roundings; the difference quotient is good to e^2.
    assert abs(got - diff) <= 1e-4 * math.sqrt(M * N)


def test_no_rows():
    e = torch.empty(0, 40, device="cuda")
    w, dw = torch.ones(40, device="cuda"), torch.ones(40, device="cuda")
    lm.rms_norm_launch(e, w, e.clone(), rstd=torch.empty(0, device="cuda"))
    lm.rms_norm_backward_launch(e, e, w, torch.empty(0, device="cuda"), e.clone(), dweight=dw)
    assert (dw == 0).all()


def test_another_stream():
    x, w = rows(64, 4096, BF16, seed=20), torch.ones(4096, device="cuda", dtype=BF16)
    y = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    lm.rms_norm_launch(x, w, y, stream=s)
    s.synchronize()
    close(y, ref.rms_norm(x, w)[0], BF16)


X = dict(M=4, N=16)


@pytest.mark.parametrize("change,error", [
    (dict(x=lambda x: x.cpu()), ValueError), (dict(x=lambda x: x.double()), TypeError),
    (dict(x=lambda x: x.t()), ValueError), (dict(x=lambda x: x[0]), ValueError),
    (dict(w=lambda w: w[:-1]), ValueError), (dict(w=lambda w: w.half()), TypeError),
    (dict(w=lambda w: torch.ones(32, device="cuda")[::2]), ValueError),
    (dict(y=lambda y: y.bfloat16()), TypeError), (dict(y=lambda y: y[:, 1:]), ValueError),
    (dict(y=lambda y: y.to(torch.int8)), ValueError), (dict(scales=lambda s: torch.ones(4, device="cuda")), ValueError),
    (dict(residual=lambda s: torch.ones(4, 15, device="cuda")), ValueError),
    (dict(rstd=lambda s: torch.ones(3, device="cuda")), ValueError),
    (dict(eps=lambda s: -1.0), RuntimeError), (dict(eps=lambda s: math.nan), RuntimeError)])
def test_refusals(change, error):
    a = dict(x=torch.ones(4, 16, device="cuda"), w=torch.ones(16, device="cuda"), y=torch.full((4, 16), 7.0, device="cuda"),
             scales=None, residual=None, rstd=None, eps=1e-6)
    for name, f in change.items():
        a[name] = f(a[name])
    with pytest.raises(error):
        lm.rms_norm_launch(a["x"], a["w"], a["y"], residual=a["residual"], scales=a["scales"], rstd=a["rstd"],
                           eps=a["eps"])


@pytest.mark.parametrize("name,make", [
    ("h", lambda: torch.ones(4, 15, device="cuda")), ("h", lambda: torch.ones(4, 16, device="cuda").half()),
    ("rstd", lambda: torch.ones(5, device="cuda")), ("dx", lambda: torch.ones(16, 4, device="cuda").t()),
    ("dweight", lambda: torch.ones(16, device="cuda").half()), ("dh", lambda: torch.ones(4, 16))])
def test_backward_refusals(name, make):
    one = lambda: torch.ones(4, 16, device="cuda")  # noqa: E731
    a = dict(dy=one(), h=one(), w=torch.ones(16, device="cuda"), rstd=torch.ones(4, device="cuda"), dx=one(),
             dweight=None, dh=None)
    a[name] = make()
    with pytest.raises((TypeError, ValueError)):
        lm.rms_norm_backward_launch(a["dy"], a["h"], a["w"], a["rstd"], a["dx"], dweight=a["dweight"], dh=a["dh"])


def test_graph_replays():
    x, w = rows(32, 1024, BF16, seed=21), torch.ones(1024, device="cuda", dtype=BF16)
    dy, rstd = rows(32, 1024, BF16, seed=22), torch.empty(32, device="cuda")
    y, dx, dw = torch.empty_like(x), torch.empty_like(x), torch.empty(1024, device="cuda")

    def step():
        lm.rms_norm_launch(x, w, y, rstd=rstd)
        lm.rms_norm_backward_launch(dy, x, w, rstd, dx, dweight=dw)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        x.copy_(rows(32, 1024, BF16, seed=30 + seed))
        step()
        torch.cuda.synchronize()
        want = y.clone(), dx.clone(), dw.clone()
        for t in (y, dx, dw):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, dx, dw), want):
            assert torch.equal(a, b)
