"""The dense layer in 8-bit integers against 64 bits.

Tolerance: the integer sum is exact and rounds to f32 once, then two products, the
bias's sum and up to two operations of the activation round, 2^-24 of |z| + |b|
each, and the output's type once."""
import pytest
import torch

import lm_layers_reference as layers
import lm_reference as ref
from mlir_edsl_hip import _native, last_plan, lm

pytestmark = pytest.mark.gpu
F32, BF16, F16, I8 = torch.float32, torch.bfloat16, torch.float16, torch.int8
ALPHA = 0.3
EPI = {"none": _native.EPI_NONE, "bias": _native.EPI_BIAS, "relu": _native.EPI_RELU,
       "bias_relu": _native.EPI_BIAS_RELU, "leaky": _native.EPI_LEAKY, "bias_leaky": _native.EPI_BIAS_LEAKY,
       "if_relu": _native.EPI_IF_RELU, "bias_if_relu": _native.EPI_BIAS_IF_RELU}


def integers(M, K, seed, pad=0, low=-128):
    v = torch.randint(low, 128, (M, K), generator=torch.Generator().manual_seed(seed)).to(I8)
    t = torch.full((M, K + pad), 77, dtype=I8, device="cuda")[:, pad:]
    t.copy_(v)
    return t


def floats(*shape, seed, dtype=F32):
    return (0.5 + torch.rand(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def check(M, K, N, y=F32, epi="none", xs=True, scales=F32, b=F32, pad=0, ypad=0, plan=None):
    x, q = integers(M, K, 1, pad), integers(K, N, 2, pad)
    s, rows = floats(N, seed=3, dtype=scales) / 512, floats(M, seed=4) if xs else None
    bias = (8 * floats(N, seed=5) - 8).to(b) if epi.startswith("bias") else None
    out = torch.full((M, N + ypad), 5.0, dtype=y, device="cuda")
    Y = out[:, ypad // 2:ypad // 2 + N]
    W = lm.i8_pack(q, s)
    lm.i8_dense_launch(x, W, bias, Y, EPI[epi], ALPHA, x_scales=rows)
    assert plan is None or plan in last_plan(), last_plan()
    want, size = layers.i8_dense(x, q, s, rows, bias, EPI[epi], ALPHA)
    bound = 7 * 2.0 ** -24 * size + ref.HALF_ULP[y] * want.abs() + ref.TINY[y]
    assert float(((ref.d(Y) - want).abs() - bound).max()) <= 0
    around = out.clone()
    around[:, ypad // 2:ypad // 2 + N] = 5.0
    assert bool((around == 5.0).all())


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 48, 49, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("K,N", [(1, 1), (16, 16), (64, 48), (63, 17), (129, 130), (1024, 96), (2113, 259)])
def test_sizes(M, K, N):
    check(M, K, N)


@pytest.mark.parametrize("M,N", [(3, 100), (40, 100), (100, 100), (700, 1502)])
@pytest.mark.parametrize("y", [F32, BF16, F16])
@pytest.mark.parametrize("epi", list(EPI))
def test_types_and_epilogues(M, N, y, epi):
    check(M, 320, N, y=y, epi=epi, scales=y, b=F16 if y == F32 else y)


@pytest.mark.parametrize("M,K,N,plan", [
    (1, 4096, 12000, "skinny rows=16 cols=32"), (1, 4096, 20000, "skinny rows=16 cols=64"), (40, 64, 9000, "direct"),
    (5, 64, 40000, "skinny rows=16 cols=64"), (64, 512, 700, "skinny rows=64 cols=16"),
    (33, 200, 6000, "skinny rows=48 cols=32"), (300, 512, 700, "skinny rows=64 cols=16"), (130, 8192, 300, "skinny rows=48"),
    (70, 63, 17, "skinny rows=48"), (2100, 384, 8200, "direct"), (4200, 192, 4000, "direct"), (600, 512, 8192, "direct"),
    (4096, 128, 4096, "direct"), (700, 512, 1500, "direct"), (701, 500, 1501, "any"), (65, 640, 40000, "direct"),
    (700, 1, 1500, "any"), (4097, 16, 130, "direct")])
def test_kernels(M, K, N, plan):
    check(M, K, N, y=BF16, epi="bias_relu", b=BF16, plan=plan)


@pytest.mark.parametrize("M,N", [(5, 130), (70, 130), (260, 130), (900, 1130)])
@pytest.mark.parametrize("pad", [1, 8, 16])
def test_strides_and_alignments(M, N, pad):
    check(M, 272, N, y=F16, pad=pad, ypad=3, xs=False)


@pytest.mark.parametrize("M,N", [(1, 33), (70, 33), (513, 1040)])
def test_largest_sums_are_exact(M, N):
    # All values at an end: the largest sum that 32 bits hold, and the deepest layer.
    K = 2 ** 17 - 1
    for a, b in ((-128, -128), (127, -128)):
        x, q = torch.full((M, K), a, dtype=I8, device="cuda"), torch.full((K, N), b, dtype=I8, device="cuda")
        Y = torch.empty(M, N, device="cuda")
        lm.i8_dense_launch(x, lm.i8_pack(q, torch.ones(N, device="cuda")), None, Y)
        assert bool((Y == float(torch.tensor(K * a * b, dtype=F32))).all())


def test_rows_of_the_norm():
    """The norm's 8-bit rows, quantized weights: the layer of the float matrices, up to their roundings."""
    M, K, N = 37, 512, 300
    g = torch.Generator().manual_seed(6)
    x, W = torch.randn(M, K, generator=g).cuda(), (torch.randn(K, N, generator=g) / 20).cuda()
    q, s = torch.empty(M, K, dtype=I8, device="cuda"), torch.empty(M, device="cuda")
    lm.rms_norm_launch(x, torch.ones(K, device="cuda"), q, scales=s)
    Q, scales = lm.i8_quantize(W)
    # A quotient rounds to the nearest integer, and the 32-bit division before that.
    assert float((ref.d(Q) * ref.d(scales) - ref.d(W)).abs().max()) <= float(ref.d(scales).max()) * 0.50001
    Y = torch.empty(M, N, device="cuda")
    lm.i8_dense_launch(q, lm.i8_pack(Q, scales), None, Y, x_scales=s)
    want, size = layers.i8_dense(q, Q, scales, s)
    assert float(((ref.d(Y) - want).abs() - 7 * 2.0 ** -24 * size - ref.TINY[F32]).max()) <= 0


def test_a_column_of_zeros_and_no_rows():
    W = torch.zeros(8, 3, device="cuda")
    W[:, 1] = 2.0
    Q, scales = lm.i8_quantize(W)
    assert Q[:, 0].tolist() == [0] * 8 and float(scales[0]) == 0 and Q[:, 1].tolist() == [127] * 8
    P = lm.i8_pack(Q, scales)
    assert "8x3" in repr(P)
    lm.i8_dense_launch(torch.zeros(0, 8, dtype=I8, device="cuda"), P, None, torch.zeros(0, 3, device="cuda"))
    assert last_plan() == "empty"


def test_another_stream_and_graph_replays():
    x, q = integers(700, 256, 1), integers(256, 1400, 2)
    P, Y = lm.i8_pack(q, floats(1400, seed=3)), torch.zeros(700, 1400, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    lm.i8_dense_launch(x, P, None, Y, stream=side)
    lm.i8_dense_launch(x[:5], P, None, Y[:5], stream=side)
    side.synchronize()
    want = Y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lm.i8_dense_launch(x, P, None, Y)
    for i in range(4):
        x.copy_(integers(700, 256, 10 + i))
        Y.zero_()
        graph.replay()
        got = Y.clone()
        lm.i8_dense_launch(x, P, None, Y)
        torch.cuda.synchronize()
        assert torch.equal(got, Y) and not torch.equal(got, want)


def test_refusals():
    x, q, s = integers(4, 32, 1), integers(32, 16, 2), floats(16, seed=3)
    P, Y = lm.i8_pack(q, s), torch.zeros(4, 16, device="cuda")
    for call, error, text in (
            (lambda: lm.i8_pack(q.float(), s), TypeError, "Q has dtype"),
            (lambda: lm.i8_pack(q[:0], s), RuntimeError, "K=0"),
            (lambda: lm.i8_pack(q, s[:-1]), ValueError, "scales has shape"),
            (lambda: lm.i8_pack(q, s.to(torch.float64)), TypeError, "scales has dtype"),
            (lambda: lm.i8_pack(q.t(), floats(32, seed=1)), ValueError, "unit inner stride"),
            (lambda: lm.i8_dense_launch(x, q, None, Y), TypeError, "not an I8Weight"),
            (lambda: lm.i8_dense_launch(x.float(), P, None, Y), TypeError, "X has dtype"),
            (lambda: lm.i8_dense_launch(x[:, :16], P, None, Y), ValueError, "shape mismatch"),
            (lambda: lm.i8_dense_launch(x, P, None, Y.int()), TypeError, "Y has dtype"),
            (lambda: lm.i8_dense_launch(x, P, None, Y[:3]), ValueError, "Y has shape"),
            (lambda: lm.i8_dense_launch(x, P, None, Y, _native.EPI_BIAS), RuntimeError, "bias is null"),
            (lambda: lm.i8_dense_launch(x, P, None, Y, 9), RuntimeError, "epilogue code 9"),
            (lambda: lm.i8_dense_launch(x, P, s[:3], Y, 1), ValueError, "b has shape"),
            (lambda: lm.i8_dense_launch(x, P, None, Y, x_scales=s), ValueError, "x_scales has shape"),
            (lambda: lm.i8_dense_launch(x.cpu(), P, None, Y), ValueError, "X must be a GPU tensor"),
            (lambda: lm.i8_quantize(q), ValueError, "2-D float")):
        with pytest.raises(error, match=text):
            call()
