"""The dense layer on 4-bit weights against 64 bits.

Tolerance: products are exact, so that an output is off by the roundings of its
sums alone. Its terms |x| s (q + z) pass through at most a group's sum (its
length), the sum over the groups and those over waves and slices (24): with one
unit of 2^-23 each (the matrix cores' sums may cut off), (min(K, 128) + K / 32 +
48) 2^-23 of the terms' sum. The row's scale, the bias and the activation cost a
few 2^-24 of the result, the output's type one rounding."""
import math

import pytest
import torch

import lm_reference as ref
from mlir_edsl_hip import _native, last_plan, lm

pytestmark = pytest.mark.gpu
F32, BF16, F16, I8, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
EPI = {"none": _native.EPI_NONE, "bias": _native.EPI_BIAS, "relu": _native.EPI_RELU,
       "bias_relu": _native.EPI_BIAS_RELU, "leaky": _native.EPI_LEAKY, "bias_leaky": _native.EPI_BIAS_LEAKY,
       "if_relu": _native.EPI_IF_RELU, "bias_if_relu": _native.EPI_BIAS_IF_RELU}
ALPHA = 0.25


def make_weights(K, N, group, scales=F32, zeros=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    G = -(-K // group)
    q = torch.randint(0, 16, (K, N), generator=g, dtype=torch.uint8).cuda()
    s = ((0.5 + torch.rand(G, N, generator=g)) / 8).to(scales).cuda()
    z = torch.randint(0, 16, (G, N), generator=g, dtype=torch.uint8).cuda() if zeros else None
    return q, s, z


def make_x(M, K, dtype, pad=0, seed=1):
    g = torch.Generator().manual_seed(seed)
    if dtype == I8:
        v = torch.randint(-128, 128, (M, K), generator=g).to(I8)
    elif dtype == E4M3:
        v = (100 * torch.randn(M, K, generator=g)).clamp(-448, 448).to(E4M3).view(I8)
    else:
        v = torch.randn(M, K, generator=g).to(dtype)
    t = torch.zeros(M, K + pad, dtype=v.dtype, device="cuda")[:, pad:]
    t.copy_(v)
    return t.view(E4M3) if dtype == E4M3 else t


def wide(x):
    return ref.d(x.float()) if x.dtype == E4M3 else ref.d(x)


def expect(x, q, s, z, group, b=None, epi="none", x_scales=None):
    """The layer, and the sum of its terms' sizes."""
    K = q.shape[0]
    at = torch.arange(K) // group
    s, z = ref.d(s)[at], ref.d(z)[at] if z is not None else 8.0
    row = ref.d(x_scales)[:, None] if x_scales is not None else 1.0
    y = wide(x) @ ((ref.d(q) - z) * s) * row
    size = wide(x).abs() @ ((ref.d(q) + z) * s) * row
    if "bias" in epi:
        y = y + ref.d(b)
    if epi.endswith("relu"):
        y = y.clamp(min=0)
    elif epi.endswith("leaky"):
        y = y.clamp(min=0) + ALPHA * y.clamp(max=0)
    return y, size


def check(got, want, size, K, b=None):
    bound = (min(K, 128) + K / 32 + 48) * 2.0 ** -23 * size
    bound = bound + 8 * 2.0 ** -24 * (want.abs() + (ref.d(b).abs() if b is not None else 0.0))
    bound = bound + ref.HALF_ULP[got.dtype] * 1.001 * (want.abs() + bound) + ref.TINY[got.dtype]
    worst = (ref.d(got) - want).abs() - bound
    assert not torch.isnan(worst).any()
    assert float(worst.max()) <= 0, float(worst.max())


def layer(M, K, N, group, x_dtype, y_dtype=None, scales=F32, zeros=True, epi="none", pad=0, seed=0):
    y_dtype = y_dtype or (x_dtype if x_dtype in (F32, BF16, F16) else BF16)
    x = make_x(M, K, x_dtype, pad, seed + 1)
    q, s, z = make_weights(K, N, group, scales, zeros, seed)
    xs = (torch.rand(M, generator=torch.Generator().manual_seed(seed + 2)) / 64).cuda() if x_dtype in (I8, E4M3) else None
    b = torch.randn(N, generator=torch.Generator().manual_seed(seed + 3)).to(y_dtype).cuda() if "bias" in epi else None
    y = torch.full((M, N + pad), 7.0, dtype=y_dtype, device="cuda")[:, pad:]
    W = lm.q4_pack(q, s, z, group_size=group)
    lm.q4_dense_launch(x, W, b, y, EPI[epi], ALPHA, x_scales=xs)
    want, size = expect(x, q, s, z, group, b, epi, xs)
    check(y, want, size, K, b)
    if pad:
        assert (y._base[:, :pad] == 7.0).all()
    return y


@pytest.mark.parametrize("x_dtype", [F32, BF16, F16, I8, E4M3])
@pytest.mark.parametrize("M,K,N,group", [
    (1, 1, 1, 32), (1, 128, 16, 128), (2, 31, 17, 32), (1, 1000, 100, 64), (16, 257, 33, 128), (5, 4096, 130, 128),
    (3, 2050, 520, 256), (16, 640, 4200, 64), (1, 384, 20000, 32), (17, 100, 20, 32), (31, 300, 129, 64),
    (33, 1024, 300, 128), (64, 129, 70, 32), (65, 512, 1000, 256), (130, 1000, 257, 64), (300, 384, 2100, 128),
    (513, 256, 4100, 32), (1100, 300, 4100, 64), (1060, 384, 4097, 32), (2000, 512, 2200, 128)])
def test_sizes(M, K, N, group, x_dtype):
    layer(M, K, N, group, x_dtype, zeros=(M + N) % 2 == 0, pad=N % 3, seed=M + K)


@pytest.mark.parametrize("M", [3, 40, 200])
@pytest.mark.parametrize("scales", [F32, BF16, F16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128, 384])
def test_groups_and_scales(group, zeros, scales, M):
    layer(M, 900, 150, group, BF16, F32, scales, zeros)


@pytest.mark.parametrize("M", [1, 50])
@pytest.mark.parametrize("epi", list(EPI))
@pytest.mark.parametrize("y_dtype", [F32, BF16, F16])
def test_epilogues(epi, y_dtype, M):
    layer(M, 256, 100, 64, F32, y_dtype, epi=epi)
    layer(M, 2048, 100, 128, I8, y_dtype, epi=epi)


def test_plans():
    for M, K, N, what in [(1, 16384, 64, "q4_small bf16 cols=16 ksplit=4 +join"), (16, 512, 8192, "cols=32 ksplit=1"),
                          (20, 512, 512, "q4_small bf16 cols=16 ksplit=1"), (20, 128, 20000, "q4_tile bf16 tile=32x128 teams=2 ksplit=1"),
                          (64, 4096, 8192, "q4_tile bf16 tile=64x128 teams=2 ksplit=4 +join"),
                          (512, 128, 4096, "q4_prep+q4_tile bf16 tile=64x128 teams=2 ksplit=1"),
                          (2048, 128, 4096, "q4_prep+q4_tile bf16 tile=64x128 teams=1 ksplit=1"),
                          (2048, 130, 4096, "q4_prep_copy+q4_tile")]:
        layer(M, K, N, 128, BF16)
        assert what in last_plan(), last_plan()


@pytest.mark.parametrize("M", [1, 16, 20, 100])
def test_integers_are_exact(M):
    """8-bit integers against integer weights: exact sums, whatever the order."""
    K, N = 1024, 200
    x, (q, _, _) = make_x(M, K, I8), make_weights(K, N, 128)
    one = torch.ones(K // 128, N, device="cuda")
    y = torch.empty(M, N, device="cuda")
    lm.q4_dense_launch(x, lm.q4_pack(q, one), None, y)
    assert torch.equal(ref.d(y), ref.d(x) @ (ref.d(q) - 8))


@pytest.mark.parametrize("M", [4, 64])
def test_f32_keeps_its_bits(M):
    """One non-zero weight a column picks elements of x: all 24 bits come back."""
    K = N = 256
    x = make_x(M, K, F32) * torch.logspace(-12, 12, M, device="cuda")[:, None]
    q = torch.full((K, N), 8, dtype=torch.uint8, device="cuda")
    q.fill_diagonal_(9)
    zeros = torch.zeros(K // 32, N, dtype=torch.uint8, device="cuda")
    y = torch.empty(M, N, device="cuda")
    picked = torch.zeros(K, N, dtype=torch.uint8, device="cuda").fill_diagonal_(1)
    lm.q4_dense_launch(x, lm.q4_pack(picked, torch.ones(K // 32, N, device="cuda"), zeros, group_size=32), None, y)
    assert torch.equal(y, x)


@pytest.mark.parametrize("M", [2, 70])
def test_rows_that_are_not_numbers(M):
    x = make_x(M, 300, BF16)
    x[1, 299] = math.inf
    x[0, 0] = math.nan
    q, s, z = make_weights(300, 90, 64)
    y = torch.empty(M, 90, dtype=BF16, device="cuda")
    lm.q4_dense_launch(x, lm.q4_pack(q, s, z, group_size=64), None, y)
    assert torch.isnan(y[:2]).all() and not torch.isnan(y[2:]).any()


def test_what_lies_around_x_is_not_read_into_it():
    """Rows end inside a block: what follows them in memory is NaN."""
    for M in (3, 40):
        for dtype in (F32, BF16, F16):
            mem = torch.full((M, 500), math.nan, dtype=dtype, device="cuda")
            mem[:, 100:333] = make_x(M, 233, dtype)
            q, s, z = make_weights(233, 40, 128)
            y = torch.empty(M, 40, dtype=dtype, device="cuda")
            lm.q4_dense_launch(mem[:, 100:333], lm.q4_pack(q, s, z), None, y)
            want, size = expect(mem[:, 100:333], q, s, z, 128)
            check(y, want, size, 233)


# Wide layers on four and two waves of a workgroup: blocks of K that the waves do
# not share evenly, odd widths, whole and broken last blocks.
@pytest.mark.parametrize("x_dtype", [F32, BF16, F16, I8, E4M3])
@pytest.mark.parametrize("M,K,N,group,waves", [
    (1, 130, 8161, 64, 4), (7, 1024, 8200, 128, 4), (16, 897, 4129, 32, 4), (3, 1200, 25000, 128, 4),
    (1, 1, 33001, 32, 2), (16, 448, 33000, 256, 2), (5, 512, 32801, 64, 2)])
def test_fewer_waves(M, K, N, group, waves, x_dtype):
    layer(M, K, N, group, x_dtype, zeros=(M + N) % 2 == 0, epi="bias", pad=N % 3, seed=M + K)
    assert f"cols=32 ksplit=1 waves={waves}" in last_plan(), last_plan()


def test_no_rows_no_columns_no_depth():
    q, s, z = make_weights(64, 40, 64)
    W = lm.q4_pack(q, s, z, group_size=64)
    lm.q4_dense_launch(torch.empty(0, 64, device="cuda"), W, None, torch.empty(0, 40, device="cuda"))
    lm.q4_dense_launch(torch.ones(3, 64, device="cuda"), lm.q4_pack(q[:, :0], s[:, :0], group_size=64), None,
                       torch.empty(3, 0, device="cuda"))
    empty = lm.q4_pack(q[:0], s[:0])
    for M in (3, 30):
        y, b = torch.full((M, 40), 7.0, device="cuda"), torch.arange(40.0, device="cuda") - 20
        lm.q4_dense_launch(torch.empty(M, 0, device="cuda"), empty, b, y, _native.EPI_BIAS_RELU)
        assert torch.equal(y, b.clamp(min=0).expand(M, 40))


@pytest.mark.parametrize("symmetric", [False, True])
def test_quantize(symmetric):
    """Every weight is within half a step of what its integer stands for (or at the range's end)."""
    g = torch.Generator().manual_seed(5)
    W = torch.randn(300, 70, generator=g).cuda()
    W[:, 3] = 0
    q, s, z = lm.q4_quantize(W, 64, symmetric)
    at = torch.arange(300, device="cuda") // 64
    back = s[at] * (q.float() - (z[at].float() if z is not None else 8.0))
    assert ((back - W).abs() <= s[at] * 0.5001 + (0 if symmetric else 1) * s[at] * 0.5).all()
    y = torch.empty(5, 70, device="cuda")
    x = make_x(5, 300, F32)
    lm.q4_dense_launch(x, lm.q4_pack(q, s, z, group_size=64), None, y)
    want, size = expect(x, q, s, z, 64)
    check(y, want, size, 300)


def test_another_stream_and_graph_replays():
    for M in (1, 48):
        x, (q, s, z) = make_x(M, 4096, BF16), make_weights(4096, 256, 128)
        W, y = lm.q4_pack(q, s, z), torch.empty(M, 256, dtype=BF16, device="cuda")
        lm.q4_dense_launch(x, W, None, y)
        want = y.clone()
        s2 = torch.cuda.Stream()
        s2.wait_stream(torch.cuda.current_stream())
        y.zero_()
        s2.wait_stream(torch.cuda.current_stream())
        lm.q4_dense_launch(x, W, None, y, stream=s2)
        s2.synchronize()
        assert torch.equal(y, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lm.q4_dense_launch(x, W, None, y)
        for seed in range(3):
            x.copy_(make_x(M, 4096, BF16, seed=50 + seed))
            lm.q4_dense_launch(x, W, None, y)
            torch.cuda.synchronize()
            want = y.clone()
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_refusals():
    q, s, z = make_weights(128, 40, 64)
    for bad, error in [(dict(Q=q.int()), TypeError), (dict(Q=q.cpu()), ValueError), (dict(Q=q.t()), ValueError),
                       (dict(scales=s[:1]), ValueError), (dict(scales=s.double()), TypeError),
                       (dict(zeros=z[:, 1:]), ValueError), (dict(zeros=z.float()), TypeError),
                       (dict(group_size=48), RuntimeError), (dict(group_size=0), RuntimeError),
                       (dict(group_size=192), RuntimeError)]:
        with pytest.raises(error):
            lm.q4_pack(**(dict(Q=q, scales=s, zeros=z, group_size=64) | bad))
    W = lm.q4_pack(q, s, z, group_size=64)
    x, y, b = make_x(4, 128, F32), torch.full((4, 40), 7.0, device="cuda"), torch.ones(40, device="cuda")
    for bad, error in [(dict(X=x[:, 1:]), ValueError), (dict(X=x.double()), TypeError), (dict(X=x.cpu()), ValueError),
                       (dict(W=q), TypeError), (dict(Y=y.int()), TypeError), (dict(Y=y[:3]), ValueError),
                       (dict(b=b[1:]), ValueError), (dict(b=None, epilogue=_native.EPI_BIAS), RuntimeError),
                       (dict(epilogue=8), RuntimeError), (dict(x_scales=b), ValueError),
                       (dict(x_scales=b[:4].half()), TypeError)]:
        with pytest.raises(error):
            lm.q4_dense_launch(**(dict(X=x, W=W, b=b, Y=y) | bad))
    torch.cuda.synchronize()
    assert (y == 7.0).all()
