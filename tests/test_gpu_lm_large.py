"""Offsets past 32 bits in the language-model operators: strided rows and whole
operands beyond 2^31 elements (or bytes), checked on sampled rows with the last
ones among them, against 64 bits. Tolerances are those of the operators' own
tests."""
import pytest
import torch

import lm_reference as ref
from mlir_edsl_hip import lm

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
FAR = 2 ** 30 + 7  # a row stride: row 2 starts past 2^31 elements


@pytest.fixture(autouse=True)
def freed():
    yield
    torch.cuda.empty_cache()


def far_rows(values, fill=float("nan")):
    """The rows of a matrix, FAR elements apart; around them `fill`."""
    M, N = values.shape
    t = torch.empty((M - 1) * FAR + N + 8, dtype=values.dtype, device="cuda").as_strided((M, N), (FAR, 1))
    for r in range(M):
        t[r].copy_(values[r])
    return t


def normal(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def close(got, want, units):
    """Within so many roundings of the type's, of a value of size 1."""
    bound = units * ref.HALF_ULP[got.dtype] * (1 + want.abs())
    assert float(((ref.d(got) - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("N", [300, 40000])
def test_norm_of_rows_far_apart(N):
    x, w, dy = normal(4, N, dtype=BF16), normal(N, seed=1), normal(4, N, seed=2, dtype=BF16)
    X, Y, rstd = far_rows(x), far_rows(torch.zeros(4, N, dtype=BF16)), torch.empty(4, device="cuda")
    lm.rms_norm_launch(X, w.cuda(), Y, rstd=rstd)
    y, h, r = ref.rms_norm(x, w)
    close(Y, y, 2)
    # dX over dY; both over Y's rows.
    for row in range(4):
        Y[row].copy_(dy[row])
    dw = torch.empty(N, device="cuda")
    lm.rms_norm_backward_launch(Y, X, w.cuda(), rstd, Y, dw)
    dx, dweight = ref.rms_norm_backward(dy, h, w, r)
    close(Y, dx, 2)
    close(dw, dweight, 2 ** 9)


def test_norm_of_many_rows():
    M, N = 2 ** 22 + 3, 520  # 2.2e9 elements
    X = torch.empty(M, N, dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    w, scales = normal(N, seed=1).cuda(), torch.empty(M, device="cuda")
    Q = torch.empty(M, N, dtype=torch.int8, device="cuda")
    lm.rms_norm_launch(X, w, Q, scales=scales)
    rows = torch.tensor([0, 1, M // 2, 4129776, 4129777, M - 2, M - 1], device="cuda")
    y, _, _ = ref.rms_norm(X[rows], w)
    s = y.abs().amax(1) / 127
    assert float(((ref.d(scales[rows]) - s).abs() / s).max()) <= 2.0 ** -20
    assert float((ref.d(Q[rows]) * s[:, None] - y).abs().div(s[:, None]).max()) <= 0.5 + 2.0 ** -12


@pytest.mark.parametrize("V", [1000, 140000])
def test_logprobs_of_rows_far_apart(V):
    M, k = 4, 3
    x, tokens = normal(M, V, dtype=BF16), torch.tensor([0, V - 1, 5, 70], device="cuda")
    X = far_rows(x)
    lp, lse, entropy, top = (torch.empty(*s, device="cuda") for s in ((M,), (M,), (M,), (M, k)))
    ids = torch.empty(M, k, dtype=torch.int64, device="cuda")
    lm.token_logprobs_launch(X, tokens, lp, lse, entropy, top, ids)
    want = ref.token_logprobs(x, tokens, k)
    assert torch.equal(ids.cpu(), want[4])
    for got, value in zip((lp, lse, entropy, top), want):
        close(got, value, 16)
    g = normal(M, seed=5).cuda()
    lm.token_logprobs_backward_launch(X, tokens, lse, X, g)  # in the logits' memory
    close(X, ref.token_logprobs_backward(x, tokens, lse, g), 2)


def test_logprobs_of_many_rows():
    M, V = 2 ** 22 + 5, 520
    X = torch.empty(M, V, dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    tokens = torch.arange(M, device="cuda", dtype=torch.int32) % V
    lp, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    ids, top = torch.empty(M, 2, dtype=torch.int32, device="cuda"), torch.empty(M, 2, device="cuda")
    lm.token_logprobs_launch(X, tokens, lp, lse, None, top, ids)
    rows = torch.tensor([0, 1, M // 2, 4129776, 4129777, M - 2, M - 1], device="cuda")
    want = ref.token_logprobs(X[rows], tokens[rows], 2)
    assert torch.equal(ids[rows].cpu().long(), want[4])
    close(lp[rows], want[0], 16)
    g = torch.ones(M, device="cuda")
    x = X[rows].clone()
    lm.token_logprobs_backward_launch(X, tokens, lse, X, g)
    close(X[rows], ref.token_logprobs_backward(x, tokens[rows], lse[rows], g[rows]), 2)


def q4_check(got, x, q, s, group):
    at = torch.arange(q.shape[0]) // group
    w, size = (ref.d(q) - 8) * ref.d(s)[at], (ref.d(q) + 8) * ref.d(s)[at]
    K = q.shape[0]
    bound = (min(K, 128) + K / 32 + 48) * 2.0 ** -23 * (ref.d(x).abs() @ size)
    want = ref.d(x) @ w
    bound = bound + ref.HALF_ULP[got.dtype] * 1.001 * (want.abs() + bound)
    assert float(((ref.d(got) - want).abs() - bound).max()) <= 0


def q4_weights(K, N, group):
    g = torch.Generator("cuda").manual_seed(K + N)
    q = torch.randint(0, 16, (K, N), dtype=torch.uint8, device="cuda", generator=g)
    return q, torch.rand(-(-K // group), N, device="cuda", generator=g) / 16


@pytest.mark.parametrize("M", [3, 17])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_q4_of_rows_far_apart(M, dtype):
    K, N, group = 384, 200, 128
    x = normal(M, K, dtype=dtype)
    q, s = q4_weights(K, N, group)
    X, Y = far_rows(x), far_rows(torch.zeros(M, N, dtype=BF16))
    lm.q4_dense_launch(X, lm.q4_pack(q, s, group_size=group), None, Y)
    q4_check(Y, x, q, s, group)


def test_q4_of_many_rows():
    M, K, N, group = 2 ** 24 + 65, 160, 130, 32  # X 2.7e9, Y 2.2e9 elements; x is copied, 2^24 rows a group
    X = torch.empty(M, K, dtype=torch.int8, device="cuda").random_(-127, 128)
    q, s = q4_weights(K, N, group)
    Y = torch.empty(M, N, dtype=BF16, device="cuda")
    lm.q4_dense_launch(X, lm.q4_pack(q, s, group_size=group), None, Y)
    rows = torch.tensor([0, 1, M // 2, M - 66, M - 2, M - 1], device="cuda")
    q4_check(Y[rows], X[rows], q, s, group)


@pytest.mark.parametrize("M", [2, 40])
def test_q4_of_large_weights(M):
    K, N, group = 4096, 2 ** 20 + 40, 128  # 2.1e9 bytes of weights, 4.3e9 of their integers
    q, s = q4_weights(K, N, group)
    W = lm.q4_pack(q, s, group_size=group)
    X = normal(M, K, dtype=BF16).cuda()
    Y = torch.empty(M, N, dtype=BF16, device="cuda")
    lm.q4_dense_launch(X, W, None, Y)
    cols = torch.tensor([0, 1, N // 2, 2 ** 20 - 1, 2 ** 20, N - 17, N - 1], device="cuda")
    q4_check(Y[:, cols], X, q[:, cols], s[:, cols], group)


# More threads than a launch takes along one axis (2^32).
def test_norm_backward_of_a_row_of_many_columns():
    N = 2 ** 26 + 21
    g = torch.Generator("cuda").manual_seed(3)
    dy, h = (torch.empty(1, N, device="cuda").normal_(generator=g) for _ in range(2))
    w, rstd = torch.ones(N, device="cuda"), torch.ones(1, device="cuda")
    dX, dw = torch.empty_like(dy), torch.full((N,), float("nan"), device="cuda")
    lm.rms_norm_backward_launch(dy, h, w, rstd, dX, dw)
    assert torch.equal(dw, (dy * h)[0])  # one row, rstd 1: the rounded product


def test_q4_of_many_columns():
    K, N, group = 1, 2 ** 30, 128  # 2^26 tiles of columns, 6.9e10 bytes of packed weights
    q, s = q4_weights(K, N, group)
    W = lm.q4_pack(q, s, group_size=group)
    X, Y = normal(1, K, dtype=BF16).cuda(), torch.full((1, N), float("nan"), dtype=BF16, device="cuda")
    lm.q4_dense_launch(X, W, None, Y)
    cols = torch.tensor([0, 1, N // 2 - 1, N // 2, 2 ** 29 + 2 ** 24, N - 17, N - 1], device="cuda")
    q4_check(Y[:, cols], X, q[:, cols], s[:, cols], group)
    assert not bool(Y.isnan().any())


def test_q4_without_depth_of_many_rows():
    M, N = 2 ** 30, 1  # 2^24 tiles of rows; no element of X is there: Y is the bias
    W = lm.q4_pack(torch.empty(0, N, dtype=torch.uint8, device="cuda"), torch.empty(0, N, device="cuda"))
    Y = torch.full((M, N), float("nan"), dtype=BF16, device="cuda")
    lm.q4_dense_launch(torch.empty(M, 0, dtype=BF16, device="cuda"), W, torch.full((N,), 1.5, device="cuda"), Y, 1)
    assert bool((Y == 1.5).all())
