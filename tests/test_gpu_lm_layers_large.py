"""Offsets past 32 bits, and axes longer than a launch's, in the layers on groups of rows and in 8-bit
integers and in sampling: strided rows, whole operands beyond 2^31 elements, very many columns or rows,
checked on some of them with the last ones among them. Small integers: results are exact."""
import pytest
import torch

import lm_layers_reference as layers
from mlir_edsl_hip import _native, last_plan, lm

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
FAR = 2 ** 30 + 8  # a row stride: row 2 starts past 2^31 elements


@pytest.fixture(autouse=True)
def freed():
    yield
    torch.cuda.empty_cache()


def whole(*shape, seed, dtype, most=2):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, dtype=torch.int8, device="cuda").to(dtype)


def far_rows(values, stride=FAR):
    M, N = values.shape
    t = torch.empty((M - 1) * stride + N, dtype=values.dtype, device="cuda").as_strided((M, N), (stride, 1))
    for r in range(M):
        t[r].copy_(values[r])
    return t


def same(got, want):
    assert torch.equal(got.double(), want.to(got.dtype).double())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("E", [1, 3])
def test_groups_of_rows_far_apart(dtype, E):
    # One group streams in none, three in all: both kernels.
    counts = [40] if E == 1 else [2, 1, 4]
    T, K, N = sum(counts), 72, 40
    far = FAR // 8 if E == 1 else FAR  # 40 rows: past 2^32 bytes all the same
    off = torch.tensor([0, *counts]).cumsum(0).cuda()
    x, w, dy = whole(T, K, seed=1, dtype=dtype), whole(E, K, N, seed=2, dtype=dtype), whole(T, N, seed=3, dtype=dtype)
    X, Y = far_rows(x, far), far_rows(torch.zeros_like(dy), far)
    lm.grouped_dense_launch(X, w, off, None, Y)
    same(Y, layers.grouped_dense(x, w, off))
    DY = far_rows(dy, far)
    dx, dw, db = far_rows(torch.zeros_like(x), far), torch.empty(E, K, N, device="cuda"), torch.empty(E, N, device="cuda")
    lm.grouped_dense_backward_launch(DY, X, w, off, dx, dw, db, Y, _native.EPI_RELU)
    for got, right in zip((dx, dw, db), layers.grouped_dense_backward(dy, x, w, off, Y.contiguous(), _native.EPI_RELU)):
        same(got, right)


@pytest.mark.parametrize("counts", [[0, 3, 2], [0, 200, 150]], ids=str)
@pytest.mark.parametrize("order", ["kn", "nk"])
def test_weights_of_groups_far_apart(counts, order):
    E, T, K, N = 3, sum(counts), 72, 40
    off = torch.tensor([0, *counts]).cumsum(0).cuda()
    values = whole(E, K, N, seed=2, dtype=F16)

    def apart(fill):
        flat = torch.empty(2 * FAR + K * N, dtype=F16, device="cuda")
        w = flat.as_strided((E, K, N), (FAR, N, 1) if order == "kn" else (FAR, 1, K))
        w.copy_(fill)
        return w
    w, dw = apart(values), apart(torch.zeros_like(values))
    x, dy = whole(T, K, seed=1, dtype=F16), whole(T, N, seed=3, dtype=F16)
    y, dx = torch.empty(T, N, dtype=F16, device="cuda"), torch.empty(T, K, dtype=F16, device="cuda")
    lm.grouped_dense_launch(x, w, off, None, y)
    same(y, layers.grouped_dense(x, values, off))
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw)
    for got, right in zip((dx, dw), layers.grouped_dense_backward(dy, x, values, off)):
        same(got, right)


def test_one_group_of_many_rows_and_weights_past_32_bits():
    T, K, N = 2 ** 22 + 130, 520, 16  # x 2.2e9 elements
    x, w = whole(T, K, seed=1, dtype=BF16, most=1), whole(1, K, N, seed=2, dtype=BF16, most=1)
    y, off = torch.empty(T, N, dtype=BF16, device="cuda"), torch.tensor([0, T], device="cuda")
    lm.grouped_dense_launch(x, w, off, None, y)
    rows = torch.tensor([0, 1, T // 2, T - 131, T - 2, T - 1], device="cuda")
    same(y[rows], layers.grouped_dense(x[rows], w, torch.tensor([0, len(rows)])))
    del x, y
    K, N = 66000, 33000  # w 2.2e9 elements, its last rows past 2^32 bytes
    w = whole(1, K, N, seed=2, dtype=BF16, most=1)
    for T in (2, 70):
        x, y = whole(T, K, seed=1, dtype=BF16, most=1), torch.empty(T, N, dtype=BF16, device="cuda")
        lm.grouped_dense_launch(x, w, torch.tensor([0, T], device="cuda"), None, y)
        cols = torch.tensor([0, 1, N // 2, N - 2, N - 1], device="cuda")
        same(y[:, cols], layers.grouped_dense(x, w[:, :, cols], torch.tensor([0, T])))


@pytest.mark.parametrize("order", ["kn", "nk"])
def test_groups_of_very_many_columns(order):
    # More threads than a launch takes along one axis, were each 16 columns a workgroup.
    K, N = 1, 2 ** 27 + 9
    x, w = whole(2, K, seed=1, dtype=BF16), whole(1, K, N, seed=2, dtype=BF16)
    if order == "nk":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    y = torch.full((2, N), float("nan"), dtype=BF16, device="cuda")
    lm.grouped_dense_launch(x, w, torch.tensor([0, 2], device="cuda"), None, y)
    assert "stream" not in last_plan()
    assert torch.equal(y, x * w[0])


@pytest.mark.parametrize("M", [3, 40])
def test_i8_rows_far_apart(M):
    K, N, far = 272, 130, FAR if M == 3 else FAR // 8
    x, q = whole(M, K, seed=1, dtype=I8, most=100), whole(K, N, seed=2, dtype=I8, most=100)
    X, Y = far_rows(x, far), far_rows(torch.zeros(M, N, device="cuda"), far)
    lm.i8_dense_launch(X, lm.i8_pack(q, torch.ones(N, device="cuda")), None, Y)
    same(Y, x.double() @ q.double())


def test_i8_of_many_rows():
    M, K, N = 2 ** 24 + 65, 144, 136  # X 2.4e9, Y 2.3e9 elements
    X, q = whole(M, K, seed=1, dtype=I8, most=100), whole(K, N, seed=2, dtype=I8, most=100)
    Y = torch.empty(M, N, dtype=F32, device="cuda")
    lm.i8_dense_launch(X, lm.i8_pack(q, torch.ones(N, device="cuda")), None, Y)
    rows = torch.tensor([0, 1, M // 2, M - 66, M - 2, M - 1], device="cuda")
    same(Y[rows], X[rows].double() @ q.double())


@pytest.mark.parametrize("M", [2, 70])
def test_i8_of_large_weights(M):
    K, N = 4096, 2 ** 20 + 40  # 4.3e9 bytes
    X, q = whole(M, K, seed=1, dtype=I8, most=100), whole(K, N, seed=2, dtype=I8, most=100)
    Y = torch.empty(M, N, dtype=F32, device="cuda")
    lm.i8_dense_launch(X, lm.i8_pack(q, torch.ones(N, device="cuda")), None, Y)
    cols = torch.tensor([0, 1, N // 2, 2 ** 20 - 1, 2 ** 20, N - 17, N - 1], device="cuda")
    same(Y[:, cols], X.double() @ q[:, cols].double())


def test_bias_sums_of_very_many_rows():
    """More workgroups than a row of the grid has, and offsets that fall: as many tiles again as there is room for."""
    T, N = 2 ** 25 + 40, 8
    dy = whole(T, N, seed=1, dtype=BF16, most=1)
    db = torch.empty(3, N, device="cuda")
    lm.grouped_dense_backward_launch(dy, None, None, torch.tensor([0, T // 2, T // 2, T], device="cuda"), db=db)
    same(db, torch.stack((dy[:T // 2].double().sum(0), torch.zeros(N, device="cuda").double(), dy[T // 2:].double().sum(0))))
    # Unspecified sums; the workspace's neighbours stay.
    guard = whole(2 ** 22, seed=2, dtype=F32)
    kept = guard.clone()
    lm.grouped_dense_backward_launch(dy, None, None, torch.tensor([0, T, 0, T], device="cuda"), db=db)
    torch.cuda.synchronize()
    assert torch.equal(guard, kept)


def test_logits_far_apart_and_the_largest_vocabulary():
    x = (2.5 * torch.randn(3, 1000, generator=torch.Generator().manual_seed(1))).cuda()
    u = torch.tensor([0.1, 0.5, 0.9], device="cuda")
    tokens = torch.zeros(3, dtype=torch.int64, device="cuda")
    lm.sample_tokens_launch(far_rows(x), u, tokens, top_k=50, top_p=0.9)
    assert tokens.tolist() == [layers.sample(x[m], u[m], 1.0, 50, 0.9)[0] for m in range(3)]
    V = 2 ** 21
    x = (2.5 * torch.randn(3, V, generator=torch.Generator().manual_seed(2))).to(BF16).cuda()
    for settings in ({}, dict(top_k=1000, top_p=0.9), dict(top_p=0.95), dict(min_p=0.001)):
        lm.sample_tokens_launch(x, u, tokens, **settings)
        assert tokens.tolist() == [layers.sample(x[m], u[m], **settings)[0] for m in range(3)]
    # The longest sums: every logit the same.
    lm.sample_tokens_launch(torch.zeros_like(x), torch.tensor([0.0, 0.5, 1 - 2.0 ** -24], device="cuda"), tokens)
    assert tokens.tolist() == [0, V // 2, V - 1]
