"""The dense layer on groups of rows and its gradients.

Most inputs are small integers, so that products and sums are exact in 32 bits in
any order and a result is its definition's, rounded once to its type: compared
bit for bit. With real values a sum of n terms is off by at most n + 64 roundings of
2^-23 (matrix cores may cut off) of the terms' absolute sum, and the type's one."""
import pytest
import torch

import lm_layers_reference as layers
import lm_reference as ref
from mlir_edsl_hip import _native, last_plan, lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}
ALPHA = 0.25  # a power of two: products with it are exact
FILL = -7.0
EPIS = [_native.EPI_NONE, _native.EPI_BIAS, _native.EPI_RELU, _native.EPI_BIAS_RELU, _native.EPI_LEAKY,
        _native.EPI_BIAS_LEAKY, _native.EPI_IF_RELU, _native.EPI_BIAS_IF_RELU]


def whole(*shape, seed, dtype, most=3):
    v = torch.randint(-most, most + 1, shape, generator=torch.Generator().manual_seed(seed))
    return v.to(dtype).cuda()


def offsets_of(counts, first=0, dtype=torch.int32):
    return (torch.tensor([0, *counts]).cumsum(0) + first).to(dtype).cuda()


def stack(values, order):
    """[E, K, N] with N ("kn") or K ("nk") contiguous."""
    return values if order == "kn" else values.transpose(1, 2).contiguous().transpose(1, 2)


def framed(t, left, right, fill=float("nan")):
    """The matrix as a view of one with more columns, which hold `fill`."""
    big = torch.full((t.shape[0], left + t.shape[1] + right), fill, dtype=t.dtype, device="cuda")
    view = big[:, left:left + t.shape[1]]
    view.copy_(t)
    return view


def same(got, want, dtype=None):
    assert torch.equal(got.double(), want.to(dtype or got.dtype).double())


def forward(counts, K, N, dtype, order, epi=0, first=0, behind=0, ids=torch.int32, frame=None, plan=None, most=3):
    E, T = len(counts), first + sum(counts) + behind
    x, w = whole(T, K, seed=1, dtype=dtype, most=most), stack(whole(E, K, N, seed=2, dtype=dtype, most=most), order)
    b = whole(E, N, seed=3, dtype=dtype, most=50) if epi & 1 else None
    y = torch.full((T, N), FILL, dtype=dtype, device="cuda")
    if frame:
        x, y = framed(x, *frame), framed(y, *frame, fill=FILL)
    off = offsets_of(counts, first, ids)
    want = layers.grouped_dense(x, w, off, b, epi, ALPHA, before=y)
    lm.grouped_dense_launch(x, w, off, b, y, epi, ALPHA)
    assert plan is None or plan in last_plan(), last_plan()
    same(y, want)
    if frame:
        around = y._base.clone()
        around[:, frame[0]:frame[0] + N] = FILL
        assert bool((around == FILL).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("counts", [[1], [3, 0, 16], [17, 32, 0, 1], [0, 33, 5], [130, 0, 64, 1]], ids=str)
@pytest.mark.parametrize("K,N", [(1, 1), (8, 3), (37, 45), (64, 128), (129, 65), (264, 200)])
def test_sizes(dtype, order, counts, K, N):
    forward(counts, K, N, TYPES[dtype], order)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("counts", [[5, 20], [300, 40]], ids=str)
@pytest.mark.parametrize("epi", EPIS)
def test_epilogues(dtype, order, counts, epi):
    forward(counts, 72, 56, TYPES[dtype], order, epi)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("order", ["kn", "nk"])
def test_kernels(dtype, order):
    t = TYPES[dtype]
    forward([2, 5, 0, 9], 512, 640, t, order, plan="stream")
    forward([2, 40, 0, 9], 512, 640, t, order, plan="stream+tiles direct")
    forward([2, 60, 0, 9], 512, 640, t, order, plan=" +tiles direct")
    forward([200, 500], 128, 384, t, order, plan="tiles direct")
    # Rows off 16 bytes.
    forward([200, 500], 130, 382, t, order, plan="tiles any")
    forward([200, 500], 129, 381, t, order, plan="tiles any")
    # Whole rounds of large tiles with halves, with quarters and with none left; quarters alone.
    for counts, N in (([700, 0, 1500, 900], 8192), ([1500, 2000, 700], 4000), ([4096], 4096), ([300, 130], 2048)):
        forward(counts, 192, N, t, order, epi=_native.EPI_BIAS_RELU, plan="tiles direct")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("frame", [(0, 8), (1, 2), (8, 8), (3, 0)], ids=str)
@pytest.mark.parametrize("counts", [[4, 17], [150, 20]], ids=str)
def test_strides_alignments_and_rows_of_no_group(dtype, order, frame, counts):
    # NaN around the rows of x; rows before and behind the groups keep what they hold.
    forward(counts, 80, 96, TYPES[dtype], order, first=3, behind=5, ids=torch.int64, frame=frame)


@pytest.mark.parametrize("E", [1, 64, 65, 200, 1500])
@pytest.mark.parametrize("most", [3, 90])
def test_many_groups(E, most):
    counts = torch.randint(0, most, (E,), generator=torch.Generator().manual_seed(E)).tolist()
    if E > 3:
        counts[:3] = [0, 0, 150]
    forward(counts, 40, 48, BF16, "kn", _native.EPI_BIAS)
    backward(counts, 40, 48, BF16, "nk", _native.EPI_BIAS)


def backward(counts, K, N, dtype, order, epi=0, first=0, behind=0, frame=None, grad=F32, dw_order=None, plan=None):
    E, T = len(counts), first + sum(counts) + behind
    x, w = whole(T, K, seed=1, dtype=dtype, most=2), stack(whole(E, K, N, seed=2, dtype=dtype, most=2), order)
    dy, y = whole(T, N, seed=3, dtype=dtype, most=2) * 4, whole(T, N, seed=4, dtype=dtype, most=2)
    dx = torch.full((T, K), FILL, dtype=dtype, device="cuda")
    if frame:
        x, dy, y, dx = framed(x, *frame), framed(dy, *frame), framed(y, *frame), framed(dx, *frame, fill=FILL)
    dw = stack(torch.full((E, K, N), FILL, dtype=grad, device="cuda"), dw_order or order)
    db = torch.full((E, N), FILL, dtype=grad, device="cuda")
    off = offsets_of(counts, first)
    want = layers.grouped_dense_backward(dy, x, w, off, y, epi, ALPHA, before=dx)
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db, y, epi, ALPHA)
    assert plan is None or plan in last_plan(), last_plan()
    for got, right in zip((dx, dw, db), want):
        same(got, right)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("counts", [[1], [3, 0, 16], [0, 33, 5], [130, 0, 64, 1]], ids=str)
@pytest.mark.parametrize("K,N", [(1, 1), (8, 3), (37, 45), (64, 128), (129, 65), (264, 200)])
def test_gradients_of_all_sizes(dtype, order, counts, K, N):
    backward(counts, K, N, TYPES[dtype], order, grad=TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("epi", EPIS)
@pytest.mark.parametrize("counts", [[5, 20], [300, 40]], ids=str)
def test_gradients_through_epilogues(dtype, epi, counts):
    backward(counts, 72, 56, TYPES[dtype], "kn", epi)
    backward(counts, 71, 53, TYPES[dtype], "nk", epi, dw_order="kn")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("frame", [(0, 8), (1, 2), (3, 0)], ids=str)
def test_gradients_strides_and_rows_of_no_group(dtype, frame):
    backward([40, 0, 33], 80, 96, TYPES[dtype], "kn", _native.EPI_RELU, first=3, behind=5, frame=frame, dw_order="nk")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradients_of_large_groups(dtype):
    wide = dtype != "f32"
    backward([1100, 1300, 0], 4096, 1536, TYPES[dtype], "kn", _native.EPI_BIAS_RELU,
             plan="dW 256x256" if wide else "dW 128x128")
    backward([150, 90, 0], 130, 258, TYPES[dtype], "kn", _native.EPI_BIAS_RELU, plan="dW any")
    backward([150, 90, 0], 131, 259, TYPES[dtype], "kn", plan="dW any")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("counts", [[7, 30], [200, 90, 500]], ids=str)
def test_real_values(dtype, counts):
    t, K, N = TYPES[dtype], 500, 260
    T, E, g = sum(counts), len(counts), torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).to(t).cuda()  # noqa: E731
    x, w, b, dy = r(T, K), r(E, K, N), r(E, N), r(T, N)
    off, y = offsets_of(counts), torch.empty(T, N, dtype=t, device="cuda")
    lm.grouped_dense_launch(x, w, off, b, y, _native.EPI_BIAS)
    want = layers.grouped_dense(x, w, off, b, _native.EPI_BIAS)
    terms = layers.grouped_dense(x.abs(), w.abs(), off, b.abs(), _native.EPI_BIAS)
    near(y, want, terms, K + 1)
    dx, dw, db = torch.empty_like(x), torch.empty(E, K, N, device="cuda"), torch.empty(E, N, device="cuda")
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db)
    want = layers.grouped_dense_backward(dy, x, w, off)
    terms = layers.grouped_dense_backward(dy.abs(), x.abs(), w.abs(), off)
    for got, right, size, n in zip((dx, dw, db), want, terms, (N, max(counts), max(counts))):
        near(got, right, size, n)


def near(got, want, terms, n):
    bound = (n + 64) * 2.0 ** -23 * terms + ref.HALF_ULP[got.dtype] * want.abs() + ref.TINY[got.dtype]
    assert float(((got.double() - want).abs() - bound).max()) <= 0


def test_gradients_against_differences():
    """f32: the loss sum(dY * Y) changes with an input as its gradient says. Y is linear in each input, so that
    a central difference of exact sums over a power of two is the derivative."""
    counts, K, N = [6, 0, 40], 24, 20
    T, E = sum(counts), len(counts)
    x, w, b, dy = (whole(*s, seed=i, dtype=F32) for i, s in enumerate(((T, K), (E, K, N), (E, N), (T, N))))
    off = offsets_of(counts)

    def loss():
        y = torch.empty(T, N, device="cuda")
        lm.grouped_dense_launch(x, w, off, b, y, _native.EPI_BIAS)
        return float((y.double() * dy.double()).sum())
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db)
    for t, grad, at in ((x, dx, (5, 3)), (x, dx, (30, 23)), (w, dw, (0, 2, 7)), (w, dw, (1, 2, 7)), (w, dw, (2, 23, 19)),
                        (b, db, (2, 1)), (b, db, (1, 1))):
        t[at] += 1
        up = loss()
        t[at] -= 2
        down = loss()
        t[at] += 1
        assert (up - down) / 2 == float(grad[at])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("counts", [[5, 9], [200, 140]], ids=str)
def test_nan_and_infinity_stay_in_their_group(dtype, counts):
    t, K, N = TYPES[dtype], 72, 56
    T, off = sum(counts), offsets_of(counts)
    x, w, dy = whole(T, K, seed=1, dtype=t), whole(2, K, N, seed=2, dtype=t), whole(T, N, seed=3, dtype=t)
    clean = layers.grouped_dense(x, w, off), layers.grouped_dense_backward(dy, x, w, off)
    x[counts[0]:] = float("nan")
    w[1] = float("inf")
    dy[counts[0]:] = float("-inf")
    y, dx, dw, db = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w), torch.empty(2, N, device="cuda")
    lm.grouped_dense_launch(x, w, off, None, y)
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db)
    same(y[:counts[0]], clean[0][:counts[0]])
    same(dx[:counts[0]], clean[1][0][:counts[0]])
    same(dw[0], clean[1][1][0])
    same(db[0], clean[1][2][0])
    assert bool(y[counts[0]:].isnan().all() and dw[1].isnan().all())


@pytest.mark.parametrize("epi,value", [(_native.EPI_RELU, float("nan")), (_native.EPI_IF_RELU, 0.0)])
def test_nan_through_the_activations(epi, value):
    x = torch.full((3, 8), float("nan"), device="cuda")
    y = torch.zeros(3, 8, device="cuda")
    lm.grouped_dense_launch(x, whole(1, 8, 8, seed=1, dtype=F32), offsets_of([3]), None, y, epi)
    assert bool(y.isnan().all()) if value != value else bool((y == value).all())


@pytest.mark.parametrize("offsets", [[0, 40, 10, 50], [-5, 20, 70, 300], [50, 40, 30, 0], [0, 50, 0, 50], [9, 9, 9, 9]], ids=str)
@pytest.mark.parametrize("K", [64, 67])
def test_offsets_without_order_stay_inside(offsets, K):
    """Unspecified rows, but nothing outside the operands changes."""
    T, N = 50, 64
    y, dx = framed(torch.zeros(T, N, device="cuda"), 4, 4, FILL), framed(torch.zeros(T, K, device="cuda"), 4, 4, FILL)
    x, w, dy = whole(T, K, seed=1, dtype=F32), whole(3, K, N, seed=2, dtype=F32), whole(T, N, seed=3, dtype=F32)
    off = torch.tensor(offsets, dtype=torch.int64, device="cuda")
    dw, db = torch.zeros(3, K, N, device="cuda"), torch.zeros(3, N, device="cuda")
    lm.grouped_dense_launch(x, w, off, None, y)
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db, y, _native.EPI_RELU)
    torch.cuda.synchronize()
    for t in (y, dx):
        assert bool((t._base[:, :4] == FILL).all() and (t._base[:, -4:] == FILL).all())


def test_empty_sides():
    t = lambda *s: torch.full(s, FILL, device="cuda")  # noqa: E731
    off = offsets_of([0, 0])
    lm.grouped_dense_launch(t(0, 8), t(2, 8, 4), off, None, t(0, 4))
    assert last_plan() == "empty"
    lm.grouped_dense_launch(t(3, 8), t(0, 8, 4), off[:1], None, t(3, 4))
    assert last_plan() == "empty"
    # No k: the bias alone. No rows: gradients of 0. No columns: dX 0.
    y = t(5, 4)
    lm.grouped_dense_launch(t(5, 0), t(2, 0, 4), offsets_of([2, 3]), whole(2, 4, seed=1, dtype=F32), y, _native.EPI_BIAS)
    same(y, whole(2, 4, seed=1, dtype=F32).double()[[0, 0, 1, 1, 1]])
    dw, db = t(2, 8, 4), t(2, 4)
    lm.grouped_dense_backward_launch(t(0, 4), t(0, 8), t(2, 8, 4), off, t(0, 8), dw, db, t(0, 4), _native.EPI_RELU)
    assert not dw.any() and not db.any()
    dx = t(5, 8)
    lm.grouped_dense_backward_launch(t(5, 0), t(5, 8), t(2, 8, 0), offsets_of([2, 3]), dx, t(2, 8, 0), t(2, 0))
    assert not dx.any()


def test_parts_of_the_gradients():
    counts, K, N = [20, 50], 40, 24
    x, w, dy = whole(70, K, seed=1, dtype=BF16), whole(2, K, N, seed=2, dtype=BF16), whole(70, N, seed=3, dtype=BF16)
    off = offsets_of(counts)
    want = layers.grouped_dense_backward(dy, x, w, off)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(2, N, dtype=BF16, device="cuda")
    lm.grouped_dense_backward_launch(dy, None, w, off, dX=dx)
    lm.grouped_dense_backward_launch(dy, x, None, off, dW=dw)
    lm.grouped_dense_backward_launch(dy, None, None, off, db=db)
    for got, right in zip((dx, dw, db), want):
        same(got, right)
    lm.grouped_dense_backward_launch(dy, x, w, off)
    assert last_plan() == "empty"


def test_one_bias_for_all_and_shared_weights():
    counts, K, N = [4, 70], 48, 32
    x, w, b = whole(74, K, seed=1, dtype=F16), whole(1, K, N, seed=2, dtype=F16).expand(2, K, N), \
        whole(1, N, seed=3, dtype=F16).expand(2, N)
    y = torch.empty(74, N, dtype=F16, device="cuda")
    lm.grouped_dense_launch(x, w, offsets_of(counts), b, y, _native.EPI_BIAS)
    same(y, layers.grouped_dense(x, w, offsets_of(counts), b, _native.EPI_BIAS))


def test_another_stream_and_graph_replays():
    """A captured step, forward and backward, replayed with other rows, other group sizes and eager calls between."""
    K, N, T = 96, 64, 160
    x, w, dy = whole(T, K, seed=1, dtype=BF16), whole(3, K, N, seed=2, dtype=BF16), whole(T, N, seed=3, dtype=BF16)
    off, b = offsets_of([100, 20, 40]), whole(3, N, seed=4, dtype=BF16)
    y, dx, dw, db = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)

    def step(stream=None):
        lm.grouped_dense_launch(x, w, off, b, y, _native.EPI_BIAS_RELU, stream=stream)
        lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db, y, _native.EPI_BIAS_RELU, stream=stream)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    step(side)
    side.synchronize()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i, counts in enumerate(([0, 160, 0], [1, 30, 129], [60, 60, 40], [10, 5, 2])):
        x.copy_(whole(T, K, seed=10 + i, dtype=BF16))
        off.copy_(offsets_of(counts))
        for t in (y, dx):
            t.fill_(FILL)
        graph.replay()
        torch.cuda.synchronize()
        same(y, layers.grouped_dense(x, w, off, b, _native.EPI_BIAS_RELU, before=torch.full_like(y, FILL)))
        for got, right in zip((dx, dw, db), layers.grouped_dense_backward(dy, x, w, off, y, _native.EPI_BIAS_RELU,
                                                                          before=torch.full_like(dx, FILL))):
            same(got, right)
        backward([33, 50], 300, 200, F32, "kn", _native.EPI_BIAS_RELU)  # the workspace between the replays


def test_refusals():
    x, w, off, y = (torch.zeros(6, 8, device="cuda"), torch.zeros(2, 8, 4, device="cuda"), offsets_of([2, 4]),
                    torch.zeros(6, 4, device="cuda"))
    f, g = lm.grouped_dense_launch, lm.grouped_dense_backward_launch
    for call, error, text in (
            (lambda: f(x, w[0], off, None, y), ValueError, "W must be 3-D"),
            (lambda: f(x, w.half(), off, None, y), TypeError, "W has dtype"),
            (lambda: f(x, w[:, :5], off, None, y), ValueError, "W has shape"),
            (lambda: f(x, torch.zeros(2, 8, 8, device="cuda")[:, :, ::2], off, None, y), ValueError, "unit stride along"),
            (lambda: f(x, w, off[:2], None, y), ValueError, "offsets has shape"),
            (lambda: f(x, w, off.float(), None, y), TypeError, "offsets has dtype"),
            (lambda: f(x, w, off.cpu(), None, y), ValueError, "offsets must be a GPU tensor"),
            (lambda: f(x, w, off, None, y, _native.EPI_BIAS), RuntimeError, "bias is null"),
            (lambda: f(x, w, off, torch.zeros(4, device="cuda"), y, 1), ValueError, "b has shape"),
            (lambda: f(x, w, off, torch.zeros(2, 4, device="cuda").half(), y, 1), TypeError, "b has dtype"),
            (lambda: f(x, w, off, None, y.half()), TypeError, "Y has dtype"),
            (lambda: f(x, w, off, None, y[:5]), ValueError, "Y has shape"),
            (lambda: f(x, w, off, None, y, 8), RuntimeError, "epilogue code 8"),
            (lambda: f(x.int(), w, off, None, y), TypeError, "X has dtype"),
            (lambda: g(y, x, None, off, dX=x), ValueError, "dX needs W"),
            (lambda: g(y, None, w, off, dW=w), ValueError, "dW needs X"),
            (lambda: g(y, x, w, off, x, w, epilogue=_native.EPI_RELU), RuntimeError, "needs Y"),
            (lambda: g(y, x, w, off, x, w, Y=y, epilogue=_native.EPI_LEAKY, alpha=-0.5), RuntimeError, "alpha >= 0"),
            (lambda: g(y, x, w, off, dW=w[:1].expand(2, 8, 4)), ValueError, "one matrix for several"),
            (lambda: g(y, x, w, off, dW=w.half()), TypeError, "dW has dtype"),
            (lambda: g(y, x, w, off, db=y[:3]), ValueError, "db has shape"),
            (lambda: g(y, x, w, off[:0], dX=x), ValueError, "offsets must be a vector")):
        with pytest.raises(error, match=text):
            call()
