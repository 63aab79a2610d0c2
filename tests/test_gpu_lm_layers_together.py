"""The layers and sampling as a model uses them: steps of a decoder with experts, eager and captured, each
operator against 64 bits on what it was given; a two-layer expert's training step; and their calls from two
streams and several threads at once."""
import math
import threading

import pytest
import torch

import lm_layers_reference as layers
import lm_reference as ref
from mlir_edsl_hip import _native, last_plan, lm
from test_gpu_lm_grouped import near, offsets_of, same, whole
from test_gpu_lm_streams import MAKERS, SPIN_CYCLES, alone

pytestmark = pytest.mark.gpu
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


class Decoder:
    """A block with an 8-bit layer and experts over a table of tokens, and a head in 8 bits; the next token is drawn."""

    def __init__(self, rows, hidden, inner, experts, vocabulary):
        g = torch.Generator().manual_seed(5)
        r = lambda *s, dtype=F32: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
        self.experts, self.rows = experts, rows
        self.table, self.norm = r(vocabulary, hidden, dtype=BF16), [r(hidden) * 0.1 + 1 for _ in range(3)]
        self.mixed, self.head_q = (lm.i8_quantize(r(hidden, n) / hidden ** 0.5) for n in (hidden, vocabulary))
        self.mix, self.head = lm.i8_pack(*self.mixed), lm.i8_pack(*self.head_q)
        self.router = r(hidden, experts)
        self.up, self.b, self.down = r(experts, hidden, inner, dtype=BF16) / hidden ** 0.5, r(experts, inner, dtype=BF16), \
            r(experts, inner, hidden, dtype=BF16) / inner ** 0.5
        e = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.q, self.scales = e(rows, hidden, dtype=I8), e(rows, dtype=F32)
        self.x1, self.total, self.x2 = e(rows, hidden), e(rows, hidden), e(rows, hidden)
        self.h, self.y = e(rows, inner), e(rows, hidden)
        self.last_q, self.last_scales, self.logits = e(rows, hidden, dtype=I8), e(rows, dtype=F32), e(rows, vocabulary, dtype=F32)
        self.tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
        self.logprobs, self.uniforms = e(rows, dtype=F32), torch.empty(rows, device="cuda")

    def step(self):
        self.x = self.table[self.tokens]
        lm.rms_norm_launch(self.x, self.norm[0], self.q, scales=self.scales)
        lm.i8_dense_launch(self.q, self.mix, None, self.x1, x_scales=self.scales)
        lm.rms_norm_launch(self.x1, self.norm[1], self.x2, residual=self.x, total=self.total)
        # Rows in the order of their experts.
        expert = (self.x2.float() @ self.router).argmax(1)
        order = expert.argsort(stable=True)
        ends = torch.searchsorted(expert[order], torch.arange(self.experts + 1, device="cuda"))
        self.offsets, self.sorted = ends, self.x2[order]
        lm.grouped_dense_launch(self.sorted, self.up, ends, self.b, self.h, _native.EPI_BIAS_RELU)
        lm.grouped_dense_launch(self.h, self.down, ends, None, self.y)
        self.back = torch.empty_like(self.y).index_copy_(0, order, self.y)
        lm.rms_norm_launch(self.back, self.norm[2], self.last_q, residual=self.total, scales=self.last_scales)
        lm.i8_dense_launch(self.last_q, self.head, None, self.logits, x_scales=self.last_scales)
        lm.sample_tokens_launch(self.logits, self.uniforms, self.tokens, self.logprobs, temperature=0.8, top_k=50, top_p=0.95)

    def check(self):
        for q, s, w, y in ((self.q, self.scales, self.mixed, self.x1), (self.last_q, self.last_scales, self.head_q, self.logits)):
            want, size = layers.i8_dense(q, *w, s)
            bound = 7 * 2.0 ** -24 * size + ref.HALF_ULP[y.dtype] * want.abs() + ref.TINY[y.dtype]
            assert float(((ref.d(y) - want).abs() - bound).max()) <= 0
        args = self.sorted, self.up, self.offsets, self.b, _native.EPI_BIAS_RELU
        near(self.h, layers.grouped_dense(*args), layers.grouped_dense(*(t.abs() if torch.is_tensor(t) else t for t in args)),
             self.up.shape[1] + 1)
        near(self.y, layers.grouped_dense(self.h, self.down, self.offsets),
             layers.grouped_dense(self.h.abs(), self.down.abs(), self.offsets), self.up.shape[2])
        for m in range(self.rows):
            token, logprob = layers.sample(self.logits[m], self.uniforms[m], 0.8, 50, 0.95)
            # One rounding to 32 bits, and masses in units of 2^-46 of the largest weight.
            bound = 2.0 ** -23 * abs(logprob) + self.logits.shape[1] * 2.0 ** -45 * math.exp(-logprob)
            assert int(self.tokens[m]) == token and abs(float(self.logprobs[m]) - logprob) <= bound


@pytest.mark.parametrize("rows", [1, 7, 150])
def test_steps_of_a_decoder(rows):
    net, u = Decoder(rows, 256, 512, 6, 3001), torch.rand(5, rows, generator=torch.Generator().manual_seed(9)).cuda()
    eager = []
    for i in range(5):
        net.uniforms.copy_(u[i])
        net.step()
        net.check()
        eager.append((net.tokens.clone(), net.logprobs.clone()))
    assert rows == 1 or len({tuple(t.tolist()) for t, _ in eager}) > 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        net.step()
    net.tokens.zero_()
    for i in range(5):
        net.uniforms.copy_(u[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(net.tokens, eager[i][0]) and torch.equal(net.logprobs, eager[i][1])
        other = Decoder(3, 256, 512, 6, 3001)  # eager work between the replays
        other.uniforms.fill_(0.5)
        other.step()


@pytest.mark.parametrize("counts", [[1, 0, 5], [200, 40, 0, 90]], ids=str)
def test_training_step_of_two_layers(counts):
    """Integers: the gradients of the whole are exact, and equal to those of automatic differentiation in 64 bits."""
    T, E, K, H, N = sum(counts), len(counts), 40, 56, 24
    x, w1, b1, w2, dy = (whole(*s, seed=i, dtype=F32, most=2) for i, s in
                         enumerate(((T, K), (E, K, H), (E, H), (E, H, N), (T, N))))
    off = offsets_of(counts)
    h, y = torch.empty(T, H, device="cuda"), torch.empty(T, N, device="cuda")
    lm.grouped_dense_launch(x, w1, off, b1, h, _native.EPI_BIAS_RELU)
    lm.grouped_dense_launch(h, w2, off, None, y)
    dh, dx = torch.empty_like(h), torch.empty_like(x)
    dw1, db1, dw2 = torch.empty_like(w1), torch.empty_like(b1), torch.empty_like(w2)
    lm.grouped_dense_backward_launch(dy, h, w2, off, dh, dw2)
    lm.grouped_dense_backward_launch(dh, x, w1, off, dx, dw1, db1, h, _native.EPI_BIAS_RELU)
    X, W1, B1, W2 = (t.double().cpu().requires_grad_() for t in (x, w1, b1, w2))
    parts = [((X[r] @ W1[e] + B1[e]).relu() @ W2[e]) for e, r in layers.runs(off)]
    Y = torch.cat(parts)
    Y.backward(dy.double().cpu())
    for got, want in ((y, Y.detach()), (dx, X.grad), (dw1, W1.grad), (db1, B1.grad), (dw2, W2.grad)):
        same(got.cpu(), want)


def normal(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def gradients(seed):
    counts = [300, 10, 90]
    T, K, N = sum(counts), 512, 640
    dy, x, w, y = normal(T, N, seed=seed), normal(T, K, seed=seed + 1), normal(3, K, N, seed=2), normal(T, N, seed=seed + 3)
    off, outs = offsets_of(counts), (torch.zeros_like(x), torch.zeros(3, K, N, device="cuda"), torch.zeros(3, N, device="cuda"))
    return lambda s: lm.grouped_dense_backward_launch(dy, x, w, off, *outs, y, _native.EPI_RELU, stream=s), outs, "mask"


def sampled(seed):
    x, u = normal(20, 30000, seed=seed), torch.rand(20, generator=torch.Generator().manual_seed(seed)).cuda()
    outs = torch.zeros(20, dtype=torch.int64, device="cuda"), torch.zeros(20, device="cuda")
    return lambda s: lm.sample_tokens_launch(x, u, *outs, top_k=40, top_p=0.9, stream=s), outs, "sample"


OURS = {"gradients": gradients, "sampled": sampled}
ALL = {**OURS, "norm": MAKERS["backward"], "logits": MAKERS["logits"]}


@pytest.mark.parametrize("first", list(OURS))
@pytest.mark.parametrize("second", list(ALL))
def test_two_streams(first, second):
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rounds = [[alone(ALL[name], 10 * r + 5 * j) for j, name in enumerate((first, second))] for r in range(3)]
    for pair in rounds:
        for s, (call, _, _) in zip(streams, pair):
            with torch.cuda.stream(s):
                torch.cuda._sleep(SPIN_CYCLES)
                call(s)
    torch.cuda.synchronize()
    for r, pair in enumerate(rounds):
        for j, (_, outputs, want) in enumerate(pair):
            assert all(torch.equal(a, b) for a, b in zip(outputs, want)), (r, j)


def test_threads():
    names = list(ALL) * 2
    cases = [[alone(ALL[names[(t + i) % len(names)]], 7 * t + i) for i in range(4)] for t in range(4)]
    errors = []

    def worker(mine):
        try:
            s = torch.cuda.Stream()
            for call, outputs, want in mine:
                for _ in range(3):
                    call(s)
                s.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(outputs, want))
        except BaseException as e:  # noqa: BLE001 -- reported by the test's own thread
            errors.append(e)
    threads = [threading.Thread(target=worker, args=(mine,)) for mine in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_two_graphs_that_share_the_workspace():
    """Captured one after the other and replayed in both orders on one stream, with eager calls between."""
    cases, graphs = [alone(gradients, 3), alone(gradients, 30)], []
    for call, _, _ in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(None)
    eager = alone(MAKERS["backward"], 5)
    for order in ((0, 1), (1, 0), (0, 1), (1, 1)):
        for i in order:
            for t in cases[i][1]:
                t.zero_()
            eager[0](None)
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in set(order):
            assert all(torch.equal(a, b) for a, b in zip(cases[i][1], cases[i][2])), (order, i)
    assert last_plan()
