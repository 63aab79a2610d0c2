"""The language-model operators that use the library's workspace, from two streams
and from several threads at once: partial sums of the norm's backward pass, of split
4-bit layers (up to 32 rows, and tiles with prepared x), parts of long rows of
logits, and the dense layer's split between them. Each call's results are those of
the same call alone, bit for bit; in the streams' test every call is queued behind a
wait on its stream, so that two would start together if nothing ordered them."""
import threading

import pytest
import torch

from mlir_edsl_hip import _native, last_plan, lm
from mlir_edsl_hip.device import dense_launch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
SPIN_CYCLES = 200_000  # ~0.1 ms


def normal(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def backward(seed):
    M, N = 700, 2048
    dy, h, w, rstd = normal(M, N, seed=seed, dtype=BF16), normal(M, N, seed=seed + 1, dtype=BF16), normal(N, seed=2), \
        normal(M, seed=seed + 3).abs()
    dx, dw = torch.zeros_like(dy), torch.zeros(N, device="cuda")
    return lambda s: lm.rms_norm_backward_launch(dy, h, w, rstd, dx, dw, stream=s), (dx, dw), "+dweight"


def layer(seed, M, K, N, dtype):
    q = torch.randint(0, 16, (K, N), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8).cuda()
    W = lm.q4_pack(q, normal(K // 128, N, seed=seed).abs())
    x, y = normal(M, K, seed=seed + 1, dtype=dtype), torch.zeros(M, N, device="cuda")
    return (lambda s: lm.q4_dense_launch(x, W, None, y, stream=s)), (y,), "+join"


def logits(seed):
    M, V, k = 3, 300000, 8
    x, tokens = normal(M, V, seed=seed), torch.arange(M, device="cuda")
    lp, lse, top, ids = torch.zeros(M, device="cuda"), torch.zeros(M, device="cuda"), torch.zeros(M, k, device="cuda"), \
        torch.zeros(M, k, dtype=torch.int64, device="cuda")
    return lambda s: lm.token_logprobs_launch(x, tokens, lp, lse, None, top, ids, stream=s), (lp, lse, top, ids), "+join"


def dense(seed):
    X, W, Y = normal(16, 2048, seed=seed), normal(2048, 2048, seed=seed + 1), torch.zeros(16, 2048, device="cuda")
    return lambda s: dense_launch(X, W, None, Y, _native.EPI_NONE, stream=s), (Y,), "+reduce"


MAKERS = {"backward": backward, "q4 small": lambda seed: layer(seed, 2, 16384, 512, BF16),
          "q4 tiles": lambda seed: layer(seed, 40, 4096, 1024, F32), "logits": logits, "dense": dense}


def alone(maker, seed):
    """The call and what it gives with nothing else on the device."""
    call, outputs, plan = maker(seed)
    torch.cuda.synchronize()
    call(None)
    assert plan in last_plan(), last_plan()
    torch.cuda.synchronize()
    want = [t.clone() for t in outputs]
    for t in outputs:
        t.zero_()
    torch.cuda.synchronize()
    return call, outputs, want


@pytest.mark.parametrize("first", list(MAKERS))
@pytest.mark.parametrize("second", list(MAKERS))
def test_two_streams(first, second):
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rounds = [[alone(MAKERS[name], 10 * r + 5 * j) for j, name in enumerate((first, second))] for r in range(3)]
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
    names = list(MAKERS) * 2
    cases = [[alone(MAKERS[names[(t + i) % len(names)]], 7 * t + i) for i in range(5)] for t in range(5)]
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
