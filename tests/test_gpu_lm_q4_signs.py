"""The 4-bit layer where the sum of x is as large as that of its sizes: x of one sign,
as a ReLU leaves it, and x with one large element.

Tolerance: 16-bit and 8-bit x meet weights held as 16 + q, less 16 + z times x's sum, so
that the terms that pass through the 32-bit sums amount to |x| s (32 + q + z). With the
roundings of test_gpu_lm_q4.py, (min(K, 128) + K / 32 + 48) 2^-23 of that, then those of
the result: 8 * 2^-24 and one to its type."""
import pytest
import torch

import lm_reference as ref
from mlir_edsl_hip import lm
from test_gpu_lm_q4 import BF16, E4M3, F16, F32, I8, expect, make_weights, make_x, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["relu", "one large", "equal"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, I8, E4M3])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,K,N,group", [(1, 4096, 130, 128), (12, 1000, 8300, 32), (24, 2048, 300, 64),
                                         (100, 4096, 520, 128), (600, 1000, 2100, 32)])
def test_one_sign(M, K, N, group, zeros, dtype, kind):
    x = make_x(M, K, dtype)
    if kind == "relu":
        x = x.float().clamp(min=0).to(dtype)
    elif kind == "equal":
        x = torch.full((M, K), 1.75 if dtype != I8 else 127.0, device="cuda").to(dtype)
    else:
        x = x.float()
        x[:, K // 3] = {F32: 1e6, BF16: 1e6, F16: 6e4, I8: 127.0, E4M3: 448.0}[dtype]
        x = x.to(dtype)
    q, s, z = make_weights(K, N, group, BF16, zeros)
    y = torch.empty(M, N, device="cuda")
    lm.q4_dense_launch(x, lm.q4_pack(q, s, z, group_size=group), None, y)
    want, _ = expect(x, q, s, z, group)
    at = torch.arange(K) // group
    size = wide(x).abs() @ ((32 + ref.d(q) + (ref.d(z)[at] if zeros else 8.0)) * ref.d(s)[at])
    bound = (min(K, 128) + K / 32 + 48) * 2.0 ** -23 * size + 9 * 2.0 ** -24 * want.abs() + ref.TINY[F32]
    worst = float(((ref.d(y) - want).abs() - bound).max())
    assert worst <= 0, worst
