"""The norm's 8-bit codes, bit for bit.

A code is y / scale = h w Q / max |h w| rounded to nearest even, whatever the norm.
h and w here are integers of 8 bits at most by a power of two (another one in some
rows), so that h w (16 bits) and h w Q by a power of two (3 bits more for 448, 7 for
127) are exact in 32 bits. The quotient's 32-bit rounding does not reach a midpoint
between codes: where h w Q is not the midpoint m max |h w| itself it is off by a
unit of a number under 2^24 (8 bits of m, 16 of the maximum), and half a unit in the
last place of the quotient is no more than that. So the codes are those of 64 bits."""
import pytest
import torch

import lm_reference as ref
from mlir_edsl_hip import lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def codes(q, out):
    """64-bit values to the codes of an 8-bit type, ties to even."""
    if out == I8:
        return q.round()
    step = 2.0 ** (torch.frexp(q)[1] - 1).clamp(min=-6).double() / 8  # 3 bits after the first; 2^-9 near zero
    return (q / step).round() * step


@pytest.mark.parametrize("out", [I8, E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("N", [7, 120, 250, 512, 1000, 2001, 4000, 8192, 16000, 40000])
def test_codes_are_the_nearest_even(N, residual, dtype, out):
    M = 40
    g = torch.Generator().manual_seed(N)
    h = torch.randint(-255, 256, (M, N), generator=g) / 16
    # Rows of ordinary, large and small values: norms from 2^40 down to where eps is all of it.
    size = torch.tensor([1.0, 2.0 ** 40, 2.0 ** -20, 2.0 ** -70, 2.0 ** -110, 2.0 ** -121])[torch.arange(M) % 6, None]
    r = torch.randint(-127, 128, (M, N), generator=g) / 16 if residual else None
    if residual:
        h = (h / 2).mul(16).trunc() / 16
    x, w = (h * size).to(dtype), torch.randint(1, 129, (N,), generator=g) / 64
    assert torch.equal(ref.d(x), ref.d(h) * ref.d(size))
    res = (r * size).to(dtype).cuda() if residual else None
    y, scales = torch.empty(M, N, dtype=I8, device="cuda").view(out), torch.empty(M, device="cuda")
    lm.rms_norm_launch(x.cuda(), w.cuda(), y, residual=res, scales=scales)
    hw = (ref.d(x) + (ref.d(res) if residual else 0.0)) * ref.d(w)
    want = codes(hw * (127.0 if out == I8 else 448.0) / hw.abs().amax(1, keepdim=True), out)
    assert torch.equal(ref.d(y.to(F32)), want)
