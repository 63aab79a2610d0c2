"""Sampling from finite logits further apart than the largest 32-bit number, at temperatures at which their weights are
of the same size, against 64 bits. Bounds as for other logits (test_gpu_lm_sample.py)."""
import math

import pytest
import torch

from test_gpu_lm_sample import TYPES, check, draw, uniforms

pytestmark = pytest.mark.gpu
SETTINGS = [{}, dict(top_k=1), dict(top_k=2), dict(top_k=30), dict(top_k=1500), dict(top_p=0.999), dict(top_p=0.5),
            dict(min_p=0.003), dict(min_p=0.5), dict(top_k=2, top_p=0.9), dict(top_k=1500, top_p=0.9, min_p=0.2)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1e37, 1e38, 3e38])
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_both_ends_of_the_type(dtype, temperature, settings):
    t = TYPES[dtype]
    most = torch.finfo(t).max
    few = torch.tensor([[3e38, -3e38, -3.1e38], [-3.1e38, 3e38, -3e38], [most, -most, most], [-most, -most, -math.inf],
                        [most, -math.inf, 0.0]]).to(t).cuda()
    check(few, uniforms(5, seed=1), temperature=temperature, **settings)
    for V in (700, 5003, 40000):
        x = (2 * torch.rand(6, V, generator=torch.Generator().manual_seed(V)) - 1) * 3.3e38
        x[3:, ::3] = -math.inf
        check(x.to(t).cuda(), uniforms(6, seed=V), temperature=temperature, **settings)


def test_top_k_of_the_far_ones():
    """Weights 1, 0.0025 and 0.0022: of the two largest, the second is drawn at the end of the range and the third never."""
    x = torch.tensor([[3e38, -3e38, -3.1e38]], device="cuda").expand(2, 3).contiguous()
    u = torch.tensor([0.5, 1 - 2.0 ** -24], device="cuda")
    assert draw(x, u, temperature=1e38, top_k=2)[0].tolist() == [0, 1]
    assert draw(x, u, temperature=1e38, top_p=0.999)[0].tolist() == [0, 2]
    assert draw(x, u, temperature=1e38, top_p=0.997)[0].tolist() == [0, 1]
