"""Sampling where the kept logits are few, thousands, and more than are held apart from the row: each setting
at sizes on both sides, against 64 bits."""
import pytest
import torch

from test_gpu_lm_sample import TYPES, check, logits, uniforms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("settings", [
    dict(top_p=0.8), dict(top_p=0.9), dict(top_p=0.95), dict(top_p=0.99), dict(top_p=0.9999), dict(min_p=1e-3),
    dict(min_p=1e-5), dict(top_k=1024), dict(top_k=1025), dict(top_k=5000), dict(top_k=12288), dict(top_k=12289),
    dict(top_k=5000, top_p=0.97), dict(top_k=14000, top_p=0.999, min_p=1e-7), dict(temperature=3.0, top_p=0.5)], ids=str)
def test_numbers_of_candidates(dtype, settings):
    x = logits(3, 50257, seed=21, dtype=TYPES[dtype])
    check(x, uniforms(3, seed=22), **settings)
    x[:, 100:13000] = x[:, 100:101]  # as many equal ones as are held apart, and more
    check(x, uniforms(3, seed=23), **settings)
