"""The native operand checks (csrc/lm_torch.cpp) of the launches of the 8-bit layer, the layer on groups of rows and
sampling against the Python ones of lm.py: the same calls are taken, with the same bits, and the same refused, with the same error."""
import pytest
import torch

from mlir_edsl_hip import lm
from test_gpu_lm_binding import CHANGES

pytestmark = pytest.mark.gpu


def arguments(op):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    if op == "i8_dense_launch":
        i = lambda *s: torch.randint(-128, 128, s, generator=g).to(torch.int8).cuda()  # noqa: E731
        return dict(X=i(6, 40), W=lm.i8_pack(i(40, 24), r(24)), b=r(24), Y=torch.zeros(6, 24, device="cuda"), epilogue=3,
                    alpha=0.5, x_scales=r(6))
    off = torch.tensor([0, 2, 6], dtype=torch.int32).cuda()
    if op == "grouped_dense_launch":
        return dict(X=r(6, 40), W=r(2, 40, 24), offsets=off, b=r(2, 24), Y=torch.zeros(6, 24, device="cuda"), epilogue=3,
                    alpha=0.5)
    if op == "grouped_dense_backward_launch":
        return dict(dY=r(6, 24), X=r(6, 40), W=r(2, 40, 24), offsets=off, dX=torch.zeros(6, 40, device="cuda"),
                    dW=torch.zeros(2, 40, 24, device="cuda"), db=torch.zeros(2, 24, device="cuda"), Y=r(6, 24), epilogue=5,
                    alpha=0.5)
    f = lambda v: torch.full((6,), v, device="cuda")  # noqa: E731
    return dict(logits=r(6, 40), uniforms=torch.rand(6, generator=g).cuda(), tokens=torch.zeros(6, dtype=torch.int64, device="cuda"),
                logprobs=f(0.0), temperature=f(0.7), top_k=torch.full((6,), 9, dtype=torch.int32, device="cuda"), top_p=f(0.9),
                min_p=f(0.01))


OPS = ["i8_dense_launch", "grouped_dense_launch", "grouped_dense_backward_launch", "sample_tokens_launch"]
MORE = {**CHANGES, "one": lambda t: 1, "half_number": lambda t: 0.5, "swapped": lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)
        if t.dim() > 1 else t, "expanded": lambda t: t[:1].expand_as(t)}


def call(op, name, change):
    args = arguments(op)
    if name:
        args[name] = MORE[change](args[name])
    try:
        getattr(lm, op)(**args)
    except Exception as e:  # noqa: BLE001 -- what is compared
        return type(e), str(e)
    return [v.detach().cpu().clone() for v in args.values() if isinstance(v, torch.Tensor)]


@pytest.mark.parametrize("op", OPS)
def test_native_checks_agree_with_python(op, monkeypatch):
    lm._torch()
    native = lm._native_module
    assert native is not None, "the torch launch module is not built"
    names = list(arguments(op))
    taken = 0
    for name in names:
        number = not isinstance(arguments(op)[name], torch.Tensor)
        for change in (("none", "text", "left_out") if number else MORE):
            if change == "expanded" and name in ("tokens", "logprobs", "db", "Y", "dX"):
                continue  # one memory for several results has no one value
            monkeypatch.setattr(lm, "_native_module", native)
            got = call(op, name, change)
            monkeypatch.setattr(lm, "_native_module", None)
            want = call(op, name, change)
            if isinstance(want, tuple):
                assert got == want, (name, change)
            else:
                taken += 1
                assert isinstance(got, list), (name, change, got)
                assert all(torch.equal(a, b) or bool((a.isnan() & b.isnan() | (a == b)).all()) for a, b in zip(got, want)), \
                    (name, change)
    assert taken > len(names) // 2
