"""The native operand checks of the language-model launches (csrc/lm_torch.cpp)
against the Python ones of lm.py: the same calls are taken, with the same bits,
and the same refused, with the same error."""
import pytest
import torch

from mlir_edsl_hip import lm

pytestmark = pytest.mark.gpu


class Sub(torch.Tensor):
    pass


def arguments(op):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x = r(6, 40)
    vec = lambda: torch.zeros(6, device="cuda")  # noqa: E731
    if op == "rms_norm_launch":
        return dict(X=x, weight=r(40), Y=torch.zeros_like(x), residual=r(6, 40), total=torch.zeros_like(x),
                    scales=None, rstd=vec(), eps=1e-5)
    if op == "rms_norm_backward_launch":
        return dict(dY=r(6, 40), H=x, weight=r(40), rstd=vec() + 1, dX=torch.zeros_like(x),
                    dweight=torch.zeros(40, device="cuda"), dh=r(6, 40))
    tokens = torch.randint(0, 40, (6,), generator=g).cuda()
    if op == "token_logprobs_launch":
        return dict(logits=x, tokens=tokens, logprobs=vec(), lse=vec(), entropy=vec(),
                    top_logprobs=torch.zeros(6, 3, device="cuda"),
                    top_ids=torch.zeros(6, 3, dtype=torch.int64, device="cuda"), scale=0.5)
    if op == "token_logprobs_backward_launch":
        return dict(logits=x, tokens=tokens, lse=vec() + 4, dlogits=torch.zeros_like(x), dlogprobs=r(6),
                    entropy=vec() + 1, dentropy=r(6), scale=0.5)
    q = torch.randint(0, 16, (40, 24), generator=g, dtype=torch.uint8).cuda()
    return dict(X=x, W=lm.q4_pack(q, r(2, 24), group_size=32), b=r(24), Y=torch.zeros(6, 24, device="cuda"),
                epilogue=3, alpha=0.5, x_scales=vec() + 2)


OPS = ["rms_norm_launch", "rms_norm_backward_launch", "q4_dense_launch", "token_logprobs_launch",
       "token_logprobs_backward_launch"]
CHANGES = {
    "none": lambda t: t, "left_out": lambda t: None, "host": lambda t: t.cpu(), "half": lambda t: t.half(),
    "int32": lambda t: t.int(), "float64": lambda t: t.double(), "fewer": lambda t: t[:-1],
    "transposed": lambda t: t.t() if t.dim() == 2 else t, "parameter": lambda t: torch.nn.Parameter(t.clone(), False),
    "strided": lambda t: torch.stack((t, t), -1).flatten(-2)[..., ::2], "subclass": lambda t: t.as_subclass(Sub),
    "padded_rows": lambda t: torch.cat((t, t), -1)[..., :t.shape[-1]] if t.dim() == 2 else t, "text": lambda t: "x",
}


def call(op, name, change):
    args = arguments(op)
    if name:
        args[name] = CHANGES[change](args[name])
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
    names = [n for n, v in arguments(op).items() if isinstance(v, torch.Tensor)] + [
        n for n in ("eps", "scale", "epilogue", "alpha") if n in arguments(op)]
    taken = 0
    for name in names:
        number = name in ("eps", "scale", "epilogue", "alpha")
        for change in (("none", "text", "left_out") if number else CHANGES):
            monkeypatch.setattr(lm, "_native_module", native)
            got = call(op, name, change)
            monkeypatch.setattr(lm, "_native_module", None)
            want = call(op, name, change)
            if isinstance(want, tuple):
                assert got == want, (name, change)
            else:
                taken += 1
                assert isinstance(got, list), (name, change, got)
                assert all(torch.equal(a, b) for a, b in zip(got, want)), (name, change)
    assert taken >= len(names)
