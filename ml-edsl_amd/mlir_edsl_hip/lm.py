"""Operators of language models around the dense layer, on torch GPU tensors.

Thin wrappers over the entries of include/edsl_hip_lm.h, in the manner of
``device.dense_launch``: operands and outputs are tensors in HBM that the caller
owns, the kernels are enqueued on a torch stream (the current one by default)
and the call returns without waiting. Matrices have unit inner stride and any
row stride and alignment; vectors are contiguous. An argument that is not taken
raises ``TypeError`` or ``ValueError`` naming it before anything is launched,
and what the library refuses raises ``RuntimeError``.

* ``rms_norm_launch``, ``rms_norm_backward_launch``: the root-mean-square norm
  with the residual's addition, its output in the input's type or in 8 bits.
* ``token_logprobs_launch``, ``token_logprobs_backward_launch``: log
  probabilities of given tokens, log-sum-exp, entropy, top alternatives.
"""
from __future__ import annotations

from . import _native, device

_types = None  # torch dtype -> EDSL_LM_* code


def _torch():
    """torch; the first call also maps the library and the stream accessor (device.py)."""
    global _types
    torch = device._torch if device._torch is not None else device._torch_module()
    if _types is None:
        _types = {torch.float32: _native.LM_F32, torch.bfloat16: _native.LM_BF16, torch.float16: _native.LM_F16,
                  torch.int8: _native.LM_I8, torch.float8_e4m3fn: _native.LM_E4M3}
    return torch


def _stream(stream):
    return stream.cuda_stream if stream is not None else device._raw_stream()


def _operand(t, name, shape, dtypes, like):
    """Checks a tensor: on the GPU of `like`, one of `dtypes`, of this shape,
    rows of unit stride (a vector contiguous)."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dim() >= 1 and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit inner stride")


def _matrix(t, name, dtypes):
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {tuple(t.shape)}")
    _operand(t, name, t.shape, dtypes, t)
    return t.shape


def _list(t, name, shape, dtypes, like):
    """A vector, or [M, k] values in one piece."""
    _operand(t, name, shape, dtypes, like)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _ld(t):
    return t.stride(0) if t is not None else 0


def _floats(torch):
    return torch.float32, torch.bfloat16, torch.float16


def rms_norm_launch(X, weight, Y, residual=None, total=None, scales=None, rstd=None, eps: float = 1e-6,
                    stream=None) -> None:
    """``h = X (+ residual); total = h; Y = h * rstd * weight`` with
    ``rstd = (mean(h**2, 1) + eps) ** -0.5``.

    X, residual and total are [M, N] in f32, bf16 or f16, weight [N] in that
    type or f32. Y has X's type, or is int8 or float8_e4m3fn with ``scales`` [M]
    in f32: ``Y * scales[:, None]`` stands for the output, the largest value of
    a row at 127 or 448. rstd [M] f32 is what the backward pass needs. The norm
    is that of h in 32 bits. total may be X or residual, and Y any of the three
    in their type."""
    torch = _torch()
    shape = _matrix(X, "X", _floats(torch))
    eight = (torch.int8, torch.float8_e4m3fn)
    _list(weight, "weight", shape[1:], (X.dtype, torch.float32), X)
    _operand(Y, "Y", shape, (X.dtype, *eight), X)
    for t, name in ((residual, "residual"), (total, "total")):
        if t is not None:
            _operand(t, name, shape, (X.dtype,), X)
    if (scales is None) == (Y.dtype in eight):
        raise ValueError("scales belong to an int8 or float8_e4m3fn Y" if scales is not None else
                         f"Y in {Y.dtype} needs scales")
    for t, name in ((scales, "scales"), (rstd, "rstd")):
        if t is not None:
            _list(t, name, shape[:1], (torch.float32,), X)
    M, N = shape
    if _native.lib().edsl_hip_rms_norm_launch(
            X.data_ptr(), X.stride(0), _ptr(residual), _ld(residual), weight.data_ptr(), _types[weight.dtype],
            _ptr(total), _ld(total), Y.data_ptr(), Y.stride(0), _types[Y.dtype], _ptr(scales), _ptr(rstd), M, N,
            _types[X.dtype], eps, _stream(stream)):
        _native.raise_on_error("rms_norm_launch")


def rms_norm_backward_launch(dY, H, weight, rstd, dX, dweight=None, dh=None, stream=None) -> None:
    """The gradients of ``rms_norm_launch``: H is the total that was normalised
    (X where there is no residual), dY the gradient of Y, dh that of total.
    dX receives the gradient of X, which is the residual's too, and dweight [N]
    f32 the weight's, summed over the rows in a fixed order. dX may be dY, H or
    dh."""
    torch = _torch()
    shape = _matrix(dY, "dY", _floats(torch))
    _operand(H, "H", shape, (dY.dtype,), dY)
    _list(weight, "weight", shape[1:], (dY.dtype, torch.float32), dY)
    _list(rstd, "rstd", shape[:1], (torch.float32,), dY)
    _operand(dX, "dX", shape, (dY.dtype,), dY)
    if dweight is not None:
        _list(dweight, "dweight", shape[1:], (torch.float32,), dY)
    if dh is not None:
        _operand(dh, "dh", shape, (dY.dtype,), dY)
    M, N = shape
    if _native.lib().edsl_hip_rms_norm_backward_launch(
            dY.data_ptr(), dY.stride(0), H.data_ptr(), H.stride(0), weight.data_ptr(), _types[weight.dtype],
            rstd.data_ptr(), _ptr(dh), _ld(dh), dX.data_ptr(), dX.stride(0), _ptr(dweight), M, N, _types[dY.dtype],
            _stream(stream)):
        _native.raise_on_error("rms_norm_backward_launch")


def _tokens(torch, tokens, logits):
    _list(tokens, "tokens", logits.shape[:1], (torch.int64, torch.int32), logits)
    return tokens.dtype == torch.int64


def token_logprobs_launch(logits, tokens=None, logprobs=None, lse=None, entropy=None, top_logprobs=None, top_ids=None,
                          scale: float = 1.0, stream=None) -> None:
    """Log probabilities under ``softmax(scale * logits)`` of each row.

    logits are [M, V] in f32, bf16 or f16, tokens [M] in int64 or int32 (one
    outside 0 .. V-1, as padding has, gets 0). Each output is written where it
    is given: logprobs, lse and entropy [M] f32, and the k largest of each row
    in falling order, equal logits by their index, in top_logprobs [M, k] f32
    and top_ids [M, k] int64 or int32 (as tokens; k at most 32 and V).
    A logit of -inf has probability 0; in a row of nothing else lse and the log
    probabilities are -inf and the entropy 0. A row with a NaN or +inf gives
    NaN and ids -1."""
    torch = _torch()
    M, V = _matrix(logits, "logits", _floats(torch))
    ids64 = _tokens(torch, tokens, logits) if tokens is not None else True
    for t, name in ((logprobs, "logprobs"), (lse, "lse"), (entropy, "entropy")):
        if t is not None:
            _list(t, name, (M,), (torch.float32,), logits)
    if logprobs is not None and tokens is None:
        raise ValueError("logprobs need tokens")
    if (top_logprobs is None) != (top_ids is None):
        raise ValueError("top_logprobs and top_ids come together")
    k = 0
    if top_ids is not None:
        if top_ids.dim() != 2:
            raise ValueError(f"top_ids must be 2-D, got {tuple(top_ids.shape)}")
        k = top_ids.shape[1]
        _list(top_logprobs, "top_logprobs", (M, k), (torch.float32,), logits)
        _list(top_ids, "top_ids", (M, k),
              (torch.int64, torch.int32) if tokens is None else (tokens.dtype,), logits)
        ids64 = top_ids.dtype == torch.int64
    if _native.lib().edsl_hip_token_logprobs_launch(
            logits.data_ptr(), logits.stride(0), _types[logits.dtype], _ptr(tokens), ids64, _ptr(logprobs), _ptr(lse),
            _ptr(entropy), _ptr(top_logprobs), _ptr(top_ids), k, M, V, scale, _stream(stream)):
        _native.raise_on_error("token_logprobs_launch")


def token_logprobs_backward_launch(logits, tokens, lse, dlogits, dlogprobs=None, entropy=None, dentropy=None,
                                   scale: float = 1.0, stream=None) -> None:
    """The gradient of the logits, in their type, given those of logprobs
    (dlogprobs [M] f32, with tokens) and of entropy (dentropy [M] f32, with the
    entropy that the forward pass gave); either may be left out. lse is the
    forward pass's. A padding token's dlogprobs counts as 0, and so does
    everything in a row of -inf alone. dlogits may be logits."""
    torch = _torch()
    M, V = _matrix(logits, "logits", _floats(torch))
    ids64 = _tokens(torch, tokens, logits) if tokens is not None else True
    _list(lse, "lse", (M,), (torch.float32,), logits)
    _operand(dlogits, "dlogits", (M, V), (logits.dtype,), logits)
    for t, name in ((dlogprobs, "dlogprobs"), (entropy, "entropy"), (dentropy, "dentropy")):
        if t is not None:
            _list(t, name, (M,), (torch.float32,), logits)
    if dlogprobs is not None and tokens is None:
        raise ValueError("dlogprobs need tokens")
    if dentropy is not None and entropy is None:
        raise ValueError("dentropy needs entropy")
    if _native.lib().edsl_hip_token_logprobs_backward_launch(
            logits.data_ptr(), logits.stride(0), _types[logits.dtype], _ptr(tokens), ids64, lse.data_ptr(),
            _ptr(dlogprobs), _ptr(entropy), _ptr(dentropy), dlogits.data_ptr(), dlogits.stride(0), M, V, scale,
            _stream(stream)):
        _native.raise_on_error("token_logprobs_backward_launch")
