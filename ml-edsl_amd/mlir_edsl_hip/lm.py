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
* ``q4_pack``, ``q4_dense_launch``: the dense layer on 4-bit weights with group
  scales, and ``q4_quantize`` to make them.
* ``token_logprobs_launch``, ``token_logprobs_backward_launch``: log
  probabilities of given tokens, log-sum-exp, entropy, top alternatives.
"""
from __future__ import annotations

from . import _native, device

_types = None  # torch dtype -> EDSL_LM_* code
_native_module = None  # the checks below and the calls, natively (csrc/lm_torch.cpp), where device.py may use it


def _torch():
    """torch; the first call also maps the library and the stream accessor (device.py)."""
    global _types, _native_module
    torch = device._torch if device._torch is not None else device._torch_module()
    if _types is None:
        _types = {torch.float32: _native.LM_F32, torch.bfloat16: _native.LM_BF16, torch.float16: _native.LM_F16,
                  torch.int8: _native.LM_I8, torch.float8_e4m3fn: _native.LM_E4M3}
        if device._native_launch is not None:
            from . import _torch_launch as _native_module
    return torch


def _done(rc, what) -> bool:
    """Whether a native call was taken; its error is raised. None: the Python
    path runs, and names what is wrong with the arguments."""
    if rc == 0:
        return True
    if rc is not None:
        _native.raise_on_error(what)
    return rc is not None


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
    if _native_module is not None and _done(
            _native_module.rms_norm(X, weight, Y, residual, total, scales, rstd, eps, stream, device._raw_stream),
            "rms_norm_launch"):
        return
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
    if _native_module is not None and _done(
            _native_module.rms_norm_backward(dY, H, weight, rstd, dX, dweight, dh, stream, device._raw_stream),
            "rms_norm_backward_launch"):
        return
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


class Q4Weight:
    """4-bit weights of a [K, N] layer as ``q4_pack`` laid them out."""

    __slots__ = ("packed", "K", "N", "group_size", "scale_type", "has_zeros")

    def __init__(self, packed, K, N, group_size, scale_type, has_zeros):
        self.packed, self.K, self.N = packed, K, N
        self.group_size, self.scale_type, self.has_zeros = group_size, scale_type, has_zeros

    def __repr__(self):
        return (f"Q4Weight({self.K}x{self.N}, group_size={self.group_size}, "
                f"{'zeros, ' if self.has_zeros else ''}{self.packed.numel()} bytes on {self.packed.device})")


def q4_quantize(W, group_size: int = 128, symmetric: bool = False):
    """4-bit integers, scales and zero points (None when symmetric) of a float
    matrix [K, N], each group's extremes at the ends of its range: what
    ``q4_pack`` takes. Torch arithmetic, for the time a model is loaded."""
    torch = _torch()
    if W.dim() != 2 or not W.is_floating_point():
        raise ValueError(f"W must be a 2-D float matrix, got {tuple(W.shape)} {W.dtype}")
    K, N = W.shape
    G = -(-K // group_size)
    w = torch.nn.functional.pad(W.float(), (0, 0, 0, G * group_size - K)).view(G, group_size, N)
    if symmetric:
        scales, zeros, z = w.abs().amax(1) / 7, None, 8.0
    else:
        low, high = w.amin(1).clamp(max=0), w.amax(1).clamp(min=0)
        scales = (high - low) / 15
        z = torch.where(scales > 0, -low / scales, 0.0).round()
        zeros, z = z.to(torch.uint8), z[:, None]
    q = torch.where(scales[:, None] > 0, w / scales[:, None], 0.0).round() + z
    return q.clamp(0, 15).to(torch.uint8).view(G * group_size, N)[:K].contiguous(), scales, zeros


def q4_pack(Q, scales, zeros=None, group_size: int = 128) -> Q4Weight:
    """Lays 4-bit weights out for ``q4_dense_launch``, once:
    ``W[k, n] = scales[k // group_size, n] * (Q[k, n] - zeros[k // group_size, n])``.

    Q [K, N] uint8 of 0 .. 15; scales [G, N] f32, bf16 or f16 with G = K /
    group_size rounded up; zeros [G, N] uint8 of 0 .. 15, 8 where left out.
    group_size is 32, 64 or a multiple of 128. Enqueued on the current stream."""
    torch = _torch()
    K, N = _matrix(Q, "Q", (torch.uint8,))
    scale_type = _types.get(scales.dtype, -1) if scales.dtype in _floats(torch) else -1
    bytes_ = _native.lib().edsl_hip_q4_packed_bytes(K, N, group_size, max(scale_type, 0), zeros is not None)
    if bytes_ < 0:
        _native.raise_on_error("q4_pack")
    G = -(-K // group_size)
    _operand(scales, "scales", (G, N), _floats(torch), Q)
    if zeros is not None:
        _operand(zeros, "zeros", (G, N), (torch.uint8,), Q)
    packed = torch.empty(bytes_, dtype=torch.uint8, device=Q.device)
    if _native.lib().edsl_hip_q4_pack_launch(
            Q.data_ptr(), Q.stride(0), scales.data_ptr(), scales.stride(0), scale_type, _ptr(zeros), _ld(zeros), K, N,
            group_size, packed.data_ptr(), bytes_, _stream(None)):
        _native.raise_on_error("q4_pack")
    return Q4Weight(packed, K, N, group_size, scale_type, zeros is not None)


def q4_dense_launch(X, W: Q4Weight, b, Y, epilogue: int = _native.EPI_NONE, alpha: float = 0.0, x_scales=None,
                    stream=None) -> None:
    """``Y = epilogue(x_scales[:, None] * X @ W (+ b))``, with the epilogues of
    ``device.dense_launch``.

    X is [M, K] in f32, bf16, f16, int8 or float8_e4m3fn, x_scales [M] f32
    (the 8-bit norm's, say), W from ``q4_pack``, Y [M, N] and b [N] in f32, bf16
    or f16. Nothing is rounded before the 32-bit sums. A row of X with an
    infinity or NaN gives a row of NaN, or of 0 under the IF_RELU epilogues
    (y > 0 ? y : 0)."""
    torch = _torch()
    if not isinstance(W, Q4Weight):
        raise TypeError("W is not a Q4Weight")
    if _native_module is not None and _done(
            _native_module.q4_dense(X, W.packed, W.K, W.N, W.group_size, W.scale_type, W.has_zeros, b, Y, epilogue,
                                    alpha, x_scales, stream, device._raw_stream), "q4_dense_launch"):
        return
    M, K = _matrix(X, "X", tuple(_types))
    if K != W.K:
        raise ValueError(f"shape mismatch: X{tuple(X.shape)} W{(W.K, W.N)}")
    if W.packed.device != X.device:
        raise ValueError(f"W is on {W.packed.device}, not on {X.device}")
    _operand(Y, "Y", (M, W.N), _floats(torch), X)
    if b is not None:
        _list(b, "b", (W.N,), _floats(torch), X)
    if x_scales is not None:
        _list(x_scales, "x_scales", (M,), (torch.float32,), X)
    if _native.lib().edsl_hip_q4_dense_launch(
            X.data_ptr(), X.stride(0), _types[X.dtype], _ptr(x_scales), W.packed.data_ptr(), _ptr(b),
            _types[b.dtype] if b is not None else 0, Y.data_ptr(), Y.stride(0), _types[Y.dtype], M, W.N, K,
            W.group_size, W.scale_type, W.has_zeros, epilogue, alpha, _stream(stream)):
        _native.raise_on_error("q4_dense_launch")


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
    if _native_module is not None and _done(
            _native_module.token_logprobs(logits, tokens, logprobs, lse, entropy, top_logprobs, top_ids, scale, stream,
                                          device._raw_stream), "token_logprobs_launch"):
        return
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
    if _native_module is not None and _done(
            _native_module.token_logprobs_backward(logits, tokens, lse, dlogits, dlogprobs, entropy, dentropy, scale,
                                                   stream, device._raw_stream), "token_logprobs_backward_launch"):
        return
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
