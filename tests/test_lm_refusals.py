"""What the entries of include/edsl_hip_lm.h refuse, and the calls with nothing to
do: decided on the host before any device is looked at, so checked without one."""
import ctypes

import pytest

from mlir_edsl_hip import _native, last_plan

P = 0x1000  # an address; nothing is read there


def message():
    buf = ctypes.create_string_buffer(512)
    _native.lib().edsl_hip_last_error(buf, len(buf))
    return buf.value.decode()


# Arguments of a call that would be taken, in the header's order.
CALLS = {
    "rms_norm": dict(x=P, ldx=8, residual=None, ldr=0, weight=P, weight_type=0, total=None, ldt=0, y=P, ldy=8, y_type=0,
                     scales=None, rstd=None, M=4, N=8, type=0, eps=1e-6, stream=None),
    "rms_norm_backward": dict(dy=P, lddy=8, h=P, ldh=8, weight=P, weight_type=0, rstd=P, dh=None, lddh=0, dx=P, lddx=8,
                              dweight=None, M=4, N=8, type=0, stream=None),
    "token_logprobs": dict(logits=P, ldl=8, type=0, tokens=P, ids64=1, logprobs=P, lse=P, entropy=P, top_logprobs=P,
                           top_ids=P, k=2, M=4, V=8, scale=1.0, stream=None),
    "token_logprobs_backward": dict(logits=P, ldl=8, type=0, tokens=P, ids64=1, lse=P, dlogprobs=P, entropy=P,
                                    dentropy=P, dlogits=P, lddl=8, M=4, V=8, scale=1.0, stream=None),
    "q4_pack": dict(q=P, ldq=16, scales=P, lds=16, scale_type=0, zeros=None, ldz=0, K=128, N=16, group=128, packed=P,
                    packed_bytes=1 << 20, stream=None),
    "q4_dense": dict(X=P, ldx=128, x_type=0, x_scales=None, packed=P, bias=P, bias_type=0, Y=P, ldy=16, y_type=0, M=4,
                     N=16, K=128, group=128, scale_type=0, has_zeros=0, epilogue=1, alpha=0.0, stream=None),
}
MORE = (1 << 30) + 1
REFUSED = [
    ("rms_norm", dict(type=3), "x: type 3"), ("rms_norm", dict(weight_type=1), "weight: type 1"),
    ("rms_norm", dict(y_type=2), "y: type 2"), ("rms_norm", dict(y_type=3), "needs scales"),
    ("rms_norm", dict(scales=P), "scales are of an 8-bit y"), ("rms_norm", dict(eps=-1.0), "eps"),
    ("rms_norm", dict(eps=float("nan")), "eps"), ("rms_norm", dict(N=0), "no norm"),
    ("rms_norm", dict(M=-1), "negative"), ("rms_norm", dict(M=MORE), "2^30"),
    ("rms_norm", dict(x=None), "x is null"), ("rms_norm", dict(weight=None), "weight is null"),
    ("rms_norm", dict(y=None), "y is null"), ("rms_norm", dict(ldx=7), "x: row stride 7"),
    ("rms_norm", dict(ldy=7), "y: row stride 7"), ("rms_norm", dict(residual=P), "residual: row stride 0"),
    ("rms_norm", dict(total=P, ldt=7), "total: row stride 7"),
    ("rms_norm_backward", dict(type=4), "dy: type 4"), ("rms_norm_backward", dict(weight_type=2), "weight: type 2"),
    ("rms_norm_backward", dict(N=0), "no norm"), ("rms_norm_backward", dict(h=None), "h is null"),
    ("rms_norm_backward", dict(rstd=None), "rstd is null"), ("rms_norm_backward", dict(weight=None), "weight is null"),
    ("rms_norm_backward", dict(dh=P, lddh=7), "dh: row stride 7"), ("rms_norm_backward", dict(lddx=0), "dx: row stride"),
    ("token_logprobs", dict(type=5), "logits: type 5"), ("token_logprobs", dict(scale=0.0), "scale"),
    ("token_logprobs", dict(scale=float("inf")), "scale"), ("token_logprobs", dict(k=33), "k=33"),
    ("token_logprobs", dict(k=-1), "k=-1"), ("token_logprobs", dict(k=9), "k=9 alternatives of V=8"),
    ("token_logprobs", dict(top_ids=None), "top_ids"), ("token_logprobs", dict(tokens=None), "need tokens"),
    ("token_logprobs", dict(V=0), "no logits"), ("token_logprobs", dict(V=(1 << 21) + 1, ldl=1 << 22), "2^21"),
    ("token_logprobs", dict(logits=None), "logits is null"), ("token_logprobs", dict(ldl=7), "row stride 7"),
    ("token_logprobs_backward", dict(M=1 << 30, V=1 << 20, ldl=1 << 20, lddl=1 << 20), "one launch"),
    ("token_logprobs_backward", dict(lse=None), "lse is null"), ("token_logprobs_backward", dict(tokens=None), "need tokens"),
    ("token_logprobs_backward", dict(entropy=None), "needs entropy"),
    ("token_logprobs_backward", dict(dlogits=None), "dlogits is null"),
    ("token_logprobs_backward", dict(lddl=7), "dlogits: row stride 7"),
    ("token_logprobs_backward", dict(scale=-1.0), "scale"), ("token_logprobs_backward", dict(type=-1), "type -1"),
    ("q4_pack", dict(group=96), "group=96"), ("q4_pack", dict(group=0), "group=0"),
    ("q4_pack", dict(scale_type=3), "scales: type 3"), ("q4_pack", dict(packed_bytes=100), "are needed"),
    ("q4_pack", dict(packed=P + 16), "256-byte aligned"), ("q4_pack", dict(packed=None), "packed is null"),
    ("q4_pack", dict(q=None), "q is null"), ("q4_pack", dict(ldq=15), "q: row stride 15"),
    ("q4_pack", dict(K=256, group=32, lds=15, packed_bytes=1 << 30), "scales: row stride 15"),
    ("q4_pack", dict(zeros=P, K=256, ldq=16, ldz=15), "zeros: row stride 15"),
    ("q4_pack", dict(K=(1 << 23) + 1), "2^23"),
    ("q4_dense", dict(x_type=5), "X: unknown type 5"), ("q4_dense", dict(y_type=3), "Y: type 3"),
    ("q4_dense", dict(bias=None), "bias is null"), ("q4_dense", dict(bias_type=4), "bias: type 4"),
    ("q4_dense", dict(epilogue=8), "epilogue code 8"), ("q4_dense", dict(group=48), "group=48"),
    ("q4_dense", dict(ldx=100), "X: row stride 100"), ("q4_dense", dict(ldy=15), "Y: row stride 15"),
    ("q4_dense", dict(packed=None), "packed is null"), ("q4_dense", dict(packed=P + 128), "256-byte aligned"),
    ("q4_dense", dict(K=-1), "negative"), ("q4_dense", dict(N=MORE, ldy=MORE), "2^30"),
    ("q4_dense", dict(X=None), "X is null"),
]
EMPTY = [("rms_norm", dict(M=0)), ("rms_norm", dict(M=0, x=None, y=None)), ("rms_norm_backward", dict(M=0)),
         ("token_logprobs", dict(M=0)), ("token_logprobs", dict(logprobs=None, lse=None, entropy=None, k=0)),
         ("token_logprobs_backward", dict(M=0)), ("q4_pack", dict(N=0)), ("q4_pack", dict(K=0)),
         ("q4_dense", dict(M=0)), ("q4_dense", dict(N=0))]


def call(op, change):
    return getattr(_native.lib(), f"edsl_hip_{op}_launch")(*{**CALLS[op], **change}.values())


@pytest.mark.parametrize("op,change,text", REFUSED, ids=[f"{op}-{'-'.join(c)}-{i}" for i, (op, c, _) in enumerate(REFUSED)])
def test_refused(op, change, text):
    assert set(change) <= set(CALLS[op])
    assert call(op, change) != 0
    assert text in message()


@pytest.mark.parametrize("op,change", EMPTY)
def test_nothing_to_do(op, change):
    assert call(op, change) == 0
    assert last_plan() == "empty"


def test_packed_bytes():
    f = _native.lib().edsl_hip_q4_packed_bytes
    # 4 bits a weight, a scale and a zero point a group, and up to three paddings of 256 bytes.
    for K, N, group, scale_type, size, zeros in ((4096, 4096, 128, 0, 4, 1), (8192, 1024, 32, 1, 2, 0), (512, 32, 256, 2, 2, 1)):
        least = K * N // 2 + K // group * N * (size + zeros)
        assert least <= f(K, N, group, scale_type, zeros) <= least + 768
    assert f(0, 16, 128, 0, 0) == f(128, 0, 128, 0, 0) == 0
    assert f(1, 1, 32, 0, 0) >= 1024
    for args in ((128, 16, 100, 0, 0), (128, 16, 128, 3, 0), (-1, 16, 128, 0, 0), ((1 << 23) + 1, 16, 128, 0, 0)):
        assert f(*args) == -1 and message()
