"""What the entries for the 8-bit layer, the layer on groups of rows and sampling refuse,
and their calls with nothing to do: decided on the host before any device is looked at, so
checked without one."""
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
    "i8_pack": dict(q=P, ldq=16, scales=P, scale_type=0, K=128, N=16, packed=P, packed_bytes=1 << 20, stream=None),
    "i8_dense": dict(X=P, ldx=128, x_scales=P, packed=P, bias=P, bias_type=0, Y=P, ldy=16, y_type=0, M=4, N=16, K=128,
                     epilogue=1, alpha=0.0, stream=None),
    "grouped_dense": dict(X=P, ldx=8, W=P, ldw=4, w_stride=32, w_turned=0, offsets=P, ids64=0, E=2, bias=P, ldbias=4, Y=P,
                          ldy=4, T=6, N=4, K=8, type=0, epilogue=1, alpha=0.0, stream=None),
    "grouped_dense_backward": dict(dY=P, lddy=4, X=P, ldx=8, W=P, ldw=4, w_stride=32, w_turned=0, offsets=P, ids64=0,
                                   E=2, Y=P, ldy=4, dX=P, lddx=8, dW=P, lddw=4, dw_stride=32, dw_turned=0, dw_type=0,
                                   db=P, lddb=4, db_type=0, T=6, N=4, K=8, type=0, epilogue=3, alpha=0.0, stream=None),
    "sample_tokens": dict(logits=P, ldl=8, type=0, uniforms=P, tokens=P, ids64=1, logprobs=P, temperature=None,
                          temperature_all=1.0, top_k=None, top_k_all=0, top_p=None, top_p_all=1.0, min_p=None,
                          min_p_all=0.0, M=4, V=8, stream=None),
}
MORE = (1 << 30) + 1
NAN = float("nan")
REFUSED = [
    ("i8_pack", dict(K=0), "K=0"), ("i8_pack", dict(K=1 << 17), "2^17"), ("i8_pack", dict(N=-1), "negative"),
    ("i8_pack", dict(scale_type=3), "scales: type 3"), ("i8_pack", dict(packed_bytes=2048), "are needed"),
    ("i8_pack", dict(packed=P + 16), "256-byte aligned"), ("i8_pack", dict(packed=None), "packed is null"),
    ("i8_pack", dict(q=None), "q is null"), ("i8_pack", dict(ldq=15), "q: row stride 15"),
    ("i8_pack", dict(scales=None), "scales is null"),
    ("i8_dense", dict(K=0), "K=0"), ("i8_dense", dict(K=1 << 17, ldx=1 << 17), "2^17"),
    ("i8_dense", dict(M=-1), "negative"), ("i8_dense", dict(M=MORE), "2^30"), ("i8_dense", dict(y_type=3), "Y: type 3"),
    ("i8_dense", dict(bias=None), "bias is null"), ("i8_dense", dict(bias_type=3), "bias: type 3"),
    ("i8_dense", dict(epilogue=8), "epilogue code 8"), ("i8_dense", dict(epilogue=-1), "epilogue code -1"),
    ("i8_dense", dict(ldx=100), "X: row stride 100"), ("i8_dense", dict(ldy=15), "Y: row stride 15"),
    ("i8_dense", dict(X=None), "X is null"), ("i8_dense", dict(Y=None), "Y is null"),
    ("i8_dense", dict(packed=None), "packed is null"), ("i8_dense", dict(packed=P + 64), "256-byte aligned"),
    ("grouped_dense", dict(E=-1), "negative"), ("grouped_dense", dict(E=65536), "65536 groups"),
    ("grouped_dense", dict(T=-1), "T=-1"), ("grouped_dense", dict(T=MORE), "2^30"),
    ("grouped_dense", dict(N=MORE, ldw=MORE, ldy=MORE, ldbias=MORE), "2^30"),
    ("grouped_dense", dict(offsets=None), "offsets is null"), ("grouped_dense", dict(type=3), "X: type 3"),
    ("grouped_dense", dict(epilogue=8), "epilogue code 8"), ("grouped_dense", dict(bias=None), "bias is null"),
    ("grouped_dense", dict(ldbias=3), "bias: row stride 3"), ("grouped_dense", dict(X=None), "X is null"),
    ("grouped_dense", dict(ldx=7), "X: row stride 7"), ("grouped_dense", dict(W=None), "W is null"),
    ("grouped_dense", dict(ldw=3), "W: row stride 3"), ("grouped_dense", dict(w_turned=1, ldw=7), "W: row stride 7"),
    ("grouped_dense", dict(w_stride=-32), "negative stride"), ("grouped_dense", dict(ldy=3), "Y: row stride 3"),
    ("grouped_dense", dict(Y=None), "Y is null"),
    ("grouped_dense_backward", dict(type=4), "dY: type 4"), ("grouped_dense_backward", dict(E=-2), "negative"),
    ("grouped_dense_backward", dict(dY=None), "dY is null"), ("grouped_dense_backward", dict(lddy=3), "dY: row stride 3"),
    ("grouped_dense_backward", dict(Y=None), "needs Y"), ("grouped_dense_backward", dict(ldy=3), "Y: row stride 3"),
    ("grouped_dense_backward", dict(epilogue=5, alpha=-0.1), "alpha >= 0"),
    ("grouped_dense_backward", dict(epilogue=4, alpha=NAN), "alpha >= 0"),
    ("grouped_dense_backward", dict(dw_type=1), "dW: type 1"), ("grouped_dense_backward", dict(db_type=2), "db: type 2"),
    ("grouped_dense_backward", dict(X=None), "X is null"), ("grouped_dense_backward", dict(W=None), "W is null"),
    ("grouped_dense_backward", dict(lddx=7), "dX: row stride 7"), ("grouped_dense_backward", dict(lddw=3), "dW: row stride 3"),
    ("grouped_dense_backward", dict(dw_turned=1), "dW: row stride 4"),
    ("grouped_dense_backward", dict(dw_stride=-1), "dW: negative stride"),
    ("grouped_dense_backward", dict(lddb=3), "db: row stride 3"), ("grouped_dense_backward", dict(offsets=None), "offsets"),
    ("sample_tokens", dict(type=3), "logits: type 3"), ("sample_tokens", dict(V=0), "no logits"),
    ("sample_tokens", dict(V=(1 << 21) + 1, ldl=1 << 22), "2^21"), ("sample_tokens", dict(M=-1), "negative"),
    ("sample_tokens", dict(logits=None), "logits is null"), ("sample_tokens", dict(ldl=7), "row stride 7"),
    ("sample_tokens", dict(uniforms=None), "uniforms is null"), ("sample_tokens", dict(tokens=None), "tokens is null"),
    ("sample_tokens", dict(temperature_all=-1.0), "temperature"), ("sample_tokens", dict(temperature_all=NAN), "temperature"),
    ("sample_tokens", dict(temperature_all=float("inf")), "temperature"), ("sample_tokens", dict(top_p_all=NAN), "top_p"),
    ("sample_tokens", dict(min_p_all=NAN), "min_p"),
]
EMPTY = [("i8_pack", dict(N=0)), ("i8_dense", dict(M=0)), ("i8_dense", dict(N=0)), ("grouped_dense", dict(T=0)),
         ("grouped_dense", dict(E=0, offsets=None)), ("grouped_dense", dict(N=0)),
         ("grouped_dense_backward", dict(E=0)), ("grouped_dense_backward", dict(dX=None, dW=None, db=None)),
         ("sample_tokens", dict(M=0))]


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
    f = _native.lib().edsl_hip_i8_packed_bytes
    assert f(4096, 4096) == 4096 * 4096 + 4 * 4096
    assert f(1, 1) == 2048 + 64 and f(128, 0) == 0
    for args in ((0, 16), (1 << 17, 16), (-1, 16), (16, -1)):
        assert f(*args) == -1 and message()
