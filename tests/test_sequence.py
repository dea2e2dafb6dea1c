"""The sequence operators' C entry points refuse what they cannot compute before anything reaches a device: every call here
carries made-up pointers and must come back with an error code and a message."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

from tacotron2_amd import _native, sequence  # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists(_native.LIB_PATH), reason="libmelvoc.so is not built")
P = 1 << 20  # a made-up, well aligned device address


def _norm(**k):
    a = _native.mv_group_norm_args(P, 320, 32, 2 * P, 320, 32, P, P, None, 2, 10, 32, 4, 0, 0, 0, 1, 0.1, 1e-5)
    for f, v in k.items():
        setattr(a, f, v)
    return _native.lib().mv_group_norm(ctypes.byref(a), None, 0, None)


def _conv(**k):
    a = _native.mv_causal_conv_args(P, 320, 32, 2 * P, 320, 32, P, P, 3 * P, 3 * P, None, 2, 10, 32, 4, 0, 0, 1, 0.1)
    for f, v in k.items():
        setattr(a, f, v)
    return _native.lib().mv_causal_conv(ctypes.byref(a), None)


def _scan(**k):
    a = _native.mv_selective_scan_args(P, 320, 32, P, 320, 32, None, 0, 0, P, 160, 16, P, 160, 16, 0, 0, 2 * P, 320, 32, P, P,
                                       P, 3 * P, 3 * P, None, 2, 10, 32, 16, 1, 0, 1)
    for f, v in k.items():
        setattr(a, f, v)
    return _native.lib().mv_selective_scan(ctypes.byref(a), None, 0, None)


BAD = [
    (_norm, dict(groups=0), b"groups"), (_norm, dict(groups=5), b"groups"), (_norm, dict(B=-1), b"sizes"),
    (_norm, dict(T=-1), b"sizes"), (_norm, dict(C=0), b"sizes"), (_norm, dict(dtype=3), b"dtype"),
    (_norm, dict(weight_dtype=1), b"weight_dtype"), (_norm, dict(activation=4), b"activation"),
    (_norm, dict(eps=-1e-5), b"eps"), (_norm, dict(eps=float("nan")), b"eps"), (_norm, dict(eps=float("inf")), b"eps"),
    (_norm, dict(x=None), b"x needs"), (_norm, dict(y=None), b"output needs"), (_norm, dict(x=P + 2), b"x needs"),
    (_norm, dict(x_row_stride=-32), b"strides"), (_norm, dict(y_row_stride=31), b"overlap"),
    (_norm, dict(y_batch_stride=319), b"overlap"), (_norm, dict(y_batch_stride=31, y_row_stride=64), b"overlap"),
    (_conv, dict(K=0), b"taps"), (_conv, dict(K=9), b"taps"), (_conv, dict(weight=None), b"weight"),
    (_conv, dict(weight_dtype=2), b"weight"), (_conv, dict(activation=-1), b"activation"), (_conv, dict(dtype=-1), b"dtype"),
    (_conv, dict(state_out=3 * P + 64), b"overlap"), (_conv, dict(state_out=3 * P - 64), b"overlap"),
    (_conv, dict(x=None), b"x needs"), (_conv, dict(y=P + 1), b"output needs"), (_conv, dict(y_row_stride=16), b"overlap"),
    (_scan, dict(N=0), b"states"), (_scan, dict(N=65), b"states"), (_scan, dict(G=0), b"groups"), (_scan, dict(G=3), b"groups"),
    (_scan, dict(A=None), b"needs A"), (_scan, dict(u=None), b"u needs"), (_scan, dict(delta=None), b"delta needs"),
    (_scan, dict(Bm=None), b"Bm needs"), (_scan, dict(Cm=None), b"Cm needs"), (_scan, dict(z=P + 2), b"z needs"),
    (_scan, dict(y=None), b"output needs"), (_scan, dict(y_batch_stride=0), b"overlap"),
    (_scan, dict(state_out=3 * P + 4), b"overlap"), (_scan, dict(dtype=7), b"dtype"), (_scan, dict(D=0), b"sizes"),
    (_scan, dict(B=-2), b"sizes"), (_scan, dict(Bg_stride=-16), b"strides"), (_scan, dict(Cg_stride=-1), b"strides"),
    (_scan, dict(A=P + 2), b"aligned"), (_scan, dict(state_in=P + 1, state_out=None), b"aligned"),
    (_scan, dict(lengths=P + 2), b"aligned"), (_conv, dict(weight=P + 2), b"aligned"), (_conv, dict(bias=P + 3), b"aligned"),
    (_norm, dict(weight=P + 2), b"aligned"), (_norm, dict(lengths=P + 1), b"aligned"),
    (_norm, dict(T=2 ** 30 + 1), b"sizes"), (_norm, dict(x_row_stride=2 ** 25 + 1), b"row stride"),
    (_conv, dict(C=2 ** 27 + 1, K=1), b"channels"), (_scan, dict(D=2 ** 22 + 1), b"channels"),
    (_scan, dict(B=2 ** 20, D=2 ** 10), b"2^29"),
]


@pytest.mark.parametrize("call,fields,message", BAD, ids=lambda v: v if isinstance(v, str) else None)
def test_bad_arguments_are_refused_before_a_launch(call, fields, message):
    assert call(**fields) == -1
    assert message in _native.lib().mv_last_error(), _native.lib().mv_last_error()


def test_null_arguments_and_empty_calls():
    lib = _native.lib()
    assert lib.mv_group_norm(None, None, 0, None) == -1
    assert lib.mv_causal_conv(None, None) == -1
    assert lib.mv_selective_scan(None, None, 0, None) == -1
    assert lib.mv_group_norm_workspace(None) == 0 and lib.mv_selective_scan_workspace(None) == 0
    # nothing to do: no pointer is looked at, nothing is launched
    assert _norm(B=0, x=None, y=None) == 0 and _norm(T=0, x=None, y=None) == 0
    assert _conv(B=0, x=None, y=None) == 0 and _conv(T=0, x=None, y=None) == 0  # (the state stays where it is)
    assert _scan(B=0, u=None, A=None, y=None) == 0 and _scan(T=0, u=None, y=None) == 0


def test_there_is_no_cpu_path():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(RuntimeError, match="MI355X only"):
        sequence.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="MI355X only"):
        sequence.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="MI355X only"):
        sequence.selective_scan(x, x, torch.zeros(8, 4), torch.zeros(2, 5, 4), torch.zeros(2, 5, 4))


def test_single_frames_never_need_scratch():
    """What the header promises and the Python layer relies on, up to batches that no grid of whole tiles holds."""
    lib = _native.lib()
    for dtype, C, G in ((1, 8, 1), (0, 4, 2), (2, 1, 1), (1, 1024, 1024), (0, 1024, 8), (1, 4096, 1), (0, 20000, 4), (1, 1 << 20, 2)):
        for B in (1, 3, 1 << 12, 1 << 16, 1 << 20, 1 << 21, 1 << 25, 1 << 28):
            for per_frame in (0, 1):
                for far in (C, 1 << 40):  # (of a single row its stride says nothing)
                    a = _native.mv_group_norm_args(P, C, far, 2 * P, C, far, None, None, None, B, 1, C, G, dtype, 0, per_frame,
                                                   0, 0.0, 1e-5)
                    assert lib.mv_group_norm_workspace(ctypes.byref(a)) == 0, (dtype, C, G, B, per_frame, far)
    for D, N in ((64, 16), (1024, 64)):
        for B in (1, 1 << 12, 1 << 19):
            a = _native.mv_selective_scan_args(P, D, D, P, D, D, None, 0, 0, P, N, N, P, N, N, 0, 0, 2 * P, D, D, P, None, None,
                                               None, None, None, B, 1, D, N, 1, 1, 1)
            assert lib.mv_selective_scan_workspace(ctypes.byref(a)) == 0


OVERLAPS = [
    # in place with other strides; shifted by channels, by a frame, by a sequence; rows inside the other's rows
    (_norm, dict(y=P, y_row_stride=64, y_batch_stride=640)), (_norm, dict(y=P, y_batch_stride=384)),
    (_norm, dict(y=P + 16)), (_norm, dict(y=P + 128)), (_norm, dict(y=P + 1280)), (_norm, dict(y=P - 2 * 1280 + 4)),
    (_norm, dict(y=P + 124, x_row_stride=64, x_batch_stride=640, y_row_stride=64, y_batch_stride=640)),
    (_norm, dict(y=P + 4 * 64 * 9 + 4, x_row_stride=64, x_batch_stride=640, y_row_stride=64, y_batch_stride=640)),
    (_norm, dict(y=P + 4, x_row_stride=64, x_batch_stride=32, y_row_stride=64, y_batch_stride=32)),  # [T][B][C]
    (_norm, dict(y=P + 256, x_row_stride=64, x_batch_stride=640)),  # strides differ, y one piece
    (_norm, dict(y=P + 4, x_row_stride=0, x_batch_stride=0)), (_norm, dict(weight=2 * P + 64)), (_norm, dict(bias=2 * P + 2556)),
    (_norm, dict(lengths=2 * P + 1280)),
    (_conv, dict(y=P)), (_conv, dict(y=P + 128)), (_conv, dict(y=P - 64)), (_conv, dict(y=3 * P)), (_conv, dict(y=3 * P - 4)),
    (_conv, dict(state_in=None, state_out=P + 128)), (_conv, dict(state_in=None, state_out=2 * P + 2556)),
    (_conv, dict(state_in=None, state_out=P - 2 * 384 + 4)), (_conv, dict(weight=2 * P)), (_conv, dict(bias=3 * P)),
    (_conv, dict(state_in=None, state_out=P + 128 + 4, x_row_stride=64, x_batch_stride=640, B=1)),
    (_scan, dict(y=P)), (_scan, dict(y=P + 8, z=2 * P, z_batch_stride=320, z_row_stride=32)), (_scan, dict(y=3 * P)),
    (_scan, dict(y=P + 64, Bm=5 * P, Cm=P + 128)), (_scan, dict(Bm=2 * P + 2556)), (_scan, dict(Cm=2 * P, Cm_row_stride=0)),
    (_scan, dict(G=2, N=16, Bg_stride=2 ** 18, Bm=P)),  # only the second group of B lies in y
    (_scan, dict(A=2 * P)), (_scan, dict(Dskip=2 * P + 128)), (_scan, dict(delta_bias=3 * P)), (_scan, dict(A=3 * P + 4092)),
    (_scan, dict(state_in=None, state_out=P)), (_scan, dict(state_in=None, state_out=2 * P - 4)), (_scan, dict(delta=3 * P + 64)),
]


@pytest.mark.parametrize("call,fields", OVERLAPS)
def test_outputs_over_inputs_are_refused(call, fields):
    assert call(**fields) == -1
    assert b"overlap" in _native.lib().mv_last_error(), _native.lib().mv_last_error()


def test_outputs_beside_inputs_are_not():
    """Rows that lie between the other's rows get past the checks: what then stops these calls is that they bring no scratch."""
    T = 100000
    for x, y, b, r in ((P, P + 128, 64 * T, 64), (P + 128, P, 64 * T, 64), (P, P + 128, 64, 128), (P, P + 4 * 64 * T, 32 * T, 32),
                       (P, P, 32 * T, 32)):  # halves of rows, also of [T][B] memory; one behind the other; in place
        rows = dict(x=x, x_batch_stride=b, x_row_stride=r, y=y, y_batch_stride=b, y_row_stride=r, weight=None, bias=None)
        assert _norm(T=T, **rows) == -4, _native.lib().mv_last_error()
    T = 5000
    far = P + 8 * 160 * T  # behind both sequences' rows
    scan = dict(T=T, delta=far, delta_batch_stride=32 * T, A=2 * far, Dskip=None, delta_bias=None, state_in=3 * far, state_out=3 * far)
    # u, B, C and y side by side in rows of 160: the groups of B and C 32 apart, y between them
    side = dict(u=P, u_batch_stride=160 * T, u_row_stride=160, G=2, N=16, Bm=P + 4 * 32, Bm_batch_stride=160 * T, Bm_row_stride=160,
                Bg_stride=64, Cm=P + 4 * 48, Cm_batch_stride=160 * T, Cm_row_stride=160, Cg_stride=64, y_batch_stride=160 * T,
                y_row_stride=160)
    for y in (64, 128):
        assert _scan(**scan, **side, y=P + 4 * y) == -4, _native.lib().mv_last_error()
    for y in (1, 33, 65, 80, 127):
        assert _scan(**scan, **side, y=P + 4 * y) == -1 and b"overlap" in _native.lib().mv_last_error()
