"""Sequence layers on channels-last tensors, computed on the MI355X by libmelvoc: what an acoustic or vocoder model built
beside this package's convolutions needs and the reference's models do not hold.

    y = group_norm(x, groups, weight, bias, activation="silu", lengths=n)           # normalisation + activation
    y = causal_conv(x, weight, bias, activation="silu", state=s, state_out=s)       # short depthwise causal convolution
    y = selective_scan(u, delta, A, B, C, D=D, z=z, state=h, state_out=h)           # state space recurrence

Data are `[B, T, channels]` float32, bfloat16 or float16 with adjacent channels and any other strides (halves of a
projection's output, `[T, B, C]` memory: taken as they lie, rows at most 2^25 elements apart; a tensor whose channels are not
adjacent is copied first).  A
tensor without the frame axis, `[B, channels]`, is one frame of each sequence: a decode step.  Arithmetic is float32 and is
rounded once, at the result.

`lengths=` (host or device, as in the vocoders) holds the true frame counts of a right-padded batch: row b is the call on
`x[b, :lengths[b]]` (to float32 rounding: how sums are cut goes by the size of the call), whatever the padding holds, and its
frames past the end are written as 0.  Host-side lengths outside `[0, T]` raise, lengths already on the device are clamped
there.

`state=` is where a sequence stands before the call (None: at its beginning), `state_out=` a tensor that receives where it
stands after its last true frame; they may be the same tensor (but share memory with no other argument), so a sequence cut
into calls (prompt, then frame by frame) gives the results of one call: the convolution bit for bit, the scan to float32
rounding.  Calls can be captured into HIP graphs, with `lengths` on the device (host-side ones are refused there); a decode
step on static tensors with its state replaced in place is one kernel.

These are synthesis-time layers: inputs that require a gradient are refused (outside `no_grad`), and so are those with a
forward-mode tangent.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _native

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # MV_DTYPE_*
_ACTIVATIONS = {None: 0, "silu": 1, "leaky_relu": 2, "relu": 2, "tanh": 3}  # MV_ACT_*
MAX_TAPS, MAX_STATES = 8, 64


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, slope=0.1, per_frame=False, lengths=None):
    """act((x - mean) / sqrt(var + eps) * weight + bias) over `groups` groups of adjacent channels.

    x             [B, T, C] or [B, C] (a frame each)
    weight, bias  [C] (float32 or x's type) or None
    per_frame     False: mean and (biased) variance over a sequence's true frames and a group's channels, as
                  `torch.nn.GroupNorm` on `[B, C, T]` without padding; True: over a frame's group alone, which does not look
                  ahead and is the same in a whole call as frame by frame
    activation    None, "silu", "relu", "leaky_relu" (with `slope`) or "tanh"
    """
    x, shape, B, T, ch, sb, st, dtype, dev = _data("group_norm", "x", x)
    if groups < 1 or ch % groups:
        raise RuntimeError(f"group_norm: {ch} channels do not split into {groups} groups")
    if not 0.0 <= eps < _INF:
        raise RuntimeError("group_norm: eps must be finite and not negative")
    act, slope = _activation("group_norm", activation, slope)
    wtype, wp, bp = 0, 0, 0
    if weight is not None or bias is not None:
        weight, bias = _one_type(weight, bias)
        if weight is not None:
            weight, wtype, wp = _weight("group_norm", "weight", weight, (ch,), dtype, dev)
        if bias is not None:
            bias, wtype, bp = _weight("group_norm", "bias", bias, (ch,), dtype, dev)
    if _grad() or _forward_ad._current_level >= 0:
        _no_grad("group_norm", x, weight, bias)
    y = _like(x, memory_format=_DENSE)
    if B and T:
        if lengths is not None:
            lengths = _lengths(lengths, B, T, x)
        _call(_native.GROUP_NORM, x, dev, T > 1, _native.GROUP_NORM.pack(
            x.data_ptr(), sb, st, y.data_ptr(), T * ch, ch, wp, bp, 0 if lengths is None else lengths.data_ptr(), B, T, ch,
            groups, _DTYPES[dtype], wtype, 1 if per_frame else 0, act, slope, eps))
    return y


def causal_conv(x, weight, bias=None, activation=None, slope=0.1, state=None, state_out=None, lengths=None):
    """act(bias + sum_k weight[:, k] * x[t - K + 1 + k]): each channel convolved by itself with its own K taps, looking
    back only.

    x          [B, T, C] or [B, C] (a frame each)
    weight     [C, K] or [C, 1, K] (a depthwise `torch.nn.Conv1d`'s), 1 <= K <= 8, float32 or x's type; bias [C] or None
    state      [B, K - 1, C] of x's type, the frames before the first, oldest first (None: zeros); state_out likewise
    """
    x, shape, B, T, ch, sb, st, dtype, dev = _data("causal_conv", "x", x)
    w = weight.shape
    K = w[-1] if len(w) > 1 else 0
    if not (w == (ch, K) or w == (ch, 1, K)) or not 1 <= K <= MAX_TAPS:
        raise RuntimeError(f"causal_conv: expected a weight [{ch}, K] with 1 <= K <= {MAX_TAPS}, got {tuple(w)}")
    act, slope = _activation("causal_conv", activation, slope)
    weight, bias = _one_type(weight, bias)
    weight, wtype, wp = _weight("causal_conv", "weight", weight, w, dtype, dev)
    bp = sp = op = 0
    if bias is not None:
        bias, wtype, bp = _weight("causal_conv", "bias", bias, (ch,), dtype, dev)
    if state is not None:
        sp = _state("causal_conv", "state", state, (B, K - 1, ch), dtype, dev)
    if state_out is state:
        op = sp
    elif state_out is not None:
        op = _state("causal_conv", "state_out", state_out, (B, K - 1, ch), dtype, dev)
    if _grad() or _forward_ad._current_level >= 0:
        _no_grad("causal_conv", x, weight, bias, state, state_out)
    y = _like(x, memory_format=_DENSE)
    if B and (T or state_out is not None):
        if lengths is not None:
            lengths = _lengths(lengths, B, T, x)
        _call(_native.CAUSAL_CONV, x, dev, False, _native.CAUSAL_CONV.pack(
            x.data_ptr(), sb, st, y.data_ptr(), T * ch, ch, wp, bp, sp, op, 0 if lengths is None else lengths.data_ptr(), B, T,
            ch, K, _DTYPES[dtype], wtype, act, slope))
    return y


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, state=None, state_out=None,
                   lengths=None):
    """The state space recurrence of D channels with N states each, per frame:

        dt = delta + delta_bias  (softplus of it with `delta_softplus`)
        h  = exp(dt * A) * h + dt * u * B          [D, N]
        y  = (sum_n C * h + D * u) * silu(z)       [D]

    u, delta, z   [B, T, D] or [B, D] (a frame each); z None: no gate
    A             [D, N], 1 <= N <= 64 (decays: A < 0); D, delta_bias [D] or None.  Held in float32
    B, C          [B, T, N], or [B, T, G, N] with D / G adjacent channels to a group ([B, N], [B, G, N] for a frame)
    state         [B, D, N] float32 (None: zeros); state_out likewise
    u, delta, z, B, C share one type.
    """
    u, shape, nb, T, ch, sb, st, dtype, dev = _data("selective_scan", "u", u)
    a, m = A.shape, B.shape
    N = a[1] if len(a) == 2 else 0
    if not 1 <= N <= MAX_STATES or a[0] != ch:
        raise RuntimeError(f"selective_scan: expected A [{ch}, N] with 1 <= N <= {MAX_STATES}, got {tuple(a)}")
    axes = len(shape)
    G = m[-2] if len(m) == axes + 1 else 1
    if C.shape != m or len(m) - axes not in (0, 1) or m[-1] != N or m[0] != nb or (axes == 3 and m[1] != T):
        raise RuntimeError(f"selective_scan: B and C must be {list(shape[:-1])} + [{N}] or [G, {N}], got {tuple(m)} and "
                           f"{tuple(C.shape)}")
    if G < 1 or ch % G:
        raise RuntimeError(f"selective_scan: {ch} channels do not split into {G} groups")
    delta, sd = _rows("delta", delta, shape, dtype, dev)
    B, sB = _rows("B", B, m, dtype, dev)
    C, sC = _rows("C", C, m, dtype, dev)
    zp, sz = 0, _NO_STRIDES
    if z is not None:
        z, sz = _rows("z", z, shape, dtype, dev)
        zp = z.data_ptr()
    Dp = bp = sp = op = 0
    A = _float32("A", A, a, dev)
    if D is not None:
        D = _float32("D", D, (ch,), dev)
        Dp = D.data_ptr()
    if delta_bias is not None:
        delta_bias = _float32("delta_bias", delta_bias, (ch,), dev)
        bp = delta_bias.data_ptr()
    if state is not None:
        sp = _state("selective_scan", "state", state, (nb, ch, N), torch.float32, dev)
    if state_out is state:
        op = sp
    elif state_out is not None:
        op = _state("selective_scan", "state_out", state_out, (nb, ch, N), torch.float32, dev)
    if _grad() or _forward_ad._current_level >= 0:
        _no_grad("selective_scan", u, delta, z, B, C, A, D, delta_bias, state, state_out)
    y = _like(u, memory_format=_DENSE)
    if nb and (T or state_out is not None):
        if lengths is not None:
            lengths = _lengths(lengths, nb, T, u)
        # a row's stride is the second one; of a single row it says nothing
        td, tz, tB, tC = (sd[1], sz[1], sB[1], sC[1]) if T > 1 else (0, 0, 0, 0)
        gB, gC = (sB[-2], sC[-2]) if G > 1 else (0, 0)
        _call(_native.SELECTIVE_SCAN, u, dev, T > 1, _native.SELECTIVE_SCAN.pack(
            u.data_ptr(), sb, st, delta.data_ptr(), sd[0], td, zp, sz[0], tz, B.data_ptr(), sB[0], tB, C.data_ptr(), sC[0], tC,
            gB, gC, y.data_ptr(), T * ch, ch, A.data_ptr(), Dp, bp, sp, op,
            0 if lengths is None else lengths.data_ptr(), nb, T, ch, N, G, _DTYPES[dtype], 1 if delta_softplus else 0))
    return y


# --- arguments.  A decode step's call is short against what Python adds to it: checks are plain comparisons, messages are made
# --- where one fails.
_INF, _NO_STRIDES, _DENSE = float("inf"), (0, 0, 0), torch.contiguous_format
_empty, _like, _grad = torch.empty, torch.empty_like, torch.is_grad_enabled


def _data(who, name, x):
    """-> (x with adjacent channels, its shape, B, T, channels, batch stride, row stride, type, device index)"""
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    if dev < 0:
        raise RuntimeError(f"tacotron2_amd.sequence.{who} computes on an MI355X only (no CPU fallback)")
    if dtype not in _DTYPES:
        raise RuntimeError(f"{who}: {name} must be float32, bfloat16 or float16, got {dtype}")
    s = x.stride()
    if len(shape) not in (2, 3) or shape[-1] < 1:
        raise RuntimeError(f"{who}: {name} must be [B, T, channels] or [B, channels], got {tuple(shape)}")
    if s[-1] != 1 and shape[-1] != 1:
        x = x.contiguous()
        s = x.stride()
    if len(shape) == 3:
        T = shape[1]
        return x, shape, shape[0], T, shape[2], s[0], s[1] if T > 1 else 0, dtype, dev  # (of one row the stride says nothing)
    return x, shape, shape[0], 1, shape[1], s[0], 0, dtype, dev


def _rows(name, t, shape, dtype, dev):
    """-> (t with adjacent channels, its strides)"""
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev:
        raise RuntimeError(f"selective_scan: {name} must be {list(shape)}, {dtype}, on the device of u; got {list(t.shape)}, "
                           f"{t.dtype}, on {t.device}")
    s = t.stride()
    if s[-1] != 1 and shape[-1] != 1:
        t = t.contiguous()
        s = t.stride()
    return t, s


def _activation(who, activation, slope):
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{who}: unknown activation {activation!r} (one of {sorted(a for a in _ACTIVATIONS if a)}, None)")
    return act, 0.0 if activation == "relu" else slope


def _one_type(weight, bias):
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        return weight.float(), bias.float()
    return weight, bias


def _weight(who, name, t, shape, dtype, dev):
    """-> (t contiguous, its MV_DTYPE_*, its address)"""
    if t.shape != shape or t.get_device() != dev or not (t.dtype == torch.float32 or t.dtype == dtype):
        raise RuntimeError(f"{who}: {name} must be {list(shape)}, float32 or {dtype}, on the device of x; got {list(t.shape)}, "
                           f"{t.dtype}, on {t.device}")
    if not t.is_contiguous():
        t = t.contiguous()
    return t, _DTYPES[t.dtype], t.data_ptr()


def _float32(name, t, shape, dev):
    if t.shape != shape or t.get_device() != dev or t.dtype not in _DTYPES:
        raise RuntimeError(f"selective_scan: {name} must be {list(shape)} floats on the device of u, got {list(t.shape)}, "
                           f"{t.dtype}, on {t.device}")
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _state(who, name, t, shape, dtype, dev):
    """-> its address"""
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev or not t.is_contiguous():
        raise RuntimeError(f"{who}: {name} must be contiguous {list(shape)}, {dtype}, on the device of the data; got "
                           f"{list(t.shape)}, {t.dtype}, on {t.device}")
    return t.data_ptr()


def _no_grad(who, *tensors):
    reverse, forward = _grad(), _forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()
    for t in tensors:
        if t is not None and (reverse and t.requires_grad or forward and _forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError(f"tacotron2_amd.sequence.{who} has no gradient: call it under torch.no_grad(), without "
                               "forward-mode tangents")


def _lengths(lengths, B, T, x):
    if not isinstance(lengths, torch.Tensor):
        lengths = torch.as_tensor(lengths)
    if lengths.numel() != B:
        raise RuntimeError("lengths must hold B frame counts in [0, T]")
    if lengths.dtype == torch.int32 and lengths.get_device() == x.get_device() and lengths.is_contiguous():
        return lengths
    if lengths.is_floating_point() or lengths.is_complex():
        raise RuntimeError("lengths must be whole numbers")
    return _native.device_lengths(lengths, B, T, x.device)


def _call(op, x, dev, scratch, args):
    """One call of the library on x's device and its current stream.  Scratch (which calls of one frame do without) comes from
    torch's allocator, in a capture from the graph's own pool: a new piece for every call, so that no two calls or graphs
    share one."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _call(op, x, dev, scratch, args)
    if op.fn is None:
        op.bind()
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if not op.scratch:
        rc = op.fn(args, stream)
    else:
        n = op.fn_workspace(args) if scratch else 0
        ws = _empty(n, dtype=torch.uint8, device=x.device) if n else None
        rc = op.fn(args, 0 if ws is None else ws.data_ptr(), n, stream)
    if rc:
        _native.check(rc, op.name)
