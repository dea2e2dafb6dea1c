"""Sequence layers on channels-last tensors, computed on the MI355X by libmelvoc: what an acoustic or vocoder model built
beside this package's convolutions needs and the reference's models do not hold.

    y = group_norm(x, groups, weight, bias, activation="silu", lengths=n)           # normalisation + activation
    y = causal_conv(x, weight, bias, activation="silu", state=s, state_out=s)       # short depthwise causal convolution
    y = selective_scan(u, delta, A, B, C, D=D, z=z, state=h, state_out=h)           # state space recurrence

Data are `[B, T, channels]` float32, bfloat16 or float16 with adjacent channels and any other strides (halves of a
projection's output, `[T, B, C]` memory: taken as they lie; a tensor whose channels are not adjacent is copied first).  A
tensor without the frame axis, `[B, channels]`, is one frame of each sequence: a decode step.  Arithmetic is float32 and is
rounded once, at the result.

`lengths=` (host or device, as in the vocoders) holds the true frame counts of a right-padded batch: row b equals the call
on `x[b, :lengths[b]]`, whatever the padding holds, and its frames past the end are written as 0.  Host-side lengths outside
`[0, T]` raise, lengths already on the device are clamped there.

`state=` is where a sequence stands before the call (None: at its beginning), `state_out=` a tensor that receives where it
stands after its last true frame; they may be the same tensor, so a sequence cut into calls (prompt, then frame by frame)
gives the results of one call.  With `state_out` given and no allocation of the caller's in between, a call can be captured
into a HIP graph.  These are synthesis-time layers: inputs that require a gradient are refused (outside `no_grad`).
"""
from __future__ import annotations

import torch

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
    x, shape, B, T, ch, sb, st = _data("group_norm", "x", x)
    if groups < 1 or ch % groups:
        raise RuntimeError(f"group_norm: {ch} channels do not split into {groups} groups")
    if not 0.0 <= eps < float("inf"):
        raise RuntimeError("group_norm: eps must be finite and not negative")
    act, slope = _activation("group_norm", activation, slope)
    weight, bias, wtype = _weights("group_norm", x, weight, (ch,), bias, ch)
    if torch.is_grad_enabled():
        _no_grad("group_norm", x, weight, bias)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    if B and T:
        lengths = _lengths(lengths, B, T, x)
        _call(_native.GROUP_NORM, x, T > 1, _native.GROUP_NORM.pack(
            x.data_ptr(), sb, st, y.data_ptr(), T * ch, ch, _ptr(weight), _ptr(bias), _ptr(lengths), B, T, ch, groups,
            _DTYPES[x.dtype], wtype, 1 if per_frame else 0, act, slope, eps))
    return y


def causal_conv(x, weight, bias=None, activation=None, slope=0.1, state=None, state_out=None, lengths=None):
    """act(bias + sum_k weight[:, k] * x[t - K + 1 + k]): each channel convolved by itself with its own K taps, looking
    back only.

    x          [B, T, C] or [B, C] (a frame each)
    weight     [C, K] or [C, 1, K] (a depthwise `torch.nn.Conv1d`'s), 1 <= K <= 8, float32 or x's type; bias [C] or None
    state      [B, K - 1, C] of x's type, the frames before the first, oldest first (None: zeros); state_out likewise
    """
    x, shape, B, T, ch, sb, st = _data("causal_conv", "x", x)
    w = weight.shape
    K = w[-1] if len(w) > 1 else 0
    if not (w == (ch, K) or w == (ch, 1, K)) or not 1 <= K <= MAX_TAPS:
        raise RuntimeError(f"causal_conv: expected a weight [{ch}, K] with 1 <= K <= {MAX_TAPS}, got {tuple(w)}")
    act, slope = _activation("causal_conv", activation, slope)
    weight, bias, wtype = _weights("causal_conv", x, weight, w, bias, ch)
    _states("causal_conv", x, state, state_out, (B, K - 1, ch), x.dtype)
    if torch.is_grad_enabled():
        _no_grad("causal_conv", x, weight, bias, state, state_out)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    if B and (T or state_out is not None):
        lengths = _lengths(lengths, B, T, x)
        _call(_native.CAUSAL_CONV, x, False, _native.CAUSAL_CONV.pack(
            x.data_ptr(), sb, st, y.data_ptr(), T * ch, ch, weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(state_out),
            _ptr(lengths), B, T, ch, K, _DTYPES[x.dtype], wtype, act, slope))
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
    u, shape, nb, T, ch, sb, st = _data("selective_scan", "u", u)
    for name, t in (("delta", delta), ("z", z)):
        if t is not None and t.shape != shape:
            raise RuntimeError(f"selective_scan: {name} has shape {tuple(t.shape)}, u {tuple(shape)}")
    a = A.shape
    if len(a) != 2 or a[0] != ch or not 1 <= a[1] <= MAX_STATES:
        raise RuntimeError(f"selective_scan: expected A [{ch}, N] with 1 <= N <= {MAX_STATES}, got {tuple(a)}")
    N = a[1]
    lead, m = shape[:-1], B.shape
    G = m[-2] if len(m) == len(shape) + 1 else 1
    if C.shape != m or not (m == (*lead, N) or m == (*lead, G, N)):
        raise RuntimeError(f"selective_scan: B and C must be {list(lead)} + [{N}] or [G, {N}], got {tuple(m)} and "
                           f"{tuple(C.shape)}")
    if G < 1 or ch % G:
        raise RuntimeError(f"selective_scan: {ch} channels do not split into {G} groups")
    dev = u.get_device()
    for name, t in (("delta", delta), ("z", z), ("B", B), ("C", C)):
        if t is not None and (t.dtype != u.dtype or t.get_device() != dev):
            raise RuntimeError(f"selective_scan: {name} must be {u.dtype} on {u.device} like u, got {t.dtype} on {t.device}")
    A = _float32("selective_scan", u, "A", A, (ch, N))
    D = _float32("selective_scan", u, "D", D, (ch,))
    delta_bias = _float32("selective_scan", u, "delta_bias", delta_bias, (ch,))
    _states("selective_scan", u, state, state_out, (nb, ch, N), torch.float32)
    if torch.is_grad_enabled():
        _no_grad("selective_scan", u, delta, z, B, C, A, D, delta_bias, state, state_out)
    y = torch.empty(shape, dtype=u.dtype, device=u.device)
    if nb and (T or state_out is not None):
        lengths = _lengths(lengths, nb, T, u)
        delta, sd = _adjacent(delta)
        z, sz = _adjacent(z) if z is not None else (None, (0, 0, 0))
        B, sB = _adjacent(B)
        C, sC = _adjacent(C)
        f = len(shape) == 3  # with a frame axis
        _call(_native.SELECTIVE_SCAN, u, T > 1, _native.SELECTIVE_SCAN.pack(
            u.data_ptr(), sb, st, delta.data_ptr(), sd[0], sd[1] if f else 0, _ptr(z), sz[0], sz[1] if f else 0,
            B.data_ptr(), sB[0], sB[1] if f else 0, C.data_ptr(), sC[0], sC[1] if f else 0, sB[-2] if G > 1 else 0,
            sC[-2] if G > 1 else 0, y.data_ptr(), T * ch, ch, A.data_ptr(), _ptr(D), _ptr(delta_bias), _ptr(state),
            _ptr(state_out), _ptr(lengths), nb, T, ch, N, G, _DTYPES[u.dtype], 1 if delta_softplus else 0))
    return y


# --- arguments (checks are plain comparisons: a decode step's call is short against what Python adds to it) -----------
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _adjacent(t):
    """-> (t with channels side by side, its strides)"""
    s = t.stride()
    if s[-1] == 1 or t.shape[-1] == 1:
        return t, s
    t = t.contiguous()
    return t, t.stride()


def _data(who, name, x):
    """-> (x with adjacent channels, its shape, B, T, channels, batch and row stride)"""
    shape = x.shape
    if len(shape) not in (2, 3) or shape[-1] < 1:
        raise RuntimeError(f"{who}: {name} must be [B, T, channels] or [B, channels], got {tuple(shape)}")
    if not x.is_cuda:
        raise RuntimeError(f"tacotron2_amd.sequence.{who} computes on an MI355X only (no CPU fallback)")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"{who}: {name} must be float32, bfloat16 or float16, got {x.dtype}")
    x, s = _adjacent(x)
    if len(shape) == 3:
        return x, shape, shape[0], shape[1], shape[2], s[0], s[1]
    return x, shape, shape[0], 1, shape[1], s[0], 0


def _activation(who, activation, slope):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{who}: unknown activation {activation!r} (one of {sorted(a for a in _ACTIVATIONS if a)}, None)")
    return _ACTIVATIONS[activation], 0.0 if activation == "relu" else float(slope)


def _weights(who, x, weight, shape, bias, ch):
    """-> (weight, bias, MV_DTYPE_* of both): contiguous, of one type, float32 or x's."""
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        weight, bias = weight.float(), bias.float()
    wtype = 0
    for name, t, want in (("weight", weight, shape), ("bias", bias, (ch,))):
        if t is not None:
            if t.shape != want or t.get_device() != x.get_device() or not (t.dtype == torch.float32 or t.dtype == x.dtype):
                raise RuntimeError(f"{who}: {name} must be {list(want)}, float32 or {x.dtype}, on {x.device}; got "
                                   f"{list(t.shape)}, {t.dtype}, on {t.device}")
            wtype = _DTYPES[t.dtype]
    return (weight if weight is None else weight.contiguous()), (bias if bias is None else bias.contiguous()), wtype


def _float32(who, x, name, t, shape):
    if t is None:
        return None
    if t.shape != shape or t.get_device() != x.get_device() or t.dtype not in _DTYPES:
        raise RuntimeError(f"{who}: {name} must be {list(shape)} floats on {x.device}, got {list(t.shape)}, {t.dtype}, on "
                           f"{t.device}")
    return t.contiguous() if t.dtype == torch.float32 else t.float().contiguous()


def _states(who, x, state, state_out, shape, dtype):
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None and (t.shape != shape or t.dtype != dtype or t.get_device() != x.get_device()
                              or not t.is_contiguous()):
            raise RuntimeError(f"{who}: {name} must be contiguous {list(shape)}, {dtype}, on {x.device}; got "
                               f"{list(t.shape)}, {t.dtype}, on {t.device}")


def _no_grad(who, *tensors):
    for t in tensors:
        if t is not None and t.requires_grad:
            raise RuntimeError(f"tacotron2_amd.sequence.{who} has no gradient: call it under torch.no_grad()")


def _lengths(lengths, B, T, x):
    if lengths is None:
        return None
    if isinstance(lengths, torch.Tensor) and lengths.is_cuda:
        if lengths.numel() != B or lengths.is_floating_point():
            raise RuntimeError("lengths must hold B frame counts in [0, T]")
        if lengths.dtype != torch.int32:
            lengths = lengths.clamp(0, T)  # (a 64-bit count must not wrap around in 32)
        elif lengths.get_device() == x.get_device() and lengths.is_contiguous():
            return lengths
    return _native.device_lengths(lengths, B, T, x.device)


def _call(op, x, scratch, args):
    """One call of the library on x's device and its current stream.  Scratch (which calls of one frame do without) comes from
    torch's allocator, in a capture from the graph's own pool: a new piece for every call, so that no two calls or graphs
    share one."""
    dev = x.get_device()
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _call(op, x, scratch, args)
    if op.fn is None:
        op.bind()
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if not op.scratch:
        rc = op.fn(args, stream)
    else:
        n = op.fn_workspace(args) if scratch else 0
        ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        rc = op.fn(args, _ptr(ws), n, stream)
    if rc:
        _native.check(rc, op.name)
