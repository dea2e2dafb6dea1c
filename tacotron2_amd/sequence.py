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

import ctypes

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
    x, B, T, ch, squeeze = _data("group_norm", "x", x)
    if groups < 1 or ch % groups:
        raise RuntimeError(f"group_norm: {ch} channels do not split into {groups} groups")
    if not 0.0 <= eps < float("inf"):
        raise RuntimeError("group_norm: eps must be finite and not negative")
    act, slope = _activation("group_norm", activation, slope)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        weight, bias = weight.float(), bias.float()
    weight, bias = _weights("group_norm", x, (("weight", weight, (ch,)), ("bias", bias, (ch,))))
    _no_grad("group_norm", x, weight, bias)
    y = x.new_empty((B, T, ch))
    if y.numel() == 0:
        return y
    lengths = _lengths(lengths, B, T, x)
    sx = x.stride()
    w = weight if weight is not None else bias
    a = _native.mv_group_norm_args(
        x.data_ptr(), sx[0], sx[-2] if not squeeze else 0, y.data_ptr(), T * ch, ch,
        weight.data_ptr() if weight is not None else None, bias.data_ptr() if bias is not None else None,
        lengths.data_ptr() if lengths is not None else None, B, T, ch, groups, _DTYPES[x.dtype],
        _DTYPES[w.dtype] if w is not None else 0, 1 if per_frame else 0, act, slope, eps)
    _call("mv_group_norm", a, x, True)
    return y[:, 0] if squeeze else y


def causal_conv(x, weight, bias=None, activation=None, slope=0.1, state=None, state_out=None, lengths=None):
    """act(bias + sum_k weight[:, k] * x[t - K + 1 + k]): each channel convolved by itself with its own K taps, looking
    back only.

    x          [B, T, C] or [B, C] (a frame each)
    weight     [C, K] or [C, 1, K] (a depthwise `torch.nn.Conv1d`'s), 1 <= K <= 8, float32 or x's type; bias [C] or None
    state      [B, K - 1, C] of x's type, the frames before the first, oldest first (None: zeros); state_out likewise
    """
    x, B, T, ch, squeeze = _data("causal_conv", "x", x)
    if weight.dim() == 3 and weight.size(1) == 1:
        weight = weight[:, 0]
    if weight.dim() != 2 or weight.size(0) != ch or not 1 <= weight.size(1) <= MAX_TAPS:
        raise RuntimeError(f"causal_conv: expected a weight [{ch}, K] with 1 <= K <= {MAX_TAPS}, got {tuple(weight.shape)}")
    K = weight.size(1)
    act, slope = _activation("causal_conv", activation, slope)
    if bias is not None and weight.dtype != bias.dtype:
        weight, bias = weight.float(), bias.float()
    weight, bias = _weights("causal_conv", x, (("weight", weight, (ch, K)), ("bias", bias, (ch,))))
    state, state_out = _states("causal_conv", x, state, state_out, (B, K - 1, ch), x.dtype)
    _no_grad("causal_conv", x, weight, bias, state, state_out)
    y = x.new_empty((B, T, ch))
    if B and (T or state_out is not None):
        lengths = _lengths(lengths, B, T, x)
        sx = x.stride()
        a = _native.mv_causal_conv_args(
            x.data_ptr(), sx[0], sx[-2] if not squeeze else 0, y.data_ptr(), T * ch, ch, weight.data_ptr(),
            bias.data_ptr() if bias is not None else None, state.data_ptr() if state is not None else None,
            state_out.data_ptr() if state_out is not None else None, lengths.data_ptr() if lengths is not None else None,
            B, T, ch, K, _DTYPES[x.dtype], _DTYPES[weight.dtype], act, slope)
        _call("mv_causal_conv", a, x, False)
    return y[:, 0] if squeeze else y


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
    u, nb, T, ch, squeeze = _data("selective_scan", "u", u)
    for name, t in (("delta", delta), ("z", z)):
        if t is not None and t.shape != u.shape:
            raise RuntimeError(f"selective_scan: {name} has shape {tuple(t.shape)}, u {tuple(u.shape)}")
    if A.dim() != 2 or A.size(0) != ch or not 1 <= A.size(1) <= MAX_STATES:
        raise RuntimeError(f"selective_scan: expected A [{ch}, N] with 1 <= N <= {MAX_STATES}, got {tuple(A.shape)}")
    N = A.size(1)
    lead = u.dim() - 1
    G = B.size(-2) if B.dim() == lead + 2 else 1
    for name, t in (("B", B), ("C", C)):
        if (t.shape[:lead] != u.shape[:lead] or t.size(-1) != N or t.dim() not in (lead + 1, lead + 2)
                or (t.size(-2) if t.dim() == lead + 2 else 1) != G):
            raise RuntimeError(f"selective_scan: {name} must be {list(u.shape[:lead])} + [{N}] or [G, {N}], B and C alike, got "
                               f"{tuple(t.shape)}")
    if G < 1 or ch % G:
        raise RuntimeError(f"selective_scan: {ch} channels do not split into {G} groups")
    for name, t in (("delta", delta), ("z", z), ("B", B), ("C", C)):
        if t is not None and (t.dtype != u.dtype or t.get_device() != u.get_device()):
            raise RuntimeError(f"selective_scan: {name} must be {u.dtype} on {u.device} like u, got {t.dtype} on {t.device}")
    delta, B, C, z = _adjacent(delta), _adjacent(B), _adjacent(C), _adjacent(z) if z is not None else None
    A, D, delta_bias = (_float32("selective_scan", u, n, t, s)
                        for n, t, s in (("A", A, (ch, N)), ("D", D, (ch,)), ("delta_bias", delta_bias, (ch,))))
    state, state_out = _states("selective_scan", u, state, state_out, (nb, ch, N), torch.float32)
    _no_grad("selective_scan", u, delta, z, B, C, A, D, delta_bias, state, state_out)
    y = u.new_empty((nb, T, ch))
    if nb and (T or state_out is not None):
        lengths = _lengths(lengths, nb, T, u)

        def rows(t):
            s = t.stride()
            return t.data_ptr(), s[0], 0 if squeeze else s[1]

        p = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        a = _native.mv_selective_scan_args(
            *rows(u), *rows(delta), *(rows(z) if z is not None else (None, 0, 0)), *rows(B), *rows(C),
            B.stride(-2) if G > 1 else 0, C.stride(-2) if G > 1 else 0, y.data_ptr(), T * ch, ch, A.data_ptr(), p(D),
            p(delta_bias), p(state), p(state_out), p(lengths), nb, T, ch, N, G, _DTYPES[u.dtype], 1 if delta_softplus else 0)
        _call("mv_selective_scan", a, u, True)
    return y[:, 0] if squeeze else y


# --- arguments -----------------------------------------------------------------------------------------------------
def _adjacent(t):
    """Channels side by side, other strides as they are."""
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _data(who, name, x):
    """-> (x with adjacent channels, B, T, channels, whether the frame axis is absent)"""
    if x.dim() not in (2, 3) or x.size(-1) < 1:
        raise RuntimeError(f"{who}: {name} must be [B, T, channels] or [B, channels], got {tuple(x.shape)}")
    if not x.is_cuda:
        raise RuntimeError(f"tacotron2_amd.sequence.{who} computes on an MI355X only (no CPU fallback)")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"{who}: {name} must be float32, bfloat16 or float16, got {x.dtype}")
    x = _adjacent(x)
    s = x.shape
    return (x, s[0], s[1], s[2], False) if len(s) == 3 else (x, s[0], 1, s[1], True)


def _activation(who, activation, slope):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{who}: unknown activation {activation!r} (one of {sorted(a for a in _ACTIVATIONS if a)}, None)")
    return _ACTIVATIONS[activation], 0.0 if activation == "relu" else float(slope)


def _weights(who, x, named):
    """Contiguous weights of one type: float32 or x's."""
    out = []
    for name, t, shape in named:
        if t is not None:
            if tuple(t.shape) != shape or t.get_device() != x.get_device() or t.dtype not in (torch.float32, x.dtype):
                raise RuntimeError(f"{who}: {name} must be {list(shape)}, float32 or {x.dtype}, on {x.device}; got "
                                   f"{list(t.shape)}, {t.dtype}, on {t.device}")
            t = t.contiguous()
        out.append(t)
    return out


def _float32(who, x, name, t, shape):
    if t is None:
        return None
    if tuple(t.shape) != shape or t.get_device() != x.get_device() or t.dtype not in _DTYPES:
        raise RuntimeError(f"{who}: {name} must be {list(shape)} floats on {x.device}, got {list(t.shape)}, {t.dtype}, on "
                           f"{t.device}")
    return t.float().contiguous()


def _states(who, x, state, state_out, shape, dtype):
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None and (tuple(t.shape) != shape or t.dtype != dtype or t.get_device() != x.get_device()
                              or not t.is_contiguous()):
            raise RuntimeError(f"{who}: {name} must be contiguous {list(shape)}, {dtype}, on {x.device}; got "
                               f"{list(t.shape)}, {t.dtype}, on {t.device}")
    return state, state_out


def _no_grad(who, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
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


def _call(name, args, x, scratch):
    """One call of the library on x's device and its current stream; scratch comes from torch's allocator (in a capture:
    from the graph's own pool), a new piece for every call, so that no two calls or graphs share one."""
    lib, dev = _native.lib(), x.get_device()
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _call(name, args, x, scratch)
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if scratch:
        n = getattr(lib, name + "_workspace")(ctypes.byref(args))
        ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        rc = getattr(lib, name)(ctypes.byref(args), ws.data_ptr() if n else None, n, stream)
    else:
        rc = getattr(lib, name)(ctypes.byref(args), stream)
    if rc:
        _native.check(rc, name)
