"""Sequence operators of a frame classifier on channels-last CUDA (ROCm) tensors, the inference forms.

``group_norm``              normalisation over the frames and a group of channels, with an activation;
``causal_conv1d``           depthwise convolution over the current and a few earlier frames;
``selective_scan``          selective state space scan: a linear recurrence whose step size, input and output
                            vectors change from frame to frame;
``causal_conv1d_step``, ``selective_step``
                            one new frame of every stream, the state updated in place.

They stand beside the models' own stages (BatchNorm inside the conv blocks, GRU recurrences, attention) for frame
classifiers that normalise without batch statistics and that have to answer frame by frame; the reference has none of
them.  The arithmetic runs in the HIP kernels of csrc/norm.hip, csrc/conv1d.hip and csrc/scan.hip through the C ABI
(``sedmi_group_norm``, ``sedmi_causal_conv1d``, ``sedmi_selective_scan``, ``sedmi_selective_step``).  Inference only:
there is no backward and no CPU path.

Common to all: activations are float32, float16 or bfloat16, one type per call, and the results have that type;
parameters are taken as float32 (others are converted in the call), sums, statistics and the scan's states are
float32, each result is rounded once.  The channel dimension has to be adjacent in memory (a tensor where it is not is
copied), the other strides are free, so slices of a wider projection are read in place (``group_norm`` copies what is
not contiguous).  ``lengths`` gives the valid frames of each clip (an int tensor or a sequence, values outside
0 .. frames are taken as the nearer end): frames behind them are never read and come out as zeros.  An int64 tensor on
the device is used as it is; anything else is copied there first, which waits for the copy and cannot be captured into
a graph.  ``reverse=True`` runs from a clip's last valid frame to its first, the second direction of a bidirectional
layer.  Tensors that require a gradient (while gradients are recorded) or carry a tangent are refused.  Nothing is kept
between calls; all work goes to the current stream of the tensors' device, and apart from that copy nothing waits for it.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_ACTIVATIONS = {None: _lib.ACT_NONE, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
MAX_CONV_WIDTH = 8
MAX_STATES = 128


def _check_input(x, who):
    if not torch.is_tensor(x) or not x.is_cuda:
        raise _lib.SedmiError(f"{who} needs a CUDA (ROCm) tensor: it runs in HIP kernels only")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{who}: float32, float16 or bfloat16, not {x.dtype}")
    return _DTYPES[x.dtype]


def _refuse_grad(who, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{who} is inference-only: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:                 # within a dual_level, which no_grad() does not end
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{who} is inference-only: it has no forward derivative either, unpack the dual tensors")


def _activation(name, who):
    code = _ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"{who}: activation must be one of {sorted(a for a in _ACTIVATIONS if a)} or None, not {name!r}")
    return code


def _like(t, x, shape, what):
    """``t`` checked to be of x's type and device and of the given shape, its last dimension adjacent."""
    if t.dtype is not x.dtype or t.get_device() != x.get_device():
        raise TypeError(f"{what}: {x.dtype} on {x.device} like x, not {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _param(t, x, shape, what):
    """``t`` checked to be on x's device and of the given shape, as contiguous float32; None stays."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != x.get_device():
        raise TypeError(f"{what}: on {t.device}, x is on {x.device}")
    return t.to(torch.float32).contiguous() if t.dtype is not torch.float32 else t.contiguous()


def _lengths(lengths, n, device, who):
    if lengths is None:
        return None
    t = lengths if torch.is_tensor(lengths) else torch.as_tensor(lengths)
    if t.dtype is torch.int64 and t.is_cuda and t.shape == (n,) and t.device == device:
        return t.contiguous()
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{who}: lengths needs one entry per clip ({n}), got shape {tuple(t.shape)}")
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError(f"{who}: lengths must be whole numbers, not {t.dtype}")
    return t.to(device, torch.int64).contiguous()


def _call(device, entry, *args):
    """One entry point on the current stream of ``device``, with that device current.  ``args``: numbers, and addresses as
    ``_address`` gives them."""
    fn, index = getattr(_lib.lib(), entry), device.index
    # raw handles, as the tensors have initialised torch: with the public forms a call takes 0.4 us longer
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc < 0:
        _lib.check(rc, entry)


def _address(t):
    return 0 if t is None else t.data_ptr()


# ----------------------------------------------------------------------------------------------------------- group norm
def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation=None, lengths=None):
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` per clip and group of channels, channels last.

    x [clips, frames, ..., channels] (or [clips, channels]): mean and biased variance run over everything between
    the clip and the channels and over the ``channels / num_groups`` channels of a group.  ``num_groups=1`` is a
    normalisation over the whole clip.  ``activation``: None, "relu", "silu" or "gelu" (the erf form)."""
    dtype = _check_input(x, "group_norm")
    _refuse_grad("group_norm", x, weight, bias)
    if x.dim() < 2:
        raise ValueError(f"group_norm: expected [clips, frames, ..., channels], got {tuple(x.shape)}")
    if lengths is not None and x.dim() < 3:
        raise ValueError("group_norm: lengths need a frame dimension behind the clips")
    n, c, whole = x.shape[0], x.shape[-1], int(num_groups)
    if whole != num_groups or whole < 1 or c == 0 or c % whole:
        raise ValueError(f"group_norm: {c} channels do not divide into {num_groups} groups")
    num_groups = whole
    if not eps >= 0:
        raise ValueError("group_norm: eps must not be negative")
    act = _activation(activation, "group_norm")
    x = x.contiguous()
    frames = x.shape[1] if x.dim() > 2 else 1
    inner = 1
    for s in x.shape[2:-1]:
        inner *= s
    weight, bias = _param(weight, x, (c,), "weight"), _param(bias, x, (c,), "bias")
    lengths = _lengths(lengths, n, x.device, "group_norm")
    y = torch.empty_like(x)
    if x.numel() == 0:
        return y
    ws_bytes = _lib.lib().sedmi_group_norm_workspace_bytes(n, frames, inner, c, num_groups, dtype)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    _call(x.device, "sedmi_group_norm", x.data_ptr(), _address(weight), _address(bias), _address(lengths), y.data_ptr(), n,
          frames, inner, c, num_groups, float(eps), act, dtype, _address(ws), ws_bytes)
    return y


# --------------------------------------------------------------------------------------------------- causal convolution
def _conv_arguments(x, weight, bias, state, who):
    n, c = x.shape[0], x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != c or not 1 <= weight.shape[1] <= MAX_CONV_WIDTH:
        raise ValueError(f"{who}: expected weight [{c}, 1 .. {MAX_CONV_WIDTH}], got {tuple(weight.shape)}")
    k = weight.shape[1]
    return n, c, k, _param(weight, x, (c, k), "weight"), _param(bias, x, (c,), "bias")


def causal_conv1d(x, weight, bias=None, activation=None, state=None, lengths=None, reverse=False, return_state=False):
    """Depthwise convolution of x [clips, frames, channels] with ``weight`` [channels, width], width 1 .. 8:
    ``y[:, t] = act(bias + sum_k weight[:, k] * x[:, t - (width - 1) + k])``.

    ``state`` [clips, width - 1, channels] (the type of x) holds the inputs before the first frame, oldest first;
    zeros when None.  With ``return_state`` the result is ``(y, state)``, the new state being the last ``width - 1``
    valid inputs: what the next stretch of the same recordings, or ``causal_conv1d_step``, continues from."""
    dtype = _check_input(x, "causal_conv1d")
    _refuse_grad("causal_conv1d", x, weight, bias, state)
    if x.dim() != 3 or x.shape[2] == 0:
        raise ValueError(f"causal_conv1d: expected [clips, frames, channels], got {tuple(x.shape)}")
    n, c, k, weight, bias = _conv_arguments(x, weight, bias, state, "causal_conv1d")
    act = _activation(activation, "causal_conv1d")
    x = x if x.stride(2) == 1 or c == 1 else x.contiguous()
    if state is not None:
        state = _like(state, x, (n, k - 1, c), "state").contiguous()
    lengths = _lengths(lengths, n, x.device, "causal_conv1d")
    frames = x.shape[1]
    y = x.new_empty((n, frames, c))
    last = x.new_empty((n, k - 1, c)) if return_state else None
    if n and (frames or return_state):
        _call(x.device, "sedmi_causal_conv1d", x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), _address(bias),
              _address(lengths), _address(state), _address(last), y.data_ptr(), n, frames, c, k, act, bool(reverse), dtype)
    return (y, last) if return_state else y


def causal_conv1d_step(x, state, weight, bias=None, activation=None):
    """One new frame x [streams, channels] of every stream: the convolution's output [streams, channels], ``state``
    [streams, width - 1, channels] (the type of x, contiguous) moved on by this frame in place; x must not be part of it."""
    dtype = _check_input(x, "causal_conv1d_step")
    _refuse_grad("causal_conv1d_step", x, weight, bias, state)
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"causal_conv1d_step: expected [streams, channels], got {tuple(x.shape)}")
    n, c, k, weight, bias = _conv_arguments(x, weight, bias, state, "causal_conv1d_step")
    act = _activation(activation, "causal_conv1d_step")
    x = x if x.stride(1) == 1 or c == 1 else x.contiguous()
    _like(state, x, (n, k - 1, c), "state")
    if not state.is_contiguous():
        raise ValueError("causal_conv1d_step: the state is updated in place and has to be contiguous")
    y = x.new_empty((n, c))
    if n:
        at = state.data_ptr()
        _call(x.device, "sedmi_causal_conv1d", x.data_ptr(), x.stride(0), 0, weight.data_ptr(), _address(bias), 0, at, at,
              y.data_ptr(), n, 1, c, k, act, 0, dtype)
        torch._C._increment_version((state,))          # for graphs that saved it; the public form takes 0.5 us longer
    return y


# ------------------------------------------------------------------------------------------------------- selective scan
def _scan_arguments(x, dt, A, B, C, D, z, dt_bias, who):
    shape = x.shape
    c, lead = shape[-1], shape[:-1]
    if A.dim() != 2 or A.shape[0] != c or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"{who}: expected A [{c}, 1 .. {MAX_STATES}], got {tuple(A.shape)}")
    m = A.shape[1]
    x = x if x.stride(-1) == 1 or c == 1 else x.contiguous()
    dt = _like(dt, x, shape, "dt")
    z = None if z is None else _like(z, x, shape, "z")
    if B.dim() == len(shape):                      # [.., states] stands for one group
        B = B.unsqueeze(-2)
    if C.dim() == len(shape):
        C = C.unsqueeze(-2)
    groups = B.shape[-2] if B.dim() == len(shape) + 1 else 0
    if groups < 1 or c % groups:
        raise ValueError(f"{who}: {c} channels and B {tuple(B.shape)}: expected {tuple(lead)} + [groups, {m}] or + [{m}], the "
                         "groups dividing the channels")
    both = (*lead, groups, m)
    return (x, dt, z, _like(B, x, both, "B"), _like(C, x, both, "C"), _param(A, x, (c, m), "A"), _param(D, x, (c,), "D"),
            _param(dt_bias, x, (c,), "dt_bias"), c, groups, m)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, state=None, lengths=None,
                   reverse=False, return_state=False):
    """Selective state space scan of x [clips, frames, channels]:

        d = softplus(dt + dt_bias)              (dt + dt_bias without ``dt_softplus``)
        h = exp(d * A) * h + d * x * B          per channel and state
        y = (sum over states of C * h + D * x) * silu(z)

    dt, z like x; A [channels, states] (negative decay rates), states 1 .. 128; B, C [clips, frames, groups, states] or
    [clips, frames, states] for one group, group g serving channels g * channels / groups and on; D, dt_bias
    [channels].  ``state`` [clips, channels, states] float32 is h before the first frame, zeros when None.  With
    ``return_state`` the result is ``(y, state)``, h behind each clip's last valid frame."""
    dtype = _check_input(x, "selective_scan")
    _refuse_grad("selective_scan", x, dt, A, B, C, D, z, dt_bias, state)
    if x.dim() != 3 or x.shape[2] == 0:
        raise ValueError(f"selective_scan: expected [clips, frames, channels], got {tuple(x.shape)}")
    x, dt, z, B, C, A, D, dt_bias, c, groups, m = _scan_arguments(x, dt, A, B, C, D, z, dt_bias, "selective_scan")
    n, frames = x.shape[0], x.shape[1]
    if state is not None:
        if state.dtype != torch.float32:
            raise TypeError(f"selective_scan: the state is float32, not {state.dtype}")
        state = _param(state, x, (n, c, m), "state")
    lengths = _lengths(lengths, n, x.device, "selective_scan")
    y = x.new_empty((n, frames, c))
    last = x.new_empty((n, c, m), dtype=torch.float32) if return_state else None
    if not n or not (frames or return_state):
        return (y, last) if return_state else y
    args = _lib.pack_scan_args(x.data_ptr(), dt.data_ptr(), _address(z), B.data_ptr(), C.data_ptr(), A.data_ptr(),
                               _address(D), _address(dt_bias), _address(lengths), _address(state), _address(last),
                               y.data_ptr(), *x.stride()[:2], *dt.stride()[:2], *((0, 0) if z is None else z.stride()[:2]),
                               *B.stride()[:3], *C.stride()[:3], n, frames, c, groups, m, dtype, bool(dt_softplus),
                               bool(reverse))
    ws_bytes = _lib.lib().sedmi_selective_scan_workspace_bytes(n, frames, c, groups, m)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    _call(x.device, "sedmi_selective_scan", args, _address(ws), ws_bytes)
    return (y, last) if return_state else y


def selective_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=False):
    """One new frame x [streams, channels] of every stream through ``selective_scan``'s formulas: y [streams,
    channels]; ``state`` [streams, channels, states] (float32, contiguous) is updated in place.  B, C [streams,
    groups, states] or [streams, states]."""
    dtype = _check_input(x, "selective_step")
    _refuse_grad("selective_step", x, dt, A, B, C, D, z, dt_bias, state)
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"selective_step: expected [streams, channels], got {tuple(x.shape)}")
    x, dt, z, B, C, A, D, dt_bias, c, groups, m = _scan_arguments(x, dt, A, B, C, D, z, dt_bias, "selective_step")
    n = x.shape[0]
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("selective_step: the state is updated in place and has to be float32 and contiguous")
    _param(state, x, (n, c, m), "state")
    y = x.new_empty((n, c))
    if n:
        at = state.data_ptr()
        b0, b1, _ = B.stride()
        c0, c1, _ = C.stride()
        args = _lib.pack_scan_args(x.data_ptr(), dt.data_ptr(), _address(z), B.data_ptr(), C.data_ptr(), A.data_ptr(),
                                   _address(D), _address(dt_bias), 0, at, at, y.data_ptr(), x.stride(0), 0, dt.stride(0), 0,
                                   0 if z is None else z.stride(0), 0, b0, 0, b1, c0, 0, c1, n, 1, c, groups, m, dtype,
                                   bool(dt_softplus), 0)
        _call(x.device, "sedmi_selective_step", args)
        torch._C._increment_version((state,))
    return y
