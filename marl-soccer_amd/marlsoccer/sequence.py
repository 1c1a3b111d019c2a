"""Sequence memory on the GPU: the short causal convolution and the selective state-space scan a
recurrent policy is built of (csrc/ms_conv.hip, csrc/ms_scan.hip; the C entry points and the formulas
are in include/marl_soccer.h).

Sequences are time-major, (T, R, D), as DeviceRollout stores them: T steps of R rows (one for every
agent of every env) of D channels. Any step and row strides will do while the channels lie next to
each other, so a batch-first tensor goes in as x.transpose(0, 1), uncopied. `starts` (T, R), bool or
uint8, says which rows begin a new episode at which step: nothing before it, the given state
included, reaches that step or a later one, and no gradient crosses it. Rows are independent.

    y, conv_state = short_conv(x, weight, bias, state=conv_state, starts=starts, return_state=True)
    y, state = ssm_scan(y, delta, A, B, C, D=D, z=z, delta_bias=b, state=state, starts=starts, return_state=True)

and for one step, with the states renewed in place:

    y = short_conv_step(x, conv_state, weight, bias, starts=starts)
    y = ssm_step(state, y, delta, A, B, C, D=D, z=z, delta_bias=b, starts=starts)

Everything that varies in time has one type (float32, bfloat16 or float16); weights, A, D, biases and
the scan's states are float32. Results are rounded once, and repeat bit for bit (no atomics). The
sequence forms carry gradients to every input but `starts` (once: no double backward); forward-mode
derivatives are refused (NotImplementedError), by the steps too. Calls are
asynchronous on the current stream of the tensors' device and may be captured into a HIP graph; a
captured backward needs its forward in the same capture, and leaves (the inputs', or those they were
computed from) that no eager autograd graph of these operators holds any more.
"""
from __future__ import annotations

import struct
import threading
import weakref

import torch
from torch.autograd import forward_ad

from . import _native as N

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_STATES = 64


# ms_conv_io and ms_scan_io (include/marl_soccer.h), packed in one go: a step's latency is the host's
_CONV_HEAD, _CONV_TAIL = "<4i3q" + "Qqq" + "QQQ" + "Qqq" + "Qqq" + "Q", "Qqq" + "Q" + "Qqq" + "QQQ" + "Qq"
_CONV = struct.Struct(_CONV_HEAD + _CONV_TAIL)
_SCAN_HEAD, _SCAN_TAIL = "<4i3q" + "Qqq" * 3 + "Qqqq" * 2 + "QQQQ" + "Qqq" * 2 + "Q", "Q" + "Qqq" + "Q" + "Qqq" * 3 + "Q" * 7 + "q"
_SCAN = struct.Struct(_SCAN_HEAD + _SCAN_TAIL)
_POINTER, _WORKSPACE, _KEEP_AT = struct.Struct("<Q"), struct.Struct("<Qq"), struct.calcsize("<" + _SCAN_HEAD.lstrip("<"))
assert _CONV.size == N.C.sizeof(N.MsConvIO) and _SCAN.size == N.C.sizeof(N.MsScanIO)
_NONE3 = (0, 0, 0)
# a step's: the head alone, and zeros from dout (ms_conv_io) or checkpoints (ms_scan_io) on
_CONV_STEP, _CONV_ZEROS = struct.Struct(_CONV_HEAD), bytes(struct.calcsize("<" + _CONV_TAIL))
_SCAN_STEP, _SCAN_ZEROS = struct.Struct(_SCAN_HEAD), bytes(struct.calcsize("<" + _SCAN_TAIL))


def _fail(rc: int) -> None:
    raise (ValueError if rc == N.MS_ERR_INVALID_ARGUMENT else N.NativeError)(
        N.lib().ms_sequence_last_error().decode(errors="replace"))


def _call(fn, io, index) -> None:
    rc = N.on_current_stream(index, fn, io)
    if rc:
        _fail(rc)


def _renewed(t):
    """t was written behind autograd's back: a graph that saved it refuses its backward."""
    if not t.is_inference():  # those carry no version, and no graph saves them
        torch.autograd.graph.increment_version(t)


# the autograd nodes of eager forwards that some graph still holds
_living, _living_lock = weakref.WeakSet(), threading.Lock()


def _leaves(nodes):
    """The leaves whose gradient accumulators lie behind these autograd nodes (their ids)."""
    found, seen, todo = set(), set(), list(nodes)
    while todo:
        node = todo.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        leaf = getattr(node, "variable", None)
        if isinstance(leaf, torch.Tensor):
            found.add(id(leaf))
        todo.extend(f for f, _ in node.next_functions)
    return found


def _refuse_held(*inputs):
    """Refuses a forward under graph capture whose leaves, or those its inputs were computed from, an
    eager graph still holds: their gradient accumulators belong to that graph's stream, and the captured
    backward would have to wait for it, at which torch ends the process."""
    here = torch.cuda.current_stream().cuda_stream
    with _living_lock:
        others = [node for node in _living if node.stream != here]
    if not others:
        return
    grad = [t for t in inputs if t is not None and t.requires_grad]
    mine = {id(t) for t in grad if t.is_leaf} | _leaves(t.grad_fn for t in grad if not t.is_leaf)
    if mine & _leaves(others):
        raise RuntimeError("a graph capture needs leaves that no eager autograd graph holds: drop the outputs and losses "
                           "of earlier forward passes before capturing")


def _lives(ctx, stream=None):
    """A forward's node, noted with its stream (None: the current one) for as long as a graph holds it."""
    ctx.stream = torch.cuda.current_stream().cuda_stream if stream is None else stream
    with _living_lock:
        _living.add(ctx)


def _refuse_tangents(who, *inputs):
    """A dual tensor has no requires_grad: without this its tangent would be lost silently."""
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in inputs):
        raise NotImplementedError(f"{who}: forward-mode derivatives are not implemented")


def _with_workspace(io, work):
    """The packed arguments with their last two, the workspace and its size, filled in."""
    return io[:-_WORKSPACE.size] + _WORKSPACE.pack(work.data_ptr(), work.numel())


def _p(t):
    return 0 if t is None else t.data_ptr()


def _p3(t):
    """Pointer, step stride, row stride of (T, R, ...)."""
    return _NONE3 if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


def _g4(t):
    """The same with the group's stride, of (T, R, [G,] N)."""
    return (t.data_ptr(), t.stride(0), t.stride(1), t.stride(2) if t.dim() == 4 else 0)


def _row3(t):
    """Pointer, no step stride, row stride of (R, ...)."""
    return _NONE3 if t is None else (t.data_ptr(), 0, t.stride(0))


def _check(who, name, t, shape, dtype, device, rows_contiguous=False):
    """A tensor argument: its type, shape and device, and channels next to each other."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{who}: {name} must be a tensor, got {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{who}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{who}: {name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{who}: {name} must be on {device}, got {t.device}")
    if rows_contiguous:
        if not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be contiguous")
    elif t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{who}: {name}'s last dimension must be contiguous (stride 1)")


def _right(t, shape, dtype, index):
    """Whether a time-dependent argument is right as it stands, without saying what is wrong."""
    return t.shape == shape and t.dtype is dtype and t.get_device() == index and t.stride(-1) == 1


def _right_weight(t, shape, index):
    return t is None or (t.shape == shape and t.dtype is torch.float32 and t.get_device() == index and t.is_contiguous())


def _right_starts(t, shape, index):
    return t is None or (t.shape == shape and (t.dtype is torch.bool or t.dtype is torch.uint8) and t.get_device() == index)


def _check_starts(who, starts, shape, device):
    if starts is None:
        return
    if not isinstance(starts, torch.Tensor) or starts.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"{who}: starts must be a bool or uint8 tensor")
    if starts.shape != shape or starts.device != device:
        raise ValueError(f"{who}: starts must have shape {tuple(shape)} and be on {device}, got {tuple(starts.shape)} on {starts.device}")


def _sequence(who, name, x, dims):
    if not isinstance(x, torch.Tensor) or x.dim() != dims:
        raise ValueError(f"{who}: {name} must be a tensor of {dims} dimensions")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{who}: {name} must be float32, bfloat16 or float16, got {x.dtype}")
    if x.shape[-1] < 1:
        raise ValueError(f"{who}: {name} has no channels")


def _on_gpu(who, device):
    if device.type != "cuda":
        raise ValueError(f"{who}: tensors must be on a HIP device, got {device}")


def _like(x):
    """An output beside x: the same order of steps and rows, packed."""
    T, R, D = x.shape
    if R > 1 and T > 1 and x.stride(1) > x.stride(0):
        return torch.empty((R, T, D), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((T, R, D), dtype=x.dtype, device=x.device)


def _rows(t):
    """A gradient as the kernels read it: channels next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


# ---------------------------------------------------------------- short convolution

def _conv_io(x, weight, bias, state, starts, silu, out=None, new=None, dout=None, dnew=None, dx=None, dstate=None,
             dweight=None, dbias=None):
    T, R, D = x.shape
    return _CONV.pack(_DTYPES[x.dtype], weight.shape[1], silu, 0, T, R, D, *_p3(x), weight.data_ptr(), _p(bias), _p(state),
                      *_p3(starts), *_p3(out), _p(new), *_p3(dout), _p(dnew), *_p3(dx), _p(dstate), _p(dweight), _p(dbias),
                      0, 0)


def _conv_right(x, weight, bias, state, starts, activation, dims):
    """Everything that _conv_check looks for, in one go."""
    try:
        shape, i = x.shape, x.get_device()
        D, W = shape[-1], weight.shape[1]
        return (i >= 0 and len(shape) == dims and x.dtype in _DTYPES and D > 0 and x.stride(-1) == 1 and 2 <= W <= 4
                and (activation is None or activation == "silu") and _right_weight(weight, (D, W), i) and _right_weight(bias, (D,), i)
                and (state is None or (_right(state, (shape[-2], W - 1, D), x.dtype, i) and state.is_contiguous()))
                and _right_starts(starts, shape[:-1], i))
    except (AttributeError, IndexError):
        return False


def _conv_check(who, x, weight, bias, state, starts, activation, dims):
    if _conv_right(x, weight, bias, state, starts, activation, dims):
        return
    _sequence(who, "x", x, dims)
    device, D = x.device, x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"{who}: weight must be a (channels, width) tensor of width 2, 3 or 4")
    if activation not in (None, "silu"):
        raise ValueError(f"{who}: activation must be None or 'silu', got {activation!r}")
    R = x.shape[-2]
    _check(who, "x", x, x.shape, x.dtype, device)
    _check(who, "weight", weight, (D, weight.shape[1]), torch.float32, device, True)
    if bias is not None:
        _check(who, "bias", bias, (D,), torch.float32, device, True)
    if state is not None:
        _check(who, "state", state, (R, weight.shape[1] - 1, D), x.dtype, device, True)
    _check_starts(who, starts, x.shape[:-1], device)
    _on_gpu(who, device)


def _conv_forward(x, weight, bias, state, starts, silu, want_state):
    out = _like(x)
    new = torch.empty((x.shape[1], weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device) if want_state else None
    _call(N.lib().ms_conv_forward, _conv_io(x, weight, bias, state, starts, silu, out, new), x.get_device())
    return out, new


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, starts, silu, want_state):
        out, new = _conv_forward(x, weight, bias, state, starts, silu, want_state)
        ctx.save_for_backward(x, weight, bias, state, starts)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        _lives(ctx, N.current_raw_stream(x.get_device()))
        return out, new

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dnew):
        x, weight, bias, state, starts = ctx.saved_tensors
        if dout is None and dnew is None:
            return (None,) * 7
        need = ctx.needs_input_grad
        dout = torch.zeros_like(x) if dout is None else _rows(dout)
        dx = _like(x)
        dweight = torch.empty_like(weight) if need[1] else None
        dbias = torch.empty_like(bias) if bias is not None and need[2] else None
        dstate = torch.empty_like(state) if state is not None and need[3] else None
        dnew = None if dnew is None else dnew.contiguous()
        L = N.lib()
        io = _conv_io(x, weight, bias, state, starts, ctx.silu, None, None, dout, dnew, dx, dstate, dweight, dbias)
        work = torch.empty((L.ms_conv_workspace(io),), dtype=torch.uint8, device=x.device)
        _call(L.ms_conv_backward, _with_workspace(io, work), x.get_device())
        return dx if need[0] else None, dweight, dbias, dstate, None, None, None


def short_conv(x, weight, bias=None, state=None, starts=None, activation=None, return_state=False):
    """Causal convolution along time with a kernel of 2 to 4 steps per channel:
    y[t] = act(bias + sum_k weight[:, k] x[t - W + 1 + k]).

    x (T, R, D); weight (D, W), bias (D) float32; state (R, W - 1, D) of x's type, the inputs before
    step 0, oldest first (None: zeros); starts (T, R). activation: None or "silu". Returns y like x,
    and with return_state the state after the last step (inputs from before the last start as
    zeros). Gradients flow to x, weight, bias, state and back from the returned state."""
    _refuse_tangents("short_conv", x, weight, bias, state)
    _conv_check("short_conv", x, weight, bias, state, starts, activation, 3)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, state)):
        if torch.cuda.is_current_stream_capturing():
            _refuse_held(x, weight, bias, state)
        out, new = _ShortConv.apply(x, weight, bias, state, starts, activation == "silu", return_state)
    else:
        out, new = _conv_forward(x, weight, bias, state, starts, activation == "silu", return_state)
    return (out, new) if return_state else out


def short_conv_step(x, state, weight, bias=None, starts=None, activation=None):
    """One step of short_conv for every row: x (R, D), starts (R,); state (R, W - 1, D) is renewed in
    place. Returns y (R, D). No gradients."""
    who = "short_conv_step"
    _refuse_tangents(who, x, state, weight, bias)
    if not isinstance(state, torch.Tensor):
        raise ValueError(f"{who}: state must be a tensor")
    _conv_check(who, x, weight, bias, state, starts, activation, 2)
    R, D = x.shape
    out = torch.empty((R, D), dtype=x.dtype, device=x.device)
    at = state.data_ptr()
    _call(N.lib().ms_conv_forward,
          _CONV_STEP.pack(_DTYPES[x.dtype], weight.shape[1], activation == "silu", 0, 1, R, D, x.data_ptr(), 0, x.stride(0),
                          weight.data_ptr(), _p(bias), at, *_row3(starts), out.data_ptr(), 0, D, at) + _CONV_ZEROS, x.get_device())
    _renewed(state)
    return out


# ---------------------------------------------------------------- state-space scan

def _scan_right(u, delta, A, B, Cm, D, z, delta_bias, state, starts, dims):
    """Everything that _scan_check looks for, in one go."""
    try:
        shape, dt, i = u.shape, u.dtype, u.get_device()
        ch, (_, n), given = shape[-1], A.shape, B.shape
        if not (i >= 0 and len(shape) == dims and dt in _DTYPES and ch > 0 and u.stride(-1) == 1 and 1 <= n <= MAX_STATES):
            return False
        lead = shape[:-1]
        if len(given) > dims:
            if given[-2] < 1 or ch % given[-2] or given != (*lead, given[-2], n):
                return False
        elif given != (*lead, n):
            return False
        return (_right(delta, shape, dt, i) and _right(B, given, dt, i) and _right(Cm, given, dt, i)
                and (z is None or _right(z, shape, dt, i)) and _right_weight(A, (ch, n), i) and _right_weight(D, (ch,), i)
                and _right_weight(delta_bias, (ch,), i) and _right_weight(state, (shape[-2], ch, n), i)
                and _right_starts(starts, lead, i))
    except (AttributeError, IndexError, ValueError):
        return False


def _scan_check(who, u, delta, A, B, Cm, D, z, delta_bias, state, starts, dims):
    if _scan_right(u, delta, A, B, Cm, D, z, delta_bias, state, starts, dims):
        return
    _sequence(who, "u", u, dims)
    device, dt, ch = u.device, u.dtype, u.shape[-1]
    lead = u.shape[:-1]
    _check(who, "u", u, u.shape, dt, device)
    _check(who, "delta", delta, u.shape, dt, device)
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"{who}: A must be a (channels, states) tensor of 1 to {MAX_STATES} states")
    n = A.shape[1]
    _check(who, "A", A, (ch, n), torch.float32, device, True)
    for name, t in (("B", B), ("C", Cm)):
        if not isinstance(t, torch.Tensor) or t.dim() not in (dims, dims + 1):
            raise ValueError(f"{who}: {name} must be a tensor of {dims} or {dims + 1} dimensions (time, row, [group,] state)")
        if t.dim() != B.dim():
            raise ValueError(f"{who}: B and C must have the same shape")
        groups = B.shape[-2] if t.dim() > dims else 1
        if groups < 1 or ch % groups:
            raise ValueError(f"{who}: {groups} groups do not divide {ch} channels")
        _check(who, name, t, (*lead, groups, n) if t.dim() > dims else (*lead, n), dt, device)
    if D is not None:
        _check(who, "D", D, (ch,), torch.float32, device, True)
    if z is not None:
        _check(who, "z", z, u.shape, dt, device)
    if delta_bias is not None:
        _check(who, "delta_bias", delta_bias, (ch,), torch.float32, device, True)
    if state is not None:
        _check(who, "state", state, (lead[-1], ch, n), torch.float32, device, True)
    _check_starts(who, starts, lead, device)
    _on_gpu(who, device)


def _scan_io(u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft, out=None, new=None, keep=None, dout=None, dnew=None,
             du=None, ddelta=None, dz=None, dB=None, dC=None, dA=None, dD=None, dbias=None, dstate=None):
    T, R, ch = u.shape
    return _SCAN.pack(_DTYPES[u.dtype], soft, A.shape[1], B.shape[2] if B.dim() == 4 else 1, T, R, ch, *_p3(u), *_p3(delta),
                      *_p3(z), *_g4(B), *_g4(Cm), A.data_ptr(), _p(D), _p(delta_bias), _p(state), *_p3(starts), *_p3(out),
                      _p(new), _p(keep), *_p3(dout), _p(dnew), *_p3(du), *_p3(ddelta), *_p3(dz), _p(dB), _p(dC), _p(dA), _p(dD),
                      _p(dbias), _p(dstate), 0, 0)


def _scan_forward(u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft, want_state, want_grad):
    """The outputs, the last states, and what the backward reads beside the inputs."""
    L = N.lib()
    out = _like(u)
    new = torch.empty((u.shape[1], *A.shape), dtype=torch.float32, device=u.device) if want_state else None
    io = _scan_io(u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft, out, new)
    keep = None
    if want_grad:
        keep = torch.empty((L.ms_scan_checkpoints(io),), dtype=torch.uint8, device=u.device)
        io = io[:_KEEP_AT] + _POINTER.pack(keep.data_ptr()) + io[_KEEP_AT + _POINTER.size:]
    size = L.ms_scan_workspace(io, 0)
    if size:
        work = torch.empty((size,), dtype=torch.uint8, device=u.device)
        io = _with_workspace(io, work)
    _call(L.ms_scan_forward, io, u.get_device())
    return out, new, keep


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft, want_state):
        out, new, keep = _scan_forward(u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft, want_state, True)
        ctx.save_for_backward(u, delta, A, B, Cm, D, z, delta_bias, state, starts, keep)
        ctx.soft = soft
        ctx.set_materialize_grads(False)
        _lives(ctx, N.current_raw_stream(u.get_device()))
        return out, new

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dnew):
        u, delta, A, B, Cm, D, z, delta_bias, state, starts, keep = ctx.saved_tensors
        if dout is None and dnew is None:
            return (None,) * 12
        need = ctx.needs_input_grad
        L = N.lib()
        dout = torch.zeros_like(u) if dout is None else _rows(dout)
        dnew = None if dnew is None else dnew.contiguous()
        du, ddelta, dz = _like(u), _like(u), _like(u) if z is not None else None
        dB = torch.empty_like(B, memory_format=torch.contiguous_format)
        dC = torch.empty_like(Cm, memory_format=torch.contiguous_format)
        dA = torch.empty_like(A)
        dD = torch.empty_like(D) if D is not None and need[5] else None
        dbias = torch.empty_like(delta_bias) if delta_bias is not None and need[7] else None
        dstate = torch.empty_like(state) if state is not None and need[8] else None
        io = _scan_io(u, delta, A, B, Cm, D, z, delta_bias, state, starts, ctx.soft, None, None, keep, dout, dnew, du, ddelta,
                      dz, dB, dC, dA, dD, dbias, dstate)
        work = torch.empty((L.ms_scan_workspace(io, 1),), dtype=torch.uint8, device=u.device)
        _call(L.ms_scan_backward, _with_workspace(io, work), u.get_device())
        grads = (du, ddelta, dA, dB, dC, dD, dz, dbias, dstate)
        return tuple(g if n else None for g, n in zip(grads, need)) + (None,) * 3


def ssm_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, starts=None, delta_softplus=True,
             return_state=False):
    """Selective state-space scan along time. For every row, channel d and state n, with
    rate = softplus(delta + delta_bias) (without the softplus if not delta_softplus):
        h[n] = exp(rate A[d, n]) h[n] + rate u B[n],   y = (sum_n C[n] h[n] + D u) silu(z).

    u, delta, z (T, R, D); B, C (T, R, N), or (T, R, G, N) with each group shared by D / G
    neighbouring channels; A (D, N), D (D), delta_bias (D) float32, A negative for states that decay;
    N 1 to 64; state (R, D, N) float32 before step 0 (None: zeros); starts (T, R); z None: no gate.
    Returns y like u, and with return_state the states after the last step. Gradients flow to every
    input but starts, and back from the returned state; with them the forward also keeps the states
    of every 8th step (4 N bytes a channel), and B and C in float32, until the backward."""
    _refuse_tangents("ssm_scan", u, delta, A, B, C, D, z, delta_bias, state)
    _scan_check("ssm_scan", u, delta, A, B, C, D, z, delta_bias, state, starts, 3)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (u, delta, A, B, C, D, z, delta_bias, state)):
        if torch.cuda.is_current_stream_capturing():
            _refuse_held(u, delta, A, B, C, D, z, delta_bias, state)
        out, new = _Scan.apply(u, delta, A, B, C, D, z, delta_bias, state, starts, bool(delta_softplus), return_state)
    else:
        out, new, _ = _scan_forward(u, delta, A, B, C, D, z, delta_bias, state, starts, bool(delta_softplus), return_state, False)
    return (out, new) if return_state else out


def ssm_step(state, u, delta, A, B, C, D=None, z=None, delta_bias=None, starts=None, delta_softplus=True):
    """One step of ssm_scan for every row: u, delta, z (R, D), B, C (R, N) or (R, G, N), starts (R,);
    state (R, D, N) is renewed in place. Returns y (R, D). No gradients."""
    who = "ssm_step"
    _refuse_tangents(who, state, u, delta, A, B, C, D, z, delta_bias)
    if not isinstance(state, torch.Tensor):
        raise ValueError(f"{who}: state must be a tensor")
    _scan_check(who, u, delta, A, B, C, D, z, delta_bias, state, starts, 2)
    R, ch = u.shape
    out = torch.empty((R, ch), dtype=u.dtype, device=u.device)
    grouped, at = B.dim() == 3, state.data_ptr()
    _call(N.lib().ms_scan_step,
          _SCAN_STEP.pack(_DTYPES[u.dtype], bool(delta_softplus), A.shape[1], B.shape[1] if grouped else 1, 1, R, ch, u.data_ptr(),
                          0, u.stride(0), delta.data_ptr(), 0, delta.stride(0), *_row3(z), B.data_ptr(), 0, B.stride(0),
                          B.stride(1) if grouped else 0, C.data_ptr(), 0, C.stride(0), C.stride(1) if grouped else 0, A.data_ptr(),
                          _p(D), _p(delta_bias), at, *_row3(starts), out.data_ptr(), 0, ch, at) + _SCAN_ZEROS, u.get_device())
    _renewed(state)
    return out
