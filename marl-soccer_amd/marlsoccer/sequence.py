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
sequence forms carry gradients to every input but `starts` (once: no double backward). Calls are
asynchronous on the current stream of the tensors' device and may be captured into a HIP graph.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _native as N

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_STATES = 64


def _fail(rc: int) -> None:
    raise (ValueError if rc == N.MS_ERR_INVALID_ARGUMENT else N.NativeError)(
        N.lib().ms_sequence_last_error().decode(errors="replace"))


def _call(fn, io, device) -> None:
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        rc = fn(C.byref(io), stream)
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(io), stream)
    if rc:
        _fail(rc)


def _p(t):
    return None if t is None else t.data_ptr()


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

def _conv_io(x, weight, bias, state, starts, silu):
    T, R, D = x.shape
    io = N.MsConvIO(dtype=_DTYPES[x.dtype], width=weight.shape[1], silu=silu, steps=T, rows=R, channels=D, x=_p(x),
                    x_t=x.stride(0), x_r=x.stride(1), weight=_p(weight), bias=_p(bias), state=_p(state))
    if starts is not None:
        io.starts, io.starts_t, io.starts_r = starts.data_ptr(), starts.stride(0), starts.stride(1)
    return io


def _conv_check(who, x, weight, bias, state, starts, activation, dims):
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


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, starts, silu, want_state):
        out = _like(x)
        new = torch.empty((x.shape[1], weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device) if want_state else None
        io = _conv_io(x, weight, bias, state, starts, silu)
        io.out, io.out_t, io.out_r, io.new_state = _p(out), out.stride(0), out.stride(1), _p(new)
        _call(N.lib().ms_conv_forward, io, x.device)
        ctx.save_for_backward(x, weight, bias, state, starts)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
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
        io = _conv_io(x, weight, bias, state, starts, ctx.silu)
        io.dout, io.dout_t, io.dout_r, io.dnew_state = _p(dout), dout.stride(0), dout.stride(1), _p(dnew)
        io.dx, io.dx_t, io.dx_r, io.dstate, io.dweight, io.dbias = _p(dx), dx.stride(0), dx.stride(1), _p(dstate), _p(dweight), _p(dbias)
        L = N.lib()
        io.workspace_bytes = L.ms_conv_workspace(C.byref(io))
        work = torch.empty((io.workspace_bytes,), dtype=torch.uint8, device=x.device)
        io.workspace = work.data_ptr()
        _call(L.ms_conv_backward, io, x.device)
        return dx if need[0] else None, dweight, dbias, dstate, None, None, None


def short_conv(x, weight, bias=None, state=None, starts=None, activation=None, return_state=False):
    """Causal convolution along time with a kernel of 2 to 4 steps per channel:
    y[t] = act(bias + sum_k weight[:, k] x[t - W + 1 + k]).

    x (T, R, D); weight (D, W), bias (D) float32; state (R, W - 1, D) of x's type, the inputs before
    step 0, oldest first (None: zeros); starts (T, R). activation: None or "silu". Returns y like x,
    and with return_state the state after the last step (inputs from before the last start as
    zeros). Gradients flow to x, weight, bias, state and back from the returned state."""
    _conv_check("short_conv", x, weight, bias, state, starts, activation, 3)
    out, new = _ShortConv.apply(x, weight, bias, state, starts, activation == "silu", return_state)
    return (out, new) if return_state else out


@torch.no_grad()
def short_conv_step(x, state, weight, bias=None, starts=None, activation=None):
    """One step of short_conv for every row: x (R, D), starts (R,); state (R, W - 1, D) is renewed in
    place. Returns y (R, D). No gradients."""
    who = "short_conv_step"
    if not isinstance(state, torch.Tensor):
        raise ValueError(f"{who}: state must be a tensor")
    _conv_check(who, x, weight, bias, state, starts, activation, 2)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    io = N.MsConvIO(dtype=_DTYPES[x.dtype], width=weight.shape[1], silu=activation == "silu", steps=1, rows=x.shape[0],
                    channels=x.shape[1], x=x.data_ptr(), x_r=x.stride(0), weight=weight.data_ptr(), bias=_p(bias),
                    state=state.data_ptr(), starts=_p(starts), starts_r=0 if starts is None else starts.stride(0),
                    out=out.data_ptr(), out_r=out.stride(0), new_state=state.data_ptr())
    _call(N.lib().ms_conv_forward, io, x.device)
    return out


# ---------------------------------------------------------------- state-space scan

def _scan_check(who, u, delta, A, B, Cm, D, z, delta_bias, state, starts, dims):
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


def _scan_io(u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft):
    T, R, ch = u.shape
    io = N.MsScanIO(dtype=_DTYPES[u.dtype], softplus=soft, states=A.shape[1], groups=B.shape[2] if B.dim() == 4 else 1,
                    steps=T, rows=R, channels=ch, u=_p(u), u_t=u.stride(0), u_r=u.stride(1), delta=_p(delta),
                    delta_t=delta.stride(0), delta_r=delta.stride(1), B=_p(B), B_t=B.stride(0), B_r=B.stride(1),
                    C=_p(Cm), C_t=Cm.stride(0), C_r=Cm.stride(1), A=_p(A), D=_p(D), delta_bias=_p(delta_bias),
                    state=_p(state))
    if B.dim() == 4:
        io.B_g, io.C_g = B.stride(2), Cm.stride(2)
    if z is not None:
        io.z, io.z_t, io.z_r = z.data_ptr(), z.stride(0), z.stride(1)
    if starts is not None:
        io.starts, io.starts_t, io.starts_r = starts.data_ptr(), starts.stride(0), starts.stride(1)
    return io


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft, want_state, want_grad):
        L = N.lib()
        out = _like(u)
        new = torch.empty((u.shape[1], *A.shape), dtype=torch.float32, device=u.device) if want_state else None
        io = _scan_io(u, delta, A, B, Cm, D, z, delta_bias, state, starts, soft)
        io.out, io.out_t, io.out_r, io.new_state = _p(out), out.stride(0), out.stride(1), _p(new)
        keep = None
        if want_grad:
            keep = torch.empty((L.ms_scan_checkpoints(C.byref(io)),), dtype=torch.uint8, device=u.device)
            io.checkpoints = keep.data_ptr()
        io.workspace_bytes = L.ms_scan_workspace(C.byref(io), 0)
        work = None
        if io.workspace_bytes:
            work = torch.empty((io.workspace_bytes,), dtype=torch.uint8, device=u.device)
            io.workspace = work.data_ptr()
        _call(L.ms_scan_forward, io, u.device)
        ctx.save_for_backward(u, delta, A, B, Cm, D, z, delta_bias, state, starts, keep)
        ctx.soft = soft
        ctx.set_materialize_grads(False)
        return out, new

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dnew):
        u, delta, A, B, Cm, D, z, delta_bias, state, starts, keep = ctx.saved_tensors
        if dout is None and dnew is None:
            return (None,) * 13
        need = ctx.needs_input_grad
        L = N.lib()
        dout = torch.zeros_like(u) if dout is None else _rows(dout)
        dnew = None if dnew is None else dnew.contiguous()
        io = _scan_io(u, delta, A, B, Cm, D, z, delta_bias, state, starts, ctx.soft)
        io.checkpoints = keep.data_ptr()
        du, ddelta, dz = _like(u), _like(u), _like(u) if z is not None else None
        dB = torch.empty_like(B, memory_format=torch.contiguous_format)
        dC = torch.empty_like(Cm, memory_format=torch.contiguous_format)
        dA = torch.empty_like(A)
        dD = torch.empty_like(D) if D is not None and need[5] else None
        dbias = torch.empty_like(delta_bias) if delta_bias is not None and need[7] else None
        dstate = torch.empty_like(state) if state is not None and need[8] else None
        io.dout, io.dout_t, io.dout_r, io.dnew_state = _p(dout), dout.stride(0), dout.stride(1), _p(dnew)
        io.du, io.du_t, io.du_r = _p(du), du.stride(0), du.stride(1)
        io.ddelta, io.ddelta_t, io.ddelta_r = _p(ddelta), ddelta.stride(0), ddelta.stride(1)
        if dz is not None:
            io.dz, io.dz_t, io.dz_r = _p(dz), dz.stride(0), dz.stride(1)
        io.dB, io.dC, io.dA, io.dD, io.ddelta_bias, io.dstate = _p(dB), _p(dC), _p(dA), _p(dD), _p(dbias), _p(dstate)
        io.workspace_bytes = L.ms_scan_workspace(C.byref(io), 1)
        work = torch.empty((io.workspace_bytes,), dtype=torch.uint8, device=u.device)
        io.workspace = work.data_ptr()
        _call(L.ms_scan_backward, io, u.device)
        grads = (du, ddelta, dA, dB, dC, dD, dz, dbias, dstate)
        return tuple(g if n else None for g, n in zip(grads, need)) + (None,) * 4


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
    of every 16th step (4 N bytes a channel) until the backward."""
    _scan_check("ssm_scan", u, delta, A, B, C, D, z, delta_bias, state, starts, 3)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (u, delta, A, B, C, D, z, delta_bias, state))
    out, new = _Scan.apply(u, delta, A, B, C, D, z, delta_bias, state, starts, bool(delta_softplus), return_state, grad)
    return (out, new) if return_state else out


@torch.no_grad()
def ssm_step(state, u, delta, A, B, C, D=None, z=None, delta_bias=None, starts=None, delta_softplus=True):
    """One step of ssm_scan for every row: u, delta, z (R, D), B, C (R, N) or (R, G, N), starts (R,);
    state (R, D, N) is renewed in place. Returns y (R, D). No gradients."""
    who = "ssm_step"
    if not isinstance(state, torch.Tensor):
        raise ValueError(f"{who}: state must be a tensor")
    _scan_check(who, u, delta, A, B, C, D, z, delta_bias, state, starts, 2)
    out = torch.empty_like(u, memory_format=torch.contiguous_format)
    io = N.MsScanIO(dtype=_DTYPES[u.dtype], softplus=bool(delta_softplus), states=A.shape[1],
                    groups=B.shape[1] if B.dim() == 3 else 1, steps=1, rows=u.shape[0], channels=u.shape[1],
                    u=u.data_ptr(), u_r=u.stride(0), delta=delta.data_ptr(), delta_r=delta.stride(0), B=B.data_ptr(),
                    B_r=B.stride(0), B_g=B.stride(1) if B.dim() == 3 else 0, C=C.data_ptr(), C_r=C.stride(0),
                    C_g=C.stride(1) if B.dim() == 3 else 0, z=_p(z), z_r=0 if z is None else z.stride(0), A=A.data_ptr(),
                    D=_p(D), delta_bias=_p(delta_bias), state=state.data_ptr(), starts=_p(starts),
                    starts_r=0 if starts is None else starts.stride(0), out=out.data_ptr(), out_r=out.stride(0),
                    new_state=state.data_ptr())
    _call(N.lib().ms_scan_step, io, u.device)
    return out
