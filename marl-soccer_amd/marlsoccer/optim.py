"""AdamW over many tensors in one launch (csrc/ms_optim.hip), for the PPO update of a policy.

The reference's update (marl-soccer.ipynb train cell) is clip_grad_norm_ and Adam over the Agent's 21
tensors, small ones: a launch an operation and tensor. Here the norm is one launch and the step
another, for any list; parameters change in place, so a captured rollout graph (DeviceRollout) goes on
reading them, and step counts, clip factor and, if wanted, the learning rate stay on the device, so
the step itself may be captured.

    opt = AdamW(agent.parameters(), lr=2.5e-4, eps=1e-5, weight_decay=0.0, max_grad_norm=0.5)
    loss.backward(); opt.step(); opt.zero_grad()

state_bits=8 holds both moments as OCP e4m3 bytes with a float32 scale for every 256 values: 2 B a
value instead of 8. The second moment is held as its root. A step of the codes is 2^-4 to 2^-3 of the value
down to 2^-14.8 of its block's largest, and 2^-17.8 of the largest below that.

rounding="stochastic" is for training: each value goes to one of its two neighbours with the odds that
keep its expectation, from a hash of the step count and its place (the same step gives the same bits). The
moments then follow the 32-bit ones in the mean; with beta2 = 0.999 a held root wanders by some 17 % about
the 32-bit one. rounding="nearest" holds each step's moments to half a step of the codes, but what a step
changes by less than that is lost, at every step, however many follow: with beta2 = 0.999 a root moves by
some 0.05 % a step, so all but the block's largest only follow that one, through the scale. When gradients
change in size their roots stay off: by 0.3 to 9 times after thousands of steps where some of a block's
values grew four times or shrank ten times against the others. With either a
root below the smallest code (2^-17.8 of its block's largest) is held as that code: held as 0 it would leave
the next step's gradient and eps alone to divide by. A moment that is infinite or no number is
held as no number, and reaches no other value of its block.
"""
from __future__ import annotations

import struct
import warnings
from itertools import chain, repeat
from operator import attrgetter

import torch

from . import _native as N

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
WORKSPACE = 4096   # MS_OPTIM_WORKSPACE, floats
BLOCK = 256        # MS_ADAMW_BLOCK: values that share a scale
F8 = torch.float8_e4m3fn
ROUNDINGS = {"nearest": 0, "stochastic": 256}  # MS_ADAMW_STOCHASTIC


def scales_for(numel: int) -> int:
    """How many scales an 8-bit moment of numel values has."""
    return -(-numel // BLOCK)


def moment_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 values that an 8-bit moment holds (for exp_avg_sq: their squares are the second
    moment)."""
    flat = codes.reshape(-1).to(torch.float32)
    return (flat * scales.repeat_interleave(BLOCK)[: flat.numel()]).view(codes.shape)


def _raise(rc: int) -> None:
    raise (ValueError if rc == N.MS_ERR_INVALID_ARGUMENT else N.NativeError)(
        N.lib().ms_optim_last_error().decode(errors="replace"))


def _bad(name, want):
    raise ValueError(f"adamw_step: {name} must be {want}")


_ROW = "6QQq2i"  # ms_optim_tensor
_ROW_BYTES = struct.calcsize("<" + _ROW)
_DTYPE, _SHAPE = attrgetter("dtype"), attrgetter("shape")
_where, _ptr_of, _numel, _packed = (getattr(torch.Tensor, k) for k in ("get_device", "data_ptr", "numel", "is_contiguous"))


def _entries(params, grads, exp_avg, exp_avg_sq, steps, scales, sq_scales):
    """The checked list as ms_optim_tensor rows (bytes), and its device. The lists are gone through
    attribute by attribute: a short list of small tensors takes longer on the host than on the GPU."""
    n, bits8 = len(params), scales is not None
    for name, ts in (("grads", grads), ("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq), ("steps", steps),
                     ("exp_avg_scales", scales), ("exp_avg_sq_scales", sq_scales)):
        if ts is not None and len(ts) != n:
            _bad(name, f"a list of {n} tensors, one for every parameter")
    every = [*params, *grads, *exp_avg, *exp_avg_sq]
    dts, shapes, moment = list(map(_DTYPE, every)), list(map(_SHAPE, every)), F8 if bits8 else torch.float32
    of_params = dts[:n]
    if not (dts[n:2 * n] == of_params and dts[2 * n:] == [moment] * (2 * n) and all(dt in _DTYPES for dt in set(of_params))
            and shapes[:n] == shapes[n:2 * n] == shapes[2 * n:3 * n] == shapes[3 * n:] and all(map(_packed, every))
            and all(dt is torch.int64 for dt in map(_DTYPE, steps)) and all(k == 1 for k in map(_numel, steps))
            and len({*map(_where, every), *map(_where, steps)}) == 1):
        for p, g, m, v, s in zip(params, grads, exp_avg, exp_avg_sq, steps):
            _explain(p, g, m, v, s, moment, params[0].device)
    sizes = list(map(_numel, params))
    if bits8:
        both = [*scales, *sq_scales]
        if not (list(map(_numel, both)) == [-(-k // BLOCK) for k in sizes] * 2 and set(map(_DTYPE, both)) == {torch.float32}
                and all(map(_packed, both)) and set(map(_where, both)) == {params[0].get_device()}):
            _bad("scales", f"contiguous float32 on {params[0].device}, one for every {BLOCK} values of their parameter")
        a, b = list(map(_ptr_of, scales)), list(map(_ptr_of, sq_scales))
    else:
        a = b = repeat(0)
    at, counts = list(map(_ptr_of, every)), list(map(_ptr_of, steps))
    written = [q for q, k in zip(at[:n] + at[2 * n:] + (a + b if bits8 else []), sizes * 5) if k]
    alone = set(written)
    if (len(alone) != len(written) or len(set(counts)) != n
            or not alone.isdisjoint(at[n:2 * n]) and any(k and q in alone for q, k in zip(at[n:2 * n], sizes))):
        _bad("every parameter, moment, scale and step count", "a tensor of its own: one is given twice")
    rows = zip(at[:n], at[n:2 * n], at[2 * n:3 * n], at[3 * n:], a, b, counts, sizes,
               [_DTYPES[dt] for dt in of_params], repeat(0))
    return struct.pack("<" + _ROW * n, *chain.from_iterable(rows)), params[0].device


def _explain(p, g, m, v, s, moment, device):
    """Raises for the first thing that is wrong with a parameter's tensors."""
    if p.dtype not in _DTYPES:
        _bad("a parameter", f"float32, bfloat16 or float16, got {p.dtype}")
    if not all(t.is_contiguous() for t in (p, g, m, v)):
        _bad("every tensor", "contiguous")
    if g.dtype != p.dtype or g.shape != p.shape:
        _bad("a gradient", "of its parameter's type and shape")
    if any(t.dtype != moment or t.shape != p.shape for t in (m, v)):
        _bad("a moment", f"{moment} of its parameter's shape")
    if s.dtype != torch.int64 or s.numel() != 1:
        _bad("a step count", "one int64")
    if any(t.device != device for t in (p, g, m, v, s)):
        _bad("every tensor", f"on one device ({device})")


def _check_workspace(workspace, device):
    if workspace.dtype != torch.float32 or workspace.numel() < WORKSPACE or not workspace.is_contiguous() or workspace.device != device:
        _bad("workspace", f"{WORKSPACE} contiguous float32 on {device}, zeroed when made")


def _launch(device, params, calls):
    if device.type != "cuda":
        raise ValueError(f"adamw_step: tensors must be on a HIP device, got {device}")
    for fn, *args in calls:
        rc = N.on_current_stream(device.index, fn, *args)
        if rc:
            _raise(rc)
    torch.autograd.graph.increment_version(params)  # a graph that saved a parameter refuses its backward


def adamw_step(params, grads, exp_avg, exp_avg_sq, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               max_grad_norm=None, exp_avg_scales=None, exp_avg_sq_scales=None, workspace=None, grad_norm=None, rounding="nearest"):
    """One AdamW step over a list of tensors, in place (see ms_adamw_step in include/marl_soccer.h):
    parameters and gradients float32, bfloat16 or float16, contiguous; moments float32, or float8_e4m3fn
    with scales; steps: one int64 on the device for each. What is written must not overlap what else is
    read or written (the same tensor twice is refused). lr: a float, or one float32 on the device.
    max_grad_norm: clip all gradients together by their norm (the gradients themselves stay as they
    are); grad_norm: one float32 on the device that receives the norm (max_grad_norm inf: the norm alone). workspace: WORKSPACE zeroed
    floats, kept by a caller that steps often (None: made here); one step at a time may use it.
    rounding: of moments with scales, "nearest" or "stochastic" (the module's comment)."""
    if not len(params):
        return
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        _bad("exp_avg_scales and exp_avg_sq_scales", "both given or both None")
    if rounding not in ROUNDINGS:
        _bad("rounding", f"'nearest' or 'stochastic', got {rounding!r}")
    rows, device = _entries(params, grads, exp_avg, exp_avg_sq, steps, exp_avg_scales, exp_avg_sq_scales)
    if max_grad_norm is not None and not max_grad_norm > 0:
        _bad("max_grad_norm", "positive")
    if grad_norm is not None and max_grad_norm is None:
        _bad("grad_norm", "given with max_grad_norm: without it no norm is computed (inf computes it and clips nothing)")
    if grad_norm is not None and (grad_norm.dtype != torch.float32 or grad_norm.numel() != 1 or grad_norm.device != device):
        _bad("grad_norm", f"one float32 on {device}")
    if device.type == "cuda" and workspace is None:
        workspace = torch.zeros(WORKSPACE, dtype=torch.float32, device=device)
    if workspace is not None:
        _check_workspace(workspace, device)
    calls = []
    if max_grad_norm is not None:
        calls.append(_clip_call(rows, max_grad_norm, grad_norm, workspace))
    calls.append(_step_call(rows, 8 | ROUNDINGS[rounding] if exp_avg_scales is not None else 32, lr, betas, eps, weight_decay,
                            max_grad_norm is not None, workspace, device))
    _launch(device, params, calls)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _clip_call(rows, max_norm, grad_norm, workspace):
    return N.lib().ms_grad_clip, rows, len(rows) // _ROW_BYTES, float(max_norm), _ptr(grad_norm), _ptr(workspace)


def _step_call(rows, bits, lr, betas, eps, weight_decay, clip, workspace, device):
    lr_device = None
    if isinstance(lr, torch.Tensor):
        if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != device:
            _bad("lr", f"a float or one float32 on {device}")
        lr, lr_device = 0.0, lr.data_ptr()
    return (N.lib().ms_adamw_step, rows, len(rows) // _ROW_BYTES, bits, float(lr), lr_device, float(betas[0]), float(betas[1]),
            float(eps), float(weight_decay), int(clip), _ptr(workspace))


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (decoupled weight decay, no amsgrad) with every tensor of a group in
    one launch; weight_decay=0 is the notebook's Adam. max_grad_norm clips the gradients of all groups
    together inside the step (.grad stays unclipped; `last_grad_norm`, on the device, holds the norm).
    A parameter without a gradient is left alone, its step count too. state_bits: 32 or 8; rounding: of 8
    bits, "stochastic" or "nearest" (the module's comment; None: nearest, with a warning). lr may be one float32 on the device, which a captured step reads anew. State:
    step, exp_avg, exp_avg_sq and, with 8 bits, their scales; state_dict() carries all of it."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_grad_norm=None, state_bits=32,
                 rounding=None):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must be >= 0, got {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError("betas must be in [0, 1), eps and weight_decay >= 0")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"max_grad_norm must be positive, got {max_grad_norm}")
        if rounding is not None and (rounding not in ROUNDINGS or state_bits != 8):
            raise ValueError(f"rounding must be 'nearest' or 'stochastic', of moments in 8 bits, got {rounding!r} with {state_bits}")
        if state_bits == 8 and rounding is None:
            warnings.warn("AdamW: moments in 8 bits, rounded to nearest, lose small changes for good; rounding='stochastic' keeps them "
                          "in the mean", stacklevel=2)
        self.max_grad_norm, self.state_bits, self.rounding = max_grad_norm, state_bits, rounding
        self._work, self._clipped = {}, False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "state_bits": self.state_bits, "rounding": self.rounding}

    def __setstate__(self, state):
        super().__setstate__(state)
        self.rounding = state.get("rounding")
        self._work, self._clipped = {}, False  # a copy's own

    @property
    def last_grad_norm(self):
        """The norm of the last clipped step, one float32 on the device (None before it)."""
        return next((w[1] for w in self._work.values()), None) if self._clipped else None

    def _state_of(self, p):
        s = self.state[p]
        if not s:
            self._refuse_capture(p)
            dt = F8 if self.state_bits == 8 else torch.float32
            s["step"] = torch.zeros((), dtype=torch.int64, device=p.device)
            s["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device).to(dt)
            s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device).to(dt)
            if self.state_bits == 8:
                for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                    s[k] = torch.zeros(scales_for(p.numel()), dtype=torch.float32, device=p.device)
        return s

    @staticmethod
    def _refuse_capture(p):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take one step before the capture: a graph that made the moments would zero them at every replay")

    @staticmethod
    def _refuse_settings(group):
        for name in ("maximize", "amsgrad"):
            if group.get(name):
                raise ValueError(f"AdamW: {name}=True is set, which this update does not do")
        if group.get("weight_decay", 0) != 0 and not group.get("decoupled_weight_decay", True):
            raise ValueError("AdamW: a weight decay that is part of the gradient (torch.optim.Adam's) is set; this one's is decoupled")

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            self._refuse_settings(param_group)
        super().add_param_group(param_group)

    def load_state_dict(self, state_dict):
        """Its own state_dict() or that of torch.optim.AdamW. One whose update is another is refused:
        maximize, amsgrad, a weight decay that is not decoupled (torch.optim.Adam's), moments of other bits."""
        for g in state_dict["param_groups"]:
            self._refuse_settings(g)
        for s in state_dict["state"].values():
            if "exp_avg" in s and (s["exp_avg"].dtype == F8) != (self.state_bits == 8):
                raise ValueError(f"AdamW: the saved moments are {s['exp_avg'].dtype}, this optimizer holds them in {self.state_bits} bits")
        super().load_state_dict(state_dict)
        # Optimizer.load_state_dict casts floating-point state to the parameter's type: take it as it was saved
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, own):
            if i in state_dict["state"]:
                self.state[p] = {k: v.to(device=p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                 for k, v in state_dict["state"][i].items()}
                step = self.state[p].get("step")
                if isinstance(step, (int, float, torch.Tensor)):  # torch's own AdamW counts in float32, on the host
                    self.state[p]["step"] = torch.as_tensor(step).to(device=p.device, dtype=torch.int64)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups, device, every_param = [], None, []
        for group in self.param_groups:
            ps = [p for p in group["params"] if p.grad is not None]
            if not ps:
                continue
            if any(p.grad.is_sparse for p in ps):
                raise ValueError("adamw_step: sparse gradients are not supported")
            ss = [self._state_of(p) for p in ps]
            get = lambda k: [s[k] for s in ss]  # noqa: E731
            eight = self.state_bits == 8
            grads = [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in ps]
            rows, dev = _entries(ps, grads, get("exp_avg"), get("exp_avg_sq"), get("step"),
                                 get("exp_avg_scale") if eight else None, get("exp_avg_sq_scale") if eight else None)
            if device is not None and dev != device:
                _bad("every tensor", f"on one device ({device})")
            device = dev
            every_param += ps
            groups.append((group, rows, grads))  # copies among them live until the launches are in the stream
        if not groups:
            return loss
        if device.type == "cuda" and device not in self._work:
            self._refuse_capture(every_param[0])
            self._work[device] = (torch.zeros(WORKSPACE, dtype=torch.float32, device=device),
                                  torch.zeros((), dtype=torch.float32, device=device))
        work, norm = self._work.get(device, (None, None))
        calls = []
        if self.max_grad_norm is not None:
            every = b"".join(rows for _, rows, _ in groups)
            calls.append(_clip_call(every, self.max_grad_norm, norm, work))
        bits = self.state_bits | ROUNDINGS[self.rounding or "nearest"]
        for group, rows, _ in groups:
            calls.append(_step_call(rows, bits, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                                    self.max_grad_norm is not None, work, device))
        _launch(device, every_param, calls)
        self._clipped |= self.max_grad_norm is not None
        return loss
