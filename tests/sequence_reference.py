"""64-bit references of the sequence operators (marlsoccer.sequence), step by step on the CPU, and the
error bounds their tests use.

The bounds: an output is a sum of products of the inputs, computed in float32 in some order. Along
any chain of K roundings a term's relative error is at most K u / (1 - K u), u = 2^-24; so an output
is off by at most gamma times the same expression with every term's absolute value, which the same
functions return with absolute=True (inputs and slopes by their absolute values, decays as they are).
K counts, for the longest chain, `per` operations a step of the recurrence, the sums over states,
channels and rows, and the activations. A decay's error is that of v_exp_f32 (2 u) and of its argument
rate A, which two roundings and the rate's own error move by less than (6 + 2) u of |rate A| <= RATE_A
here. A 16-bit output is rounded once more: half a step, finfo.eps / 2 of its value.
"""
import torch

U = 2.0 ** -24
RATE_A = 16.0   # |rate A| is below it in the tests, where a decay is exp(-16) = 1e-7 already
PER_STEP = 4 + 2 + 8 * RATE_A / 4  # mean of |rate A| over a chain is below RATE_A / 4


def gamma(k):
    return k * U / (1 - k * U)


def sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def silu(x):
    return x * sigmoid(x)


def silu_slope(x):
    s = sigmoid(x)
    return s * (1 + x * (1 - s))


def silu_slope_size(x):
    """The slope's terms by their absolute values. s (1 + x (1 - s)) passes through zero at x = -1.28,
    where 1 and x (1 - s) cancel: the rounding of the sum's terms, u (1 + |x| (1 - s)) s a rounding,
    stays while the slope itself vanishes, so |slope| would be no bound."""
    s = sigmoid(x)
    return s * (1 + x.abs() * (1 - s))


def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, starts=None, soft=True, dout=None, dnew=None, absolute=False):
    """(out, last state, gradients by name) in float64; gradients where dout is given."""
    mag = (lambda x: x.abs()) if absolute else (lambda x: x)
    d64 = lambda x: None if x is None else x.detach().double().cpu()  # noqa: E731
    u, delta, A, B, C, D, z, delta_bias, state, dout, dnew = map(d64, (u, delta, A, B, C, D, z, delta_bias, state, dout, dnew))
    T, R, ch = u.shape
    grouped = B.dim() == 4
    if not grouped:
        B, C = B[:, :, None], C[:, :, None]
    G, N = B.shape[2:]
    per = ch // G
    raw = delta + (0 if delta_bias is None else delta_bias)
    rate = softplus(raw) if soft else raw
    slope = sigmoid(raw) if soft else torch.ones_like(raw)
    u, B, C, rate_m = mag(u), mag(B), mag(C), mag(rate)
    if absolute:
        D, state = (None if x is None else x.abs() for x in (D, state))
    skip = torch.zeros(ch, dtype=torch.float64) if D is None else D
    h = torch.zeros((R, ch, N), dtype=torch.float64) if state is None else state
    st = None if starts is None else starts.cpu().bool()
    wide = lambda x: x.repeat_interleave(per, 1)  # noqa: E731  (R, G, N) -> (R, D, N)
    hs, ys, decays, befores = [], [], [], []
    for t in range(T):
        if st is not None:
            h = torch.where(st[t][:, None, None], torch.zeros_like(h), h)
        a = torch.exp(rate[t][..., None] * A)
        decays.append(a)
        befores.append(h)
        h = a * h + (rate_m[t] * u[t])[..., None] * wide(B[t])
        hs.append(h)
        ys.append((h * wide(C[t])).sum(-1) + skip * u[t])
    y = torch.stack(ys) if T else torch.zeros_like(u)
    gate = torch.ones_like(u) if z is None else mag(silu(z))
    out = y * gate
    if dout is None:
        return out, h, None
    dout = mag(dout)
    zero = lambda x: torch.zeros_like(x)  # noqa: E731
    du, ddelta, dB, dC, dA = zero(u), zero(delta), zero(B), zero(C), zero(A)
    dz = None if z is None else dout * y * (silu_slope_size(z) if absolute else silu_slope(z))
    dy = dout * gate
    carry = zero(h) if dnew is None else mag(dnew)
    Am = mag(A)
    for t in reversed(range(T)):
        g = dy[t][..., None] * wide(C[t]) + carry
        fold = lambda x: x.view(R, G, per, N).sum(2)  # noqa: E731
        dC[t] = fold(dy[t][..., None] * hs[t])
        dB[t] = fold((rate_m[t] * u[t])[..., None] * g)
        gb = (g * wide(B[t])).sum(-1)
        q = g * decays[t] * befores[t]
        ddelta[t] = (gb * u[t] + (q * Am).sum(-1)) * slope[t]
        du[t] = rate_m[t] * gb + skip * dy[t]
        dA += (q * rate_m[t][..., None]).sum(0)
        carry = decays[t] * g
        if st is not None:
            carry = torch.where(st[t][:, None, None], zero(carry), carry)
    if not grouped:
        dB, dC = dB[:, :, 0], dC[:, :, 0]
    return out, h, dict(u=du, delta=ddelta, A=dA, B=dB, C=dC, D=(dy * u).sum((0, 1)), z=dz, delta_bias=ddelta.sum((0, 1)), state=carry)


def scan_chain(T, R, ch, N, grads):
    """K of the module's comment."""
    k = PER_STEP * T + N + 40
    return 2 * k + ch + T + R if grads else k


def conv(x, weight, bias=None, state=None, starts=None, act=True, dout=None, dnew=None, absolute=False):
    """(out, last state, gradients by name) in float64."""
    d64 = lambda v: None if v is None else v.detach().double().cpu()  # noqa: E731
    x, weight, bias, state, dout, dnew = map(d64, (x, weight, bias, state, dout, dnew))
    T, R, D = x.shape
    W = weight.shape[1]
    st = torch.zeros((T, R), dtype=torch.bool) if starts is None else starts.cpu().bool()
    bias = torch.zeros(D, dtype=torch.float64) if bias is None else bias
    ext = torch.cat([(torch.zeros((R, W - 1, D), dtype=torch.float64) if state is None else state).transpose(0, 1), x])
    taps, pres = [], []
    for t in range(T):
        row = []
        for k in range(W):
            s = t - (W - 1) + k  # the tap's step
            cut = torch.zeros(R, dtype=torch.bool)
            for m in range(max(s + 1, 0), t + 1):
                cut |= st[m]
            row.append(torch.where(cut[:, None], 0.0, ext[s + W - 1]))
        taps.append(row)
        pres.append(bias + sum(weight[:, k] * row[k] for k in range(W)))
    pre = torch.stack(pres) if T else torch.zeros_like(x)
    amount = (bias.abs() + torch.stack([sum((weight[:, k] * r[k]).abs() for k in range(W)) for r in taps])) if T else torch.zeros_like(x)
    out = silu(pre) if act else pre
    new = []
    for k in range(W - 1):
        s = T - (W - 1) + k
        cut = torch.zeros(R, dtype=torch.bool)
        for m in range(max(s + 1, 0), T):
            cut |= st[m]
        new.append(torch.where(cut[:, None], 0.0, ext[s + W - 1]))
    new = torch.stack(new, 1)
    if absolute:  # |d out| <= max slope (1.1) x |d pre|, and the product of the activation
        out = 1.1 * amount + out.abs() if act else amount
    if dout is None:
        return out, new, None
    slope = silu_slope(pre) if act else torch.ones_like(pre)
    if absolute:  # silu'' is below 0.5 in size: the error of pre moves the slope
        slope, dout, weight = (silu_slope_size(pre) + 0.5 * amount if act else slope), dout.abs(), weight.abs()
        taps = [[r.abs() for r in row] for row in taps]
        dnew = None if dnew is None else dnew.abs()
    dpre = dout * slope
    dext, dw = torch.zeros_like(ext), torch.zeros_like(weight)
    for t in range(T):
        for k in range(W):
            s = t - (W - 1) + k
            cut = torch.zeros(R, dtype=torch.bool)
            for m in range(max(s + 1, 0), t + 1):
                cut |= st[m]
            dext[s + W - 1] += torch.where(cut[:, None], 0.0, weight[:, k] * dpre[t])
            dw[:, k] += (dpre[t] * taps[t][k]).sum(0)
    if dnew is not None:
        for k in range(W - 1):
            s = T - (W - 1) + k
            cut = torch.zeros(R, dtype=torch.bool)
            for m in range(max(s + 1, 0), T):
                cut |= st[m]
            dext[s + W - 1] += torch.where(cut[:, None], 0.0, dnew[:, k])
    return out, new, dict(x=dext[W - 1:], weight=dw, bias=dpre.sum((0, 1)), state=dext[: W - 1].transpose(0, 1))


def assert_close(name, got, want, size, k):
    """got (any type) against the 64-bit value and the magnitude of its terms: the module's bound."""
    g = got.detach().double().cpu()
    assert g.shape == want.shape, (name, g.shape, want.shape)
    eps = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a step among the subnormals
    if got.dtype != torch.float16:
        tiny = torch.finfo(got.dtype).smallest_normal  # float32's and bfloat16's are flushed in places
    bound = gamma(k) * size + eps * (want.abs() + gamma(k) * size) + tiny
    off = (g - want).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = int((off / bound).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got {float(g.reshape(-1)[i])}, want "
                             f"{float(want.reshape(-1)[i])}, off {float(off.reshape(-1)[i]):.3g}, allowed {float(bound.reshape(-1)[i]):.3g}")
