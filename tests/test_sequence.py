"""The sequence operators (marlsoccer.sequence) against 64-bit references, their gradients against the
formulas and against differences, and what they refuse."""
import pytest

torch = pytest.importorskip("torch")

import sequence_reference as ref  # noqa: E402

from marlsoccer import sequence as seq  # noqa: E402

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}
gpu = pytest.mark.gpu


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def scan_inputs(T, R, D, N, G, dtype, seed=0, device="cpu", starts=False, state=False, gate=True, grouped=None):
    g = gen(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    grouped = G > 1 if grouped is None else grouped
    lead = (T, R, G) if grouped else (T, R)
    v = dict(u=r(T, R, D).to(dtype), delta=(0.5 * r(T, R, D)).to(dtype), A=-torch.exp(0.4 * r(D, N)) * torch.linspace(0.5, 4, N),
             B=r(*lead, N).to(dtype), C=r(*lead, N).to(dtype), D=r(D), z=r(T, R, D).to(dtype) if gate else None,
             delta_bias=r(D) - 1.5, state=r(R, D, N) if state else None,
             starts=(torch.rand((T, R), generator=g) < 0.2) if starts else None)
    return {k: None if t is None else t.to(device) for k, t in v.items()}


def conv_inputs(T, R, D, W, dtype, seed=0, device="cpu", starts=False, state=False, bias=True):
    g = gen(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    v = dict(x=r(T, R, D).to(dtype), weight=r(D, W) * 0.6, bias=r(D) * 0.2 if bias else None,
             state=r(R, W - 1, D).to(dtype) if state else None, starts=(torch.rand((T, R), generator=g) < 0.25) if starts else None)
    return {k: None if t is None else t.to(device) for k, t in v.items()}


# ---------------------------------------------------------------- the references themselves (CPU)

@pytest.mark.parametrize("starts,state,gate,G", [(False, False, True, 1), (True, True, True, 2), (True, True, False, 1)])
def test_scan_reference_gradients_match_differences(starts, state, gate, G):
    v = scan_inputs(5, 2, 4, 3, G, torch.float32, 1, starts=starts, state=state, gate=gate)
    v = {k: t.double() if t is not None and t.is_floating_point() else t for k, t in v.items()}
    g = gen(2)
    dout, dnew = torch.randn((5, 2, 4), generator=g).double(), torch.randn((2, 4, 3), generator=g).double()
    _, _, grads = ref.scan(**v, dout=dout, dnew=dnew)

    def value(w):
        out, h, _ = ref.scan(**w)
        return float((out * dout).sum() + (h * dnew).sum())

    for name in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"):
        if v[name] is None:
            continue
        for i in range(0, v[name].numel(), 3):
            d = torch.zeros(v[name].numel(), dtype=torch.float64)
            d[i] = 1e-6
            d = d.view(v[name].shape)
            fd = (value({**v, name: v[name] + d}) - value({**v, name: v[name] - d})) / 2e-6
            assert abs(fd - float(grads[name].reshape(-1)[i])) < 1e-7 * (1 + abs(fd)), name


@pytest.mark.parametrize("W", [2, 3, 4])
def test_conv_reference_gradients_match_differences(W):
    v = conv_inputs(6, 2, 3, W, torch.float32, 3, starts=True, state=True)
    v = {k: t.double() if t.is_floating_point() else t for k, t in v.items()}
    g = gen(4)
    dout, dnew = torch.randn((6, 2, 3), generator=g).double(), torch.randn((2, W - 1, 3), generator=g).double()
    _, _, grads = ref.conv(**v, dout=dout, dnew=dnew)

    def value(w):
        out, new, _ = ref.conv(**w)
        return float((out * dout).sum() + (new * dnew).sum())

    for name in ("x", "weight", "bias", "state"):
        for i in range(v[name].numel()):
            d = torch.zeros(v[name].numel(), dtype=torch.float64)
            d[i] = 1e-6
            d = d.view(v[name].shape)
            fd = (value({**v, name: v[name] + d}) - value({**v, name: v[name] - d})) / 2e-6
            assert abs(fd - float(grads[name].reshape(-1)[i])) < 1e-7 * (1 + abs(fd)), name


# ---------------------------------------------------------------- refusals (CPU)

def refuses(fn, match, *a, **k):
    with pytest.raises(ValueError, match=match):
        fn(*a, **k)


def test_short_conv_refusals():
    v = conv_inputs(4, 2, 6, 4, torch.float32, state=True, starts=True)
    x, w, b, s, st = (v[k] for k in ("x", "weight", "bias", "state", "starts"))
    refuses(seq.short_conv, "3 dimensions", x[0], w)
    refuses(seq.short_conv, "float32, bfloat16 or float16", x.double(), w)
    refuses(seq.short_conv, "width 2, 3 or 4", x, torch.randn(6, 5))
    refuses(seq.short_conv, "width 2, 3 or 4", x, torch.randn(6, 1))
    refuses(seq.short_conv, "weight must have shape", x, torch.randn(5, 4))
    refuses(seq.short_conv, "weight must be torch.float32", x, w.double())
    refuses(seq.short_conv, "weight must be contiguous", x, torch.randn(4, 6).t())
    refuses(seq.short_conv, "bias must have shape", x, w, b[:5])
    refuses(seq.short_conv, "state must have shape", x, w, b, s[:, :2])
    refuses(seq.short_conv, "state must be torch.float32", x, w, b, s.half())
    refuses(seq.short_conv, "last dimension must be contiguous", torch.randn(4, 6, 2).transpose(1, 2), w)
    refuses(seq.short_conv, "starts must be a bool or uint8", x, w, starts=st.float())
    refuses(seq.short_conv, "starts must have shape", x, w, starts=st[:3])
    refuses(seq.short_conv, "activation", x, w, activation="tanh")
    refuses(seq.short_conv, "HIP device", x, w, b, s, st)
    refuses(seq.short_conv_step, "state must be a tensor", x[0], None, w)
    refuses(seq.short_conv_step, "2 dimensions", x, s, w)
    refuses(seq.short_conv_step, "HIP device", x[0], s, w, b, st[0])


def test_ssm_scan_refusals():
    v = scan_inputs(4, 2, 6, 5, 1, torch.float32, state=True, starts=True)
    ok = lambda **k: seq.ssm_scan(**{**v, **k})  # noqa: E731
    refuses(ok, "HIP device")
    refuses(ok, "u must be a tensor of 3", u=v["u"][0])
    refuses(ok, "delta must have shape", delta=v["delta"][:3])
    refuses(ok, "delta must be torch.float32", delta=v["delta"].half())
    refuses(ok, "states", A=torch.randn(6, 65))
    refuses(ok, "A must have shape", A=torch.randn(5, 5))
    refuses(ok, "A must be contiguous", A=torch.randn(5, 6).t())
    refuses(ok, "B must have shape", B=v["B"][..., :4])
    refuses(ok, "B must be a tensor of 3 or 4", B=v["B"][0])
    refuses(ok, "same shape", C=v["C"][:, :, None])
    refuses(ok, "groups do not divide", B=torch.randn(4, 2, 4, 5), C=torch.randn(4, 2, 4, 5))
    refuses(ok, "C must be torch.float32", C=v["C"].half())
    refuses(ok, "D must have shape", D=torch.randn(5))
    refuses(ok, "z must have shape", z=v["z"][:, :1])
    refuses(ok, "delta_bias must be torch.float32", delta_bias=v["delta_bias"].double())
    refuses(ok, "state must be torch.float32", state=v["state"].half())
    refuses(ok, "starts", starts=torch.zeros(4, 3, dtype=torch.bool))
    refuses(ok, "last dimension must be contiguous", u=torch.randn(4, 6, 2).transpose(1, 2))
    step = {k: (t[0] if k in ("u", "delta", "B", "C", "z", "starts") else t) for k, t in v.items()}
    refuses(seq.ssm_step, "HIP device", **step)
    refuses(seq.ssm_step, "state must be a tensor", **{**step, "state": None})
    refuses(seq.ssm_step, "B must be a tensor of 2 or 3", **{**step, "B": v["B"][0, 0]})


def test_c_entries_refuse_bad_arguments():
    """The C entry points check what they are given before any launch."""
    import ctypes as C

    from marlsoccer import _native as N
    L = N.lib()
    for fn, io in ((L.ms_conv_forward, N.MsConvIO), (L.ms_conv_backward, N.MsConvIO), (L.ms_scan_forward, N.MsScanIO),
                   (L.ms_scan_step, N.MsScanIO), (L.ms_scan_backward, N.MsScanIO)):
        assert fn(None, None) == N.MS_ERR_INVALID_ARGUMENT
        assert fn(C.byref(io()), None) == N.MS_ERR_INVALID_ARGUMENT
        assert L.ms_sequence_last_error()
        bad = io(steps=1, rows=1, channels=4, width=4, weight=16) if io is N.MsConvIO else io(steps=1, rows=1, channels=4, states=4, groups=3, A=16)
        assert fn(C.byref(bad), None) == N.MS_ERR_INVALID_ARGUMENT
        bad.dtype = 7
        assert fn(C.byref(bad), None) == N.MS_ERR_INVALID_ARGUMENT and b"dtype" in L.ms_sequence_last_error()
    # a backward without its workspace, and an in-place state over several steps
    io = N.MsConvIO(dtype=0, width=4, steps=2, rows=1, channels=4, x=16, weight=16, out=16, dout=16, dx=16)
    assert L.ms_conv_backward(C.byref(io), None) == N.MS_ERR_INVALID_ARGUMENT and b"workspace" in L.ms_sequence_last_error()
    io.state = io.new_state = 16
    assert L.ms_conv_forward(C.byref(io), None) == N.MS_ERR_INVALID_ARGUMENT and b"one step" in L.ms_sequence_last_error()


# ---------------------------------------------------------------- against the references (GPU)

CONV = [(1, 1, 1, 4), (1, 3, 66, 4), (2, 2, 7, 3), (3, 1, 4, 4), (17, 3, 64, 4), (40, 2, 130, 3), (100, 2, 24, 4), (65, 5, 8, 2), (33, 1, 2050, 4)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("T,R,D,W", CONV)
@pytest.mark.parametrize("full", [False, True], ids=["bare", "full"])
def test_short_conv(T, R, D, W, dtype, full):
    need_gpu()
    v = conv_inputs(T, R, D, W, dtype, 7, "cuda", starts=full, state=full, bias=full)
    leaves = {k: t.requires_grad_() for k, t in v.items() if t is not None and k != "starts"}
    out, new = seq.short_conv(**v, activation="silu" if full else None, return_state=True)
    g = gen(8)
    dout = torch.randn((T, R, D), generator=g).to(dtype).cuda()
    dnew = torch.randn((R, W - 1, D), generator=g).to(dtype).cuda() if full else None
    loss = [(out, dout)] + ([(new, dnew)] if full else [])
    grads = dict(zip(leaves, torch.autograd.grad([a for a, _ in loss], list(leaves.values()), [b for _, b in loss])))
    kw = dict(act=full, dout=dout, dnew=dnew)
    want_out, want_new, want = ref.conv(**v, **kw)
    size_out, _, size = ref.conv(**v, **kw, absolute=True)
    ref.assert_close("out", out, want_out, size_out, W + 20)
    assert torch.equal(new.double().cpu(), want_new)
    for k in leaves:
        ref.assert_close(k, grads[k], want[k], size[k], 2 * W + 30 + (T * R if k in ("weight", "bias") else 0))


SCAN = [(1, 1, 1, 1, 1), (1, 2, 66, 16, 1), (2, 3, 5, 3, 1), (16, 2, 64, 16, 1), (17, 1, 65, 5, 1), (33, 3, 130, 16, 2), (40, 2, 24, 8, 3),
        (50, 1, 64, 4, 1), (31, 2, 72, 33, 1), (20, 1, 40, 64, 1), (48, 2, 256, 16, 2), (64, 1, 9, 32, 1)]


def check_scan(v, soft=True, dout=None, dnew=None):
    names = [k for k, t in v.items() if t is not None and k != "starts"]
    leaves = {k: v[k].detach().requires_grad_() for k in names}
    out, new = seq.ssm_scan(**{**v, **leaves}, delta_softplus=soft, return_state=True)
    T, R, D = v["u"].shape
    N = v["A"].shape[1]
    loss = [(out, dout)] + ([(new, dnew)] if dnew is not None else [])
    grads = dict(zip(names, torch.autograd.grad([a for a, _ in loss], list(leaves.values()), [b for _, b in loss])))
    kw = dict(soft=soft, dout=dout, dnew=dnew)
    want_out, want_new, want = ref.scan(**v, **kw)
    size_out, size_new, size = ref.scan(**v, **kw, absolute=True)
    ref.assert_close("out", out, want_out, size_out, ref.scan_chain(T, R, D, N, False))
    ref.assert_close("new", new, want_new, size_new, ref.scan_chain(T, R, D, N, False))
    for k in names:
        assert grads[k].dtype == v[k].dtype
        ref.assert_close(k, grads[k], want[k], size[k], ref.scan_chain(T, R, D, N, True))
    return out, new, grads


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("T,R,D,N,G", SCAN)
@pytest.mark.parametrize("full", [False, True], ids=["bare", "full"])
def test_ssm_scan(T, R, D, N, G, dtype, full):
    need_gpu()
    v = scan_inputs(T, R, D, N, G, dtype, 11, "cuda", starts=full, state=full, gate=full)
    if not full:
        v["D"] = v["delta_bias"] = None
    g = gen(12)
    check_scan(v, True, torch.randn((T, R, D), generator=g).to(dtype).cuda(),
               torch.randn((R, D, N), generator=g).cuda() if full else None)


@gpu
def test_ssm_scan_without_softplus_and_with_one_named_group():
    need_gpu()
    v = scan_inputs(20, 2, 48, 16, 1, torch.float32, 13, "cuda", state=True, grouped=True)
    v["delta"], v["delta_bias"] = v["delta"].abs(), None
    check_scan(v, False, torch.randn((20, 2, 48), generator=gen(14)).cuda())


@gpu
@pytest.mark.parametrize("T,R,D,N,dtype", [(1000, 1, 64, 16, torch.float32), (517, 2, 70, 5, torch.bfloat16), (2100, 1, 16, 4, torch.float32)])
@pytest.mark.parametrize("starts", [False, True])
def test_ssm_scan_long(T, R, D, N, dtype, starts):
    """Few rows and many steps: the time axis is split into chunks."""
    need_gpu()
    v = scan_inputs(T, R, D, N, 1, dtype, 15, "cuda", state=True)
    if starts:
        v["starts"] = (torch.rand((T, R), generator=gen(16)) < 0.004).cuda()
    g = gen(17)
    check_scan(v, True, torch.randn((T, R, D), generator=g).to(dtype).cuda(), torch.randn((R, D, N), generator=g).cuda())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS.get)
def test_strides_and_alignment(dtype):
    """Row-major storage, cut-out channels at odd offsets, and gradients given in other strides give
    what packed tensors give."""
    need_gpu()
    T, R, D, N, W = 37, 3, 40, 16, 4
    v = scan_inputs(T, R, D, N, 1, dtype, 21, "cuda", starts=True, state=True)
    c = conv_inputs(T, R, D, W, dtype, 22, "cuda", starts=True, state=True)

    def odd(t):  # a view at an odd offset inside a wider buffer, rows first
        if t is None or t.dim() < 3 or t.shape[:2] != (T, R):
            return t
        wide = torch.empty((R, T, *t.shape[2:-1], t.shape[-1] + 3), dtype=t.dtype, device=t.device)
        view = wide[..., 1:1 + t.shape[-1]].transpose(0, 1)
        view.copy_(t)
        return view

    dout = torch.randn((T, R, D), generator=gen(23)).to(dtype).cuda()
    for fn, args, kw in ((seq.ssm_scan, v, {}), (seq.short_conv, c, dict(activation="silu"))):
        got = []
        for change in (lambda t: t, odd, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t is not None and t.shape[:2] == (T, R) else t):
            leaves = {k: change(t).detach().requires_grad_() if t is not None and k != "starts" else change(t) for k, t in args.items()}
            out, new = fn(**leaves, **kw, return_state=True)
            names = [k for k in leaves if k != "starts"]
            grads = torch.autograd.grad(out, [leaves[k] for k in names], change(dout))
            got.append([out, new, *grads])
        for other in got[1:]:
            for a, b in zip(got[0], other):
                assert torch.equal(a, b)


@gpu
def test_broadcast_gradient_and_expanded_inputs():
    """out.sum() hands an expanded gradient back; an input expanded over rows is read with a stride of 0."""
    need_gpu()
    v = scan_inputs(9, 1, 32, 8, 1, torch.float32, 24, "cuda")
    wide = {k: t.expand(9, 4, *t.shape[2:]) if t is not None and k in ("u", "delta", "B", "C", "z") else t for k, t in v.items()}
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    out = seq.ssm_scan(**{k: leaves[k].expand(9, 4, *t.shape[2:]) if t is not None and k in ("u", "delta", "B", "C", "z") else leaves.get(k)
                          for k, t in v.items()})
    grads = torch.autograd.grad(out.sum(), list(leaves.values()))
    _, _, want = ref.scan(**wide, dout=torch.ones(9, 4, 32))
    _, _, size = ref.scan(**wide, dout=torch.ones(9, 4, 32), absolute=True)
    for k, g in zip(leaves, grads):
        w, s = (x.sum(1, keepdim=True) if k in ("u", "delta", "B", "C", "z") else x for x in (want[k], size[k]))
        ref.assert_close(k, g, w, s, ref.scan_chain(9, 4, 32, 8, True) + 4)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS.get)
@pytest.mark.parametrize("R,D,N,G", [(1, 1, 1, 1), (2, 128, 16, 1), (5, 66, 16, 2), (3, 7, 5, 1), (4, 33, 64, 1), (3, 20, 8, 1), (2, 9, 12, 3), (70, 8, 4, 1), (2, 16, 32, 1)])
def test_steps_match_the_sequences(R, D, N, G, dtype):
    """Steps in turn give the references' values, and the states that the sequence forms end with."""
    need_gpu()
    T, W = 6, 4
    v = scan_inputs(T, R, D, N, G, dtype, 31, "cuda", starts=True, state=True)
    c = conv_inputs(T, R, D, W, dtype, 32, "cuda", starts=True, state=True)
    state, cstate = v["state"].clone(), c["state"].clone()
    ys, cs = [], []
    for t in range(T):
        at = {k: (x[t] if x is not None and k in ("u", "delta", "B", "C", "z", "starts") else x) for k, x in v.items()}
        ys.append(seq.ssm_step(**{**at, "state": state}))
        cs.append(seq.short_conv_step(c["x"][t], cstate, c["weight"], c["bias"], starts=c["starts"][t], activation="silu"))
    want, h, _ = ref.scan(**v)
    size, hsize, _ = ref.scan(**v, absolute=True)
    k = ref.scan_chain(T, R, D, N, False)
    ref.assert_close("steps", torch.stack(ys), want, size, k)
    ref.assert_close("state", state, h, hsize, k)
    out, new = seq.short_conv(**c, activation="silu", return_state=True)
    assert torch.equal(torch.stack(cs), out) and torch.equal(cstate, new)


@gpu
def test_nothing_crosses_a_start():
    """NaN and infinity in an episode, in the given state and in the gradient handed back stay in their
    episode: the other one's values and gradients are those of inputs without them."""
    need_gpu()
    T, R, D, N = 40, 2, 64, 16
    v = scan_inputs(T, R, D, N, 1, torch.float32, 41, "cuda", state=True)
    c = conv_inputs(T, R, D, 4, torch.float32, 42, "cuda", state=True)
    starts = torch.zeros((T, R), dtype=torch.bool, device="cuda")
    starts[20] = True
    for args, fn, timed, kw in ((v, seq.ssm_scan, ("u", "delta", "B", "C", "z"), {}), (c, seq.short_conv, ("x",), dict(activation="silu"))):
        args["starts"] = starts
        main = timed[0]
        dout = torch.randn((T, R, D), generator=gen(43)).cuda()
        res = []
        for poison in (False, True):
            w = {k: None if t is None else t.clone() for k, t in args.items()}
            if poison:
                w[main][3] = float("nan")
                w[main][5] = float("inf")
                w["state"][:] = float("nan")
            w[main].requires_grad_()
            out = fn(**w, **kw)
            d = dout.clone()
            (g,) = torch.autograd.grad(out, w[main], d)
            res.append((out[20:], g[20:]))
        assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
        # and a gradient that is not a number in the later episode leaves the earlier one's alone
        w = {k: None if t is None else t.clone() for k, t in args.items()}
        w[main].requires_grad_()
        d = dout.clone()
        (clean,) = torch.autograd.grad(fn(**w, **kw), w[main], d)
        d[25:] = float("nan")
        (g,) = torch.autograd.grad(fn(**w, **kw), w[main], d)
        assert torch.equal(g[:20], clean[:20]) and torch.isnan(g[25:]).all()


@gpu
def test_empty_sequences_and_rows():
    need_gpu()
    for T, R in ((0, 3), (4, 0), (0, 0)):
        v = scan_inputs(T, R, 8, 4, 1, torch.float32, 51, "cuda", state=True, starts=True)
        leaves = {k: t.detach().requires_grad_() if t is not None and k != "starts" else t for k, t in v.items()}
        out, new = seq.ssm_scan(**leaves, return_state=True)
        assert out.shape == (T, R, 8) and (torch.equal(new, v["state"]) if T == 0 else new.shape == (R, 8, 4))
        names = [k for k in leaves if k != "starts"]
        grads = dict(zip(names, torch.autograd.grad([out, new], [leaves[k] for k in names], [torch.ones_like(out), torch.full_like(new, 3.0)])))
        assert torch.equal(grads["state"], torch.full_like(new, 3.0))
        assert all(not grads[k].any() for k in names if k != "state")
        c = conv_inputs(T, R, 8, 4, torch.float32, 52, "cuda", state=True, starts=True)
        leaves = {k: t.detach().requires_grad_() if k != "starts" else t for k, t in c.items()}
        out, new = seq.short_conv(**leaves, return_state=True)
        assert out.shape == (T, R, 8) and torch.equal(new, c["state"])
        grads = torch.autograd.grad([out, new], [leaves[k] for k in ("x", "weight", "bias", "state")], [torch.ones_like(out), torch.full_like(new, 3.0)])
        assert not grads[1].any() and not grads[2].any() and torch.equal(grads[3], torch.full_like(new, 3.0))


@gpu
def test_results_repeat_bit_for_bit_and_on_another_stream():
    need_gpu()
    v = scan_inputs(70, 3, 200, 16, 1, torch.bfloat16, 61, "cuda", starts=True, state=True)
    dout = torch.randn((70, 3, 200), generator=gen(62)).bfloat16().cuda()

    def once():
        leaves = {k: t.detach().requires_grad_() if k != "starts" else t for k, t in v.items()}
        out = seq.ssm_scan(**leaves)
        return [out, *torch.autograd.grad(out, [leaves[k] for k in leaves if k != "starts"], dout)]

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = once()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@gpu
def test_captured_training_step_and_steps_replay():
    """Forward, backward and single steps captured into graphs and replayed several times, with eager
    work between, against the eager results."""
    need_gpu()
    T, R, D, N = 30, 2, 48, 16
    v = scan_inputs(T, R, D, N, 1, torch.float32, 71, "cuda", starts=True, state=True)
    c = conv_inputs(T, R, D, 4, torch.float32, 72, "cuda", starts=True, state=True)
    dout = torch.randn((T, R, D), generator=gen(73)).cuda()
    state, cstate = v["state"].clone(), c["state"].clone()

    def train():
        leaves = {k: t.detach().requires_grad_() if k != "starts" else t for k, t in v.items()}
        x = c["x"].detach().requires_grad_()
        y = seq.short_conv(x, c["weight"], c["bias"], c["state"], c["starts"], "silu")
        out = seq.ssm_scan(**{**leaves, "u": y})
        return [out, *torch.autograd.grad(out, [x] + [leaves[k] for k in leaves if k not in ("starts", "u")], dout)]

    def step():
        y = seq.short_conv_step(c["x"][0], cstate, c["weight"], c["bias"], starts=c["starts"][0], activation="silu")
        return seq.ssm_step(state, y, v["delta"][0], v["A"], v["B"][0], v["C"][0], D=v["D"], z=v["z"][0], delta_bias=v["delta_bias"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for fn in (train, step):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = fn()
        graphs.append((g, got))
    for k in range(4):
        with torch.no_grad():
            c["x"].add_(0.25)
            v["delta"].mul_(0.9)
        want = train()
        at = state.clone(), cstate.clone()
        want_step = step()
        after = state.clone(), cstate.clone()
        state.copy_(at[0])
        cstate.copy_(at[1])
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, graphs[0][1]):
            assert torch.equal(a, b), k
        assert torch.equal(want_step, graphs[1][1]) and torch.equal(state, after[0]) and torch.equal(cstate, after[1])


@gpu
def test_a_chain_of_both_matches_the_references():
    """The operators as a memory uses them, one after the other, over two calls that hand the states on:
    the same as one call over the whole sequence."""
    need_gpu()
    T, R, D, N = 50, 3, 64, 16
    v = scan_inputs(T, R, D, N, 1, torch.float32, 81, "cuda", starts=True, state=True)
    c = conv_inputs(T, R, D, 4, torch.float32, 82, "cuda", starts=True, state=True)
    v["starts"] = c["starts"]

    def chain(a, b, state, cstate):
        cut = lambda x: None if x is None else x[a:b]  # noqa: E731
        y, cs = seq.short_conv(c["x"][a:b], c["weight"], c["bias"], cstate, c["starts"][a:b], "silu", return_state=True)
        out, s = seq.ssm_scan(y, cut(v["delta"]), v["A"], cut(v["B"]), cut(v["C"]), D=v["D"], z=cut(v["z"]),
                              delta_bias=v["delta_bias"], state=state, starts=cut(v["starts"]), return_state=True)
        return out, s, cs

    whole = chain(0, T, v["state"], c["state"])
    first = chain(0, 23, v["state"], c["state"])
    second = chain(23, T, first[1], first[2])
    _, cnew, _ = ref.conv(**c)
    y = seq.short_conv(**c, activation="silu")  # the convolution's own error is test_short_conv's matter
    want, h, _ = ref.scan(**{**v, "u": y})
    size, hs, _ = ref.scan(**{**v, "u": y}, absolute=True)
    k = ref.scan_chain(T, R, D, N, False)
    for out, s, cs in (whole, (torch.cat([first[0], second[0]]), second[1], second[2])):
        ref.assert_close("out", out, want, size, k)
        ref.assert_close("state", s, h, hs, k)
        assert torch.equal(cs.double().cpu(), cnew)


@gpu
@pytest.mark.parametrize("R,D,N,G", [(70, 130, 16, 1), (100, 130, 12, 1), (200, 80, 16, 2), (260, 64, 5, 1)])
def test_ssm_scan_many_rows(R, D, N, G):
    """Row counts on both sides of the launch's choices: one block a compute unit and more."""
    need_gpu()
    T = 21
    v = scan_inputs(T, R, D, N, G, torch.float32, 91, "cuda", starts=True, state=True)
    g = gen(92)
    check_scan(v, True, torch.randn((T, R, D), generator=g).cuda(), torch.randn((R, D, N), generator=g).cuda())


@gpu
@pytest.mark.parametrize("N", [3, 8, 12, 16, 17, 40, 64])
@pytest.mark.parametrize("T", [63, 64, 65, 129, 300])
def test_ssm_scan_chunk_edges(T, N):
    """Lengths around the chunks and tiles a split time axis has, for every way the states are shared."""
    need_gpu()
    v = scan_inputs(T, 2, 70, N, 1, torch.float32, 93, "cuda", state=True)
    v["starts"] = (torch.rand((T, 2), generator=gen(94)) < 0.02).cuda()
    g = gen(95)
    check_scan(v, True, torch.randn((T, 2, 70), generator=g).cuda(), torch.randn((2, 70, N), generator=g).cuda())


@gpu
@pytest.mark.parametrize("N", [9, 16])
@pytest.mark.parametrize("T", [1, 31, 32, 33, 95, 191, 193, 225, 352])
def test_ssm_scan_around_the_split_of_16_states(T, N):
    """Lengths around whole tiles of the unsplit form of 9 to 16 states, and around those where it splits."""
    need_gpu()
    v = scan_inputs(T, 3, 100, N, 1, torch.bfloat16, 131, "cuda", state=True)
    v["starts"] = (torch.rand((T, 3), generator=gen(132)) < 0.02).cuda()
    g = gen(133)
    check_scan(v, True, torch.randn((T, 3, 100), generator=g).bfloat16().cuda(), torch.randn((3, 100, N), generator=g).cuda())


@gpu
@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("R,D,dtype", [(1500, 2048, torch.bfloat16), (700, 1028, torch.float32), (4200, 516, torch.float16), (9, 3001, torch.float32),
                                       (11, 1030, torch.bfloat16)])
def test_short_conv_many_rows_and_every_width_of_access(T, R, D, dtype):
    """More rows than the blocks take at once, and channels that 8, 4, 2 or 1 of them a thread divide; the
    step's form against the sequence's, whose first step it is."""
    need_gpu()
    c = conv_inputs(T, R, D, 4, dtype, 141, "cuda", starts=True, state=True)
    out, new = seq.short_conv(**c, activation="silu", return_state=True)
    want, want_new = ref.conv(**c)[:2]
    ref.assert_close("out", out, want, ref.conv(**c, absolute=True)[0], 4 + 20)
    assert torch.equal(new.double().cpu(), want_new)
    state = c["state"].clone()
    for t in range(T):
        y = seq.short_conv_step(c["x"][t], state, c["weight"], c["bias"], starts=c["starts"][t], activation="silu")
        assert torch.equal(y, out[t])
    assert torch.equal(state, new)


@gpu
@pytest.mark.parametrize("G", [1, 2])
@pytest.mark.parametrize("D,N,T", [(132, 16, 70), (130, 16, 70), (268, 5, 40), (262, 16, 400), (136, 33, 40)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS.get)
def test_ssm_scan_every_width_of_access(D, N, T, G, dtype):
    """Channels whose rows are aligned to 16, 8 or 4 B, in groups that end inside them."""
    need_gpu()
    v = scan_inputs(T, 3, D, N, G, dtype, 151, "cuda", state=True, starts=True)
    g = gen(152)
    check_scan(v, True, torch.randn((T, 3, D), generator=g).to(dtype).cuda(), torch.randn((3, D, N), generator=g).cuda())


@gpu
def test_strides_past_32_bits():
    """Steps that lie more than 2^31 elements apart."""
    need_gpu()
    far = 2 ** 31 + 64
    T, R, D, N = 3, 2, 64, 16
    big = torch.empty(2 * far + 8 * R * (D + N), dtype=torch.bfloat16, device="cuda")

    def place(t, at):
        view = big.as_strided((T, *t.shape[1:]), (far, *t[0].stride()), at)
        view.copy_(t)
        return view

    v = scan_inputs(T, R, D, N, 1, torch.bfloat16, 101, "cuda", state=True, starts=True)
    c = conv_inputs(T, R, D, 4, torch.bfloat16, 102, "cuda", state=True, starts=True)
    dout = torch.randn((T, R, D), generator=gen(103)).bfloat16().cuda()
    w, at = dict(v), 0
    for k in ("u", "delta", "z", "B", "C"):
        w[k] = place(v[k], at)
        at += v[k][0].numel()
    cw = dict(c, x=place(c["x"], at))
    for fn, a, b, kw in ((seq.ssm_scan, v, w, {}), (seq.short_conv, c, cw, dict(activation="silu"))):
        got = []
        for args in (a, b):
            leaves = {k: t.detach().requires_grad_() if k != "starts" else t for k, t in args.items()}
            out, new = fn(**leaves, **kw, return_state=True)
            got.append([out, new, *torch.autograd.grad(out, [leaves[k] for k in leaves if k != "starts"], dout)])
        for x, y in zip(*got):
            assert torch.equal(x, y)


@gpu
def test_steps_in_inference_mode_and_a_saved_state_that_was_renewed():
    need_gpu()
    v = scan_inputs(1, 2, 16, 4, 1, torch.float32, 111, "cuda", state=True)
    at = {k: (t[0] if t is not None and k in ("u", "delta", "B", "C", "z") else t) for k, t in v.items()}
    c = conv_inputs(1, 2, 16, 4, torch.float32, 112, "cuda", state=True)
    with torch.inference_mode():
        state, cstate = v["state"].clone(), c["state"].clone()
        y = seq.ssm_step(**{**at, "state": state})
        seq.short_conv_step(c["x"][0], cstate, c["weight"], c["bias"])
    assert torch.isfinite(y).all() and not torch.equal(state, v["state"])
    u = v["u"].clone().requires_grad_()
    out = seq.ssm_scan(**{**v, "u": u})
    seq.ssm_step(**at)  # renews the state that the scan saved
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_nodes_are_noted_while_a_graph_holds_them(monkeypatch):
    """The bookkeeping behind the refusal below, without a device: an eager forward's node is seen from
    another stream's capture while its graph lives, and goes with it."""
    stream = [1]
    monkeypatch.setattr(seq.torch.cuda, "current_stream", lambda device=None: type("S", (), {"cuda_stream": stream[0]}))

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            seq._lives(ctx)
            return x * 2

        @staticmethod
        def backward(ctx, g):
            return g * 2, None

    leaf, other = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    out = Twice.apply(leaf, torch.ones(3))
    seq._refuse_held(leaf)  # the same stream
    stream[0] = 2
    seq._refuse_held(None, other, torch.ones(3), other * 2)
    with pytest.raises(RuntimeError, match="no eager autograd graph"):
        seq._refuse_held(other, leaf)
    out = (out * 3).sum()
    with pytest.raises(RuntimeError, match="no eager autograd graph"):
        seq._refuse_held(leaf)
    out.backward()
    with pytest.raises(RuntimeError, match="no eager autograd graph"):
        seq._refuse_held(leaf)  # a graph that has run its backward still holds the leaf
    del out
    seq._refuse_held(leaf)


def test_nodes_are_found_behind_other_operations(monkeypatch):
    """The same where the leaves feed the operators through torch's own: A = -exp(A_log), a projection."""
    stream = [1]
    monkeypatch.setattr(seq.torch.cuda, "current_stream", lambda device=None: type("S", (), {"cuda_stream": stream[0]}))

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            seq._lives(ctx)
            return x * 2

        @staticmethod
        def backward(ctx, g):
            return g * 2, None

    a_log, other = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    out = Twice.apply(-torch.exp(a_log), other.detach())
    stream[0] = 2
    seq._refuse_held(other, -torch.exp(other))
    for t in (a_log, -torch.exp(a_log), (other * a_log).sum()):
        with pytest.raises(RuntimeError, match="no eager autograd graph"):
            seq._refuse_held(other, t)
    del out
    seq._refuse_held(a_log, -torch.exp(a_log))


@gpu
def test_capture_refuses_leaves_that_an_eager_graph_holds():
    need_gpu()
    v = scan_inputs(5, 2, 16, 4, 1, torch.float32, 121, "cuda")
    leaves = {k: t.detach().requires_grad_() if t is not None and k != "starts" else t for k, t in v.items()}
    dout = torch.ones((5, 2, 16), device="cuda")

    def train():
        out = seq.ssm_scan(**leaves)
        return torch.autograd.grad(out, [t for t in leaves.values() if t is not None], dout)

    held = seq.ssm_scan(**leaves)  # an eager graph that goes on living
    torch.cuda.synchronize()
    count = torch.zeros(1, device="cuda")
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        count.add_(1)
        with pytest.raises(RuntimeError, match="no eager autograd graph"):
            seq.ssm_scan(**leaves)
    del held
    want = train()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = train()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def tangent_calls(device):
    """Each operator with one of its inputs a dual tensor, by name."""
    v = scan_inputs(4, 2, 6, 5, 1, torch.float32, 161, device, state=True, starts=True)
    c = conv_inputs(4, 2, 6, 4, torch.float32, 162, device, state=True, starts=True)
    at = {k: (t[0] if k in ("u", "delta", "B", "C", "z", "starts") else t) for k, t in v.items()}
    cat = {k: (t[0] if k in ("x", "starts") else t) for k, t in c.items()}
    for fn, args in ((seq.ssm_scan, v), (seq.ssm_step, at), (seq.short_conv, c), (seq.short_conv_step, cat)):
        for k in args:
            if k != "starts":
                yield fn, args, k


def test_forward_mode_derivatives_are_refused():
    """Raised before anything runs, so without a device too; an input without a tangent is none of its business."""
    from torch.autograd import forward_ad
    for fn, args, k in tangent_calls("cpu"):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(**{**args, k: dual})
            refuses(fn, "HIP device", **args)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: seq.short_conv(x, torch.ones(6, 4)), (torch.ones(4, 2, 6),), (torch.ones(4, 2, 6),))


@gpu
def test_a_level_of_forward_mode_alone_changes_nothing():
    need_gpu()
    from torch.autograd import forward_ad
    v = scan_inputs(4, 2, 6, 5, 1, torch.float32, 163, "cuda")
    with forward_ad.dual_level():
        again = seq.ssm_scan(**v)
        other = forward_ad.make_dual(torch.ones(3, device="cuda"), torch.ones(3, device="cuda")) * 2
    assert torch.equal(seq.ssm_scan(**v), again) and other is not None
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        seq.ssm_scan(**{**v, "u": forward_ad.make_dual(v["u"], torch.ones_like(v["u"]))})


LARGE = [0.0, 1e-30, 0.5, 1.0, 1.28, 5.0, 17.0, 20.0, 40.0, 80.0, 87.0, 87.5, 88.0, 89.0, 100.0, 127.5, 1e3, 6e4, 1e10, 1e30, 1e37, 3e38]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS.get)
def test_activations_of_large_values(dtype):
    """The convolution's activation and the scan's gate, and their slopes, from 1e-30 to the types' ends and of
    both signs. exp's argument is off by |x| 2 u, so its value by that much of itself; 1 - s is known to u,
    which the slope multiplies by x while s is not yet 1 (x < 17); a sigmoid below 2^-126 is 0, which costs at
    most 89 x 2^-126. The products and sums: 24 u as in test_short_conv."""
    need_gpu()
    x = torch.tensor([v for v in LARGE if v < torch.finfo(dtype).max])
    x = torch.cat([x, -x]).to(dtype)
    n = x.numel()
    d = x.double()
    s = 1 / (1 + torch.exp(-d))
    want, slope = torch.where(s > 0, d * s, 0.0), s * (1 + d * (1 - s))
    u, lost = 2.0 ** -24, 89 * 2.0 ** -126
    near = d.abs().clamp(max=100)
    err = (24 + 2 * near) * u * want.abs() + lost
    slope_err = (24 + 2 * near) * u * s * (1 + d.abs() * (1 - s)) + 2 * u * near * s * (d > 0) + lost

    def check(name, got, want, err):
        eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
        tiny = torch.finfo(dtype).smallest_normal * (torch.finfo(dtype).eps if dtype == torch.float16 else 1.0)
        off = (got.double().cpu() - want).abs()
        bad = ~(off <= err + eps * (want.abs() + err) + tiny)
        assert not bad.any(), (name, d[bad], got.double().cpu()[bad], want[bad])

    weight = torch.zeros((n, 4), device="cuda")
    weight[:, 3] = 1
    at = x.cuda()[None, None].requires_grad_()
    out = seq.short_conv(at, weight, activation="silu")
    (g,) = torch.autograd.grad(out, at, torch.ones_like(out))
    check("convolution", out[0, 0], want, err)
    check("its slope", g[0, 0], slope, slope_err)
    one, zero = torch.ones((1, 1, n), dtype=dtype, device="cuda"), torch.zeros((1, 1, 1), dtype=dtype, device="cuda")
    A, skip = -torch.ones((n, 1), device="cuda"), torch.ones(n, device="cuda")
    out = seq.ssm_scan(one, one, A, zero, zero, D=skip, z=at)
    (g,) = torch.autograd.grad(out, at, torch.ones_like(out))
    check("gate", out[0, 0], want, err)
    check("its slope", g[0, 0], slope, slope_err)
    y = seq.ssm_step(torch.zeros((1, n, 1), device="cuda"), one[0], one[0], A, zero[0], zero[0], D=skip, z=at.detach()[0])
    check("a step's gate", y[0], want, err)
    wide = at.detach().expand(40, 3, n).requires_grad_()  # several tiles and rows
    out = seq.ssm_scan(one.expand(40, 3, n), one.expand(40, 3, n), A, zero.expand(40, 3, 1), zero.expand(40, 3, 1), D=skip, z=wide)
    (g,) = torch.autograd.grad(out, wide, torch.ones_like(out))
    check("gate of a sequence", out, want.expand(40, 3, n), err)
    check("its slope", g, slope.expand(40, 3, n), slope_err)


def drifting(n):
    """A float32 constant whose n-fold sum, added up one by one in float32, drifts far from n times it."""
    import numpy as np
    c = np.linspace(0.1, 0.2, 257, dtype=np.float32)
    total = np.zeros_like(c)
    for _ in range(n):
        total += c
    off = np.abs(total.astype(np.float64) / (n * c.astype(np.float64)) - 1)
    return float(c[off.argmax()]), float(off.max())


@gpu
def test_short_conv_sums_long_sequences_in_short_chains():
    """dweight and dbias over 2^30 steps and rows, all adding the same: each thread adds at most 512 of them
    in float32 (511 roundings of half a unit, of sums no larger than the last), the rest is float64, with
    one rounding for a block's part and one at the end. Chains of 4,096, which these rows would make, drift further."""
    need_gpu()
    T, R, W = 4096, 262144, 4
    c, off = drifting(T)
    bound = 514 * 2.0 ** -24
    assert off > bound  # the input shows it
    x = torch.ones((1, 1, 1), device="cuda").expand(T, R, 1)
    weight, bias = torch.ones((1, W), device="cuda", requires_grad=True), torch.zeros(1, device="cuda", requires_grad=True)
    out = seq.short_conv(x, weight, bias)
    dout = torch.full((1, 1, 1), c, device="cuda").expand(T, R, 1)
    dw, db = torch.autograd.grad(out, (weight, bias), dout)
    value = float(torch.tensor(c))
    want = torch.tensor([value * R * (T - W + 1 + k) for k in range(W)], dtype=torch.float64)
    assert float((dw.double().cpu()[0] / want - 1).abs().max()) <= bound
    assert abs(float(db) / (value * R * T) - 1) <= bound


@gpu
def test_ssm_scan_sums_long_sequences_in_short_chains():
    """dA, dD and ddelta_bias over 65,536 steps of 512 rows that all add nearly the same: at most 512 steps are
    added up in float32, the rest in float64. The 64-bit values: every row is the same, and once the states have
    settled (exp(-0.5) a step at the slowest) each step adds the same again. dD's terms are exact: 514 u as for
    the convolution. A term of dA or ddelta_bias has two states that have settled, each off by at most 12 u (a
    decay by (3 x 0.5 + 2) u, which 1 / (1 - a) = 2.5 makes 9, and two roundings a step), the slope, the products
    and the sum over 16 states: below 64 u."""
    need_gpu()
    T, R, N, short = 65536, 512, 16, 512
    c, off = drifting(T // 8)  # of the eight sums in turn that a row's steps make
    u = 2.0 ** -24
    assert off > 578 * u
    one = lambda x: torch.tensor([[[x]]], dtype=torch.float32)  # noqa: E731
    A, B, C = -torch.arange(1, N + 1, dtype=torch.float32)[None], torch.full((1, 1, N), 0.75), torch.linspace(0.5, 1.0, N)[None, None]
    skip, bias = torch.ones(1), torch.zeros(1)
    wants = []
    for t in (short - 1, short):
        far = lambda x: x.expand(t, 1, x.shape[2])  # noqa: E731
        wants.append(ref.scan(far(one(1.0)), far(one(0.5)), A, far(B), far(C), skip, None, bias, soft=False, dout=far(one(c)))[2])
    leaves = [x.cuda().requires_grad_() for x in (A, skip, bias)]
    far = lambda x: x.cuda().expand(T, R, x.shape[2])  # noqa: E731
    out = seq.ssm_scan(far(one(1.0)), far(one(0.5)), leaves[0], far(B), far(C), D=leaves[1], delta_bias=leaves[2], delta_softplus=False)
    grads = torch.autograd.grad(out, leaves, far(one(c)))
    for name, g, k in (("A", grads[0], 578), ("D", grads[1], 514), ("delta_bias", grads[2], 578)):
        want = (wants[1][name] + (T - short) * (wants[1][name] - wants[0][name])) * R
        rel = float((g.double().cpu() / want - 1).abs().max())
        assert rel <= k * u, (name, rel / u)


@gpu
@pytest.mark.parametrize("T,R,D,N", [(513, 520, 64, 16), (1030, 520, 3, 5), (1600, 2, 64, 16), (4200, 1, 70, 33)])
def test_ssm_scan_around_the_segments_of_its_sums(T, R, D, N):
    """Lengths past whole segments, with the time axis whole (many rows) and in chunks."""
    need_gpu()
    v = scan_inputs(T, R, D, N, 1, torch.float32, 171, "cuda", state=True)
    v["starts"] = (torch.rand((T, R), generator=gen(172)) < 0.01).cuda()
    g = gen(173)
    dout, dnew = torch.randn((T, R, D), generator=g).cuda(), torch.randn((R, D, N), generator=g).cuda()
    check_scan(v, True, dout, dnew)


@gpu
@pytest.mark.parametrize("N", [16, 1])
def test_a_step_of_more_rows_than_a_launch_has_threads(N):
    """2^32 threads and some (four states a thread, or a channel each): the same as the rows by themselves."""
    need_gpu()
    D = 64 if N == 16 else 256
    R = 2 ** 24 + 3
    if torch.cuda.mem_get_info()[0] < 120 * 2 ** 30:
        pytest.skip("needs 120 GiB of device memory")
    g = torch.Generator(device="cuda").manual_seed(181)
    r = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    u, delta, B, C = r(R, D), r(1, D).expand(R, D), r(R, N), r(R, N)
    A, state = -torch.rand((D, N), generator=g, device="cuda") - 0.5, torch.ones((R, D, N), device="cuda")
    y = seq.ssm_step(state, u, delta, A, B, C)
    for at in (slice(0, 5), slice(R // 2, R // 2 + 5), slice(2 ** 24 - 2, R)):
        alone = torch.ones((at.stop - at.start, D, N), device="cuda")
        same = torch.equal(y[at], seq.ssm_step(alone, u[at], delta[at], A, B[at], C[at])), torch.equal(state[at], alone)
        assert same == (True, True), at


def test_sequences_past_a_launchs_threads_are_refused_before_anything_runs():
    """No device is needed to hear it: nothing was launched."""
    import ctypes as C

    from marlsoccer import _native as N
    L = N.lib()
    many = 2 ** 27  # rows of 64 channels: 2^27 blocks of 256 threads
    io = N.MsScanIO(dtype=1, states=16, groups=1, steps=1, rows=many, channels=64, u=16, delta=16, B=16, C=16, A=16, out=16, workspace=16,
                    workspace_bytes=2 ** 62, dout=16, du=16, ddelta=16, dB=16, dC=16, dA=16, checkpoints=16)
    for fn in (L.ms_scan_forward, L.ms_scan_backward):
        assert fn(C.byref(io), None) == N.MS_ERR_INVALID_ARGUMENT and b"too large" in L.ms_sequence_last_error()


@gpu
@pytest.mark.parametrize("T,R,D,N,G,dtype", [(100, 2, 24, 16, 24, torch.float32), (300, 1, 63, 16, 3, torch.bfloat16), (70, 3, 127, 4, 1, torch.float16),
                                             (33, 2, 130, 8, 130, torch.float32), (3, 2, 1, 1, 1, torch.float32), (9, 600, 2, 2, 1, torch.bfloat16),
                                             (257, 3, 192, 16, 3, torch.bfloat16), (40, 2, 66, 20, 6, torch.float16)])
@pytest.mark.parametrize("every", [False, True], ids=["some starts", "all starts"])
def test_ssm_scan_odd_groups_and_every_step_a_start(T, R, D, N, G, dtype, every):
    """Groups of one channel and of odd numbers; starts of any non-zero value, expanded over the rows."""
    need_gpu()
    v = scan_inputs(T, R, D, N, G, dtype, 191, "cuda", starts=True, state=True, grouped=True)
    if every:
        v["starts"] = torch.full((T, 1), 255, dtype=torch.uint8, device="cuda").expand(T, R)
    g = gen(192)
    check_scan(v, True, torch.randn((T, R, D), generator=g).to(dtype).cuda(), torch.randn((R, D, N), generator=g).cuda())


@gpu
def test_only_the_states_gradient_and_a_graph_used_twice():
    need_gpu()
    T, R, D, N = 20, 2, 40, 16
    v = scan_inputs(T, R, D, N, 1, torch.float32, 193, "cuda", state=True)
    dnew = torch.randn((R, D, N), generator=gen(194)).cuda()
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    _, new = seq.ssm_scan(**{**v, **leaves}, return_state=True)
    names = ["u", "delta", "A", "B", "delta_bias", "state"]
    first = torch.autograd.grad(new, [leaves[k] for k in names], dnew, retain_graph=True)
    again = torch.autograd.grad(new, [leaves[k] for k in names], dnew)
    none = torch.zeros(T, R, D)
    want, size = (ref.scan(**v, dout=none, dnew=dnew, absolute=a)[2] for a in (False, True))
    for k, x, y in zip(names, first, again):
        assert torch.equal(x, y)
        ref.assert_close(k, x, want[k], size[k], ref.scan_chain(T, R, D, N, True))


@gpu
def test_calls_from_several_threads():
    """Each on its own stream, with gradients: the bits of a call by itself."""
    import threading
    need_gpu()
    v = scan_inputs(60, 3, 70, 16, 1, torch.float32, 195, "cuda", starts=True, state=True)
    c = conv_inputs(60, 3, 70, 4, torch.float32, 196, "cuda", starts=True, state=True)
    dout = torch.randn((60, 3, 70), generator=gen(197)).cuda()

    def once():
        leaves = {k: t.detach().requires_grad_() if k != "starts" else t for k, t in v.items()}
        x = c["x"].detach().requires_grad_()
        out = seq.ssm_scan(**{**leaves, "u": seq.short_conv(x, c["weight"], c["bias"], c["state"], c["starts"], "silu")})
        return [out, *torch.autograd.grad(out, [x, leaves["A"], leaves["B"]], dout)]

    want, wrong = once(), []
    torch.cuda.synchronize()

    def work():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = once()
                    stream.synchronize()
                    wrong.extend(i for i, (a, b) in enumerate(zip(want, got)) if not torch.equal(a, b))
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
